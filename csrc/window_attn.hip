// Causal attention with a sliding window and a few first tokens that stay
// visible, forward and backward (ops/attention.py).
//
// Row i of sequence b stands at position p = i + start_b and sees key j iff
//   j <= p < len_b  and  (p - j < W  or  j < S).
// A row outside its sequence (p < 0 or p >= len_b) is padding: output 0, no
// gradient.  Keys that no row of a block can see are never read; keys at or
// behind a sequence's length are read as zeros, whatever the memory holds.
//
// G query heads share a key / value head.  The kernels work on "rows"
// r = t G + g, all heads of a group in one list: K and V tiles are fetched
// once for the group, the gradients of a shared head are summed in the
// accumulators in a fixed order, and a single token's G rows fill a tile
// instead of G tiles of one row.
//
// All products are 32x32 tiles with 8 contraction elements a lane
// (v_mfma_f32_32x32x16 for 16-bit types, eight v_mfma_f32_32x32x2f32 for
// fp32: exact fp32 products, the same operand layout).  A wave owns 32 rows
// (keys in the key-gradient kernel), one per column of the accumulator: the
// transposed scores S^T = K Q^T put a row's keys into the registers of the
// two lanes (l, l + 32), so the softmax needs one exchange, the rescale of
// O^T is a factor per lane, and P^T is the next product's right operand
// without leaving its registers.  The contraction order of that product is
// the accumulator's own row order; the left operand (V^T, read transposed
// out of LDS) follows it.
#include "common.h"

#include "lm_ops.h"

#include <algorithm>
#include <type_traits>

namespace kfac {

namespace {

constexpr int NT = 256;      // 4 waves
constexpr int BM = 128;      // rows (or keys) of a block, 32 a wave
constexpr int BN = 64;       // streamed tile
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kInf = __builtin_inff();

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef short v8i16 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// x of lane l ^ 32
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

template <typename T> struct Ops;
template <> struct Ops<__bf16> {
  typedef v8bf frag;
  typedef v4bf quad;
  __device__ __forceinline__ static v16f mma(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Ops<_Float16> {
  typedef v8h frag;
  typedef v4h quad;
  __device__ __forceinline__ static v16f mma(frag a, frag b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct Ops<float> {
  typedef v8f frag;
  typedef v4f quad;
  __device__ __forceinline__ static v16f mma(frag a, frag b, v16f c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

template <typename T> constexpr int kUnit = 16 / (int)sizeof(T);  // elements of 16 bytes

// LDS row stride: rows 16 bytes past a multiple of 256 (or of 128) keep the
// 16-byte row reads of neighbouring rows on different banks
template <typename T, int DP> constexpr int kLd = DP + kUnit<T>;

// waves a SIMD that the row kernels and the key-gradient kernel leave
// registers for (256 a wave at 2, 512 at 1)
template <typename T, int DP> constexpr int kRowWaves = sizeof(T) == 2 || DP <= 64 ? 2 : 1;
template <typename T, int DP> constexpr int kKeyWaves = (sizeof(T) == 2 ? DP <= 64 : DP <= 32) ? 2 : 1;

// accumulator register e of lane half h is tile row (e & 3) + 8 (e >> 2) + 4 h
__device__ __forceinline__ int acc_row(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

__device__ __forceinline__ v4f quad_of(const v16f& x, int e4) {
  return v4f{x[e4 * 4], x[e4 * 4 + 1], x[e4 * 4 + 2], x[e4 * 4 + 3]};
}

__device__ __forceinline__ v4f add4(v4f a, v4f b) {
  return v4f{a[0] + b[0], a[1] + b[1], a[2] + b[2], a[3] + b[3]};
}

__device__ __forceinline__ v16f zero16() {
  v16f z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

// Left operand from rows: lane l holds row r0 + (l & 31), elements
// k0 + 8 (l >> 5) .. + 7 of a row-major LDS tile
template <typename T, int DP>
__device__ __forceinline__ typename Ops<T>::frag row_frag(const T* L, int r0, int k0) {
  const int l = threadIdx.x & 63;
  const T* p = L + (r0 + (l & 31)) * kLd<T, DP> + k0 + 8 * (l >> 5);
  typename Ops<T>::frag f;
  if constexpr (sizeof(T) == 2) {
    f = *reinterpret_cast<const typename Ops<T>::frag*>(p);
  } else {
    const v4f a = *reinterpret_cast<const v4f*>(p), b = *reinterpret_cast<const v4f*>(p + 4);
    f = v8f{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
  return f;
}

// Left operand from columns: lane l holds column c0 + (l & 31) of tile rows
// r0 + 4h + {0..3} and r0 + 8 + 4h + {0..3}: the order in which registers
// 8s .. 8s + 7 of an accumulator hold its rows (r0 = 16 s)
template <typename T, int DP>
__device__ __forceinline__ typename Ops<T>::frag col_frag(const T* L, int r0, int c0) {
  const int l = threadIdx.x & 63;
  if constexpr (sizeof(T) == 2) {
    // ds_read_b64_tr_b16: 16 lanes read 4 rows x 16 columns (lane 4q + p row
    // q, columns 4p ..) and get a column's 4 rows each
    const int i = l & 15, g = l >> 4;
    const T* p = L + (r0 + 4 * (g >> 1) + (i >> 2)) * kLd<T, DP> + c0 + 16 * (g & 1) + 4 * (i & 3);
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)p);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + 8 * kLd<T, DP>));
    const v8i16 f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(typename Ops<T>::frag, f);
  } else {
    const T* p = L + (r0 + 4 * (l >> 5)) * kLd<T, DP> + c0 + (l & 31);
    v8f f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = p[i * kLd<T, DP>];
      f[4 + i] = p[(8 + i) * kLd<T, DP>];
    }
    return f;
  }
}

// registers 8s .. 8s + 7 of an accumulator as a right operand, rounded once
// to the operands' type (16-bit probabilities and their gradients are the
// price of the matrix units; they are at most 2^-9 off relative each, and
// the sums over them stay in 32 bits)
template <typename T>
__device__ __forceinline__ typename Ops<T>::frag acc_frag(const v16f& a, int s) {
  v8f f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = a[8 * s + i];
  return __builtin_convertvector(f, typename Ops<T>::frag);
}

// 8 elements of a global row from element d on; zeros behind D (D % 8 == 0)
template <typename T>
__device__ __forceinline__ typename Ops<T>::frag global_frag(const T* row, int d, int D, bool ok) {
  typename Ops<T>::frag f;
  if (ok && d < D) {
    if constexpr (sizeof(T) == 2) {
      f = *reinterpret_cast<const typename Ops<T>::frag*>(row + d);
    } else {
      const v4f a = *reinterpret_cast<const v4f*>(row + d);
      const v4f b = *reinterpret_cast<const v4f*>(row + d + 4);
      f = v8f{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (T)0.f;
  }
  return f;
}

// a BN-row tile on its way from global memory through registers into LDS
template <typename T, int DP>
struct Tile {
  static constexpr int CR = DP / kUnit<T>;          // 16-byte chunks of a row
  static constexpr int CH = BN * CR / NT;           // chunks a thread
  static_assert(BN * CR % NT == 0, "tile");
  uint4 r[CH];

  // row_ptr(i): row i's address, or null where it is to be zeros
  template <typename F>
  __device__ __forceinline__ void load(F row_ptr, int D) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int id = threadIdx.x + c * NT;
      const int d = (id % CR) * kUnit<T>;
      const T* p = row_ptr(id / CR);
      r[c] = p != nullptr && d < D ? *reinterpret_cast<const uint4*>(p + d)
                                   : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void store(T* L) const {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int id = threadIdx.x + c * NT;
      *reinterpret_cast<uint4*>(L + (id / CR) * kLd<T, DP> + (id % CR) * kUnit<T>) = r[c];
    }
  }
};

struct Seq {
  int len, start;
};

// row -> (token, head of the group); a.Gmagic = floor(2^32 / G), so the
// product is the quotient or one less
struct Row {
  int t, g;
  __device__ __forceinline__ Row(int r, const AttnArgs& a) {
    t = (int)__umulhi((uint32_t)r, a.Gmagic);
    g = r - t * a.G;
    if (g >= a.G) {
      ++t;
      g -= a.G;
    }
  }
};

__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  Seq s;
  s.len = a.Tk;
  if (a.lengths != nullptr) {
    const int n = a.lengths[b];
    s.len = n < 0 ? 0 : (n < a.Tk ? n : a.Tk);
  }
  s.start = a.starts != nullptr ? a.starts[b] : (a.start_given ? a.start : s.len - a.Tq);
  return s;
}

// 64-bit: a start near the type's ends must not wrap into the sequence
__device__ __forceinline__ int position(int64_t t, const Seq& s) {
  const int64_t p = t + s.start;
  return p < 0 || p >= s.len ? -1 : (int)p;
}

// The keys that the positions [pmin, pmax] see, as tiles of BN: the sinks'
// tiles first, then the window's.
struct KeyTiles {
  int lo, hi;       // the window's keys
  int sinks, first, total;
  __device__ __forceinline__ KeyTiles(int pmin, int pmax, int W, int S) {
    lo = pmin - W + 1 > 0 ? pmin - W + 1 : 0;
    hi = pmax + 1;
    const int s = S < lo ? S : lo;
    sinks = (s + BN - 1) / BN;
    first = lo / BN > sinks ? lo / BN : sinks;
    const int end = (hi + BN - 1) / BN;
    total = sinks + (end > first ? end - first : 0);
  }
  __device__ __forceinline__ int key0(int it) const {
    return (it < sinks ? it : first + it - sinks) * BN;
  }
};

// first and last position of rows [r0, r1) that lie in the sequence; false:
// none does
__device__ __forceinline__ bool span(int r0, int r1, const AttnArgs& args, const Seq& s, int& pmin,
                                     int& pmax) {
  if (r1 <= r0 || s.len <= 0) return false;
  const int64_t a = (int64_t)Row(r0, args).t + s.start, b = (int64_t)Row(r1 - 1, args).t + s.start;
  if (b < 0 || a >= s.len) return false;
  pmin = (int)(a > 0 ? a : 0);
  pmax = (int)(b < s.len - 1 ? b : s.len - 1);
  return true;
}

__device__ __forceinline__ bool sees(int p, int j, int W, int S) {
  return j <= p && (p - j < W || j < S);
}

// what a run of rows sees of 32 keys from j0 on: 0 nothing, 2 all, 1 mixed
__device__ __forceinline__ int coverage(int pmin, int pmax, int j0, int W, int S) {
  const int j1 = j0 + 31;
  if (j0 > pmax || (pmin - j1 >= W && j0 >= S)) return 0;
  if (j1 <= pmin && (pmax - j0 < W || j1 < S)) return 2;
  return 1;
}

// scores that rows do not see become -inf: their probability is 0
template <bool KEYS_IN_REGS>
__device__ __forceinline__ void hide(v16f& s, int fixed, const int* others, int j0, int h, int W,
                                     int S) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int p = KEYS_IN_REGS ? fixed : others[acc_row(e, h)];
    const int j = KEYS_IN_REGS ? j0 + acc_row(e, h) : fixed;
    if (!sees(p, j, W, S)) s[e] = -kInf;
  }
}

// a row's 32 x ND accumulators as T (or fp32), times f
template <typename T, typename O, int ND>
__device__ __forceinline__ void put(O* out, const v16f (&x)[ND], float f, bool zero, int D, int h) {
  typedef O quad __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int dd = d * 32 + acc_row(e4 * 4, h);
      if (dd < D) {
        v4f v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = zero ? 0.f : x[d][e4 * 4 + i] * f;
        *reinterpret_cast<quad*>(out + dd) = __builtin_convertvector(v, quad);
      }
    }
}

// What a block of the row kernels (forward, dq) works on.
struct RowBlock {
  int b, hk, bh, r0, r, t, head, p, h, wave;
  int wmin, wmax, tiles;
  bool live, wany;
  Seq seq;
  __device__ __forceinline__ RowBlock(const AttnArgs& a) {
    bh = blockIdx.x;
    b = bh / a.Hkv;
    hk = bh - b * a.Hkv;
    const int rows = a.Tq * a.G;
    r0 = (int)(gridDim.y - 1 - blockIdx.y) * BM;  // longest rows first
    const int l = threadIdx.x & 63;
    wave = threadIdx.x >> 6;
    h = l >> 5;
    seq = sequence(a, b);
    r = r0 + wave * 32 + (l & 31);
    const Row rw(r, a);
    t = rw.t;
    head = hk * a.G + rw.g;
    live = r < rows;
    p = live ? position(t, seq) : -1;
    const int w0 = r0 + wave * 32;
    wmin = 0;
    wmax = -1;
    wany = span(w0, w0 + 32 < rows ? w0 + 32 : rows, a, seq, wmin, wmax);
  }
  __device__ __forceinline__ KeyTiles keys(const AttnArgs& a) {
    const int rows = a.Tq * a.G;
    int pmin = 0, pmax = -1;
    const bool any = span(r0, r0 + BM < rows ? r0 + BM : rows, a, seq, pmin, pmax);
    const KeyTiles kt(pmin, pmax, a.W, a.S);
    tiles = any ? kt.total : 0;
    return kt;
  }
};

// ---------------------------------------------------------------- forward
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(NT, (kRowWaves<T, DP>)) fwd_kernel(AttnArgs a) {
  constexpr int KD = DP / 16, ND = DP / 32, LD = kLd<T, DP>;
  typedef typename Ops<T>::frag frag;
  __shared__ __attribute__((aligned(16))) T Ks[2][BN * LD];
  __shared__ __attribute__((aligned(16))) T Vs[2][BN * LD];
  RowBlock w(a);
  const KeyTiles kt = w.keys(a);
  const int h = w.h;
  const float c = a.scale * kLog2e;
  int it0 = 0, it1 = w.tiles;
  if (SPLIT) {
    const int per = (it1 + a.splits - 1) / a.splits;
    it0 = per * (int)blockIdx.z < it1 ? per * (int)blockIdx.z : it1;
    it1 = it0 + per < it1 ? it0 + per : it1;
  }

  const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.qs[0] + w.head * a.qs[1] + w.t * a.qs[2];
  frag qf[KD];
#pragma unroll
  for (int k = 0; k < KD; ++k) qf[k] = global_frag<T>(q, k * 16 + 8 * h, a.D, w.p >= 0);

  v16f o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = zero16();
  float m = -kInf, sum = 0.f;

  const T* kb = reinterpret_cast<const T*>(a.k) + w.b * a.ks[0] + w.hk * a.ks[1];
  const T* vb = reinterpret_cast<const T*>(a.v) + w.b * a.vs[0] + w.hk * a.vs[1];
  Tile<T, DP> tk, tv;
  auto fetch = [&](int it) {
    const int j0 = kt.key0(it);
    auto ok = [&](int i) { return j0 + i < kt.hi && (j0 + i >= kt.lo || j0 + i < a.S); };
    tk.load([&](int i) { return ok(i) ? kb + (int64_t)(j0 + i) * a.ks[2] : nullptr; }, a.D);
    tv.load([&](int i) { return ok(i) ? vb + (int64_t)(j0 + i) * a.vs[2] : nullptr; }, a.D);
  };
  if (it0 < it1) fetch(it0);
  for (int it = it0; it < it1; ++it) {
    const int buf = (it - it0) & 1;
    tk.store(Ks[buf]);
    tv.store(Vs[buf]);
    __syncthreads();
    if (it + 1 < it1) fetch(it + 1);
    const int j0 = kt.key0(it);
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int js = j0 + sub * 32;
      const int cover = w.wany ? coverage(w.wmin, w.wmax, js, a.W, a.S) : 0;
      if (cover == 0) continue;
      v16f s = zero16();
#pragma unroll
      for (int k = 0; k < KD; ++k)
        s = Ops<T>::mma(row_frag<T, DP>(Ks[buf], sub * 32, k * 16), qf[k], s);
      if (cover == 1) hide<true>(s, w.p, nullptr, js, h, a.W, a.S);
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
      // c > 0: the maximum of the products is the product of the maximum
      mx = fmaxf(mx, other_half(mx)) * c;
      const float mn = fmaxf(m, mx);
      const float base = mn == -kInf ? 0.f : mn;
      const float alpha = ex2(m - base);
      m = mn;
      float add = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = ex2(__builtin_fmaf(s[e], c, -base));
        add += s[e];
      }
      sum = sum * alpha + add;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        const frag pf = acc_frag<T>(s, ss);
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[d] = Ops<T>::mma(col_frag<T, DP>(Vs[buf], sub * 32 + ss * 16, d * 32), pf, o[d]);
      }
    }
  }

  sum += other_half(sum);
  const bool none = w.p < 0 || sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  const float lse = none ? kInf : m + log2f(sum);
  if (!w.live) return;
  if (SPLIT) {
    const int64_t at = ((int64_t)blockIdx.z * gridDim.x + w.bh) * (a.Tq * a.G) + w.r;
    if (h == 0) a.lpart[at] = none ? -kInf : lse;
    put<T, float, ND>(a.opart + at * a.D, o, inv, none, a.D, h);
    return;
  }
  if (h == 0 && a.lse != nullptr) a.lse[((int64_t)w.b * a.Hq + w.head) * a.Tq + w.t] = lse;
  put<T, T, ND>(reinterpret_cast<T*>(a.out) + w.b * a.os[0] + w.head * a.os[1] + w.t * a.os[2], o,
                inv, none, a.D, h);
}

// Joins the key slices of a row: one block a row, 8 lanes groups of 32 (4
// elements of D a lane) walk every eighth slice, and the groups' sums are
// added in order.
template <typename T>
__global__ void __launch_bounds__(NT) join_kernel(AttnArgs a) {
  __shared__ float wts[256];
  __shared__ v4f part[8][32];
  __shared__ float red[NT / 64];
  const int rows = a.Tq * a.G;
  const int64_t row = blockIdx.x, all = (int64_t)a.B * a.Hkv * rows;
  const int tid = threadIdx.x;
  float lp = tid < a.splits ? a.lpart[tid * all + row] : -kInf;
  float m = lp;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float base = m == -kInf ? 0.f : m;
  // a slice that saw nothing has weight 0; one with a NaN keeps it
  wts[tid] = ex2(lp - base);
  __syncthreads();
  const int grp = tid >> 5, d = (tid & 31) * 4;
  v4f o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  for (int z = grp; z < a.splits; z += 8) {
    const float wt = wts[z];
    sum += wt;
    if (d < a.D) {
      const v4f x = *reinterpret_cast<const v4f*>(a.opart + (z * all + row) * a.D + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] += wt * x[i];
    }
  }
  part[grp][tid & 31] = o;
  __syncthreads();
  if (tid < 32) wts[tid] = 0.f;
  __syncthreads();
  if ((tid & 31) == 0) wts[grp] = sum;
  __syncthreads();
  if (tid >= 32) return;
  o = part[0][tid];
  sum = wts[0];
#pragma unroll
  for (int g = 1; g < 8; ++g) {
    sum += wts[g];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += part[g][tid][i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] *= inv;
  const int bh = (int)(row / rows), b = bh / a.Hkv;
  const Row rw((int)(row - (int64_t)bh * rows), a);
  const int head = (bh - b * a.Hkv) * a.G + rw.g;
  if (d < a.D)
    *reinterpret_cast<typename Ops<T>::quad*>(reinterpret_cast<T*>(a.out) + b * a.os[0] +
                                              head * a.os[1] + rw.t * a.os[2] + d) =
        __builtin_convertvector(o, typename Ops<T>::quad);
  if (tid == 0 && a.lse != nullptr)
    a.lse[((int64_t)b * a.Hq + head) * a.Tq + rw.t] = sum == 0.f ? kInf : base + log2f(sum);
}

// --------------------------------------------------------------- backward
// dq, and delta = do . o for the key-gradient kernel.  The forward's tiles
// and layout once more: S^T = K Q^T, dP^T = V dO^T, dS^T = P (dP - delta),
// dQ^T += K^T dS^T.
template <typename T, int DP>
__global__ void __launch_bounds__(NT, (kRowWaves<T, DP>)) dq_kernel(AttnArgs a) {
  constexpr int KD = DP / 16, ND = DP / 32, LD = kLd<T, DP>;
  typedef typename Ops<T>::frag frag;
  __shared__ __attribute__((aligned(16))) T Ks[2][BN * LD];
  __shared__ __attribute__((aligned(16))) T Vs[2][BN * LD];
  RowBlock w(a);
  const KeyTiles kt = w.keys(a);
  const int h = w.h, it1 = w.tiles;
  const float c = a.scale * kLog2e;

  const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.qs[0] + w.head * a.qs[1] + w.t * a.qs[2];
  const T* g =
      reinterpret_cast<const T*>(a.dout) + w.b * a.dos[0] + w.head * a.dos[1] + w.t * a.dos[2];
  const T* o = reinterpret_cast<const T*>(a.out) + w.b * a.os[0] + w.head * a.os[1] + w.t * a.os[2];
  frag qf[KD], gf[KD];
  float delta = 0.f;
#pragma unroll
  for (int k = 0; k < KD; ++k) {
    qf[k] = global_frag<T>(q, k * 16 + 8 * h, a.D, w.p >= 0);
    gf[k] = global_frag<T>(g, k * 16 + 8 * h, a.D, w.p >= 0);
    const frag of = global_frag<T>(o, k * 16 + 8 * h, a.D, w.p >= 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) delta += (float)gf[k][i] * (float)of[i];
  }
  delta += other_half(delta);
  const int64_t at = ((int64_t)w.b * a.Hq + w.head) * a.Tq + w.t;
  if (w.live && h == 0) a.delta[at] = delta;
  const float lse = w.p >= 0 ? a.lse[at] : kInf;

  v16f dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = zero16();
  const T* kb = reinterpret_cast<const T*>(a.k) + w.b * a.ks[0] + w.hk * a.ks[1];
  const T* vb = reinterpret_cast<const T*>(a.v) + w.b * a.vs[0] + w.hk * a.vs[1];
  Tile<T, DP> tk, tv;
  auto fetch = [&](int it) {
    const int j0 = kt.key0(it);
    auto ok = [&](int i) { return j0 + i < kt.hi && (j0 + i >= kt.lo || j0 + i < a.S); };
    tk.load([&](int i) { return ok(i) ? kb + (int64_t)(j0 + i) * a.ks[2] : nullptr; }, a.D);
    tv.load([&](int i) { return ok(i) ? vb + (int64_t)(j0 + i) * a.vs[2] : nullptr; }, a.D);
  };
  if (it1 > 0) fetch(0);
  for (int it = 0; it < it1; ++it) {
    const int buf = it & 1;
    tk.store(Ks[buf]);
    tv.store(Vs[buf]);
    __syncthreads();
    if (it + 1 < it1) fetch(it + 1);
    const int j0 = kt.key0(it);
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int js = j0 + sub * 32;
      const int cover = w.wany ? coverage(w.wmin, w.wmax, js, a.W, a.S) : 0;
      if (cover == 0) continue;
      v16f s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        s = Ops<T>::mma(row_frag<T, DP>(Ks[buf], sub * 32, k * 16), qf[k], s);
        dp = Ops<T>::mma(row_frag<T, DP>(Vs[buf], sub * 32, k * 16), gf[k], dp);
      }
      if (cover == 1) hide<true>(s, w.p, nullptr, js, h, a.W, a.S);
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = ex2(__builtin_fmaf(s[e], c, -lse)) * (dp[e] - delta);
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        const frag sf = acc_frag<T>(s, ss);
#pragma unroll
        for (int d = 0; d < ND; ++d)
          dq[d] = Ops<T>::mma(col_frag<T, DP>(Ks[buf], sub * 32 + ss * 16, d * 32), sf, dq[d]);
      }
    }
  }
  if (!w.live) return;
  put<T, T, ND>(reinterpret_cast<T*>(a.dq) + w.b * a.dqs[0] + w.head * a.dqs[1] + w.t * a.dqs[2],
                dq, a.scale, w.p < 0, a.D, h);
}

// Rows that look at the keys [k0, k0 + BM): the near ones, whose window
// reaches there, and, where the block holds sinks, the far ones behind them.
struct RowRange {
  int n0, n1, f1;  // near [n0, n1), far [n1, f1)
  __device__ __forceinline__ RowRange(int k0, const AttnArgs& a, const Seq& s) {
    const int64_t last = (int64_t)s.len - 1;        // last position
    const int64_t kend = k0 + BM - 1 < last ? k0 + BM - 1 : last;
    const int64_t near_end = kend + a.W - 1 < last ? kend + a.W - 1 : last;
    n0 = clip((int64_t)k0 - s.start, a) * a.G;
    n1 = clip(near_end + 1 - s.start, a) * a.G;
    if (k0 > last) n0 = n1 = 0;
    if (n1 < n0) n1 = n0;
    f1 = k0 < a.S && k0 <= last ? clip(last + 1 - s.start, a) * a.G : n1;
    if (f1 < n1) f1 = n1;
  }
  __device__ __forceinline__ static int clip(int64_t t, const AttnArgs& a) {
    return (int)(t < 0 ? 0 : (t < a.Tq ? t : a.Tq));
  }
};

constexpr int kSinkKeys = 32;  // keys of a far item

// fp32 sums of (group of sink keys, share) in AttnArgs::kvpart: share 0 from
// the near rows, 1 + i from chunk i of the far ones; [dk, dv][key][D]
__device__ __forceinline__ float* sink_part(const AttnArgs& a, int bh, int group, int share) {
  return a.kvpart + (((int64_t)bh * a.sink_groups + group) * (1 + a.far_chunks) + share) * 2 *
                        kSinkKeys * a.D;
}

// 64 rows of q and do, and their statistics
template <typename T, int DP>
struct RowTile {
  Tile<T, DP> q, g;
  float lse, delta;
  int p;
  __device__ __forceinline__ void load(const AttnArgs& a, const Seq& seq, int b, int hk, int t0,
                                       int end) {
    const T* qb = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + hk * a.G * a.qs[1];
    const T* gb = reinterpret_cast<const T*>(a.dout) + b * a.dos[0] + hk * a.G * a.dos[1];
    q.load([&](int i) {
      const Row r(t0 + i, a);
      return t0 + i < end ? qb + r.g * a.qs[1] + r.t * a.qs[2] : nullptr;
    }, a.D);
    g.load([&](int i) {
      const Row r(t0 + i, a);
      return t0 + i < end ? gb + r.g * a.dos[1] + r.t * a.dos[2] : nullptr;
    }, a.D);
    if (threadIdx.x < BN) {
      const int r = t0 + threadIdx.x;
      const Row rw(r, a);
      // rows outside the sequence have lse = +inf: P = 0
      p = r < end ? position(rw.t, seq) : -1;
      lse = kInf;
      delta = 0.f;
      if (p >= 0) {
        const int64_t at = ((int64_t)b * a.Hq + hk * a.G + rw.g) * a.Tq + rw.t;
        lse = a.lse[at];
        delta = a.delta[at];
      }
    }
  }
  __device__ __forceinline__ void store(T* Q, T* G, float* L, float* D, int* P) const {
    q.store(Q);
    g.store(G);
    if (threadIdx.x < BN) {
      L[threadIdx.x] = lse;
      D[threadIdx.x] = delta;
      P[threadIdx.x] = p;
    }
  }
};

// dk and dv: a wave owns 32 keys.  S = Q K^T and dP = dO V^T have a row's
// scores in register order, so dV^T += dO^T P and dK^T += Q^T dS take P and
// dS from where they are.
template <typename T, int DP>
struct KeyGrad {
  static constexpr int KD = DP / 16, ND = DP / 32;
  typedef typename Ops<T>::frag frag;
  frag kf[KD], vf[KD];
  v16f dk[ND], dv[ND];

  __device__ __forceinline__ void init(const AttnArgs& a, int b, int hk, int key, bool ok) {
    const int h = (threadIdx.x & 63) >> 5;
    const T* kp = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2];
    const T* vp = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2];
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      kf[k] = global_frag<T>(kp, k * 16 + 8 * h, a.D, ok);
      vf[k] = global_frag<T>(vp, k * 16 + 8 * h, a.D, ok);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();
  }

  // 32 rows from tile row i0 on
  __device__ __forceinline__ void rows(const AttnArgs& a, const T* Q, const T* G, const float* L,
                                       const float* D, const int* P, int i0, int key, int cover) {
    const int h = (threadIdx.x & 63) >> 5;
    const float c = a.scale * kLog2e;
    v16f s = zero16(), dp = zero16();
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      s = Ops<T>::mma(row_frag<T, DP>(Q, i0, k * 16), kf[k], s);
      dp = Ops<T>::mma(row_frag<T, DP>(G, i0, k * 16), vf[k], dp);
    }
    if (cover == 1) hide<false>(s, key, P + i0, 0, h, a.W, a.S);
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const v4f le = *reinterpret_cast<const v4f*>(L + i0 + acc_row(e4 * 4, h));
      const v4f de = *reinterpret_cast<const v4f*>(D + i0 + acc_row(e4 * 4, h));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e4 * 4 + i;
        s[e] = ex2(__builtin_fmaf(s[e], c, -le[i]));
        dp[e] = s[e] * (dp[e] - de[i]);
      }
    }
#pragma unroll
    for (int ss = 0; ss < 2; ++ss) {
      const frag pf = acc_frag<T>(s, ss), sf = acc_frag<T>(dp, ss);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        dv[d] = Ops<T>::mma(col_frag<T, DP>(G, i0 + ss * 16, d * 32), pf, dv[d]);
        dk[d] = Ops<T>::mma(col_frag<T, DP>(Q, i0 + ss * 16, d * 32), sf, dk[d]);
      }
    }
  }
};

// blockIdx.y < key_blocks: the near rows of 128 keys, 32 a wave, the rows
// streamed in tiles of 64.  Above: a chunk of the far rows of 32 sink keys,
// which all waves own together, 32 rows each of a tile of 128; their sums
// are added in wave order.  Sinks are few and the rows behind the window
// many, so a far item has its rows spread over the waves and not its keys.
template <typename T, int DP>
__global__ void __launch_bounds__(NT, (kKeyWaves<T, DP>)) dkv_kernel(AttnArgs a, int key_blocks) {
  constexpr int ND = DP / 32, LD = kLd<T, DP>;
  __shared__ __attribute__((aligned(16))) T Qs[2][BN * LD];
  __shared__ __attribute__((aligned(16))) T Gs[2][BN * LD];
  __shared__ __attribute__((aligned(16))) float Ls[2][BN], Ds[2][BN];
  __shared__ int Ps[2][BN];
  static_assert(2 * BN * LD * sizeof(T) >= kSinkKeys * DP * sizeof(float), "sums of a far item");
  const int bh = blockIdx.x, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, h = l >> 5;
  const Seq seq = sequence(a, b);
  RowTile<T, DP> tile;
  KeyGrad<T, DP> kg;

  if ((int)blockIdx.y >= key_blocks) {
    const int item = (int)blockIdx.y - key_blocks;
    const int group = item / a.far_chunks, chunk = item - group * a.far_chunks;
    const int j0 = group * kSinkKeys, key = j0 + (l & 31);
    const RowRange rr(j0 / BM * BM, a, seq);
    const int tiles = (rr.f1 - rr.n1 + BM - 1) / BM;
    const int per = (tiles + a.far_chunks - 1) / a.far_chunks;
    int ra = rr.n1 + per * chunk * BM, rb = ra + per * BM;
    if (rb > rr.f1) rb = rr.f1;
    kg.init(a, b, hk, key, key < seq.len);
    for (int t0 = ra; t0 < rb; t0 += BM) {
      __syncthreads();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        tile.load(a, seq, b, hk, t0 + half * BN, rb);
        tile.store(Qs[half], Gs[half], Ls[half], Ds[half], Ps[half]);
      }
      __syncthreads();
      const int s0 = t0 + wave * 32;
      int pmin, pmax;
      const int cover = span(s0, s0 + 32 < rb ? s0 + 32 : rb, a, seq, pmin, pmax)
                            ? coverage(pmin, pmax, j0, a.W, a.S) : 0;
      if (cover != 0)
        kg.rows(a, Qs[0], Gs[0], Ls[0], Ds[0], Ps[0], wave * 32, key, cover);
    }
    float* sk = reinterpret_cast<float*>(&Qs[0][0]);
    float* sv = reinterpret_cast<float*>(&Gs[0][0]);
    for (int turn = 0; turn < NT / 64; ++turn) {
      __syncthreads();
      if (wave == turn) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e4 = 0; e4 < 4; ++e4) {
            const int at = (l & 31) * DP + d * 32 + acc_row(e4 * 4, h);
            v4f fk = quad_of(kg.dk[d], e4), fv = quad_of(kg.dv[d], e4);
            if (turn > 0) {
              fk = add4(fk, *reinterpret_cast<const v4f*>(sk + at));
              fv = add4(fv, *reinterpret_cast<const v4f*>(sv + at));
            }
            *reinterpret_cast<v4f*>(sk + at) = fk;
            *reinterpret_cast<v4f*>(sv + at) = fv;
          }
      }
    }
    __syncthreads();
    float* part = sink_part(a, bh, group, 1 + chunk);
    for (int i = threadIdx.x; i < kSinkKeys * (DP / 4); i += NT) {
      const int kk = i / (DP / 4), d = i % (DP / 4) * 4;
      if (d >= a.D || j0 + kk >= a.S) continue;
      const v4f fk = *reinterpret_cast<const v4f*>(sk + kk * DP + d);
      *reinterpret_cast<v4f*>(part + kk * a.D + d) =
          v4f{fk[0] * a.scale, fk[1] * a.scale, fk[2] * a.scale, fk[3] * a.scale};
      *reinterpret_cast<v4f*>(part + (kSinkKeys + kk) * a.D + d) =
          *reinterpret_cast<const v4f*>(sv + kk * DP + d);
    }
    return;
  }

  const int k0 = (int)blockIdx.y * BM;
  const RowRange rr(k0, a, seq);
  const int key = k0 + wave * 32 + (l & 31);
  kg.init(a, b, hk, key, key < seq.len);
  if (rr.n0 < rr.n1) tile.load(a, seq, b, hk, rr.n0, rr.n1);
  int buf = 0;
  for (int t0 = rr.n0; t0 < rr.n1; t0 += BN, buf ^= 1) {
    tile.store(Qs[buf], Gs[buf], Ls[buf], Ds[buf], Ps[buf]);
    __syncthreads();
    if (t0 + BN < rr.n1) tile.load(a, seq, b, hk, t0 + BN, rr.n1);
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int s0 = t0 + sub * 32;
      int pmin, pmax;
      const int cover = span(s0, s0 + 32 < rr.n1 ? s0 + 32 : rr.n1, a, seq, pmin, pmax)
                            ? coverage(pmin, pmax, k0 + wave * 32, a.W, a.S) : 0;
      if (cover != 0)
        kg.rows(a, Qs[buf], Gs[buf], Ls[buf], Ds[buf], Ps[buf], sub * 32, key, cover);
    }
  }
  if (a.far_chunks > 0 && key < a.S) {
    float* part = sink_part(a, bh, key / kSinkKeys, 0) + key % kSinkKeys * a.D;
    put<T, float, ND>(part, kg.dk, a.scale, false, a.D, h);
    put<T, float, ND>(part + kSinkKeys * a.D, kg.dv, 1.f, false, a.D, h);
  } else if (key < a.Tk) {
    put<T, T, ND>(reinterpret_cast<T*>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2],
                  kg.dk, a.scale, false, a.D, h);
    put<T, T, ND>(reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2],
                  kg.dv, 1.f, false, a.D, h);
  }
}

// the shares of the sinks' gradients, summed in order
template <typename T>
__global__ void __launch_bounds__(NT) join_kv_kernel(AttnArgs a) {
  const int D4 = a.D / 4;
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (id >= (int64_t)a.B * a.Hkv * a.S * 2 * D4) return;
  const int d = (int)(id % D4) * 4;
  const int64_t rest = id / D4;
  const int which = (int)(rest & 1), key = (int)((rest >> 1) % a.S);
  const int bh = (int)((rest >> 1) / a.S), b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const float* part = sink_part(a, bh, key / kSinkKeys, 0) +
                      (which * kSinkKeys + key % kSinkKeys) * a.D + d;
  const int64_t step = (int64_t)2 * kSinkKeys * a.D;
  v4f f = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int ch = 0; ch <= a.far_chunks; ++ch) f = add4(f, *reinterpret_cast<const v4f*>(part + ch * step));
  T* out = which == 0
               ? reinterpret_cast<T*>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2]
               : reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2];
  *reinterpret_cast<typename Ops<T>::quad*>(out + d) =
      __builtin_convertvector(f, typename Ops<T>::quad);
}

unsigned row_blocks(const AttnArgs& a) {
  return (unsigned)ceil_div((int64_t)a.Tq * a.G, BM);
}

template <typename T, int DP>
void forward_dp(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.Hkv), row_blocks(a), (unsigned)a.splits);
  if (a.splits > 1) {
    fwd_kernel<T, DP, true><<<grid, NT, 0, st>>>(a);
    join_kernel<T><<<(unsigned)(a.B * a.Hq * a.Tq), NT, 0, st>>>(a);
  } else {
    fwd_kernel<T, DP, false><<<grid, NT, 0, st>>>(a);
  }
}

template <typename T, int DP>
void backward_dp(const AttnArgs& a, hipStream_t st) {
  const unsigned bh = (unsigned)(a.B * a.Hkv);
  dq_kernel<T, DP><<<dim3(bh, row_blocks(a)), NT, 0, st>>>(a);
  const int kb = (int)ceil_div(a.Tk, BM);
  dkv_kernel<T, DP><<<dim3(bh, (unsigned)(kb + a.sink_groups * a.far_chunks)), NT, 0, st>>>(a, kb);
  if (a.far_chunks > 0) {
    const int64_t n = (int64_t)bh * a.S * 2 * (a.D / 4);
    join_kv_kernel<T><<<(unsigned)ceil_div(n, NT), NT, 0, st>>>(a);
  }
}

template <typename T>
void forward_type(const AttnArgs& a, hipStream_t st) {
  if (a.D <= 32) forward_dp<T, 32>(a, st);
  else if (a.D <= 64) forward_dp<T, 64>(a, st);
  else if (a.D <= 96) forward_dp<T, 96>(a, st);
  else forward_dp<T, 128>(a, st);
}

template <typename T>
void backward_type(const AttnArgs& a, hipStream_t st) {
  if (a.D <= 32) backward_dp<T, 32>(a, st);
  else if (a.D <= 64) backward_dp<T, 64>(a, st);
  else if (a.D <= 96) backward_dp<T, 96>(a, st);
  else backward_dp<T, 128>(a, st);
}

}  // namespace

void attn_plan(const AttnArgs& a, int* splits, int64_t* floats) {
  const int64_t rows = (int64_t)a.Tq * a.G;
  const int64_t blocks = (int64_t)a.B * a.Hkv * ceil_div(rows, BM);
  // tiles that the longest row block can see
  const int64_t most = ceil_div(std::min<int64_t>((int64_t)a.W + BM, a.Tk), BN) +
                       ceil_div(std::min<int64_t>(a.S, a.Tk), BN) + 1;
  int64_t s = 1;
  if (blocks > 0 && blocks < 256) {
    s = ceil_div(1024, blocks);
    if (s > ceil_div(most, 4)) s = ceil_div(most, 4);
    if (s > 256) s = 256;
  }
  *splits = (int)s;
  *floats = s > 1 ? s * a.B * a.Hkv * rows * (a.D + 1) : 0;
}

void attn_forward(int dtype, const AttnArgs& a, hipStream_t st) {
  if ((int64_t)a.B * a.Hq * a.Tq == 0) return;
  if (dtype == kBF16) forward_type<__bf16>(a, st);
  else if (dtype == kF16) forward_type<_Float16>(a, st);
  else forward_type<float>(a, st);
}

void attn_bwd_plan(const AttnArgs& a, int* sink_groups, int* far_chunks, int64_t* floats) {
  *sink_groups = *far_chunks = 0;
  *floats = 0;
  // far rows exist only behind the window of a sink's key
  if (a.S <= 0 || a.W >= a.Tk) return;
  const int64_t groups = ceil_div(a.S, kSinkKeys), bh = (int64_t)a.B * a.Hkv;
  // chunks of at least two tiles until there are items for 4 blocks a CU
  int64_t ch = ceil_div(1024, bh * groups);
  ch = std::min(ch, ceil_div((int64_t)a.Tq * a.G, 2 * BM));
  ch = std::max<int64_t>(1, std::min<int64_t>(ch, 32));
  *sink_groups = (int)groups;
  *far_chunks = (int)ch;
  *floats = bh * groups * (1 + ch) * 2 * kSinkKeys * a.D;
}

void attn_backward(int dtype, const AttnArgs& a, hipStream_t st) {
  if ((int64_t)a.B * a.Hkv * a.Tk == 0 || a.Tq == 0) return;
  if (dtype == kBF16) backward_type<__bf16>(a, st);
  else if (dtype == kF16) backward_type<_Float16>(a, st);
  else backward_type<float>(a, st);
}

}  // namespace kfac

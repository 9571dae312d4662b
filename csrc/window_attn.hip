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

// accumulator register e of lane half h is tile row (e & 3) + 8 (e >> 2) + 4 h
__device__ __forceinline__ int acc_row(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

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
__device__ __forceinline__ bool span(int64_t r0, int64_t r1, int G, const Seq& s, int& pmin,
                                     int& pmax) {
  const int64_t a = r0 / G + s.start, b = (r1 - 1) / G + s.start;
  if (r1 <= r0 || b < 0 || a >= s.len || s.len <= 0) return false;
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

// ---------------------------------------------------------------- forward
template <typename T, int DP, bool SPLIT>
__global__ void __launch_bounds__(NT) fwd_kernel(AttnArgs a) {
  constexpr int KD = DP / 16, ND = DP / 32, LD = kLd<T, DP>;
  typedef typename Ops<T>::frag frag;
  __shared__ __attribute__((aligned(16))) T Ks[2][BN * LD];
  __shared__ __attribute__((aligned(16))) T Vs[2][BN * LD];
  const int bh = blockIdx.x, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int64_t rows = (int64_t)a.Tq * a.G;
  const int64_t r0 = (int64_t)(gridDim.y - 1 - blockIdx.y) * BM;  // longest rows first
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, h = l >> 5;
  const Seq seq = sequence(a, b);
  const int64_t r = r0 + wave * 32 + (l & 31);
  const int t = (int)(r / a.G), head = hk * a.G + (int)(r % a.G);
  const bool live = r < rows;
  const int p = live ? position(t, seq) : -1;
  const float c = a.scale * kLog2e;

  int pmin = 0, pmax = -1;
  const int64_t rend = r0 + BM < rows ? r0 + BM : rows;
  const bool any = span(r0, rend, a.G, seq, pmin, pmax);
  const int64_t w0 = r0 + wave * 32;
  int wmin = 0, wmax = -1;
  const bool wany = span(w0, w0 + 32 < rows ? w0 + 32 : rows, a.G, seq, wmin, wmax);
  const KeyTiles kt(pmin, pmax, a.W, a.S);
  int it0 = 0, it1 = any ? kt.total : 0;
  if (SPLIT) {
    const int per = (it1 + a.splits - 1) / a.splits;
    it0 = per * (int)blockIdx.z < it1 ? per * (int)blockIdx.z : it1;
    it1 = it0 + per < it1 ? it0 + per : it1;
  }

  const T* q = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[1] + t * a.qs[2];
  frag qf[KD];
#pragma unroll
  for (int k = 0; k < KD; ++k) qf[k] = global_frag<T>(q, k * 16 + 8 * h, a.D, p >= 0);

  v16f o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = zero16();
  float m = -kInf, sum = 0.f;

  const T* kb = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1];
  const T* vb = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1];
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
      const int cover = wany ? coverage(wmin, wmax, js, a.W, a.S) : 0;
      if (cover == 0) continue;
      v16f s = zero16();
#pragma unroll
      for (int k = 0; k < KD; ++k)
        s = Ops<T>::mma(row_frag<T, DP>(Ks[buf], sub * 32, k * 16), qf[k], s);
      float mx = -kInf;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = cover == 2 || sees(p, js + acc_row(e, h), a.W, a.S) ? s[e] * c : -kInf;
        mx = fmaxf(mx, s[e]);
      }
      mx = fmaxf(mx, other_half(mx));
      const float mn = fmaxf(m, mx);
      const float base = mn == -kInf ? 0.f : mn;
      const float alpha = ex2(m - base);
      m = mn;
      float add = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = ex2(s[e] - base);
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
  const bool none = p < 0 || sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  const float lse = none ? kInf : m + log2f(sum);
  if (!live) return;
  if (SPLIT) {
    const int64_t at = ((int64_t)blockIdx.z * gridDim.x + bh) * rows + r;
    if (h == 0) a.lpart[at] = none ? -kInf : lse;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = d * 32 + acc_row(e4 * 4, h);
        if (dd < a.D)
          *reinterpret_cast<float4*>(a.opart + at * a.D + dd) =
              none ? make_float4(0.f, 0.f, 0.f, 0.f)
                   : make_float4(o[d][e4 * 4] * inv, o[d][e4 * 4 + 1] * inv,
                                 o[d][e4 * 4 + 2] * inv, o[d][e4 * 4 + 3] * inv);
      }
    return;
  }
  if (h == 0 && a.lse != nullptr) a.lse[((int64_t)b * a.Hq + head) * a.Tq + t] = lse;
  T* out = reinterpret_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int dd = d * 32 + acc_row(e4 * 4, h);
      if (dd < a.D) {
        v4f f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = none ? 0.f : o[d][e4 * 4 + i] * inv;
        *reinterpret_cast<typename Ops<T>::quad*>(out + dd) =
            __builtin_convertvector(f, typename Ops<T>::quad);
      }
    }
}

// joins the key slices of a row, in order: one thread per 4 elements of D
template <typename T>
__global__ void __launch_bounds__(NT) join_kernel(AttnArgs a) {
  const int64_t rows = (int64_t)a.Tq * a.G, D4 = a.D / 4;
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  const int64_t all = (int64_t)a.B * a.Hkv * rows;
  if (id >= all * D4) return;
  const int64_t row = id / D4;
  const int d = (int)(id % D4) * 4;
  float m = -kInf;
  for (int z = 0; z < a.splits; ++z) m = fmaxf(m, a.lpart[z * all + row]);
  const float base = m == -kInf ? 0.f : m;
  float sum = 0.f;
  v4f o = {0.f, 0.f, 0.f, 0.f};
  for (int z = 0; z < a.splits; ++z) {
    const float lp = a.lpart[z * all + row];
    // a slice that saw nothing left zeros; one with a NaN has a NaN sum and
    // must not be skipped
    const float w = ex2(lp - base);
    const v4f x = *reinterpret_cast<const v4f*>(a.opart + (z * all + row) * a.D + d);
    sum += w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += w * x[i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] *= inv;
  const int64_t bh = row / rows, r = row % rows;
  const int64_t b = bh / a.Hkv, t = r / a.G, head = (bh % a.Hkv) * a.G + r % a.G;
  *reinterpret_cast<typename Ops<T>::quad*>(reinterpret_cast<T*>(a.out) + b * a.os[0] +
                                            head * a.os[1] + t * a.os[2] + d) =
      __builtin_convertvector(o, typename Ops<T>::quad);
  if (d == 0 && a.lse != nullptr)
    a.lse[(b * a.Hq + head) * a.Tq + t] = sum == 0.f ? kInf : base + log2f(sum);
}

// --------------------------------------------------------------- backward
// dq, and delta = do . o for the key-gradient kernel.  The forward's tiles
// and layout once more: S^T = K Q^T, dP^T = V dO^T, dS^T = P (dP - delta),
// dQ^T += K^T dS^T.
template <typename T, int DP>
__global__ void __launch_bounds__(NT) dq_kernel(AttnArgs a) {
  constexpr int KD = DP / 16, ND = DP / 32, LD = kLd<T, DP>;
  typedef typename Ops<T>::frag frag;
  __shared__ __attribute__((aligned(16))) T Ks[2][BN * LD];
  __shared__ __attribute__((aligned(16))) T Vs[2][BN * LD];
  const int bh = blockIdx.x, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int64_t rows = (int64_t)a.Tq * a.G;
  const int64_t r0 = (int64_t)(gridDim.y - 1 - blockIdx.y) * BM;
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, h = l >> 5;
  const Seq seq = sequence(a, b);
  const int64_t r = r0 + wave * 32 + (l & 31);
  const int t = (int)(r / a.G), head = hk * a.G + (int)(r % a.G);
  const bool live = r < rows;
  const int p = live ? position(t, seq) : -1;
  const float c = a.scale * kLog2e;

  int pmin = 0, pmax = -1;
  const bool any = span(r0, r0 + BM < rows ? r0 + BM : rows, a.G, seq, pmin, pmax);
  const int64_t w0 = r0 + wave * 32;
  int wmin = 0, wmax = -1;
  const bool wany = span(w0, w0 + 32 < rows ? w0 + 32 : rows, a.G, seq, wmin, wmax);
  const KeyTiles kt(pmin, pmax, a.W, a.S);
  const int it1 = any ? kt.total : 0;

  const T* q = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[1] + t * a.qs[2];
  const T* g = reinterpret_cast<const T*>(a.dout) + b * a.dos[0] + head * a.dos[1] + t * a.dos[2];
  const T* o = reinterpret_cast<const T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
  frag qf[KD], gf[KD];
  float delta = 0.f;
#pragma unroll
  for (int k = 0; k < KD; ++k) {
    qf[k] = global_frag<T>(q, k * 16 + 8 * h, a.D, p >= 0);
    gf[k] = global_frag<T>(g, k * 16 + 8 * h, a.D, p >= 0);
    const frag of = global_frag<T>(o, k * 16 + 8 * h, a.D, p >= 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) delta += (float)gf[k][i] * (float)of[i];
  }
  delta += other_half(delta);
  const int64_t at = ((int64_t)b * a.Hq + head) * a.Tq + t;
  if (live && h == 0) a.delta[at] = delta;
  const float lse = p >= 0 ? a.lse[at] : kInf;

  v16f dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = zero16();
  const T* kb = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1];
  const T* vb = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1];
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
      const int cover = wany ? coverage(wmin, wmax, js, a.W, a.S) : 0;
      if (cover == 0) continue;
      v16f s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        s = Ops<T>::mma(row_frag<T, DP>(Ks[buf], sub * 32, k * 16), qf[k], s);
        dp = Ops<T>::mma(row_frag<T, DP>(Vs[buf], sub * 32, k * 16), gf[k], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float pr = ex2(s[e] * c - lse);
        s[e] = cover == 2 || sees(p, js + acc_row(e, h), a.W, a.S) ? pr * (dp[e] - delta) : 0.f;
      }
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        const frag sf = acc_frag<T>(s, ss);
#pragma unroll
        for (int d = 0; d < ND; ++d)
          dq[d] = Ops<T>::mma(col_frag<T, DP>(Ks[buf], sub * 32 + ss * 16, d * 32), sf, dq[d]);
      }
    }
  }
  if (!live) return;
  T* out = reinterpret_cast<T*>(a.dq) + b * a.dqs[0] + head * a.dqs[1] + t * a.dqs[2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int dd = d * 32 + acc_row(e4 * 4, h);
      if (dd < a.D) {
        v4f f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = p < 0 ? 0.f : dq[d][e4 * 4 + i] * a.scale;
        *reinterpret_cast<typename Ops<T>::quad*>(out + dd) =
            __builtin_convertvector(f, typename Ops<T>::quad);
      }
    }
}

// Rows that look at the keys [k0, k0 + BM): the near ones, whose window
// reaches there, and, where the block holds sinks, the far ones behind them.
struct RowRange {
  int64_t n0, n1, f1;  // near [n0, n1), far [n1, f1)
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
  __device__ __forceinline__ static int64_t clip(int64_t t, const AttnArgs& a) {
    return t < 0 ? 0 : (t < a.Tq ? t : a.Tq);
  }
};

// far rows [f0, f1) of chunk `ch` of `chunks`, in whole tiles
__device__ __forceinline__ void far_chunk(const RowRange& rr, int ch, int chunks, int64_t& f0,
                                          int64_t& f1) {
  const int64_t tiles = (rr.f1 - rr.n1 + BN - 1) / BN;
  const int64_t per = (tiles + chunks - 1) / chunks;
  f0 = rr.n1 + per * ch * BN;
  f1 = f0 + per * BN;
  if (f1 > rr.f1) f1 = rr.f1;
  if (f0 > f1) f0 = f1;
}

// dk and dv: a wave owns 32 keys and the block walks the rows that look at
// them.  S = Q K^T and dP = dO V^T have a row's scores in register order, so
// dV^T += dO^T P and dK^T += Q^T dS take P and dS from where they are.
// blockIdx.y < key blocks: the near rows; above: a chunk of the far rows of
// a block with sinks, whose sums join_kv_kernel adds up.
template <typename T, int DP>
__global__ void __launch_bounds__(NT) dkv_kernel(AttnArgs a, int key_blocks) {
  constexpr int KD = DP / 16, ND = DP / 32, LD = kLd<T, DP>;
  typedef typename Ops<T>::frag frag;
  __shared__ __attribute__((aligned(16))) T Qs[2][BN * LD];
  __shared__ __attribute__((aligned(16))) T Gs[2][BN * LD];
  __shared__ float Ls[2][BN], Ds[2][BN];
  __shared__ int Ps[2][BN];
  const int bh = blockIdx.x, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, h = l >> 5;
  const Seq seq = sequence(a, b);
  const bool far = (int)blockIdx.y >= key_blocks;
  const int item = far ? (int)blockIdx.y - key_blocks : (int)blockIdx.y;
  const int kblock = far ? item / a.far_chunks : item;
  const int k0 = kblock * BM;
  const RowRange rr(k0, a, seq);
  int64_t ra = rr.n0, rb = rr.n1;
  if (far) far_chunk(rr, item % a.far_chunks, a.far_chunks, ra, rb);

  const int key = k0 + wave * 32 + (l & 31);
  const bool kok = key < seq.len;
  const float c = a.scale * kLog2e;
  frag kf[KD], vf[KD];
  {
    const T* kp = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2];
    const T* vp = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2];
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      kf[k] = global_frag<T>(kp, k * 16 + 8 * h, a.D, kok);
      vf[k] = global_frag<T>(vp, k * 16 + 8 * h, a.D, kok);
    }
  }
  v16f dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();

  const T* qb = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + hk * a.G * a.qs[1];
  const T* gb = reinterpret_cast<const T*>(a.dout) + b * a.dos[0] + hk * a.G * a.dos[1];
  Tile<T, DP> tq, tg;
  float nl = 0.f, nd = 0.f;
  int np = -1;
  auto fetch = [&](int64_t t0) {
    tq.load([&](int i) {
      const int64_t r = t0 + i;
      return r < rb ? qb + (r % a.G) * a.qs[1] + (r / a.G) * a.qs[2] : nullptr;
    }, a.D);
    tg.load([&](int i) {
      const int64_t r = t0 + i;
      return r < rb ? gb + (r % a.G) * a.dos[1] + (r / a.G) * a.dos[2] : nullptr;
    }, a.D);
    if (threadIdx.x < BN) {
      const int64_t r = t0 + threadIdx.x;
      np = r < rb ? position(r / a.G, seq) : -1;
      nl = kInf;
      nd = 0.f;
      if (np >= 0) {
        const int64_t at = ((int64_t)b * a.Hq + hk * a.G + r % a.G) * a.Tq + r / a.G;
        nl = a.lse[at];
        nd = a.delta[at];
      }
    }
  };
  if (ra < rb) fetch(ra);
  int buf = 0;
  for (int64_t t0 = ra; t0 < rb; t0 += BN, buf ^= 1) {
    tq.store(Qs[buf]);
    tg.store(Gs[buf]);
    if (threadIdx.x < BN) {
      Ls[buf][threadIdx.x] = nl;
      Ds[buf][threadIdx.x] = nd;
      Ps[buf][threadIdx.x] = np;
    }
    __syncthreads();
    if (t0 + BN < rb) fetch(t0 + BN);
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int64_t s0 = t0 + sub * 32;
      int pmin, pmax;
      const bool any = span(s0, s0 + 32 < rb ? s0 + 32 : rb, a.G, seq, pmin, pmax);
      const int cover = any ? coverage(pmin, pmax, k0 + wave * 32, a.W, a.S) : 0;
      if (cover == 0) continue;
      v16f s = zero16(), dp = zero16();
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        s = Ops<T>::mma(row_frag<T, DP>(Qs[buf], sub * 32, k * 16), kf[k], s);
        dp = Ops<T>::mma(row_frag<T, DP>(Gs[buf], sub * 32, k * 16), vf[k], dp);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int i = sub * 32 + acc_row(e, h);
        const bool see = cover == 2 || sees(Ps[buf][i], key, a.W, a.S);
        // rows outside the sequence have lse = +inf: P = 0
        const float pr = see ? ex2(s[e] * c - Ls[buf][i]) : 0.f;
        dp[e] = see ? pr * (dp[e] - Ds[buf][i]) : 0.f;
        s[e] = pr;
      }
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        const frag pf = acc_frag<T>(s, ss), sf = acc_frag<T>(dp, ss);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          dv[d] = Ops<T>::mma(col_frag<T, DP>(Gs[buf], sub * 32 + ss * 16, d * 32), pf, dv[d]);
          dk[d] = Ops<T>::mma(col_frag<T, DP>(Qs[buf], sub * 32 + ss * 16, d * 32), sf, dk[d]);
        }
      }
    }
  }

  if (a.far_chunks > 0 && kblock < a.sink_blocks) {
    // a share of a sink block's sums: [slot][dk, dv][key][D], fp32
    const int64_t slot = ((int64_t)bh * a.sink_blocks + kblock) * (1 + a.far_chunks) +
                         (far ? 1 + item % a.far_chunks : 0);
    float* part = a.kvpart + (slot * 2 * BM + wave * 32 + (l & 31)) * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const int dd = d * 32 + acc_row(e4 * 4, h);
        if (dd < a.D) {
          v4f fk, fv;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            fk[i] = dk[d][e4 * 4 + i] * a.scale;
            fv[i] = dv[d][e4 * 4 + i];
          }
          *reinterpret_cast<v4f*>(part + dd) = fk;
          *reinterpret_cast<v4f*>(part + (int64_t)BM * a.D + dd) = fv;
        }
      }
    return;
  }
  if (key >= a.Tk) return;
  T* ok = reinterpret_cast<T*>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2];
  T* ov = reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int dd = d * 32 + acc_row(e4 * 4, h);
      if (dd < a.D) {
        v4f fk, fv;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          fk[i] = dk[d][e4 * 4 + i] * a.scale;
          fv[i] = dv[d][e4 * 4 + i];
        }
        *reinterpret_cast<typename Ops<T>::quad*>(ok + dd) =
            __builtin_convertvector(fk, typename Ops<T>::quad);
        *reinterpret_cast<typename Ops<T>::quad*>(ov + dd) =
            __builtin_convertvector(fv, typename Ops<T>::quad);
      }
    }
}

// the shares of the sink blocks' keys, summed in order
template <typename T>
__global__ void __launch_bounds__(NT) join_kv_kernel(AttnArgs a) {
  const int64_t D4 = a.D / 4;
  const int64_t per = (int64_t)BM * D4;
  const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (id >= (int64_t)a.B * a.Hkv * a.sink_blocks * per) return;
  const int64_t blk = id / per;                       // (b, head, sink block)
  const int i = (int)(id % per / D4), d = (int)(id % D4) * 4;
  const int64_t bh = blk / a.sink_blocks, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int64_t key = (blk % a.sink_blocks) * BM + i;
  if (key >= a.Tk) return;
  v4f fk = {0.f, 0.f, 0.f, 0.f}, fv = fk;
  for (int ch = 0; ch <= a.far_chunks; ++ch) {
    const float* part =
        a.kvpart + (((blk * (1 + a.far_chunks) + ch) * 2) * BM + i) * (int64_t)a.D + d;
    fk += *reinterpret_cast<const v4f*>(part);
    fv += *reinterpret_cast<const v4f*>(part + (int64_t)BM * a.D);
  }
  *reinterpret_cast<typename Ops<T>::quad*>(reinterpret_cast<T*>(a.dk) + b * a.dks[0] +
                                            hk * a.dks[1] + key * a.dks[2] + d) =
      __builtin_convertvector(fk, typename Ops<T>::quad);
  *reinterpret_cast<typename Ops<T>::quad*>(reinterpret_cast<T*>(a.dv) + b * a.dvs[0] +
                                            hk * a.dvs[1] + key * a.dvs[2] + d) =
      __builtin_convertvector(fv, typename Ops<T>::quad);
}

unsigned row_blocks(const AttnArgs& a) {
  return (unsigned)ceil_div((int64_t)a.Tq * a.G, BM);
}

template <typename T, int DP>
void forward_dp(const AttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.Hkv), row_blocks(a), (unsigned)a.splits);
  if (a.splits > 1) {
    fwd_kernel<T, DP, true><<<grid, NT, 0, st>>>(a);
    const int64_t n = (int64_t)a.B * a.Hq * a.Tq * (a.D / 4);
    join_kernel<T><<<(unsigned)ceil_div(n, NT), NT, 0, st>>>(a);
  } else {
    fwd_kernel<T, DP, false><<<grid, NT, 0, st>>>(a);
  }
}

template <typename T, int DP>
void backward_dp(const AttnArgs& a, hipStream_t st) {
  const unsigned bh = (unsigned)(a.B * a.Hkv);
  dq_kernel<T, DP><<<dim3(bh, row_blocks(a)), NT, 0, st>>>(a);
  const int kb = (int)ceil_div(a.Tk, BM);
  dkv_kernel<T, DP><<<dim3(bh, (unsigned)(kb + a.sink_blocks * a.far_chunks)), NT, 0, st>>>(a, kb);
  if (a.far_chunks > 0) {
    const int64_t n = (int64_t)bh * a.sink_blocks * BM * (a.D / 4);
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

void attn_plan(const AttnArgs& a, int, int* splits, int64_t* floats) {
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

void attn_bwd_plan(const AttnArgs& a, int, int* sink_blocks, int* far_chunks, int64_t* floats) {
  *sink_blocks = *far_chunks = 0;
  *floats = 0;
  // far rows exist only behind the window of a sink's key
  if (a.S <= 0 || a.W >= a.Tk || a.Tk == 0) return;
  const int64_t sb = ceil_div(std::min<int64_t>(a.S, a.Tk), BM);
  const int64_t tiles = ceil_div((int64_t)a.Tq * a.G, BN);
  int64_t ch = ceil_div(tiles, 16);
  if (ch > 64) ch = 64;
  if (ch < 1) ch = 1;
  *sink_blocks = (int)sb;
  *far_chunks = (int)ch;
  *floats = (int64_t)a.B * a.Hkv * sb * (1 + ch) * 2 * BM * a.D;
}

void attn_backward(int dtype, const AttnArgs& a, hipStream_t st) {
  if ((int64_t)a.B * a.Hkv * a.Tk == 0 || a.Tq == 0) return;
  if (dtype == kBF16) backward_type<__bf16>(a, st);
  else if (dtype == kF16) backward_type<_Float16>(a, st);
  else backward_type<float>(a, st);
}

}  // namespace kfac

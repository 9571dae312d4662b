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
#include <utility>

namespace kfac {

namespace {

constexpr int NT = 256;      // threads of the joining kernels
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

// (x of lane l & 31, x of lane l | 32)
__device__ __forceinline__ void halves(float x, float& lo, float& hi) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x),
                                                  __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t a = r[0], b = r[1];
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}
__device__ __forceinline__ float halves_sum(float x) {
  float lo, hi;
  halves(x, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ float halves_max(float x) {
  float lo, hi;
  halves(x, lo, hi);
  return fmaxf(lo, hi);
}

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

// fp16 holds numbers from 2^-14 on (2^-24 with one bit) and up to 2^16.
// Probabilities are at most 1 and a long row has many small ones, so they are
// rounded 2^kLift larger than they are, and the sums that they enter are
// divided by it, a power of two, in 32 bits.  Forward: 2^7, the base of a
// row's powers lies up to 2^8 below its maximum, so they end at 2^15.  Key
// gradients, whose powers have the row's sum in their base: 2^15.  Their
// products with dP - delta follow the upstream gradient's size and get a power
// of two of their own (lift_of).
template <typename T> constexpr int kLift = 0;
template <> constexpr int kLift<_Float16> = 7;
template <typename T> constexpr int kKeyLift = 0;
template <> constexpr int kKeyLift<_Float16> = 15;
template <typename T> constexpr bool kLifts = kLift<T> != 0;

// f(0), f(1) .. f(N - 1), each with its number as a constant
template <typename F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
  each_of(f, std::make_integer_sequence<int, N>());
}

template <typename T> constexpr int kUnit = 16 / (int)sizeof(T);  // elements of 16 bytes

// An LDS tile is BN rows of CR 16-byte chunks (a power of two), chunk c of
// row r at place c ^ place_of(r).  Row reads (16 bytes of 32 rows) and
// transposed reads (64 bytes of 4 rows) then both meet every bank once; a
// padded row stride can serve only one of the two.
template <typename T, int DP> constexpr int kChunks = DP * (int)sizeof(T) <= 64 ? 4
                                                   : DP * (int)sizeof(T) <= 128 ? 8
                                                   : DP * (int)sizeof(T) <= 256 ? 16 : 32;
template <typename T, int DP> constexpr int kLd = kChunks<T, DP> * kUnit<T>;  // elements of a row

template <int CR>
__device__ __forceinline__ int place_of(int r) {
  if constexpr (CR >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
  else if constexpr (CR == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
  else return (r >> 2) & 3;
}

// Waves a SIMD that the row kernels and the key-gradient kernel leave
// registers for (256 a wave at 2, 512 at 1).
template <typename T, int DP> constexpr int kRowFit = sizeof(T) == 2 || DP <= 64 ? 2 : 1;
template <typename T, int DP> constexpr int kKeyFit = (sizeof(T) == 2 ? DP <= 64 : DP <= 32) ? 2 : 1;

// Waves of a block.  Rows: 4 (GPT-NeoX batch: forward 39 us, 44 with 2 and 42
// with 8; 8192 tokens with heads of 128: 94, 148, 115).  Keys: 2 up to heads
// of 64, where the shorter blocks even out the load (67 us, 74 with 4; fp32
// padded batch 60, 78), 4 above, where the traffic of the rows weighs more
// (228 us, 243 with 2, before the fixed order of KeyGrad::rows64).
constexpr int kRowWaves = 4;
template <int DP> constexpr int kKeyWaves = DP <= 64 ? 2 : 4;

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

// Where a lane reads a tile, in bytes from its start.  Rows and chunks lie in
// different bits and place_of is linear over the bits of a row, so every
// other operand's place is one exclusive or and a constant away.
template <typename T, int DP>
struct Lane {
  static constexpr int CR = kChunks<T, DP>, ROW = kLd<T, DP> * (int)sizeof(T);
  uint32_t row, col;
  __device__ __forceinline__ Lane() {
    const int l = threadIdx.x & 63, h = l >> 5;
    if constexpr (sizeof(T) == 2) {
      const int i = l & 15, g = l >> 4, r = 4 * (g >> 1) + (i >> 2);
      row = (l & 31) * ROW + (h ^ place_of<CR>(l & 31)) * 16;
      col = r * ROW + ((2 * (g & 1) + ((i & 3) >> 1)) ^ place_of<CR>(r)) * 16 + 8 * (i & 1);
    } else {
      row = (l & 31) * ROW + ((2 * h) ^ place_of<CR>(l & 31)) * 16;
      col = 4 * h * ROW + (((l & 31) / 4) ^ place_of<CR>(4 * h)) * 16 + (l & 3) * 4;
    }
  }
  // Once a tile: the compiler would keep every operand's address of every
  // tile in a register of its own (100 and more) instead of these two.
  __device__ __forceinline__ void fresh() { asm volatile("" : "+v"(row), "+v"(col)); }
};

// Left operand from rows: lane l holds row r0 + (l & 31), elements
// 16 k + 8 (l >> 5) .. + 7 (r0 a multiple of 16)
template <typename T, int DP>
__device__ __forceinline__ typename Ops<T>::frag row_frag(const T* L, const Lane<T, DP>& at, int r0,
                                                          int k) {
  const char* p = reinterpret_cast<const char*>(L) + r0 * Lane<T, DP>::ROW;
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const typename Ops<T>::frag*>(p + (at.row ^ (k * 32)));
  } else {
    const v4f a = *reinterpret_cast<const v4f*>(p + (at.row ^ (k * 64)));
    const v4f b = *reinterpret_cast<const v4f*>(p + (at.row ^ (k * 64 + 16)));
    return v8f{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  }
}

// Left operand from columns: lane l holds column c0 + (l & 31) of tile rows
// r0 + 4h + {0..3} and r0 + 8 + 4h + {0..3}: the order in which registers
// 8s .. 8s + 7 of an accumulator hold its rows (r0 = 16 s)
template <typename T, int DP>
__device__ __forceinline__ typename Ops<T>::frag col_frag(const T* L, const Lane<T, DP>& at, int r0,
                                                          int c0) {
  constexpr int CR = Lane<T, DP>::CR, ROW = Lane<T, DP>::ROW;
  const char* p = reinterpret_cast<const char*>(L) + r0 * ROW;
  if constexpr (sizeof(T) == 2) {
    // ds_read_b64_tr_b16: 16 lanes read 4 rows x 16 columns (lane 4q + p row
    // q, columns 4p ..) and get a column's 4 rows each
    const char* lp = p + (at.col ^ (c0 * 2));
    const char* hp = p + 8 * ROW + (at.col ^ (c0 * 2 ^ place_of<CR>(8) * 16));
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)lp);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)hp);
    const v8i16 f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(typename Ops<T>::frag, f);
  } else {
    v8f f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int x = (i & 3) + 8 * (i >> 2);
      f[i] = *reinterpret_cast<const float*>(p + x * ROW +
                                             (at.col ^ (c0 * 4 ^ place_of<CR>(x) * 16)));
    }
    return f;
  }
}

// registers 8s .. 8s + 7 of an accumulator as a right operand, rounded once
// to the operands' type (16-bit probabilities and their gradients are the
// price of the matrix units; each is off by half a step, 2^-8 of itself in
// bf16 and 2^-11 in fp16, and the sums over them stay in 32 bits).  fp16's
// stay clear of its subnormals and of its end: kLift.  What falls below 2^-14
// there all the same is off by 2^-25, that is 2^-32 of a row's largest
// probability (forward), 2^-40 (key gradients), and 2^-40 of what dP - delta
// can be.
template <typename T>
__device__ __forceinline__ typename Ops<T>::frag acc_frag(const v16f& a, int s) {
  v8f f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = a[8 * s + i];
  return __builtin_convertvector(f, typename Ops<T>::frag);
}

// what that rounding took away, rounded itself
template <typename T>
__device__ __forceinline__ typename Ops<T>::frag acc_rest(const v16f& a, int s,
                                                          typename Ops<T>::frag rounded) {
  v8f f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = a[8 * s + i] - (float)rounded[i];
  return __builtin_convertvector(f, typename Ops<T>::frag);
}

// 8 elements of a global row from element d on; zeros behind D (D % 8 == 0)
// and where the row is not `ok`.  Those lanes read `there`, the tensor's
// beginning: with a branch round the load, a row's loads would wait for each
// other.
template <typename T>
__device__ __forceinline__ typename Ops<T>::frag global_frag(const void* there, const T* row, int d,
                                                             int D, bool ok) {
  ok = ok && d < D;
  const T* p = ok ? row + d : reinterpret_cast<const T*>(there);
  typename Ops<T>::frag f;
  if constexpr (sizeof(T) == 2) {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    v4u u = *reinterpret_cast<const v4u*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = ok ? u[i] : 0u;
    f = __builtin_bit_cast(typename Ops<T>::frag, u);
  } else {
    const v4f a = *reinterpret_cast<const v4f*>(p);
    const v4f b = *reinterpret_cast<const v4f*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i] = ok ? a[i] : 0.f;
      f[4 + i] = ok ? b[i] : 0.f;
    }
  }
  return f;
}

constexpr uint32_t kNowhere = 0x80000000u;  // an offset that no buffer reaches: reads 0

// One wave's share of a BN-row tile, straight from global memory into LDS
// (16 bytes a lane, no registers in between).  The places in LDS follow the
// lanes; which chunk belongs there is in the offsets, which a tile of rows
// at a constant stride keeps for its whole life.  Offsets behind the
// buffer's last byte read zeros.
template <typename T, int DP, int NW>
struct Dma {
  static constexpr int NT = 64 * NW, CR = kChunks<T, DP>, CH = BN * CR / NT;
  __device__ __forceinline__ static int row(int n) { return (n * NT + (int)threadIdx.x) / CR; }
  __device__ __forceinline__ static int chunk(int n) {
    return ((n * NT + (int)threadIdx.x) % CR) ^ place_of<CR>(row(n));
  }
  // byte offset of this lane's chunk n in a row at `at` bytes
  __device__ __forceinline__ static uint32_t offset(int n, uint32_t at, int D) {
    return chunk(n) * kUnit<T> < D ? at + chunk(n) * 16 : kNowhere;
  }
  template <typename F>
  __device__ __forceinline__ static void run(T* L, const void* base, uint32_t bytes, int wave,
                                             F offset_of) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
#pragma unroll
    for (int n = 0; n < CH; ++n)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(L + (n * NT + wave * 64) * kUnit<T>), 16,
          offset_of(n), 0, 0, 0);
  }
};

// this wave's loads into LDS have arrived, then everybody's
__device__ __forceinline__ void arrived() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

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

// bits below n set, n clamped to [0, 32]
__device__ __forceinline__ uint32_t below(int n) {
  return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u);
}

// Scores become -inf where bit acc_row(e, 0) of `keep` is clear: their
// probability is 0.  Two instructions an element (sign-extended bit, select).
__device__ __forceinline__ void hide(v16f& s, uint32_t keep) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t m = (uint32_t)((int)(keep << (31 - acc_row(e, 0))) >> 31);
    s[e] = __uint_as_float((__float_as_uint(s[e]) & m) | (0xff800000u & ~m));
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

// what rounding x times f to T takes away, rounded to T itself
template <typename T, int ND>
__device__ __forceinline__ void put_rest(T* out, const v16f (&x)[ND], float f, bool zero, int D,
                                         int h) {
  typedef T quad __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const int dd = d * 32 + acc_row(e4 * 4, h);
      if (dd < D) {
        v4f v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = zero ? 0.f : x[d][e4 * 4 + i] * f;
          v[i] -= (float)(T)v[i];
        }
        *reinterpret_cast<quad*>(out + dd) = __builtin_convertvector(v, quad);
      }
    }
}

// What a block of the row kernels (forward, dq) works on.
template <int NW>
struct RowBlock {
  static constexpr int BM = 32 * NW;
  int b, hk, bh, r0, r, t, head, p, h, wave;
  int tiles;
  // keys that some row of this wave sees, and those that all rows see:
  // [0, S) or [any0, any1), and [full0, full1) or [0, fulls)
  int any0, any1, full0, full1, fulls;
  bool live;
  Seq seq;
  __device__ __forceinline__ RowBlock(const AttnArgs& a) {
    bh = blockIdx.x;
    b = bh / a.Hkv;
    hk = bh - b * a.Hkv;
    const int rows = a.Tq * a.G;
    r0 = (int)(gridDim.y - 1 - blockIdx.y) * BM;  // longest rows first
    const int l = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    h = l >> 5;
    seq = sequence(a, b);
    r = r0 + wave * 32 + (l & 31);
    const Row rw(r, a);
    t = rw.t;
    head = hk * a.G + rw.g;
    live = r < rows;
    p = live ? position(t, seq) : -1;
    const int w0 = r0 + wave * 32;
    int wmin = 0, wmax = -1;  // no rows: no keys
    span(w0, w0 + 32 < rows ? w0 + 32 : rows, a, seq, wmin, wmax);
    any0 = wmin - a.W + 1;
    any1 = wmax + 1;
    full0 = wmax - a.W + 1;
    full1 = wmin + 1;
    fulls = a.S < full1 ? a.S : full1;
  }
  // what the wave's rows see of 32 keys from j0 on: 0 nothing, 2 all, 1 mixed
  __device__ __forceinline__ int coverage(int j0, int S) const {
    if (j0 >= any1 || (j0 + 32 <= any0 && j0 >= S)) return 0;
    return (j0 >= full0 && j0 + 32 <= full1) || j0 + 32 <= fulls ? 2 : 1;
  }
  // which of the 32 keys from j0 on this lane's row sees: bit o is key
  // j0 + 4h + o
  __device__ __forceinline__ uint32_t seen(int j0, const AttnArgs& a) const {
    const int first = j0 + 4 * h;
    return below(p - first + 1) & (~below(p - a.W + 1 - first) | below(a.S - first));
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

// The K and V tiles of a row block, one after the other.
template <typename T, int DP, int NW>
struct KeyStream {
  typedef Dma<T, DP, NW> D;
  const char *k, *v;
  uint32_t ko[D::CH], vo[D::CH];
  uint32_t ks, vs;  // bytes from a key to the next
  int wave;
  __device__ __forceinline__ KeyStream(const AttnArgs& a, const RowBlock<NW>& w) {
    k = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.k) + w.b * a.ks[0] +
                                      w.hk * a.ks[1]);
    v = reinterpret_cast<const char*>(reinterpret_cast<const T*>(a.v) + w.b * a.vs[0] +
                                      w.hk * a.vs[1]);
    ks = (uint32_t)(a.ks[2] * sizeof(T));
    vs = (uint32_t)(a.vs[2] * sizeof(T));
    wave = w.wave;
#pragma unroll
    for (int n = 0; n < D::CH; ++n) {
      ko[n] = D::offset(n, D::row(n) * ks, a.D);
      vo[n] = D::offset(n, D::row(n) * vs, a.D);
    }
  }
  // keys behind kt.hi, and those before the window that are no sinks, read
  // as zeros: nobody sees them, and they may hold anything
  __device__ __forceinline__ void fetch(const AttnArgs& a, const KeyTiles& kt, int j0, T* K,
                                        T* V) const {
    const uint32_t last = kt.hi - j0 < BN ? kt.hi - j0 - 1 : BN - 1, row = a.D * sizeof(T);
    const uint32_t kb = last * ks + row, vb = last * vs + row;
    const char* kp = k + (uint64_t)(uint32_t)j0 * ks;
    const char* vp = v + (uint64_t)(uint32_t)j0 * vs;
    if (j0 >= kt.lo) {
      D::run(K, kp, kb, wave, [&](int i) { return ko[i]; });
      D::run(V, vp, vb, wave, [&](int i) { return vo[i]; });
    } else {
      auto seen = [&](int i) { return j0 + D::row(i) >= kt.lo || j0 + D::row(i) < a.S; };
      D::run(K, kp, kb, wave, [&](int i) { return seen(i) ? ko[i] : kNowhere; });
      D::run(V, vp, vb, wave, [&](int i) { return seen(i) ? vo[i] : kNowhere; });
    }
  }
};

// Runs step(K tile, V tile, first key) over key tiles [it0, it1), the next
// tile on its way while one is worked on.  Two buffers that the compiler can
// tell apart: it would otherwise wait for the loads before every LDS read.
template <typename T, int DP, int NW, typename F>
__device__ __forceinline__ void stream_keys(const AttnArgs& a, const RowBlock<NW>& w,
                                            const KeyTiles& kt, int it0, int it1, F step) {
  __shared__ __attribute__((aligned(16))) T K0[BN * kLd<T, DP>];
  __shared__ __attribute__((aligned(16))) T K1[BN * kLd<T, DP>];
  __shared__ __attribute__((aligned(16))) T V0[BN * kLd<T, DP>];
  __shared__ __attribute__((aligned(16))) T V1[BN * kLd<T, DP>];
  const KeyStream<T, DP, NW> ks(a, w);
  if (it0 < it1) ks.fetch(a, kt, kt.key0(it0), K0, V0);
  for (int it = it0; it < it1; it += 2) {
    arrived();
    if (it + 1 < it1) ks.fetch(a, kt, kt.key0(it + 1), K1, V1);
    step(K0, V0, kt.key0(it));
    if (it + 1 >= it1) break;
    arrived();
    if (it + 2 < it1) ks.fetch(a, kt, kt.key0(it + 2), K0, V0);
    step(K1, V1, kt.key0(it + 1));
  }
}

// ---------------------------------------------------------------- forward
// 8192 tokens, 16 heads of 128 over 4, window 1024: 95 us, 690 TFLOP/s, the
// matrix units busy for 32% and the vector unit for 36% of it with two waves a
// SIMD, as many as the tiles leave room for.  GPT-NeoX batch (8 x 2048 tokens,
// 12 heads of 64, window 256): 38 us; a block sees 7 tiles there, one of them
// the sinks', and a product of 64 elements is shorter than its powers.
// SPLIT, for few rows: the keys over blockIdx.z.  16 sequences of one token,
// 32 heads of 128 over 8, 4096 keys each: 54 us and 5 to join, 4.6 TB/s of
// keys and values.
template <typename T, int DP, int NW, bool SPLIT>
__global__ void __launch_bounds__(64 * NW, (kRowFit<T, DP>)) fwd_kernel(AttnArgs a) {
  constexpr int KD = DP / 16, ND = DP / 32;
  typedef typename Ops<T>::frag frag;
  RowBlock<NW> w(a);
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
  for (int k = 0; k < KD; ++k) qf[k] = global_frag<T>(a.q, q, k * 16 + 8 * h, a.D, w.p >= 0);

  v16f o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = zero16();
  float m = -kInf, sum = 0.f;
  Lane<T, DP> at;

  stream_keys<T, DP, NW>(a, w, kt, it0, it1, [&](const T* K, const T* V, int j0) {
    at.fresh();
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int js = j0 + sub * 32;
      const int cover = w.coverage(js, a.S);
      if (cover == 0) continue;
      v16f s = zero16();
#pragma unroll
      for (int k = 0; k < KD; ++k) s = Ops<T>::mma(row_frag<T, DP>(K, at, sub * 32, k), qf[k], s);
      if (cover == 1) hide(s, w.seen(js, a));
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
      // c > 0: the maximum of the products is the product of the maximum
      mx = halves_max(mx) * c;
      // The base of a row's powers may lie up to 2^8 below its maximum: sums
      // and accumulators have the exponents for that (fp16: kLift), the
      // quotient at the end does not change, and most tiles of a row leave its
      // accumulators alone.
      if (__any(mx > m + 8.f)) {
        const float mn = fmaxf(m, mx);
        const float alpha = ex2(m - (mn == -kInf ? 0.f : mn));
        m = mn;
        sum *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
      }
      const float base = (m == -kInf ? 0.f : m) - kLift<T>;
      float add = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[e] = ex2(__builtin_fmaf(s[e], c, -base));
        add += s[e];
      }
      sum += add;
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        const frag pf = acc_frag<T>(s, ss);
#pragma unroll
        for (int d = 0; d < ND; ++d)
          o[d] = Ops<T>::mma(col_frag<T, DP>(V, at, sub * 32 + ss * 16, d * 32), pf, o[d]);
      }
    }
  });

  sum = halves_sum(sum);
  const bool none = w.p < 0 || sum == 0.f;
  const float inv = none ? 0.f : 1.f / sum;
  const float lse = none ? kInf : (m - kLift<T>) + log2f(sum);
  if (!w.live) return;
  if (SPLIT) {
    const int64_t row = ((int64_t)blockIdx.z * gridDim.x + w.bh) * (a.Tq * a.G) + w.r;
    if (h == 0) a.lpart[row] = none ? -kInf : lse;
    put<T, float, ND>(a.opart + row * a.D, o, inv, none, a.D, h);
    return;
  }
  if (h == 0 && a.lse != nullptr) a.lse[(int64_t)w.bh * (a.Tq * a.G) + w.r] = lse;
  const int64_t at_out = w.b * a.os[0] + w.head * a.os[1] + w.t * a.os[2];
  put<T, T, ND>(reinterpret_cast<T*>(a.out) + at_out, o, inv, none, a.D, h);
  if (sizeof(T) == 2 && a.rest != nullptr)
    put_rest<T, ND>(reinterpret_cast<T*>(a.rest) + at_out, o, inv, none, a.D, h);
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
#pragma unroll 8
  for (int z = grp; z < a.splits; z += 8) {
    const float wt = wts[z];
    sum += wt;
    // lanes behind D read its last elements again and are not stored
    const v4f x = *reinterpret_cast<const v4f*>(a.opart + (z * all + row) * a.D +
                                                (d < a.D ? d : a.D - 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += wt * x[i];
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
  if (d < a.D) {
    const int64_t at = b * a.os[0] + head * a.os[1] + rw.t * a.os[2] + d;
    *reinterpret_cast<typename Ops<T>::quad*>(reinterpret_cast<T*>(a.out) + at) =
        __builtin_convertvector(o, typename Ops<T>::quad);
    if (sizeof(T) == 2 && a.rest != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] -= (float)(T)o[i];
      *reinterpret_cast<typename Ops<T>::quad*>(reinterpret_cast<T*>(a.rest) + at) =
          __builtin_convertvector(o, typename Ops<T>::quad);
    }
  }
  if (tid == 0 && a.lse != nullptr)
    a.lse[row] = sum == 0.f ? kInf : base + log2f(sum);
}

__device__ __forceinline__ int clip(int64_t t, const AttnArgs& a) {
  return (int)(t < 0 ? 0 : (t < a.Tq ? t : a.Tq));
}

// The rows that see a wave's 32 keys, as rows: first and behind the last
// that see some of them, that see all of them, and that see this lane's.
struct KeyRows {
  int any0, any1, full0, full1, mine0, mine1;
  __device__ __forceinline__ KeyRows(int j0, int key, const AttnArgs& a, const Seq& s) {
    // row of the first token at position p or later
    auto row = [&](int64_t p) { return clip(p - s.start, a) * a.G; };
    const int64_t last = s.len, w = a.W;
    any0 = row(j0);
    any1 = row(j0 < a.S || j0 + 31 + w > last ? last : j0 + 31 + w);
    full0 = row((int64_t)j0 + 31);
    full1 = row(j0 + 31 < a.S || j0 + w > last ? last : j0 + w);
    mine0 = row(key);
    mine1 = row(key < a.S || key + w > last ? last : key + w);
  }
  __device__ __forceinline__ int coverage(int r0) const {
    if (r0 + 32 <= any0 || r0 >= any1) return 0;
    return r0 >= full0 && r0 + 32 <= full1 ? 2 : 1;
  }
  // some row sees this lane's key
  __device__ __forceinline__ bool key_seen() const { return mine0 < mine1; }
  // bit o is row r0 + 4h + o
  __device__ __forceinline__ uint32_t seen(int r0, int h) const {
    const int first = r0 + 4 * h;
    return below(mine1 - first) & ~below(mine0 - first);
  }
};

// fp16's products P (dP - delta) would pass 65504 under a large loss scale, and
// lie among the subnormals, or below them, for small upstream gradients and
// long windows: they are rounded 2^n larger than they are, n from the bound
// |dP - delta| <= 2 |do| |v|, so that none reaches 2^15.  n of a row for dq,
// whose sums are a row's own; of a (sequence, key head) for dk.
__device__ __forceinline__ int lift_of(float do2, float v2) {
  const float b = 4.f * do2 * v2;
  // nothing to bound, or no bound: infinities are the caller's
  if (!(b > 0.f && b < kInf)) return 0;
  return 15 - ((__builtin_amdgcn_frexp_expf(b) + 1) >> 1);  // sqrt(b) < 2^that
}

__device__ __forceinline__ float power2(int n) { return __builtin_amdgcn_ldexpf(1.f, n); }

// The largest |do|^2 and |v|^2 of a chunk of the rows and keys that take part:
// blockIdx.y of a.bound_chunks.  One read of do and v, 16 lanes a row of them.
// fp16, GPT-NeoX batch (8 x 2048 tokens, 12 heads of 64): 13 us of the pass's
// 157, with the factors on dS 4 us each in dq and dk/dv; 140 us without all of
// it, and then products under 2^-25 are lost and those over 65504 infinite.
template <typename T>
__global__ void __launch_bounds__(NT) bounds_kernel(AttnArgs a) {
  constexpr int U = 8;  // rows in flight
  __shared__ float red[2][NT / 64];
  const int bh = blockIdx.x, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int d = ((int)threadIdx.x & 15) * 8, first = (int)threadIdx.x >> 4;
  const Seq seq = sequence(a, b);
  const int chunk = blockIdx.y;
  float best[2];
  auto largest = [&](int n, auto load) {
    const int per = (n + a.bound_chunks - 1) / a.bound_chunks;
    const int from = per * chunk < n ? per * chunk : n, to = from + per < n ? from + per : n;
    float mx = 0.f;
    for (int i = from + first; i < to; i += U * (NT / 16)) {
      typename Ops<T>::frag f[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = i + u * (NT / 16);
        f[u] = load(at < to ? at : i);
      }
      float s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[u] += (float)f[u][e] * (float)f[u][e];
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] += __shfl_xor(s[u], off, 64);
      // leaves out a NaN, which is in the gradient anyway
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    return fmaxf(mx, __shfl_xor(mx, 32, 64));
  };
  best[0] = largest(a.Tq * a.G, [&](int i) {
    const Row r(i, a);
    const T* p = reinterpret_cast<const T*>(a.dout) + b * a.dos[0] + (hk * a.G + r.g) * a.dos[1] +
                 r.t * a.dos[2];
    return global_frag<T>(a.dout, p, d, a.D, position(r.t, seq) >= 0);
  });
  best[1] = largest(a.Tk, [&](int j) {
    const T* p = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1] + j * a.vs[2];
    return global_frag<T>(a.v, p, d, a.D, KeyRows(j, j, a, seq).key_seen());
  });
  if ((threadIdx.x & 63) == 0)
    for (int i = 0; i < 2; ++i) red[i][threadIdx.x >> 6] = best[i];
  __syncthreads();
  if (threadIdx.x >= 2) return;
  const float* x = red[threadIdx.x];
  a.bounds[((int64_t)bh * a.bound_chunks + chunk) * 2 + threadIdx.x] =
      fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
}

// which: 0 the largest |do|^2 of a (sequence, key head), 1 |v|^2
__device__ __forceinline__ float bound_of(const AttnArgs& a, int bh, int which) {
  const int l = threadIdx.x & 63;
  float x = l < a.bound_chunks ? a.bounds[((int64_t)bh * a.bound_chunks + l) * 2 + which] : 0.f;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

// The factor of the gradients to q and k.  Where a row sees itself alone its
// probability is 1 whatever they are, and the gradient exactly 0: not the
// difference of two sums that were taken in different orders.
__device__ __forceinline__ float score_factor(const AttnArgs& a) {
  return a.W == 1 && (a.S == 0 || a.Tk == 1) ? 0.f : a.scale;
}

// --------------------------------------------------------------- backward
// dq, and -delta = -do . o for the key-gradient kernel.  The forward's tiles
// and layout once more: S^T = K Q^T, dP^T = V dO^T, dS^T = P (dP - delta),
// dQ^T += K^T dS^T.  8192 tokens, heads of 128: 130 us, 750 TFLOP/s; GPT-NeoX
// batch 49 us.  The fixed order of KeyGrad::rows64 costs the second wave of a
// SIMD its registers here (57 us for the latter), four waves a SIMD with 128
// registers are no faster (49).
// FINE: see attn_keeps_rest.
template <typename T, int DP, int NW, bool FINE>
__global__ void __launch_bounds__(64 * NW, (kRowFit<T, DP>)) dq_kernel(AttnArgs a) {
  constexpr int KD = DP / 16, ND = DP / 32;
  typedef typename Ops<T>::frag frag;
  RowBlock<NW> w(a);
  const KeyTiles kt = w.keys(a);
  const int h = w.h;
  const float c = a.scale * kLog2e;

  const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.qs[0] + w.head * a.qs[1] + w.t * a.qs[2];
  const T* g =
      reinterpret_cast<const T*>(a.dout) + w.b * a.dos[0] + w.head * a.dos[1] + w.t * a.dos[2];
  const int64_t at_out = w.b * a.os[0] + w.head * a.os[1] + w.t * a.os[2];
  const T* o = reinterpret_cast<const T*>(a.out) + at_out;
  const T* rest = reinterpret_cast<const T*>(a.rest) + at_out;
  frag qf[KD], gf[KD];
  float delta = 0.f;
#pragma unroll
  for (int k = 0; k < KD; ++k) {
    qf[k] = global_frag<T>(a.q, q, k * 16 + 8 * h, a.D, w.p >= 0);
    gf[k] = global_frag<T>(a.dout, g, k * 16 + 8 * h, a.D, w.p >= 0);
    const frag of = global_frag<T>(a.out, o, k * 16 + 8 * h, a.D, w.p >= 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) delta += (float)gf[k][i] * (float)of[i];
  }
  if (FINE) {
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      const frag rf = global_frag<T>(a.rest, rest, k * 16 + 8 * h, a.D, w.p >= 0);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += (float)gf[k][i] * (float)rf[i];
    }
  }
  delta = -halves_sum(delta);
  const int64_t row = (int64_t)w.bh * (a.Tq * a.G) + w.r;
  if (w.live && h == 0) a.delta[row] = delta;
  const float lse = w.p >= 0 ? a.lse[row] : kInf;
  // multiplied on, not put into the base of the powers: a power of two more on
  // the upstream gradient is then one on dq, bit for bit
  float more = 1.f, back = 1.f;
  if constexpr (kLifts<T>) {
    if (w.live && h == 0) a.lse_keys[row] = lse - kKeyLift<T>;
    float do2 = 0.f;
#pragma unroll
    for (int k = 0; k < KD; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) do2 += (float)gf[k][i] * (float)gf[k][i];
    const int lift = lift_of(halves_sum(do2), bound_of(a, w.bh, 1));
    more = power2(lift);
    back = power2(-lift);
  }

  // dP - delta comes out of the matrix units: they start from -delta (in fp32
  // with heads over 32, whose registers are full, it is added afterwards)
  constexpr bool kStart = sizeof(T) == 2 || DP <= 32;
  v16f minus = zero16();
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (kStart) minus[e] = delta;
  v16f dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dq[d] = zero16();
  Lane<T, DP> at;
  stream_keys<T, DP, NW>(a, w, kt, 0, w.tiles, [&](const T* K, const T* V, int j0) {
    at.fresh();
#pragma unroll
    for (int sub = 0; sub < BN / 32; ++sub) {
      const int js = j0 + sub * 32;
      const int cover = w.coverage(js, a.S);
      if (cover == 0) continue;
      v16f s = zero16(), dp = minus;
#pragma unroll
      for (int k = 0; k < KD; ++k) {
        s = Ops<T>::mma(row_frag<T, DP>(K, at, sub * 32, k), qf[k], s);
        dp = Ops<T>::mma(row_frag<T, DP>(V, at, sub * 32, k), gf[k], dp);
      }
      if (cover == 1) hide(s, w.seen(js, a));
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = ex2(__builtin_fmaf(s[e], c, -lse));
        s[e] = (kLifts<T> ? x * more : x) * (kStart ? dp[e] : dp[e] + delta);
      }
#pragma unroll
      for (int ss = 0; ss < 2; ++ss) {
        const frag sf = acc_frag<T>(s, ss);
        frag rest;
        if constexpr (FINE) rest = acc_rest<T>(s, ss, sf);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const frag kf = col_frag<T, DP>(K, at, sub * 32 + ss * 16, d * 32);
          dq[d] = Ops<T>::mma(kf, sf, dq[d]);
          if constexpr (FINE) dq[d] = Ops<T>::mma(kf, rest, dq[d]);
        }
      }
    }
  });
  if (!w.live) return;
  put<T, T, ND>(reinterpret_cast<T*>(a.dq) + w.b * a.dqs[0] + w.head * a.dqs[1] + w.t * a.dqs[2],
                dq, score_factor(a) * back, w.p < 0, a.D, h);
}

// Rows that look at the keys [k0, k0 + BM): the near ones, whose window
// reaches there, and, where the block holds sinks, the far ones behind them.
template <int KG>
struct RowRange {
  static constexpr int BM = 32 * KG;
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
    if (a.far_chunks == 0) n1 = f1;  // no far items: the block takes all rows
  }
};

constexpr int kSinkKeys = 32;  // keys of a far item

// fp32 sums of (group of sink keys, share) in AttnArgs::kvpart: share 0 from
// the near rows, 1 + i from chunk i of the far ones; [dk, dv][key][D]
__device__ __forceinline__ float* sink_part(const AttnArgs& a, int bh, int group, int share) {
  return a.kvpart + (((int64_t)bh * a.sink_groups + group) * (1 + a.far_chunks) + share) * 2 *
                        kSinkKeys * a.D;
}

// 64 rows of q and do with their statistics
template <typename T>
struct RowBuf {
  T *q, *g;
  float *lse, *delta;
};

template <typename T, int DP, int NW>
struct RowStream {
  typedef Dma<T, DP, NW> D;
  const T *q, *g;
  const float *lse, *delta;
  uint32_t qo[D::CH], go[D::CH];
  int wave;
  bool repeats;  // every tile begins with a token's first head
  __device__ __forceinline__ RowStream(const AttnArgs& a, int b, int hk, int wv) {
    wave = wv;
    q = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + hk * a.G * a.qs[1];
    g = reinterpret_cast<const T*>(a.dout) + b * a.dos[0] + hk * a.G * a.dos[1];
    const int64_t at = ((int64_t)b * a.Hkv + hk) * (a.Tq * a.G);
    lse = (kLifts<T> ? a.lse_keys : a.lse) + at;
    delta = a.delta + at;
    repeats = BN % a.G == 0;
    if (repeats) offsets(a, 0, BN, qo, go);
  }
  // of the tile's rows r0 .. r0 + BN - 1, from r0's token on
  __device__ __forceinline__ void offsets(const AttnArgs& a, int r0, int count, uint32_t (&x)[D::CH],
                                          uint32_t (&y)[D::CH]) const {
    const int t0 = Row(r0, a).t;
#pragma unroll
    for (int n = 0; n < D::CH; ++n) {
      const Row r(r0 + D::row(n), a);
      const bool in = D::row(n) < count;
      x[n] = in ? D::offset(n, (uint32_t)((r.g * a.qs[1] + (r.t - t0) * a.qs[2]) * sizeof(T)), a.D)
                : kNowhere;
      y[n] = in ? D::offset(n, (uint32_t)((r.g * a.dos[1] + (r.t - t0) * a.dos[2]) * sizeof(T)), a.D)
                : kNowhere;
    }
  }
  // rows [r0, r0 + BN) that lie before `end`; the others read as zeros (q
  // and do of 0 add nothing, whatever the statistics)
  __device__ __forceinline__ void fetch(const AttnArgs& a, int r0, int end, const RowBuf<T>& to) const {
    const int count = end - r0 < BN ? end - r0 : BN;
    const int t0 = Row(r0, a).t;
    const T *qb = q + t0 * a.qs[2], *gb = g + t0 * a.dos[2];
    if (repeats && count == BN) {
      D::run(to.q, qb, kNowhere - 1, wave, [&](int n) { return qo[n]; });
      D::run(to.g, gb, kNowhere - 1, wave, [&](int n) { return go[n]; });
    } else {
      uint32_t x[D::CH], y[D::CH];
      offsets(a, r0, count, x, y);
      D::run(to.q, qb, kNowhere - 1, wave, [&](int n) { return x[n]; });
      D::run(to.g, gb, kNowhere - 1, wave, [&](int n) { return y[n]; });
    }
    const int l = threadIdx.x & 63;
    if (wave < 2) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<float*>((wave == 0 ? lse : delta) + r0), (short)0, (count > 0 ? count : 0) * 4,
          0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(wave == 0 ? to.lse : to.delta), 4, l * 4,
          0, 0, 0);
    }
  }
};

// dk and dv: a wave owns 32 keys.  S = Q K^T and dP = dO V^T have a row's
// scores in register order, so dV^T += dO^T P and dK^T += Q^T dS take P and
// dS from where they are.
template <typename T, int DP, bool FINE>
struct KeyGrad {
  static constexpr int KD = DP / 16, ND = DP / 32;
  typedef typename Ops<T>::frag frag;
  static constexpr int kAhead = 4;
  frag kf[KD], vf[KD];
  v16f dk[ND], dv[ND];
  Lane<T, DP> at;
  // Probabilities carry 2^kKeyLift (in lse), their products with dP - delta
  // times `more` the power of two that suits them; k_back and v_back take both
  // out of the sums again.
  float more = 1.f, k_back = 1.f, v_back = 1.f;

  // A key that no row sees is taken for zeros, as the row kernels do: it may
  // hold anything, and 0 times that need not be 0.
  __device__ __forceinline__ void init(const AttnArgs& a, int b, int hk, int key,
                                       const KeyRows& kr) {
    const bool ok = kr.key_seen();
    if constexpr (kLifts<T>) {
      const int bh = b * a.Hkv + hk;
      const int lift = __builtin_amdgcn_readfirstlane(lift_of(bound_of(a, bh, 0), bound_of(a, bh, 1)));
      more = power2(lift - kKeyLift<T>);
      k_back = power2(-lift);
      v_back = power2(-kKeyLift<T>);
    }
    const int h = (threadIdx.x & 63) >> 5;
    const T* kp = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1] + key * a.ks[2];
    const T* vp = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1] + key * a.vs[2];
    // with a branch each: the sums' registers fall out worse without (heads of
    // 128: 200 us against 185)
    auto load = [&](const T* p, int d) {
      if (ok && d < a.D) return global_frag<T>(p, p, d, a.D, true);
      frag f;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (T)0.f;
      return f;
    };
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      kf[k] = load(kp, k * 16 + 8 * h);
      vf[k] = load(vp, k * 16 + 8 * h);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = zero16();
  }

  // 32 rows, r0 on, that lie in the tile from its row i0 on
  __device__ __forceinline__ void rows(const AttnArgs& a, const RowBuf<T>& b, int i0, int r0,
                                       const KeyRows& kr) {
    const int cover = kr.coverage(r0);
    if (cover == 0) return;
    const int h = (threadIdx.x & 63) >> 5;
    v16f s = zero16(), dp;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const v4f de = *reinterpret_cast<const v4f*>(b.delta + i0 + acc_row(e4 * 4, h));
#pragma unroll
      for (int i = 0; i < 4; ++i) dp[e4 * 4 + i] = de[i];
    }
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      s = Ops<T>::mma(row_frag<T, DP>(b.q, at, i0, k), kf[k], s);
      dp = Ops<T>::mma(row_frag<T, DP>(b.g, at, i0, k), vf[k], dp);
    }
    if (cover == 1) hide(s, kr.seen(r0, h));
    weigh(a, b, i0, s, dp);
    add(b, i0, s, dp);
  }

  // The 64 rows of a tile in one fixed sequence of products: those of one
  // half run beside the powers of the other, and a product's left operand is
  // read kAhead products before it.  The compiler's own order reads an operand
  // right before its product and keeps the powers apart from the products.
  // 8192 tokens, heads of 128: 217 -> 187 us (32% of the matrix units' time,
  // one wave a SIMD: an instruction of a lone wave takes 6 cycles to issue,
  // 33 ns for a product of 17 with all that goes with it); heads of 64: 69 ->
  // 67 us.  Reading 8 ahead, or a second copy of the sequence without masks,
  // is not faster (195, 227 us).
  __device__ __forceinline__ void rows64(const AttnArgs& a, const RowBuf<T>& b, int r0,
                                         const KeyRows& kr) {
    constexpr int HALF = 2 * KD, SUMS = 4 * ND, ALL = 2 * (HALF + SUMS);
    constexpr int E = (16 + HALF - 1) / HALF;  // powers beside a product
    const int h = (threadIdx.x & 63) >> 5;
    const float c = a.scale * kLog2e;
    auto left = [&](auto ic) {
      constexpr int i = decltype(ic)::value, j = i - 2 * HALF;
      if constexpr (i < 2 * HALF)
        return row_frag<T, DP>(i % 2 == 0 ? b.q : b.g, at, i / HALF * 32, i % HALF / 2);
      else
        return col_frag<T, DP>(i % 2 == 0 ? b.g : b.q, at, j / (2 * ND) * 16, j / 2 % ND * 32);
    };
    frag ring[kAhead];
    v16f s[2] = {zero16(), zero16()}, dp[2];
    v4f le[2][4];
    frag pf[2][2], sf[2][2];
#pragma unroll
    for (int sub = 0; sub < 2; ++sub)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4) {
        const v4f de = *reinterpret_cast<const v4f*>(b.delta + sub * 32 + acc_row(e4 * 4, h));
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[sub][e4 * 4 + i] = de[i];
      }
    const bool mixed[2] = {kr.coverage(r0) != 2, kr.coverage(r0 + 32) != 2};
    each<kAhead>([&](auto ic) { ring[decltype(ic)::value] = left(ic); });
    each<ALL>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      const frag f = ring[i % kAhead];
      if constexpr (i == HALF || i == 2 * HALF) {
        constexpr int sub = i / HALF - 1;
        if (mixed[sub]) hide(s[sub], kr.seen(r0 + sub * 32, h));
      }
      if constexpr (i < 2 * HALF) {
        constexpr int sub = i / HALF, k = i % HALF / 2;
        if constexpr (i % 2 == 0) s[sub] = Ops<T>::mma(f, kf[k], s[sub]);
        else dp[sub] = Ops<T>::mma(f, vf[k], dp[sub]);
      } else {
        constexpr int j = i - 2 * HALF, sub = j / SUMS, ss = j % SUMS / (2 * ND), d = j / 2 % ND;
        if constexpr (i % 2 == 0) dv[d] = Ops<T>::mma(f, pf[sub][ss], dv[d]);
        else dk[d] = Ops<T>::mma(f, sf[sub][ss], dk[d]);
      }
      if constexpr (i + kAhead < ALL)
        ring[i % kAhead] = left(std::integral_constant<int, i + kAhead>());
      // the first half's powers beside the second half's scores, the second
      // half's beside the first half's sums
      each<2>([&](auto subc) {
        constexpr int sub = decltype(subc)::value, o = i - HALF * (1 + sub) - 1;
        if constexpr (o == -2)
          each<4>([&](auto e4) {
            le[sub][e4] = *reinterpret_cast<const v4f*>(b.lse + sub * 32 + acc_row(e4 * 4, h));
          });
        if constexpr (o >= 0 && o * E < 16)
          each<E>([&](auto ec) {
            constexpr int e = o * E + decltype(ec)::value;
            if constexpr (e < 16) {
              const float x = __builtin_fmaf(s[sub][e], c, -le[sub][e / 4][e % 4]);
              s[sub][e] = ex2(x);
              dp[sub][e] *= kLifts<T> ? s[sub][e] * more : s[sub][e];
              if constexpr (e % 8 == 7) {
                pf[sub][e / 8] = acc_frag<T>(s[sub], e / 8);
                sf[sub][e / 8] = acc_frag<T>(dp[sub], e / 8);
              }
            }
          });
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // scores and dO V^T - delta become P and dS
  __device__ __forceinline__ void weigh(const AttnArgs& a, const RowBuf<T>& b, int i0, v16f& s,
                                        v16f& dp) {
    const int h = (threadIdx.x & 63) >> 5;
    const float c = a.scale * kLog2e;
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      const v4f le = *reinterpret_cast<const v4f*>(b.lse + i0 + acc_row(e4 * 4, h));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = e4 * 4 + i;
        s[e] = ex2(__builtin_fmaf(s[e], c, -le[i]));
        dp[e] *= kLifts<T> ? s[e] * more : s[e];
      }
    }
  }

  __device__ __forceinline__ void add(const RowBuf<T>& b, int i0, const v16f& s, const v16f& dp) {
#pragma unroll
    for (int ss = 0; ss < 2; ++ss) {
      const frag pf = acc_frag<T>(s, ss), sf = acc_frag<T>(dp, ss);
      frag rest;
      if constexpr (FINE) rest = acc_rest<T>(dp, ss, sf);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        dv[d] = Ops<T>::mma(col_frag<T, DP>(b.g, at, i0 + ss * 16, d * 32), pf, dv[d]);
        const frag qf = col_frag<T, DP>(b.q, at, i0 + ss * 16, d * 32);
        dk[d] = Ops<T>::mma(qf, sf, dk[d]);
        if constexpr (FINE) dk[d] = Ops<T>::mma(qf, rest, dk[d]);
      }
    }
  }
};

// blockIdx.y < key_blocks: the near rows of 32 KG keys, 32 a wave, the rows
// streamed in tiles of 64.  Above: a chunk of the far rows of 32 sink keys,
// which all waves own together, 32 rows each of a tile of one or two times
// 64; their sums are added in wave order.  Sinks are few and the rows behind the window
// many, so a far item has its rows spread over the waves and not its keys.
//
// KG groups of 32 keys and, for each, RS waves that take every RS-th 32 rows
// of a tile and add up at the end: where there are fewer waves than the chip
// can hold, a key's rows are the time that is left to divide.
template <typename T, int DP, int KG, int RS, bool FINE>
__global__ void __launch_bounds__(64 * KG * RS, (kKeyFit<T, DP>))
dkv_kernel(AttnArgs a, int key_blocks) {
  constexpr int ND = DP / 32, LD = kLd<T, DP>, NW = KG * RS, NT = 64 * NW, BM = 32 * KG;
  __shared__ __attribute__((aligned(16))) T Q0[BN * LD];
  __shared__ __attribute__((aligned(16))) T Q1[BN * LD];
  __shared__ __attribute__((aligned(16))) T G0[BN * LD];
  __shared__ __attribute__((aligned(16))) T G1[BN * LD];
  __shared__ __attribute__((aligned(16))) float L0[BN], L1[BN], D0[BN], D1[BN];
  static_assert(BN * LD * sizeof(T) >= kSinkKeys * DP * sizeof(float), "sums of a far item");
  static_assert(NW == 2 || NW == 4, "two waves or four");
  const RowBuf<T> b0{Q0, G0, L0, D0}, b1{Q1, G1, L1, D1};
  const int bh = blockIdx.x, b = bh / a.Hkv, hk = bh - b * a.Hkv;
  const int l = threadIdx.x & 63, h = l >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Seq seq = sequence(a, b);
  const RowStream<T, DP, NW> rs(a, b, hk, wave);
  KeyGrad<T, DP, FINE> kg;

  if ((int)blockIdx.y >= key_blocks) {
    const int item = (int)blockIdx.y - key_blocks;
    const int group = item / a.far_chunks, chunk = item - group * a.far_chunks;
    const int j0 = group * kSinkKeys, key = j0 + (l & 31);
    const RowRange<KG> rr(j0 / BM * BM, a, seq);
    const int tokens = (rr.f1 - rr.n1) / a.G;
    const int per = (tokens + a.far_chunks - 1) / a.far_chunks * a.G;
    const int ra = rr.n1 + per * chunk < rr.f1 ? rr.n1 + per * chunk : rr.f1;
    const int rb = ra + per < rr.f1 ? ra + per : rr.f1;
    const KeyRows kr(j0, key, a, seq);
    kg.init(a, b, hk, key, kr);
    for (int t0 = ra; t0 < rb; t0 += 32 * NW) {
      __syncthreads();
      rs.fetch(a, t0, rb, b0);
      if (NW > 2) rs.fetch(a, t0 + BN, rb, b1);
      arrived();
      kg.at.fresh();
      if (t0 + wave * 32 < rb)
        kg.rows(a, NW <= 2 || wave < 2 ? b0 : b1, (wave & 1) * 32, t0 + wave * 32, kr);
    }
    float* sk = reinterpret_cast<float*>(Q0);
    float* sv = reinterpret_cast<float*>(G0);
    for (int turn = 0; turn < NW; ++turn) {
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
      const v4f fv = *reinterpret_cast<const v4f*>(sv + kk * DP + d);
      const float f = a.scale * kg.k_back, g = kg.v_back;
      *reinterpret_cast<v4f*>(part + kk * a.D + d) = v4f{fk[0] * f, fk[1] * f, fk[2] * f, fk[3] * f};
      *reinterpret_cast<v4f*>(part + (kSinkKeys + kk) * a.D + d) =
          v4f{fv[0] * g, fv[1] * g, fv[2] * g, fv[3] * g};
    }
    return;
  }

  const int k0 = (int)blockIdx.y * BM, group = wave % KG, turn = wave / KG;
  const RowRange<KG> rr(k0, a, seq);
  const int key = k0 + group * 32 + (l & 31);
  const KeyRows kr(k0 + group * 32, key, a, seq);
  kg.init(a, b, hk, key, kr);
  auto step = [&](const RowBuf<T>& buf, int t0) {
    kg.at.fresh();
    if constexpr (RS == 1 && sizeof(T) == 2 && !FINE) {
      if (kr.coverage(t0) != 0 || kr.coverage(t0 + 32) != 0) kg.rows64(a, buf, t0, kr);
      return;
    }
#pragma unroll
    for (int sub = 0; sub < BN / 32; sub += RS) {
      const int i0 = (sub + (RS > 1 ? turn : 0)) * 32;
      kg.rows(a, buf, i0, t0 + i0, kr);
    }
  };
  if (rr.n0 < rr.n1) rs.fetch(a, rr.n0, rr.n1, b0);
  for (int t0 = rr.n0; t0 < rr.n1; t0 += 2 * BN) {
    arrived();
    if (t0 + BN < rr.n1) rs.fetch(a, t0 + BN, rr.n1, b1);
    step(b0, t0);
    if (t0 + BN >= rr.n1) break;
    arrived();
    if (t0 + 2 * BN < rr.n1) rs.fetch(a, t0 + 2 * BN, rr.n1, b0);
    step(b1, t0 + BN);
  }
  if (RS > 1) {
    float* sk = reinterpret_cast<float*>(group == 0 ? Q0 : Q1) + l * 4;
    float* sv = reinterpret_cast<float*>(group == 0 ? G0 : G1) + l * 4;
    __syncthreads();
    if (turn == 1)
#pragma unroll
      for (int i = 0; i < 4 * ND; ++i) {
        *reinterpret_cast<v4f*>(sk + i * 256) = quad_of(kg.dk[i / 4], i % 4);
        *reinterpret_cast<v4f*>(sv + i * 256) = quad_of(kg.dv[i / 4], i % 4);
      }
    __syncthreads();
    if (turn == 1) return;
#pragma unroll
    for (int i = 0; i < 4 * ND; ++i) {
      const v4f fk = *reinterpret_cast<const v4f*>(sk + i * 256);
      const v4f fv = *reinterpret_cast<const v4f*>(sv + i * 256);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kg.dk[i / 4][i % 4 * 4 + e] += fk[e];
        kg.dv[i / 4][i % 4 * 4 + e] += fv[e];
      }
    }
  }
  const float f = score_factor(a) * kg.k_back;
  if (a.far_chunks > 0 && key < a.S) {
    float* part = sink_part(a, bh, key / kSinkKeys, 0) + key % kSinkKeys * a.D;
    put<T, float, ND>(part, kg.dk, f, false, a.D, h);
    put<T, float, ND>(part + kSinkKeys * a.D, kg.dv, kg.v_back, false, a.D, h);
  } else if (key < a.Tk) {
    put<T, T, ND>(reinterpret_cast<T*>(a.dk) + b * a.dks[0] + hk * a.dks[1] + key * a.dks[2],
                  kg.dk, f, false, a.D, h);
    put<T, T, ND>(reinterpret_cast<T*>(a.dv) + b * a.dvs[0] + hk * a.dvs[1] + key * a.dvs[2],
                  kg.dv, kg.v_back, false, a.D, h);
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

template <typename T, int DP>
void forward_dp(const AttnArgs& a, hipStream_t st) {
  constexpr int NW = kRowWaves;
  const dim3 grid((unsigned)(a.B * a.Hkv), (unsigned)ceil_div((int64_t)a.Tq * a.G, 32 * NW),
                  (unsigned)a.splits);
  if (a.splits > 1) {
    fwd_kernel<T, DP, NW, true><<<grid, 64 * NW, 0, st>>>(a);
    join_kernel<T><<<(unsigned)(a.B * a.Hq * a.Tq), NT, 0, st>>>(a);
  } else {
    fwd_kernel<T, DP, NW, false><<<grid, 64 * NW, 0, st>>>(a);
  }
}

template <typename T, int DP, bool FINE>
void backward_fine(const AttnArgs& a, hipStream_t st) {
  constexpr int QN = kRowWaves, KG = kKeyWaves<DP>;
  const unsigned bh = (unsigned)(a.B * a.Hkv);
  dq_kernel<T, DP, QN, FINE><<<dim3(bh, (unsigned)ceil_div((int64_t)a.Tq * a.G, 32 * QN)), 64 * QN,
                               0, st>>>(a);
  const int kb = (int)ceil_div(a.Tk, 32 * KG);
  const dim3 grid(bh, (unsigned)(kb + a.sink_groups * a.far_chunks));
  // up to one wave a SIMD: two share a group of keys (fp32 padded batch, 520
  // waves: 60 -> 44 us)
  if (KG == 2 && (int64_t)bh * kb * KG <= 1024)
    dkv_kernel<T, DP, KG, KG == 2 ? 2 : 1, FINE><<<grid, 64 * KG * 2, 0, st>>>(a, kb);
  else
    dkv_kernel<T, DP, KG, 1, FINE><<<grid, 64 * KG, 0, st>>>(a, kb);
  if (a.far_chunks > 0) {
    const int64_t n = (int64_t)bh * a.S * 2 * (a.D / 4);
    join_kv_kernel<T><<<(unsigned)ceil_div(n, NT), NT, 0, st>>>(a);
  }
}

template <typename T, int DP>
void backward_dp(const AttnArgs& a, hipStream_t st) {
  if constexpr (sizeof(T) == 2)
    if (a.rest != nullptr) return backward_fine<T, DP, true>(a, st);
  backward_fine<T, DP, false>(a, st);
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

// dP - delta is small where few keys share the weight, and two roundings then
// weigh in the gradients of q and k: that of o, which delta goes by, and that
// of P (dP - delta) itself.  With a window of 2 and neither mended they are off
// by 0.0037 of their norm (bf16), of 6 0.0027, of 30 0.0025; with delta counting
// what o's rounding took away by 0.0025 at each, and with the product taken in
// two parts (FINE: two matrix instructions for one, and no rows64) by 0.0018,
// where their own rounding is 0.0017.  The first rows of a short sequence see
// as few keys.  GPT-NeoX batch with window 100: 135 us without the two parts,
// 142 with; 8192 tokens, heads of 128, window 100: 171, 194.  Over 128 keys
// neither is done (0.0025; window 256, delta's part alone: 155 -> 171 us).
bool attn_keeps_rest(const AttnArgs& a) { return std::min<int64_t>((int64_t)a.W + a.S, a.Tk) <= 128; }

void attn_plan(const AttnArgs& a, int* splits, int64_t* floats) {
  const int64_t rows = (int64_t)a.Tq * a.G;
  const int64_t blocks = (int64_t)a.B * a.Hkv * ceil_div(rows, 32 * kRowWaves);
  // tiles that the longest row block can see
  const int64_t most = ceil_div(std::min<int64_t>((int64_t)a.W + 128, a.Tk), BN) +
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
  // far rows exist only behind the window of a sink's key; up to 512 rows
  // (8 tiles) the block of keys takes them itself: a launch that adds up the
  // shares costs more (2 x 64 tokens, 4 heads of 16: 17 us for the pass
  // against 20)
  if (a.S <= 0 || a.W >= a.Tk || (int64_t)a.Tq * a.G <= 512) return;
  const int64_t groups = ceil_div(a.S, kSinkKeys), bh = (int64_t)a.B * a.Hkv;
  // chunks of at least two tiles until there are items for 4 blocks a CU
  int64_t ch = ceil_div(1024, bh * groups);
  ch = std::min(ch, ceil_div((int64_t)a.Tq * a.G, 256));
  ch = std::max<int64_t>(1, std::min<int64_t>(ch, 32));
  *sink_groups = (int)groups;
  *far_chunks = (int)ch;
  *floats = bh * groups * (1 + ch) * 2 * kSinkKeys * a.D;
}

int attn_bound_chunks(int dtype, const AttnArgs& a) {
  if (dtype != kF16) return 0;
  // a wave reads them all at once
  const int64_t most = std::max<int64_t>((int64_t)a.Tq * a.G, a.Tk);
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(most, 256), 64));
}

void attn_backward(int dtype, const AttnArgs& a, hipStream_t st) {
  if ((int64_t)a.B * a.Hkv * a.Tk == 0 || a.Tq == 0) return;
  if (dtype == kBF16) {
    backward_type<__bf16>(a, st);
  } else if (dtype == kF16) {
    bounds_kernel<_Float16><<<dim3((unsigned)(a.B * a.Hkv), (unsigned)a.bound_chunks), NT, 0, st>>>(a);
    backward_type<_Float16>(a, st);
  } else {
    backward_type<float>(a, st);
  }
}

}  // namespace kfac

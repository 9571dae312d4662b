// Distillation from a teacher's top logits (ops/distill.py).
//
// Student row z of V logits, temperature T, u = z / T; teacher entries
// (index_k, t_k), k < K, and optionally the log-sum rest of its other
// logits.  p = softmax over (t_k / T, rest), r the part of the rest,
// I the set of the row's indices, q = softmax(u), R = sum of q outside I:
//
//   loss = T^2 [ sum_k p_k (ln p_k - ln q_k) + r (ln r - ln R) ]
//   dloss/dz_j = T (q_j - sum_{k: index_k = j} p_k)   j in I
//              = T q_j (1 - r / R)                    elsewhere
//
// Without a rest r = 0 and both are the divergence from the teacher's
// renormalised top entries.  R is summed over the columns outside I, not
// formed as 1 - sum of the others: next to 1 that difference has no digits
// left.  The columns of I are told apart by a bitmap of the block's slice
// of the row in LDS, one bit a column.
//
// All of it is bound by memory.  Where a backward pass is to follow and
// there are rows for the whole chip, a row's logits are read once into the
// registers of one block (1024 threads hold 16 x 16 bytes each: 131072
// 16-bit logits), which forms the statistics and writes the gradient from
// there: one read and one write of [N, V], with the factors of the loss that
// are known by then (mean, weight).  A factor that the caller puts on the
// loss afterwards is multiplied into the gradient in place by the backward
// pass, which costs a read and a write more and, where it is no power of
// two, a second rounding.  16384 rows of 50304 bf16 logits: 0.67 ms for loss
// and gradient, 4.9 TB/s, a copy's rate.  The other calls (fp16, whose range does not hold
// the unscaled gradient of a mean over thousands of rows; few rows, each cut
// into slices; reduction 'none'; more columns) read the logits once forward
// and once more backward.
#include "common.h"

#include "lm_ops.h"

#include <algorithm>

namespace kfac {

namespace {

constexpr int NT = 256;
constexpr int kMaxK = 1024;
constexpr int kMaxVpt = 16;  // 16-byte accesses that each of
constexpr int kMaxRowThreads = 1024;  // threads of row_kernel holds, at most
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
#define KFAC_NEG_INF (-__builtin_inff())

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename E> __device__ __forceinline__ float up(E v) { return (float)v; }

template <typename E> struct Wide { static constexpr int N = 16 / (int)sizeof(E); };

// N elements from p: one 16-byte access where rows are aligned, and where
// the row length is odd the widest one that the element's alignment allows
template <typename E, bool ALIGNED>
__device__ __forceinline__ void load_wide(const E* p, float* f) {
  constexpr int N = Wide<E>::N;
  typedef E vec __attribute__((ext_vector_type(N)));
  typedef vec uvec __attribute__((aligned(sizeof(E))));
  const vec v = ALIGNED ? *reinterpret_cast<const vec*>(p)
                        : (vec)*reinterpret_cast<const uvec*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = up<E>(v[i]);
}

template <typename E, bool ALIGNED>
__device__ __forceinline__ void store_wide(E* p, const float* f) {
  constexpr int N = Wide<E>::N;
  typedef E vec __attribute__((ext_vector_type(N)));
  typedef vec uvec __attribute__((aligned(sizeof(E))));
  vec v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (E)f[i];
  if (ALIGNED) *reinterpret_cast<vec*>(p) = v;
  else *reinterpret_cast<uvec*>(p) = v;
}

// A sum of powers, as (base m, sum s of 2^(y - m)); s = 0 is empty.  It stays
// in two parts to the end: m + log2 s rounds to a step of m's size, which
// would put the same 2^-24 m on every probability of the row.
struct Run {
  float m, s;
  // 2^(b - base) with b as it was rounded: contracted with the product that
  // formed either, the difference of two equal numbers would be that rounding
  __device__ __forceinline__ static float down(float b, float base) {
#pragma clang fp contract(off)
    return ex2(b - base);
  }
  __device__ __forceinline__ void join(float m2, float s2) {
    const float mm = fmaxf(m, m2);
    const float base = mm == KFAC_NEG_INF ? 0.f : mm;
    s = s * down(m, base) + s2 * down(m2, base);
    m = mm;
  }
  // 2^(x c), the product not rounded
  __device__ __forceinline__ void add(float x, float c) {
    const float y = x * c;
    join(y, y == KFAC_NEG_INF ? 0.f : ex2(__builtin_fmaf(x, c, -y)));
  }
  // 2^(x c) as a part of the sum
  __device__ __forceinline__ float part(float x, float c) const {
    return ex2(__builtin_fmaf(x, c, -m)) / s;
  }
  __device__ __forceinline__ float log2part(float x, float c) const {
    return __builtin_fmaf(x, c, -m) - log2f(s);
  }
};

__device__ __forceinline__ Run joined(Run a, Run b) {
  a.join(b.m, b.s);
  return a;
}

__device__ __forceinline__ Run wave_join(Run r) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float m2 = __shfl_xor(r.m, off, 64), s2 = __shfl_xor(r.s, off, 64);
    r.join(m2, s2);
  }
  return r;
}

// The floor of finite logits, for the lowest value of bf16 or fp32 that a row
// may be masked with: its product with c passes the end of fp32 or has no
// digits left to cancel.  -2^30 over c, or 2^24 where that is more, rounded to
// a power of two, so that its own product with c is exact.  Beside a logit
// above it everything at it has probability 0; a row with none above it
// ("floored") is uniform over its finite logits.  That takes no operation of
// the loops over a row: their bases are kept at the floor or above, and a row
// whose base is the floor is counted once more.
__device__ __forceinline__ float floor_of(float c) {
  const int e = 30 - __builtin_amdgcn_frexp_expf(c);
  return -__builtin_amdgcn_ldexpf(1.f, e > 24 ? e : 24);
}
__device__ __forceinline__ float floored(float x, float low) {
  return x == KFAC_NEG_INF ? x : fmaxf(x, low) + (x - x);  // NaN stays
}

__device__ __forceinline__ int64_t index_at(const DistillArgs& a, int64_t i) {
  return a.index64 ? reinterpret_cast<const int64_t*>(a.index)[i]
                   : (int64_t)reinterpret_cast<const int32_t*>(a.index)[i];
}

template <typename E>
__device__ __forceinline__ const E* row_of(const DistillArgs& a, int64_t n) {
  return reinterpret_cast<const E*>(a.z) + (n / a.inner) * a.zs0 + (n % a.inner) * a.zs1;
}

// nothing above the floor, and no NaN
__device__ __forceinline__ bool is_floored(const Run& all, float low, float c) {
  return all.m <= low * c && all.s == all.s;
}

// A row's statistics, as the backward pass finds them.
struct RowInfo {
  Run all, tail;  // the student's columns; those outside I (with a rest)
  Run teacher;
  float r;        // the rest's share of the teacher; -1: the row does not count
  float unused;
};

__device__ __forceinline__ RowInfo load_info(const DistillArgs& a, int64_t n) {
  const float4 u = a.info[2 * n], v = a.info[2 * n + 1];
  return RowInfo{{u.x, u.y}, {u.z, u.w}, {v.x, v.y}, v.z, v.w};
}

__device__ __forceinline__ void store_info(const DistillArgs& a, int64_t n, const RowInfo& i) {
  a.info[2 * n] = make_float4(i.all.m, i.all.s, i.tail.m, i.tail.s);
  a.info[2 * n + 1] = make_float4(i.teacher.m, i.teacher.s, i.r, i.unused);
}

// the log-sum of the teacher's other logits
__device__ __forceinline__ float rest_of(const DistillArgs& a, int64_t n) {
  return a.rest != nullptr ? floored(a.rest[n], floor_of(kLog2e)) : KFAC_NEG_INF;
}

// The teacher's part of a row's info, by one wave.  An index behind the
// vocabulary makes the teacher's sum NaN, and with it the loss and gradient.
__device__ __forceinline__ void teacher_of(const DistillArgs& a, int64_t n, RowInfo& info) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / a.temperature;
  const float low = floor_of(c);
  const float rest = rest_of(a, n);
  Run t{KFAC_NEG_INF, 0.f};
  bool some = false, far = false;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t j = index_at(a, n * a.K + k);
    if (j < 0) continue;
    some = true;
    far |= j >= a.V;
    t.add(floored(a.teacher[n * a.K + k], low), c);
  }
  t = wave_join(t);
  t.add(rest, kLog2e);
  if (__any(far)) t.s = __builtin_nanf("");
  info.teacher = t;
  info.r = !__any(some) || t.s == 0.f ? -1.f
           : rest == KFAC_NEG_INF     ? 0.f
                                      : t.part(rest, kLog2e);
}

// A row's loss, by one wave; raw(k, j) is the student's logit of entry k.
// Each entry's two log-probabilities meet before they are weighted: apart,
// the rounding of the weights would be multiplied by the row's logarithm.
template <typename F>
__device__ __forceinline__ float row_loss(const DistillArgs& a, int64_t n, const RowInfo& i,
                                          F raw) {
  const float c = kLog2e / a.temperature, low = floor_of(c);
  float loss = 0.f;
  for (int k = threadIdx.x & 63; k < a.K; k += 64) {
    const int64_t j = index_at(a, n * a.K + k);
    if (j < 0 || j >= a.V) continue;
    const float tl = floored(a.teacher[n * a.K + k], low);
    const float p = i.teacher.part(tl, c);
    if (p > 0.f)
      loss += p * (i.teacher.log2part(tl, c) - i.all.log2part(floored(raw(k, j), low), c));
  }
  loss = wave_reduce_sum(loss);
  if (i.r > 0.f)
    loss += i.r * (i.teacher.log2part(rest_of(a, n), kLog2e) -
                   ((i.tail.m - i.all.m) + (log2f(i.tail.s) - log2f(i.all.s))));
  // p = 0 terms drop out, but not what makes the row undefined
  if (i.all.s != i.all.s || i.all.s == 0.f || i.teacher.s != i.teacher.s) loss = __builtin_nanf("");
  return i.r < 0.f ? 0.f : loss * kLn2 * a.temperature * a.temperature;
}

template <typename E>
__device__ void finish_row(const DistillArgs& a, int64_t n, const Run& all, const Run& tail) {
  RowInfo info{all, tail, {0.f, 0.f}, 0.f, 0.f};
  teacher_of(a, n, info);
  const E* z = row_of<E>(a, n);
  const float loss = row_loss(a, n, info, [&](int, int64_t j) { return up<E>(z[j]); });
  if ((threadIdx.x & 63) == 0) {
    store_info(a, n, info);
    a.row_loss[n] = loss;
  }
}

// The gradient of the columns outside I is f power(x).
struct Outside {
  float base, f;
  __device__ __forceinline__ Outside(const RowInfo& i, float g, bool rest) {
    if (rest && i.tail.s > 0.f) {
      const float share = i.tail.s * ex2(i.tail.m - i.all.m) / i.all.s;  // R
      base = i.tail.m;
      f = g * (share - i.r) / i.tail.s;
    } else {
      base = i.all.m;
      f = g / i.all.s;
    }
    if (i.teacher.s != i.teacher.s) f = i.teacher.s;
  }
  __device__ __forceinline__ float power(float x, float c) const {
    return ex2(__builtin_fmaf(x, c, -base));
  }
  // of a floored row: uniform over its finite logits
  __device__ __forceinline__ float flat(float x) const { return x > KFAC_NEG_INF ? 1.f : 0.f; }
};

// Statistics of a slice of a row: part = {tail m, s, member m, s}.
template <typename E, bool ALIGNED, bool REST>
__global__ void __launch_bounds__(NT) stats_kernel(DistillArgs a) {
  constexpr int N = Wide<E>::N;
  constexpr int U = 4;  // accesses in flight
  extern __shared__ uint32_t bits[];
  __shared__ float4 red[NT / 64];
  const int64_t n = blockIdx.x / a.splits;
  const int64_t c0 = (int64_t)(blockIdx.x % a.splits) * a.slice;
  const int64_t c1 = c0 + a.slice < a.V ? c0 + a.slice : a.V;
  const int tid = threadIdx.x;
  const E* z = row_of<E>(a, n);
  const float c = kLog2e / a.temperature;

  if (REST) {
    const int words = (int)((c1 - c0 + 31) >> 5);
    for (int w = tid; w < words; w += NT) bits[w] = 0;
    __syncthreads();
  }
  int some = 0;
  for (int k = tid; k < a.K; k += NT) {
    const int64_t j = index_at(a, n * a.K + k);
    some |= j >= 0;
    if (REST && j >= c0 && j < c1)
      atomicOr(&bits[(j - c0) >> 5], 1u << ((j - c0) & 31));
  }
  some = __syncthreads_or(some);

  const float low = floor_of(c);
  Run out{KFAC_NEG_INF, 0.f}, in{KFAC_NEG_INF, 0.f};
  float raw = low;  // largest logit so far, the floor at least
  if (some) {
    const int64_t nv = (c1 - c0) / N;
    for (int64_t v0 = tid; v0 < nv; v0 += (int64_t)NT * U) {
      float y[U][N];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const int64_t v = v0 + (int64_t)q * NT;
        if (v < nv) {
          load_wide<E, ALIGNED>(z + c0 + v * N, y[q]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) y[q][i] = KFAC_NEG_INF;
        }
      }
      float mx = raw;
#pragma unroll
      for (int q = 0; q < U; ++q) {
        if (REST) {
          const int64_t v = v0 + (int64_t)q * NT;
          const int at = (int)(v * N);
          const uint32_t b = v < nv ? (bits[at >> 5] >> (at & 31)) & ((1u << N) - 1u) : 0u;
          if (b != 0) {  // rare: K columns of V
#pragma unroll
            for (int i = 0; i < N; ++i)
              if ((b >> i) & 1u) {
                in.add(floored(y[q][i], low), c);
                y[q][i] = KFAC_NEG_INF;
              }
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) mx = fmaxf(mx, y[q][i]);
      }
      raw = mx;
      const float m = mx * c;
      float s = out.s * Run::down(out.m, m);
#pragma unroll
      for (int q = 0; q < U; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i) s += ex2(__builtin_fmaf(y[q][i], c, -m));
      out.s = s;
      out.m = m;
    }
    const int64_t rem = c0 + nv * N + tid;  // the last, partial access
    if (rem < c1) {
      const int at = (int)(rem - c0);
      const bool member = REST && ((bits[at >> 5] >> (at & 31)) & 1u);
      (member ? in : out).add(floored(up<E>(z[rem]), low), c);
    }
  }
  out = wave_join(out);
  if (REST) in = wave_join(in);
  if ((tid & 63) == 0) red[tid >> 6] = make_float4(out.m, out.s, in.m, in.s);
  __syncthreads();
  out = Run{red[0].x, red[0].y};
  in = Run{red[0].z, red[0].w};
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) {
    out.join(red[w].x, red[w].y);
    in.join(red[w].z, red[w].w);
  }
  if (some && is_floored(joined(out, in), low, c)) {
    float count = 0.f;
    for (int64_t i = c0 + tid; i < c1; i += NT) {
      const bool member = REST && ((bits[(i - c0) >> 5] >> ((i - c0) & 31)) & 1u);
      count += !member && up<E>(z[i]) > KFAC_NEG_INF ? 1.f : 0.f;
    }
    count = wave_reduce_sum(count);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6].x = count;
    __syncthreads();
    out = Run{low * c, 0.f};
    for (int w = 0; w < NT / 64; ++w) out.s += red[w].x;
  }
  if (tid >= 64) return;
  if (a.splits > 1) {
    if (tid == 0) a.part[blockIdx.x] = make_float4(out.m, out.s, in.m, in.s);
    return;
  }
  finish_row<E>(a, n, REST ? joined(out, in) : out, out);
}

// rows of several slices: one wave joins them, in order
template <typename E, bool REST>
__global__ void __launch_bounds__(64) join_kernel(DistillArgs a) {
  const int64_t n = blockIdx.x;
  Run out{KFAC_NEG_INF, 0.f}, in{KFAC_NEG_INF, 0.f};
  for (int q = threadIdx.x; q < a.splits; q += 64) {
    const float4 p = a.part[n * a.splits + q];
    out.join(p.x, p.y);
    if (REST) in.join(p.z, p.w);
  }
  out = wave_join(out);
  if (REST) in = wave_join(in);
  finish_row<E>(a, n, REST ? joined(out, in) : out, out);
}

// sum or mean of the rows' losses (loss null: not yet known), and the factor
// of a row's gradient (weight, or weight / rows that count); 64-bit sums in a
// fixed order
__global__ void __launch_bounds__(1024) reduce_kernel(const float* row_loss, const float4* info,
                                                      int64_t N, int mean, float weight,
                                                      float* loss, float* factor) {
  __shared__ double sum[16];
  __shared__ double cnt[16];
  double s = 0.0, c = 0.0;
  for (int64_t n = threadIdx.x; n < N; n += 1024) {
    s += loss != nullptr ? row_loss[n] : 0.f;
    c += info[2 * n + 1].z < 0.f ? 0.0 : 1.0;
  }
  s = wave_reduce_sum(s);
  c = wave_reduce_sum(c);
  if ((threadIdx.x & 63) == 0) {
    sum[threadIdx.x >> 6] = s;
    cnt[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = c = 0.0;
    for (int i = 0; i < 16; ++i) {
      s += sum[i];
      c += cnt[i];
    }
    const double f = (mean ? 1.0 / (c > 0.0 ? c : 1.0) : 1.0) * weight;
    if (loss != nullptr) *loss = (float)(s * f);
    if (factor != nullptr) *factor = (float)f;
  }
}

// the teacher's side of every row, one wave each, before the fused kernel
__global__ void __launch_bounds__(NT) teacher_kernel(DistillArgs a) {
  const int64_t n = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
  if (n >= a.N) return;
  RowInfo info{{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, 0.f, 0.f};
  teacher_of(a, n, info);
  if ((threadIdx.x & 63) == 0) store_info(a, n, info);
}

// Keeps 16 bytes packed: without it the compiler carries their fp32 values,
// twice the registers, from the statistics to the gradient.
template <typename V>
__device__ __forceinline__ void stay_packed(V& x) {
  uint4 u = __builtin_bit_cast(uint4, x);
  asm volatile("" : "+v"(u.x), "+v"(u.y), "+v"(u.z), "+v"(u.w));
  x = __builtin_bit_cast(V, u);
}

// A row in one block: its logits stay in registers between the statistics
// and the gradient.
// Waves a SIMD are chosen so that two blocks or more share a CU where their
// logits leave the registers for it: one loads while another forms its sums.
template <typename E, int VPT, int kRowThreads, bool ALIGNED, bool REST>
__global__ void __launch_bounds__(kRowThreads, VPT <= 7 ? 8 : 4)
row_kernel(DistillArgs a) {
  constexpr int N = Wide<E>::N;
  extern __shared__ uint32_t bits[];  // with a rest: one bit a column
  __shared__ float4 red[kRowThreads / 64];
  __shared__ int at[kMaxK];     // the entries' columns, -1: none
  __shared__ float pk[kMaxK];   // their share of the teacher
  __shared__ float xk[kMaxK];   // the student's logits there
  __shared__ float pj[kMaxK];   // the teacher's share of the column, all entries that name it
  const int64_t n = blockIdx.x;
  const int tid = threadIdx.x, V = (int)a.V, nv = V / N;
  const E* z = row_of<E>(a, n);
  E* d = reinterpret_cast<E*>(a.dz) + n * a.V;
  const float c = kLog2e / a.temperature;
  RowInfo info = load_info(a, n);
  typedef E vec __attribute__((ext_vector_type(N)));
  typedef vec uvec __attribute__((aligned(sizeof(E))));
  auto put = [&](E* p, const vec& x) {
    if (ALIGNED) *reinterpret_cast<vec*>(p) = x;
    else *reinterpret_cast<uvec*>(p) = x;
  };
  if (info.r < 0.f) {  // the row does not count (a NaN does)
    vec zero;
#pragma unroll
    for (int i = 0; i < N; ++i) zero[i] = (E)0.f;
    for (int v = tid; v < nv; v += kRowThreads) put(d + (int64_t)v * N, zero);
    if (nv * N + tid < V) d[nv * N + tid] = (E)0.f;
    if (tid == 0) a.row_loss[n] = 0.f;
    return;
  }
  vec x[VPT];
#pragma unroll
  for (int q = 0; q < VPT; ++q) {
    const int v = tid + q * kRowThreads;
    if (v < nv)
      x[q] = ALIGNED ? *reinterpret_cast<const vec*>(z + (int64_t)v * N)
                     : (vec)*reinterpret_cast<const uvec*>(z + (int64_t)v * N);
    else
#pragma unroll
      for (int i = 0; i < N; ++i) x[q][i] = (E)KFAC_NEG_INF;
  }
  const int rem = nv * N + tid;  // the last, partial access
  const float last = rem < V ? up<E>(z[rem]) : KFAC_NEG_INF;
  if (REST) {
    for (int w = tid; w < (V + 31) / 32; w += kRowThreads) bits[w] = 0;
    __syncthreads();
  }
  for (int k = tid; k < a.K; k += kRowThreads) {
    const int64_t j = index_at(a, n * a.K + k);
    const bool in = j >= 0 && j < V;
    at[k] = in ? (int)j : -1;
    pk[k] = in ? info.teacher.part(floored(a.teacher[n * a.K + k], floor_of(c)), c) : 0.f;
    xk[k] = in ? up<E>(z[j]) : 0.f;
    if (REST && in) atomicOr(&bits[j >> 5], 1u << (j & 31));
  }
  __syncthreads();
  {
    // an index given twice counts with both its parts: `team` lanes of a wave
    // add up the entries that name the column of entry k (with more entries
    // than threads, those of entry k + kRowThreads afterwards)
    int team = 64;
    while (team > 1 && team * a.K > kRowThreads) team >>= 1;
    const int part = tid & (team - 1);
    for (int k0 = 0; k0 < a.K; k0 += kRowThreads / team) {
      const int k = k0 + tid / team;
      float p = 0.f;
      if (k < a.K && at[k] >= 0)
        for (int i = part; i < a.K; i += team) p += at[i] == at[k] ? pk[i] : 0.f;
      for (int off = team >> 1; off > 0; off >>= 1) p += __shfl_xor(p, off, 64);
      if (k < a.K && part == 0) pj[k] = p;
    }
  }
  const float low = floor_of(c);
  Run out{KFAC_NEG_INF, 0.f}, in{KFAC_NEG_INF, 0.f};
  float raw = low;  // largest logit so far, the floor at least
#pragma unroll
  for (int q = 0; q < VPT; ++q) {
    if (REST) {
      const int col = (tid + q * kRowThreads) * N;
      const uint32_t b = col < V ? (bits[col >> 5] >> (col & 31)) & ((1u << N) - 1u) : 0u;
      if (b != 0) {  // rare: K columns of V; their gradient is written below
#pragma unroll
        for (int i = 0; i < N; ++i)
          if ((b >> i) & 1u) {
            in.add(floored(up<E>(x[q][i]), low), c);
            x[q][i] = (E)KFAC_NEG_INF;
          }
      }
      stay_packed(x[q]);
    }
    float y[N], mx = raw;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      y[i] = up<E>(x[q][i]);
      mx = fmaxf(mx, y[i]);
    }
    raw = mx;
    const float m = mx * c;
    float s = out.s * Run::down(out.m, m);
#pragma unroll
    for (int i = 0; i < N; ++i) s += ex2(__builtin_fmaf(y[i], c, -m));
    out.s = s;
    out.m = m;
  }
  if (rem < V) {
    const bool member = REST && ((bits[rem >> 5] >> (rem & 31)) & 1u);
    (member ? in : out).add(floored(last, low), c);
  }
  out = wave_join(out);
  if (REST) in = wave_join(in);
  if ((tid & 63) == 0) red[tid >> 6] = make_float4(out.m, out.s, in.m, in.s);
  __syncthreads();
  out = Run{red[0].x, red[0].y};
  in = Run{red[0].z, red[0].w};
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) {
    out.join(red[w].x, red[w].y);
    if (REST) in.join(red[w].z, red[w].w);
  }
  info.all = REST ? joined(out, in) : out;
  const bool flat = is_floored(info.all, low, c);
  if (flat) {
    float count = 0.f;
    for (int i = tid; i < V; i += kRowThreads) {
      const bool member = REST && ((bits[i >> 5] >> (i & 31)) & 1u);
      count += !member && up<E>(z[i]) > KFAC_NEG_INF ? 1.f : 0.f;
    }
    count = wave_reduce_sum(count);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6].x = count;
    __syncthreads();
    out = Run{low * c, 0.f};
    for (int w = 0; w < kRowThreads / 64; ++w) out.s += red[w].x;
    info.all = REST ? joined(out, in) : out;
  }
  info.tail = out;
  const float g = a.temperature * a.mean[0];
  const Outside o(info, g, REST);
  if (flat) {
    for (int i = tid; i < V; i += kRowThreads) d[i] = (E)(o.f * o.flat(up<E>(z[i])));
  } else {
#pragma unroll
    for (int q = 0; q < VPT; ++q) {
      const int v = tid + q * kRowThreads;
      stay_packed(x[q]);
      if (v < nv) {
        vec y;
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = (E)(o.f * o.power(up<E>(x[q][i]), c));
        put(d + (int64_t)v * N, y);
      }
    }
    if (rem < V) d[rem] = (E)(o.f * o.power(last, c));
  }
  if (tid < 64) {
    const float loss = row_loss(a, n, info, [&](int k, int64_t) { return xk[k]; });
    if (tid == 0) {
      a.row_loss[n] = loss;
      store_info(a, n, info);
    }
  }
  __syncthreads();
  const float nan = info.teacher.s != info.teacher.s ? info.teacher.s : 0.f;
  for (int k = tid; k < a.K; k += kRowThreads)
    if (at[k] >= 0) d[at[k]] = (E)(g * (info.all.part(floored(xk[k], low), c) - pj[k]) + nan);
}

// dz *= *factor, in place; nothing to do where that is 1
template <typename E>
__global__ void __launch_bounds__(NT) scale_kernel(E* dz, int64_t n, const float* factor) {
  constexpr int N = Wide<E>::N;
  const float f = *factor;
  if (f == 1.f) return;
  const int64_t nv = n / N;
  for (int64_t v = (int64_t)blockIdx.x * NT + threadIdx.x; v < nv; v += (int64_t)gridDim.x * NT) {
    float y[N];
    load_wide<E, true>(dz + v * N, y);
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] *= f;
    store_wide<E, true>(dz + v * N, y);
  }
  const int64_t rem = nv * N + threadIdx.x;
  if (blockIdx.x == 0 && rem < n) dz[rem] = (E)(up<E>(dz[rem]) * f);
}

// dz of a slice of a row.  Every column is first written as one outside I,
// the block's members are written over it behind a barrier.
template <typename E, bool ALIGNED_Z, bool ALIGNED_D, bool REST>
__global__ void __launch_bounds__(NT) grad_kernel(DistillArgs a) {
  constexpr int N = Wide<E>::N;
  constexpr int U = 4;
  __shared__ int at[kMaxK];    // column within the slice, -1: not here
  __shared__ float pk[kMaxK];
  const int64_t n = blockIdx.x / a.splits;
  const int64_t c0 = (int64_t)(blockIdx.x % a.splits) * a.slice;
  const int64_t c1 = c0 + a.slice < a.V ? c0 + a.slice : a.V;
  const int tid = threadIdx.x;
  const E* z = row_of<E>(a, n);
  E* d = reinterpret_cast<E*>(a.dz) + n * a.V;
  const float c = kLog2e / a.temperature;
  const RowInfo info = load_info(a, n);
  const bool counts = !(info.r < 0.f);
  const float low = floor_of(c);
  const bool flat = counts && is_floored(info.all, low, c);
  float g = a.upstream[a.upstream_rows ? n : 0] * a.temperature;
  g *= a.mean != nullptr ? a.mean[0] : a.weight;
  const Outside o(info, g, REST);
  if (counts) {
    for (int k = tid; k < a.K; k += NT) {
      const int64_t j = index_at(a, n * a.K + k);
      at[k] = j >= c0 && j < c1 ? (int)(j - c0) : -1;
      pk[k] = info.teacher.part(floored(a.teacher[n * a.K + k], low), c);
    }
  }
  const int64_t nv = flat ? 0 : (c1 - c0) / N;
  if (flat)
    for (int64_t i = c0 + tid; i < c1; i += NT) d[i] = (E)(o.f * o.flat(up<E>(z[i])));
  for (int64_t v0 = tid; v0 < nv; v0 += (int64_t)NT * U) {
    float y[U][N];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int64_t v = v0 + (int64_t)q * NT;
      if (v < nv && counts) load_wide<E, ALIGNED_Z>(z + c0 + v * N, y[q]);
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int64_t v = v0 + (int64_t)q * NT;
      if (v < nv) {
#pragma unroll
        for (int i = 0; i < N; ++i) y[q][i] = counts ? o.f * o.power(y[q][i], c) : 0.f;
        store_wide<E, ALIGNED_D>(d + c0 + v * N, y[q]);
      }
    }
  }
  const int64_t rem = c0 + nv * N + tid;
  if (rem < c1 && !flat) d[rem] = (E)(counts ? o.f * o.power(up<E>(z[rem]), c) : 0.f);
  if (!counts) return;
  __syncthreads();
  for (int k = tid; k < a.K; k += NT) {
    const int j = at[k];
    if (j < 0) continue;
    float p = 0.f;  // an index given twice counts with both its parts
    for (int i = 0; i < a.K; ++i) p += at[i] == j ? pk[i] : 0.f;
    d[c0 + j] = (E)(g * (info.all.part(floored(up<E>(z[c0 + j]), low), c) - p));
  }
}

template <typename E>
void forward_type(const DistillArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.N * a.splits);
  const bool rest = a.rest != nullptr;
  const size_t lds = rest ? (size_t)((a.slice + 31) / 32) * 4 : 0;
  if (rest) {
    if (a.aligned) stats_kernel<E, true, true><<<grid, NT, lds, st>>>(a);
    else stats_kernel<E, false, true><<<grid, NT, lds, st>>>(a);
    if (a.splits > 1) join_kernel<E, true><<<(unsigned)a.N, 64, 0, st>>>(a);
  } else {
    if (a.aligned) stats_kernel<E, true, false><<<grid, NT, lds, st>>>(a);
    else stats_kernel<E, false, false><<<grid, NT, lds, st>>>(a);
    if (a.splits > 1) join_kernel<E, false><<<(unsigned)a.N, 64, 0, st>>>(a);
  }
}

template <typename E, bool AZ, bool AD>
void backward_aligned(const DistillArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)(a.N * a.splits);
  if (a.rest != nullptr) grad_kernel<E, AZ, AD, true><<<grid, NT, 0, st>>>(a);
  else grad_kernel<E, AZ, AD, false><<<grid, NT, 0, st>>>(a);
}

template <typename E>
void backward_type(const DistillArgs& a, hipStream_t st) {
  if (a.aligned && a.dz_aligned) backward_aligned<E, true, true>(a, st);
  else if (a.dz_aligned) backward_aligned<E, false, true>(a, st);
  else if (a.aligned) backward_aligned<E, true, false>(a, st);
  else backward_aligned<E, false, false>(a, st);
}

template <typename E, int VPT, int THREADS>
void row_vpt(const DistillArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)a.N;
  const bool al = a.aligned && a.dz_aligned;
  const size_t lds = a.rest != nullptr ? (size_t)((a.V + 31) / 32) * 4 : 0;
  if (a.rest != nullptr) {
    if (al) row_kernel<E, VPT, THREADS, true, true><<<grid, THREADS, lds, st>>>(a);
    else row_kernel<E, VPT, THREADS, false, true><<<grid, THREADS, lds, st>>>(a);
  } else {
    if (al) row_kernel<E, VPT, THREADS, true, false><<<grid, THREADS, lds, st>>>(a);
    else row_kernel<E, VPT, THREADS, false, false><<<grid, THREADS, lds, st>>>(a);
  }
}

template <typename E>
void row_type(const DistillArgs& a, hipStream_t st) {
  // 1024 threads up to 7 accesses each (50304 bf16 logits, 16384 rows: 0.67
  // ms, 0.80 as 512 x 13, whose registers do not suffice); where 1024 x 9
  // would not fit a CU twice, 512 x 18 does (33278 fp32, 1280 rows: 83 us for
  // the pass against 99)
  const int64_t vpt = ceil_div(a.V / Wide<E>::N, kMaxRowThreads);
  if (vpt <= 1) row_vpt<E, 1, kMaxRowThreads>(a, st);
  else if (vpt <= 2) row_vpt<E, 2, kMaxRowThreads>(a, st);
  else if (vpt <= 4) row_vpt<E, 4, kMaxRowThreads>(a, st);
  else if (vpt <= 7) row_vpt<E, 7, kMaxRowThreads>(a, st);
  else if (vpt <= 9) row_vpt<E, 18, kMaxRowThreads / 2>(a, st);
  else row_vpt<E, kMaxVpt, kMaxRowThreads>(a, st);
}

}  // namespace

void distill_split(int64_t N, int64_t V, bool bitmap, int64_t* slice, int* splits) {
  // one block a row where there are rows for 8 blocks a CU, else slices of
  // at least 2048 columns; a bitmap of at most 32 KB
  int64_t want = N >= 2048 ? 1 : ceil_div(2048, N > 0 ? N : 1);
  const int64_t most = ceil_div(V, 2048);
  if (want > most) want = most;
  const int64_t least = bitmap ? ceil_div(V, 262144) : 1;
  if (want < least) want = least;
  *slice = ceil_div(ceil_div(V, want), 8) * 8;
  *splits = (int)ceil_div(V, *slice);
}

void distill_forward(int dtype, const DistillArgs& a, float* loss, float* factor, int reduction,
                     hipStream_t st) {
  if (a.N > 0) {
    if (dtype == kBF16) forward_type<__bf16>(a, st);
    else if (dtype == kF16) forward_type<_Float16>(a, st);
    else forward_type<float>(a, st);
  }
  if (reduction != 0)
    reduce_kernel<<<1, 1024, 0, st>>>(a.row_loss, a.info, a.N, reduction == 2, a.weight,
                                       loss, factor);
}

bool distill_fuses(int dtype, int64_t N, int64_t V) {
  // 256 rows: a block on every CU; a launch has at most 2^32 threads
  const int64_t n = dtype == kBF16 ? 8 : 4;
  return dtype != kF16 && N >= 256 && N < (1LL << 22) && V <= kMaxRowThreads * kMaxVpt * n;
}

void distill_forward_grad(int dtype, const DistillArgs& a, float* loss, int reduction,
                          hipStream_t st) {
  teacher_kernel<<<(unsigned)ceil_div(a.N, NT / 64), NT, 0, st>>>(a);
  reduce_kernel<<<1, 1024, 0, st>>>(a.row_loss, a.info, a.N, reduction == 2, a.weight, nullptr,
                                    const_cast<float*>(a.mean));
  if (dtype == kBF16) row_type<__bf16>(a, st);
  else row_type<float>(a, st);
  reduce_kernel<<<1, 1024, 0, st>>>(a.row_loss, a.info, a.N, reduction == 2, a.weight, loss,
                                    nullptr);
}

void distill_scale(int dtype, void* dz, int64_t n, const float* factor, hipStream_t st) {
  const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n, 8 * NT), 2048);
  if (dtype == kBF16)
    scale_kernel<__bf16><<<grid, NT, 0, st>>>(static_cast<__bf16*>(dz), n, factor);
  else
    scale_kernel<float><<<grid, NT, 0, st>>>(static_cast<float*>(dz), n, factor);
}

void distill_backward(int dtype, const DistillArgs& a, hipStream_t st) {
  if (a.N == 0) return;
  if (dtype == kBF16) backward_type<__bf16>(a, st);
  else if (dtype == kF16) backward_type<_Float16>(a, st);
  else backward_type<float>(a, st);
}

}  // namespace kfac

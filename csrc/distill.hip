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
// two, a second rounding.  The other calls (fp16, whose range does not hold
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
constexpr int kMaxVpt = 16;  // 16-byte accesses a thread of row_kernel holds
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

// running (maximum, sum of 2^(y - maximum)); (-inf, 0) is empty
struct Run {
  float m, s;
  __device__ __forceinline__ void join(float m2, float s2) {
    const float mm = fmaxf(m, m2);
    const float base = mm == KFAC_NEG_INF ? 0.f : mm;
    s = s * ex2(m - base) + s2 * ex2(m2 - base);
    m = mm;
  }
  __device__ __forceinline__ float log2sum() const {
    return s == 0.f ? KFAC_NEG_INF : m + log2f(s);
  }
};

__device__ __forceinline__ float add_log2(float a, float b) {
  Run r{a, a == KFAC_NEG_INF ? 0.f : 1.f};
  r.join(b, b == KFAC_NEG_INF ? 0.f : 1.f);
  return r.log2sum();
}

__device__ __forceinline__ Run wave_join(Run r) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float m2 = __shfl_xor(r.m, off, 64), s2 = __shfl_xor(r.s, off, 64);
    r.join(m2, s2);
  }
  return r;
}

__device__ __forceinline__ int64_t index_at(const DistillArgs& a, int64_t i) {
  return a.index64 ? reinterpret_cast<const int64_t*>(a.index)[i]
                   : (int64_t)reinterpret_cast<const int32_t*>(a.index)[i];
}

template <typename E>
__device__ __forceinline__ const E* row_of(const DistillArgs& a, int64_t n) {
  return reinterpret_cast<const E*>(a.z) + (n / a.inner) * a.zs0 + (n % a.inner) * a.zs1;
}

// The teacher's side of a row, by one wave.
struct Teacher {
  float norm, rest, r;  // log2 sum of its entries and rest; log2 rest; the rest's share
  bool counts;          // the row has entries, and they or the rest have mass
  bool outside;         // an index behind the vocabulary
  __device__ __forceinline__ Teacher(const DistillArgs& a, int64_t n) {
    const int lane = threadIdx.x & 63;
    const float c = kLog2e / a.temperature;
    rest = a.rest != nullptr ? a.rest[n] * kLog2e : KFAC_NEG_INF;
    Run t{KFAC_NEG_INF, 0.f};
    bool some = false, far = false;
    for (int k = lane; k < a.K; k += 64) {
      const int64_t j = index_at(a, n * a.K + k);
      if (j < 0) continue;
      some = true;
      far |= j >= a.V;
      const float y = a.teacher[n * a.K + k] * c;
      t.join(y, y == KFAC_NEG_INF ? 0.f : 1.f);
    }
    t = wave_join(t);
    outside = __any(far);
    norm = add_log2(t.log2sum(), rest);
    r = a.rest != nullptr && rest != KFAC_NEG_INF ? ex2(rest - norm) : 0.f;
    counts = __any(some) && norm != KFAC_NEG_INF;
  }
};

// A row's loss, by one wave.  tail / lse: log2 sums of the student's columns
// outside I (with a rest) and of all columns; both NaN where an index lies
// behind the vocabulary.
template <typename E>
__device__ float row_loss(const DistillArgs& a, int64_t n, const Teacher& t, float lse,
                          float tail) {
  const float c = kLog2e / a.temperature;
  const E* z = row_of<E>(a, n);
  float loss = 0.f;
  for (int k = threadIdx.x & 63; k < a.K; k += 64) {
    const int64_t j = index_at(a, n * a.K + k);
    if (j < 0 || j >= a.V) continue;
    const float lp = a.teacher[n * a.K + k] * c - t.norm;
    const float p = ex2(lp);
    if (p > 0.f) loss += p * (lp - (up<E>(z[j]) * c - lse));
  }
  loss = wave_reduce_sum(loss);
  if (t.r > 0.f) loss += t.r * ((t.rest - t.norm) - (tail - lse));
  // p = 0 terms drop out, but not what makes the row undefined
  if (lse != lse || t.norm != t.norm) loss = lse + t.norm;
  return t.counts ? loss * kLn2 * a.temperature * a.temperature : 0.f;
}

// info: {lse, tail, r (-1: the row does not count), teacher norm}
template <typename E>
__device__ void finish_row(const DistillArgs& a, int64_t n, float lse, float tail) {
  const Teacher t(a, n);
  if (t.outside) lse = tail = __builtin_nanf("");
  const float loss = row_loss<E>(a, n, t, lse, tail);
  if ((threadIdx.x & 63) == 0) {
    a.info[n] = make_float4(lse, tail, t.counts ? t.r : -1.f, t.norm);
    a.row_loss[n] = loss;
  }
}

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

  Run out{KFAC_NEG_INF, 0.f}, in{KFAC_NEG_INF, 0.f};
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
      float mx = out.m;
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
                const float e = y[q][i] * c;
                in.join(e, e == KFAC_NEG_INF ? 0.f : 1.f);
                y[q][i] = KFAC_NEG_INF;
              }
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          y[q][i] *= c;
          mx = fmaxf(mx, y[q][i]);
        }
      }
      const float base = mx == KFAC_NEG_INF ? 0.f : mx;
      float s = out.s * ex2(out.m - base);
#pragma unroll
      for (int q = 0; q < U; ++q)
#pragma unroll
        for (int i = 0; i < N; ++i) s += ex2(y[q][i] - base);
      out.s = s;
      out.m = mx;
    }
    const int64_t rem = c0 + nv * N + tid;  // the last, partial access
    if (rem < c1) {
      const float e = up<E>(z[rem]) * c;
      const int at = (int)(rem - c0);
      const bool member = REST && ((bits[at >> 5] >> (at & 31)) & 1u);
      (member ? in : out).join(e, e == KFAC_NEG_INF ? 0.f : 1.f);
    }
  }
  out = wave_join(out);
  if (REST) in = wave_join(in);
  if ((tid & 63) == 0) red[tid >> 6] = make_float4(out.m, out.s, in.m, in.s);
  __syncthreads();
  if (tid >= 64) return;
  out = Run{red[0].x, red[0].y};
  in = Run{red[0].z, red[0].w};
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) {
    out.join(red[w].x, red[w].y);
    in.join(red[w].z, red[w].w);
  }
  if (a.splits > 1) {
    if (tid == 0) a.part[blockIdx.x] = make_float4(out.m, out.s, in.m, in.s);
    return;
  }
  const float tail = out.log2sum();
  finish_row<E>(a, n, REST ? add_log2(tail, in.log2sum()) : tail, tail);
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
  const float tail = out.log2sum();
  finish_row<E>(a, n, REST ? add_log2(tail, in.log2sum()) : tail, tail);
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
    c += info[n].z < 0.f ? 0.0 : 1.0;
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
  const Teacher t(a, n);
  if ((threadIdx.x & 63) == 0)
    a.info[n] = make_float4(t.outside ? __builtin_nanf("") : 0.f, 0.f, t.counts ? t.r : -1.f,
                            t.norm);
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
constexpr int kRowThreads = 1024;

// Two blocks a CU (64 registers a thread) up to 9 accesses a thread, so that
// one loads while the other forms its sums; one block above.
template <typename E, int VPT, bool ALIGNED, bool REST>
__global__ void __launch_bounds__(kRowThreads, VPT <= 9 ? 8 : 4) row_kernel(DistillArgs a) {
  constexpr int N = Wide<E>::N;
  extern __shared__ uint32_t bits[];  // with a rest: one bit a column
  __shared__ float4 red[kRowThreads / 64];
  __shared__ int at[kMaxK];     // the entries' columns, -1: none
  __shared__ float pk[kMaxK];   // their share of the teacher
  __shared__ float yk[kMaxK];   // the student's logits there, in units of log2
  __shared__ float pj[kMaxK];   // the teacher's share of the column, all entries that name it
  __shared__ float sums[2];     // sum p (ln p - y) and sum p, over the entries
  const int64_t n = blockIdx.x;
  const int tid = threadIdx.x, V = (int)a.V, nv = V / N;
  const E* z = row_of<E>(a, n);
  E* d = reinterpret_cast<E*>(a.dz) + n * a.V;
  const float c = kLog2e / a.temperature;
  const float4 info = a.info[n];
  typedef E vec __attribute__((ext_vector_type(N)));
  typedef vec uvec __attribute__((aligned(sizeof(E))));
  auto put = [&](E* p, const vec& x) {
    if (ALIGNED) *reinterpret_cast<vec*>(p) = x;
    else *reinterpret_cast<uvec*>(p) = x;
  };
  if (info.z < 0.f) {  // the row does not count (a NaN does)
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
    pk[k] = in ? ex2(a.teacher[n * a.K + k] * c - info.w) : 0.f;
    yk[k] = in ? up<E>(z[j]) * c : 0.f;
    if (REST && in) atomicOr(&bits[j >> 5], 1u << (j & 31));
  }
  __syncthreads();
  {
    // an index given twice counts with both its parts: `team` lanes of a wave
    // add up the entries that name the column of entry k
    int team = 64;
    while (team > 1 && team * a.K > kRowThreads) team >>= 1;
    const int k = tid / team, part = tid & (team - 1);
    float p = 0.f;
    if (k < a.K && at[k] >= 0)
      for (int i = part; i < a.K; i += team) p += at[i] == at[k] ? pk[i] : 0.f;
    for (int off = team >> 1; off > 0; off >>= 1) p += __shfl_xor(p, off, 64);
    if (k < a.K && part == 0) pj[k] = p;
  }
  if (tid < 64) {
    float sa = 0.f, sp = 0.f;
    for (int k = tid; k < a.K; k += 64)
      if (pk[k] > 0.f) {
        sa += pk[k] * ((a.teacher[n * a.K + k] * c - info.w) - yk[k]);
        sp += pk[k];
      }
    sa = wave_reduce_sum(sa);
    sp = wave_reduce_sum(sp);
    if (tid == 0) {
      sums[0] = sa;
      sums[1] = sp;
    }
  }

  Run out{KFAC_NEG_INF, 0.f}, in{KFAC_NEG_INF, 0.f};
#pragma unroll
  for (int q = 0; q < VPT; ++q) {
    if (REST) {
      const int col = (tid + q * kRowThreads) * N;
      const uint32_t b = col < V ? (bits[col >> 5] >> (col & 31)) & ((1u << N) - 1u) : 0u;
      if (b != 0) {  // rare: K columns of V; their gradient is written below
#pragma unroll
        for (int i = 0; i < N; ++i)
          if ((b >> i) & 1u) {
            const float e = up<E>(x[q][i]) * c;
            in.join(e, e == KFAC_NEG_INF ? 0.f : 1.f);
            x[q][i] = (E)KFAC_NEG_INF;
          }
      }
      stay_packed(x[q]);
    }
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = up<E>(x[q][i]) * c;
    float mx = out.m;
#pragma unroll
    for (int i = 0; i < N; ++i) mx = fmaxf(mx, y[i]);
    const float base = mx == KFAC_NEG_INF ? 0.f : mx;
    float s = out.s * ex2(out.m - base);
#pragma unroll
    for (int i = 0; i < N; ++i) s += ex2(y[i] - base);
    out.s = s;
    out.m = mx;
  }
  if (rem < V) {
    const float e = last * c;
    const bool member = REST && ((bits[rem >> 5] >> (rem & 31)) & 1u);
    (member ? in : out).join(e, e == KFAC_NEG_INF ? 0.f : 1.f);
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
  float tail = out.log2sum();
  float lse = REST ? add_log2(tail, in.log2sum()) : tail;
  if (info.x != info.x) lse = tail = info.x;  // an index behind the vocabulary
  const float r = info.z, g = a.temperature * a.mean[0];
  float base = lse, f = g;
  if (REST && tail != KFAC_NEG_INF) {
    base = tail;
    f = g * (ex2(tail - lse) - r);
  }
#pragma unroll
  for (int q = 0; q < VPT; ++q) {
    const int v = tid + q * kRowThreads;
    stay_packed(x[q]);
    if (v < nv) {
      vec y;
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = (E)(f * ex2(up<E>(x[q][i]) * c - base));
      put(d + (int64_t)v * N, y);
    }
  }
  if (rem < V) d[rem] = (E)(f * ex2(last * c - base));
  if (tid == 0) {
    float loss = sums[0] + sums[1] * lse;
    if (r > 0.f) loss += r * ((a.rest[n] * kLog2e - info.w) - (tail - lse));
    if (lse != lse || info.w != info.w) loss = lse + info.w;
    a.row_loss[n] = loss * kLn2 * a.temperature * a.temperature;
    a.info[n] = make_float4(lse, tail, r, info.w);
  }
  __syncthreads();
  for (int k = tid; k < a.K; k += kRowThreads)
    if (at[k] >= 0) d[at[k]] = (E)(g * (ex2(yk[k] - lse) - pj[k]));
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

// dz of a slice of a row.  Every column is first written as one outside I
// (e = 2^(y - tail), factor R - r; without a rest 2^(y - lse)), the block's
// members are written over it behind a barrier.
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
  const float4 info = a.info[n];
  const float lse = info.x, tail = info.y, r = info.z, norm = info.w;
  const bool counts = !(r < 0.f);
  float g = a.upstream[a.upstream_rows ? n : 0] * a.temperature;
  if (a.mean != nullptr) g *= a.mean[0];
  float base = lse, f = g;
  if (REST && tail != KFAC_NEG_INF) {
    base = tail;
    f = g * (ex2(tail - lse) - r);
  }
  if (counts) {
    for (int k = tid; k < a.K; k += NT) {
      const int64_t j = index_at(a, n * a.K + k);
      at[k] = j >= c0 && j < c1 ? (int)(j - c0) : -1;
      pk[k] = ex2(a.teacher[n * a.K + k] * c - norm);
    }
  }
  const int64_t nv = (c1 - c0) / N;
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
        for (int i = 0; i < N; ++i) y[q][i] = counts ? f * ex2(y[q][i] * c - base) : 0.f;
        store_wide<E, ALIGNED_D>(d + c0 + v * N, y[q]);
      }
    }
  }
  const int64_t rem = c0 + nv * N + tid;
  if (rem < c1) d[rem] = (E)(counts ? f * ex2(up<E>(z[rem]) * c - base) : 0.f);
  if (!counts) return;
  __syncthreads();
  for (int k = tid; k < a.K; k += NT) {
    const int j = at[k];
    if (j < 0) continue;
    float p = 0.f;  // an index given twice counts with both its parts
    for (int i = 0; i < a.K; ++i) p += at[i] == j ? pk[i] : 0.f;
    d[c0 + j] = (E)(g * (ex2(up<E>(z[c0 + j]) * c - lse) - p));
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

template <typename E, int VPT>
void row_vpt(const DistillArgs& a, hipStream_t st) {
  const unsigned grid = (unsigned)a.N;
  const bool al = a.aligned && a.dz_aligned;
  const size_t lds = a.rest != nullptr ? (size_t)((a.V + 31) / 32) * 4 : 0;
  if (a.rest != nullptr) {
    if (al) row_kernel<E, VPT, true, true><<<grid, kRowThreads, lds, st>>>(a);
    else row_kernel<E, VPT, false, true><<<grid, kRowThreads, lds, st>>>(a);
  } else {
    if (al) row_kernel<E, VPT, true, false><<<grid, kRowThreads, lds, st>>>(a);
    else row_kernel<E, VPT, false, false><<<grid, kRowThreads, lds, st>>>(a);
  }
}

template <typename E>
void row_type(const DistillArgs& a, hipStream_t st) {
  const int64_t vpt = ceil_div(a.V / Wide<E>::N, kRowThreads);
  if (vpt <= 1) row_vpt<E, 1>(a, st);
  else if (vpt <= 2) row_vpt<E, 2>(a, st);
  else if (vpt <= 4) row_vpt<E, 4>(a, st);
  else if (vpt <= 7) row_vpt<E, 7>(a, st);
  else if (vpt <= 9) row_vpt<E, 9>(a, st);
  else row_vpt<E, kMaxVpt>(a, st);
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
  // 256 rows: a block on every CU
  const int64_t n = dtype == kBF16 ? 8 : 4;
  return dtype != kF16 && N >= 256 && V <= kRowThreads * kMaxVpt * n;
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

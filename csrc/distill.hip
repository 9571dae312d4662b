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
// Both passes are bound by memory: the forward reads the logits once
// (running maximum and sum, 32 bits, in units of log2), the backward reads
// them again and writes the gradient.  Keeping a gradient from the forward
// would save that second read only where the upstream factor is 1 and costs
// a second rounding where it is not, and in fp16 the unscaled gradient of a
// mean over thousands of rows is below the type's smallest value.
#include "common.h"

#include "lm_ops.h"

namespace kfac {

namespace {

constexpr int NT = 256;
constexpr int kMaxK = 1024;
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

// The teacher's side of a row and its loss, by one wave.  tail / lse: log2
// sums of the student's columns outside I (with a rest) and of all columns.
// info: {lse, tail, r (-1: no entry, the row does not count), teacher norm}.
template <typename E>
__device__ void finish_row(const DistillArgs& a, int64_t n, float lse, float tail) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / a.temperature;
  const E* z = row_of<E>(a, n);
  const float rest2 = a.rest != nullptr ? a.rest[n] * kLog2e : KFAC_NEG_INF;
  Run t{KFAC_NEG_INF, 0.f};
  bool some = false, outside = false;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t j = index_at(a, n * a.K + k);
    if (j < 0) continue;
    some = true;
    outside |= j >= a.V;
    const float y = a.teacher[n * a.K + k] * c;
    t.join(y, y == KFAC_NEG_INF ? 0.f : 1.f);
  }
  t = wave_join(t);
  some = __any(some);
  // an index behind the vocabulary: NaN, in the loss and in the gradient
  if (__any(outside)) lse = tail = __builtin_nanf("");
  const float norm = add_log2(t.log2sum(), rest2);
  const float r = a.rest != nullptr && rest2 != KFAC_NEG_INF ? ex2(rest2 - norm) : 0.f;
  float loss = 0.f;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t j = index_at(a, n * a.K + k);
    if (j < 0 || j >= a.V) continue;
    const float lp = a.teacher[n * a.K + k] * c - norm;
    const float p = ex2(lp);
    if (p > 0.f) loss += p * (lp - (up<E>(z[j]) * c - lse));
  }
  loss = wave_reduce_sum(loss);
  if (r > 0.f) loss += r * ((rest2 - norm) - (tail - lse));
  // p = 0 terms drop out, but not what makes the row undefined
  if (lse != lse || norm != norm) loss = lse + norm;
  if (lane == 0) {
    // no entry, or entries and a rest without any mass: the row does not count
    some = some && norm != KFAC_NEG_INF;
    a.info[n] = make_float4(lse, tail, some ? r : -1.f, norm);
    a.row_loss[n] = some ? loss * kLn2 * a.temperature * a.temperature : 0.f;
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

// sum or mean of the rows' losses, and the factor of a row's gradient (1, or
// 1 / rows that count); 64-bit sums in a fixed order
__global__ void __launch_bounds__(1024) reduce_kernel(const float* row_loss, const float4* info,
                                                      int64_t N, int mean, float* loss,
                                                      float* factor) {
  __shared__ double sum[16];
  __shared__ double cnt[16];
  double s = 0.0, c = 0.0;
  for (int64_t n = threadIdx.x; n < N; n += 1024) {
    s += row_loss[n];
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
    const double f = mean ? 1.0 / (c > 0.0 ? c : 1.0) : 1.0;
    *loss = (float)(s * f);
    *factor = (float)f;
  }
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
    reduce_kernel<<<1, 1024, 0, st>>>(a.row_loss, a.info, a.N, reduction == 2, loss,
                                       factor);
}

void distill_backward(int dtype, const DistillArgs& a, hipStream_t st) {
  if (a.N == 0) return;
  if (dtype == kBF16) backward_type<__bf16>(a, st);
  else if (dtype == kF16) backward_type<_Float16>(a, st);
  else backward_type<float>(a, st);
}

}  // namespace kfac

// Rotary positions with several axes, q and k in one launch (ops/rotary.py).
//
// Pair i of a head belongs to axis a(i) and turns by the angle
//   pos[token][a(i)] * f(i):  (x1, x2) -> (x1 c - x2 s, x1 s + x2 c),
// the backward pass is the same launch with the angle's sign flipped.  The
// elements behind the last pair are copied.
//
// The kernel moves 2 bytes in and 2 out per bf16 element and has to do
// little else, so it is bound by memory as long as the trigonometry is done
// once per (token, pair) and not once per head: a thread owns one 16-byte
// unit of a token's head and walks the heads, q's first and k's after them.
// GPT-NeoX batch (8 x 2048 tokens, q and k of 12 heads of 64, bf16): 27 us,
// 3.7 TB/s; 2 x 4719 video tokens, 16 + 4 heads of 128 in fp32, three axes: 48
// us, 4 TB/s.
// Angles are formed in turns in 64 bits (position 10^6 times frequency 1 is
// 0.06 rad off in 32 bits), reduced to [-1/2, 1/2] turn there, and only the
// rest goes to sincospif.
#include "common.h"

#include "lm_ops.h"

namespace kfac {

namespace {

template <typename E> struct Elem;
template <> struct Elem<float> {
  __device__ __forceinline__ static float up(float v) { return v; }
  __device__ __forceinline__ static float down(float v) { return v; }
};
template <> struct Elem<__bf16> {
  __device__ __forceinline__ static float up(__bf16 v) { return (float)v; }
  __device__ __forceinline__ static __bf16 down(float v) { return (__bf16)v; }
};
template <> struct Elem<_Float16> {
  __device__ __forceinline__ static float up(_Float16 v) { return (float)v; }
  __device__ __forceinline__ static _Float16 down(float v) { return (_Float16)v; }
};

template <typename E, int N, bool VEC>
__device__ __forceinline__ void load_unit(const E* p, E* v) {
  if (VEC) {
    typedef E vec __attribute__((ext_vector_type(N)));
    const vec t = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = t[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}

template <typename E, int N, bool VEC>
__device__ __forceinline__ void store_unit(E* p, const E* v) {
  if (VEC) {
    typedef E vec __attribute__((ext_vector_type(N)));
    vec t;
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = v[i];
    *reinterpret_cast<vec*>(p) = t;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v[i];
  }
}

// N elements per access.  Interleaved: a unit is N consecutive elements,
// N / 2 pairs (2i, 2i + 1).  Halves: a unit is N elements of the first half
// and the N of the second that they pair with (i, i + pairs); units behind
// the pairs are N plain elements to copy.
template <typename E, int N, bool VEC, bool HALVES>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  constexpr int NP = HALVES ? N : N / 2;  // pairs of a unit
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)a.B * a.T * a.units) return;
  const int unit = (int)(id % a.units);
  const int64_t bt = id / a.units;
  const int t = (int)(bt % a.T);
  const int64_t b = bt / a.T;
  const int rot_units = HALVES ? a.pairs / N : a.units;
  const bool copy = HALVES && unit >= rot_units;
  const int pair0 = unit * NP;
  const int d0 = HALVES ? (copy ? 2 * a.pairs + (unit - rot_units) * N : unit * N) : unit * N;

  float c[NP], s[NP];
  bool turns[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int pr = pair0 + i;
    turns[i] = !copy && pr < a.pairs;
    c[i] = 1.f;
    s[i] = 0.f;
    if (turns[i]) {
      const int64_t at = b * a.psB + t * a.psT + a.tab.axis[pr] * a.psA;
      const double p = a.pos64 ? (double)reinterpret_cast<const int64_t*>(a.pos)[at]
                               : (double)reinterpret_cast<const int32_t*>(a.pos)[at];
      const double rev = p * a.tab.turn[pr];
      const float rest = (float)(rev - rint(rev));
      sincospif(2.f * rest, &s[i], &c[i]);
      s[i] *= a.sign;
    }
  }

  const int heads = a.Hq + a.Hk;
  const int per = (heads + gridDim.y - 1) / gridDim.y;
  const int h0 = blockIdx.y * per;
  const int h1 = h0 + per < heads ? h0 + per : heads;
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const bool isq = h < a.Hq;
    const int hh = isq ? h : h - a.Hq;
    const E* x = isq ? reinterpret_cast<const E*>(a.q) + b * a.qs[0] + hh * a.qs[1] + t * a.qs[2]
                     : reinterpret_cast<const E*>(a.k) + b * a.ks[0] + hh * a.ks[1] + t * a.ks[2];
    E* y = isq ? reinterpret_cast<E*>(a.qo) + ((b * a.Hq + hh) * a.T + t) * a.D
               : reinterpret_cast<E*>(a.ko) + ((b * a.Hk + hh) * a.T + t) * a.D;
    E v[N], w[N];
    load_unit<E, N, VEC>(x + d0, v);
    if (HALVES) {
      if (!copy) {
        load_unit<E, N, VEC>(x + d0 + a.pairs, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float x1 = Elem<E>::up(v[i]), x2 = Elem<E>::up(w[i]);
          v[i] = Elem<E>::down(x1 * c[i] - x2 * s[i]);
          w[i] = Elem<E>::down(x2 * c[i] + x1 * s[i]);
        }
        store_unit<E, N, VEC>(y + d0 + a.pairs, w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const float x1 = Elem<E>::up(v[2 * i]), x2 = Elem<E>::up(v[2 * i + 1]);
        // a pair that does not turn is copied, whatever it holds
        if (turns[i]) {
          v[2 * i] = Elem<E>::down(x1 * c[i] - x2 * s[i]);
          v[2 * i + 1] = Elem<E>::down(x2 * c[i] + x1 * s[i]);
        }
      }
    }
    store_unit<E, N, VEC>(y + d0, v);
  }
}

template <typename E, int N, bool VEC>
void launch(const RotaryArgs& a, bool halves, dim3 grid, hipStream_t st) {
  if (halves) rotary_kernel<E, N, VEC, true><<<grid, 256, 0, st>>>(a);
  else rotary_kernel<E, N, VEC, false><<<grid, 256, 0, st>>>(a);
}

template <typename E>
void launch_type(RotaryArgs& a, bool halves, bool vec, hipStream_t st) {
  constexpr int NV = 16 / (int)sizeof(E);
  const int n = vec ? NV : (halves ? 1 : 2);
  a.units = halves ? (a.pairs + a.D - 2 * a.pairs) / n : a.D / n;
  const int64_t threads = (int64_t)a.B * a.T * a.units;
  const int64_t bx = ceil_div(threads, 256);
  // heads over blockIdx.y until the chip has work for 8 waves a SIMD
  const int heads = a.Hq + a.Hk;
  int64_t hy = ceil_div(2048, bx);
  if (hy > heads) hy = heads;
  const dim3 grid((unsigned)bx, (unsigned)hy);
  if (vec) launch<E, NV, true>(a, halves, grid, st);
  else if (halves) rotary_kernel<E, 1, false, true><<<grid, 256, 0, st>>>(a);
  else rotary_kernel<E, 2, false, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace

// dtype: kF32, kBF16 or kF16; vec: strides and pointers allow 16-byte units
// and, for halves, pairs and D - 2 pairs are multiples of a unit (the host
// checks); D even; at least one pair
void rotary_axes(int dtype, RotaryArgs a, bool halves, bool vec, hipStream_t st) {
  if (a.B == 0 || a.T == 0 || a.D == 0 || a.Hq + a.Hk == 0) return;
  if (dtype == kBF16) launch_type<__bf16>(a, halves, vec, st);
  else if (dtype == kF16) launch_type<_Float16>(a, halves, vec, st);
  else launch_type<float>(a, halves, vec, st);
}

}  // namespace kfac

// Argument blocks of the decoder operators (window attention, rotary
// positions, distillation), shared by their kernels and lm_ops.cpp.
#pragma once

#include <cstdint>

#include <hip/hip_runtime.h>

namespace kfac {

// ---------------------------------------------------------------- rotary
constexpr int kMaxRotaryPairs = 128;

struct RotaryTable {
  double turn[kMaxRotaryPairs];   // frequency of a pair, in turns per position
  uint8_t axis[kMaxRotaryPairs];  // its axis
};

struct RotaryArgs {
  const void* q;
  const void* k;
  void* qo;  // contiguous [B, Hq, T, D]
  void* ko;  // contiguous [B, Hk, T, D]
  const void* pos;
  int64_t qs[3], ks[3];   // strides of q and k: batch, head, token
  int64_t psB, psT, psA;  // strides of the positions
  int B, T, D, Hq, Hk, pairs, units, pos64;
  float sign;  // +1 forward, -1 backward
  RotaryTable tab;
};

void rotary_axes(int dtype, RotaryArgs a, bool halves, bool vec, hipStream_t st);

// ---------------------------------------------------------------- distill
struct DistillArgs {
  const void* z;         // student logits: row n = (n / inner, n % inner)
  int64_t zs0, zs1;      // strides of the two row indices
  int64_t inner;
  const float* teacher;  // [N, K]
  const void* index;     // [N, K] int32 / int64, negative = no entry
  const float* rest;     // [N] or null
  int64_t N, V;
  int K, index64, aligned;
  float temperature, weight;
  float4* part;          // [N, splits]: running statistics of a slice of a row
  float4* info;          // [N, 2]: RowInfo of distill.hip
  float* row_loss;       // [N]
  int splits;
  int64_t slice;         // columns of a split (a multiple of 8)
  // backward
  const float* upstream;    // scalar, or one value a row
  int upstream_rows;        // 1: one a row
  const float* mean;        // factor of the rows' gradients; null: 1
  void* dz;                 // contiguous [N, V]
  int dz_aligned;
};

// reduction: 0 none (row_loss is the answer), 1 sum, 2 mean: loss, and the
// factor of a row's gradient
void distill_forward(int dtype, const DistillArgs& a, float* loss, float* factor, int reduction,
                     hipStream_t st);
void distill_backward(int dtype, const DistillArgs& a, hipStream_t st);
// loss and gradient in one pass over the logits (a.dz, a.mean to be written;
// reduction 1 or 2), where distill_fuses says so
bool distill_fuses(int dtype, int64_t N, int64_t V);
void distill_forward_grad(int dtype, const DistillArgs& a, float* loss, int reduction,
                          hipStream_t st);
// dz *= *factor in place (16-byte aligned)
void distill_scale(int dtype, void* dz, int64_t n, const float* factor, hipStream_t st);
// columns of a split for N rows of V columns, and how many there are
void distill_split(int64_t N, int64_t V, bool bitmap, int64_t* slice, int* splits);

// --------------------------------------------------------- window attention
struct AttnArgs {
  const void *q, *k, *v;
  int64_t qs[3], ks[3], vs[3];  // strides: batch, head, token
  const void* dout;             // backward
  int64_t dos[3];
  void* out;                    // [B, Hq, Tq, D] with strides os
  int64_t os[3];
  void* rest;                   // what out's rounding took away, laid out like out, or null
  float* lse;                   // [B * Hkv, Tq * G] (rows), log2 units; +inf: sees nothing
  float* delta;                 // the same: -do . o
  void *dq, *dk, *dv;
  int64_t dqs[3], dks[3], dvs[3];
  const int* lengths;           // [B] or null
  const int* starts;            // [B] or null
  int start;                    // where starts is null and start_given
  int start_given;
  int B, Hq, Hkv, Tq, Tk, D, W, S, G;
  float scale;
  int splits;                   // key slices of a row block (forward)
  float* opart;                 // [splits, B * Hkv, rows, D]
  float* lpart;                 // [splits, B * Hkv, rows]
  uint32_t Gmagic;              // floor(2^32 / G)
  int sink_groups, far_chunks;  // backward: groups of sink keys, chunks of their far rows
  float* kvpart;                // their shares
  // fp16 backward: of each chunk of a (sequence, key head) the largest |do|^2
  // of its rows and |v|^2 of its keys; the rows' lse for the key gradients
  int bound_chunks;
  float* bounds;                // [B * Hkv, bound_chunks, 2]
  float* lse_keys;              // like lse
};

// how a forward call is split over the keys, and the floats of its partial
// results; the same for the backward call's sinks
bool attn_keeps_rest(const AttnArgs& a);
void attn_plan(const AttnArgs& a, int* splits, int64_t* floats);
void attn_bwd_plan(const AttnArgs& a, int* sink_groups, int* far_chunks, int64_t* floats);
// chunks of AttnArgs::bounds, 0: the type needs none
int attn_bound_chunks(int dtype, const AttnArgs& a);
void attn_forward(int dtype, const AttnArgs& a, hipStream_t st);
void attn_backward(int dtype, const AttnArgs& a, hipStream_t st);

}  // namespace kfac

// Torch side of the decoder operators: window attention with sinks, rotary
// positions with several axes, distillation from a teacher's top logits
// (kernels in window_attn.hip, rotary.hip, distill.hip).  Argument checks of
// the public functions are in ops/attention.py, ops/rotary.py and
// ops/distill.py; the checks here are those that keep a kernel in bounds.
// Each operator is a C++ autograd node, so that neither its forward nor its
// backward runs Python.
#include <torch/extension.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <tuple>
#include <vector>

#include "common.h"
#include "lm_ops.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

hipStream_t stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

int tag(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return kfac::kF32;
    case at::kBFloat16: return kfac::kBF16;
    case at::kHalf: return kfac::kF16;
    default: TORCH_CHECK(false, "kfac native: unsupported dtype ", t.scalar_type());
  }
  return -1;
}

bool aligned16(const at::Tensor& t) {
  return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
}

// contiguous and at a multiple of 16 bytes, a copy if need be
at::Tensor packed16(const at::Tensor& t) {
  const at::Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone();
}

// rows that 16-byte accesses can read: unit last stride, every other stride
// of a dimension with more than one element a multiple of 16 bytes
bool rows16(const at::Tensor& t) {
  const int64_t unit = 16 / (int64_t)t.element_size();
  const int64_t n = t.dim();
  if (!aligned16(t) || (t.stride(n - 1) != 1 && t.size(n - 1) > 1)) return false;
  for (int64_t i = 0; i + 1 < n; ++i)
    if (t.size(i) > 1 && t.stride(i) % unit != 0) return false;
  return true;
}

// batch, head, token of [B, H, T, D].  The stride of a single token may be
// anything and a tile's rows behind it are still placed by it: a row's length
// keeps them apart and aligned.
void strides3(const at::Tensor& t, int64_t* s) {
  s[0] = t.stride(0);
  s[1] = t.stride(1);
  s[2] = t.size(2) > 1 ? t.stride(2) : t.size(3);
}

// An attention operand [B, H, T, D]: rows that 16-byte accesses can read, a
// token's row no longer than the stride to the next (an expanded one is
// not), and 64 rows of `group` heads within 2^31 bytes of the first, which
// is what the kernels' 32-bit offsets reach.  Else a copy laid out
// [B, T, H, D].
bool in_reach(const at::Tensor& t, int64_t group) {
  int64_t s[3];
  strides3(t, s);
  return ((group - 1) * s[1] + 64 * s[2]) * (int64_t)t.element_size() < ((int64_t)1 << 31) - 1024;
}
at::Tensor operand(const at::Tensor& t, int64_t group) {
  if (rows16(t) && (t.size(2) <= 1 || t.stride(2) >= t.size(3)) && in_reach(t, group)) return t;
  const at::Tensor c = t.transpose(1, 2).clone(at::MemoryFormat::Contiguous).transpose(1, 2);
  TORCH_CHECK(in_reach(c, group), "window_attention: too large: 64 tokens of ", t.size(1),
              " heads pass 2^31 bytes");
  return c;
}

void once_only(const char* op) {
  // the backward pass is made of kernels: nothing records it for a second one
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": gradients of gradients are not supported");
}

// A tangent would be dropped without a word: the kernels have no forward-mode
// derivative.
void reverse_only(const char* op, std::initializer_list<const at::Tensor*> ts) {
  for (const auto* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(), op,
                ": forward-mode derivatives are not supported");
}

bool records(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto* t : ts)
    if (t->requires_grad()) return true;
  return false;
}

void on_device(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "kfac native: ", what,
              " must be on the operands' GPU");
}

// ----------------------------------------------------------- attention
struct AttnConf {
  int64_t window, sinks, start;
  bool start_given;
  double scale;
};

// what a node keeps besides tensors, as one entry (each is exact in a double)
std::vector<double> pack(const AttnConf& c) {
  return {(double)c.window, (double)c.sinks, (double)c.start, c.start_given ? 1.0 : 0.0, c.scale};
}
AttnConf unpack(const std::vector<double>& v) {
  return {(int64_t)v[0], (int64_t)v[1], (int64_t)v[2], v[3] != 0.0, v[4]};
}

kfac::AttnArgs attn_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                         const OptTensor& lengths, const OptTensor& starts, const AttnConf& c) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && k.dim() == 4 && v.sizes() == k.sizes(),
              "window_attention: q, k, v must be 4-D GPU tensors, v like k");
  on_device(k, q, "k");
  on_device(v, q, "v");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "window_attention: q, k, v must share a dtype");
  kfac::AttnArgs a{};
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(3) == q.size(3) && k.size(1) > 0 &&
                  q.size(1) % k.size(1) == 0,
              "window_attention: shapes of q and k do not fit");
  TORCH_CHECK(q.size(3) % 8 == 0 && q.size(3) >= 8 && q.size(3) <= 128,
              "window_attention: head size must be a multiple of 8, at most 128");
  const int64_t lim = (int64_t)1 << 30;
  // a launch has at most 2^32 threads along x
  TORCH_CHECK(q.size(2) < lim && k.size(2) < lim && q.size(0) * q.size(1) < ((int64_t)1 << 24),
              "window_attention: too large");
  a.B = (int)q.size(0);
  a.Hq = (int)q.size(1);
  a.Tq = (int)q.size(2);
  a.D = (int)q.size(3);
  a.Hkv = (int)k.size(1);
  a.Tk = (int)k.size(2);
  a.G = a.Hq / a.Hkv;
  TORCH_CHECK(((int64_t)a.Tq * a.G + 127) / 128 <= 65535,
              "window_attention: more than 65535 row blocks");
  TORCH_CHECK(c.window >= 1 && c.sinks >= 0, "window_attention: window >= 1, sinks >= 0");
  a.W = (int)std::min<int64_t>(c.window, std::max<int64_t>(a.Tk, 1));
  a.S = (int)std::min<int64_t>(c.sinks, a.Tk);
  for (const auto* o : {&lengths, &starts})
    if (o->has_value()) {
      on_device(**o, q, "lengths / q_start");
      TORCH_CHECK((*o)->scalar_type() == at::kInt && (*o)->is_contiguous() &&
                      (*o)->numel() == a.B,
                  "window_attention: lengths and q_start must be contiguous int32 [B]");
    }
  a.lengths = lengths.has_value() ? lengths->data_ptr<int>() : nullptr;
  a.starts = starts.has_value() ? starts->data_ptr<int>() : nullptr;
  a.start = (int)std::max<int64_t>(std::min<int64_t>(c.start, lim), -lim);
  a.start_given = c.start_given;
  a.scale = (float)c.scale;
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  strides3(q, a.qs);
  strides3(k, a.ks);
  strides3(v, a.vs);
  a.splits = 1;
  a.Gmagic = a.G > 1 ? (uint32_t)(((uint64_t)1 << 32) / a.G) : 0xffffffffu;
  return a;
}

// out [B, Hq, Tq, D] over memory laid out [B, Tq, Hq, D] (what the output
// projection reads), and where a backward pass may follow the rows' lse and,
// for 16-bit types and short windows, what out's rounding took away
std::tuple<at::Tensor, at::Tensor, at::Tensor> attn_forward(const at::Tensor& q,
                                                            const at::Tensor& k,
                                                            const at::Tensor& v,
                                                            const OptTensor& lengths,
                                                            const OptTensor& starts,
                                                            const AttnConf& c, bool training) {
  c10::hip::HIPGuardMasqueradingAsCUDA g(q.device());
  kfac::AttnArgs a = attn_args(q, k, v, lengths, starts, c);
  // no transposed view of a buffer: in-place operations on a view that was made
  // without recording are refused later
  const int64_t row = (int64_t)a.Hq * a.D;
  at::Tensor out =
      at::empty_strided({a.B, a.Hq, a.Tq, a.D}, {a.Tq * row, a.D, row, 1}, q.options());
  at::Tensor lse, rest;
  if (training) {
    lse = at::empty({a.B * a.Hkv, (int64_t)a.Tq * a.G}, q.options().dtype(at::kFloat));
    if (q.scalar_type() != at::kFloat && kfac::attn_keeps_rest(a))
      rest = at::empty({a.B, a.Tq, a.Hq, a.D}, q.options());
  }
  a.out = out.data_ptr();
  strides3(out, a.os);
  a.rest = rest.defined() ? rest.data_ptr() : nullptr;
  a.lse = training ? lse.data_ptr<float>() : nullptr;
  int64_t floats = 0;
  kfac::attn_plan(a, &a.splits, &floats);
  at::Tensor ws;
  if (floats > 0) {
    ws = at::empty({floats}, q.options().dtype(at::kFloat));
    const int64_t rows = (int64_t)a.splits * a.B * a.Hkv * a.Tq * a.G;
    a.opart = ws.data_ptr<float>();
    a.lpart = a.opart + rows * a.D;
  }
  kfac::attn_forward(tag(q), a, stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {out, lse, rest};
}

int64_t groups(const at::Tensor& q, const at::Tensor& k) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.size(1) > 0,
              "window_attention: q, k, v must be 4-D");
  return q.size(1) / k.size(1);
}

struct WindowAttnFn : public torch::autograd::Function<WindowAttnFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q_, const at::Tensor& k_,
                            const at::Tensor& v_, const OptTensor& lengths,
                            const OptTensor& starts, int64_t window, int64_t sinks, int64_t start,
                            bool start_given, double scale) {
    const AttnConf c{window, sinks, start, start_given, scale};
    const int64_t G = groups(q_, k_);
    const at::Tensor q = operand(q_, G), k = operand(k_, 1), v = operand(v_, 1);
    auto [out, lse, rest] = attn_forward(q, k, v, lengths, starts, c, true);
    ctx->save_for_backward({q, k, v, out, lse, rest, lengths.has_value() ? *lengths : at::Tensor(),
                            starts.has_value() ? *starts : at::Tensor()});
    ctx->saved_data["conf"] = pack(c);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("window_attention");
    auto sv = ctx->get_saved_variables();
    // saved-tensor hooks may hand tensors back with other strides: out and rest
    // are read with the strides that the forward gave them
    const int64_t G = groups(sv[0], sv[1]);
    const at::Tensor q = operand(sv[0], G), k = operand(sv[1], 1), v = operand(sv[2], 1);
    const at::Tensor out = packed16(sv[3].transpose(1, 2)), lse = packed16(sv[4]);
    const at::Tensor rest = sv[5].defined() ? packed16(sv[5]) : sv[5];
    for (const auto* t : {&out, &lse, &rest})
      if (t->defined()) on_device(*t, q, "what the forward saved");
    const AttnConf c = unpack(ctx->saved_data["conf"].toDoubleVector());
    const OptTensor lengths = sv[6].defined() ? OptTensor(sv[6]) : c10::nullopt;
    const OptTensor starts = sv[7].defined() ? OptTensor(sv[7]) : c10::nullopt;
    c10::hip::HIPGuardMasqueradingAsCUDA g(q.device());
    kfac::AttnArgs a = attn_args(q, k, v, lengths, starts, c);
    const at::Tensor go = operand(grads[0], a.G);
    int64_t floats = 0;
    kfac::attn_bwd_plan(a, &a.sink_groups, &a.far_chunks, &floats);
    TORCH_CHECK((int64_t)(a.Tk + 63) / 64 + (int64_t)a.sink_groups * a.far_chunks <= 65535,
                "window_attention: more than 65535 key blocks");
    // the sinks' shares are joined by a thread for 4 elements
    TORCH_CHECK(a.far_chunks == 0 ||
                    (int64_t)a.B * a.Hkv * a.S * (a.D / 2) < ((int64_t)1 << 32) - 256,
                "window_attention: too large: sinks of all sequences and heads");
    at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
    if (a.Tq == 0 || q.numel() == 0) {
      dk.zero_();
      dv.zero_();
    } else {
      a.out = out.data_ptr();
      strides3(out.transpose(1, 2), a.os);
      a.rest = rest.defined() ? rest.data_ptr() : nullptr;
      a.dout = go.data_ptr();
      strides3(go, a.dos);
      a.dq = dq.data_ptr();
      a.dk = dk.data_ptr();
      a.dv = dv.data_ptr();
      strides3(dq, a.dqs);
      strides3(dk, a.dks);
      strides3(dv, a.dvs);
      a.bound_chunks = kfac::attn_bound_chunks(tag(q), a);
      const int64_t rows = lse.numel(), bounds = (int64_t)a.B * a.Hkv * a.bound_chunks * 2;
      // the sinks' shares (16-byte aligned), the bounds (8), delta, lse_keys
      const at::Tensor ws =
          at::empty({floats + bounds + (bounds > 0 ? 2 : 1) * rows}, lse.options());
      a.lse = lse.data_ptr<float>();
      a.kvpart = ws.data_ptr<float>();
      a.bounds = a.kvpart + floats;
      a.delta = a.bounds + bounds;
      a.lse_keys = bounds > 0 ? a.delta + rows : nullptr;
      if (a.Tk == 0) dq.zero_();
      kfac::attn_backward(tag(q), a, stream());
      C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    at::Tensor u;
    return {dq, dk, dv, u, u, u, u, u, u, u};
  }
};

at::Tensor window_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const OptTensor& lengths, const OptTensor& starts, int64_t window,
                            int64_t sinks, int64_t start, bool start_given, double scale) {
  reverse_only("window_attention", {&q, &k, &v});
  if (records({&q, &k, &v}))
    return WindowAttnFn::apply(q, k, v, lengths, starts, window, sinks, start, start_given, scale);
  const AttnConf c{window, sinks, start, start_given, scale};
  return std::get<0>(
      attn_forward(operand(q, groups(q, k)), operand(k, 1), operand(v, 1), lengths, starts, c,
                   false));
}

// -------------------------------------------------------------- rotary
// a pair's frequency in turns per position, and its axis: fp64 [pairs, 2] on
// the CPU
struct RotaryConf {
  at::Tensor table;
  bool halves;
};

// both operands turned by the positions' angles (sign -1: turned back)
std::tuple<at::Tensor, at::Tensor> rotary_run(const at::Tensor& q, const at::Tensor& k,
                                              const at::Tensor& pos, const RotaryConf& c,
                                              double sign) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && k.dim() == 4 && q.scalar_type() == k.scalar_type() &&
                  q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
              "rotary_axes: q and k must be 4-D GPU tensors of one dtype that differ in heads only");
  on_device(k, q, "k");
  on_device(pos, q, "positions");
  const int64_t B = q.size(0), T = q.size(2), D = q.size(3);
  TORCH_CHECK(c.table.device().is_cpu() && c.table.scalar_type() == at::kDouble &&
                  c.table.dim() == 2 && c.table.size(1) == 2 && c.table.is_contiguous(),
              "rotary_axes: table must be a contiguous fp64 CPU tensor [pairs, 2]");
  const int64_t pairs = c.table.size(0);
  TORCH_CHECK(pairs >= 1 && pairs <= kfac::kMaxRotaryPairs && 2 * pairs <= D && D % 2 == 0,
              "rotary_axes: pairs do not fit the head");
  TORCH_CHECK((pos.scalar_type() == at::kLong || pos.scalar_type() == at::kInt) &&
                  (pos.dim() == 2 || (pos.dim() == 3 && pos.size(0) == B)) &&
                  pos.size(-2) == T,
              "rotary_axes: positions must be int32 / int64 [T, axes] or [B, T, axes]");
  TORCH_CHECK(B * T < (1LL << 31) && B < (1LL << 30) && q.size(1) + k.size(1) < (1LL << 30),
              "rotary_axes: too large");
  c10::hip::HIPGuardMasqueradingAsCUDA g(q.device());
  kfac::RotaryArgs a{};
  const double* entry = c.table.data_ptr<double>();
  for (int64_t i = 0; i < pairs; ++i, entry += 2) {
    TORCH_CHECK(entry[1] >= 0 && entry[1] < pos.size(-1), "rotary_axes: axis of a pair");
    a.tab.turn[i] = entry[0];
    a.tab.axis[i] = (uint8_t)entry[1];
  }
  at::Tensor qo = at::empty({B, q.size(1), T, D}, q.options());
  at::Tensor ko = at::empty({B, k.size(1), T, D}, k.options());
  a.q = q.data_ptr();
  a.k = k.data_ptr();
  a.qo = qo.data_ptr();
  a.ko = ko.data_ptr();
  strides3(q, a.qs);
  strides3(k, a.ks);
  a.pos = pos.data_ptr();
  a.pos64 = pos.scalar_type() == at::kLong;
  a.psB = pos.dim() == 3 ? pos.stride(0) : 0;
  a.psT = pos.stride(-2);
  a.psA = pos.stride(-1);
  a.B = (int)B;
  a.T = (int)T;
  a.D = (int)D;
  a.Hq = (int)q.size(1);
  a.Hk = (int)k.size(1);
  a.pairs = (int)pairs;
  a.sign = (float)sign;
  const int64_t unit = 16 / (int64_t)q.element_size();
  const bool vec = rows16(q) && rows16(k) && D % unit == 0 &&
                   (!c.halves || (pairs % unit == 0 && (D - 2 * pairs) % unit == 0));
  // a thread a unit of a token's head, at most 2^32 of a launch
  TORCH_CHECK(B * T * (vec ? D / unit : D) < (1LL << 32) - 256, "rotary_axes: too large");
  kfac::rotary_axes(tag(q), a, c.halves, vec, stream());
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return {qo, ko};
}

at::Tensor unit_last(const at::Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
}

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k,
                               const at::Tensor& pos, const at::Tensor& table, bool halves) {
    const RotaryConf c{table, halves};
    auto [qo, ko] = rotary_run(unit_last(q), unit_last(k), pos, c, 1.0);
    ctx->save_for_backward({pos});
    ctx->saved_data[halves ? "halves" : "interleaved"] = table;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("rotary_axes");
    const auto kept = ctx->saved_data.begin();
    const RotaryConf c{kept->second.toTensor(), kept->first == "halves"};
    // no heads of an operand that needs no gradient
    const bool need[2] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1)};
    for (int i = 0; i < 2; ++i)
      grads[i] = need[i] ? unit_last(grads[i]) : grads[i].narrow(1, 0, 0);
    auto [dq, dk] = rotary_run(grads[0], grads[1], ctx->get_saved_variables()[0], c, -1.0);
    at::Tensor u;
    return {need[0] ? dq : u, need[1] ? dk : u, u, u, u};
  }
};

std::tuple<at::Tensor, at::Tensor> rotary_axes(const at::Tensor& q, const at::Tensor& k,
                                               const at::Tensor& pos, const at::Tensor& table,
                                               bool halves) {
  reverse_only("rotary_axes", {&q, &k});
  if (records({&q, &k})) {
    auto r = RotaryFn::apply(q, k, pos, table, halves);
    return {r[0], r[1]};
  }
  return rotary_run(unit_last(q), unit_last(k), pos, RotaryConf{table, halves}, 1.0);
}

// ------------------------------------------------------------- distill
kfac::DistillArgs distill_args(const at::Tensor& z, const at::Tensor& teacher,
                               const at::Tensor& index, const OptTensor& rest,
                               double temperature, double weight) {
  TORCH_CHECK(z.is_cuda() && z.dim() == 3 && (z.stride(2) == 1 || z.size(2) == 1),
              "topk_distill_loss: logits must be a GPU tensor [.., .., V] with unit last stride");
  on_device(teacher, z, "teacher_logits");
  on_device(index, z, "teacher_index");
  kfac::DistillArgs a{};
  a.N = z.size(0) * z.size(1);
  a.V = z.size(2);
  a.inner = std::max<int64_t>(z.size(1), 1);
  a.zs0 = z.stride(0);
  a.zs1 = z.stride(1);
  TORCH_CHECK(teacher.scalar_type() == at::kFloat && teacher.is_contiguous() &&
                  index.is_contiguous() && index.numel() == teacher.numel() &&
                  (index.scalar_type() == at::kInt || index.scalar_type() == at::kLong),
              "topk_distill_loss: teacher entries must be contiguous fp32 / int32 or int64");
  TORCH_CHECK(a.V >= 1 && teacher.dim() >= 1, "topk_distill_loss: no columns");
  a.K = (int)teacher.size(-1);
  TORCH_CHECK(teacher.size(-1) >= 1 && teacher.size(-1) <= 1024 &&
                  teacher.numel() == a.N * a.K,
              "topk_distill_loss: 1 to 1024 teacher entries for each row");
  if (rest.has_value()) {
    on_device(*rest, z, "teacher_rest");
    TORCH_CHECK(rest->scalar_type() == at::kFloat && rest->is_contiguous() &&
                    rest->numel() == a.N,
                "topk_distill_loss: teacher_rest must be contiguous fp32, one a row");
    a.rest = rest->data_ptr<float>();
  }
  a.z = z.data_ptr();
  a.teacher = teacher.data_ptr<float>();
  a.index = index.data_ptr();
  a.index64 = index.scalar_type() == at::kLong;
  a.temperature = (float)temperature;
  a.weight = (float)weight;
  a.aligned = rows16(z);
  kfac::distill_split(a.N, a.V, rest.has_value(), &a.slice, &a.splits);
  // blocks of 256 threads, at most 2^32 of a launch
  TORCH_CHECK(a.N * a.splits < (1LL << 24), "topk_distill_loss: too many rows");
  return a;
}

struct DistillOut {
  at::Tensor loss, info, mean, dz;
};

// reduction: 0 none (of the shape `lead`), 1 sum, 2 mean; grad: a backward pass
// will follow
DistillOut distill_run(const at::Tensor& z, const at::Tensor& teacher, const at::Tensor& index,
                       const OptTensor& rest, double temperature, double weight,
                       int64_t reduction, const std::vector<int64_t>& lead, bool grad) {
  c10::hip::HIPGuardMasqueradingAsCUDA g(z.device());
  kfac::DistillArgs a = distill_args(z, teacher, index, rest, temperature, weight);
  const auto f32 = z.options().dtype(at::kFloat);
  DistillOut o;
  o.info = at::empty({a.N, 8}, f32);
  at::Tensor rows = at::empty(lead, f32);
  TORCH_CHECK(rows.numel() == a.N, "topk_distill_loss: rows");
  a.info = reinterpret_cast<float4*>(o.info.data_ptr<float>());
  a.row_loss = rows.data_ptr<float>();
  o.loss = rows;
  float *loss = nullptr, *mean = nullptr;
  if (reduction != 0) {
    o.loss = at::empty({}, f32);
    o.mean = at::empty({1}, f32);
    loss = o.loss.data_ptr<float>();
    mean = o.mean.data_ptr<float>();
  }
  if (grad && reduction != 0 && kfac::distill_fuses(tag(z), a.N, a.V)) {
    o.dz = at::empty(z.sizes(), z.options());
    a.dz = o.dz.data_ptr();
    a.dz_aligned = rows16(o.dz);
    a.mean = mean;
    kfac::distill_forward_grad(tag(z), a, loss, (int)reduction, stream());
  } else {
    at::Tensor part;
    if (a.splits > 1) {
      part = at::empty({a.N * a.splits, 4}, f32);
      a.part = reinterpret_cast<float4*>(part.data_ptr<float>());
    }
    kfac::distill_forward(tag(z), a, loss, mean, (int)reduction, stream());
    if (reduction == 0 && weight != 1.0) rows.mul_(weight);
  }
  C10_HIP_KERNEL_LAUNCH_CHECK();
  return o;
}

struct DistillFn : public torch::autograd::Function<DistillFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& teacher,
                            const at::Tensor& index, const OptTensor& rest, double temperature,
                            double weight, int64_t reduction, const std::vector<int64_t>& lead) {
    auto o = distill_run(z, teacher, index, rest, temperature, weight, reduction, lead, true);
    // the gradient as well: saved-tensor hooks (offloading, checkpoints) see it
    ctx->save_for_backward({z, teacher, index, rest.has_value() ? *rest : at::Tensor(), o.info,
                            o.mean, o.dz});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["reduction"] = reduction;
    return o.loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("topk_distill_loss");
    auto sv = ctx->get_saved_variables();
    // saved-tensor hooks may hand tensors back with other strides
    const at::Tensor z = unit_last(sv[0]);
    c10::hip::HIPGuardMasqueradingAsCUDA g(z.device());
    const at::Tensor up = grads[0].to(at::kFloat).contiguous();
    at::Tensor dz, u;
    if (sv[6].defined() && ctx->saved_data.count("spent") == 0) {
      // the gradient that the forward wrote is given away and scaled in
      // place, so it serves one backward pass; another one of the same graph
      // (retain_graph) computes its own below.  Whatever becomes of it, the
      // saved tensor's version stays: that other pass still unpacks it.
      ctx->saved_data["spent"] = true;
      dz = sv[6].variable_data();
      TORCH_CHECK(dz.sizes() == z.sizes() && dz.scalar_type() == z.scalar_type() &&
                      dz.device() == z.device(),
                  "topk_distill_loss: a saved-tensor hook changed the stored gradient");
      dz = packed16(dz);  // a hook may hand it back otherwise
      if (dz.numel() > 0)
        kfac::distill_scale(tag(z), dz.data_ptr(), dz.numel(), up.data_ptr<float>(), stream());
      C10_HIP_KERNEL_LAUNCH_CHECK();
      return {dz, u, u, u, u, u, u, u};
    }
    const OptTensor rest = sv[3].defined() ? OptTensor(sv[3].contiguous()) : c10::nullopt;
    const at::Tensor teacher = sv[1].contiguous(), index = sv[2].contiguous();
    kfac::DistillArgs a =
        distill_args(z, teacher, index, rest, ctx->saved_data["temperature"].toDouble(),
                     ctx->saved_data["weight"].toDouble());
    const bool rows = ctx->saved_data["reduction"].toInt() == 0;
    dz = at::empty(z.sizes(), z.options());
    const at::Tensor info = packed16(sv[4]);
    TORCH_CHECK(info.is_cuda() && info.numel() == a.N * 8, "topk_distill_loss: saved statistics");
    a.info = reinterpret_cast<float4*>(info.data_ptr<float>());
    a.upstream = up.data_ptr<float>();
    a.upstream_rows = rows;
    a.mean = rows ? nullptr : sv[5].data_ptr<float>();
    a.dz = dz.data_ptr();
    a.dz_aligned = rows16(dz);
    kfac::distill_backward(tag(z), a, stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {dz, u, u, u, u, u, u, u};
  }
};

at::Tensor topk_distill_loss(const at::Tensor& z, const at::Tensor& teacher,
                             const at::Tensor& index, const OptTensor& rest, double temperature,
                             double weight, int64_t reduction, const std::vector<int64_t>& lead) {
  reverse_only("topk_distill_loss", {&z});
  if (records({&z}))
    return DistillFn::apply(z, teacher, index, rest, temperature, weight, reduction, lead);
  return distill_run(z, teacher, index, rest, temperature, weight, reduction, lead, false).loss;
}

}  // namespace

void bind_lm_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("window_attention", &window_attention, py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("lengths"), py::arg("starts"), py::arg("window"), py::arg("sinks"),
        py::arg("start"), py::arg("start_given"), py::arg("scale"));
  m.def("rotary_axes", &rotary_axes, py::arg("q"), py::arg("k"), py::arg("positions"),
        py::arg("table"), py::arg("halves"));
  m.def("topk_distill_loss", &topk_distill_loss, py::arg("logits"), py::arg("teacher"),
        py::arg("index"), py::arg("rest"), py::arg("temperature"),
        py::arg("weight"), py::arg("reduction"), py::arg("lead"));
}

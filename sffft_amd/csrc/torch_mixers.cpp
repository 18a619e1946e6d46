// PyTorch operators over the C ABI of libsffft_ops.so (sffft_ops.h), registered from C++ beside the
// convolution's (torch_ops.cpp), in the same library and namespace. No counterparts in the reference.
//
//   sffft::linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, float scale,
//                           Tensor? initial_state=None, Tensor? lengths=None) -> (Tensor, Tensor)
//       q [B, T, H, Dk], k [B, T, Hk, Dk], v [B, T, Hk, Dv] -> o [B, T, H, Dv], final state
//       [B, H, Dk, Dv] fp32; differentiable in q, k, v and initial_state
//   sffft::linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state,
//                           float scale, Tensor? slots=None) -> Tensor
//       one token: q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv]; state [slots, H, Dk, Dv] in place
//   sffft::rotary(Tensor q, Tensor k, Tensor table, Tensor? positions=None, bool interleaved=False,
//                 bool inverse=False) -> (Tensor, Tensor)      differentiable in q and k
//   sffft::rotary_(Tensor(a!) q, Tensor(b!) k, ...) -> ()       the same in place
//   sffft::block_norm(Tensor x, Tensor y, Tensor w_pre, Tensor? w_post=None, Tensor? gate=None,
//                 Tensor? scale=None, str activation="none", float eps=1e-6) -> (Tensor, Tensor)
//       r = x + scale . act(gate) . norm(y) w_post, h = norm(r) w_pre; differentiable in all
//   sffft::pre_norm(Tensor x, Tensor w, float eps=1e-6) -> Tensor     the first norm alone
//
// Each launches on the current stream of its input's device; outputs and workspaces come from torch's
// allocator, which ties them to that stream. Inputs whose channels are not contiguous, or whose
// rows are not aligned to 16 bytes where the kernel needs that, are copied first.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "sffft_ops.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

void* stream_of() { return c10::hip::getCurrentHIPStream().stream(); }

void check(int rc, const char* what) {
  TORCH_CHECK(rc == SFFFT_OK, what, " failed: ", sffft_strerror(rc), " (", rc, ") ", rc == SFFFT_EHIP ? sffft_ops_last_error() : "");
}

const void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.const_data_ptr() : nullptr; }
const void* ptr(const OptTensor& t) { return t ? ptr(*t) : nullptr; }
float* fptr(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
const float* cfptr(const OptTensor& t) { return t ? t->const_data_ptr<float>() : nullptr; }

int io_of(const Tensor& t, const char* op) {
  TORCH_CHECK(t.is_cuda() && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16), op,
              ": inputs must be float32 or bfloat16 GPU tensors, got ", t.scalar_type(), " on ", t.device());
  return t.scalar_type() == at::kBFloat16 ? SFFFT_IO_BF16 : SFFFT_IO_F32;
}
// a fp32 parameter or state on x's device
void check_f32(const char* op, const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.device() == x.device(), op, ": ", name, " must be float32 on ",
              x.device(), ", got ", t.scalar_type(), " on ", t.device());
}
void check_like(const char* op, const char* name, const Tensor& t, const Tensor& x) {
  TORCH_CHECK(t.scalar_type() == x.scalar_type() && t.device() == x.device(), op, ": ", name, " must be ",
              x.scalar_type(), " on ", x.device(), ", got ", t.scalar_type(), " on ", t.device());
}
OptTensor dense(const OptTensor& t) { return t ? OptTensor(t->contiguous()) : t; }
Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// t itself where its channels are contiguous and its rows aligned to 16 bytes, else a copy
Tensor rows16(const Tensor& t) {
  const int64_t e = t.element_size();
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < t.dim(); d++) ok = ok && t.stride(d) >= 0 && t.stride(d) * e % 16 == 0;
  if (t.dim() == 4) ok = ok && t.stride(1) <= (1 << 24) - 128;  // sffft_linattn's token stride
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ---- linear attention ----

constexpr const char* LA = "sffft::linear_attention";

struct Attention {
  sffft_linattn p;
  Tensor q, k, v, decay;
  OptTensor state, lengths;
};

// The arguments checked, and laid out as the kernels take them. `step`: one token, no T dimension.
Attention attention_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, double scale,
                       const OptTensor& state, const OptTensor& lengths, bool step) {
  Attention a;
  a.p = {};
  a.p.io = io_of(q, LA);
  check_like(LA, "k", k, q);
  check_like(LA, "v", v, q);
  const int64_t d = step ? 3 : 4;
  TORCH_CHECK(q.dim() == d && k.dim() == d && v.dim() == d, LA, ": q, k, v must have ", d, " dimensions, got ",
              q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  const int64_t B = q.size(0), T = step ? 1 : q.size(1), H = q.size(-2), Dk = q.size(-1);
  const int64_t Hk = k.size(-2), Dv = v.size(-1);
  TORCH_CHECK(k.size(0) == B && v.size(0) == B && (step || (k.size(1) == T && v.size(1) == T)) && v.size(-2) == Hk &&
                  k.size(-1) == Dk && Hk >= 1 && H % Hk == 0,
              LA, ": k and v must be the keys [.., Hk, Dk] and values [.., Hk, Dv] of q's tokens, H a multiple of Hk, got ",
              q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  TORCH_CHECK(Dk >= 8 && Dv >= 8 && Dk <= 128 && Dv <= 128 && Dk % 8 == 0 && Dv % 8 == 0, LA,
              ": head channels must be multiples of 8 up to 128, got ", Dk, " and ", Dv);
  TORCH_CHECK(B <= INT32_MAX && T <= INT32_MAX && H * std::max(Dk, Dv) <= (1 << 23) - 64, LA, ": shape too large");
  check_f32(LA, "log_decay", log_decay, q);
  TORCH_CHECK(log_decay.dim() == 1 && log_decay.size(0) == H, LA, ": log_decay must be [H] = [", H, "], got ",
              log_decay.sizes());
  if (state) {
    check_f32(LA, "the state", *state, q);
    TORCH_CHECK(state->dim() == 4 && (step || state->size(0) == B) && state->size(1) == H && state->size(2) == Dk &&
                    state->size(3) == Dv,
                LA, ": the state must be [", step ? "slots" : "B", ", H, Dk, Dv] for q ", q.sizes(), " and v ",
                v.sizes(), ", got ", state->sizes());
  }
  if (lengths)
    TORCH_CHECK(lengths->scalar_type() == at::kInt && lengths->device() == q.device() && lengths->dim() == 1 &&
                    lengths->size(0) == B,
                LA, ": ", step ? "slots" : "lengths", " must be int32 [B] on ", q.device(), ", got ",
                lengths->scalar_type(), " ", lengths->sizes());
  a.q = rows16(q), a.k = rows16(k), a.v = rows16(v), a.decay = log_decay.contiguous();
  a.state = step ? state : dense(state), a.lengths = dense(lengths);
  a.p.B = (int)B, a.p.T = (int)T, a.p.H = (int)H, a.p.Hk = (int)Hk, a.p.Dk = (int)Dk, a.p.Dv = (int)Dv;
  a.p.scale = (float)scale;
  auto strides = [&](const Tensor& t, long long* s) {
    s[0] = t.stride(0), s[1] = step ? 0 : t.stride(1), s[2] = t.stride(-2);
  };
  strides(a.q, a.p.q), strides(a.k, a.p.k), strides(a.v, a.p.v);
  return a;
}

std::tuple<Tensor, Tensor> attention_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay,
                                         double scale, const OptTensor& state, const OptTensor& lengths) {
  const c10::DeviceGuard guard(q.device());
  const Attention a = attention_of(q, k, v, log_decay, scale, state, lengths, false);
  const int64_t B = a.p.B, T = a.p.T, H = a.p.H, Dk = a.p.Dk, Dv = a.p.Dv;
  Tensor o = at::empty({B, T, H, Dv}, q.options());
  Tensor s = at::empty({B, H, Dk, Dv}, q.options().dtype(at::kFloat));
  if (B == 0 || H == 0) return {o, s};
  if (T == 0) {
    if (a.state) s.copy_(*a.state);
    else s.zero_();
    return {o, s};
  }
  const size_t wb = sffft_linattn_work_bytes(&a.p, 0);
  Tensor work = workspace(wb, q);
  check(sffft_linattn_fwd(&a.p, ptr(a.q), ptr(a.k), ptr(a.v), a.decay.const_data_ptr<float>(), cfptr(a.state),
                          a.lengths ? a.lengths->const_data_ptr<int>() : nullptr, o.data_ptr(), fptr(s),
                          wb ? work.data_ptr() : nullptr, wb, stream_of()),
        LA);
  return {o, s};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> attention_backward_gpu(
    const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, double scale, const OptTensor& state,
    const OptTensor& lengths, const OptTensor& go_in, const OptTensor& ds_in) {
  const c10::DeviceGuard guard(q.device());
  Attention a = attention_of(q, k, v, log_decay, scale, state, lengths, false);
  const int64_t B = a.p.B, T = a.p.T, H = a.p.H, Hk = a.p.Hk, Dk = a.p.Dk, Dv = a.p.Dv;
  Tensor dq = at::empty({B, T, H, Dk}, q.options()), dk = at::empty({B, T, Hk, Dk}, q.options());
  Tensor dv = at::empty({B, T, Hk, Dv}, q.options());
  // no gradient of a state that there is not
  Tensor ds0 = a.state ? at::empty({B, H, Dk, Dv}, q.options().dtype(at::kFloat)) : at::empty({0}, q.options().dtype(at::kFloat));
  if (ds_in) {
    check_f32(LA, "the final state's gradient", *ds_in, q);
    TORCH_CHECK(ds_in->sizes() == at::IntArrayRef({B, H, Dk, Dv}), LA,
                ": the final state's gradient must be [B, H, Dk, Dv], got ", ds_in->sizes());
  }
  const OptTensor ds = dense(ds_in);
  if (B == 0 || H == 0) return {dq, dk.zero_(), dv.zero_(), ds0};  // keys without queries
  if (T == 0) {
    if (a.state && ds) ds0.copy_(*ds);
    else ds0.zero_();
    return {dq, dk, dv, ds0};
  }
  Tensor go = go_in ? *go_in : at::zeros({B, T, H, Dv}, q.options());
  check_like(LA, "the output's gradient", go, q);
  TORCH_CHECK(go.sizes() == at::IntArrayRef({B, T, H, Dv}), LA, ": the output's gradient must be [B, T, H, Dv], got ",
              go.sizes());
  go = rows16(go);
  for (int i = 0; i < 3; i++) a.p.go[i] = go.stride(i);
  const size_t wb = sffft_linattn_work_bytes(&a.p, 1);
  Tensor work = workspace(wb, q);
  check(sffft_linattn_bwd(&a.p, ptr(a.q), ptr(a.k), ptr(a.v), a.decay.const_data_ptr<float>(), cfptr(a.state),
                          a.lengths ? a.lengths->const_data_ptr<int>() : nullptr, ptr(go), cfptr(ds), dq.data_ptr(),
                          dk.data_ptr(), dv.data_ptr(), a.state ? fptr(ds0) : nullptr, wb ? work.data_ptr() : nullptr, wb, stream_of()),
        LA);
  return {dq, dk, dv, ds0};
}

Tensor step_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                double scale, const OptTensor& slots) {
  const c10::DeviceGuard guard(q.device());
  const Attention a = attention_of(q, k, v, log_decay, scale, state, slots, true);
  TORCH_CHECK(state.is_contiguous(), "sffft::linear_attention_step: the state must be contiguous");
  TORCH_CHECK(slots || state.size(0) >= q.size(0), "sffft::linear_attention_step: ", q.size(0),
              " sequences need as many rows of state or slots, got ", state.size(0));
  Tensor o = at::empty({a.p.B, a.p.H, a.p.Dv}, q.options());
  if (o.numel() == 0) return o;
  TORCH_CHECK(state.size(0) >= 1 && state.size(0) <= INT32_MAX, "sffft::linear_attention_step: the state has ",
              state.size(0), " slots");
  check(sffft_linattn_step(&a.p, ptr(a.q), ptr(a.k), ptr(a.v), a.decay.const_data_ptr<float>(),
                           static_cast<float*>(state.data_ptr()), (int)state.size(0),
                           a.lengths ? a.lengths->const_data_ptr<int>() : nullptr, o.data_ptr(), stream_of()),
        "sffft::linear_attention_step");
  return o;
}

// ---- rotary ----

constexpr const char* ROT = "sffft::rotary";

void rotary_run(const Tensor& q, const Tensor& k, const Tensor& table_in, const OptTensor& positions,
                bool interleaved, bool inverse, const Tensor& qo, const Tensor& ko) {
  sffft_rotary p = {};
  p.io = io_of(q, ROT);
  check_like(ROT, "k", k, q);
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3),
              ROT, ": q and k must be [B, T, H, D] and [B, T, Hk, D], got ", q.sizes(), " and ", k.sizes());
  const int64_t B = q.size(0), T = q.size(1);
  check_f32(ROT, "table", table_in, q);
  TORCH_CHECK(table_in.dim() == 2 && table_in.size(0) >= 1 && table_in.size(1) >= 2 && table_in.size(1) % 2 == 0 &&
                  table_in.size(1) <= q.size(3) && q.size(3) % 2 == 0,
              ROT, ": table must be [positions, R] with R even and at most D = ", q.size(3), " (even too), got ",
              table_in.sizes());
  TORCH_CHECK(B <= INT32_MAX && T <= INT32_MAX && q.size(2) <= INT32_MAX && k.size(2) <= INT32_MAX &&
                  q.size(3) <= INT32_MAX && table_in.size(0) <= INT32_MAX && B * T <= INT32_MAX &&
                  (q.size(2) + k.size(2)) * (q.size(3) / 2) <= 65535,
              ROT, ": shape too large");
  OptTensor pos = dense(positions);
  if (pos) {
    TORCH_CHECK((pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong) && pos->device() == q.device() &&
                    pos->dim() == 2 && pos->size(0) == B && pos->size(1) == T,
                ROT, ": positions must be int32 or int64 [B, T] on ", q.device(), ", got ", pos->scalar_type(), " ",
                pos->sizes());
    p.pos_bits = pos->scalar_type() == at::kLong ? 64 : 32;
  }
  if (B * T * (q.size(2) + k.size(2)) == 0) return;
  const Tensor table = table_in.contiguous();
  // the call's first array has heads: k's where q has none
  const bool alone = q.size(2) == 0;
  const Tensor &a = alone ? k : q, &c = alone ? q : k, &ao = alone ? ko : qo, &co = alone ? qo : ko;
  p.B = (int)B, p.T = (int)T, p.H = (int)a.size(2), p.Hk = (int)c.size(2), p.D = (int)a.size(3);
  p.R = (int)table.size(1), p.interleaved = interleaved, p.inverse = inverse, p.positions = (int)table.size(0);
  for (int i = 0; i < 3; i++) p.q[i] = a.stride(i), p.k[i] = c.stride(i), p.qo[i] = ao.stride(i), p.ko[i] = co.stride(i);
  const int rc = sffft_rotary_apply(&p, ptr(a), ptr(c), table.const_data_ptr<float>(), ptr(pos), ao.data_ptr(),
                                    p.Hk ? co.data_ptr() : nullptr, stream_of());
  TORCH_CHECK(rc != SFFFT_EINVAL || !ao.is_same(a), ROT, "_: q and k may overlap neither themselves nor each other, nor the table "
              "or positions; got strides ", q.strides(), " and ", k.strides());
  check(rc, ROT);
}

Tensor channels_last(const Tensor& t) {
  bool ok = t.dim() > 0 && t.stride(-1) == 1;
  for (int64_t d = 0; d < t.dim(); d++) ok = ok && t.stride(d) >= 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::tuple<Tensor, Tensor> rotary_gpu(const Tensor& q, const Tensor& k, const Tensor& table, const OptTensor& positions,
                                      bool interleaved, bool inverse) {
  const c10::DeviceGuard guard(q.device());
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  rotary_run(channels_last(q), channels_last(k), table, positions, interleaved, inverse, qo, ko);
  return {qo, ko};
}

void rotary_inplace_gpu(const Tensor& q, const Tensor& k, const Tensor& table, const OptTensor& positions,
                        bool interleaved) {
  const c10::DeviceGuard guard(q.device());
  for (const Tensor* t : {&q, &k})
    TORCH_CHECK(t->dim() == 4 && (t->numel() == 0 || t->stride(3) == 1), ROT,
                "_: q and k must be [B, T, H, D] with contiguous channels, got ", t->sizes(), " strides ", t->strides());
  rotary_run(q, k, table, positions, interleaved, false, q, k);
}

// ---- norms ----

constexpr const char* BN = "sffft::block_norm";

int act_of(c10::string_view name) {
  if (name == "none") return SFFFT_ACT_NONE;
  if (name == "sigmoid") return SFFFT_ACT_SIGMOID;
  TORCH_CHECK(name == "silu", BN, ": activation must be none, sigmoid or silu, got ", std::string(name));
  return SFFFT_ACT_SILU;
}

// rows [n, C] of x at one stride, without a copy where its dimensions allow it
Tensor rows_of(const Tensor& x) {
  const int64_t C = x.size(-1);
  if (x.dim() == 1 || x.numel() == 0) return x.contiguous().view({-1, C});
  int64_t stride = x.stride(-2), n = x.size(-2);
  bool ok = x.stride(-1) == 1 && (n == 1 || stride >= C);
  if (n == 1) stride = 0;
  for (int64_t d = x.dim() - 3; d >= 0; d--) {
    if (x.size(d) == 1) continue;
    if (n == 1) stride = x.stride(d), ok = ok && stride >= C;
    else ok = ok && x.stride(d) == stride * n;
    n *= x.size(d);
  }
  if (!ok) return x.contiguous().view({-1, C});
  return x.as_strided({n, C}, {n == 1 ? C : stride, 1});
}

struct Norm {
  sffft_blocknorm p;
  Tensor x, y, gate;
  OptTensor w_pre, w_post, scale;
};

Norm norm_of(const Tensor& x, const OptTensor& y, const Tensor& w_pre, const OptTensor& w_post, const OptTensor& gate,
             const OptTensor& scale, c10::string_view activation, double eps) {
  Norm n;
  n.p = {};
  n.p.io = io_of(x, BN);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384, BN, ": x must be [.., C] with C from 1 to 16384, got ",
              x.sizes());
  const int64_t C = x.size(-1);
  n.p.act = act_of(activation);
  auto vector = [&](const OptTensor& w, const char* name) -> OptTensor {
    if (!w) return w;
    check_f32(BN, name, *w, x);
    TORCH_CHECK(w->dim() == 1 && w->size(0) == C, BN, ": ", name, " must be [C] = [", C, "], got ", w->sizes());
    return OptTensor(w->contiguous());
  };
  n.w_pre = vector(w_pre, "w_pre"), n.w_post = vector(w_post, "w_post"), n.scale = vector(scale, "scale");
  n.x = rows_of(x);
  n.p.rows = n.x.size(0), n.p.C = (int)C, n.p.gate_rows = 1, n.p.eps = (float)eps;
  TORCH_CHECK(n.p.eps >= 0.f && std::isfinite(n.p.eps), BN, ": eps must be finite and not negative, got ", eps);
  n.p.x = n.x.stride(0);
  if (y) {
    check_like(BN, "y", *y, x);
    TORCH_CHECK(y->sizes() == x.sizes(), BN, ": y must have x's shape ", x.sizes(), ", got ", y->sizes());
    n.y = rows_of(*y);
    n.p.y = n.y.stride(0);
  }
  if (gate) {
    check_like(BN, "gate", *gate, x);
    // [.., T, C] or [.., 1, C]: one row for each token, or for each sequence
    bool ok = gate->dim() == x.dim() && gate->size(-1) == C;
    for (int64_t d = 0; ok && d + 2 < x.dim(); d++) ok = gate->size(d) == x.size(d);
    const bool each = ok && (x.dim() == 1 || gate->size(-2) == x.size(-2));
    TORCH_CHECK(ok && (each || gate->size(-2) == 1), BN, ": gate must have x's shape ", x.sizes(),
                ", or 1 in place of its tokens, got ", gate->sizes());
    n.gate = rows_of(*gate);
    n.p.gate = n.gate.stride(0);
    n.p.gate_rows = each ? 1 : x.size(-2);
  }
  return n;
}

std::tuple<Tensor, Tensor> norm_gpu(const Tensor& x, const OptTensor& y, const Tensor& w_pre, const OptTensor& w_post,
                                    const OptTensor& gate, const OptTensor& scale, c10::string_view activation,
                                    double eps) {
  const c10::DeviceGuard guard(x.device());
  const Norm n = norm_of(x, y, w_pre, w_post, gate, scale, activation, eps);
  Tensor h = at::empty(x.sizes(), x.options()), r = y ? at::empty(x.sizes(), x.options()) : Tensor();
  if (x.numel())
    check(sffft_blocknorm_fwd(&n.p, ptr(n.x), ptr(n.y), ptr(n.gate), cfptr(n.w_pre), cfptr(n.w_post), cfptr(n.scale),
                              y ? r.data_ptr() : nullptr, h.data_ptr(), stream_of()),
          BN);
  return {r, h};
}

std::tuple<Tensor, Tensor> block_norm_gpu(const Tensor& x, const Tensor& y, const Tensor& w_pre, const OptTensor& w_post,
                                          const OptTensor& gate, const OptTensor& scale, c10::string_view activation,
                                          double eps) {
  return norm_gpu(x, y, w_pre, w_post, gate, scale, activation, eps);
}
Tensor pre_norm_gpu(const Tensor& x, const Tensor& w, double eps) {
  return std::get<1>(norm_gpu(x, std::nullopt, w, std::nullopt, std::nullopt, std::nullopt, "none", eps));
}

// dx, dy, dgate, dw_pre, dw_post, dscale; those of absent inputs are empty
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> norm_backward_gpu(
    const OptTensor& gr_in, const OptTensor& gh_in, const Tensor& x, const OptTensor& y, const Tensor& w_pre,
    const OptTensor& w_post, const OptTensor& gate, const OptTensor& scale, c10::string_view activation, double eps) {
  const c10::DeviceGuard guard(x.device());
  Norm n = norm_of(x, y, w_pre, w_post, gate, scale, activation, eps);
  const auto f32 = x.options().dtype(at::kFloat);
  const Tensor none = at::empty({0}, f32);
  auto like = [&](const OptTensor& t) { return t ? at::empty(t->sizes(), t->options()) : none; };
  Tensor dx = like(x), dy = like(y), dg = like(gate), dwq = like(w_pre), dwp = like(w_post), ds = like(scale);
  if (x.numel() == 0 || (!gr_in && !gh_in)) {
    for (Tensor t : {dx, dy, dg, dwq, dwp, ds}) t.zero_();
    return {dx, dy, dg, dwq, dwp, ds};
  }
  auto grad = [&](const OptTensor& t, const char* name, long long* stride) {
    if (!t) return Tensor();
    check_like(BN, name, *t, x);
    TORCH_CHECK(t->sizes() == x.sizes(), BN, ": ", name, " must have x's shape ", x.sizes(), ", got ", t->sizes());
    const Tensor rows = rows_of(*t);
    *stride = rows.stride(0);
    return rows;
  };
  const Tensor gr = grad(gr_in, "the gradient of r", &n.p.gr), gh = grad(gh_in, "the gradient of h", &n.p.gh);
  const size_t wb = sffft_blocknorm_work_bytes(&n.p, y.has_value(), gate.has_value());
  Tensor work = workspace(wb, x);
  check(sffft_blocknorm_bwd(&n.p, ptr(n.x), ptr(n.y), ptr(n.gate), cfptr(n.w_pre), cfptr(n.w_post), cfptr(n.scale),
                            ptr(gr), ptr(gh), dx.data_ptr(), y ? dy.data_ptr() : nullptr,
                            gate ? dg.data_ptr() : nullptr, fptr(dwq), w_post ? fptr(dwp) : nullptr,
                            scale ? fptr(ds) : nullptr, work.data_ptr(), wb, stream_of()),
        BN);
  return {dx, dy, dg, dwq, dwp, ds};
}

// ---- dispatch and gradients ----

template <class Sig>
auto op_handle(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

using AttentionSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, double,
                                                const OptTensor&, const OptTensor&);
using AttentionBackwardSig = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&,
                                                                        const Tensor&, double, const OptTensor&,
                                                                        const OptTensor&, const OptTensor&,
                                                                        const OptTensor&);
using StepSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, double,
                       const OptTensor&);
using RotarySig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, bool, bool);
using RotaryInplaceSig = void(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, bool);
using BlockNormSig = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                                                const OptTensor&, const OptTensor&, c10::string_view, double);
using PreNormSig = Tensor(const Tensor&, const Tensor&, double);
using NormBackwardSig = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>(
    const OptTensor&, const OptTensor&, const Tensor&, const OptTensor&, const Tensor&, const OptTensor&,
    const OptTensor&, const OptTensor&, c10::string_view, double);

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
Tensor plain(const OptTensor& t) { return t ? *t : Tensor(); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && wants_grad(*t); }
// Whether a call is recorded: a node of the graph costs the host a microsecond or two, as much as a small kernel.
template <class... A>
bool recorded(const A&... t) {
  return at::GradMode::is_enabled() && (wants_grad(t) || ...);
}

// No operator has a forward-mode derivative. A tangent needs no requires_grad and no recording: a call below autograd
// would drop it, and its output's would read as zero.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <class... A>
void refuse_tangents(const char* op, const A&... t) {
  TORCH_CHECK(!(has_tangent(t) || ...), op, " has no forward-mode derivative (jvp)");
}

void refuse_second_derivative(const char* op, const variable_list& grads) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, " has no second derivative (backward with create_graph)");
  for (const Variable& g : grads) refuse_tangents(op, g);
}

class AttentionFn : public torch::autograd::Function<AttentionFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& log_decay, double scale, const OptTensor& state, const OptTensor& lengths) {
    static const auto op = op_handle<AttentionSig>("sffft::linear_attention");
    ctx->save_for_backward({q, k, v, log_decay, plain(state), plain(lengths)});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView guard;
    auto out = op.call(q, k, v, log_decay, scale, state, lengths);
    return {std::get<0>(out), std::get<1>(out)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_handle<AttentionBackwardSig>("sffft::linear_attention_backward");
    refuse_second_derivative(LA, grads);
    const variable_list s = ctx->get_saved_variables();
    variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    auto g = op.call(s[0], s[1], s[2], s[3], ctx->saved_data["scale"].toDouble(), opt(s[4]), opt(s[5]), opt(grads[0]),
                     opt(grads[1]));
    out[0] = std::get<0>(g), out[1] = std::get<1>(g), out[2] = std::get<2>(g);
    if (s[4].defined()) out[5] = std::get<3>(g);
    return out;
  }
};

std::tuple<Tensor, Tensor> attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                                              const Tensor& log_decay, double scale, const OptTensor& state,
                                              const OptTensor& lengths) {
  TORCH_CHECK(!log_decay.requires_grad() || !at::GradMode::is_enabled(), LA,
              ": log_decay has no gradient (the decays are constants of the layer)");
  refuse_tangents(LA, q, k, v, log_decay, state);
  if (!recorded(q, k, v, state)) {
    static const auto op = op_handle<AttentionSig>("sffft::linear_attention");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(q, k, v, log_decay, scale, state, lengths);
  }
  auto out = AttentionFn::apply(q, k, v, log_decay, scale, state, lengths);
  return {out[0], out[1]};
}

Tensor step_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& log_decay, const Tensor& state,
                     double scale, const OptTensor& slots) {
  static const auto op = op_handle<StepSig>("sffft::linear_attention_step");
  TORCH_CHECK(!recorded(q, k, v, state, log_decay),
              "sffft::linear_attention_step has no gradient: use sffft::linear_attention");
  refuse_tangents("sffft::linear_attention_step", q, k, v, log_decay, state);
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor o = op.call(q, k, v, log_decay, state, scale, slots);
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return o;
}

std::tuple<Tensor, Tensor> rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& table,
                                           const OptTensor& positions, bool interleaved, bool inverse);

// Its gradient is the rotation by the negative angle, itself differentiable.
class RotaryFn : public torch::autograd::Function<RotaryFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& table,
                               const OptTensor& positions, bool interleaved, bool inverse) {
    static const auto op = op_handle<RotarySig>("sffft::rotary");
    ctx->save_for_backward({table, plain(positions)});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    at::AutoDispatchBelowADInplaceOrView guard;
    auto out = op.call(q, k, table, positions, interleaved, inverse);
    return {std::get<0>(out), std::get<1>(out)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_handle<RotarySig>("sffft::rotary");
    const variable_list s = ctx->get_saved_variables();
    auto g = op.call(grads[0], grads[1], s[0], opt(s[1]), ctx->saved_data["interleaved"].toBool(),
                     !ctx->saved_data["inverse"].toBool());
    return {std::get<0>(g), std::get<1>(g), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> rotary_autograd(const Tensor& q, const Tensor& k, const Tensor& table,
                                           const OptTensor& positions, bool interleaved, bool inverse) {
  TORCH_CHECK(!table.requires_grad() || !at::GradMode::is_enabled(), ROT, ": the table has no gradient");
  refuse_tangents(ROT, q, k, table);
  if (!recorded(q, k)) {
    static const auto op = op_handle<RotarySig>("sffft::rotary");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(q, k, table, positions, interleaved, inverse);
  }
  auto out = RotaryFn::apply(q, k, table, positions, interleaved, inverse);
  return {out[0], out[1]};
}

void rotary_inplace_autograd(const Tensor& q, const Tensor& k, const Tensor& table, const OptTensor& positions,
                             bool interleaved) {
  static const auto op = op_handle<RotaryInplaceSig>("sffft::rotary_");
  TORCH_CHECK(!recorded(q, k),
              "sffft::rotary_ records no gradient: use sffft::rotary");
  refuse_tangents("sffft::rotary_", q, k, table);
  at::AutoDispatchBelowADInplaceOrView guard;
  op.call(q, k, table, positions, interleaved);
  for (const Tensor* t : {&q, &k})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

class BlockNormFn : public torch::autograd::Function<BlockNormFn> {
 public:
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& y, const Tensor& w_pre,
                               const OptTensor& w_post, const OptTensor& gate, const OptTensor& scale,
                               c10::string_view activation, double eps) {
    static const auto op = op_handle<BlockNormSig>("sffft::block_norm");
    ctx->save_for_backward({x, y, w_pre, plain(w_post), plain(gate), plain(scale)});
    ctx->saved_data["activation"] = std::string(activation);
    ctx->saved_data["eps"] = eps;
    ctx->set_materialize_grads(false);
    at::AutoDispatchBelowADInplaceOrView guard;
    auto out = op.call(x, y, w_pre, w_post, gate, scale, activation, eps);
    return {std::get<0>(out), std::get<1>(out)};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_handle<NormBackwardSig>("sffft::block_norm_backward");
    refuse_second_derivative(BN, grads);
    const variable_list s = ctx->get_saved_variables();
    variable_list out(8);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    auto g = op.call(opt(grads[0]), opt(grads[1]), s[0], s[1], s[2], opt(s[3]), opt(s[4]), opt(s[5]),
                     ctx->saved_data["activation"].toStringRef(), ctx->saved_data["eps"].toDouble());
    out[0] = std::get<0>(g), out[1] = std::get<1>(g), out[2] = std::get<3>(g);
    if (s[3].defined()) out[3] = std::get<4>(g);
    if (s[4].defined()) out[4] = std::get<2>(g);
    if (s[5].defined()) out[5] = std::get<5>(g);
    return out;
  }
};

std::tuple<Tensor, Tensor> block_norm_autograd(const Tensor& x, const Tensor& y, const Tensor& w_pre,
                                               const OptTensor& w_post, const OptTensor& gate, const OptTensor& scale,
                                               c10::string_view activation, double eps) {
  refuse_tangents(BN, x, y, w_pre, w_post, gate, scale);
  if (!recorded(x, y, w_pre, w_post, gate, scale)) {
    static const auto op = op_handle<BlockNormSig>("sffft::block_norm");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, y, w_pre, w_post, gate, scale, activation, eps);
  }
  auto out = BlockNormFn::apply(x, y, w_pre, w_post, gate, scale, activation, eps);
  return {out[0], out[1]};
}

class PreNormFn : public torch::autograd::Function<PreNormFn> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, double eps) {
    static const auto op = op_handle<PreNormSig>("sffft::pre_norm");
    ctx->save_for_backward({x, w});
    ctx->saved_data["eps"] = eps;
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, w, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_handle<NormBackwardSig>("sffft::block_norm_backward");
    refuse_second_derivative("sffft::pre_norm", grads);
    const variable_list s = ctx->get_saved_variables();
    auto g = op.call(std::nullopt, grads[0], s[0], std::nullopt, s[1], std::nullopt, std::nullopt, std::nullopt, "none",
                     ctx->saved_data["eps"].toDouble());
    return {std::get<0>(g), std::get<3>(g), Tensor()};
  }
};

Tensor pre_norm_autograd(const Tensor& x, const Tensor& w, double eps) {
  refuse_tangents("sffft::pre_norm", x, w);
  if (!recorded(x, w)) {
    static const auto op = op_handle<PreNormSig>("sffft::pre_norm");
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, w, eps);
  }
  return PreNormFn::apply(x, w, eps);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(sffft, m) {
  m.def(
      "linear_attention(Tensor q, Tensor k, Tensor v, Tensor log_decay, float scale, Tensor? initial_state=None, "
      "Tensor? lengths=None) -> (Tensor, Tensor)");
  m.def(
      "linear_attention_backward(Tensor q, Tensor k, Tensor v, Tensor log_decay, float scale, Tensor? initial_state, "
      "Tensor? lengths, Tensor? grad_o, Tensor? grad_state) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor log_decay, Tensor(a!) state, float scale, "
      "Tensor? slots=None) -> Tensor");
  m.def(
      "rotary(Tensor q, Tensor k, Tensor table, Tensor? positions=None, bool interleaved=False, bool inverse=False) -> "
      "(Tensor, Tensor)");
  m.def("rotary_(Tensor(a!) q, Tensor(b!) k, Tensor table, Tensor? positions=None, bool interleaved=False) -> ()");
  m.def(
      "block_norm(Tensor x, Tensor y, Tensor w_pre, Tensor? w_post=None, Tensor? gate=None, Tensor? scale=None, "
      "str activation=\"none\", float eps=1e-6) -> (Tensor, Tensor)");
  m.def("pre_norm(Tensor x, Tensor w, float eps=1e-6) -> Tensor");
  m.def(
      "block_norm_backward(Tensor? grad_r, Tensor? grad_h, Tensor x, Tensor? y, Tensor w_pre, Tensor? w_post, "
      "Tensor? gate, Tensor? scale, str activation, float eps) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(sffft, CUDA, m) {
  m.impl("linear_attention", &attention_gpu);
  m.impl("linear_attention_backward", &attention_backward_gpu);
  m.impl("linear_attention_step", &step_gpu);
  m.impl("rotary", &rotary_gpu);
  m.impl("rotary_", &rotary_inplace_gpu);
  m.impl("block_norm", &block_norm_gpu);
  m.impl("pre_norm", &pre_norm_gpu);
  m.impl("block_norm_backward", &norm_backward_gpu);
}

TORCH_LIBRARY_IMPL(sffft, Autograd, m) {
  m.impl("linear_attention", &attention_autograd);
  m.impl("linear_attention_step", &step_autograd);
  m.impl("rotary", &rotary_autograd);
  m.impl("rotary_", &rotary_inplace_autograd);
  m.impl("block_norm", &block_norm_autograd);
  m.impl("pre_norm", &pre_norm_autograd);
}

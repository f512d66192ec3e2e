// Torch operators of the packed-sequence entry points with their outputs, workspaces and gradient (the generated ones in
// ops.cpp write into given tensors): echosparse_gfx950::packed_attention and ::shared_prefix_attention, called by packed.py,
// which checks the arguments against the documentation. (Host time of a training call with a Python autograd function 150 us,
// with this one 99; the kernels of 2300 tokens of 24 heads run about as long.)
//
// Every kernel checks what the C entry points rely on (device, dtype, layout, sizes), so a direct call cannot reach them with
// other pointers than it names.
#include "../../../include/packed_hip.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <tuple>
#include <utility>

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

void check_tokens(const char* name, const Tensor& t, const Tensor& q, int64_t dims) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name, " must be on q's GPU (got ", t.device(), ")");
  TORCH_CHECK(t.scalar_type() == q.scalar_type(), name, " must have q's dtype (got ", t.scalar_type(), ")");
  TORCH_CHECK(t.dim() == dims && t.is_contiguous(), name, " must be a contiguous ", dims, "-dimensional tensor");
}
void check_ints(const char* name, const Tensor& t, const Tensor& q, int64_t n) {
  TORCH_CHECK(t.is_cuda() && t.device() == q.device(), name, " must be on q's GPU (got ", t.device(), ")");
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && (n < 0 || t.size(0) == n), name,
              " must be a contiguous int32 tensor of its length");
}
bool half(const Tensor& q) {
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be bfloat16 or float16 (got ",
              q.scalar_type(), ")");
  return q.scalar_type() == at::kHalf;
}
int as_int(int64_t x) {
  TORCH_CHECK(x >= 0 && x <= INT32_MAX, "size ", x, " is out of range");
  return static_cast<int>(x);
}
void check_status(const char* name, int status) {
  TORCH_CHECK(status == 0, name, " failed (status ", status, "): ", es_last_error_string());
}
Tensor workspace(size_t bytes, const Tensor& q) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)) : Tensor();
}

// a tensor that starts inside another's storage at an address the kernels' 16-byte loads do not take is copied
Tensor aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) & 15 ? t.clone() : t; }

// the checked arguments of one packed call
struct Packed {
  Tensor bias, cu_q, cu_k, buckets;
  int B, Tq, Tk, H, Hk, D, num_buckets = 0, R = 0;
  bool f16;
  hipStream_t stream;

  Packed(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias_, const OptTensor& cu_q_,
         const OptTensor& cu_k_, const OptTensor& buckets_, int64_t B_)
      : cu_q(given(cu_q_)), cu_k(given(cu_k_)), buckets(given(buckets_)), B(as_int(B_)), f16(half(q)) {
    check_tokens("q", q, q, 3);
    check_tokens("k", k, q, 3);
    check_tokens("v", v, q, 3);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(2) == q.size(2), "q, k and v do not go together");
    Tq = as_int(q.size(0)), H = as_int(q.size(1)), D = as_int(q.size(2));
    Tk = as_int(k.size(0)), Hk = as_int(k.size(1));
    if (cu_q.defined()) check_ints("cu_q", cu_q, q, B_ + 1);
    if (cu_k.defined()) check_ints("cu_k", cu_k, q, B_ + 1);
    if (bias_.has_value()) {
      bias = bias_->detach().to(at::kFloat).contiguous();
      TORCH_CHECK(bias.is_cuda() && bias.device() == q.device() && bias.dim() == 2 && bias.size(1) == H,
                  "bias must be [num_buckets, heads] on q's GPU");
      TORCH_CHECK(buckets.defined(), "bias needs buckets");
      check_ints("buckets", buckets, q, -1);
      TORCH_CHECK(buckets.size(0) % 2 == 1, "buckets must hold 2 R + 1 values");
      num_buckets = as_int(bias.size(0));
      R = as_int(buckets.size(0)) / 2;
    }
    stream = c10::hip::getCurrentHIPStream(q.device().index()).stream();
  }
  const float* weights() const { return static_cast<const float*>(data(bias)); }
  const int* ints(const Tensor& t) const { return static_cast<const int*>(data(t)); }
};

std::tuple<Tensor, Tensor> packed_forward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& bias,
                                          const OptTensor& cu_q, const OptTensor& cu_k, const OptTensor& buckets, int64_t B,
                                          bool causal, double scale) {
  const c10::OptionalDeviceGuard guard(q_.device());
  const Packed a(q_, k_, v_, bias, cu_q, cu_k, buckets, B);
  const Tensor q = aligned(q_), k = aligned(k_), v = aligned(v_);
  Tensor out = at::empty_like(q), lse = at::empty({a.Tq, a.H}, q.options().dtype(at::kFloat));
  const size_t bytes = es_packed_fwd_workspace(a.B, a.Tq, a.Tk, a.H, a.Hk, a.D);
  const Tensor ws = workspace(bytes, q);
  check_status("es_packed_fwd", (a.f16 ? es_packed_fwd_f16 : es_packed_fwd)(
      data(q), data(k), data(v), a.ints(a.cu_q), a.ints(a.cu_k), a.weights(), a.ints(a.buckets), a.num_buckets, a.R, data(out),
      static_cast<float*>(data(lse)), data(ws), bytes, a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, causal, static_cast<float>(scale),
      a.stream));
  return {out, lse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> packed_backward(const Tensor& dout_, const Tensor& q_, const Tensor& k_,
                                                           const Tensor& v_, const Tensor& out, const Tensor& lse,
                                                           const OptTensor& bias, const OptTensor& cu_q,
                                                           const OptTensor& cu_k, const OptTensor& buckets, int64_t B,
                                                           bool causal, double scale) {
  const c10::OptionalDeviceGuard guard(q_.device());
  const Packed a(q_, k_, v_, bias, cu_q, cu_k, buckets, B);
  const Tensor q = aligned(q_), k = aligned(k_), v = aligned(v_), dout = aligned(dout_.contiguous());
  check_tokens("dout", dout, q, 3);
  check_tokens("out", out, q, 3);
  TORCH_CHECK(dout.sizes() == q.sizes() && out.sizes() == q.sizes(), "out and its gradient must be like q");
  TORCH_CHECK(lse.is_cuda() && lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.numel() == static_cast<int64_t>(a.Tq) * a.H,
              "lse must be the forward's");
  Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  Tensor dbias = a.bias.defined() ? at::empty_like(a.bias) : at::empty({0}, q.options().dtype(at::kFloat));
  const size_t bytes = es_packed_bwd_workspace(a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.R, a.bias.defined(), causal);
  const Tensor ws = workspace(bytes, q);
  check_status("es_packed_bwd", (a.f16 ? es_packed_bwd_f16 : es_packed_bwd)(
      data(q), data(k), data(v), data(dout), data(out), static_cast<const float*>(data(lse)), a.ints(a.cu_q), a.ints(a.cu_k),
      a.weights(), a.ints(a.buckets), a.num_buckets, a.R, data(dq), data(dk), data(dv),
      a.bias.defined() ? static_cast<float*>(data(dbias)) : nullptr, data(ws), bytes, a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, causal,
      static_cast<float>(scale), a.stream));
  if (bias.has_value()) dbias = dbias.to(bias->scalar_type());
  return {dq, dk, dv, dbias};
}

std::tuple<Tensor, Tensor> shared_forward(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& k,
                                          const Tensor& v, const Tensor& lens, double scale) {
  const c10::OptionalDeviceGuard guard(q.device());
  const bool f16 = half(q);
  check_tokens("q", q, q, 4);
  check_tokens("k_prefix", kp, q, 3);
  check_tokens("v_prefix", vp, q, 3);
  check_tokens("k", k, q, 4);
  check_tokens("v", v, q, 4);
  check_ints("lens", lens, q, q.size(0));
  const int B = as_int(q.size(0)), n = as_int(q.size(1)), H = as_int(q.size(2)), D = as_int(q.size(3));
  const int P = as_int(kp.size(0)), S = as_int(k.size(1)), Hk = as_int(k.size(2));
  TORCH_CHECK(k.sizes() == v.sizes() && kp.sizes() == vp.sizes() && k.size(0) == B && k.size(3) == D &&
                  kp.size(1) == Hk && kp.size(2) == D,
              "q, the prefix and the caches do not go together");
  Tensor out = at::empty_like(q), lse = at::empty({B, n, H}, q.options().dtype(at::kFloat));
  const size_t bytes = es_shared_prefix_workspace(B, n, P, S, H, Hk, D);
  const Tensor ws = workspace(bytes, q);
  check_status("es_shared_prefix_fwd", (f16 ? es_shared_prefix_fwd_f16 : es_shared_prefix_fwd)(
      data(q), data(kp), data(vp), data(k), data(v), static_cast<const int*>(data(lens)), data(out),
      static_cast<float*>(data(lse)), data(ws), bytes, B, n, P, S, H, Hk, D, static_cast<float>(scale),
      c10::hip::getCurrentHIPStream(q.device().index()).stream()));
  return {out, lse};
}

// ------------------------------------------------------------------------------------------------ shapes alone
std::tuple<Tensor, Tensor> packed_forward_meta(const Tensor& q, const Tensor&, const Tensor&, const OptTensor&,
                                               const OptTensor&, const OptTensor&, const OptTensor&, int64_t, bool, double) {
  return {at::empty_like(q), at::empty_symint({q.sym_size(0), q.sym_size(1)}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> packed_backward_meta(const Tensor&, const Tensor& q, const Tensor& k,
                                                                const Tensor& v, const Tensor&, const Tensor&,
                                                                const OptTensor& bias, const OptTensor&, const OptTensor&,
                                                                const OptTensor&, int64_t, bool, double) {
  return {at::empty_like(q), at::empty_like(k), at::empty_like(v),
          bias.has_value() ? at::empty_like(*bias) : at::empty({0}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor> shared_forward_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                               const Tensor&, double) {
  return {at::empty_like(q),
          at::empty_symint({q.sym_size(0), q.sym_size(1), q.sym_size(2)}, q.options().dtype(at::kFloat))};
}

// ------------------------------------------------------------------------------------------------ gradient
using BackwardSignature = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&,
                                                                     const Tensor&, const Tensor&, const Tensor&,
                                                                     const OptTensor&, const OptTensor&, const OptTensor&,
                                                                     const OptTensor&, int64_t, bool, double);
using ForwardSignature = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                                                    const OptTensor&, const OptTensor&, const OptTensor&, int64_t, bool,
                                                    double);
using SharedSignature = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                   const Tensor&, double);

OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

const c10::TypedOperatorHandle<BackwardSignature>& backward_op() {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("echosparse_gfx950::packed_attention_backward", "")
                             .typed<BackwardSignature>();
  return op;
}

// the backward is an operator of its own, whose gradient is refused rather than left out
struct PackedBackward : torch::autograd::Function<PackedBackward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& out, const Tensor& lse, const OptTensor& bias, const OptTensor& cu_q,
                               const OptTensor& cu_k, const OptTensor& buckets, int64_t B, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dq, dk, dv, dbias] = backward_op().call(dout, q, k, v, out, lse, bias, cu_q, cu_k, buckets, B, causal, scale);
    return {dq, dk, dv, dbias};
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "the backward of packed_attention is not differentiable");
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor> packed_backward_autograd(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                                    const Tensor& v, const Tensor& out, const Tensor& lse,
                                                                    const OptTensor& bias, const OptTensor& cu_q,
                                                                    const OptTensor& cu_k, const OptTensor& buckets, int64_t B,
                                                                    bool causal, double scale) {
  if (!at::GradMode::is_enabled()) {  // (a backward without create_graph: no node to make)
    at::AutoDispatchBelowADInplaceOrView below;
    return backward_op().call(dout, q, k, v, out, lse, bias, cu_q, cu_k, buckets, B, causal, scale);
  }
  auto r = PackedBackward::apply(dout, q, k, v, out, lse, bias, cu_q, cu_k, buckets, B, causal, scale);
  return {r[0], r[1], r[2], r[3]};
}

struct PackedForward : torch::autograd::Function<PackedForward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias,
                               const OptTensor& cu_q, const OptTensor& cu_k, const OptTensor& buckets, int64_t B, bool causal,
                               double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("echosparse_gfx950::packed_attention", "")
                               .typed<ForwardSignature>();
    auto [out, lse] = op.call(q, k, v, bias, cu_q, cu_k, buckets, B, causal, scale);
    ctx->save_for_backward({q, k, v, out, lse, given(bias), given(cu_q), given(cu_k), given(buckets)});
    ctx->saved_data["B"] = B;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    return {out, lse};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list res(10);
    if (!grads[0].defined()) return res;
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dv, dbias] = backward_op().call(grads[0], s[0], s[1], s[2], s[3], s[4], maybe(s[5]), maybe(s[6]),
                                                  maybe(s[7]), maybe(s[8]), ctx->saved_data["B"].toInt(),
                                                  ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    res[0] = dq;
    res[1] = dk;
    res[2] = dv;
    if (s[5].defined()) res[3] = dbias;
    return res;
  }
};
std::tuple<Tensor, Tensor> packed_forward_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias,
                                                   const OptTensor& cu_q, const OptTensor& cu_k, const OptTensor& buckets,
                                                   int64_t B, bool causal, double scale) {
  auto r = PackedForward::apply(q, k, v, bias, cu_q, cu_k, buckets, B, causal, scale);
  return {r[0], r[1]};
}

// no derivative of either mode: refused rather than left out (packed.py refuses requires_grad by itself, but a tangent is seen
// here only)
std::tuple<Tensor, Tensor> shared_forward_autograd(const Tensor& q, const Tensor& kp, const Tensor& vp, const Tensor& k,
                                                   const Tensor& v, const Tensor& lens, double scale) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("echosparse_gfx950::shared_prefix_attention", "")
                             .typed<SharedSignature>();
  const bool grad = at::GradMode::is_enabled();
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>{"q", q}, {"k_prefix", kp}, {"v_prefix", vp}, {"k", k},
                                {"v", v}}) {
    TORCH_CHECK(!t._fw_grad(0).defined(), "shared_prefix_attention has no forward-mode derivative, and ", name,
                " has a tangent");
    TORCH_CHECK(!grad || !t.requires_grad(), "shared_prefix_attention has no backward, and ", name, " requires a gradient");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, kp, vp, k, v, lens, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(echosparse_gfx950, m) {
  m.def("packed_attention(Tensor q, Tensor k, Tensor v, Tensor? bias, Tensor? cu_q, Tensor? cu_k, Tensor? buckets, int B, "
        "bool causal, float scale) -> (Tensor, Tensor)");
  m.def("packed_attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor? bias, "
        "Tensor? cu_q, Tensor? cu_k, Tensor? buckets, int B, bool causal, float scale) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("shared_prefix_attention(Tensor q, Tensor k_prefix, Tensor v_prefix, Tensor k, Tensor v, Tensor lens, float scale) "
        "-> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(echosparse_gfx950, CUDA, m) {
  m.impl("packed_attention", TORCH_FN(packed_forward));
  m.impl("packed_attention_backward", TORCH_FN(packed_backward));
  m.impl("shared_prefix_attention", TORCH_FN(shared_forward));
}
TORCH_LIBRARY_IMPL(echosparse_gfx950, Meta, m) {
  m.impl("packed_attention", TORCH_FN(packed_forward_meta));
  m.impl("packed_attention_backward", TORCH_FN(packed_backward_meta));
  m.impl("shared_prefix_attention", TORCH_FN(shared_forward_meta));
}
TORCH_LIBRARY_IMPL(echosparse_gfx950, Autograd, m) {
  m.impl("packed_attention", TORCH_FN(packed_forward_autograd));
  m.impl("packed_attention_backward", TORCH_FN(packed_backward_autograd));
  m.impl("shared_prefix_attention", TORCH_FN(shared_forward_autograd));
}

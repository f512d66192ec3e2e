// Torch operators of norms with rotation and of paged caches with their outputs, workspaces and gradient:
// echosparse_gfx950::norm_rotate, ::append_paged, ::paged_rows and ::paged_attention, called by rotary.py and paged.py, which check
// the arguments against the documentation.
//
// Every operator checks what the C entry points rely on (device, dtype, layout, sizes), so a direct call cannot reach them with
// other pointers than it names.
#include "../../../include/paged_hip.h"

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <initializer_list>
#include <tuple>
#include <utility>

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor given(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor maybe(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
const int* ints(const Tensor& t) { return static_cast<const int*>(data(t)); }

bool half_type(at::ScalarType t) {
  TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf, "tokens must be bfloat16 or float16 (got ", t, ")");
  return t == at::kHalf;
}
int as_int(int64_t x) {
  TORCH_CHECK(x >= 0 && x <= INT32_MAX, "size ", x, " is out of range");
  return static_cast<int>(x);
}
void check_status(const char* name, int status) {
  TORCH_CHECK(status == 0, name, " failed (status ", status, "): ", es_last_error_string());
}
hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool misaligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) & 15; }
Tensor aligned(const Tensor& t) { return misaligned(t) ? t.clone() : t; }

void check_on(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the tokens' GPU (got ", t.device(), ")");
}
void check_ints(const char* name, const Tensor& t, const Tensor& like, at::IntArrayRef shape) {
  check_on(name, t, like);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.sizes() == shape && t.is_contiguous(), name,
              " must be a contiguous int32 tensor of ", shape);
}

// [T, heads, D] rows of one stride: as they are, or copied where the kernels' loads do not take their layout
Tensor rows(const char* name, const Tensor& t, const Tensor& like) {
  check_on(name, t, like);
  TORCH_CHECK(t.dim() == 3 && t.scalar_type() == like.scalar_type(), name, " must be [T, heads, D] of the tokens' dtype");
  const int64_t D = t.size(2);
  const bool packed = t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == D) &&
                      (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) * D));
  return packed && !misaligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}
// the distance of its rows (a dimension of one row may have any stride, and heads of one may have any, too)
int64_t row_stride(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0); }

// the norm and rotation of a call
struct Turn {
  Tensor q_weight, k_weight, table;
  int R = 0, P = 0, f32 = 0;
  Turn(const Tensor& like, int64_t D, const OptTensor& qw, const OptTensor& kw, const OptTensor& table_) : table(given(table_)) {
    auto weight = [&](const char* name, const OptTensor& w) -> Tensor {
      if (!w.has_value()) return Tensor();
      check_on(name, *w, like);
      TORCH_CHECK(w->dim() == 1 && w->size(0) == D, name, " must be [", D, "]");
      TORCH_CHECK(w->scalar_type() == at::kFloat || w->scalar_type() == like.scalar_type(), name,
                  " must be float32 or of the tokens' dtype");
      return w->is_contiguous() && !misaligned(*w) ? *w : aligned(w->contiguous());
    };
    q_weight = weight("q_weight", qw);
    k_weight = weight("k_weight", kw);
    TORCH_CHECK(!q_weight.defined() || !k_weight.defined() || q_weight.scalar_type() == k_weight.scalar_type(),
                "q_weight and k_weight must have one dtype");
    const Tensor& w = q_weight.defined() ? q_weight : k_weight;
    f32 = w.defined() && w.scalar_type() == at::kFloat;
    if (table.defined()) {
      check_on("table", table, like);
      TORCH_CHECK(table.scalar_type() == at::kFloat && table.dim() == 3 && table.size(2) == 2 && table.is_contiguous(),
                  "table must be a contiguous float32 [positions, R / 2, 2] tensor");
      P = as_int(table.size(0));
      R = as_int(2 * table.size(1));
      TORCH_CHECK(R > 0 && R % 16 == 0 && R <= D && P > 0, "table must hold angles of R channels, a multiple of 16 up to ", D);
      table = aligned(table);
    }
  }
  const float* angles() const { return static_cast<const float*>(data(table)); }
};

// ------------------------------------------------------------------------------------------------ norm and rotation
struct Rotation {
  Tensor q, k, positions;
  Turn turn;
  int T, H, Hk, D;
  bool f16;
  Rotation(const Tensor& q_, const Tensor& k_, const OptTensor& qw, const OptTensor& kw, const OptTensor& table,
           const OptTensor& positions_, int64_t L)
      : q(rows("q", q_, q_)), k(rows("k", k_, q_)), positions(given(positions_)), turn(q_, q_.size(2), qw, kw, table),
        f16(half_type(q_.scalar_type())) {
    TORCH_CHECK(k.size(0) == q.size(0) && k.size(2) == q.size(2), "q and k do not go together");
    T = as_int(q.size(0)), H = as_int(q.size(1)), D = as_int(q.size(2)), Hk = as_int(k.size(1));
    TORCH_CHECK(H > 0 && Hk > 0, "q and k must have heads");
    TORCH_CHECK(turn.q_weight.defined() == turn.k_weight.defined(), "q_weight and k_weight go together");
    TORCH_CHECK(turn.q_weight.defined() || turn.table.defined(), "norm_rotate needs weights, a table or both");
    if (positions.defined()) {
      TORCH_CHECK(turn.table.defined(), "positions go with a table");
      check_ints("positions", positions, q, {q.size(0)});
    } else {
      TORCH_CHECK(!turn.table.defined() || turn.P >= L, "the table has ", turn.P, " positions for ", L, " rows");
    }
  }
};

std::tuple<Tensor, Tensor> rotate_forward(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                          const OptTensor& table, const OptTensor& positions, int64_t L, bool halves, double eps) {
  const c10::OptionalDeviceGuard guard(q.device());
  const Rotation a(q, k, qw, kw, table, positions, L);
  Tensor qo = at::empty(a.q.sizes(), q.options()), ko = at::empty(a.k.sizes(), q.options());
  check_status("es_norm_rotate", (a.f16 ? es_norm_rotate_f16 : es_norm_rotate)(
      data(a.q), data(a.k), data(a.turn.q_weight), data(a.turn.k_weight), a.turn.angles(), ints(a.positions), data(qo), data(ko),
      a.T, as_int(L), a.H, a.Hk, a.D, a.turn.R, a.turn.P, halves, a.turn.f32, eps, row_stride(a.q), row_stride(a.k),
      stream_of(q)));
  return {qo, ko};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> rotate_backward(const Tensor& dqo_, const Tensor& dko_, const Tensor& q,
                                                           const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                                           const OptTensor& table, const OptTensor& positions, int64_t L,
                                                           bool halves, double eps) {
  const c10::OptionalDeviceGuard guard(q.device());
  const Rotation a(q, k, qw, kw, table, positions, L);
  auto gradient = [&](const char* name, const Tensor& d, const Tensor& x) {
    check_on(name, d, x);
    TORCH_CHECK(d.scalar_type() == x.scalar_type() && d.sizes() == x.sizes(), name, " must be like its output");
    return d.is_contiguous() && !misaligned(d) ? d : aligned(d.contiguous());
  };
  const Tensor dqo = gradient("the gradient of q", dqo_, a.q), dko = gradient("the gradient of k", dko_, a.k);
  Tensor dq = at::empty(a.q.sizes(), q.options()), dk = at::empty(a.k.sizes(), q.options());
  auto like = [&](const Tensor& w) { return at::empty({w.defined() ? a.D : 0}, (w.defined() ? w : q).options()); };
  Tensor dqw = like(a.turn.q_weight), dkw = like(a.turn.k_weight);
  const bool norm = a.turn.q_weight.defined();
  const size_t bytes = norm ? es_norm_rotate_workspace(a.T, a.H, a.Hk, a.D) : 0;
  const Tensor ws = bytes ? at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)) : Tensor();
  check_status("es_norm_rotate_bwd", (a.f16 ? es_norm_rotate_bwd_f16 : es_norm_rotate_bwd)(
      data(a.q), data(a.k), data(dqo), data(dko), data(a.turn.q_weight), data(a.turn.k_weight), a.turn.angles(),
      ints(a.positions), data(dq), data(dk), norm ? data(dqw) : nullptr, norm ? data(dkw) : nullptr, data(ws), bytes, a.T,
      as_int(L), a.H, a.Hk, a.D, a.turn.R, a.turn.P, halves, a.turn.f32, eps, row_stride(a.q), row_stride(a.k), stream_of(q)));
  return {dq, dk, dqw, dkw};
}

// ------------------------------------------------------------------------------------------------ caches
// the checked cache and places of a call
struct Cache {
  const Tensor &k, &v;
  Tensor ks, vs, cu;
  const Tensor &pages, &lens;
  int B, T, max_pages, num_pages, page_size, Hk, D;
  bool four;
  Cache(const Tensor& k_, const Tensor& v_, const OptTensor& ks_, const OptTensor& vs_, const Tensor& pages_, const Tensor& lens_,
        const OptTensor& cu_, at::ScalarType dtype, int64_t rows)
      : k(k_), v(v_), ks(given(ks_)), vs(given(vs_)), cu(given(cu_)), pages(pages_), lens(lens_) {
    TORCH_CHECK(k.is_cuda(), "the cache must be on the GPU (got ", k.device(), ")");
    check_on("v of the cache", v, k);
    TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes(), "k and v of the cache must have one shape [pages, heads, page size, D]");
    TORCH_CHECK(ks.defined() == vs.defined(), "a cache has both scales or none");
    four = ks.defined();
    num_pages = as_int(k.size(0)), Hk = as_int(k.size(1)), page_size = as_int(k.size(2));
    D = as_int(k.size(3)) * (four ? 2 : 1);
    if (four) {
      TORCH_CHECK(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte && k.is_contiguous() && v.is_contiguous(),
                  "codes of a cache must be contiguous uint8 tensors");
      for (const Tensor& s : {ks, vs}) {
        check_on("scales of the cache", s, k);
        TORCH_CHECK(s.scalar_type() == at::kByte && s.is_contiguous() && s.dim() == 4 && s.size(0) == num_pages &&
                        s.size(1) == Hk && s.size(2) == page_size && s.size(3) == D / 32,
                    "scales of a cache must be contiguous uint8 [pages, heads, page size, D / 32] tensors");
      }
    } else {
      TORCH_CHECK(k.scalar_type() == dtype && v.scalar_type() == dtype, "a cache of 16 bits must have the tokens' dtype (got ",
                  k.scalar_type(), " and ", v.scalar_type(), ")");
      TORCH_CHECK(k.strides() == v.strides() && k.stride(3) == 1,
                  "k and v of a cache must have the same strides, channels 1 apart");
      // each dimension steps over all that those of smaller strides hold (a dimension of one may have any stride)
      int order[3] = {2, 1, 0};
      std::sort(order, order + 3, [&](int i, int j) { return k.stride(i) < k.stride(j); });
      int64_t span = D;
      for (int i : order) {
        if (k.size(i) <= 1) continue;
        TORCH_CHECK(k.stride(i) >= span && k.stride(i) % 8 == 0, "rows of a cache must not overlap, their strides be multiples of 8");
        span += (k.size(i) - 1) * k.stride(i);
      }
    }
    for (const Tensor* t : {&k, &v, (const Tensor*)&ks, (const Tensor*)&vs})
      TORCH_CHECK(!t->defined() || t->numel() == 0 || !misaligned(*t), "the cache must be aligned to 16 bytes");
    TORCH_CHECK(pages.dim() == 2, "pages must be [sequences, pages]");
    B = as_int(pages.size(0)), max_pages = as_int(pages.size(1));
    check_ints("pages", pages, k, {B, max_pages});
    check_ints("lens", lens, k, {B});
    if (cu.defined()) check_ints("cu", cu, k, {B + 1});
    T = as_int(rows);
  }
  // (a dimension of one page, head or row may have any stride, which no address uses)
  long long page_stride() const { return num_pages <= 1 ? 0 : k.stride(0); }
  long long head_stride() const { return Hk <= 1 ? 0 : k.stride(1); }
  long long row_stride() const { return page_size <= 1 ? D : k.stride(2); }
  static uint8_t* bytes(const Tensor& t) { return static_cast<uint8_t*>(data(t)); }
};

Tensor append_forward(const OptTensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& qw, const OptTensor& kw,
                      const OptTensor& table, const Tensor& pages, const Tensor& lens, const OptTensor& cu, const Tensor& kp,
                      const Tensor& vp, const OptTensor& ks, const OptTensor& vs, bool halves, double eps) {
  const c10::OptionalDeviceGuard guard(k_.device());
  const bool f16 = half_type(k_.scalar_type());
  const Cache c(kp, vp, ks, vs, pages, lens, cu, k_.scalar_type(), k_.size(0));
  check_on("the cache", kp, k_);
  const Tensor q = q_.has_value() ? rows("q", *q_, k_) : Tensor(), k = rows("k", k_, k_), v = rows("v", v_, k_);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(1) == c.Hk && k.size(2) == c.D &&
                  (!q.defined() || (q.size(0) == k.size(0) && q.size(2) == c.D)),
              "q, k, v and the cache do not go together");
  TORCH_CHECK(q.defined() ? q.size(1) > 0 && qw.has_value() == kw.has_value() : !qw.has_value(),
              "q_weight goes with q and k_weight, q has heads");
  const Turn turn(k_, c.D, qw, kw, table);
  const int H = q.defined() ? as_int(q.size(1)) : 0;
  Tensor out = q.defined() ? at::empty(q.sizes(), q.options()) : at::empty({0}, k.options());
  void* qo = q.defined() ? data(out) : nullptr;
  const long long qs = q.defined() ? row_stride(q) : 0;
  if (c.four)
    check_status("es_append_paged4", (f16 ? es_append_paged4_f16 : es_append_paged4)(
        data(q), data(k), data(v), data(turn.q_weight), data(turn.k_weight), turn.angles(), ints(pages), ints(lens), ints(c.cu), qo,
        c.bytes(kp), c.bytes(c.ks), c.bytes(vp), c.bytes(c.vs), c.B, c.T, c.max_pages, c.num_pages, c.page_size, H, c.Hk, c.D,
        turn.R, turn.P, halves, turn.f32, eps, qs, row_stride(k), row_stride(v), stream_of(k)));
  else
    check_status("es_append_paged", (f16 ? es_append_paged_f16 : es_append_paged)(
        data(q), data(k), data(v), data(turn.q_weight), data(turn.k_weight), turn.angles(), ints(pages), ints(lens), ints(c.cu), qo,
        data(kp), data(vp), c.B, c.T, c.max_pages, c.num_pages, c.page_size, H, c.Hk, c.D, turn.R, turn.P, halves, turn.f32, eps,
        qs, row_stride(k), row_stride(v), c.page_stride(), c.head_stride(), c.row_stride(), stream_of(k)));
  return out;
}

std::tuple<Tensor, Tensor> rows_forward(const Tensor& kp, const Tensor& vp, const OptTensor& ks, const OptTensor& vs,
                                        const Tensor& pages, const Tensor& lens, const OptTensor& cu, int64_t count,
                                        at::ScalarType dtype) {
  const c10::OptionalDeviceGuard guard(kp.device());
  const bool f16 = half_type(dtype);
  const Cache c(kp, vp, ks, vs, pages, lens, cu, dtype, count);
  Tensor k = at::empty({count, c.Hk, c.D}, kp.options().dtype(dtype)), v = at::empty_like(k);
  if (c.four)
    check_status("es_paged_rows4", (f16 ? es_paged_rows4_f16 : es_paged_rows4)(
        c.bytes(kp), c.bytes(c.ks), c.bytes(vp), c.bytes(c.vs), ints(pages), ints(lens), ints(c.cu), data(k), data(v), c.B, c.T,
        c.max_pages, c.num_pages, c.page_size, c.Hk, c.D, stream_of(kp)));
  else
    check_status("es_paged_rows", (f16 ? es_paged_rows_f16 : es_paged_rows)(
        data(kp), data(vp), ints(pages), ints(lens), ints(c.cu), data(k), data(v), c.B, c.T, c.max_pages, c.num_pages, c.page_size,
        c.Hk, c.D, c.page_stride(), c.head_stride(), c.row_stride(), stream_of(kp)));
  return {k, v};
}

std::tuple<Tensor, Tensor> attention_forward(const Tensor& q_, const Tensor& kp, const Tensor& vp, const OptTensor& ks,
                                             const OptTensor& vs, const Tensor& pages, const Tensor& lens, const OptTensor& cu,
                                             bool causal, double scale) {
  const c10::OptionalDeviceGuard guard(q_.device());
  const bool f16 = half_type(q_.scalar_type());
  check_on("q", q_, q_);
  TORCH_CHECK(q_.dim() == 3 && q_.is_contiguous(), "q must be a contiguous [T, heads, D] tensor");
  const Cache c(kp, vp, ks, vs, pages, lens, cu, q_.scalar_type(), q_.size(0));
  check_on("the cache", kp, q_);
  TORCH_CHECK(q_.size(2) == c.D, "q and the cache do not go together");
  const Tensor q = q_.numel() ? aligned(q_) : q_;
  const int H = as_int(q.size(1));
  Tensor out = at::empty(q.sizes(), q.options()), lse = at::empty({c.T, H}, q.options().dtype(at::kFloat));
  const size_t bytes = es_paged_workspace(c.B, c.T, c.max_pages, c.page_size, H, c.Hk, c.D, c.four ? 4 : 16);
  const Tensor ws = bytes ? at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)) : Tensor();
  float* l = static_cast<float*>(data(lse));
  if (c.four)
    check_status("es_paged4_fwd", (f16 ? es_paged4_fwd_f16 : es_paged4_fwd)(
        data(q), c.bytes(kp), c.bytes(c.ks), c.bytes(vp), c.bytes(c.vs), ints(pages), ints(lens), ints(c.cu), data(out), l,
        data(ws), bytes, c.B, c.T, c.max_pages, c.num_pages, c.page_size, H, c.Hk, c.D, causal, static_cast<float>(scale), stream_of(q)));
  else
    check_status("es_paged_fwd", (f16 ? es_paged_fwd_f16 : es_paged_fwd)(
        data(q), data(kp), data(vp), ints(pages), ints(lens), ints(c.cu), data(out), l, data(ws), bytes, c.B, c.T, c.max_pages,
        c.num_pages, c.page_size, H, c.Hk, c.D, causal, static_cast<float>(scale), c.page_stride(), c.head_stride(), c.row_stride(),
        stream_of(q)));
  return {out, lse};
}

// ------------------------------------------------------------------------------------------------ shapes alone
std::tuple<Tensor, Tensor> attention_meta(const Tensor& q, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                          const Tensor&, const Tensor&, const OptTensor&, bool, double) {
  return {at::empty_like(q), at::empty_symint({q.sym_size(0), q.sym_size(1)}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor> rotate_meta(const Tensor& q, const Tensor& k, const OptTensor&, const OptTensor&, const OptTensor&,
                                       const OptTensor&, c10::SymInt, bool, double) {
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options())};
}
std::tuple<Tensor, Tensor, Tensor, Tensor> rotate_backward_meta(const Tensor&, const Tensor&, const Tensor& q, const Tensor& k,
                                                                const OptTensor& qw, const OptTensor& kw, const OptTensor&,
                                                                const OptTensor&, c10::SymInt, bool, double) {
  auto like = [&](const OptTensor& w) { return w.has_value() ? at::empty_like(*w) : at::empty({0}, q.options()); };
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options()), like(qw), like(kw)};
}
Tensor append_meta(const OptTensor& q, const Tensor& k, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                   const Tensor&, const Tensor&, const OptTensor&, const Tensor&, const Tensor&, const OptTensor&,
                   const OptTensor&, bool, double) {
  return q.has_value() ? at::empty_symint(q->sym_sizes(), q->options()) : at::empty({0}, k.options());
}
std::tuple<Tensor, Tensor> rows_meta(const Tensor& kp, const Tensor&, const OptTensor& ks, const OptTensor&, const Tensor&,
                                     const Tensor&, const OptTensor&, c10::SymInt count, at::ScalarType dtype) {
  Tensor k = at::empty_symint({std::move(count), kp.sym_size(1), kp.sym_size(3) * (ks.has_value() ? 2 : 1)}, kp.options().dtype(dtype));
  return {k, at::empty_like(k)};
}

// ------------------------------------------------------------------------------------------------ gradient
using RotateSignature = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                   const OptTensor&, const OptTensor&, c10::SymInt, bool, double);
using RotateBackwardSignature = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&,
                                                                           const Tensor&, const OptTensor&, const OptTensor&,
                                                                           const OptTensor&, const OptTensor&, c10::SymInt, bool,
                                                                           double);

template <class Signature>
c10::TypedOperatorHandle<Signature> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
const c10::TypedOperatorHandle<RotateBackwardSignature>& rotate_backward_op() {
  static const auto op = find<RotateBackwardSignature>("echosparse_gfx950::norm_rotate_backward");
  return op;
}

// the backward is an operator of its own, whose gradient is refused rather than left out
struct RotateBackward : torch::autograd::Function<RotateBackward> {
  static variable_list forward(AutogradContext*, const Tensor& dqo, const Tensor& dko, const Tensor& q, const Tensor& k,
                               const OptTensor& qw, const OptTensor& kw, const OptTensor& table, const OptTensor& positions,
                               c10::SymInt L, bool halves, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [dq, dk, dqw, dkw] = rotate_backward_op().call(dqo, dko, q, k, qw, kw, table, positions, L, halves, eps);
    return {dq, dk, dqw, dkw};
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "the backward of norm_rotate is not differentiable");
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor> rotate_backward_autograd(const Tensor& dqo, const Tensor& dko, const Tensor& q,
                                                                    const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                                                    const OptTensor& table, const OptTensor& positions,
                                                                    c10::SymInt L, bool halves, double eps) {
  if (!at::GradMode::is_enabled()) {  // (a backward without create_graph: no node to make)
    at::AutoDispatchBelowADInplaceOrView below;
    return rotate_backward_op().call(dqo, dko, q, k, qw, kw, table, positions, L, halves, eps);
  }
  auto r = RotateBackward::apply(dqo, dko, q, k, qw, kw, table, positions, L, halves, eps);
  return {r[0], r[1], r[2], r[3]};
}

struct RotateForward : torch::autograd::Function<RotateForward> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                               const OptTensor& table, const OptTensor& positions, c10::SymInt L, bool halves, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = find<RotateSignature>("echosparse_gfx950::norm_rotate");
    auto [qo, ko] = op.call(q, k, qw, kw, table, positions, L, halves, eps);
    ctx->save_for_backward({q, k, given(qw), given(kw), given(table), given(positions)});
    ctx->saved_data["L"] = L;
    ctx->saved_data["halves"] = halves;
    ctx->saved_data["eps"] = eps;
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    variable_list res(9);
    const auto s = ctx->get_saved_variables();
    auto [dq, dk, dqw, dkw] = rotate_backward_op().call(grads[0], grads[1], s[0], s[1], maybe(s[2]), maybe(s[3]), maybe(s[4]),
                                                        maybe(s[5]), ctx->saved_data["L"].toSymInt(),
                                                        ctx->saved_data["halves"].toBool(), ctx->saved_data["eps"].toDouble());
    res[0] = dq;
    res[1] = dk;
    if (s[2].defined()) res[2] = dqw;
    if (s[3].defined()) res[3] = dkw;
    return res;
  }
};
// A captured backward hands each gradient to the stream on which its input's node was made. Where that is another one, as for a
// leaf that an eager graph still holds, the capture cannot be ended any more: refused at the forward call.
void refuse_other_streams(std::initializer_list<Tensor> inputs, const Tensor& like) {
  const auto stream = c10::hip::getCurrentHIPStream(like.device().index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess) {  // (asked of the default stream beside a capture)
    (void)hipGetLastError();
    return;
  }
  if (status != hipStreamCaptureStatusActive) return;
  for (const Tensor& t : inputs) {
    if (!t.defined() || !t.requires_grad()) continue;
    const auto node = t.grad_fn() ? t.grad_fn() : torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    const auto made_on = node->stream();
    TORCH_CHECK(!made_on.has_value() || *made_on == stream.unwrap(), "norm_rotate cannot be captured with inputs whose gradients "
                "belong to another stream: take leaves made inside the capture, or free the graphs made before it");
  }
}

std::tuple<Tensor, Tensor> rotate_autograd(const Tensor& q, const Tensor& k, const OptTensor& qw, const OptTensor& kw,
                                           const OptTensor& table, const OptTensor& positions, c10::SymInt L, bool halves,
                                           double eps) {
  const bool grad = at::GradMode::is_enabled();
  auto wants = [](const OptTensor& t) { return t.has_value() && t->requires_grad(); };
  TORCH_CHECK(!grad || !wants(table), "norm_rotate has no gradient of its table");
  auto tangent = [](const OptTensor& t) { return t.has_value() && t->_fw_grad(0).defined(); };
  TORCH_CHECK(!tangent(q) && !tangent(k) && !tangent(qw) && !tangent(kw) && !tangent(table),
              "norm_rotate has no forward-mode derivative");
  if (!grad || !(q.requires_grad() || k.requires_grad() || wants(qw) || wants(kw))) {  // (nothing to keep: a third of a short call)
    static const auto op = find<RotateSignature>("echosparse_gfx950::norm_rotate");
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(q, k, qw, kw, table, positions, L, halves, eps);
  }
  if (q.is_cuda()) refuse_other_streams({q, k, given(qw), given(kw)}, q);
  auto r = RotateForward::apply(q, k, qw, kw, table, positions, L, halves, eps);
  return {r[0], r[1]};
}

// no derivative of either mode: refused rather than left out
void refuse_derivatives(const char* op, std::initializer_list<std::pair<const char*, const Tensor>> named) {
  const bool grad = at::GradMode::is_enabled();
  for (const auto& [name, t] : named) {
    if (!t.defined()) continue;
    TORCH_CHECK(!t._fw_grad(0).defined(), op, " has no forward-mode derivative, and ", name, " has a tangent");
    TORCH_CHECK(!grad || !t.requires_grad(), op, " has no backward, and ", name, " requires a gradient");
  }
}

using AppendSignature = Tensor(const OptTensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                               const Tensor&, const Tensor&, const OptTensor&, const Tensor&, const Tensor&, const OptTensor&,
                               const OptTensor&, bool, double);
Tensor append_autograd(const OptTensor& q, const Tensor& k, const Tensor& v, const OptTensor& qw, const OptTensor& kw,
                       const OptTensor& table, const Tensor& pages, const Tensor& lens, const OptTensor& cu, const Tensor& kp,
                       const Tensor& vp, const OptTensor& ks, const OptTensor& vs, bool halves, double eps) {
  static const auto op = find<AppendSignature>("echosparse_gfx950::append_paged");
  refuse_derivatives("append_paged", {{"q", given(q)}, {"k", k}, {"v", v}, {"q_weight", given(qw)}, {"k_weight", given(kw)},
                                      {"table", given(table)}, {"cache.k", kp}, {"cache.v", vp}});
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor out = op.call(q, k, v, qw, kw, table, pages, lens, cu, kp, vp, ks, vs, halves, eps);
  for (const Tensor& t : {kp, vp, given(ks), given(vs)})      // (a graph that saved the cache sees that it changed)
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return out;
}

using RowsSignature = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&,
                                                 const Tensor&, const OptTensor&, c10::SymInt, at::ScalarType);
std::tuple<Tensor, Tensor> rows_autograd(const Tensor& kp, const Tensor& vp, const OptTensor& ks, const OptTensor& vs,
                                         const Tensor& pages, const Tensor& lens, const OptTensor& cu, c10::SymInt count,
                                         at::ScalarType dtype) {
  static const auto op = find<RowsSignature>("echosparse_gfx950::paged_rows");
  refuse_derivatives("paged_rows", {{"cache.k", kp}, {"cache.v", vp}});
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(kp, vp, ks, vs, pages, lens, cu, count, dtype);
}

using AttentionSignature = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&,
                                                      const OptTensor&, const Tensor&, const Tensor&, const OptTensor&, bool,
                                                      double);
std::tuple<Tensor, Tensor> attention_autograd(const Tensor& q, const Tensor& kp, const Tensor& vp, const OptTensor& ks,
                                              const OptTensor& vs, const Tensor& pages, const Tensor& lens, const OptTensor& cu,
                                              bool causal, double scale) {
  static const auto op = find<AttentionSignature>("echosparse_gfx950::paged_attention");
  refuse_derivatives("paged_attention", {{"q", q}, {"cache.k", kp}, {"cache.v", vp}});
  at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, kp, vp, ks, vs, pages, lens, cu, causal, scale);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(echosparse_gfx950, m) {
  m.def("norm_rotate(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? table, Tensor? positions, SymInt L, "
        "bool halves, float eps) -> (Tensor, Tensor)");
  m.def("norm_rotate_backward(Tensor dq_out, Tensor dk_out, Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, "
        "Tensor? table, Tensor? positions, SymInt L, bool halves, float eps) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("append_paged(Tensor? q, Tensor k, Tensor v, Tensor? q_weight, Tensor? k_weight, Tensor? table, Tensor pages, "
        "Tensor lens, Tensor? cu, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!)? k_scales, Tensor(d!)? v_scales, "
        "bool halves, float eps) -> Tensor");
  m.def("paged_rows(Tensor k_pages, Tensor v_pages, Tensor? k_scales, Tensor? v_scales, Tensor pages, Tensor lens, Tensor? cu, "
        "SymInt rows, ScalarType dtype) -> (Tensor, Tensor)");
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor? k_scales, Tensor? v_scales, Tensor pages, "
        "Tensor lens, Tensor? cu, bool causal, float scale) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(echosparse_gfx950, CUDA, m) {
  m.impl("norm_rotate", TORCH_FN(rotate_forward));
  m.impl("norm_rotate_backward", TORCH_FN(rotate_backward));
  m.impl("append_paged", TORCH_FN(append_forward));
  m.impl("paged_rows", TORCH_FN(rows_forward));
  m.impl("paged_attention", TORCH_FN(attention_forward));
}
TORCH_LIBRARY_IMPL(echosparse_gfx950, Meta, m) {
  m.impl("norm_rotate", TORCH_FN(rotate_meta));
  m.impl("norm_rotate_backward", TORCH_FN(rotate_backward_meta));
  m.impl("append_paged", TORCH_FN(append_meta));
  m.impl("paged_rows", TORCH_FN(rows_meta));
  m.impl("paged_attention", TORCH_FN(attention_meta));
}
TORCH_LIBRARY_IMPL(echosparse_gfx950, Autograd, m) {
  m.impl("norm_rotate", TORCH_FN(rotate_autograd));
  m.impl("norm_rotate_backward", TORCH_FN(rotate_backward_autograd));
  m.impl("append_paged", TORCH_FN(append_autograd));
  m.impl("paged_rows", TORCH_FN(rows_autograd));
  m.impl("paged_attention", TORCH_FN(attention_autograd));
}

// Native host side of norms and rotation (module kv_attention._native): the dispatcher entries of alexdremov_qk_norm_rope::{forward, backward}
// and alexdremov_paged_attention::append_rope, the autograd of the first, and the eager call path of the public Python functions.
#include "kv_torch.h"

using namespace kv_native;

namespace {

using OptDouble = std::optional<double>;

// ---- argument checks and layout -------------------------------------------------------------------------------
bool is_weight(const OptTensor& w, const Tensor& q) {
  return !w || (w->dim() == 1 && w->size(0) == q.size(3) && w->device() == q.device() &&
                (w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat));
}
bool is_rotation(const Tensor& q, const Tensor& cos, const Tensor& sin, const OptTensor& q_weight, const OptTensor& k_weight,
                 const OptTensor& positions, OptDouble eps) {
  for (const Tensor* t : {&cos, &sin})
    if (t->dim() != 2 || t->scalar_type() != at::kFloat || t->device() != q.device()) return false;
  if (cos.sizes() != sin.sizes() || cos.size(1) < 8 || cos.size(1) % 8 != 0 || 2 * cos.size(1) > q.size(3) || !small(cos.size(0))) return false;
  if (!is_weight(q_weight, q) || !is_weight(k_weight, q)) return false;
  if (q_weight && k_weight && q_weight->scalar_type() != k_weight->scalar_type()) return false;
  if (positions && (positions->dim() != 2 || positions->scalar_type() != at::kInt || positions->size(0) != q.size(0) ||
                    positions->size(1) != q.size(2) || positions->device() != q.device()))
    return false;
  if (!eps) return !q_weight && !k_weight;
  return (float)*eps > 0.0f && *eps < 3.4e38;
}
// Rows that the kernels can read in place, or a copy.
Tensor table_layout(const Tensor& t) {
  const bool ok = t.stride(1) == 1 && (t.size(0) <= 1 || (t.stride(0) >= 0 && t.stride(0) % 4 == 0)) &&
                  reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
Tensor rows_layout(const Tensor& t) { return kernel_layout(t, false); }   // rows of a long projection may lie any distance apart
OptTensor weight_layout(const OptTensor& w) {
  if (!w || ((w->stride(0) == 1) && reinterpret_cast<uintptr_t>(w->const_data_ptr()) % 16 == 0)) return w;
  return w->clone(at::MemoryFormat::Contiguous);
}
const void* opt_ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : 0; }
bool weights_f32(const OptTensor& q_weight, const OptTensor& k_weight) {
  return (q_weight && q_weight->scalar_type() == at::kFloat) || (k_weight && k_weight->scalar_type() == at::kFloat);
}
struct Positions {
  const int32_t* p = nullptr;
  int64_t s[2] = {0, 0};
  explicit Positions(const OptTensor& t) {
    if (t) p = t->const_data_ptr<int32_t>(), s[0] = t->stride(0), s[1] = t->stride(1);
  }
};
float c_eps(OptDouble eps) { return eps ? (float)*eps : 0.0f; }

// ---- queries and keys --------------------------------------------------------------------------------------------
bool is_pair(const Tensor& q, const Tensor& k, const OptTensor& lens) {
  if (q.dim() != 4 || k.dim() != 4 || dtype_id(q) < 0 || !known_head_dim(q.size(3)) || !alike(q, k)) return false;
  if (k.size(0) != q.size(0) || k.size(2) != q.size(2) || k.size(3) != q.size(3) || q.size(1) < 1 || k.size(1) < 1) return false;
  return small_sizes(q) && small_sizes(k) && is_lengths(lens, q);
}
void validate_rope(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const OptTensor& q_weight, const OptTensor& k_weight,
                   const OptTensor& lens, const OptTensor& positions, OptDouble eps, std::initializer_list<const Tensor*> grads = {}) {
  bool ok = is_pair(q, k, lens) && is_rotation(q, cos, sin, q_weight, k_weight, positions, eps);
  const Tensor* x[2] = {&q, &k};
  int i = 0;
  for (const Tensor* t : grads) ok = ok && t->sizes() == x[i]->sizes() && t->device() == q.device(), ++i;
  if (C10_LIKELY(ok)) return;
  Gil gil;
  PyObject *q_ = THPVariable_Wrap(q), *k_ = THPVariable_Wrap(k), *c_ = THPVariable_Wrap(cos), *s_ = THPVariable_Wrap(sin);
  if (grads.size() == 2)
    explain("_validate_rope", {q_, k_, c_, s_, wrap(q_weight), wrap(k_weight), wrap(lens), wrap(positions), wrap(eps),
                               THPVariable_Wrap(**grads.begin()), THPVariable_Wrap(**(grads.begin() + 1))});
  explain("_validate_rope", {q_, k_, c_, s_, wrap(q_weight), wrap(k_weight), wrap(lens), wrap(positions), wrap(eps)});
}

std::tuple<Tensor, Tensor> rope_forward_gpu(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const OptTensor& q_weight,
                                            const OptTensor& k_weight, const OptTensor& lens, const OptTensor& positions, OptDouble eps,
                                            bool interleaved) {
  validate_rope(q, k, cos, sin, q_weight, k_weight, lens, positions, eps);
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor q_out = empty_same(q), k_out = empty_same(k);
  if (q.numel() == 0) return {std::move(q_out), std::move(k_out)};
  const Tensor qk = rows_layout(q), kk = rows_layout(k), ct = table_layout(cos), st = table_layout(sin);
  const OptTensor wq = weight_layout(q_weight), wk = weight_layout(k_weight);
  const Lengths l(lens);
  const Positions pos(positions);
  check_launch(api().qk_norm_rope(ptr(qk), ptr(kk), (const float*)ptr(ct), (const float*)ptr(st), row_stride(ct), row_stride(st), opt_ptr(wq),
                                  opt_ptr(wk), weights_f32(wq, wk), l.p, l.stride, pos.p, pos.s, out_ptr(q_out), out_ptr(k_out), Strides(qk),
                                  Strides(kk), (int)q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), (int)q.size(3),
                                  (int)(2 * cos.size(1)), (int)cos.size(0), interleaved, c_eps(eps), dtype_id(q), current_stream(q)),
               "kv_qk_norm_rope");
  return {std::move(q_out), std::move(k_out)};
}

// Gradients of q and k and, where `weights` says so, of the weights that there are (else empty tensors).
std::tuple<Tensor, Tensor, Tensor, Tensor> rope_backward_gpu(const Tensor& d_q, const Tensor& d_k, const Tensor& q, const Tensor& k,
                                                             const Tensor& cos, const Tensor& sin, const OptTensor& q_weight,
                                                             const OptTensor& k_weight, const OptTensor& lens, const OptTensor& positions,
                                                             OptDouble eps, bool interleaved, bool weights) {
  validate_rope(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, {&d_q, &d_k});
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor dq = empty_same(q), dk = empty_same(k);
  auto like = [&](const OptTensor& w) { return w && weights ? at::empty({w->size(0)}, w->options()) : at::empty({0}, q.options()); };
  Tensor dwq = like(q_weight), dwk = like(k_weight);
  weights = weights && (q_weight || k_weight);
  if (q.numel() == 0) {
    dwq.zero_(), dwk.zero_();
    return {std::move(dq), std::move(dk), std::move(dwq), std::move(dwk)};
  }
  const Api& a = api();
  const Tensor qk = rows_layout(q), kk = rows_layout(k), ct = table_layout(cos), st = table_layout(sin);
  // the upstream gradient may arrive in another type and with arbitrary strides
  const Tensor gq = rows_layout(d_q.to(q.scalar_type())), gk = rows_layout(d_k.to(q.scalar_type()));
  const OptTensor wq = weight_layout(q_weight), wk = weight_layout(k_weight);
  const int B = (int)q.size(0), Hq = (int)q.size(1), Hkv = (int)k.size(1), T = (int)q.size(2), D = (int)q.size(3);
  const int64_t bytes = weights ? a.qk_norm_rope_backward_workspace(B, Hq, Hkv, T, D, dtype_id(q)) : 0;
  check(bytes, "kv_qk_norm_rope_backward");
  const Tensor ws = bytes > 0 ? workspace(q, bytes) : Tensor();
  const Lengths l(lens);
  const Positions pos(positions);
  check_launch(a.qk_norm_rope_backward(ptr(qk), ptr(kk), ptr(gq), ptr(gk), (const float*)ptr(ct), (const float*)ptr(st), row_stride(ct),
                                       row_stride(st), opt_ptr(wq), opt_ptr(wk), weights_f32(wq, wk), l.p, l.stride, pos.p, pos.s, out_ptr(dq),
                                       out_ptr(dk), weights && wq ? out_ptr(dwq) : nullptr, weights && wk ? out_ptr(dwk) : nullptr,
                                       bytes > 0 ? out_ptr(ws) : nullptr, bytes, Strides(qk), Strides(kk), Strides(gq), Strides(gk), B, Hq, Hkv,
                                       T, D, (int)(2 * cos.size(1)), (int)cos.size(0), interleaved, c_eps(eps), dtype_id(q), current_stream(q)),
               "kv_qk_norm_rope_backward");
  return {std::move(dq), std::move(dk), std::move(dwq), std::move(dwk)};
}

using RopeForward = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                               const OptTensor&, const OptTensor&, OptDouble, bool);
using RopeBackward = std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                                const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                                                                const OptTensor&, OptDouble, bool, bool);
const c10::TypedOperatorHandle<RopeForward>& rope_forward_op() {
  static const auto op = find_op<RopeForward>("alexdremov_qk_norm_rope::forward");
  return op;
}
const c10::TypedOperatorHandle<RopeBackward>& rope_backward_op() {
  static const auto op = find_op<RopeBackward>("alexdremov_qk_norm_rope::backward");
  return op;
}
bool wants_grad(const OptTensor& t) { return t && kv_native::wants_grad({&*t}); }
bool has_tangent(const OptTensor& t) { return t && kv_native::has_tangent({&*t}); }

// Saves its inputs: the norms are formed again from q and k.
struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& cos,
                                                const Tensor& sin, const OptTensor& q_weight, const OptTensor& k_weight, const OptTensor& lens,
                                                const OptTensor& positions, OptDouble eps, bool interleaved, bool weights) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [q_out, k_out] = rope_forward_op().call(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved);
    auto maybe = [](const OptTensor& t) { return t ? *t : Tensor(); };
    ctx->save_for_backward({q, k, cos, sin, maybe(q_weight), maybe(k_weight), maybe(lens), maybe(positions)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["weights"] = weights;
    return {std::move(q_out), std::move(k_out)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(11);   // one per argument of forward
    const auto saved = ctx->get_saved_variables();
    auto maybe = [&](int i) { return saved[i].defined() ? OptTensor(saved[i]) : OptTensor(); };
    const bool weights = ctx->saved_data["weights"].toBool();
    auto [dq, dk, dwq, dwk] = rope_backward_op().call(grads[0], grads[1], saved[0], saved[1], saved[2], saved[3], maybe(4), maybe(5), maybe(6),
                                                      maybe(7), ctx->saved_data["eps"].toOptional<double>(),
                                                      ctx->saved_data["interleaved"].toBool(), weights);
    out[0] = std::move(dq), out[1] = std::move(dk);
    if (weights && saved[4].defined()) out[4] = std::move(dwq);
    if (weights && saved[5].defined()) out[5] = std::move(dwk);
    return out;
  }
};
std::tuple<Tensor, Tensor> rope_forward_autograd(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const OptTensor& q_weight,
                                                 const OptTensor& k_weight, const OptTensor& lens, const OptTensor& positions, OptDouble eps,
                                                 bool interleaved) {
  // a tangent must not be dropped in silence, nor a gradient of the angles
  TORCH_CHECK_NOT_IMPLEMENTED(!kv_native::has_tangent({&q, &k, &cos, &sin}) && !has_tangent(q_weight) && !has_tangent(k_weight),
                              "alexdremov_qk_norm_rope::forward has no forward-mode derivative");
  TORCH_CHECK(!kv_native::wants_grad({&cos, &sin}), "alexdremov_qk_norm_rope::forward passes no gradient on to cos and sin: detach them");
  const bool weights = wants_grad(q_weight) || wants_grad(k_weight);
  if (!weights && !kv_native::wants_grad({&q, &k})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return rope_forward_op().call(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved);
  }
  auto r = QkNormRope::apply(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved, weights);
  return {std::move(r[0]), std::move(r[1])};
}

// Marks the outputs of the backward op as not differentiable a second time.
struct NoDoubleBackward : torch::autograd::Function<NoDoubleBackward> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, const Tensor& dq, const Tensor& dk, const Tensor& dwq,
                                                const Tensor& dwk, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                const OptTensor&, const OptTensor&) {
    return {dq.view_as(dq), dk.view_as(dk), dwq.view_as(dwq), dwk.view_as(dwk)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "alexdremov_qk_norm_rope::backward has no autograd formula: differentiating through the backward pass "
                       "(double backward) is not supported");
  }
};
std::tuple<Tensor, Tensor, Tensor, Tensor> rope_backward_autograd(const Tensor& d_q, const Tensor& d_k, const Tensor& q, const Tensor& k,
                                                                  const Tensor& cos, const Tensor& sin, const OptTensor& q_weight,
                                                                  const OptTensor& k_weight, const OptTensor& lens, const OptTensor& positions,
                                                                  OptDouble eps, bool interleaved, bool weights) {
  const bool record = kv_native::wants_grad({&d_q, &d_k, &q, &k}) || wants_grad(q_weight) || wants_grad(k_weight);
  std::tuple<Tensor, Tensor, Tensor, Tensor> r;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    r = rope_backward_op().call(d_q, d_k, q, k, cos, sin, q_weight, k_weight, lens, positions, eps, interleaved, weights);
  }
  if (!record) return r;
  auto g = NoDoubleBackward::apply(std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), d_q, d_k, q, k, q_weight, k_weight);
  return {std::move(g[0]), std::move(g[1]), std::move(g[2]), std::move(g[3])};
}

// ---- into the pages ----------------------------------------------------------------------------------------------
Tensor append_rope_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                       const Tensor& lens, const Tensor& cos, const Tensor& sin, const OptTensor& q_weight, const OptTensor& k_weight,
                       const OptTensor& new_lens, const OptTensor& positions, OptDouble eps, bool interleaved) {
  if (C10_UNLIKELY(!(is_cache(q, k_pages, v_pages, page_table, lens, new_lens) && q.size(1) % k_pages.size(1) == 0 && is_pair(q, k, new_lens) &&
                     k.size(1) == k_pages.size(1) && v.sizes() == k.sizes() && alike(k, v) &&
                     is_rotation(q, cos, sin, q_weight, k_weight, positions, eps)))) {
    Gil gil;
    explain("_validate_append_rope",
            {THPVariable_Wrap(q), THPVariable_Wrap(k), THPVariable_Wrap(v), THPVariable_Wrap(k_pages), THPVariable_Wrap(v_pages),
             THPVariable_Wrap(page_table), THPVariable_Wrap(lens), THPVariable_Wrap(cos), THPVariable_Wrap(sin), wrap(q_weight), wrap(k_weight),
             wrap(new_lens), wrap(positions), wrap(eps)});
  }
  const c10::OptionalDeviceGuard guard(q.device());
  for (const Tensor* t : {&k_pages, &v_pages})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  Tensor q_out = empty_same(q);
  if (q.numel() == 0) return q_out;
  const Tensor qk = rows_layout(q), kk = rows_layout(k), vk = rows_layout(v), ct = table_layout(cos), st = table_layout(sin);
  const Tensor table = unit_rows(page_table);
  const OptTensor wq = weight_layout(q_weight), wk = weight_layout(k_weight);
  const Lengths l(lens), nl(new_lens);
  const Positions pos(positions);
  check_launch(api().paged_append_rope(ptr(qk), ptr(kk), ptr(vk), out_ptr(q_out), out_ptr(k_pages), out_ptr(v_pages), table.const_data_ptr<int32_t>(),
                                       table.stride(0), l.p, l.stride, nl.p, nl.stride, (const float*)ptr(ct), (const float*)ptr(st),
                                       row_stride(ct), row_stride(st), opt_ptr(wq), opt_ptr(wk), weights_f32(wq, wk), pos.p, pos.s, Strides(qk),
                                       Strides(kk), Strides(vk), Strides(k_pages), Strides(v_pages), (int)q.size(0), (int)q.size(1),
                                       (int)k.size(1), (int)q.size(2), (int)q.size(3), (int)k_pages.size(0), (int)k_pages.size(2),
                                       (int)table.size(1), (int)(2 * cos.size(1)), (int)cos.size(0), interleaved, c_eps(eps), dtype_id(q),
                                       current_stream(q)),
               "kv_paged_append_rope");
  return q_out;
}

using AppendRope = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                          const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, OptDouble, bool);
const c10::TypedOperatorHandle<AppendRope>& append_rope_op() {
  static const auto op = find_op<AppendRope>("alexdremov_paged_attention::append_rope");
  return op;
}
// The cache takes values, no history.
Tensor append_rope_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages,
                            const Tensor& page_table, const Tensor& lens, const Tensor& cos, const Tensor& sin, const OptTensor& q_weight,
                            const OptTensor& k_weight, const OptTensor& new_lens, const OptTensor& positions, OptDouble eps, bool interleaved) {
  TORCH_CHECK_NOT_IMPLEMENTED(!kv_native::has_tangent({&q, &k, &v, &k_pages, &v_pages, &cos, &sin}) && !has_tangent(q_weight) && !has_tangent(k_weight),
                              "alexdremov_paged_attention::append_rope has no forward-mode derivative");
  TORCH_CHECK(!kv_native::wants_grad({&q, &k, &v, &k_pages, &v_pages, &cos, &sin}) && !wants_grad(q_weight) && !wants_grad(k_weight),
              "alexdremov_paged_attention::append_rope records no gradient: call it under torch.no_grad() or on detached tensors");
  at::AutoDispatchBelowADInplaceOrView below;
  return append_rope_op().call(q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions, eps, interleaved);
}

}  // namespace

// qk_norm_rope(q, k, cos, sin, q_weight, k_weight, lens, positions, eps or None, interleaved)
PyObject* py_qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, cos, sin;
  OptTensor q_weight, k_weight, lens, positions;
  OptDouble eps;
  if (n != 10 || !tensor_arg(args[0], q) || !tensor_arg(args[1], k) || !tensor_arg(args[2], cos) || !tensor_arg(args[3], sin) ||
      !optional_arg(args[4], q_weight) || !optional_arg(args[5], k_weight) || !optional_arg(args[6], lens) || !optional_arg(args[7], positions) ||
      !eps_arg(args[8], eps) || !PyBool_Check(args[9]))
    Py_RETURN_NOTIMPLEMENTED;
  std::tuple<Tensor, Tensor> r;
  {
    pybind11::gil_scoped_release no_gil;
    r = rope_forward_op().call(q, k, cos, sin, q_weight, k_weight, lens, positions, eps, args[9] == Py_True);
  }
  PyObject* first = THPVariable_Wrap(std::get<0>(r));
  return Py_BuildValue("(NN)", first, THPVariable_Wrap(std::get<1>(r)));
  END_HANDLE_TH_ERRORS
}

// paged_append_rope(q, k, v, k_pages, v_pages, page_table, lens, cos, sin, q_weight, k_weight, new_lens, positions, eps or None, interleaved)
PyObject* py_paged_append_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor t[9];
  OptTensor o[4];
  OptDouble eps;
  if (n != 15) Py_RETURN_NOTIMPLEMENTED;
  for (int i = 0; i < 9; ++i)
    if (!tensor_arg(args[i], t[i])) Py_RETURN_NOTIMPLEMENTED;
  for (int i = 0; i < 4; ++i)
    if (!optional_arg(args[9 + i], o[i])) Py_RETURN_NOTIMPLEMENTED;
  if (!eps_arg(args[13], eps) || !PyBool_Check(args[14])) Py_RETURN_NOTIMPLEMENTED;
  Tensor r;
  {
    pybind11::gil_scoped_release no_gil;
    r = append_rope_op().call(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], o[0], o[1], o[2], o[3], eps, args[14] == Py_True);
  }
  return THPVariable_Wrap(r);
  END_HANDLE_TH_ERRORS
}

TORCH_LIBRARY(alexdremov_qk_norm_rope, m) {
  m.def("forward(Tensor q, Tensor k, Tensor cos, Tensor sin, Tensor? q_weight, Tensor? k_weight, Tensor? lens, Tensor? positions, float? eps, "
        "bool interleaved) -> (Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("backward(Tensor d_q, Tensor d_k, Tensor q, Tensor k, Tensor cos, Tensor sin, Tensor? q_weight, Tensor? k_weight, Tensor? lens, "
        "Tensor? positions, float? eps, bool interleaved, bool weights) -> (Tensor, Tensor, Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(alexdremov_qk_norm_rope, CUDA, m) {
  m.impl("forward", TORCH_FN(rope_forward_gpu));
  m.impl("backward", TORCH_FN(rope_backward_gpu));
}
TORCH_LIBRARY_IMPL(alexdremov_qk_norm_rope, Autograd, m) {
  m.impl("forward", TORCH_FN(rope_forward_autograd));
  m.impl("backward", TORCH_FN(rope_backward_autograd));
}
TORCH_LIBRARY_FRAGMENT(alexdremov_paged_attention, m) {
  m.def("append_rope(Tensor q, Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor lens, Tensor cos, Tensor sin, "
        "Tensor? q_weight, Tensor? k_weight, Tensor? new_lens, Tensor? positions, float? eps, bool interleaved) -> Tensor",
        {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(alexdremov_paged_attention, CUDA, m) { m.impl("append_rope", TORCH_FN(append_rope_gpu)); }
TORCH_LIBRARY_IMPL(alexdremov_paged_attention, Autograd, m) { m.impl("append_rope", TORCH_FN(append_rope_autograd)); }

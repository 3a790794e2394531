// Native host side of cross attention and of attention over pages (module kv_attention._native): the dispatcher entries of
// alexdremov_cross_attention::{forward, backward} and alexdremov_paged_attention::{forward, append, tree_forward, keep}, their autograd, and the eager
// call path of the public Python functions, as sa_torch.cpp has them for streaming attention.
//
// The shared library is opened on the first call, the one that KV_ATTENTION_LIB names or the one beside this module; there is no
// other implementation.  Invalid arguments are handed to the _validate functions of kv_attention.ops, which name the condition (AssertionError).
#include "kv_torch.h"

using namespace kv_native;

namespace {

// ---- the shared library -------------------------------------------------------------------------------------
Api open_library() {
  std::string path;
  if (const char* env = getenv("KV_ATTENTION_LIB")) {
    path = env;
  } else {
    Dl_info info;
    TORCH_CHECK(dladdr(reinterpret_cast<void*>(&open_library), &info) != 0, "cannot locate this module");
    path = info.dli_fname;
    path = path.substr(0, path.rfind('/') + 1) + "libkv_attention.so";
  }
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(lib, "libkv_attention.so not found at ", path, " (", dlerror(),
              "): build it with `make -C kernels_amd/csrc`. There is no fallback implementation.");
  auto symbol = [&](const char* name) {
    void* p = dlsym(lib, name);
    TORCH_CHECK(p, path, " has no symbol ", name);
    return p;
  };
  Api a;
#define KV_SYMBOL(field) a.field = reinterpret_cast<decltype(a.field)>(symbol("kv_" #field))
  KV_SYMBOL(cross_forward);
  KV_SYMBOL(cross_forward_workspace);
  KV_SYMBOL(cross_backward);
  KV_SYMBOL(cross_backward_workspace);
  KV_SYMBOL(paged_forward);
  KV_SYMBOL(paged_forward_workspace);
  KV_SYMBOL(paged_append);
  KV_SYMBOL(paged_append_rope);
  KV_SYMBOL(paged_tree_forward);
  KV_SYMBOL(paged_tree_forward_workspace);
  KV_SYMBOL(paged_keep);
  KV_SYMBOL(qk_norm_rope);
  KV_SYMBOL(qk_norm_rope_backward);
  KV_SYMBOL(qk_norm_rope_backward_workspace);
  KV_SYMBOL(error_string);
#undef KV_SYMBOL
  return a;
}
}  // namespace

const Api& kv_native::api() {
  static const Api a = open_library();   // tried again by the next call if it throws
  return a;
}

namespace {

// ---- cross attention --------------------------------------------------------------------------------------------
void validate_cross(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens, const OptTensor& q_lens, double sm_scale,
                    std::initializer_list<const Tensor*> more = {}) {
  bool ok = is_cross(q, k, v, lens, q_lens, sm_scale);
  for (const Tensor* t : more) ok = ok && t->sizes() == q.sizes() && t->device() == q.device();
  if (C10_LIKELY(ok)) return;
  Gil gil;
  PyObject *q_ = THPVariable_Wrap(q), *k_ = THPVariable_Wrap(k), *v_ = THPVariable_Wrap(v), *s_ = PyFloat_FromDouble(sm_scale);
  if (more.size() == 2)
    explain("_validate_cross", {q_, k_, v_, wrap(lens), wrap(q_lens), s_, THPVariable_Wrap(**more.begin()), THPVariable_Wrap(**(more.begin() + 1))});
  explain("_validate_cross", {q_, k_, v_, wrap(lens), wrap(q_lens), s_});
}

// The kernels' part of the forward; q, k and v in kernel_layout.
void cross_forward_into(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens, const OptTensor& q_lens, double sm_scale,
                        const Tensor& o, float* lse) {
  const Api& a = api();
  const int B = (int)q.size(0), Hq = (int)q.size(1), Tq = (int)q.size(2), D = (int)q.size(3), Hkv = (int)k.size(1), Tk = (int)k.size(2);
  const int64_t bytes = a.cross_forward_workspace(B, Hq, Hkv, Tq, Tk, D, dtype_id(q));
  check(bytes, "kv_cross_forward");
  const Tensor ws = bytes > 0 ? workspace(q, bytes) : Tensor();
  const Lengths l(lens), ql(q_lens);
  check_launch(a.cross_forward(ptr(q), ptr(k), ptr(v), l.p, l.stride, ql.p, ql.stride, out_ptr(o), lse, bytes > 0 ? out_ptr(ws) : nullptr, bytes,
                               Strides(q), Strides(k), Strides(v), B, Hq, Hkv, Tq, Tk, D, (float)sm_scale, dtype_id(q), current_stream(q)),
               "kv_cross_forward");
}

std::tuple<Tensor, Tensor> cross_forward_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens,
                                             const OptTensor& q_lens, double sm_scale, bool return_lse) {
  validate_cross(q, k, v, lens, q_lens, sm_scale);
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor o = empty_same(q);
  Tensor lse = return_lse ? empty_rows(q) : at::empty({0});
  if (q.numel() > 0)
    cross_forward_into(kernel_layout(q), kernel_layout(k), kernel_layout(v), lens, q_lens, sm_scale, o, return_lse ? (float*)out_ptr(lse) : nullptr);
  return {std::move(o), std::move(lse)};
}

std::tuple<Tensor, Tensor, Tensor> cross_backward_gpu(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens,
                                                      const OptTensor& q_lens, const Tensor& o, const Tensor& lse_in, const Tensor& d_o,
                                                      double sm_scale) {
  validate_cross(q, k, v, lens, q_lens, sm_scale, {&o, &d_o});
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor dq = empty_same(q);
  if (q.numel() == 0) return {std::move(dq), at::zeros(k.sizes(), k.options()), at::zeros(v.sizes(), v.options())};
  const Api& a = api();
  Tensor dk = empty_same(k), dv = empty_same(v);
  const Tensor qk = kernel_layout(q), kk = kernel_layout(k), vk = kernel_layout(v);
  // the upstream gradient may arrive in another type and with arbitrary strides
  const Tensor gk = kernel_layout(d_o.to(q.scalar_type())), ok = kernel_layout(o.to(q.scalar_type()));
  Tensor lse = lse_in;
  if (lse.numel() != q.numel() / q.size(3) || lse.device() != q.device()) {   // the forward ran with return_lse=False
    lse = empty_rows(q);
    cross_forward_into(qk, kk, vk, lens, q_lens, sm_scale, empty_same(q), (float*)out_ptr(lse));
  }
  lse = lse.to(at::kFloat).contiguous();
  const int B = (int)q.size(0), Hq = (int)q.size(1), Tq = (int)q.size(2), D = (int)q.size(3), Hkv = (int)k.size(1), Tk = (int)k.size(2);
  const int64_t bytes = a.cross_backward_workspace(B, Hq, Hkv, Tq, Tk, D, dtype_id(q));
  check(bytes, "kv_cross_backward");
  const Tensor ws = workspace(q, bytes);
  const Lengths l(lens), ql(q_lens);
  check_launch(a.cross_backward(ptr(qk), ptr(kk), ptr(vk), l.p, l.stride, ql.p, ql.stride, ptr(ok), ptr(gk), (const float*)ptr(lse), out_ptr(dq),
                                out_ptr(dk), out_ptr(dv), out_ptr(ws), bytes, Strides(qk), Strides(kk), Strides(vk), Strides(ok), Strides(gk), B,
                                Hq, Hkv, Tq, Tk, D, (float)sm_scale, dtype_id(q), current_stream(q)),
               "kv_cross_backward");
  return {std::move(dq), std::move(dk), std::move(dv)};
}

using CrossForward = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, double, bool);
using CrossBackward = std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                         const Tensor&, const Tensor&, const Tensor&, double);
const c10::TypedOperatorHandle<CrossForward>& cross_forward_op() {
  static const auto op = find_op<CrossForward>("alexdremov_cross_attention::forward");
  return op;
}
const c10::TypedOperatorHandle<CrossBackward>& cross_backward_op() {
  static const auto op = find_op<CrossBackward>("alexdremov_cross_attention::backward");
  return op;
}

// Saves q, k, v, O, LSE and the lengths and hands dO to the backward op.  No gradient flows through the log-sum-exp: it leaves through
// lse_out, beside the node's one output, as in sa_torch.cpp.
struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens,
                        const OptTensor& q_lens, double sm_scale, bool return_lse, Tensor* lse_out) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse] = cross_forward_op().call(q, k, v, lens, q_lens, sm_scale, return_lse);
    ctx->save_for_backward({q, k, v, o, lse, lens ? *lens : Tensor(), q_lens ? *q_lens : Tensor()});
    ctx->saved_data["sm_scale"] = sm_scale;
    ctx->set_materialize_grads(false);   // a missing gradient of O is made in backward, in O's own type and layout
    *lse_out = std::move(lse);
    return o;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(8);   // one per argument of forward
    const auto saved = ctx->get_saved_variables();
    const Tensor d_o = grads[0].defined() ? grads[0] : at::zeros_like(saved[3]);
    auto lengths = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    auto [dq, dk, dv] = cross_backward_op().call(saved[0], saved[1], saved[2], lengths(saved[5]), lengths(saved[6]), saved[3], saved[4], d_o,
                                                 ctx->saved_data["sm_scale"].toDouble());
    out[0] = std::move(dq), out[1] = std::move(dk), out[2] = std::move(dv);
    return out;
  }
};

std::tuple<Tensor, Tensor> cross_forward_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens,
                                                  const OptTensor& q_lens, double sm_scale, bool return_lse) {
  // a tangent must not be dropped in silence
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&q, &k, &v}), "alexdremov_cross_attention::forward has no forward-mode derivative");
  if (!wants_grad({&q, &k, &v})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return cross_forward_op().call(q, k, v, lens, q_lens, sm_scale, return_lse);
  }
  Tensor lse;
  Tensor o = CrossAttention::apply(q, k, v, lens, q_lens, sm_scale, return_lse, &lse);
  return {std::move(o), std::move(lse)};
}

// Marks the outputs of the backward op as not differentiable a second time.
struct NoDoubleBackward : torch::autograd::Function<NoDoubleBackward> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext*, const Tensor& dq, const Tensor& dk, const Tensor& dv,
                                                const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&) {
    return {dq.view_as(dq), dk.view_as(dk), dv.view_as(dv)};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "alexdremov_cross_attention::backward has no autograd formula: differentiating through the backward pass "
                       "(double backward) is not supported");
  }
};
std::tuple<Tensor, Tensor, Tensor> cross_backward_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens,
                                                           const OptTensor& q_lens, const Tensor& o, const Tensor& lse, const Tensor& d_o,
                                                           double sm_scale) {
  const bool record = wants_grad({&q, &k, &v, &o, &d_o});   // (gradient mode is off under an ordinary .backward())
  std::tuple<Tensor, Tensor, Tensor> r;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    r = cross_backward_op().call(q, k, v, lens, q_lens, o, lse, d_o, sm_scale);
  }
  if (!record) return r;
  auto g = NoDoubleBackward::apply(std::get<0>(r), std::get<1>(r), std::get<2>(r), q, k, v, o, d_o);
  return {std::move(g[0]), std::move(g[1]), std::move(g[2])};
}

// ---- pages --------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor> paged_forward_gpu(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                                             const Tensor& lens, int64_t context_size, int64_t back_contexts, double sm_scale,
                                             const OptTensor& new_lens, bool return_lse) {
  if (C10_UNLIKELY(!(is_cache(q, k_pages, v_pages, page_table, lens, new_lens) && q.size(1) % k_pages.size(1) == 0 && context_size >= 1 &&
                     back_contexts >= 0 && is_scale(sm_scale)))) {
    Gil gil;
    explain("_validate_paged", {THPVariable_Wrap(q), THPVariable_Wrap(k_pages), THPVariable_Wrap(v_pages), THPVariable_Wrap(page_table),
                                THPVariable_Wrap(lens), PyLong_FromLongLong(context_size), PyLong_FromLongLong(back_contexts),
                                PyFloat_FromDouble(sm_scale), wrap(new_lens)});
  }
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor o = empty_same(q);
  Tensor lse = return_lse ? empty_rows(q) : at::empty({0});
  if (q.numel() == 0) return {std::move(o), std::move(lse)};
  const Api& a = api();
  const Tensor qk = kernel_layout(q);
  const Tensor table = unit_rows(page_table);
  const int B = (int)q.size(0), Hq = (int)q.size(1), T = (int)q.size(2), D = (int)q.size(3);
  const int N = (int)k_pages.size(0), Hkv = (int)k_pages.size(1), page = (int)k_pages.size(2), W = (int)table.size(1);
  const int C = clamp_int(context_size), R = clamp_int(back_contexts);
  const int64_t bytes = a.paged_forward_workspace(B, Hq, Hkv, T, D, page, W, C, R, dtype_id(q));
  check(bytes, "kv_paged_forward");
  const Tensor ws = bytes > 0 ? workspace(q, bytes) : Tensor();
  const Lengths l(lens), nl(new_lens);
  check_launch(a.paged_forward(ptr(qk), ptr(k_pages), ptr(v_pages), table.const_data_ptr<int32_t>(), table.stride(0), l.p, l.stride, nl.p,
                               nl.stride, out_ptr(o), return_lse ? (float*)out_ptr(lse) : nullptr, bytes > 0 ? out_ptr(ws) : nullptr, bytes,
                               Strides(qk), Strides(k_pages), Strides(v_pages), B, Hq, Hkv, T, D, N, page, W, C, R, (float)sm_scale,
                               dtype_id(q), current_stream(q)),
               "kv_paged_forward");
  return {std::move(o), std::move(lse)};
}

void paged_append_gpu(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                      const Tensor& lens, const OptTensor& new_lens) {
  if (C10_UNLIKELY(!(is_cache(k, k_pages, v_pages, page_table, lens, new_lens) && k.size(1) == k_pages.size(1) && v.sizes() == k.sizes() &&
                     alike(k, v)))) {
    Gil gil;
    explain("_validate_append", {THPVariable_Wrap(k), THPVariable_Wrap(v), THPVariable_Wrap(k_pages), THPVariable_Wrap(v_pages),
                                 THPVariable_Wrap(page_table), THPVariable_Wrap(lens), wrap(new_lens)});
  }
  const c10::OptionalDeviceGuard guard(k.device());
  for (const Tensor* t : {&k_pages, &v_pages})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  if (k.numel() == 0 || k_pages.numel() == 0 || page_table.numel() == 0) return;
  const Tensor kk = kernel_layout(k), vk = kernel_layout(v);
  const Tensor table = unit_rows(page_table);
  const Lengths l(lens), nl(new_lens);
  check_launch(api().paged_append(ptr(kk), ptr(vk), out_ptr(k_pages), out_ptr(v_pages), table.const_data_ptr<int32_t>(), table.stride(0), l.p,
                                  l.stride, nl.p, nl.stride, Strides(kk), Strides(vk), Strides(k_pages), Strides(v_pages), (int)k.size(0),
                                  (int)k.size(1), (int)k.size(2), (int)k.size(3), (int)k_pages.size(0), (int)k_pages.size(2),
                                  (int)table.size(1), dtype_id(k), current_stream(k)),
               "kv_paged_append");
}

bool is_tree(const Tensor& tree, const Tensor& q) {
  const int64_t d = tree.dim();
  return (d == 2 || (d == 3 && tree.size(0) == q.size(0))) && tree.scalar_type() == at::kBool && tree.device() == q.device() &&
         tree.size(-1) == q.size(2) && tree.size(-2) == q.size(2);
}
std::tuple<Tensor, Tensor> tree_forward_gpu(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                                            const Tensor& lens, const Tensor& tree, double sm_scale, const OptTensor& new_lens,
                                            bool return_lse) {
  if (C10_UNLIKELY(!(is_cache(q, k_pages, v_pages, page_table, lens, new_lens) && q.size(1) % k_pages.size(1) == 0 && is_tree(tree, q) &&
                     is_scale(sm_scale)))) {
    Gil gil;
    explain("_validate_tree", {THPVariable_Wrap(q), THPVariable_Wrap(k_pages), THPVariable_Wrap(v_pages), THPVariable_Wrap(page_table),
                               THPVariable_Wrap(lens), THPVariable_Wrap(tree), PyFloat_FromDouble(sm_scale), wrap(new_lens)});
  }
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor o = empty_same(q);
  Tensor lse = return_lse ? empty_rows(q) : at::empty({0});
  if (q.numel() == 0) return {std::move(o), std::move(lse)};
  const Api& a = api();
  const Tensor qk = kernel_layout(q), table = unit_rows(page_table);
  const int B = (int)q.size(0), Hq = (int)q.size(1), T = (int)q.size(2), D = (int)q.size(3);
  const int N = (int)k_pages.size(0), Hkv = (int)k_pages.size(1), page = (int)k_pages.size(2), W = (int)table.size(1);
  const int64_t bytes = a.paged_tree_forward_workspace(B, Hq, Hkv, T, D, page, W, dtype_id(q));
  check(bytes, "kv_paged_tree_forward");
  const Tensor ws = bytes > 0 ? workspace(q, bytes) : Tensor();
  const Lengths l(lens), nl(new_lens);
  const int64_t tree_strides[3] = {tree.dim() == 3 ? tree.stride(0) : 0, tree.stride(-2), tree.stride(-1)};
  check_launch(a.paged_tree_forward(ptr(qk), ptr(k_pages), ptr(v_pages), table.const_data_ptr<int32_t>(), table.stride(0), l.p, l.stride, nl.p,
                                    nl.stride, ptr(tree), tree_strides, out_ptr(o), return_lse ? (float*)out_ptr(lse) : nullptr,
                                    bytes > 0 ? out_ptr(ws) : nullptr, bytes, Strides(qk), Strides(k_pages), Strides(v_pages), B, Hq, Hkv, T, D,
                                    N, page, W, (float)sm_scale, dtype_id(q), current_stream(q)),
               "kv_paged_tree_forward");
  return {std::move(o), std::move(lse)};
}

void paged_keep_gpu(const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table, const Tensor& first, const Tensor& kept) {
  if (C10_UNLIKELY(!(is_pages(k_pages, v_pages, page_table) && first.dim() == 1 && kept.dim() == 2 && first.scalar_type() == at::kInt &&
                     kept.scalar_type() == at::kInt && first.size(0) == page_table.size(0) && kept.size(0) == page_table.size(0) &&
                     small(kept.size(1)) && first.device() == k_pages.device() && kept.device() == k_pages.device()))) {
    Gil gil;
    explain("_validate_keep", {THPVariable_Wrap(k_pages), THPVariable_Wrap(v_pages), THPVariable_Wrap(page_table), THPVariable_Wrap(first),
                               THPVariable_Wrap(kept)});
  }
  const c10::OptionalDeviceGuard guard(k_pages.device());
  for (const Tensor* t : {&k_pages, &v_pages})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  if (k_pages.numel() == 0 || page_table.numel() == 0 || kept.numel() == 0) return;
  const Tensor table = unit_rows(page_table);
  const int64_t kept_strides[2] = {kept.stride(0), kept.stride(1)};
  check_launch(api().paged_keep(out_ptr(k_pages), out_ptr(v_pages), table.const_data_ptr<int32_t>(), table.stride(0), first.const_data_ptr<int32_t>(),
                                first.stride(0), kept.const_data_ptr<int32_t>(), kept_strides, Strides(k_pages), Strides(v_pages),
                                (int)table.size(0), (int)k_pages.size(1), (int)kept.size(1), (int)k_pages.size(3), (int)k_pages.size(0),
                                (int)k_pages.size(2), (int)table.size(1), dtype_id(k_pages), current_stream(k_pages)),
               "kv_paged_keep");
}

using PagedForward = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, SymInt, SymInt,
                                                double, const OptTensor&, bool);
using PagedAppend = void(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const OptTensor&);
const c10::TypedOperatorHandle<PagedForward>& paged_forward_op() {
  static const auto op = find_op<PagedForward>("alexdremov_paged_attention::forward");
  return op;
}
const c10::TypedOperatorHandle<PagedAppend>& paged_append_op() {
  static const auto op = find_op<PagedAppend>("alexdremov_paged_attention::append");
  return op;
}

using TreeForward = std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, double,
                                               const OptTensor&, bool);
using PagedKeep = void(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&);
const c10::TypedOperatorHandle<TreeForward>& tree_forward_op() {
  static const auto op = find_op<TreeForward>("alexdremov_paged_attention::tree_forward");
  return op;
}
const c10::TypedOperatorHandle<PagedKeep>& paged_keep_op() {
  static const auto op = find_op<PagedKeep>("alexdremov_paged_attention::keep");
  return op;
}

// Forward only: the result of inputs that require a gradient requires one too, and asking for it raises.
struct PagedAttention : torch::autograd::Function<PagedAttention> {
  static Tensor forward(torch::autograd::AutogradContext*, const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                        const Tensor& page_table, const Tensor& lens, SymInt context_size, SymInt back_contexts, double sm_scale,
                        const OptTensor& new_lens, bool return_lse, Tensor* lse_out) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse] = paged_forward_op().call(q, k_pages, v_pages, page_table, lens, context_size, back_contexts, sm_scale, new_lens, return_lse);
    *lse_out = std::move(lse);
    return o;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "Trying to backward through alexdremov_paged_attention.forward.default but no autograd formula was registered: "
                       "attention over pages is forward only");
  }
};
std::tuple<Tensor, Tensor> paged_forward_autograd(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                                                  const Tensor& lens, SymInt context_size, SymInt back_contexts, double sm_scale,
                                                  const OptTensor& new_lens, bool return_lse) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&q, &k_pages, &v_pages}), "alexdremov_paged_attention::forward has no forward-mode derivative");
  if (!wants_grad({&q, &k_pages, &v_pages})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return paged_forward_op().call(q, k_pages, v_pages, page_table, lens, std::move(context_size), std::move(back_contexts), sm_scale, new_lens,
                                   return_lse);
  }
  Tensor lse;
  Tensor o = PagedAttention::apply(q, k_pages, v_pages, page_table, lens, std::move(context_size), std::move(back_contexts), sm_scale, new_lens,
                                   return_lse, &lse);
  return {std::move(o), std::move(lse)};
}
struct TreeAttention : torch::autograd::Function<TreeAttention> {
  static Tensor forward(torch::autograd::AutogradContext*, const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                        const Tensor& page_table, const Tensor& lens, const Tensor& tree, double sm_scale, const OptTensor& new_lens,
                        bool return_lse, Tensor* lse_out) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [o, lse] = tree_forward_op().call(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens, return_lse);
    *lse_out = std::move(lse);
    return o;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "Trying to backward through alexdremov_paged_attention.tree_forward.default but no autograd formula was registered: "
                       "attention over pages is forward only");
  }
};
std::tuple<Tensor, Tensor> tree_forward_autograd(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                                                 const Tensor& lens, const Tensor& tree, double sm_scale, const OptTensor& new_lens,
                                                 bool return_lse) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&q, &k_pages, &v_pages}), "alexdremov_paged_attention::tree_forward has no forward-mode derivative");
  if (!wants_grad({&q, &k_pages, &v_pages})) {
    at::AutoDispatchBelowADInplaceOrView below;
    return tree_forward_op().call(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens, return_lse);
  }
  Tensor lse;
  Tensor o = TreeAttention::apply(q, k_pages, v_pages, page_table, lens, tree, sm_scale, new_lens, return_lse, &lse);
  return {std::move(o), std::move(lse)};
}
// The cache takes values, no history.
void paged_append_autograd(const Tensor& k, const Tensor& v, const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                           const Tensor& lens, const OptTensor& new_lens) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&k, &v, &k_pages, &v_pages}), "alexdremov_paged_attention::append has no forward-mode derivative");
  TORCH_CHECK(!wants_grad({&k, &v, &k_pages, &v_pages}),
              "alexdremov_paged_attention::append records no gradient: call it under torch.no_grad() or on detached tensors");
  at::AutoDispatchBelowADInplaceOrView below;
  paged_append_op().call(k, v, k_pages, v_pages, page_table, lens, new_lens);
}

void paged_keep_autograd(const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table, const Tensor& first, const Tensor& kept) {
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent({&k_pages, &v_pages}), "alexdremov_paged_attention::keep has no forward-mode derivative");
  TORCH_CHECK(!wants_grad({&k_pages, &v_pages}),
              "alexdremov_paged_attention::keep records no gradient: call it under torch.no_grad() or on detached tensors");
  at::AutoDispatchBelowADInplaceOrView below;
  paged_keep_op().call(k_pages, v_pages, page_table, first, kept);
}

// ---- eager call path of the public functions ------------------------------------------------------------------------
// As in sa_torch.cpp: arguments come positionally and complete; one that is not of the plain type returns NotImplemented, and the Python functions
// call the op itself, which converts or refuses it.
PyObject* result(const std::tuple<Tensor, Tensor>& r, bool return_lse) {
  PyObject* o = THPVariable_Wrap(std::get<0>(r));
  if (!return_lse || !o) return o;
  return Py_BuildValue("(NN)", o, THPVariable_Wrap(std::get<1>(r)));
}

// cross_attention(q, k, v, lens, q_lens, sm_scale or None, return_lse)
PyObject* py_cross_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v;
  OptTensor lens, q_lens;
  double sm_scale;
  if (n != 7 || !tensor_arg(args[0], q) || !tensor_arg(args[1], k) || !tensor_arg(args[2], v) || !optional_arg(args[3], lens) ||
      !optional_arg(args[4], q_lens) || !scale_arg(args[5], q, sm_scale) || !PyBool_Check(args[6]))
    Py_RETURN_NOTIMPLEMENTED;
  const bool return_lse = args[6] == Py_True;
  // the log-sum-exp is needed by the backward pass whenever a gradient is wanted
  const bool need_lse = return_lse || wants_grad({&q, &k, &v});
  std::tuple<Tensor, Tensor> r;
  {
    pybind11::gil_scoped_release no_gil;
    r = cross_forward_op().call(q, k, v, lens, q_lens, sm_scale, need_lse);
  }
  return result(r, return_lse);
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_pages, v_pages, page_table, lens, context_size, back_contexts, sm_scale or None, new_lens, return_lse)
PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, table, lens;
  OptTensor new_lens;
  int64_t C, R;
  double sm_scale;
  if (n != 10 || !tensor_arg(args[0], q) || !tensor_arg(args[1], k) || !tensor_arg(args[2], v) || !tensor_arg(args[3], table) ||
      !tensor_arg(args[4], lens) || !int_arg(args[5], C) || !int_arg(args[6], R) || !scale_arg(args[7], q, sm_scale) ||
      !optional_arg(args[8], new_lens) || !PyBool_Check(args[9]))
    Py_RETURN_NOTIMPLEMENTED;
  const bool return_lse = args[9] == Py_True;
  std::tuple<Tensor, Tensor> r;
  {
    pybind11::gil_scoped_release no_gil;
    r = paged_forward_op().call(q, k, v, table, lens, C, R, sm_scale, new_lens, return_lse);
  }
  return result(r, return_lse);
  END_HANDLE_TH_ERRORS
}

// paged_append(k, v, k_pages, v_pages, page_table, lens, new_lens)
PyObject* py_paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor k, v, k_pages, v_pages, table, lens;
  OptTensor new_lens;
  if (n != 7 || !tensor_arg(args[0], k) || !tensor_arg(args[1], v) || !tensor_arg(args[2], k_pages) || !tensor_arg(args[3], v_pages) ||
      !tensor_arg(args[4], table) || !tensor_arg(args[5], lens) || !optional_arg(args[6], new_lens))
    Py_RETURN_NOTIMPLEMENTED;
  {
    pybind11::gil_scoped_release no_gil;
    paged_append_op().call(k, v, k_pages, v_pages, table, lens, new_lens);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// paged_tree_attention(q, k_pages, v_pages, page_table, lens, tree, sm_scale or None, new_lens, return_lse)
PyObject* py_paged_tree_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, table, lens, tree;
  OptTensor new_lens;
  double sm_scale;
  if (n != 9 || !tensor_arg(args[0], q) || !tensor_arg(args[1], k) || !tensor_arg(args[2], v) || !tensor_arg(args[3], table) ||
      !tensor_arg(args[4], lens) || !tensor_arg(args[5], tree) || !scale_arg(args[6], q, sm_scale) || !optional_arg(args[7], new_lens) ||
      !PyBool_Check(args[8]))
    Py_RETURN_NOTIMPLEMENTED;
  const bool return_lse = args[8] == Py_True;
  std::tuple<Tensor, Tensor> r;
  {
    pybind11::gil_scoped_release no_gil;
    r = tree_forward_op().call(q, k, v, table, lens, tree, sm_scale, new_lens, return_lse);
  }
  return result(r, return_lse);
  END_HANDLE_TH_ERRORS
}

// paged_keep(k_pages, v_pages, page_table, first, kept)
PyObject* py_paged_keep(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Tensor k, v, table, first, kept;
  if (n != 5 || !tensor_arg(args[0], k) || !tensor_arg(args[1], v) || !tensor_arg(args[2], table) || !tensor_arg(args[3], first) ||
      !tensor_arg(args[4], kept))
    Py_RETURN_NOTIMPLEMENTED;
  {
    pybind11::gil_scoped_release no_gil;
    paged_keep_op().call(k, v, table, first, kept);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"cross_attention", (PyCFunction)(void (*)())py_cross_attention, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)())py_paged_attention, METH_FASTCALL, nullptr},
    {"paged_append", (PyCFunction)(void (*)())py_paged_append, METH_FASTCALL, nullptr},
    {"paged_append_rope", (PyCFunction)(void (*)())py_paged_append_rope, METH_FASTCALL, nullptr},
    {"paged_tree_attention", (PyCFunction)(void (*)())py_paged_tree_attention, METH_FASTCALL, nullptr},
    {"paged_keep", (PyCFunction)(void (*)())py_paged_keep, METH_FASTCALL, nullptr},
    {"qk_norm_rope", (PyCFunction)(void (*)())py_qk_norm_rope, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

TORCH_LIBRARY(alexdremov_cross_attention, m) {
  m.def("forward(Tensor q, Tensor k, Tensor v, Tensor? lens, Tensor? q_lens, float sm_scale, bool return_lse) -> (Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("backward(Tensor q, Tensor k, Tensor v, Tensor? lens, Tensor? q_lens, Tensor o, Tensor lse, Tensor do, float sm_scale) "
        "-> (Tensor, Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(alexdremov_cross_attention, CUDA, m) {
  m.impl("forward", TORCH_FN(cross_forward_gpu));
  m.impl("backward", TORCH_FN(cross_backward_gpu));
}
TORCH_LIBRARY_IMPL(alexdremov_cross_attention, Autograd, m) {
  m.impl("forward", TORCH_FN(cross_forward_autograd));
  m.impl("backward", TORCH_FN(cross_backward_autograd));
}
TORCH_LIBRARY(alexdremov_paged_attention, m) {
  m.def("forward(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor lens, SymInt context_size, SymInt back_contexts, "
        "float sm_scale, Tensor? new_lens, bool return_lse) -> (Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("append(Tensor k, Tensor v, Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor lens, Tensor? new_lens) -> ()",
        {at::Tag::pt2_compliant_tag});
  m.def("tree_forward(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor lens, Tensor tree, float sm_scale, Tensor? new_lens, "
        "bool return_lse) -> (Tensor, Tensor)",
        {at::Tag::pt2_compliant_tag});
  m.def("keep(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor first, Tensor kept) -> ()", {at::Tag::pt2_compliant_tag});
}
TORCH_LIBRARY_IMPL(alexdremov_paged_attention, CUDA, m) {
  m.impl("forward", TORCH_FN(paged_forward_gpu));
  m.impl("append", TORCH_FN(paged_append_gpu));
  m.impl("tree_forward", TORCH_FN(tree_forward_gpu));
  m.impl("keep", TORCH_FN(paged_keep_gpu));
}
TORCH_LIBRARY_IMPL(alexdremov_paged_attention, Autograd, m) {
  m.impl("forward", TORCH_FN(paged_forward_autograd));
  m.impl("append", TORCH_FN(paged_append_autograd));
  m.impl("tree_forward", TORCH_FN(tree_forward_autograd));
  m.impl("keep", TORCH_FN(paged_keep_autograd));
}

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }

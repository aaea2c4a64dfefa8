// Attention of drafted tokens over a cache.

#include <ATen/core/grad_mode.h>

#include "nsa_host.h"

namespace nsa_host {

static void require(bool ok, const char* what) {
  if (!ok) throw Error(std::string("tree_attend: ") + what);
}

// -> out, lse
static std::vector<OptTensor> tree_attend(Tensor q, Tensor k_cache, Tensor v_cache, OptTensor lengths_, int64_t length, Tensor k, Tensor v,
                                          OptTensor mask_, double scale, bool want_lse, int64_t impl, int64_t status) {
  for (const Tensor* t : {&q, &k_cache, &v_cache, &k, &v}) {
    require_cuda(*t);
    require(t->dim() == 4, "tensors must be [batch, heads, rows, dim_head]");
    dtype_code(*t);
    require(t->device() == q.device() && t->scalar_type() == q.scalar_type(), "tensors must share device and type");
    for (int64_t s : t->sizes()) require(s <= 0x7fffffff, "a size is above 2^31");
    require(!at::GradMode::is_enabled() || !t->requires_grad(), "no gradient passes: call it under no_grad, or with detached tensors");
    require(!t->_fw_grad(0).defined(), "no forward-mode derivative passes: call it with the tensors without their tangents");
  }
  const int64_t b = q.size(0), t = q.size(2), d = q.size(3), kv = k.size(1);
  require(k.size(0) == b && k.size(2) == t && k.size(3) == d && v.sizes() == k.sizes(),
          "keys and values of the drafted tokens must both be [batch, kv_heads, tokens, dim_head]");
  require(k_cache.size(0) == b && k_cache.size(1) == kv && k_cache.size(3) == d && v_cache.sizes() == k_cache.sizes(),
          "cached keys and values must both be [batch, kv_heads, rows, dim_head] with the drafted tokens' heads");
  require(kv > 0 && q.size(1) > 0 && q.size(1) % kv == 0, "q_heads must be a positive multiple of kv_heads");
  const c10::cuda::CUDAGuard guard(q.device());
  const at::NoGradGuard no_grad;
  auto dense = [](const Tensor& x) { return x.size(3) == 1 || x.stride(3) == 1 ? x : x.contiguous(); };
  require(k_cache.stride(3) == 1 && v_cache.stride(3) == 1, "the caches' last axis must be contiguous");
  require(!k_cache.is_neg() && !v_cache.is_neg(), "the caches must not be views that are negated when read");
  for (Tensor* t : {&q, &k, &v})
    if (t->is_neg()) *t = t->resolve_neg();
  q = dense(q);
  k = q.scalar_type() == at::kBFloat16 ? rowwise(k) : dense(k);
  v = q.scalar_type() == at::kBFloat16 ? rowwise(v) : dense(v);
  nsa_tree_args a = {};
  a.batch = b; a.q_heads = q.size(1); a.kv_heads = kv; a.tokens = t; a.dim_head = d; a.capacity = k_cache.size(2);
  a.dtype = dtype_code(q); a.impl = impl; a.scale = scale; a.length = length;
  Tensor lengths = lengths_.value_or(Tensor()), mask = mask_.value_or(Tensor());
  if (lengths.defined()) {
    require_cuda(lengths);
    require(lengths.device() == q.device() && lengths.dim() == 1 && lengths.size(0) == b && (lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong),
            "lengths must be [batch], int32 or int64, on the device of q");
    lengths = lengths.scalar_type() == at::kLong ? lengths.clamp(0, a.capacity).to(at::kInt) : lengths.contiguous();
    a.lengths = ptr<int32_t>(lengths);
  }
  if (mask.defined()) {
    require_cuda(mask);
    require(mask.device() == q.device() && (mask.scalar_type() == at::kBool || mask.scalar_type() == at::kByte), "mask must be bool on the device of q");
    require((mask.dim() == 2 || (mask.dim() == 3 && (mask.size(0) == b || mask.size(0) == 1))) && mask.size(-1) == t && mask.size(-2) == t,
            "mask must be [tokens, tokens] or [batch, tokens, tokens]");
    if (t > 1 && mask.stride(-1) != 1) mask = mask.contiguous();
    a.mask = static_cast<const uint8_t*>(mask.data_ptr());
    a.mask_stride_b = mask.dim() == 3 && mask.size(0) > 1 ? mask.stride(0) : 0;
    a.mask_stride_t = mask.stride(-2);
  }
  Tensor out = at::empty(q.sizes(), q.options()), lse;
  if (want_lse) {
    lse = empty({b, q.size(1), t}, q, at::kFloat);
    a.lse = ptr<float>(lse);
  }
  a.q = t4(q); a.k = t4(k); a.v = t4(v); a.k_cache = t4(k_cache); a.v_cache = t4(v_cache); a.out = t4(out);
  a.status = reinterpret_cast<int32_t*>(status);
  const int64_t need = nsa_tree_workspace_bytes(&a);
  if (need < 0) check(need);
  Tensor ws;
  if (need > 0) {
    ws = bytes(need, q);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = need;
  }
  check(nsa_tree_attend(&a, stream_of(q)));
  return {out, want_lse ? OptTensor(lse) : OptTensor()};
}

void bind_tree(pybind11::module_& m) {
  m.def("tree_attend", &tree_attend, pybind11::call_guard<pybind11::gil_scoped_release>());
}

}  // namespace nsa_host

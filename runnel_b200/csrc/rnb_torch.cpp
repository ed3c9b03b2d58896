// rnb_torch.cpp -- the attention-side calls on torch tensors: argument checks,
// outputs and scratch from torch's allocator, one C-ABI call on the current
// stream.  A serving step makes these calls once a layer; through ctypes each
// spent 15-20 us on the host, of which the launches are 3-6.
//
// The C functions are not linked: bind() is given their addresses from the
// library that runnel_b200._lib has loaded.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <map>
#include <optional>
#include <string>

#include "rnb_moe.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

struct Fns {
  decltype(&rnb_kv_plan) kv_plan = nullptr;
  decltype(&rnb_kv_release_bounded) kv_release = nullptr;
  decltype(&rnb_rope_append) rope_append = nullptr;
  decltype(&rnb_paged_attention_workspace_size) workspace_size = nullptr;
  decltype(&rnb_paged_attention) paged_attention = nullptr;
} fns;

void bind(const std::map<std::string, uintptr_t>& at) {
  fns.kv_plan = reinterpret_cast<decltype(fns.kv_plan)>(at.at("rnb_kv_plan"));
  fns.kv_release = reinterpret_cast<decltype(fns.kv_release)>(at.at("rnb_kv_release_bounded"));
  fns.rope_append = reinterpret_cast<decltype(fns.rope_append)>(at.at("rnb_rope_append"));
  fns.workspace_size = reinterpret_cast<decltype(fns.workspace_size)>(at.at("rnb_paged_attention_workspace_size"));
  fns.paged_attention = reinterpret_cast<decltype(fns.paged_attention)>(at.at("rnb_paged_attention"));
}

// Raises RnbError for a C call's negative status.
void check(const char* fn, int rc) {
  if (rc != RNB_OK) py::module_::import("runnel_b200._lib").attr("check")(fn, rc);
}

std::string str(const char* s) { return s; }
std::string str(int64_t v) { return std::to_string(v); }
std::string str(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
std::string str(at::ScalarType t) { return c10::toString(t); }
std::string str(const at::Device& d) { return d.str(); }

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  throw py::value_error((str(a) + ...));
}

at::Device cuda_device(const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(name, " must be a CUDA tensor: the kernels have no other implementation");
  return t.device();
}

int32_t* ints(const Tensor& t, const char* name, at::Device dev) {
  if (t.scalar_type() != at::kInt || t.device() != dev || !t.is_contiguous())
    refuse(name, " must be a contiguous int32 tensor on ", dev);
  return static_cast<int32_t*>(t.data_ptr());
}

int32_t* ints(const Tensor& t, const char* name, at::Device dev, at::IntArrayRef shape) {
  if (t.sizes() != shape) refuse(name, " must have shape ", shape, ", not ", t.sizes());
  return ints(t, name, dev);
}

int c_int(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse(name, " does not fit 32 bits");
  return static_cast<int>(v);
}

Tensor empty(at::IntArrayRef shape, at::ScalarType dt, at::Device dev) {
  return at::detail::empty_cuda(shape, dt, dev, std::nullopt);
}

// n elements of a one-dimensional buffer, sharing its storage (as narrow() gives,
// without its dispatch).
Tensor part(const Tensor& buf, int64_t off, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(buf.storage()), buf.key_set(),
                                                      buf.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(buf.storage_offset() + off);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

// A [tokens, heads, head_dim] operand: itself if the kernels take its strides,
// else a packed copy.
struct Rows {
  Tensor t;
  void* p = nullptr;
  int64_t token = 0, head = 0;  // strides
};

Rows rows(const Tensor& t, const char* name, at::ScalarType dt, at::Device dev, at::IntArrayRef shape) {
  if (t.scalar_type() != dt || t.device() != dev) refuse(name, " must be a ", dt, " tensor on ", dev);
  if (t.sizes() != shape) refuse(name, " must have shape ", shape, ", not ", t.sizes());
  Rows r;
  // (a stride over an extent of one is never used)
  const int64_t packed = shape[1] * shape[2];
  r.token = shape[0] == 1 ? packed : t.stride(0);
  r.head = shape[1] == 1 ? shape[2] : t.stride(1);
  const bool ok = t.stride(2) == 1 && !((r.token | r.head) & 7) && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
  if (ok) {
    r.t = t;
  } else {
    r.t = t.is_contiguous() ? t.clone() : t.contiguous();
    r.token = packed, r.head = shape[2];
  }
  r.p = r.t.data_ptr();
  return r;
}

int dtype_code(at::ScalarType t) { return t == at::kBFloat16 ? RNB_DTYPE_BF16 : t == at::kHalf ? RNB_DTYPE_F16 : -1; }

rnb_kv_cache cache_of(const Tensor& k, const Tensor& v, at::ScalarType dt, at::Device dev) {
  if (k.device() != dev || k.scalar_type() != dt || v.device() != dev || v.scalar_type() != dt)
    refuse("k_cache and v_cache must be ", dt, " tensors on ", dev, ", like q");
  if (k.dim() != 4 || v.sizes() != k.sizes())
    refuse("k_cache and v_cache must be [num_pages, n_kv_heads, page_size, head_dim], both alike");
  const int64_t D = k.size(3);
  if (k.stride(3) != 1 || k.stride(2) != D || v.stride(3) != 1 || v.stride(2) != D)
    refuse("a head's page must be contiguous in k_cache and v_cache");
  rnb_kv_cache c{};
  c.dtype = dtype_code(dt);
  c.num_pages = c_int(k.size(0), "num_pages"), c.n_kv_heads = c_int(k.size(1), "n_kv_heads");
  c.page_size = c_int(k.size(2), "page_size"), c.head_dim = c_int(D, "head_dim");
  c.k = k.data_ptr(), c.v = v.data_ptr();
  c.k_page_stride = k.stride(0), c.k_head_stride = k.stride(1);
  c.v_page_stride = v.stride(0), c.v_head_stride = v.stride(1);
  return c;
}

Tensor output(const OptTensor& out, at::IntArrayRef shape, at::ScalarType dt, at::Device dev) {
  if (!out) return empty(shape, dt, dev);
  if (out->scalar_type() != dt || out->device() != dev || out->sizes() != shape || !out->is_contiguous())
    refuse("out must be a contiguous ", dt, " tensor of shape ", shape, " on ", dev);
  return *out;
}

void* stream_of(at::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> kv_plan(const Tensor& table, const Tensor& ctx_lens,
                                                           const Tensor& new_lens, const Tensor& free_pages,
                                                           const Tensor& free_count, int64_t page_size,
                                                           int64_t num_pages, int64_t max_tokens) {
  const at::Device dev = cuda_device(table, "table");
  if (table.dim() != 2) refuse("table must be [requests, columns]");
  if (max_tokens < 0) refuse("max_tokens must be >= 0");
  const int64_t B = table.size(0), cols = table.size(1);
  int32_t* tp = ints(table, "table", dev);
  const int32_t* cp = ints(ctx_lens, "ctx_lens", dev, {B});
  const int32_t* np = ints(new_lens, "new_lens", dev, {B});
  const int32_t* fp = ints(free_pages, "free_pages", dev);
  const int32_t* fc = ints(free_count, "free_count", dev, {1});
  const c10::cuda::CUDAGuard guard(dev);
  // one allocation; each output starts 16 bytes aligned
  const int64_t n[5] = {B, B + 1, max_tokens, max_tokens, 1};
  int64_t off[5], all = 0;
  for (int i = 0; i < 5; ++i) off[i] = all, all += (n[i] + 3) & ~int64_t(3);
  const Tensor buf = empty({all}, at::kInt, dev);
  Tensor seq = part(buf, off[0], n[0]), cu = part(buf, off[1], n[1]), pos = part(buf, off[2], n[2]),
         slots = part(buf, off[3], n[3]), left = part(buf, off[4], n[4]);
  auto p = [](Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
  check("rnb_kv_plan", fns.kv_plan(c_int(B, "requests"), c_int(cols, "columns"), c_int(page_size, "page_size"),
                                   c_int(num_pages, "num_pages"), c_int(max_tokens, "max_tokens"), tp, cp, np, fp,
                                   c_int(free_pages.numel(), "free_pages"), fc, p(seq), p(cu), p(pos), p(slots), p(left),
                                   stream_of(dev)));
  return {seq, cu, pos, slots, left};
}

std::tuple<Tensor, Tensor> kv_release(const Tensor& table, const Tensor& lens, const Tensor& finished,
                                      const Tensor& free_pages, const Tensor& free_count, int64_t page_size,
                                      std::optional<int64_t> num_pages) {
  const at::Device dev = cuda_device(table, "table");
  if (table.dim() != 2) refuse("table must be [requests, columns]");
  const int64_t B = table.size(0), cols = table.size(1);
  const int32_t* tp = ints(table, "table", dev);
  const int32_t* lp = ints(lens, "lens", dev, {B});
  const int32_t* np = ints(finished, "finished", dev, {B});
  int32_t* fp = ints(free_pages, "free_pages", dev);
  const int32_t* fc = ints(free_count, "free_count", dev, {1});
  const c10::cuda::CUDAGuard guard(dev);
  Tensor out = empty({B}, at::kInt, dev), left = empty({1}, at::kInt, dev);
  check("rnb_kv_release",
        fns.kv_release(c_int(B, "requests"), c_int(cols, "columns"), c_int(page_size, "page_size"),
                       c_int(num_pages.value_or(INT32_MAX), "num_pages"), tp, lp, np, fp,
                       c_int(free_pages.numel(), "free_pages"), fc, static_cast<int32_t*>(out.data_ptr()),
                       static_cast<int32_t*>(left.data_ptr()), stream_of(dev)));
  return {out, left};
}

const void* norm_weight(const OptTensor& w, const char* name, at::ScalarType dt, at::Device dev, int64_t D) {
  if (!w) return nullptr;
  if (w->scalar_type() != dt || w->device() != dev || w->dim() != 1 || w->size(0) != D || !w->is_contiguous())
    refuse(name, " must be a contiguous ", dt, " tensor of ", D, " elements on ", dev);
  return w->data_ptr();
}

Tensor rope(const Tensor& q, const OptTensor& k, const OptTensor& v, const Tensor& positions, const Tensor& inv_freq,
            const OptTensor& slots, const OptTensor& k_cache, const OptTensor& v_cache,
            const std::optional<std::vector<int64_t>>& sections, bool interleaved, const OptTensor& q_norm,
            const OptTensor& k_norm, double eps, const OptTensor& out) {
  const at::Device dev = cuda_device(q, "q");
  if (q.dim() != 3) refuse("q must be [tokens, heads, head_dim]");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  const at::ScalarType dt = q.scalar_type();
  rnb_rope_desc d{};
  d.dtype = dtype_code(dt);
  if (d.dtype < 0) refuse("q must be bfloat16 or float16");
  if (inv_freq.scalar_type() != at::kFloat || inv_freq.device() != dev || !inv_freq.is_contiguous())
    refuse("inv_freq must be a contiguous float32 tensor on ", dev);
  const int64_t half = inv_freq.numel(), axes = sections ? static_cast<int64_t>(sections->size()) : 1;
  if (axes < 1 || axes > 4) refuse("sections must name one to four axes");
  const c10::cuda::CUDAGuard guard(dev);
  Tensor pos = positions;
  if (pos.scalar_type() == at::kLong) pos = pos.to(at::kInt);
  if (pos.dim() == 1 && pos.size(0) == T) {
    if (axes > 1) pos = pos.expand({axes, T}).contiguous();  // text: every axis at the token's position
  } else if (pos.dim() != 2 || pos.size(0) != axes || pos.size(1) != T) {
    refuse("positions must have shape [", axes, ", ", T, "] or [", T, "], not ", positions.sizes());
  }
  const int32_t* pp = ints(pos, "positions", dev);
  const void* qw = norm_weight(q_norm, "q_norm", dt, dev, D);
  const void* kw = norm_weight(k_norm, "k_norm", dt, dev, D);
  const Rows qr = rows(q, "q", dt, dev, {T, Hq, D});
  Rows kr, vr;
  rnb_kv_cache cache{};
  const int32_t* sp = nullptr;
  if (k_cache) {
    if (!k || !v || !v_cache || !slots) refuse("k, v, slots and both caches must be given together");
    cache = cache_of(*k_cache, *v_cache, dt, dev);
    if (cache.head_dim != D) refuse("q and the cache must have one head_dim");
    kr = rows(*k, "k", dt, dev, {T, cache.n_kv_heads, D});
    vr = rows(*v, "v", dt, dev, {T, cache.n_kv_heads, D});
    sp = ints(*slots, "slots", dev, {T});
  }
  Tensor o = output(out, {T, Hq, D}, dt, dev);
  if (T == 0) return o;
  d.T = c_int(T, "tokens"), d.n_q_heads = c_int(Hq, "heads"), d.n_kv_heads = cache.n_kv_heads;
  d.head_dim = c_int(D, "head_dim"), d.rot = c_int(2 * half, "inv_freq"), d.n_axes = static_cast<int>(axes);
  d.interleaved = interleaved;
  for (int64_t i = 0; i < axes; ++i) d.sections[i] = c_int(sections ? (*sections)[i] : half, "sections");
  d.eps = static_cast<float>(eps);
  d.q_token_stride = qr.token, d.q_head_stride = qr.head;
  d.k_token_stride = kr.token, d.k_head_stride = kr.head;
  d.v_token_stride = vr.token, d.v_head_stride = vr.head;
  check("rnb_rope_append",
        fns.rope_append(&d, qr.p, kr.p, vr.p, qw, kw, pp, static_cast<const float*>(inv_freq.data_ptr()), sp,
                        k_cache ? &cache : nullptr, o.data_ptr(), stream_of(dev)));
  return o;
}

py::object paged_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table,
                           const Tensor& seq_lens, const OptTensor& cu_q, std::optional<int64_t> max_q,
                           std::optional<double> scale, int64_t window, const OptTensor& gate, const OptTensor& out,
                           bool return_lse) {
  const at::Device dev = cuda_device(q, "q");
  if (q.dim() != 3) refuse("q must be [tokens, heads, head_dim]");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2);
  const at::ScalarType dt = q.scalar_type();
  const rnb_kv_cache cache = cache_of(k_cache, v_cache, dt, dev);
  if (cache.head_dim != D) refuse("q and the cache must have one head_dim");
  if (table.dim() != 2) refuse("table must be [requests, columns]");
  const int64_t B = table.size(0);
  const int32_t* tp = ints(table, "table", dev);
  const int32_t* sl = ints(seq_lens, "seq_lens", dev, {B});
  const int32_t* cu = nullptr;
  if (cu_q)
    cu = ints(*cu_q, "cu_q", dev, {B + 1});
  else if (T != B)
    refuse("without cu_q every request has one query row: q must have as many as table");
  const c10::cuda::CUDAGuard guard(dev);
  const Rows qr = rows(q, "q", dt, dev, {T, Hq, D});
  Rows gr;
  if (gate) gr = rows(*gate, "gate", dt, dev, {T, Hq, D});
  Tensor o = output(out, {T, Hq, D}, dt, dev);
  OptTensor lse;
  if (return_lse) lse = empty({T, Hq}, at::kFloat, dev);
  rnb_attn_desc d{};
  d.B = c_int(B, "requests"), d.T = c_int(T, "tokens"), d.n_q_heads = c_int(Hq, "heads");
  d.table_cols = c_int(table.size(1), "columns");
  d.max_q = cu ? c_int(max_q.value_or(0), "max_q") : max_q.value_or(0) < 0 ? -1 : 1;
  d.window = c_int(window, "window");
  d.scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(D)));
  d.q_token_stride = qr.token, d.q_head_stride = qr.head;
  d.gate_token_stride = gr.token, d.gate_head_stride = gr.head;
  size_t need = 0;
  check("rnb_paged_attention_workspace_size", fns.workspace_size(&d, &cache, &need));
  const Tensor ws = empty({static_cast<int64_t>(need)}, at::kByte, dev);
  check("rnb_paged_attention",
        fns.paged_attention(&d, &cache, qr.p, gr.p, tp, sl, cu, o.data_ptr(),
                            lse ? static_cast<float*>(lse->data_ptr()) : nullptr, ws.data_ptr(), need, stream_of(dev)));
  if (return_lse) return py::cast(std::make_tuple(o, *lse));
  return py::cast(o);
}

}  // namespace

PYBIND11_MODULE(_torch_calls, m) {
  m.def("bind", &bind);
  m.def("kv_plan", &kv_plan);
  m.def("kv_release", &kv_release);
  m.def("rope", &rope);
  m.def("paged_attention", &paged_attention);
}

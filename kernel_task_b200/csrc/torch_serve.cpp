// Torch binding of the serving operators (include/trring.h, tr_plan_step and what follows):
// argument checks, output tensors from torch's allocator, the caller's current stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <cmath>
#include <cstdlib>
#include <map>
#include <mutex>
#include <utility>

#include "torch_ext.h"

namespace py = pybind11;

namespace trr_torch {
namespace {

using OptTensor = c10::optional<at::Tensor>;

[[noreturn]] void refuse(const char* op, const std::string& why) {
  throw py::value_error(std::string(op) + ": " + why);
}

void need_cuda(const char* op, const char* name, const at::Tensor& t) {
  if (!t.is_cuda()) refuse(op, std::string(name) + " must be a CUDA tensor");
}
void need(const char* op, const char* name, const at::Tensor& t, at::ScalarType type, int64_t dims,
          const at::Tensor& like) {
  need_cuda(op, name, t);
  if (t.device() != like.device()) refuse(op, std::string(name) + " is on another device");
  if (t.scalar_type() != type)
    refuse(op, std::string(name) + " must be " + c10::toString(type));
  if (t.dim() != dims)
    refuse(op, std::string(name) + " must have " + std::to_string(dims) + " dimension(s)");
}
// a vector of `n` values, contiguous
void need_vector(const char* op, const char* name, const at::Tensor& t, at::ScalarType type,
                 int64_t n, const at::Tensor& like) {
  need(op, name, t, type, 1, like);
  if (t.size(0) != n)
    refuse(op, std::string(name) + " must have " + std::to_string(n) + " values");
  if (!t.is_contiguous()) refuse(op, std::string(name) + " must be contiguous");
}
void need_table(const char* op, const at::Tensor& t, int64_t requests, const at::Tensor& like) {
  need(op, "tables", t, at::kInt, 2, like);
  if (t.size(0) != requests)
    refuse(op, "tables must have " + std::to_string(requests) + " rows");
  if (t.numel() > 0 && t.size(1) > 1 && t.stride(1) != 1)
    refuse(op, "tables must be contiguous along a row");
}
// row stride of a 2-D tensor (that of a single row or an empty tensor is not used)
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

cudaStream_t current_stream(const at::Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

void check(int st, const char* what) {
  if (st != TR_OK) raise_status(st, what);
}

// The small outputs of a call.  As a rule they share one allocation (an allocation costs a
// microsecond of the host, a tensor on its storage a tenth); `apart`, for the registered torch
// ops, whose outputs may not share storage, each gets its own.
class Outputs {
 public:
  Outputs(int64_t bytes, const at::Tensor& like, bool apart) : options_(like.options()) {
    if (!apart) all_ = at::empty({bytes}, options_.dtype(at::kByte));
  }
  // n values of `type`, at byte `at` of the shared allocation
  at::Tensor take(int64_t at, int64_t n, at::ScalarType type) const {
    if (!all_.defined()) return at::empty({n}, options_.dtype(type));
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(all_.storage()), all_.key_set(), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return t;
  }

 private:
  at::TensorOptions options_;
  at::Tensor all_;
};

// ---- step plan
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> plan_step(
    const at::Tensor& lens, const at::Tensor& brings, const at::Tensor& tables,
    const at::Tensor& free_pages, const at::Tensor& free_count, int64_t page_size, int64_t tokens,
    bool inplace, bool apart) {
  const char* op = "plan_step";
  need(op, "lens", lens, at::kInt, 1, lens);
  const int64_t R = lens.size(0);
  need_vector(op, "lens", lens, at::kInt, R, lens);
  need_vector(op, "new", brings, at::kInt, R, lens);
  need_table(op, tables, R, lens);
  need(op, "free", free_pages, at::kInt, 1, lens);
  need_vector(op, "free", free_pages, at::kInt, free_pages.size(0), lens);
  need_vector(op, "free_count", free_count, at::kInt, 1, lens);
  if (page_size < 1 || page_size > INT32_MAX) refuse(op, "page_size must be positive");
  if (tokens < 0) refuse(op, "tokens must not be negative");
  if (tables.size(1) > INT32_MAX) refuse(op, "too many table columns");
  const c10::cuda::CUDAGuard guard(lens.device());
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  // slots, positions (from a multiple of 16 bytes on), starts, granted, lens, count
  const int64_t at_positions = (tokens * 8 + 15) / 16 * 16, at_starts = at_positions + tokens * 4;
  const Outputs outputs(at_starts + (3 * R + 2) * 4, lens, apart);
  const at::Tensor slots = outputs.take(0, tokens, at::kLong);
  const at::Tensor positions = outputs.take(at_positions, tokens, at::kInt);
  const at::Tensor starts = outputs.take(at_starts, R + 1, at::kInt);
  const at::Tensor granted = outputs.take(at_starts + (R + 1) * 4, R, at::kInt);
  const at::Tensor lens_out =
      inplace ? lens : outputs.take(at_starts + (2 * R + 1) * 4, R, at::kInt);
  const at::Tensor count_out =
      inplace ? free_count : outputs.take(at_starts + (3 * R + 1) * 4, 1, at::kInt);
  check(tr_plan_step(lens.data_ptr<int32_t>(), brings.data_ptr<int32_t>(), R,
                     tables.data_ptr<int32_t>(), row_stride(tables), (int32_t)tables.size(1),
                     free_pages.data_ptr<int32_t>(), free_pages.size(0),
                     free_count.data_ptr<int32_t>(), (int32_t)page_size, tokens,
                     slots.data_ptr<int64_t>(), positions.data_ptr<int32_t>(),
                     starts.data_ptr<int32_t>(), lens_out.data_ptr<int32_t>(),
                     granted.data_ptr<int32_t>(), count_out.data_ptr<int32_t>(),
                     current_stream(lens)),
        "tr_plan_step");
  return {slots, positions, starts, lens_out, granted, count_out};
}

void release_pages(const at::Tensor& lens, const at::Tensor& finished, const at::Tensor& tables,
                   const at::Tensor& free_pages, const at::Tensor& free_count,
                   int64_t page_size) {
  const char* op = "release_pages";
  need(op, "lens", lens, at::kInt, 1, lens);
  const int64_t R = lens.size(0);
  need_vector(op, "lens", lens, at::kInt, R, lens);
  need_vector(op, "finished", finished, at::kInt, R, lens);
  need_table(op, tables, R, lens);
  need(op, "free", free_pages, at::kInt, 1, lens);
  need_vector(op, "free", free_pages, at::kInt, free_pages.size(0), lens);
  need_vector(op, "free_count", free_count, at::kInt, 1, lens);
  if (page_size < 1 || page_size > INT32_MAX) refuse(op, "page_size must be positive");
  if (tables.size(1) > INT32_MAX) refuse(op, "too many table columns");
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const c10::cuda::CUDAGuard guard(lens.device());
  check(tr_release_pages(lens.data_ptr<int32_t>(), finished.data_ptr<int32_t>(), R,
                         tables.data_ptr<int32_t>(), row_stride(tables), (int32_t)tables.size(1),
                         free_pages.data_ptr<int32_t>(), free_pages.size(0),
                         free_count.data_ptr<int32_t>(), (int32_t)page_size,
                         current_stream(lens)),
        "tr_release_pages");
}

// ---- the paged cache
void need_pools(const char* op, const at::Tensor& k_pages, const at::Tensor& v_pages,
                const at::Tensor& like) {
  if (dtype_code(k_pages.scalar_type()) < 0)
    refuse(op, "k_pages must be float32, float16 or bfloat16");
  need(op, "k_pages", k_pages, k_pages.scalar_type(), 4, like);
  need(op, "v_pages", v_pages, k_pages.scalar_type(), 4, like);
  if (k_pages.sizes() != v_pages.sizes()) refuse(op, "k_pages and v_pages differ in shape");
  if (!k_pages.is_contiguous() || !v_pages.is_contiguous())
    refuse(op, "k_pages and v_pages must be contiguous");
  if (k_pages.size(1) > INT32_MAX || k_pages.size(2) > INT32_MAX || k_pages.size(3) > INT32_MAX ||
      k_pages.size(1) < 1 || k_pages.size(2) < 1 || k_pages.size(3) < 1)
    refuse(op, "pools must be [pages, kv_heads, page_size, head_dim]");
}

void append_kv(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_pages,
               const at::Tensor& v_pages, const at::Tensor& slots) {
  const char* op = "append_kv";
  need_cuda(op, "k", k);
  need_pools(op, k_pages, v_pages, k);
  if (k.scalar_type() != k_pages.scalar_type() && k.scalar_type() != at::kFloat)
    refuse(op, "k and v must have the pools' dtype or be float32");
  need(op, "k", k, k.scalar_type(), 3, k);
  need(op, "v", v, k.scalar_type(), 3, k);
  if (k.sizes() != v.sizes() || k.size(1) != k_pages.size(1) || k.size(2) != k_pages.size(3))
    refuse(op, "k and v must be [tokens, " + std::to_string(k_pages.size(1)) + ", " +
                   std::to_string(k_pages.size(3)) + "]");
  need_vector(op, "slots", slots, at::kLong, k.size(0), k);
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const c10::cuda::CUDAGuard guard(k.device());
  const at::Tensor kc = k.stride(2) == 1 || k.size(2) == 1 ? k : k.contiguous();
  const at::Tensor vc = v.stride(2) == 1 || v.size(2) == 1 ? v : v.contiguous();
  check(tr_append_kv(kc.data_ptr(), kc.stride(0), kc.stride(1), vc.data_ptr(), vc.stride(0),
                     vc.stride(1), dtype_code(k.scalar_type()), k_pages.data_ptr(),
                     v_pages.data_ptr(), dtype_code(k_pages.scalar_type()),
                     slots.data_ptr<int64_t>(), k.size(0), (int32_t)k.size(1), (int32_t)k.size(2),
                     k_pages.size(0), (int32_t)k_pages.size(2), current_stream(k)),
        "tr_append_kv");
}

// The attention's workspace: one buffer per device and stream, its state zeroed when it is made
// and left ready by every call, so calls in one stream share it and calls in two streams do not
// meet in it.  While the stream is being captured a call gets a buffer of its own, whose zeroing
// is captured with it, because the graph may be replayed next to later calls on the stream.
at::Tensor new_workspace(int64_t bytes, const at::Tensor& like, cudaStream_t stream) {
  at::Tensor ws = at::empty({bytes}, like.options().dtype(at::kByte));
  check(tr_workspace_clear(ws.data_ptr(), TR_ATTENTION_STATE_BYTES, stream), "tr_workspace_clear");
  return ws;
}
std::mutex workspaces_lock;
std::map<std::pair<int, cudaStream_t>, at::Tensor>& workspaces() {
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();
  return *kept;
}
at::Tensor attention_workspace(int64_t bytes, const at::Tensor& like, cudaStream_t stream) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &capture) != cudaSuccess)
    throw std::runtime_error("paged_attention: cudaStreamIsCapturing failed");
  if (capture != cudaStreamCaptureStatusNone) return new_workspace(bytes, like, stream);
  const std::lock_guard<std::mutex> hold(workspaces_lock);
  at::Tensor& ws = workspaces()[{like.get_device(), stream}];
  if (!ws.defined() || ws.numel() < bytes) ws = new_workspace(bytes, like, stream);
  return ws;
}

// TRR_CHECK_STATUS=1: after every call outside a capture, read the status word (a stream
// synchronisation) and raise if a bounded device-side wait gave up.  Debugging aid.
bool checks_status() {
  static const bool on = [] {
    const char* v = std::getenv("TRR_CHECK_STATUS");
    return v && v[0] == '1';
  }();
  return on;
}
// The status word of the stream's kept workspace; waits for the stream.  With `reset` a workspace
// that timed out is given up, and the next call starts from a new one: its counters are not valid
// any more.
int64_t attention_status(int64_t device, bool reset) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  at::Tensor ws;
  {
    const std::lock_guard<std::mutex> hold(workspaces_lock);
    const auto kept = workspaces().find({(int)device, stream});
    if (kept == workspaces().end()) return TR_OK;
    ws = kept->second;
  }
  int32_t status = TR_OK;
  check(tr_workspace_status(ws.data_ptr(), ws.numel(), &status, 0, stream), "tr_workspace_status");
  if (status != TR_OK && reset) {
    const std::lock_guard<std::mutex> hold(workspaces_lock);
    const auto kept = workspaces().find({(int)device, stream});
    if (kept != workspaces().end() && kept->second.is_same(ws)) workspaces().erase(kept);
  }
  return status;
}
void check_status(const at::Tensor& like, cudaStream_t stream) {
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &capture) != cudaSuccess ||
      capture != cudaStreamCaptureStatusNone)
    return;
  const int64_t status = attention_status(like.get_device(), true);
  if (status != TR_OK)
    throw std::runtime_error(std::string("paged_attention: ") + tr_status_string((int)status) +
                             " (the call's output is not valid)");
}

// Polls of a wait before it gives up (0: the built-in limit), for tests of the timeout path.
std::atomic<uint32_t> attention_polls{0};

std::pair<at::Tensor, OptTensor> paged_attention(const at::Tensor& q, const at::Tensor& k_pages,
                                                 const at::Tensor& v_pages,
                                                 const at::Tensor& tables, const at::Tensor& lens,
                                                 const at::Tensor& starts,
                                                 c10::optional<double> scale, bool return_lse) {
  const char* op = "paged_attention";
  need_cuda(op, "q", q);
  need_pools(op, k_pages, v_pages, q);
  need(op, "q", q, k_pages.scalar_type(), 3, q);
  need(op, "lens", lens, at::kInt, 1, q);
  const int64_t R = lens.size(0), T = q.size(0), H = q.size(1), D = q.size(2);
  if (D != k_pages.size(3) || H < 1 || H % k_pages.size(1))
    refuse(op, "q must be [tokens, heads, " + std::to_string(k_pages.size(3)) +
                   "] with heads a multiple of " + std::to_string(k_pages.size(1)));
  need_vector(op, "lens", lens, at::kInt, R, q);
  need_vector(op, "starts", starts, at::kInt, R + 1, q);
  need_table(op, tables, R, q);
  if (H > INT32_MAX || tables.size(1) > INT32_MAX) refuse(op, "shape too large");
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)D);
  if (!(s > 0) || !std::isfinite((float)s)) refuse(op, "scale must be positive and finite");
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const c10::cuda::CUDAGuard guard(q.device());
  // heads of the last axis contiguous and 16-byte aligned, or a copy that is
  const int64_t es = q.element_size();
  const bool fine = q.stride(2) == 1 && ((uintptr_t)q.data_ptr() & 15) == 0 &&
                    (q.stride(0) * es) % 16 == 0 && (q.stride(1) * es) % 16 == 0;
  const at::Tensor qc = fine ? q : q.clone(at::MemoryFormat::Contiguous);
  at::Tensor out = at::empty({T, H, D}, q.options());
  at::Tensor lse;
  if (return_lse) lse = at::empty({T, H}, q.options().dtype(at::kFloat));
  tr_attention a = {};
  a.q = qc.data_ptr();
  a.q_token_stride = qc.stride(0);
  a.q_head_stride = qc.stride(1);
  a.k_pages = k_pages.data_ptr();
  a.v_pages = v_pages.data_ptr();
  a.tables = tables.data_ptr<int32_t>();
  a.table_stride = row_stride(tables);
  a.lens = lens.data_ptr<int32_t>();
  a.starts = starts.data_ptr<int32_t>();
  a.out = out.data_ptr();
  a.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  a.tokens = T;
  a.requests = R;
  a.pages = k_pages.size(0);
  a.columns = (int32_t)tables.size(1);
  a.page_size = (int32_t)k_pages.size(2);
  a.heads = (int32_t)H;
  a.kv_heads = (int32_t)k_pages.size(1);
  a.head_dim = (int32_t)D;
  a.dtype = dtype_code(q.scalar_type());
  a.scale = (float)s;
  a.wait_polls = attention_polls.load(std::memory_order_relaxed);
  size_t bytes = 0;
  check(tr_attention_workspace_bytes(&a, &bytes), "tr_paged_attention");
  cudaStream_t stream = current_stream(q);
  at::Tensor ws;
  if (bytes) ws = attention_workspace((int64_t)bytes, q, stream);
  check(tr_paged_attention(&a, bytes ? ws.data_ptr() : nullptr, bytes ? ws.numel() : 0, stream),
        "tr_paged_attention");
  if (bytes && checks_status()) check_status(q, stream);
  if (!return_lse) return {out, c10::nullopt};
  return {out, lse};
}

// ---- norms
const void* parameter(const char* op, const char* name, const OptTensor& t, int64_t width,
                      const at::Tensor& like) {
  if (!t.has_value()) return nullptr;
  need_vector(op, name, *t, like.scalar_type(), width, like);
  return t->data_ptr();
}

std::pair<OptTensor, OptTensor> residual_norm(const OptTensor& y, const at::Tensor& h,
                                              const OptTensor& post, const OptTensor& pre,
                                              const OptTensor& gate, const OptTensor& post_bias,
                                              const OptTensor& pre_bias, const std::string& kind,
                                              double eps, double residual_scale,
                                              double branch_scale) {
  const char* op = "residual_norm";
  if (dtype_code(h.scalar_type()) < 0) refuse(op, "h must be float32, float16 or bfloat16");
  need(op, "h", h, h.scalar_type(), 2, h);
  const int64_t T = h.size(0), W = h.size(1);
  if (W < 1) refuse(op, "h must have columns");
  tr_norm n = {};
  if (kind == "rms") n.kind = TR_NORM_RMS;
  else if (kind == "layer") n.kind = TR_NORM_LAYER;
  else refuse(op, "kind must be \"rms\" or \"layer\"");
  if (!y.has_value() && !pre.has_value()) refuse(op, "neither y nor pre");
  if (!y.has_value() && (post.has_value() || gate.has_value()))
    refuse(op, "post and gate need y");
  if ((post_bias.has_value() && !post.has_value()) || (pre_bias.has_value() && !pre.has_value()))
    refuse(op, "a bias needs its weight");
  if (!(eps >= 0)) refuse(op, "eps must not be negative");
  n.post = parameter(op, "post", post, W, h);
  n.pre = parameter(op, "pre", pre, W, h);
  n.post_bias = parameter(op, "post_bias", post_bias, W, h);
  n.pre_bias = parameter(op, "pre_bias", pre_bias, W, h);
  const auto rows = [&](const char* name, const at::Tensor& t) {
    if (t.dim() != 2 || t.size(0) != T || t.size(1) != W)
      refuse(op, std::string(name) + " must be [" + std::to_string(T) + ", " + std::to_string(W) +
                     "]");
    return W > 1 && t.stride(1) != 1 ? t.contiguous() : t;
  };
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const c10::cuda::CUDAGuard guard(h.device());
  at::Tensor hc = rows("h", h), yc, gc;
  n.h = hc.data_ptr();
  n.h_stride = row_stride(hc);
  if (y.has_value()) {
    if (y->scalar_type() != h.scalar_type() && y->scalar_type() != at::kFloat)
      refuse(op, "y must have h's dtype or be float32");
    need(op, "y", *y, y->scalar_type(), 2, h);
    yc = rows("y", *y);
    n.y = yc.data_ptr();
    n.y_stride = row_stride(yc);
    n.y_dtype = dtype_code(yc.scalar_type());
  }
  if (gate.has_value()) {
    if (gate->dim() == 1) {
      n.gate = parameter(op, "gate", gate, W, h);
      n.gate_stride = 0;
    } else {
      need(op, "gate", *gate, h.scalar_type(), 2, h);
      gc = rows("gate", *gate);
      n.gate = gc.data_ptr();
      n.gate_stride = row_stride(gc);
    }
  }
  OptTensor h_out, x_out;
  if (y.has_value()) {
    h_out = at::empty({T, W}, h.options());
    n.h_out = h_out->data_ptr();
  }
  if (pre.has_value()) {
    x_out = at::empty({T, W}, h.options());
    n.x_out = x_out->data_ptr();
  }
  n.tokens = T;
  n.width = W;
  n.dtype = dtype_code(h.scalar_type());
  n.eps = (float)eps;
  n.residual_scale = (float)residual_scale;
  n.branch_scale = (float)branch_scale;
  check(tr_residual_norm(&n, current_stream(h)), "tr_residual_norm");
  if (!y.has_value()) h_out = h;
  return {h_out, x_out};
}

// ---- sampling
std::pair<at::Tensor, at::Tensor> sample_tokens(const at::Tensor& logits, const at::Tensor& noise,
                                                const at::Tensor& temperature,
                                                const OptTensor& top_k, const OptTensor& top_p,
                                                const OptTensor& min_p, bool apart) {
  const char* op = "sample_tokens";
  if (dtype_code(logits.scalar_type()) < 0)
    refuse(op, "logits must be float32, float16 or bfloat16");
  need(op, "logits", logits, logits.scalar_type(), 2, logits);
  need(op, "noise", noise, at::kFloat, 2, logits);
  const int64_t R = logits.size(0), V = logits.size(1);
  if (V < 1) refuse(op, "logits must have columns");
  if (noise.sizes() != logits.sizes()) refuse(op, "noise must have the shape of logits");
  need_vector(op, "temperature", temperature, at::kFloat, R, logits);
  if (top_k.has_value()) need_vector(op, "top_k", *top_k, at::kInt, R, logits);
  if (top_p.has_value()) need_vector(op, "top_p", *top_p, at::kFloat, R, logits);
  if (min_p.has_value()) need_vector(op, "min_p", *min_p, at::kFloat, R, logits);
  const at::AutoDispatchBelowADInplaceOrView no_grad;
  const c10::cuda::CUDAGuard guard(logits.device());
  const at::Tensor lc = V > 1 && logits.stride(1) != 1 ? logits.contiguous() : logits;
  const at::Tensor nc = V > 1 && noise.stride(1) != 1 ? noise.contiguous() : noise;
  const Outputs outputs(R * 12, logits, apart);
  const at::Tensor tokens = outputs.take(0, R, at::kLong);
  const at::Tensor logprobs = outputs.take(R * 8, R, at::kFloat);
  check(tr_sample(lc.data_ptr(), dtype_code(lc.scalar_type()), row_stride(lc),
                  nc.data_ptr<float>(), row_stride(nc), temperature.data_ptr<float>(),
                  top_k.has_value() ? top_k->data_ptr<int32_t>() : nullptr,
                  top_p.has_value() ? top_p->data_ptr<float>() : nullptr,
                  min_p.has_value() ? min_p->data_ptr<float>() : nullptr, R, V,
                  tokens.data_ptr<int64_t>(), logprobs.data_ptr<float>(), current_stream(logits)),
        "tr_sample");
  return {tokens, logprobs};
}

}  // namespace

void bind_serving(py::module_& m) {
  m.def("plan_step", &plan_step, py::arg("lens"), py::arg("new"), py::arg("tables"),
        py::arg("free"), py::arg("free_count"), py::arg("page_size"), py::arg("tokens"),
        py::arg("inplace") = false, py::arg("apart") = false);
  m.def("release_pages", &release_pages, py::arg("lens"), py::arg("finished"), py::arg("tables"),
        py::arg("free"), py::arg("free_count"), py::arg("page_size"));
  m.def("append_kv", &append_kv, py::arg("k"), py::arg("v"), py::arg("k_pages"),
        py::arg("v_pages"), py::arg("slots"));
  m.def("paged_attention", &paged_attention, py::arg("q"), py::arg("k_pages"), py::arg("v_pages"),
        py::arg("tables"), py::arg("lens"), py::arg("starts"), py::arg("scale") = py::none(),
        py::arg("return_lse") = false);
  m.def("attention_status", &attention_status, py::arg("device"), py::arg("reset"));
  m.def("set_attention_wait_limit", [](uint32_t polls) { attention_polls.store(polls); },
        py::arg("polls"));
  m.def("residual_norm", &residual_norm, py::arg("y"), py::arg("h"), py::arg("post"),
        py::arg("pre"), py::arg("gate"), py::arg("post_bias"), py::arg("pre_bias"),
        py::arg("kind"), py::arg("eps"), py::arg("residual_scale"), py::arg("branch_scale"));
  m.def("sample_tokens", &sample_tokens, py::arg("logits"), py::arg("noise"),
        py::arg("temperature"), py::arg("top_k") = py::none(), py::arg("top_p") = py::none(),
        py::arg("min_p") = py::none(), py::arg("apart") = false);
}

}  // namespace trr_torch

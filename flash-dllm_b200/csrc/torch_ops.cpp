// Torch binding of the quantised operators (8-bit products, appending to a
// paged cache, attention over the 4-bit cache): checks of the arguments,
// outputs, workspaces and the current stream, in front of the C ABI.
//
// The calls are made per layer and per token, and several of the kernels run
// for a few microseconds, so the host's share counts: the same checks through
// Python and a foreign-function call of 22 arguments took 20 us a call, here
// 3 to 4.
//
// Errors: ValueError for shapes, strides and devices, TypeError for types,
// FdllmError for a status of the library (the class is registered by ops.py).
// Every call runs on the device of its tensors, on torch's current stream
// there.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <optional>
#include <tuple>
#include <vector>

#include "flashdllm_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kHead = 128, kPage = 64, kBlock = 4352;
constexpr size_t kGemmFlagBytes = 4096;

py::handle g_error;  // FdllmError(name, code)

void check_status(const char* name, int rc) {
  if (rc == FDLLM_OK) return;
  py::object e = py::reinterpret_borrow<py::object>(g_error)(name, rc);
  PyErr_SetObject(g_error.ptr(), e.ptr());
  throw py::error_already_set();
}

// ------------------------------------------------------------- workspaces --
// Scratch of one stream, its first `zero` bytes zero.  Eager calls keep a
// buffer per (device, stream, tag).  A captured graph gets its own from its
// memory pool, cleared by a node of the graph, and so does every stream of one
// capture (its branches replay at the same time): two graphs, two branches of
// one, or a graph and an eager call never share one, and nothing has to run
// before the capture.  The clearing node is on the branch that uses the
// buffer.  (Buffers that were outgrown stay allocated: work of their stream
// may still use them.)
class Workspaces {
 public:
  void* get(const at::Device& dev, cudaStream_t stream, const char* tag, size_t bytes, size_t zero, size_t* size) {
    *size = 0;
    if (bytes == 0) return nullptr;
    uint64_t capture = 0;
    check_status("fdllm_stream_capture_id", fdllm_stream_capture_id(stream, &capture));
    std::lock_guard<std::mutex> lock(mu_);
    const auto opts = at::TensorOptions().dtype(at::kByte).device(dev);
    Tensor* buf;
    if (capture == 0) {
      buf = &eager_[{dev.index(), stream, tag}];
      if (!buf->defined() || static_cast<size_t>(buf->numel()) < bytes) {
        size_t n = std::max<size_t>(bytes, 1 << 16);
        if (buf->defined()) {
          n = std::max<size_t>(n, static_cast<size_t>(buf->numel()) * 3 / 2);
          retired_.push_back(*buf);
        }
        *buf = at::zeros({static_cast<int64_t>(n)}, opts);
      }
    } else {
      const Captured key{capture, dev.index(), stream, tag};
      const auto held = captured_.find(key);
      if (held == captured_.end() || static_cast<size_t>(held->second.back().numel()) < bytes) {
        // captures long ended: their memory belongs to their graphs' pools
        while (captured_.size() > 64 && std::get<0>(captured_.begin()->first) < capture)
          captured_.erase(captured_.begin());
        Tensor t = at::empty({static_cast<int64_t>(std::max<size_t>(bytes, 256))}, opts);
        if (zero > 0) t.narrow(0, 0, static_cast<int64_t>(zero)).zero_();
        captured_[key].push_back(t);
      }
      buf = &captured_[key].back();
    }
    *size = static_cast<size_t>(buf->numel());
    return buf->data_ptr();
  }
  // After a device error left flags or counters set: zeros, once nothing that
  // runs on any stream uses them, and before anything else does.
  void rezero() {
    std::lock_guard<std::mutex> lock(mu_);
    for (auto& kv : eager_) {
      const c10::cuda::CUDAGuard guard(kv.second.device());
      C10_CUDA_CHECK(cudaDeviceSynchronize());
      kv.second.zero_();
      C10_CUDA_CHECK(cudaDeviceSynchronize());
    }
  }
  void clear() {
    std::lock_guard<std::mutex> lock(mu_);
    eager_.clear();
    captured_.clear();
    retired_.clear();
  }

 private:
  std::mutex mu_;
  std::map<std::tuple<int, cudaStream_t, std::string>, Tensor> eager_;
  using Captured = std::tuple<uint64_t, int, cudaStream_t, std::string>;  // (ordered by capture first)
  std::map<Captured, std::vector<Tensor>> captured_;
  std::vector<Tensor> retired_;
};

Workspaces& workspaces() {
  static Workspaces* w = new Workspaces();  // (not destroyed: tensors must not outlive the CUDA context's end)
  return *w;
}

// ----------------------------------------------------------------- checks --
struct Call {
  const Tensor& t;
  c10::cuda::OptionalCUDAGuard guard;
  cudaStream_t stream = nullptr;
  Call(const Tensor& first, const char* name) : t(first) {
    TORCH_CHECK_VALUE(first.is_cuda(), name, ": the tensors must be CUDA tensors (no CPU path)");
    guard.set_device(first.device());
    stream = c10::cuda::getCurrentCUDAStream(first.device().index()).stream();
  }
  void same(const Tensor& o, const char* name) const {
    TORCH_CHECK_VALUE(o.device() == t.device(), name, " must be on ", t.device(), ", got ", o.device());
  }
  // contiguous, of a type and a number of dimensions
  void plain(const Tensor& o, const char* name, at::ScalarType type, int64_t dim) const {
    same(o, name);
    TORCH_CHECK_TYPE(o.scalar_type() == type, name, " must be ", type, ", got ", o.scalar_type());
    TORCH_CHECK_VALUE(dim < 0 || o.dim() == dim, name, " must be ", dim, "-D, got shape ", o.sizes());
    TORCH_CHECK_VALUE(o.is_contiguous(), name, " must be contiguous");
  }
  // bf16 rows with unit column stride; returns the row stride
  int64_t rows(const Tensor& o, const char* name, int64_t n_rows, int64_t cols) const {
    same(o, name);
    TORCH_CHECK_TYPE(o.scalar_type() == at::kBFloat16, name, " must be bfloat16, got ", o.scalar_type());
    TORCH_CHECK_VALUE(o.dim() == 2, name, " must be 2-D, got shape ", o.sizes());
    TORCH_CHECK_VALUE((n_rows < 0 || o.size(0) == n_rows) && (cols < 0 || o.size(1) == cols), name, " must be [", n_rows,
                      ", ", cols, "], got ", o.sizes());
    TORCH_CHECK_VALUE(o.size(1) <= 1 || o.stride(1) == 1, name, " must have unit column stride");
    const int64_t ld = o.size(0) > 1 ? o.stride(0) : std::max<int64_t>(o.size(1), 1);
    TORCH_CHECK_VALUE(ld >= o.size(1) && ld % 8 == 0 && reinterpret_cast<uintptr_t>(o.data_ptr()) % 16 == 0, name,
                      ": rows must not overlap and must start on 16-byte boundaries");
    return ld;
  }
};

// Bytes of `rows` rows of `width` at a stride; a contiguous tensor is one row.
struct Span {
  int64_t at, rows, stride, width;
};
Span span(const Tensor& t) { return {reinterpret_cast<int64_t>(t.data_ptr()), 1, 0, static_cast<int64_t>(t.nbytes())}; }
Span span(const Tensor& t, int64_t ld) {
  const int64_t size = t.element_size(), width = t.size(1) * size;
  if (ld == t.size(1)) return span(t);
  return {reinterpret_cast<int64_t>(t.data_ptr()), t.size(0), ld * size, width};
}
// Whether two of them share a byte (with different strides: whether their
// ranges meet).  Rows of one tensor do not overlap.
bool meet(const Span& a, const Span& b) {
  if (a.rows == 0 || b.rows == 0 || a.width == 0 || b.width == 0) return false;
  const auto end = [](const Span& s) { return s.at + (s.rows - 1) * s.stride + s.width; };
  if (end(a) <= b.at || end(b) <= a.at) return false;
  if (a.rows > 1 && b.rows == 1) return meet(b, a);
  if (a.rows > 1 && a.stride != b.stride) return true;
  if (b.rows == 1) return true;
  const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y != 0 && x < 0); };
  if (a.rows == 1) {  // the first row of b that ends behind a's begin
    const int64_t i = std::max<int64_t>(0, floor_div(a.at - b.at - b.width, b.stride) + 1);
    return i < b.rows && b.at + i * b.stride < a.at + a.width;
  }
  // b's row j begins `off` behind the begin of a's row k + j
  const int64_t k = floor_div(b.at - a.at, a.stride), off = b.at - a.at - k * a.stride;
  const auto any = [&](int64_t k0) { return std::max<int64_t>(0, -k0) <= std::min(b.rows - 1, a.rows - 1 - k0); };
  return (off < a.width && any(k)) || (off + b.width > a.stride && any(k + 1));
}

// (the allocator itself: at::empty's way through the dispatcher costs as much
// again as the allocation, at up to three outputs a call)
Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

int32_t i32(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v >= 0 && v <= INT32_MAX, name, " is out of range: ", v);
  return static_cast<int32_t>(v);
}

void* opt_ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// ------------------------------------------------------------ 8-bit rows --
std::tuple<Tensor, Tensor> quantize_int8(const Tensor& x) {
  Call c(x, "quantize_int8");
  const int64_t ld = c.rows(x, "x", -1, -1);
  Tensor codes = empty(x.sizes(), at::kChar, x);
  Tensor scale = empty({x.size(0)}, at::kFloat, x);
  check_status("fdllm_quantize_int8",
               fdllm_quantize_int8(x.data_ptr(), ld, codes.data_ptr(), static_cast<float*>(scale.data_ptr()),
                                   i32(x.size(0), "rows"), i32(x.size(1), "dim"), c.stream));
  return {codes, scale};
}

std::tuple<Tensor, Tensor> rmsnorm_int8(const Tensor& x, const Tensor& weight, double eps) {
  Call c(x, "rmsnorm_int8");
  c.plain(x, "x", at::kBFloat16, 2);
  c.plain(weight, "weight", at::kBFloat16, 1);
  TORCH_CHECK_VALUE(weight.size(0) == x.size(1), "weight must have ", x.size(1), " values, got ", weight.size(0));
  Tensor codes = empty(x.sizes(), at::kChar, x);
  Tensor scale = empty({x.size(0)}, at::kFloat, x);
  check_status("fdllm_rmsnorm_int8",
               fdllm_rmsnorm_int8(x.data_ptr(), weight.data_ptr(), codes.data_ptr(),
                                  static_cast<float*>(scale.data_ptr()), i32(x.size(0), "rows"),
                                  i32(x.size(1), "dim"), static_cast<float>(eps), c.stream));
  return {codes, scale};
}

// -------------------------------------------------------- 8-bit products --
struct Int8Shape {
  int32_t rows, n, k;
};
Int8Shape int8_operands(const Call& c, const Tensor& a, const Tensor& a_scale, const Tensor& w,
                        const Tensor& w_scale) {
  c.plain(a, "a", at::kChar, 2);
  c.plain(w, "w", at::kChar, 2);
  c.plain(a_scale, "a_scale", at::kFloat, 1);
  c.plain(w_scale, "w_scale", at::kFloat, 1);
  TORCH_CHECK_VALUE(a.size(1) == w.size(1), "shapes ", a.sizes(), " x ", w.sizes(), "^T do not match");
  TORCH_CHECK_VALUE(a_scale.size(0) == a.size(0) && w_scale.size(0) == w.size(0), "scales must be [", a.size(0),
                    "] and [", w.size(0), "], got ", a_scale.sizes(), " and ", w_scale.sizes());
  return {i32(a.size(0), "rows"), i32(w.size(0), "n"), i32(a.size(1), "k")};
}

Tensor linear_int8(const Tensor& a, const Tensor& a_scale, const Tensor& w, const Tensor& w_scale,
                   const OptTensor& residual, const OptTensor& out) {
  Call c(a, "linear_int8");
  const Int8Shape s = int8_operands(c, a, a_scale, w, w_scale);
  const int64_t ld_res = residual.has_value() ? c.rows(*residual, "residual", s.rows, s.n) : 0;
  Tensor y = out.has_value() ? *out : empty({s.rows, s.n}, at::kBFloat16, a);
  const int64_t ld_out = out.has_value() ? c.rows(y, "out", s.rows, s.n) : s.n;
  if (out.has_value()) {
    const Span o = span(y, ld_out);
    for (const Tensor* t : {&a, &a_scale, &w, &w_scale})
      TORCH_CHECK_VALUE(!meet(o, span(*t)), "out must not overlap the operands");
    if (residual.has_value()) {  // (the residual itself: a value is read by the thread that writes it)
      const bool itself = y.data_ptr() == residual->data_ptr() && ld_out == ld_res;
      TORCH_CHECK_VALUE(itself || !meet(o, span(*residual, ld_res)), "out must not overlap the residual, unless it is it");
    }
  }
  size_t size = 0;
  void* ws = workspaces().get(a.device(), c.stream, "int8", fdllm_gemm_int8_workspace_bytes(s.rows, s.n, s.k, 0),
                              kGemmFlagBytes, &size);
  check_status("fdllm_gemm_int8",
               fdllm_gemm_int8(a.data_ptr(), static_cast<const float*>(a_scale.data_ptr()), w.data_ptr(),
                               static_cast<const float*>(w_scale.data_ptr()), y.data_ptr(), opt_ptr(residual), s.rows,
                               s.n, s.k, ld_out, ld_res, ws, size, c.stream));
  return y;
}

Tensor linear_swiglu_int8(const Tensor& a, const Tensor& a_scale, const Tensor& w, const Tensor& w_scale) {
  Call c(a, "linear_swiglu_int8");
  const Int8Shape s = int8_operands(c, a, a_scale, w, w_scale);
  TORCH_CHECK_VALUE(s.n % 2 == 0, "w_gate_up must be [2H, K]");
  Tensor y = empty({s.rows, s.n / 2}, at::kBFloat16, a);
  size_t size = 0;
  void* ws = workspaces().get(a.device(), c.stream, "int8", fdllm_gemm_int8_workspace_bytes(s.rows, s.n, s.k, 1),
                              kGemmFlagBytes, &size);
  check_status("fdllm_gemm_swiglu_int8",
               fdllm_gemm_swiglu_int8(a.data_ptr(), static_cast<const float*>(a_scale.data_ptr()), w.data_ptr(),
                                      static_cast<const float*>(w_scale.data_ptr()), y.data_ptr(), s.rows, s.n / 2,
                                      s.k, s.n / 2, ws, size, c.stream));
  return y;
}

// ---------------------------------------------------------- paged caches --
// pages of a 4-bit cache pair
int64_t int4_pages(const Call& c, const Tensor& k, const Tensor& v, int64_t n_kv) {
  c.plain(k, "k_cache", at::kByte, 3);
  c.plain(v, "v_cache", at::kByte, 3);
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(1) == n_kv && k.size(2) == kBlock,
                    "4-bit caches must both be [pages, ", n_kv, ", ", kBlock, "], got ", k.sizes(), " and ", v.sizes());
  return k.size(0);
}

struct Pages {
  const int32_t* table = nullptr;
  int32_t batch = 0, per_seq = 0;
};
Pages page_table(const Call& c, const OptTensor& t, int64_t seqlen_max) {
  TORCH_CHECK_VALUE(seqlen_max > 0 && seqlen_max <= INT32_MAX, "seqlen_max must be positive");
  Pages p;
  if (!t.has_value()) {
    TORCH_CHECK_VALUE(seqlen_max % kPage == 0, "without a page table seqlen_max must be a multiple of ", kPage);
    return p;
  }
  c.plain(*t, "page_table", at::kInt, 2);
  TORCH_CHECK_VALUE(t->size(0) > 0 && t->size(1) * kPage >= seqlen_max, "page_table must be [batch, at least ",
                    (seqlen_max + kPage - 1) / kPage, "], got ", t->sizes());
  p.table = static_cast<const int32_t*>(t->data_ptr());
  p.batch = i32(t->size(0), "batch");
  p.per_seq = i32(t->size(1), "pages");
  return p;
}

Tensor rope_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& slots, const OptTensor& sin,
                   const OptTensor& cos, const Tensor& k_cache, const Tensor& v_cache, int64_t n_heads,
                   int64_t n_kv_heads, int64_t seqlen_max, const OptTensor& table, const OptTensor& q_out) {
  Call c(q, "rope_append");
  c.plain(slots, "slots", at::kLong, 1);
  TORCH_CHECK_VALUE(n_heads > 0 && n_kv_heads > 0, "n_heads and n_kv_heads must be positive");
  const int64_t rows = slots.size(0);
  const int64_t ldq = c.rows(q, "q", rows, n_heads * kHead), ldk = c.rows(k, "k", rows, n_kv_heads * kHead),
                ldv = c.rows(v, "v", rows, n_kv_heads * kHead);
  const Pages pt = page_table(c, table, seqlen_max);
  int64_t n_pages;
  int bits;
  if (k_cache.scalar_type() == at::kByte) {
    bits = 4;
    n_pages = int4_pages(c, k_cache, v_cache, n_kv_heads);
  } else {
    bits = 16;
    c.plain(k_cache, "k_cache", at::kBFloat16, 2);
    c.plain(v_cache, "v_cache", at::kBFloat16, 2);
    TORCH_CHECK_VALUE(k_cache.sizes() == v_cache.sizes() && k_cache.size(1) == n_kv_heads * kHead &&
                          k_cache.size(0) % kPage == 0,
                      "bf16 caches must both be [pages * ", kPage, ", ", n_kv_heads * kHead, "], got ", k_cache.sizes(),
                      " and ", v_cache.sizes());
    n_pages = k_cache.size(0) / kPage;
  }
  TORCH_CHECK_VALUE(sin.has_value() == cos.has_value(), "sin and cos go together");
  if (sin.has_value()) {
    c.plain(*sin, "sin", at::kFloat, 2);
    c.plain(*cos, "cos", at::kFloat, 2);
    TORCH_CHECK_VALUE(sin->size(1) == kHead && cos->size(1) == kHead && sin->size(0) >= seqlen_max &&
                          cos->size(0) >= seqlen_max,
                      "sin and cos must be [at least ", seqlen_max, ", ", kHead, "], got ", sin->sizes(), " and ",
                      cos->sizes());
  }
  Tensor out;
  if (q_out.has_value()) {
    out = *q_out;
    c.plain(out, "q_out", at::kBFloat16, 2);
    TORCH_CHECK_VALUE(out.size(0) == rows && out.size(1) == n_heads * kHead, "q_out must be [", rows, ", ",
                      n_heads * kHead, "], got ", out.sizes());
  } else if (sin.has_value()) {
    out = empty({rows, n_heads * kHead}, at::kBFloat16, q);
  }
  // what is written overlaps nothing else, but for q_out, which may be q
  const Span ks = span(k_cache), vs = span(v_cache), in[] = {span(q, ldq), span(k, ldk), span(v, ldv)};
  TORCH_CHECK_VALUE(!meet(ks, vs), "k_cache and v_cache must not overlap");
  for (const Span& x : in)
    TORCH_CHECK_VALUE(!meet(ks, x) && !meet(vs, x), "q, k and v must not overlap the caches");
  if (out.defined() && q_out.has_value()) {
    const Span o = span(out);
    const bool itself = out.data_ptr() == q.data_ptr() && ldq == n_heads * kHead;
    TORCH_CHECK_VALUE((itself || !meet(o, in[0])) && !meet(o, in[1]) && !meet(o, in[2]) && !meet(o, ks) && !meet(o, vs),
                      "q_out must not overlap k, v or the caches, nor q, unless it is q");
  }
  check_status("fdllm_rope_append",
               fdllm_rope_append(q.data_ptr(), k.data_ptr(), v.data_ptr(), ldq, ldk, ldv,
                                 static_cast<const int64_t*>(slots.data_ptr()), static_cast<const float*>(opt_ptr(sin)),
                                 static_cast<const float*>(opt_ptr(cos)), out.defined() ? out.data_ptr() : nullptr,
                                 k_cache.data_ptr(), v_cache.data_ptr(), bits, i32(rows, "rows"),
                                 i32(n_heads, "n_heads"), i32(n_kv_heads, "n_kv_heads"),
                                 static_cast<int32_t>(seqlen_max), n_pages, pt.table, pt.batch, pt.per_seq, c.stream));
  return out.defined() ? out : q;
}

std::tuple<Tensor, Tensor> read_cache_int4(const Tensor& k_cache, const Tensor& v_cache, const Tensor& slots,
                                           int64_t seqlen_max, const OptTensor& table) {
  Call c(k_cache, "read_cache_int4");
  TORCH_CHECK_VALUE(k_cache.dim() == 3, "k_cache must be 3-D, got shape ", k_cache.sizes());
  const int64_t hk = k_cache.size(1);
  const int64_t n_pages = int4_pages(c, k_cache, v_cache, hk);
  c.plain(slots, "slots", at::kLong, 1);
  const Pages pt = page_table(c, table, seqlen_max);
  Tensor k = empty({slots.size(0), hk * kHead}, at::kBFloat16, slots);
  Tensor v = empty({slots.size(0), hk * kHead}, at::kBFloat16, slots);
  check_status("fdllm_read_cache_int4",
               fdllm_read_cache_int4(k_cache.data_ptr(), v_cache.data_ptr(),
                                     static_cast<const int64_t*>(slots.data_ptr()), k.data_ptr(), v.data_ptr(),
                                     i32(slots.size(0), "rows"), i32(hk, "kv heads"),
                                     static_cast<int32_t>(seqlen_max), n_pages, pt.table, pt.batch, pt.per_seq,
                                     c.stream));
  return {k, v};
}

void attn_cache_int4(const Tensor& q, const Tensor& o, const Tensor& k_cache, const Tensor& v_cache,
                     const Tensor& plan, int64_t capacity, const OptTensor& scores, double score_scale,
                     int64_t n_heads, int64_t n_kv_heads, int64_t seqlen_max, double softmax_scale, int64_t kv_splits,
                     int64_t rows_hint, const OptTensor& table) {
  Call c(q, "attn_cache_int4");
  c.plain(q, "q", at::kBFloat16, 2);
  c.plain(o, "o", at::kBFloat16, 2);
  TORCH_CHECK_VALUE(n_kv_heads > 0 && n_heads > 0 && n_heads % n_kv_heads == 0,
                    "n_heads must be a multiple of n_kv_heads");
  TORCH_CHECK_VALUE(q.size(1) == n_heads * kHead && o.sizes() == q.sizes(), "q and o must be [rows, ",
                    n_heads * kHead, "], got ", q.sizes(), " and ", o.sizes());
  // (scores sum all masked rows of q, rows that another CTA may have answered)
  const auto* q0 = static_cast<const char*>(q.data_ptr());
  const auto* o0 = static_cast<const char*>(o.data_ptr());
  TORCH_CHECK_VALUE(q.numel() == 0 || q0 + q.nbytes() <= o0 || o0 + o.nbytes() <= q0, "o must not overlap q");
  const int64_t n_pages = int4_pages(c, k_cache, v_cache, n_kv_heads);
  c.plain(plan, "plan", at::kInt, 1);
  const Pages pt = page_table(c, table, seqlen_max);
  // (a plan holds a header, its capacity in items and a record per sequence, 8 words each)
  const int64_t rows = q.size(0), n_seqs = plan.numel() / 8 - 1 - capacity;
  TORCH_CHECK_VALUE(plan.numel() % 8 == 0 && capacity > 0 && n_seqs > 0 && n_seqs <= capacity,
                    "plan and capacity are not of one plan_cache_attention");
  if (scores.has_value()) {
    c.plain(*scores, "attn_scores", at::kFloat, -1);
    TORCH_CHECK_VALUE(scores->numel() >= n_seqs * seqlen_max,
                      "attn_scores must be [batch * seqlen_max]");
  }
  const int32_t r = i32(rows, "rows"), cap = i32(capacity, "capacity"), seqs = i32(n_seqs, "sequences"), h = i32(n_heads, "n_heads"),
                hk = i32(n_kv_heads, "n_kv_heads"), len = static_cast<int32_t>(seqlen_max),
                splits = i32(kv_splits, "kv_splits"), hint = i32(rows_hint, "rows_hint");
  size_t scratch_bytes = 0, ws_size = 0, scratch_size = 0;
  const size_t ws_bytes =
      fdllm_attn_int4_workspace_bytes(r, cap, seqs, h, hk, len, splits, hint, scores.has_value(), &scratch_bytes);
  void* ws = workspaces().get(q.device(), c.stream, "attn4", ws_bytes, ws_bytes, &ws_size);
  void* scratch = workspaces().get(q.device(), c.stream, "attn4s", scratch_bytes, 0, &scratch_size);
  check_status("fdllm_attn_cache_int4",
               fdllm_attn_cache_int4(q.data_ptr(), o.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                     plan.data_ptr(), cap, seqs, static_cast<float*>(opt_ptr(scores)),
                                     static_cast<float>(score_scale), r, h, hk, len, n_pages,
                                     static_cast<float>(softmax_scale), splits, hint, pt.table, pt.batch, pt.per_seq,
                                     ws, ws_size, scratch, scratch_size, c.stream));
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("set_error_class", [](py::object cls) { g_error = cls.release(); });
  m.def("workspace_rezero", [] { workspaces().rezero(); });
  m.def("workspace_clear", [] { workspaces().clear(); });
  m.def("quantize_int8", &quantize_int8);
  m.def("rmsnorm_int8", &rmsnorm_int8);
  m.def("linear_int8", &linear_int8);
  m.def("linear_swiglu_int8", &linear_swiglu_int8);
  m.def("rope_append", &rope_append);
  m.def("read_cache_int4", &read_cache_int4);
  m.def("attn_cache_int4", &attn_cache_int4);
}

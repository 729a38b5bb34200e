// Host side of the operators on the 8-bit key/value cache: checks of the tensors, the C ABI's structs, the launch.
// In C++ for the same reason as the single-GPU calls (rswa_torch.cpp): a decoding step calls each of them once per layer,
// and through ctypes the host would need longer than the GPU.
//
// Every function returns False instead of doing anything where the device has no status word yet or an error of an
// earlier call has not been raised: Python sees to that and calls again.  Checks that need no device come first.
#include "rswa_torch.h"

#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <cstring>
#include <map>
#include <mutex>

#include "../../include/rswa.h"

namespace rswa_host {

namespace {

constexpr int64_t kIntMax = 0x7fffffff;

at::Tensor tensor_arg(PyObject* o, const char* what, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o) && THPVariable_CheckTypeExact(Py_TYPE(o)), what, ": ", name, " must be a torch.Tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
int64_t int_arg(PyObject* o, const char* what, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, what, ": ", name, " must be an integer");
  }
  return v;
}

// These operators have no derivative, and a trace or a transform would see only the allocation of their results.
void check_plain(const at::Tensor& t, const char* what, const char* name) {
  TORCH_CHECK(!(c10::GradMode::is_enabled() && t.requires_grad()), what, ": ", name,
              " requires a gradient, which this operator has none of: call it under torch.no_grad() or with a detached tensor");
  TORCH_CHECK(!t._fw_grad(0).defined(), what, ": no forward-mode derivative");
}
void check_mode(const char* what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, ": cannot be traced");
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode), what, ": no torch.func transforms");
}
void check_16bit(const at::Tensor& t, const char* what, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, what, ": ", name, " must be bfloat16 or float16, got ", t.scalar_type());
}
void check_device(const at::Tensor& t, const at::Tensor& like, const char* what, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.layout() == at::kStrided, what, ": ", name, " must be a CUDA tensor: ring_swa has no CPU path");
  TORCH_CHECK_VALUE(t.device() == like.device(), what, ": ", name, " is on ", t.device(), ", the cache on ", like.device());
}

struct Cache {
  at::Tensor k, v, ks, vs;
};
Cache cache_args(PyObject* const* args, const char* what) {
  Cache c = {tensor_arg(args[0], what, "cache.k"), tensor_arg(args[1], what, "cache.v"), tensor_arg(args[2], what, "cache.k_scale"),
             tensor_arg(args[3], what, "cache.v_scale")};
  TORCH_CHECK_VALUE(c.k.dim() == 4 && c.v.sizes() == c.k.sizes() && c.ks.dim() == 2 && c.ks.size(0) == c.k.size(0) && c.ks.size(1) == c.k.size(1) &&
                        c.vs.sizes() == c.ks.sizes(),
                    what, ": cache.k and cache.v must be [num_blocks, num_kv_heads, block_size, head_dim], the scales [num_blocks, num_kv_heads]");
  TORCH_CHECK_VALUE((c.k.scalar_type() == at::kChar || c.k.scalar_type() == at::kFloat8_e4m3fn) && c.v.scalar_type() == c.k.scalar_type() &&
                        c.ks.scalar_type() == at::kFloat && c.vs.scalar_type() == at::kFloat,
                    what, ": cache.k and cache.v must both be int8 or both float8_e4m3fn, the scales float32");
  for (const at::Tensor* t : {&c.k, &c.v, &c.ks, &c.vs}) TORCH_CHECK_VALUE(t->is_contiguous(), what, ": the cache's tensors must be contiguous");
  TORCH_CHECK_VALUE(c.k.numel() > 0 && c.k.size(0) <= kIntMax && c.k.size(1) <= kIntMax, what, ": the cache is empty or too large");
  TORCH_CHECK_VALUE((c.k.size(3) == 64 || c.k.size(3) == 128) && (c.k.size(2) == 16 || c.k.size(2) == 32 || c.k.size(2) == 64 || c.k.size(2) == 128), what,
                    ": head_dim must be 64 or 128 and block_size 16, 32, 64 or 128, got ", c.k.size(3), " and ", c.k.size(2));
  return c;
}
void check_cache_device(const Cache& c, const char* what) {
  for (const at::Tensor* t : {&c.k, &c.v, &c.ks, &c.vs}) check_device(*t, c.k, what, "the cache");
}
rswa_cache_t cache_struct(const Cache& c) {
  rswa_cache_t r;
  r.k = c.k.data_ptr(), r.v = c.v.data_ptr();
  r.k_scale = static_cast<float*>(c.ks.data_ptr()), r.v_scale = static_cast<float*>(c.vs.data_ptr());
  r.num_blocks = c.k.size(0);
  r.n_kv_heads = static_cast<int32_t>(c.k.size(1)), r.block_size = static_cast<int32_t>(c.k.size(2)), r.head_dim = static_cast<int32_t>(c.k.size(3));
  r.kind = c.k.scalar_type() == at::kChar ? RSWA_CACHE_INT8 : RSWA_CACHE_E4M3;
  return r;
}

// block table [batch, max_blocks] and lengths [batch]
void check_table(const at::Tensor& table, const at::Tensor& lens, int64_t block_size, const char* what, const char* name = "block_table") {
  TORCH_CHECK_VALUE(table.dim() == 2 && lens.dim() == 1 && lens.size(0) == table.size(0), what, ": ", name, " must be [batch, max_blocks] and lens [batch]");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt, what, ": ", name, " and lens must be int32");
  TORCH_CHECK_VALUE((table.size(1) <= 1 || table.stride(1) == 1) && (lens.size(0) <= 1 || lens.stride(0) == 1), what, ": rows of ", name,
                    " and lens must be contiguous");
  TORCH_CHECK_VALUE(table.size(0) <= kIntMax && table.size(1) <= kIntMax / block_size, what, ": ", name, " is too large");
}
rswa_block_table_t table_struct(const at::Tensor& table) {
  rswa_block_table_t t;
  t.entries = table.const_data_ptr<int32_t>();
  // (a row expanded over the batch is passed as it is; the library refuses it where blocks are written to)
  t.stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  t.batch = static_cast<int32_t>(table.size(0)), t.max_blocks = static_cast<int32_t>(table.size(1));
  return t;
}

// The kernels load 16 bytes at a time along the head dimension; through tensor maps they want positive strides besides.
at::Tensor loadable(const at::Tensor& t, bool map = false) {
  bool ok = (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 && t.stride(-1) == 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && (!map || t.stride(i) > 0)));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

int32_t dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? RSWA_DTYPE_BF16 : RSWA_DTYPE_FP16; }

bool ready(int dev) {
  if (status_word(dev) == nullptr) return false;
  if (!reported(dev)) return true;
  // an error cannot be raised and cleared inside a stream capture
  cudaStreamCaptureStatus st;
  return cudaStreamIsCapturing(c10::cuda::getCurrentCUDAStream(dev).stream(), &st) == cudaSuccess && st != cudaStreamCaptureStatusNone;
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The zeroed counters of rswa_cache_attn.  Calls on one of torch's streams follow one another and share them, for as long as the
// process lives.  Calls that are being captured (the graph may run beside anything), and those on streams that torch did not make,
// get their own, zeroed on the stream each time: a handle from elsewhere may be another stream for every thread, or be given to
// another stream while work of the one that had it still runs.  (torch identifies its own streams by numbers, those by the handle.)
at::Tensor counters(int dev, const at::TensorOptions& options) {
  const c10::cuda::CUDAStream current = c10::cuda::getCurrentCUDAStream(dev);
  const cudaStream_t stream = current.stream();
  const bool foreign = stream != nullptr && current.id() == static_cast<c10::StreamId>(reinterpret_cast<intptr_t>(stream));
  cudaStreamCaptureStatus st;
  if (foreign || cudaStreamIsCapturing(stream, &st) != cudaSuccess || st != cudaStreamCaptureStatusNone)
    return at::zeros({RSWA_CACHE_ATTN_COUNTERS}, options.dtype(at::kInt));
  static std::mutex mutex;
  static auto* kept = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();  // (never freed: the process may end before its streams do)
  const std::lock_guard<std::mutex> lock(mutex);
  at::Tensor& t = (*kept)[{dev, stream}];
  if (!t.defined()) t = at::zeros({RSWA_CACHE_ATTN_COUNTERS}, options.dtype(at::kInt));
  return t;
}

// accumulated weights [batch, num_kv_heads, >= tokens]
void check_weights(const at::Tensor& w, int64_t batch, int64_t heads, int64_t tokens, const char* what, const char* name) {
  TORCH_CHECK_VALUE(w.scalar_type() == at::kFloat && w.dim() == 3 && w.size(0) == batch && w.size(1) == heads && w.size(2) >= tokens, what, ": ", name,
                    " must be float32 [batch, num_kv_heads, at least max_blocks * block_size = ", tokens, "], got ", w.sizes());
  // rows apart in either order of sequences and heads
  const auto apart = [&](int inner, int outer) {
    return (w.size(inner) <= 1 || w.stride(inner) >= w.size(2)) &&
           (w.size(outer) <= 1 || w.stride(outer) >= (w.size(inner) - 1) * (w.size(inner) <= 1 ? 0 : w.stride(inner)) + w.size(2));
  };
  TORCH_CHECK_VALUE((w.size(2) <= 1 || w.stride(2) == 1) && (apart(1, 0) || apart(0, 1)), what, ": ", name,
                    " must be contiguous along the tokens, without rows that overlap");
}

}  // namespace

// cache_append(k_cache, v_cache, k_scale, v_scale, k, v, block_table, lens, cu_seqlens or None)
PyObject* py_cache_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "cache_append";
  TORCH_CHECK_TYPE(n == 9, what, " takes 9 arguments");
  const Cache c = cache_args(args, what);
  at::Tensor k = tensor_arg(args[4], what, "k"), v = tensor_arg(args[5], what, "v");
  const at::Tensor table = tensor_arg(args[6], what, "block_table"), lens = tensor_arg(args[7], what, "lens");
  const at::Tensor cu = args[8] == Py_None ? at::Tensor() : tensor_arg(args[8], what, "cu_seqlens");
  check_16bit(k, what, "k");
  TORCH_CHECK_VALUE(k.dim() == (cu.defined() ? 3 : 4), what, ": k must be ", cu.defined() ? "[tokens, num_kv_heads, head_dim] with" : "[batch, tokens, num_kv_heads, head_dim] without",
                    " cu_seqlens");
  TORCH_CHECK_VALUE(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), what, ": k and v must have the same shape and type");
  TORCH_CHECK_VALUE(k.size(-2) == c.k.size(1) && k.size(-1) == c.k.size(3), what, ": k has ", k.size(-2), " heads of ", k.size(-1), ", the cache ", c.k.size(1), " of ",
                    c.k.size(3));
  check_table(table, lens, c.k.size(2), what);
  if (cu.defined()) {
    TORCH_CHECK_VALUE(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.size(0) == table.size(0) + 1 && (cu.size(0) <= 1 || cu.stride(0) == 1), what,
                      ": cu_seqlens must be contiguous int32 [batch + 1]");
  } else {
    TORCH_CHECK_VALUE(k.size(0) == table.size(0), what, ": k has ", k.size(0), " sequences, block_table ", table.size(0));
  }
  TORCH_CHECK_VALUE(k.numel() / (k.size(-1) * k.size(-2)) <= kIntMax, what, ": too many tokens");
  check_plain(k, what, "k");
  check_plain(v, what, "v");
  check_mode(what);
  check_cache_device(c, what);
  check_device(k, c.k, what, "k"), check_device(v, c.k, what, "v"), check_device(table, c.k, what, "block_table"), check_device(lens, c.k, what, "lens");
  if (cu.defined()) check_device(cu, c.k, what, "cu_seqlens");
  const int dev = c.k.get_device();
  if (!ready(dev)) Py_RETURN_FALSE;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(c.k.device());
    k = loadable(k), v = loadable(v);
    rswa_cache_append_params_t p;
    std::memset(&p, 0, sizeof(p));
    p.cache = cache_struct(c);
    p.table = table_struct(table);
    p.lens = lens.const_data_ptr<int32_t>();
    p.dtype = dtype_code(k);
    const int64_t t = k.dim() - 3;  // the token dimension
    p.tokens = t == 0 ? k.size(0) : k.size(0) * k.size(1);
    p.cu_seqlens = cu.defined() ? cu.const_data_ptr<int32_t>() : nullptr;
    p.k = k.const_data_ptr(), p.v = v.const_data_ptr();
    p.k_stride_b = t == 0 ? 0 : stride_of(k, 0), p.k_stride_t = stride_of(k, t), p.k_stride_h = stride_of(k, t + 1);
    p.v_stride_b = t == 0 ? 0 : stride_of(v, 0), p.v_stride_t = stride_of(v, t), p.v_stride_h = stride_of(v, t + 1);
    p.status = status_word(dev);
    check(rswa_cache_append(&p, stream_of(dev)), what);
    for (const at::Tensor* w : {&c.k, &c.v, &c.ks, &c.vs}) written(*w);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// cache_read(k_cache, v_cache, k_scale, v_scale, block_table, lens, rows, bf16) -> (k, v)
PyObject* py_cache_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "cache_read";
  TORCH_CHECK_TYPE(n == 8, what, " takes 8 arguments");
  const Cache c = cache_args(args, what);
  const at::Tensor table = tensor_arg(args[4], what, "block_table"), lens = tensor_arg(args[5], what, "lens");
  const int64_t rows = int_arg(args[6], what, "max_len");
  const bool bf16 = PyObject_IsTrue(args[7]);
  check_table(table, lens, c.k.size(2), what);
  TORCH_CHECK_VALUE(rows >= 0 && rows <= kIntMax - 128, what, ": max_len must be non-negative, got ", rows);
  check_mode(what);
  check_cache_device(c, what);
  check_device(table, c.k, what, "block_table"), check_device(lens, c.k, what, "lens");
  const int dev = c.k.get_device();
  if (!ready(dev)) Py_RETURN_FALSE;
  at::Tensor k, v;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(c.k.device());
    const auto options = c.k.options().dtype(bf16 ? at::kBFloat16 : at::kHalf);
    k = at::empty({table.size(0), rows, c.k.size(1), c.k.size(3)}, options);
    v = at::empty(k.sizes(), options);
    rswa_cache_read_params_t p;
    std::memset(&p, 0, sizeof(p));
    p.cache = cache_struct(c);
    p.table = table_struct(table);
    p.lens = lens.const_data_ptr<int32_t>();
    p.dtype = dtype_code(k);
    p.rows = static_cast<int32_t>(rows);
    p.k = k.data_ptr(), p.v = v.data_ptr();
    p.status = status_word(dev);
    check(rswa_cache_read(&p, stream_of(dev)), what);
  }
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  END_HANDLE_TH_ERRORS
}

// cache_attn(k_cache, v_cache, k_scale, v_scale, q, block_table, lens, window or None, n_sink, scale or None, weights or None, want_lse)
//   -> out or (out, lse)
PyObject* py_cache_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "cache_attn";
  TORCH_CHECK_TYPE(n == 12, what, " takes 12 arguments");
  const Cache c = cache_args(args, what);
  at::Tensor q = tensor_arg(args[4], what, "q");
  const at::Tensor table = tensor_arg(args[5], what, "block_table"), lens = tensor_arg(args[6], what, "lens");
  int64_t window = -1;
  if (args[7] != Py_None) {
    window = int_arg(args[7], what, "window_size");
    TORCH_CHECK_VALUE(window >= 0, what, ": window_size must be non-negative, or None for every earlier token; got ", window);
  }
  const int64_t n_sink = int_arg(args[8], what, "num_sink_tokens");
  TORCH_CHECK_VALUE(n_sink >= 0, what, ": num_sink_tokens must be non-negative, got ", n_sink);
  const at::Tensor weights = args[10] == Py_None ? at::Tensor() : tensor_arg(args[10], what, "weights");
  const bool want_lse = PyObject_IsTrue(args[11]);
  check_16bit(q, what, "q");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == c.k.size(3), what, ": q must be [batch, queries, num_q_heads, ", c.k.size(3), "], got ", q.sizes());
  TORCH_CHECK_VALUE(q.size(2) > 0 && q.size(2) % c.k.size(1) == 0, what, ": Number of query heads must be divisible by number of key/value heads, got ", q.size(2),
                    " and ", c.k.size(1));
  double scale = 1. / std::sqrt(static_cast<double>(q.size(3)));
  if (args[9] != Py_None) {
    scale = PyFloat_AsDouble(args[9]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      TORCH_CHECK_TYPE(false, what, ": softmax_scale must be a number");
    }
  }
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0.f && std::isfinite(static_cast<float>(scale)), what, ": softmax_scale must be positive, got ", scale);
  check_table(table, lens, c.k.size(2), what);
  TORCH_CHECK_VALUE(q.size(0) == table.size(0), what, ": q has ", q.size(0), " sequences, block_table ", table.size(0));
  TORCH_CHECK_VALUE(q.size(1) <= 65536 && q.size(2) <= 65536, what, ": too many queries or heads");
  if (weights.defined()) check_weights(weights, table.size(0), c.k.size(1), table.size(1) * c.k.size(2), what, "weights");
  check_plain(q, what, "q");
  if (weights.defined()) check_plain(weights, what, "weights");
  check_mode(what);
  check_cache_device(c, what);
  check_device(q, c.k, what, "q"), check_device(table, c.k, what, "block_table"), check_device(lens, c.k, what, "lens");
  if (weights.defined()) check_device(weights, c.k, what, "weights");
  const int dev = c.k.get_device();
  if (!ready(dev)) Py_RETURN_FALSE;
  at::Tensor out, lse;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(c.k.device());
    q = loadable(q);
    out = at::empty(q.sizes(), q.options());
    if (want_lse || weights.defined()) lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    rswa_cache_attn_params_t p;
    std::memset(&p, 0, sizeof(p));
    p.cache = cache_struct(c);
    p.table = table_struct(table);
    p.lens = lens.const_data_ptr<int32_t>();
    p.dtype = dtype_code(q);
    p.q_len = static_cast<int32_t>(q.size(1)), p.n_q_heads = static_cast<int32_t>(q.size(2));
    p.window = window < 0 ? -1 : static_cast<int32_t>(std::min(window, kIntMax));
    p.n_sink = static_cast<int32_t>(std::min(n_sink, kIntMax));
    p.softmax_scale = static_cast<float>(scale);
    p.q = q.const_data_ptr();
    p.q_stride_b = stride_of(q, 0), p.q_stride_t = stride_of(q, 1), p.q_stride_h = stride_of(q, 2);
    p.out = out.data_ptr();
    p.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
    if (weights.defined()) {
      p.weights = weights.data_ptr<float>();
      p.w_stride_b = stride_of(weights, 0), p.w_stride_h = stride_of(weights, 1);
    }
    p.status = status_word(dev);
    const int64_t bytes = rswa_cache_attn_workspace_bytes(&p);
    if (bytes < 0) check(static_cast<int>(bytes), what);
    // (from the allocator of the current stream: a graph that captures the call keeps it, two calls never share it)
    const at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
    p.workspace = ws.data_ptr();
    p.workspace_bytes = bytes;
    const at::Tensor arrived = counters(dev, q.options());
    p.arrived = arrived.data_ptr<int32_t>();
    check(rswa_cache_attn(&p, stream_of(dev)), what);
    if (weights.defined()) written(weights);
  }
  if (!want_lse) return THPVariable_Wrap(out);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
  END_HANDLE_TH_ERRORS
}

// cache_evict(k_cache, v_cache, k_scale, v_scale, block_table, lens, weights, budget, new_block_table, n_sink, n_recent)
//   -> (new_lens, new_weights, kept)
PyObject* py_cache_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "cache_evict";
  TORCH_CHECK_TYPE(n == 11, what, " takes 11 arguments");
  const Cache c = cache_args(args, what);
  const at::Tensor table = tensor_arg(args[4], what, "block_table"), lens = tensor_arg(args[5], what, "lens");
  const at::Tensor weights = tensor_arg(args[6], what, "weights"), new_table = tensor_arg(args[8], what, "new_block_table");
  const int64_t budget = int_arg(args[7], what, "budget"), n_sink = int_arg(args[9], what, "num_sink_tokens"), n_recent = int_arg(args[10], what, "num_recent_tokens");
  const int64_t bs = c.k.size(2);
  check_table(table, lens, bs, what);
  check_table(new_table, lens, bs, what, "new_block_table");
  check_weights(weights, table.size(0), c.k.size(1), table.size(1) * bs, what, "weights");
  TORCH_CHECK_VALUE(budget > 0 && budget <= kIntMax, what, ": budget must be positive, got ", budget);
  TORCH_CHECK_VALUE(n_sink >= 0 && n_recent >= 0 && n_sink <= budget && n_recent <= budget - n_sink, what, ": num_sink_tokens (", n_sink, ") and num_recent_tokens (", n_recent,
                    ") must not be negative and fit into the budget of ", budget);
  TORCH_CHECK_VALUE(new_table.size(1) * bs >= std::min(budget, table.size(1) * bs), what, ": new_block_table holds ", new_table.size(1) * bs,
                    " tokens per sequence, but ", std::min(budget, table.size(1) * bs), " may stay");
  check_plain(weights, what, "weights");
  check_mode(what);
  check_cache_device(c, what);
  check_device(table, c.k, what, "block_table"), check_device(lens, c.k, what, "lens"), check_device(weights, c.k, what, "weights");
  check_device(new_table, c.k, what, "new_block_table");
  const int dev = c.k.get_device();
  if (!ready(dev)) Py_RETURN_FALSE;
  at::Tensor new_lens, new_weights, kept;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(c.k.device());
    new_lens = at::empty({table.size(0)}, lens.options());
    new_weights = at::empty({table.size(0), c.k.size(1), new_table.size(1) * bs}, weights.options());
    kept = at::empty({table.size(0), c.k.size(1), budget}, lens.options());
    rswa_cache_evict_params_t p;
    std::memset(&p, 0, sizeof(p));
    p.cache = cache_struct(c);
    p.table = table_struct(table);
    p.new_table = table_struct(new_table);
    p.lens = lens.const_data_ptr<int32_t>();
    p.weights = weights.const_data_ptr<float>();
    p.w_stride_b = stride_of(weights, 0), p.w_stride_h = stride_of(weights, 1);
    p.budget = static_cast<int32_t>(budget), p.n_sink = static_cast<int32_t>(n_sink), p.n_recent = static_cast<int32_t>(n_recent);
    p.new_w_len = static_cast<int32_t>(new_weights.size(2));
    p.new_lens = new_lens.data_ptr<int32_t>();
    p.new_weights = new_weights.data_ptr<float>();
    p.kept = kept.data_ptr<int32_t>();
    p.status = status_word(dev);
    check(rswa_cache_evict(&p, stream_of(dev)), what);
    for (const at::Tensor* w : {&c.k, &c.v, &c.ks, &c.vs}) written(*w);
  }
  return Py_BuildValue("(NNN)", THPVariable_Wrap(new_lens), THPVariable_Wrap(new_weights), THPVariable_Wrap(kept));
  END_HANDLE_TH_ERRORS
}

// weight_sums(q, k, lse, window or None, n_sink, scale or None, cu_seqlens or None) -> sums
PyObject* py_weight_sums(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "attn_weight_sums";
  TORCH_CHECK_TYPE(n == 7, what, " takes 7 arguments");
  at::Tensor q = tensor_arg(args[0], what, "q"), k = tensor_arg(args[1], what, "k"), lse = tensor_arg(args[2], what, "softmax_lse");
  const at::Tensor cu = args[6] == Py_None ? at::Tensor() : tensor_arg(args[6], what, "cu_seqlens");
  int64_t window = kIntMax;
  if (args[3] != Py_None) {
    window = int_arg(args[3], what, "window_size");
    TORCH_CHECK_VALUE(window >= 0, what, ": window_size must be non-negative, or None for every earlier token; got ", window);
  }
  const int64_t n_sink = int_arg(args[4], what, "num_sink_tokens");
  TORCH_CHECK_VALUE(n_sink >= 0, what, ": num_sink_tokens must be non-negative, got ", n_sink);
  check_16bit(q, what, "q");
  const int64_t dims = cu.defined() ? 3 : 4, t = dims - 3;  // the token dimension
  TORCH_CHECK_VALUE(q.dim() == dims && k.dim() == dims, what, ": q and k must be ", cu.defined() ? "[tokens, heads, head_dim] with" : "[batch, tokens, heads, head_dim] without", " cu_seqlens");
  TORCH_CHECK_VALUE(k.scalar_type() == q.scalar_type() && k.size(-1) == q.size(-1) && k.size(t) == q.size(t) && (t == 0 || k.size(0) == q.size(0)), what,
                    ": q and k must have the same type, head dimension and number of tokens");
  TORCH_CHECK_VALUE(q.size(-1) == 64 || q.size(-1) == 128, what, ": head_dim must be 64 or 128, got ", q.size(-1));
  TORCH_CHECK_VALUE(k.size(-2) > 0 && q.size(-2) > 0 && q.size(-2) % k.size(-2) == 0, what, ": Number of query heads must be divisible by number of key/value heads, got ",
                    q.size(-2), " and ", k.size(-2));
  const int64_t batch = t == 0 ? 1 : q.size(0), len = q.size(t), hq = q.size(-2), hkv = k.size(-2);
  TORCH_CHECK_VALUE(batch <= kIntMax && len <= kIntMax && hq <= kIntMax, what, ": too large");
  TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.dim() == dims - 1 && lse.size(-1) == len && lse.size(-2) == hq && (t == 0 || lse.size(0) == batch), what,
                    ": softmax_lse must be float32 ", cu.defined() ? "[num_q_heads, tokens]" : "[batch, num_q_heads, tokens]", ", got ", lse.sizes());
  if (cu.defined())
    TORCH_CHECK_VALUE(cu.scalar_type() == at::kInt && cu.dim() == 1 && cu.size(0) >= 2 && cu.stride(0) == 1, what, ": cu_seqlens must be contiguous int32 [sequences + 1]");
  double scale = 1. / std::sqrt(static_cast<double>(q.size(-1)));
  if (args[5] != Py_None) {
    scale = PyFloat_AsDouble(args[5]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      TORCH_CHECK_TYPE(false, what, ": softmax_scale must be a number");
    }
  }
  TORCH_CHECK_VALUE(static_cast<float>(scale) > 0.f && std::isfinite(static_cast<float>(scale)), what, ": softmax_scale must be positive, got ", scale);
  check_plain(q, what, "q"), check_plain(k, what, "k"), check_plain(lse, what, "softmax_lse");
  check_mode(what);
  TORCH_CHECK(q.is_cuda() && q.layout() == at::kStrided, what, ": q must be a CUDA tensor: ring_swa has no CPU path");
  for (const at::Tensor* x : std::initializer_list<const at::Tensor*>{&k, &lse, &cu})
    if (x->defined()) TORCH_CHECK_VALUE(x->device() == q.device() && x->layout() == at::kStrided, what, ": all tensors must be on one device");
  const int dev = q.get_device();
  if (!ready(dev)) Py_RETURN_FALSE;
  at::Tensor out;
  {
    pybind11::gil_scoped_release no_gil;
    const c10::cuda::CUDAGuard guard(q.device());
    out = at::empty(t == 0 ? at::IntArrayRef({hkv, len}) : at::IntArrayRef({batch, hkv, len}), lse.options());
    if (out.numel() > 0) {
      q = loadable(q, true), k = loadable(k, true);
      if (lse.stride(-1) != 1) lse = lse.contiguous();
      rswa_weight_sums_params_t p;
      std::memset(&p, 0, sizeof(p));
      p.dtype = dtype_code(q);
      p.batch = static_cast<int32_t>(batch), p.len = static_cast<int32_t>(len), p.n_q_heads = static_cast<int32_t>(hq), p.n_kv_heads = static_cast<int32_t>(hkv);
      p.head_dim = static_cast<int32_t>(q.size(-1));
      p.window = static_cast<int32_t>(std::min(window, kIntMax)), p.n_sink = static_cast<int32_t>(std::min(n_sink, kIntMax));
      p.softmax_scale = static_cast<float>(scale);
      p.cu_seqlens = cu.defined() ? cu.const_data_ptr<int32_t>() : nullptr;
      p.n_seqs = cu.defined() ? static_cast<int32_t>(cu.size(0) - 1) : 0;
      // (strides of dimensions of size 1 mean nothing: any that the tensor maps take)
      const auto stride = [](const at::Tensor& x, int64_t dim) { return x.size(dim) <= 1 ? x.size(-1) * x.size(-2) : x.stride(dim); };
      p.q = q.const_data_ptr(), p.k = k.const_data_ptr();
      p.q_stride_b = t == 0 ? 0 : stride(q, 0), p.q_stride_t = stride(q, t), p.q_stride_h = stride(q, t + 1);
      p.k_stride_b = t == 0 ? 0 : stride(k, 0), p.k_stride_t = stride(k, t), p.k_stride_h = stride(k, t + 1);
      p.lse = lse.const_data_ptr<float>();
      p.lse_stride_b = t == 0 ? 0 : stride_of(lse, 0), p.lse_stride_h = stride_of(lse, t);
      p.out = out.data_ptr<float>();
      p.status = status_word(dev);
      const int64_t bytes = rswa_weight_sums_workspace_bytes(&p);
      if (bytes < 0) check(static_cast<int>(bytes), what);
      const at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
      p.workspace = ws.data_ptr();
      p.workspace_bytes = bytes;
      check(rswa_weight_sums(&p, stream_of(dev)), what);
    }
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace rswa_host

// The torch side of the quantized KV cache's calls, in C++: what QuantizedKVCache.store, .rope_store, .load and .attend do for the ordinary case (dense
// tensors on the cache's device, which is the current one, rows that the kernels can read where they lie). In Python, through ctypes, a call took 13 to 27 us of
// the host, some four times what its kernels take for a few tokens. Everything that is not ordinary returns None, and the Python code takes the call.
#include "torch_common.h"

#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>

#include <algorithm>
#include <mutex>

#include "../../include/xnq.h"

namespace xnq_torch {
namespace {

decltype(&xnq_kv_store) g_store = nullptr;
decltype(&xnq_kv_load) g_load = nullptr;
decltype(&xnq_kv_attend) g_attend = nullptr;
decltype(&xnq_kv_attend_workspace_bytes) g_workspace_bytes = nullptr;
PyObject *g_check = nullptr; // raises the error of a status

struct Cache { // owned by the capsule that the Python object keeps, with its tensors
  xnq_kv_cache c;
  int64_t batch;
  c10::DeviceIndex device;
};
constexpr const char *NAME = "xnq.kv_cache";
Cache *cache_of(PyObject *o) { return static_cast<Cache *>(PyCapsule_GetPointer(o, NAME)); }

// Scratch of attention (parts of rows, tickets that are zero between calls), one block for each stream: the stream keeps the calls that use it in order, and
// whoever enqueues one holds the block's lock. At most BLOCKS streams have one; they are given back with the last cache. A graph may be replayed beside anything
// else, so a stream under capture has a block of the graph's own memory, cleared in the graph by the first call of it (cleared by each, with all its parts,
// a step's attention over 512 positions took 11.9 us instead of 9.6). A call that finds none takes and clears its own.
struct Block {
  c10::DeviceIndex device;
  cudaStream_t stream;
  void *p;
  size_t bytes;
  std::mutex lock;
};
constexpr size_t BLOCK = 16 << 20; // the parts take 10 MB whatever the call; the rest is tickets
constexpr int BLOCKS = 16;
Block g_blocks[BLOCKS]; // they and the counts: under the interpreter's lock
int g_num_blocks = 0;
int64_t g_caches = 0;
struct GraphBlock {
  c10::DeviceIndex device;
  cudaStream_t stream;
  unsigned long long capture; // 0: none
  c10::DataPtr p;
  size_t bytes;
};
GraphBlock *const g_graph_blocks = new GraphBlock[BLOCKS](); // (never destroyed: the allocator may be gone by then)
int g_next_graph_block = 0;

void free_cache(PyObject *capsule) {
  delete cache_of(capsule);
  if (--g_caches > 0) return;
  const RelaxedCapture relaxed;
  for (; g_num_blocks > 0; g_num_blocks--) (void)cudaFree(g_blocks[g_num_blocks - 1].p); // (waits for the kernels that use it; fails where the process is ending)
  for (int i = 0; i < BLOCKS; i++) g_graph_blocks[i] = GraphBlock{};
  (void)cudaGetLastError();
}
// the block of a stream under capture, or null
void *graph_block_for(c10::DeviceIndex device, cudaStream_t stream, size_t bytes) {
  cudaStreamCaptureStatus status;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess || status != cudaStreamCaptureStatusActive || !id) {
    (void)cudaGetLastError();
    return nullptr;
  }
  GraphBlock *b = nullptr;
  for (int i = 0; i < BLOCKS && !b; i++)
    if (g_graph_blocks[i].stream == stream && g_graph_blocks[i].device == device && g_graph_blocks[i].capture) b = &g_graph_blocks[i];
  if (b && b->capture == id && b->bytes >= bytes) return b->p.get();
  if (!b) b = &g_graph_blocks[g_next_graph_block++ % BLOCKS]; // (a capture that loses its block this way clears another)
  *b = GraphBlock{};
  c10::DataPtr p = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  if (cudaMemsetAsync(p.get(), 0, XNQ_KV_WORKSPACE_ZEROED, stream) != cudaSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  *b = GraphBlock{device, stream, id, std::move(p), bytes};
  return b->p.get();
}
// the stream's block, or null: the call takes and clears one of its own
Block *block_for(c10::DeviceIndex device, cudaStream_t stream, size_t bytes) {
  if (bytes > BLOCK) return nullptr;
  cudaStreamCaptureStatus capture;
  if (cudaStreamIsCapturing(stream, &capture) != cudaSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  if (capture != cudaStreamCaptureStatusNone) return nullptr;
  for (int i = 0; i < g_num_blocks; i++)
    if (g_blocks[i].stream == stream && g_blocks[i].device == device) return &g_blocks[i];
  if (g_num_blocks == BLOCKS) return nullptr;
  Block &b = g_blocks[g_num_blocks];
  const RelaxedCapture relaxed;
  if (cudaMalloc(&b.p, BLOCK) != cudaSuccess || cudaMemsetAsync(b.p, 0, BLOCK, stream) != cudaSuccess) {
    (void)cudaGetLastError();
    return nullptr;
  }
  b.device = device, b.stream = stream, b.bytes = BLOCK;
  g_num_blocks++;
  return &b;
}

// [batch, seq, heads, head_dim] that the kernels can read as it lies
bool rows(const Cache &c, const at::Tensor &t, xnq_rows *out) {
  if (t.dim() != 4 || t.size(0) != c.batch || t.size(3) != c.c.head_dim || t.stride(3) != 1 || t.device().index() != c.device || t.size(1) == 0) return false;
  out->dtype = xnq_dtype(t.scalar_type());
  if (out->dtype < 0) return false;
  out->data = const_cast<void *>(t.const_data_ptr());
  const int64_t e = 16 / t.element_size();
  int64_t *const strides[3] = {&out->stride_b, &out->stride_s, &out->stride_h};
  for (int i = 0; i < 3; i++) {
    *strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (*strides[i] % e) return false;
  }
  return reinterpret_cast<uintptr_t>(out->data) % 16 == 0;
}
// A gradient or a tangent is asked for: the Python code refuses the call.
bool asks(const at::Tensor &t) { return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined(); }
bool positions(const Cache &c, PyObject *o, const long long **p, int *stride) {
  if (!plain(o)) return false;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kLong || t.device().index() != c.device || !t.is_contiguous() || (t.numel() != 1 && t.numel() != c.batch)) return false;
  *p = static_cast<const long long *>(t.const_data_ptr()), *stride = t.numel() > 1;
  return true;
}
PyObject *raise(int rc) { return PyObject_CallFunction(g_check, "i", rc); }
cudaStream_t stream_of(const Cache &c) { return c10::cuda::getCurrentCUDAStream(c.device).stream(); }
bool arguments(const char *who, Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", who, want);
  return false;
}
at::ScalarType scalar_type(long long code) { return code == XNQ_F32 ? at::kFloat : (code == XNQ_F16 ? at::kHalf : at::kBFloat16); }

} // namespace

// kv_cache(address of an xnq_kv_cache, batch, device index) -> capsule
PyObject *kv_cache(PyObject *, PyObject *args) {
  unsigned long long at;
  long long batch;
  int device;
  if (!PyArg_ParseTuple(args, "KLi", &at, &batch, &device)) return nullptr;
  PyObject *capsule = PyCapsule_New(new Cache{*reinterpret_cast<const xnq_kv_cache *>(at), batch, (c10::DeviceIndex)device}, NAME, free_cache);
  if (capsule) g_caches++;
  return capsule;
}

// kv_bind(xnq_kv_store, xnq_kv_load, xnq_kv_attend, xnq_kv_attend_workspace_bytes, check): the library that ctypes has loaded
PyObject *kv_bind(PyObject *, PyObject *args) {
  unsigned long long store, load, attend, ws;
  PyObject *check;
  if (!PyArg_ParseTuple(args, "KKKKO", &store, &load, &attend, &ws, &check)) return nullptr;
  g_store = reinterpret_cast<decltype(g_store)>(store), g_load = reinterpret_cast<decltype(g_load)>(load);
  g_attend = reinterpret_cast<decltype(g_attend)>(attend), g_workspace_bytes = reinterpret_cast<decltype(g_workspace_bytes)>(ws);
  Py_INCREF(check);
  Py_XSETREF(g_check, check);
  Py_RETURN_NONE;
}

// kv_store(cache, k, v, pos) -> True, or None
PyObject *kv_store(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!arguments("kv_store", nargs, 4)) return nullptr;
  const Cache *c = cache_of(args[0]);
  if (!c) return nullptr;
  xnq_rows k, v;
  const long long *pos;
  int stride;
  if (!plain(args[1]) || !plain(args[2]) || observed() || c10::cuda::current_device() != c->device) Py_RETURN_NONE;
  const at::Tensor &kt = THPVariable_Unpack(args[1]), &vt = THPVariable_Unpack(args[2]);
  if (asks(kt) || asks(vt) || !rows(*c, kt, &k) || !rows(*c, vt, &v) || k.dtype != v.dtype || kt.size(1) != vt.size(1) || kt.size(2) != c->c.kv_heads || vt.size(2) != c->c.kv_heads ||
      !positions(*c, args[3], &pos, &stride))
    Py_RETURN_NONE;
  int rc;
  const int64_t seq = kt.size(1);
  const cudaStream_t stream = stream_of(*c);
  Py_BEGIN_ALLOW_THREADS
  rc = g_store(&c->c, &k, &v, c->batch, seq, pos, stride, nullptr, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return raise(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// kv_rope_store(cache, qkv, cos, sin, pos, heads, type of the queries or -1) -> q, or None
PyObject *kv_rope_store(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!arguments("kv_rope_store", nargs, 7)) return nullptr;
  const Cache *c = cache_of(args[0]);
  if (!c) return nullptr;
  const long long heads = PyLong_AsLongLong(args[5]), type = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  const long long *pos;
  int stride;
  if (!plain(args[1]) || !plain(args[2]) || !plain(args[3]) || observed() || c10::cuda::current_device() != c->device) Py_RETURN_NONE;
  const at::Tensor &x = THPVariable_Unpack(args[1]), &cos = THPVariable_Unpack(args[2]), &sin = THPVariable_Unpack(args[3]);
  const int64_t hd = c->c.head_dim, kv = c->c.kv_heads;
  const int dtype = xnq_dtype(x.scalar_type());
  if (asks(x) || asks(cos) || asks(sin) || dtype < 0 || heads < 1 || heads > 65535 || x.dim() != 3 || x.size(0) != c->batch || x.size(1) == 0 || x.size(2) != (heads + 2 * kv) * hd || x.stride(2) != 1 ||
      x.device().index() != c->device || !positions(*c, args[4], &pos, &stride))
    Py_RETURN_NONE;
  for (const at::Tensor *t : {&cos, &sin})
    if (t->scalar_type() != at::kFloat || !t->is_contiguous() || t->dim() != 2 || t->size(1) != hd / 2 || t->size(0) != cos.size(0) || t->device().index() != c->device)
      Py_RETURN_NONE;
  const int64_t e = 16 / x.element_size(), sb = c->batch > 1 ? x.stride(0) : 0, ss = x.size(1) > 1 ? x.stride(1) : 0;
  char *const data = static_cast<char *>(const_cast<void *>(x.const_data_ptr()));
  if (reinterpret_cast<uintptr_t>(data) % 16 || sb % e || ss % e) Py_RETURN_NONE;
  const at::ScalarType out_type = type < 0 ? x.scalar_type() : scalar_type(type);
  at::Tensor q = empty_here({c->batch, x.size(1), (int64_t)heads, hd}, out_type);
  const int64_t width = x.element_size();
  const xnq_rows k{data + heads * hd * width, dtype, sb, ss, hd}, v{data + (heads + kv) * hd * width, dtype, sb, ss, hd};
  const xnq_kv_rope rope{static_cast<const float *>(cos.const_data_ptr()), static_cast<const float *>(sin.const_data_ptr()), cos.size(0), (int)heads,
                         xnq_rows{data, dtype, sb, ss, hd}, xnq_rows{q.mutable_data_ptr(), xnq_dtype(out_type), x.size(1) * heads * hd, heads * hd, hd}};
  int rc;
  const int64_t seq = x.size(1);
  const cudaStream_t stream = stream_of(*c);
  Py_BEGIN_ALLOW_THREADS
  rc = g_store(&c->c, &k, &v, c->batch, seq, pos, stride, &rope, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return raise(rc);
  return THPVariable_Wrap(std::move(q));
  END_HANDLE_TH_ERRORS
}

// kv_load(cache, start: a number or positions, length, type) -> (k, v), or None
PyObject *kv_load(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!arguments("kv_load", nargs, 4)) return nullptr;
  const Cache *c = cache_of(args[0]);
  if (!c) return nullptr;
  const long long n = PyLong_AsLongLong(args[2]), type = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  if (n < 1 || observed() || c10::cuda::current_device() != c->device) Py_RETURN_NONE;
  const long long *pos = nullptr;
  int stride = 0;
  long long start = 0;
  if (PyLong_Check(args[1])) {
    start = PyLong_AsLongLong(args[1]);
    if (PyErr_Occurred()) return nullptr;
  } else if (!positions(*c, args[1], &pos, &stride)) Py_RETURN_NONE;
  at::Tensor k = empty_here({c->batch, (int64_t)c->c.kv_heads, (int64_t)n, (int64_t)c->c.head_dim}, scalar_type(type));
  at::Tensor v = empty_here({c->batch, (int64_t)c->c.kv_heads, (int64_t)n, (int64_t)c->c.head_dim}, scalar_type(type));
  void *const kp = k.mutable_data_ptr(), *const vp = v.mutable_data_ptr();
  int rc;
  const cudaStream_t stream = stream_of(*c);
  Py_BEGIN_ALLOW_THREADS
  rc = g_load(&c->c, c->batch, pos, stride, start, n, (int)type, kp, vp, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return raise(rc);
  PyObject *kw = THPVariable_Wrap(std::move(k)), *vw = THPVariable_Wrap(std::move(v)), *both = kw && vw ? PyTuple_Pack(2, kw, vw) : nullptr;
  Py_XDECREF(kw);
  Py_XDECREF(vw);
  return both;
  END_HANDLE_TH_ERRORS
}

// kv_attend(cache, q, pos, causal, window, scale) -> out, or None
PyObject *kv_attend(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (!arguments("kv_attend", nargs, 6)) return nullptr;
  const Cache *c = cache_of(args[0]);
  if (!c) return nullptr;
  if (!plain(args[1]) || observed() || c10::cuda::current_device() != c->device) Py_RETURN_NONE;
  const at::Tensor &qt = THPVariable_Unpack(args[1]);
  xnq_rows q;
  const long long *pos;
  int stride;
  if (asks(qt) || !rows(*c, qt, &q) || qt.size(2) < 1 || qt.size(2) % c->c.kv_heads || !positions(*c, args[2], &pos, &stride)) Py_RETURN_NONE;
  const int causal = PyObject_IsTrue(args[3]);
  const long long window = PyLong_AsLongLong(args[4]);
  const double scale = PyFloat_AsDouble(args[5]);
  if (PyErr_Occurred()) return nullptr;
  if (window < 0) Py_RETURN_NONE;
  const int64_t seq = qt.size(1), heads = qt.size(2), hd = c->c.head_dim;
  at::Tensor out = empty_here(qt.sizes(), qt.scalar_type());
  const xnq_rows o{out.mutable_data_ptr(), q.dtype, seq * heads * hd, heads * hd, hd};
  const cudaStream_t stream = stream_of(*c);
  const size_t need = std::max<size_t>(g_workspace_bytes(c->batch, seq, (int)heads, c->c.kv_heads, c->c.head_dim), 256);
  Block *const block = block_for(c->device, stream, need);
  c10::DataPtr own;
  void *ws = block ? block->p : graph_block_for(c->device, stream, need);
  if (!ws) own = c10::cuda::CUDACachingAllocator::get()->allocate(need), ws = own.get(); // for the current device and stream, where the call launches
  int rc = 0;
  cudaError_t cleared = cudaSuccess;
  Py_BEGIN_ALLOW_THREADS // a launch may block while the device's queue is full
  if (block) block->lock.lock();
  else if (own) cleared = cudaMemsetAsync(ws, 0, XNQ_KV_WORKSPACE_ZEROED, stream);
  if (cleared == cudaSuccess) rc = g_attend(&c->c, &q, &o, nullptr, c->batch, seq, (int)heads, pos, stride, (float)scale, causal, window, ws, need, stream);
  if (block) block->lock.unlock();
  Py_END_ALLOW_THREADS
  if (cleared != cudaSuccess) {
    PyErr_Format(PyExc_RuntimeError, "attend: clearing the workspace failed: %s", cudaGetErrorString(cleared));
    return nullptr;
  }
  if (rc != 0) return raise(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

} // namespace xnq_torch

// Python binding of the key-value cache's C entries (include/ma_api.h) for
// torch tensors: argument checks, outputs, stream and workspace of
// kv_cache_write, kv_cache_read and decode_attention (kv_cache.py).
//
// One new token a call is a few microseconds of device time, so the host side
// has to be as short: built on ctypes, a call took 15 us of it.  The kernels stay in the C
// library, whose entries' addresses init() takes; nothing here computes.
//
// Each function returns its result, or an int that kv_cache.py acts on: the
// library's return code, kFailedBefore (the host mirror reports a failure of
// an earlier call) or kNoStatus (set_status() was not called for the device).
// Wrong arguments raise ValueError / TypeError / RuntimeError.
#include <ATen/ops/empty.h>
#include <ATen/ops/ne.h>
#include <ATen/ops/narrow.h>
#include <ATen/ops/zero.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>

#include <cmath>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "ma_api.h"

namespace {

constexpr int kFailedBefore = -100, kNoStatus = -101;
constexpr int kMaxDevices = 64;

int (*write_fn)(const ma_cache_write_params*, void*) = nullptr;
int (*read_fn)(const ma_cache_read_params*, void*) = nullptr;
int (*decode_fn)(const ma_decode_params*, void*) = nullptr;
size_t workspace_bytes = 0;

struct Status {
  uint32_t* word = nullptr;  // on the device
  uint32_t* host = nullptr;  // its page-locked mirror
  bool mirror = false;       // whether the kernels may write it
};
Status status_of[kMaxDevices];

int page_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MA_DTYPE_F32;
    case at::kHalf: return MA_DTYPE_F16;
    case at::kBFloat16: return MA_DTYPE_BF16;
    case at::kFloat8_e4m3fn: return MA_DTYPE_E4M3;
    case at::kChar: return MA_DTYPE_I8;
    default: return -1;
  }
}

int dense_code(at::ScalarType t) {
  const int c = page_code(t);
  return c >= 0 && c <= MA_DTYPE_BF16 ? c : -1;
}

int mask_code(at::ScalarType t) {
  switch (t) {
    case at::kBool:
    case at::kByte:
    case at::kChar: return MA_MASK_BOOL;
    case at::kInt: return MA_MASK_I32;
    case at::kLong: return MA_MASK_I64;
    case at::kFloat: return MA_MASK_F32;
    case at::kHalf: return MA_MASK_F16;
    case at::kBFloat16: return MA_MASK_BF16;
    default: return MA_MASK_NONE;
  }
}

// Numbers become text here and not in the checks' streams: those belong to
// torch's libraries, whose C++ runtime need not be this one's.
std::string dims(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

const at::Tensor& tensor_of(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor; got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

// Neither a gradient nor a tangent is dropped in silence.
void no_grad(const at::Tensor& t) {
  TORCH_CHECK((!t.requires_grad() || !c10::GradMode::is_enabled()) &&
                  (!t._fw_grad(0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode()),
              "the key-value cache operators have no gradient: call them under torch.no_grad() or "
              "detach their inputs");
}

// A cache's tensors, checked, in the library's form.  0 or kFailedBefore / kNoStatus.
int cache_arg(PyObject* k_pages, PyObject* v_pages, PyObject* page_table, PyObject* scales,
              ma_kv_cache* c, c10::Device* device) {
  const at::Tensor &k = tensor_of(k_pages, "k_pages"), &v = tensor_of(v_pages, "v_pages");
  const at::Tensor& table = tensor_of(page_table, "page_table");
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(),
                    "k_pages and v_pages must both be (num_pages, heads, page_size, head_dim); got ",
                    dims(k.sizes()), " and ", dims(v.sizes()));
  const int code = page_code(k.scalar_type());
  TORCH_CHECK_TYPE(code >= 0 && v.scalar_type() == k.scalar_type(),
                   "unsupported dtypes of the pages: ", k.scalar_type(), ", ", v.scalar_type());
  TORCH_CHECK(k.is_cuda(), "the key-value cache (B200) lives on CUDA devices only; got a tensor on ",
              k.device());
  const c10::Device dev = k.device();
  TORCH_CHECK_VALUE(k.size(3) <= 1 || (k.stride(3) == 1 && v.stride(3) == 1),
                    "the head dimension of the pages must have stride 1");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2,
                    "page_table must be an int32 tensor of shape (E, max_pages); got ",
                    table.scalar_type(), " ", dims(table.sizes()));
  TORCH_CHECK_VALUE(v.device() == dev && table.device() == dev,
                    "pages and page table are on different devices");
  no_grad(k);
  no_grad(v);
  for (int i = 0; i < 4; ++i)
    TORCH_CHECK_VALUE(k.size(i) <= INT32_MAX, "the pages have a dimension beyond 2^31 - 1");
  TORCH_CHECK_VALUE(table.size(0) <= INT32_MAX && table.size(1) <= INT32_MAX,
                    "page_table has a dimension beyond 2^31 - 1");
  c->struct_size = sizeof(*c);
  c->dtype = code;
  c->k_pages = k.data_ptr();
  c->v_pages = v.data_ptr();
  for (int i = 0; i < 3; ++i) {
    c->k_stride[i] = k.stride(i);
    c->v_stride[i] = v.stride(i);
  }
  if (code == MA_DTYPE_E4M3 || code == MA_DTYPE_I8) {
    TORCH_CHECK_VALUE(scales != Py_None && PyTuple_Check(scales) && PyTuple_GET_SIZE(scales) == 2,
                      k.scalar_type(), " pages need scales=(k_scale, v_scale)");
    for (int j = 0; j < 2; ++j) {
      const at::Tensor& s = tensor_of(PyTuple_GET_ITEM(scales, j), "scales");
      TORCH_CHECK_VALUE(s.scalar_type() == at::kFloat && s.sizes() == k.sizes().slice(0, 3),
                        "scales must be float32 tensors of shape (num_pages, heads, page_size) = ",
                        dims(k.sizes().slice(0, 3)), "; got ", s.scalar_type(), " ", dims(s.sizes()));
      TORCH_CHECK_VALUE(s.device() == dev, "scales must be on the same device as the pages");
      no_grad(s);
      (j ? c->v_scale : c->k_scale) = static_cast<float*>(s.data_ptr());
      for (int i = 0; i < 3; ++i) (j ? c->vs_stride : c->ks_stride)[i] = s.stride(i);
    }
  } else {
    TORCH_CHECK_VALUE(scales == Py_None, k.scalar_type(), " pages have no scales");
  }
  c->page_table = static_cast<const int32_t*>(table.data_ptr());
  c->page_table_stride[0] = table.stride(0);
  c->page_table_stride[1] = table.stride(1);
  c->E = (int32_t)table.size(0);
  c->Hk = (int32_t)k.size(1);
  c->D = (int32_t)k.size(3);
  c->num_pages = (int32_t)k.size(0);
  c->page_size = (int32_t)k.size(2);
  c->max_pages = (int32_t)table.size(1);
  *device = dev;
  TORCH_CHECK(dev.index() >= 0 && dev.index() < kMaxDevices, "device index out of range");
  const Status& st = status_of[dev.index()];
  if (!st.word) return kNoStatus;
  if (st.mirror && *static_cast<volatile uint32_t*>(st.host) != 0) return kFailedBefore;
  c->status = st.word;
  c->status_host = st.mirror ? st.host : nullptr;
  return 0;
}

const int32_t* seq_arg(PyObject* o, const char* name, int64_t E, c10::Device dev) {
  const at::Tensor& t = tensor_of(o, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == E && t.is_contiguous(),
                    name, " must be a contiguous int32 tensor of shape (E,) = ", dims({E}), "; got ",
                    t.scalar_type(), " ", dims(t.sizes()));
  TORCH_CHECK_VALUE(t.device() == dev, name, " must be on the same device as the pages");
  return static_cast<const int32_t*>(t.data_ptr());
}

PyObject* code_of(int rc) { return PyLong_FromLong(rc); }

void need_args(Py_ssize_t n, Py_ssize_t want) {
  TORCH_CHECK_TYPE(n == want, "wrong number of arguments");
}

// init(ma_cache_write, ma_cache_read, ma_decode: addresses, workspace bytes)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 4);
  write_fn = reinterpret_cast<decltype(write_fn)>(PyLong_AsVoidPtr(args[0]));
  read_fn = reinterpret_cast<decltype(read_fn)>(PyLong_AsVoidPtr(args[1]));
  decode_fn = reinterpret_cast<decltype(decode_fn)>(PyLong_AsVoidPtr(args[2]));
  workspace_bytes = PyLong_AsSize_t(args[3]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// set_status(device index, address of the word, address of the mirror, may the kernels write it)
PyObject* set_status(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 4);
  const long i = PyLong_AsLong(args[0]);
  TORCH_CHECK(i >= 0 && i < kMaxDevices, "device index out of range");
  Status s;
  s.word = static_cast<uint32_t*>(PyLong_AsVoidPtr(args[1]));
  s.host = static_cast<uint32_t*>(PyLong_AsVoidPtr(args[2]));
  s.mirror = PyObject_IsTrue(args[3]) == 1;
  if (PyErr_Occurred()) return nullptr;
  status_of[i] = s;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// write(k, v, k_pages, v_pages, page_table, start, scales, count)
PyObject* write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 8);
  ma_cache_write_params p{};
  c10::Device dev(c10::kCUDA, 0);
  const int before = cache_arg(args[2], args[3], args[4], args[6], &p.cache, &dev);
  const at::Tensor &k = tensor_of(args[0], "k"), &v = tensor_of(args[1], "v");
  const int64_t E = p.cache.E, Hk = p.cache.Hk, D = p.cache.D;
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes() && k.size(0) == E && k.size(1) == Hk &&
                        k.size(3) == D,
                    "k and v must be (E, Hk, T, D) with (E, Hk, D) = ", dims({E, Hk, D}), "; got ",
                    dims(k.sizes()), " and ", dims(v.sizes()));
  p.dtype = dense_code(k.scalar_type());
  TORCH_CHECK_TYPE(p.dtype >= 0 && v.scalar_type() == k.scalar_type(),
                   "unsupported dtypes of k and v: ", k.scalar_type(), ", ", v.scalar_type());
  TORCH_CHECK_VALUE(k.device() == dev && v.device() == dev,
                    "k and v must be on the same device as the pages");
  no_grad(k);
  no_grad(v);
  p.struct_size = sizeof(p);
  p.start = seq_arg(args[5], "start", E, dev);
  p.count = args[7] == Py_None ? nullptr : seq_arg(args[7], "count", E, dev);
  TORCH_CHECK_VALUE(k.size(2) <= INT32_MAX, "T exceeds 2^31 - 1");
  p.T = (int32_t)k.size(2);
  if (before) return code_of(before);
  if (E == 0 || p.T == 0) return code_of(0);
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  for (int i = 0; i < 4; ++i) {
    p.k_stride[i] = k.stride(i);
    p.v_stride[i] = v.stride(i);
  }
  const c10::cuda::CUDAGuard guard(dev);
  return code_of(write_fn(&p, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  END_HANDLE_TH_ERRORS
}

// read(k_pages, v_pages, page_table, lengths, max_len, scales, dtype, out) -> (k, v, mask)
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 8);
  ma_cache_read_params p{};
  c10::Device dev(c10::kCUDA, 0);
  const int before = cache_arg(args[0], args[1], args[2], args[5], &p.cache, &dev);
  const int64_t E = p.cache.E, Hk = p.cache.Hk, D = p.cache.D;
  p.struct_size = sizeof(p);
  p.lengths = seq_arg(args[3], "lengths", E, dev);
  const int64_t N = PyLong_AsLongLong(args[4]);
  if (N == -1 && PyErr_Occurred()) return nullptr;
  TORCH_CHECK_VALUE(N >= 0, "max_len must not be negative");
  TORCH_CHECK_VALUE(N <= INT32_MAX, "max_len exceeds 2^31 - 1");
  p.N = (int32_t)N;
  at::ScalarType dt = at::kBFloat16;
  const bool given = args[6] != Py_None;
  if (given) {
    TORCH_CHECK_TYPE(THPDtype_Check(args[6]), "dtype must be a torch.dtype");
    dt = reinterpret_cast<THPDtype*>(args[6])->scalar_type;
  } else if (p.cache.dtype == MA_DTYPE_F32 || p.cache.dtype == MA_DTYPE_F16) {
    dt = p.cache.dtype == MA_DTYPE_F32 ? at::kFloat : at::kHalf;
  }
  at::Tensor k, v;
  if (args[7] != Py_None) {
    TORCH_CHECK_TYPE(PyTuple_Check(args[7]) && PyTuple_GET_SIZE(args[7]) == 2, "out must be (k, v)");
    k = tensor_of(PyTuple_GET_ITEM(args[7], 0), "out");
    v = tensor_of(PyTuple_GET_ITEM(args[7], 1), "out");
    const int64_t want[4] = {E, Hk, N, D};
    TORCH_CHECK_VALUE(k.sizes() == at::IntArrayRef(want, 4) && v.sizes() == k.sizes(),
                      "out tensors must be (E, Hk, max_len, D) = ", dims(at::IntArrayRef(want, 4)), "; got ",
                      dims(k.sizes()), " and ", dims(v.sizes()));
    TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type() && (!given || k.scalar_type() == dt),
                     "out dtypes ", k.scalar_type(), ", ", v.scalar_type(), " do not match");
    TORCH_CHECK_VALUE(k.device() == dev && v.device() == dev,
                      "out tensors must be on the same device as the pages");
    no_grad(k);
    no_grad(v);
    dt = k.scalar_type();
  }
  p.dtype = dense_code(dt);
  TORCH_CHECK_TYPE(p.dtype >= 0, "unsupported dtype ", dt);
  if (before) return code_of(before);
  const c10::cuda::CUDAGuard guard(dev);
  if (!k.defined()) {
    k = at::empty({E, Hk, N, D}, at::TensorOptions(dev).dtype(dt));
    v = at::empty({E, Hk, N, D}, at::TensorOptions(dev).dtype(dt));
  }
  at::Tensor mask = at::empty({E, N}, at::TensorOptions(dev).dtype(at::kBool));
  if (E > 0 && N > 0) {
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.mask = static_cast<uint8_t*>(mask.data_ptr());
    for (int i = 0; i < 4; ++i) {
      p.k_stride[i] = k.stride(i);
      p.v_stride[i] = v.stride(i);
    }
    const int rc = read_fn(&p, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
    if (rc) return code_of(rc);
  }
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  if (args[7] != Py_None) {
    for (int i = 0; i < 2; ++i) {
      PyObject* o = PyTuple_GET_ITEM(args[7], i);
      Py_INCREF(o);
      PyTuple_SET_ITEM(r, i, o);
    }
  } else {
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
  }
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(mask)));
  return r;
  END_HANDLE_TH_ERRORS
}

// ma_decode's workspace: one a stream, so that calls on different streams do not
// meet in it; its counters are zero at first and every call leaves it ready.  The last
// kHeld streams' are kept (10 MB each): another one takes the place of the one that was used
// longest ago, whose memory goes back to the allocator, which gives it to that stream's later
// work alone.  A call that is being captured gets one of its own, zeroed in the graph.  The
// table is never destroyed: the allocator may be gone at the process's end.
constexpr size_t kHeld = 16;
struct Workspace {
  cudaStream_t stream;
  uint64_t used;
  at::Tensor memory;
};
at::Tensor workspace(c10::Device dev, cudaStream_t stream) {
  static std::mutex lock;
  static auto* held = new std::vector<Workspace>[kMaxDevices];
  static uint64_t calls = 0;
  const bool capturing =
      c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  const auto make = [&] {
    at::Tensor t = at::empty({(int64_t)workspace_bytes}, at::TensorOptions(dev).dtype(at::kByte));
    t.narrow(0, 0, MA_DECODE_ZERO_BYTES).zero_();
    return t;
  };
  if (capturing) return make();
  const std::lock_guard<std::mutex> g(lock);
  std::vector<Workspace>& of = held[dev.index()];
  size_t oldest = 0;
  for (size_t i = 0; i < of.size(); ++i) {
    if (of[i].stream == stream) {
      of[i].used = ++calls;
      return of[i].memory;
    }
    if (of[i].used < of[oldest].used) oldest = i;
  }
  Workspace w{stream, ++calls, make()};
  if (of.size() < kHeld) of.push_back(w);
  else of[oldest] = w;
  return w.memory;
}

// decode(q, k_pages, v_pages, page_table, lengths, mask, scales, sm_scale, out, return_lse)
// -> out or (out, lse)
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  need_args(n, 10);
  ma_decode_params p{};
  c10::Device dev(c10::kCUDA, 0);
  const int before = cache_arg(args[1], args[2], args[3], args[6], &p.cache, &dev);
  const int64_t E = p.cache.E, Hk = p.cache.Hk, D = p.cache.D;
  const at::Tensor& q = tensor_of(args[0], "q");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(0) == E && q.size(2) == 1 && q.size(3) == D,
                    "q must be (E, H, 1, D) with (E, D) = ", dims({E, D}), "; got ", dims(q.sizes()));
  const int64_t H = q.size(1);
  TORCH_CHECK_VALUE(H > 0 && H <= INT32_MAX && Hk > 0 && H % Hk == 0, "the number of query heads ",
                    std::to_string(H), " is not a multiple of the cache's ", std::to_string(Hk));
  p.struct_size = sizeof(p);
  p.dtype = dense_code(q.scalar_type());
  TORCH_CHECK_TYPE(p.dtype >= 0, "unsupported dtype of q: ", q.scalar_type());
  TORCH_CHECK_TYPE(args[6] != Py_None || p.dtype == p.cache.dtype, "q is ", q.scalar_type(),
                   " but the pages are of another type");
  TORCH_CHECK_VALUE(q.device() == dev, "q must be on the same device as the pages");
  no_grad(q);
  p.lengths = seq_arg(args[4], "lengths", E, dev);
  const c10::cuda::CUDAGuard guard(dev);
  at::Tensor mask;
  if (args[5] != Py_None) {
    mask = tensor_of(args[5], "attention_mask");
    TORCH_CHECK_VALUE(mask.dim() == 2 && mask.size(0) == E && mask.size(1) <= INT32_MAX,
                      "attention_mask must have shape (E, N) with E = ", std::to_string(E), "; got ",
                      dims(mask.sizes()));
    TORCH_CHECK_VALUE(mask.device() == dev, "attention_mask must be on the same device as the inputs");
    p.mask_dtype = mask_code(mask.scalar_type());
    if (p.mask_dtype == MA_MASK_NONE) {  // any other dtype: nonzero = valid
      mask = at::ne(mask, 0);
      p.mask_dtype = MA_MASK_BOOL;
    }
    p.mask_len = (int32_t)mask.size(1);
    p.mask_stride[0] = mask.stride(0);
    p.mask_stride[1] = mask.stride(1);
    // without columns nothing is valid: a pointer that is never read
    p.mask = p.mask_len ? mask.data_ptr() : static_cast<const void*>(p.lengths);
  }
  double scale = D > 0 ? 1.0 / std::sqrt((double)D) : 1.0;
  if (args[7] != Py_None) {
    scale = PyFloat_AsDouble(args[7]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  }
  p.sm_scale = (float)scale;
  const int want_lse = PyObject_IsTrue(args[9]);
  if (want_lse < 0) return nullptr;
  at::Tensor out, lse;
  if (args[8] != Py_None) {
    out = tensor_of(args[8], "out");
    TORCH_CHECK_VALUE(out.sizes() == q.sizes(), "out shape ", dims(out.sizes()), " != ",
                      dims(q.sizes()));
    TORCH_CHECK_TYPE(out.scalar_type() == q.scalar_type(), "out dtype ", out.scalar_type(),
                     " != ", q.scalar_type());
    TORCH_CHECK_VALUE(out.device() == dev, "out is on a different device than the inputs");
    no_grad(out);
  }
  if (before) return code_of(before);
  if (!out.defined()) out = at::empty({E, H, 1, D}, q.options());
  if (want_lse) lse = at::empty({E, H}, at::TensorOptions(dev).dtype(at::kFloat));
  if (E > 0) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const at::Tensor ws = workspace(dev, stream);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = workspace_bytes;
    p.q = q.data_ptr();
    p.out = out.data_ptr();
    p.lse = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
    for (int i = 0, j = 0; i < 4; ++i)
      if (i != 2) {
        p.q_stride[j] = q.stride(i);
        p.o_stride[j++] = out.stride(i);
      }
    p.H = (int32_t)H;
    const int rc = decode_fn(&p, stream);
    if (rc) return code_of(rc);
  }
  PyObject* o = args[8];
  if (o == Py_None) o = THPVariable_Wrap(std::move(out));
  else Py_INCREF(o);
  if (!o || !want_lse) return o;
  PyObject* l = THPVariable_Wrap(std::move(lse));
  PyObject* r = l ? PyTuple_Pack(2, o, l) : nullptr;
  Py_DECREF(o);
  Py_XDECREF(l);
  return r;
  END_HANDLE_TH_ERRORS
}

#define MA_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"init", MA_FAST(init), nullptr},
                         {"set_status", MA_FAST(set_status), nullptr},
                         {"write", MA_FAST(write), nullptr},
                         {"read", MA_FAST(read), nullptr},
                         {"decode", MA_FAST(decode), nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ma_torch", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ma_torch() { return PyModule_Create(&module); }

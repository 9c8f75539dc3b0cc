// torch_ops.cpp -- tensor-level callers of the KV-cache and beam-search entry
// points of the C ABI: argument checks, output and workspace memory (PyTorch's
// allocator), device and stream.  These calls are made per token and layer, where
// the same steps in Python take as long as the kernels (19 us of host time for a tree
// attention through ctypes); the library itself stays independent of PyTorch.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>
#include <vector>

#include "../../include/ltm_b200.h"

namespace {

PyObject* g_error = nullptr;  // ltm_b200.LtmError(status, message)

struct Refused {};  // a Python exception is set

[[noreturn]] void fail(int status, const std::string& msg) {
  PyObject* args = Py_BuildValue("(is)", status, msg.c_str());
  if (args != nullptr) {
    PyErr_SetObject(g_error, args);
    Py_DECREF(args);
  }
  throw Refused{};
}
[[noreturn]] void bad(const std::string& msg) { fail(LTM_ERR_INVALID_ARG, msg); }

using Opt = const at::Tensor*;  // nullptr: None

Opt tensor_or_none(PyObject* o) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "expected a tensor");
    throw Refused{};
  }
  return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o) {
  Opt t = tensor_or_none(o);
  if (t == nullptr) {
    PyErr_SetString(PyExc_TypeError, "expected a tensor, got None");
    throw Refused{};
  }
  return *t;
}
int integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  if (v < INT32_MIN || v > INT32_MAX) bad("a size exceeds int32");
  return static_cast<int>(v);
}
int size32(int64_t v) {
  if (v > INT32_MAX) bad("a size exceeds int32");
  return static_cast<int>(v);
}

void* ptr(Opt t) { return t ? t->data_ptr() : nullptr; }
template <class T>
T* ptr_as(Opt t) { return static_cast<T*>(ptr(t)); }

ltm_dtype dtype_of(at::ScalarType s) {
  switch (s) {
    case at::kFloat: return LTM_DTYPE_F32;
    case at::kHalf: return LTM_DTYPE_F16;
    case at::kBFloat16: return LTM_DTYPE_BF16;
    default: bad("unsupported type (f32, f16 or bf16)");
  }
}

// Device and stream of one call.  The tensors' device and the call's stream are the current
// ones while this lives.  Memory made for the call comes from the call's stream: a block of
// the caller's current stream may still be read or written by work queued there, which the
// call does not wait for.  The caller's stream is recorded as a user of the outputs, so that
// they are not given out again while its work reads them.
class Call {
 public:
  Call(const at::Tensor& first, PyObject* stream)
      : device_(first.device()), guard_(first.device()),
        stream_(c10::cuda::getCurrentCUDAStream(first.device().index())), raw_(stream_.stream()) {
    if (stream != Py_None) {
      PyObject* v = PyObject_GetAttrString(stream, "cuda_stream");
      if (v == nullptr) throw Refused{};
      void* s = PyLong_AsVoidPtr(v);
      Py_DECREF(v);
      if (PyErr_Occurred()) throw Refused{};
      if (s != static_cast<void*>(raw_)) {
        raw_ = static_cast<cudaStream_t>(s);
        other_.emplace(c10::cuda::getStreamFromExternal(raw_, device_.index()).unwrap());
      }
    }
  }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    at::Tensor t(at::detail::empty_cuda(shape, type, device_, std::nullopt));  // no dispatch
    if (other_ && t.numel() > 0) t.record_stream(stream_.unwrap());
    return t;
  }
  void* stream() const { return static_cast<void*>(raw_); }
  // Workspace of the allocator's, given back to the call's stream when the launches are
  // queued.
  class Workspace {
   public:
    Workspace(size_t bytes, cudaStream_t stream)
        : p_(bytes ? c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(bytes, stream)
                   : nullptr) {}
    ~Workspace() {
      if (p_ != nullptr) c10::cuda::CUDACachingAllocator::raw_delete(p_);
    }
    Workspace(const Workspace&) = delete;
    Workspace& operator=(const Workspace&) = delete;
    void* get() const { return p_; }

   private:
    void* p_;
  };
  Workspace workspace(size_t bytes) const { return Workspace(bytes, raw_); }

 private:
  c10::Device device_;
  c10::cuda::CUDAGuard guard_;
  c10::cuda::CUDAStream stream_;  // the caller's
  cudaStream_t raw_;              // the call's
  std::optional<c10::cuda::CUDAStreamGuard> other_;  // where they differ
};

void done(ltm_status st) {
  if (st != LTM_OK) fail(st, ltm_last_error_string());
}

void check_cuda(const at::Tensor& first) {
  if (!first.is_cuda()) {
    PyErr_SetString(PyExc_ValueError, "ltm_b200 operates on CUDA tensors only");
    throw Refused{};
  }
}
void check_device(const at::Tensor& first, std::initializer_list<Opt> others) {
  check_cuda(first);
  for (Opt t : others)
    if (t != nullptr && t->device() != first.device()) bad("all tensors must be on one device");
}

// A contiguous int32 tensor of the shape (or None).
void check_index(Opt t, at::IntArrayRef shape) {
  if (t != nullptr && (t->scalar_type() != at::kInt || t->sizes() != shape || !t->is_contiguous()))
    bad("lengths and indices must be contiguous int32 tensors of one value per sequence (beam, token)");
}

void check_cache(const at::Tensor& c, Opt scale, const char* what) {
  const std::string name(what);
  if (c.dim() != 4 || !c.is_contiguous())
    bad(name + " must be contiguous [B, kv_heads, max_positions, head_dim]");
  if (scale == nullptr) {
    if (c.scalar_type() == at::kChar) bad(name + ": int8 caches need scales");
  } else if (c.scalar_type() != at::kChar || scale->scalar_type() != at::kFloat ||
             scale->sizes() != c.sizes().slice(0, 3) || !scale->is_contiguous()) {
    bad(name + ": an int8 cache takes contiguous fp32 scales [B, kv_heads, max_positions], "
               "other caches none");
  }
}
void check_pair(const at::Tensor& k, const at::Tensor& v, Opt ks, Opt vs) {
  check_cache(k, ks, "k_cache");
  check_cache(v, vs, "v_cache");
  if (k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
    bad("k_cache and v_cache must have one shape and type");
}
// Strides of a 4-dimensional tensor's first three dimensions; those of one entry
// count as 0, whatever the tensor says.
struct RowStrides {
  int64_t s[3];
  RowStrides(const at::Tensor& t, const char* what) {
    if (t.stride(3) != 1) bad(std::string(what) + " must have unit stride in head_dim");
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) == 1 ? 0 : t.stride(i);
  }
};

// Whether the spans of two tensors' elements meet.
bool meet(const at::Tensor& a, const at::Tensor& b) {
  auto end = [](const at::Tensor& t) {
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return static_cast<const char*>(t.data_ptr()) + last * static_cast<int64_t>(t.element_size());
  };
  return a.numel() > 0 && b.numel() > 0 && static_cast<const char*>(a.data_ptr()) < end(b) &&
         static_cast<const char*>(b.data_ptr()) < end(a);
}
void apart(const at::Tensor& a, std::initializer_list<Opt> others, const char* msg) {
  for (Opt t : others)
    if (t != nullptr && meet(a, *t)) bad(msg);
}

template <class F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& f) {
  if (given != wanted) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  HANDLE_TH_ERRORS  // PyTorch's errors (out of memory) as its own exceptions
  try {
    return f();
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* none() { Py_RETURN_NONE; }

// (k, v, k_cache, v_cache, cache_lens, k_scale, v_scale, num_tokens, stream)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &kc = tensor(a[2]), &vc = tensor(a[3]);
    const at::Tensor& lens = tensor(a[4]);
    Opt ks = tensor_or_none(a[5]), vs = tensor_or_none(a[6]), num = tensor_or_none(a[7]);
    check_device(k, {&v, &kc, &vc, &lens, ks, vs, num});
    check_pair(kc, vc, ks, vs);
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type())
      bad("k and v must both be [B, T, kv_heads, head_dim]");
    const int64_t B = k.size(0), T = k.size(1), h = k.size(2), d = k.size(3);
    if (kc.size(0) != B || kc.size(1) != h || kc.size(3) != d) bad("the caches do not fit k and v");
    if (ks == nullptr && kc.scalar_type() != k.scalar_type())
      bad("the caches must be int8 or have k's type");
    check_index(&lens, {B});
    check_index(num, {B});
    const RowStrides sk(k, "k"), sv(v, "v");
    for (Opt t : {&k, &v}) apart(*t, {&kc, &vc, ks, vs}, "k and v must not overlap the caches");
    const ltm_dtype dt = dtype_of(k.scalar_type());
    Call c(k, a[8]);
    done(ltm_kv_cache_append(k.data_ptr(), sk.s, v.data_ptr(), sv.s, dt, kc.data_ptr(), vc.data_ptr(),
                             ptr_as<float>(ks), ptr_as<float>(vs), kc.size(2),
                             ptr_as<int32_t>(&lens), ptr_as<int32_t>(num), size32(B), size32(T),
                             size32(h), size32(d), c.stream()));
    return none();
  });
}

at::ScalarType dtype_arg(PyObject* o, at::ScalarType otherwise) {
  if (o == Py_None) return otherwise;
  if (!THPDtype_Check(o)) {
    PyErr_SetString(PyExc_TypeError, "expected a torch.dtype");
    throw Refused{};
  }
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// (cache, scale, length, first, cache_lens, dtype, out, stream)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&] {
    const at::Tensor& cache = tensor(a[0]);
    Opt scale = tensor_or_none(a[1]), first = tensor_or_none(a[3]), lens = tensor_or_none(a[4]);
    Opt given = tensor_or_none(a[6]);
    const int length = integer(a[2]);
    check_device(cache, {scale, first, lens, given});
    check_cache(cache, scale, "cache");
    if (length < 0) bad("length must not be negative");
    const at::ScalarType type = dtype_arg(a[5], scale ? at::kFloat : cache.scalar_type());
    if (scale == nullptr && type != cache.scalar_type()) bad("a 16-bit cache is read in its own type");
    const int64_t B = cache.size(0), h = cache.size(1), P = cache.size(2), d = cache.size(3);
    check_index(first, {B});
    check_index(lens, {B});
    const ltm_dtype dt = dtype_of(type);
    const int64_t shape[4] = {B, h, length, d};
    if (given != nullptr && (given->sizes() != at::IntArrayRef(shape, 4) ||
                             given->scalar_type() != type || !given->is_contiguous()))
      bad("out must be contiguous [B, kv_heads, length, head_dim] of the read type");
    if (given != nullptr) apart(*given, {&cache, scale}, "out must not overlap the cache");
    Call c(cache, a[7]);
    const at::Tensor out = given ? *given : c.empty(at::IntArrayRef(shape, 4), type);
    done(ltm_kv_cache_read(cache.data_ptr(), ptr_as<float>(scale), dt, P, ptr_as<int32_t>(first),
                           ptr_as<int32_t>(lens), size32(B), size32(h), size32(d), length,
                           out.data_ptr(), c.stream()));
    return given ? Py_NewRef(a[6]) : THPVariable_Wrap(out);
  });
}

// (q, k_cache, v_cache, cache_lens, parents, k_scale, v_scale, num_tokens, out, stream)
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 10, [&] {
    const at::Tensor &q = tensor(a[0]), &kc = tensor(a[1]), &vc = tensor(a[2]), &lens = tensor(a[3]);
    Opt parents = tensor_or_none(a[4]), ks = tensor_or_none(a[5]), vs = tensor_or_none(a[6]);
    Opt num = tensor_or_none(a[7]), given = tensor_or_none(a[8]);
    check_device(q, {&kc, &vc, &lens, parents, ks, vs, num, given});
    check_pair(kc, vc, ks, vs);
    if (q.dim() != 4 || kc.size(0) != q.size(0) || kc.size(3) != q.size(3))
      bad("q must be [B, T, heads, head_dim] for the caches' B and head_dim");
    if (ks == nullptr && kc.scalar_type() != q.scalar_type())
      bad("the caches must be int8 or have q's type");
    const int64_t B = q.size(0), T = q.size(1), heads = q.size(2), d = q.size(3);
    check_index(&lens, {B});
    check_index(num, {B});
    check_index(parents, {B, T});
    if (given != nullptr && (given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type()))
      bad("out must have q's shape and type");
    bool aside = false;
    if (given != nullptr) {
      apart(*given, {&kc, &vc, ks, vs}, "out must not overlap the caches");
      // More than 512 sequences are several launches, and a later one reads q after an earlier
      // one has written: into memory of its own, then, where out may share some with q other
      // than as q itself.
      bool itself = given->data_ptr() == q.data_ptr();
      for (int i = 0; i < 4; ++i) itself &= q.size(i) == 1 || q.stride(i) == given->stride(i);
      aside = B > 512 && !itself && meet(*given, q);
      if (at::has_internal_overlap(*given) == at::MemOverlap::Yes)
        bad("elements of out share memory");
    }
    const RowStrides sq(q, "q");
    const ltm_dtype dt = dtype_of(q.scalar_type());
    size_t bytes = 0;
    done(ltm_tree_attention_workspace(size32(B), size32(T), size32(heads), size32(kc.size(1)),
                                      size32(d), &bytes));
    Call c(q, a[9]);
    const at::Tensor out = given && !aside ? *given : c.empty(q.sizes(), q.scalar_type());
    const RowStrides so(out, "out");
    if (aside) RowStrides(*given, "out");
    const Call::Workspace ws = c.workspace(bytes);
    done(ltm_tree_attention(q.data_ptr(), sq.s, kc.data_ptr(), vc.data_ptr(), ptr_as<float>(ks),
                            ptr_as<float>(vs), kc.size(2), ptr_as<int32_t>(&lens),
                            ptr_as<int32_t>(num), ptr_as<int32_t>(parents), out.data_ptr(),
                            so.s, size32(B), size32(T), size32(heads),
                            size32(kc.size(1)), size32(d), dt, ws.get(), bytes, c.stream()));
    if (aside) given->copy_(out);
    return given ? Py_NewRef(a[8]) : THPVariable_Wrap(out);
  });
}

// (logits, scores, num_out or None, done, end_token, stream)
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&] {
    const at::Tensor &logits = tensor(a[0]), &scores = tensor(a[1]);
    Opt fin = tensor_or_none(a[3]);
    check_device(logits, {&scores, fin});
    if (logits.dim() != 3 || (logits.size(2) > 1 && logits.stride(2) != 1))
      bad("logits must be [B, W, V] with unit stride in V");
    const int64_t B = logits.size(0), W = logits.size(1), V = logits.size(2);
    if (scores.scalar_type() != at::kFloat || scores.sizes() != at::IntArrayRef({B, W}) ||
        !scores.is_contiguous())
      bad("scores must be contiguous fp32 [B, W]");
    if (fin != nullptr && (fin->scalar_type() != at::kBool ||
                           fin->sizes() != at::IntArrayRef({B, W}) || !fin->is_contiguous()))
      bad("done must be contiguous bool [B, W]");
    const int K = a[2] == Py_None ? size32(W) : integer(a[2]), end = integer(a[4]);
    if (K < 1) bad("num_out must be at least 1");
    const ltm_dtype dt = dtype_of(logits.scalar_type());
    size_t bytes = 0;
    done(ltm_beam_select_workspace(size32(B), size32(W), size32(V), K, &bytes));
    Call c(logits, a[5]);
    const at::Tensor best = c.empty({B, K}, at::kFloat), beams = c.empty({B, K}, at::kInt);
    const at::Tensor tokens = c.empty({B, K}, at::kInt);
    at::Tensor out_fin;
    if (fin != nullptr) out_fin = c.empty({B, K}, at::kBool);
    const Call::Workspace ws = c.workspace(bytes);
    done(ltm_beam_select(logits.data_ptr(), dt, logits.stride(0), logits.stride(1),
                         ptr_as<float>(&scores), ptr_as<uint8_t>(fin), end, size32(B), size32(W),
                         size32(V), K, ptr_as<float>(&best), ptr_as<int32_t>(&beams),
                         ptr_as<int32_t>(&tokens), fin ? ptr_as<uint8_t>(&out_fin) : nullptr,
                         ws.get(), bytes, c.stream()));
    PyObject* r = PyTuple_New(fin ? 4 : 3);
    if (r == nullptr) throw Refused{};
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(best));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(beams));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(tokens));
    if (fin) PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(out_fin));
    return r;
  });
}

// (caches, beams, cache_lens, first, stream); caches: a list or tuple of tensors
PyObject* reorder(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const at::Tensor& beams = tensor(a[1]);
    Opt lens = tensor_or_none(a[2]), first = tensor_or_none(a[3]);
    check_device(beams, {lens, first});
    if (beams.dim() != 2) bad("beams must be int32 [B, W]");
    const int64_t B = beams.size(0), W = beams.size(1);
    check_index(&beams, {B, W});
    check_index(lens, {B});
    check_index(first, {B});
    PyObject* seq = PySequence_Fast(a[0], "caches must be a sequence of tensors");
    if (seq == nullptr) throw Refused{};
    struct Release {
      PyObject* o;
      ~Release() { Py_DECREF(o); }
    } release{seq};
    const Py_ssize_t count = PySequence_Fast_GET_SIZE(seq);
    if (count == 0) return none();
    std::vector<void*> ptrs;
    std::vector<int64_t> rows;
    int64_t h = 0, P = 0;
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor& t = tensor(PySequence_Fast_GET_ITEM(seq, i));
      if (t.device() != beams.device()) bad("all tensors must be on one device");
      if (t.dim() < 3 || t.dim() > 4 || !t.is_contiguous())
        bad("caches must be contiguous [B * W, kv_heads, max_positions(, head_dim)]");
      if (i == 0) {
        h = t.size(1);
        P = t.size(2);
      }
      if (t.size(0) != B * W || t.size(1) != h || t.size(2) != P)
        bad("caches must all be [B * W, kv_heads, max_positions(, head_dim)]");
      ptrs.push_back(t.data_ptr());
      rows.push_back(static_cast<int64_t>(t.element_size()) * (t.dim() == 4 ? t.size(3) : 1));
    }
    Call c(beams, a[4]);
    done(ltm_kv_cache_reorder(ptrs.data(), rows.data(), static_cast<int>(count),
                              ptr_as<int32_t>(&beams), ptr_as<int32_t>(first),
                              ptr_as<int32_t>(lens), size32(B), size32(W), size32(h), P,
                              c.stream()));
    return none();
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XDECREF(g_error);
  g_error = cls;
  Py_RETURN_NONE;
}

template <class F>
PyCFunction fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"kv_cache_append", fast(append), METH_FASTCALL, nullptr},
    {"kv_cache_read", fast(read), METH_FASTCALL, nullptr},
    {"tree_attention", fast(tree), METH_FASTCALL, nullptr},
    {"beam_select", fast(beam_select), METH_FASTCALL, nullptr},
    {"kv_cache_reorder", fast(reorder), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }

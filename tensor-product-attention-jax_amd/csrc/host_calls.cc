// Host side of the Python operator API: argument checks, output and workspace allocation, and the call into the C ABI,
// as one native call per operator, plus the operator's autograd node.
//
// What bounds it: a decode of one sequence is two kernels of a few microseconds, and the same work written in Python
// (shape checks, three torch allocations, six factor descriptors and an argument structure through ctypes, a stream
// look-up) took 24 us per call, a differentiable call 100 us - longer than the kernels it launches.  Here a call costs
// what its allocations and launches cost.
//
// Every function takes its operands as torch GPU tensors and returns NotImplemented if one of them is something else
// (numpy arrays, CPU tensors): the Python layer then converts them and calls again.  The shape and type rules are those
// of tpa/tpa.py:144-163,474-475; a violated one raises the exception a Python `assert` / `raise` would.
#include <Python.h>
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "tpa_abi.h"

namespace {

using at::Tensor;

// ------------------------------------------------------------------------------------------------ the C ABI, by name
#define TPA_CALLS(X)                                                                                             \
  X(tpa_fwd) X(tpa_decode) X(tpa_cache_append) X(tpa_bwd) X(tpa_strerror) X(tpa_fwd_call_workspace_bytes) \
  X(tpa_decode_call_workspace_bytes) X(tpa_cache_append_workspace_bytes) X(tpa_bwd_workspace_bytes)             \
  X(tpa_page_tables) X(tpa_norm_rope) X(tpa_norm_rope_bwd) X(tpa_norm_rope_bwd_workspace_bytes) X(tpa_decode_shared) \
  X(tpa_decode_shared_workspace_bytes) X(tpa_fp4_row_bytes) X(tpa_cache_write_fp4) X(tpa_cache_read_fp4) X(tpa_decode_fp4) \
  X(tpa_decode_fp4_workspace_bytes) X(tpa_beam_select) X(tpa_beam_select_workspace_bytes) X(tpa_pages_fork) X(tpa_pages_compact) X(tpa_pages_workspace_bytes)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
  TPA_CALLS(X)
#undef X
} lib;

// ------------------------------------------------------------------------------------------------ errors
PyObject* error_class = nullptr;  // TpaError(function, code, text)

struct Raise {  // a Python exception of a built-in type
  PyObject* type;
  std::string text;
};
struct CallFailed {  // a non-zero return code of the C ABI
  const char* function;
  int code;
};
void check(const char* function, int code) {
  if (code != TPA_OK) throw CallFailed{function, code};
}
std::string sizes_of(const Tensor& t) {
  std::string s = "torch.Size([";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "])";
}
void expect(bool ok, const Tensor& t) {
  if (!ok) throw Raise{PyExc_AssertionError, sizes_of(t)};
}
void set_python_error(const CallFailed& e) {  // with the GIL held
  PyObject* exc = PyObject_CallFunction(error_class, "sis", e.function, e.code, lib.tpa_strerror(e.code));
  if (!exc) return;
  PyErr_SetObject(error_class, exc);
  Py_DECREF(exc);
}

#define BEGIN_CALL HANDLE_TH_ERRORS try {
#define END_CALL                                   \
  }                                                \
  catch (const Raise& e) {                         \
    PyErr_SetString(e.type, e.text.c_str());       \
    return nullptr;                                \
  }                                                \
  catch (const CallFailed& e) {                    \
    set_python_error(e);                           \
    return nullptr;                                \
  }                                                \
  END_HANDLE_TH_ERRORS

struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// ------------------------------------------------------------------------------------------------ arguments
// `need` tensors at the front of `args` must be GPU tensors; false: let Python convert them
bool gpu_tensors(PyObject* const* args, int n) {
  for (int i = 0; i < n; ++i)
    if (!THPVariable_Check(args[i]) || !THPVariable_Unpack(args[i]).is_cuda()) return false;
  return true;
}
bool none_or_gpu(PyObject* arg) { return arg == Py_None || gpu_tensors(&arg, 1); }
Tensor tensor_or_none(PyObject* arg) { return arg == Py_None ? Tensor() : THPVariable_Unpack(arg); }
constexpr int64_t kNotGiven = INT64_MIN;  // a size that has a default
int64_t integer(PyObject* arg) {
  const long long v = PyLong_AsLongLong(arg);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double real(PyObject* arg) {
  const double v = PyFloat_AsDouble(arg);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
void count(const char* name, Py_ssize_t got, Py_ssize_t want) {
  if (got != want) throw Raise{PyExc_TypeError, std::string(name) + ": " + std::to_string(want) + " arguments expected, got " + std::to_string(got)};
}

int dtype_code(at::ScalarType t) {
  if (t == at::kFloat) return TPA_DTYPE_F32;
  if (t == at::kBFloat16) return TPA_DTYPE_BF16;
  throw Raise{PyExc_TypeError, std::string("unsupported dtype ") + c10::toString(t) + ": the kernels take float32 or bfloat16"};
}

// A [b, l, r, x] array whose last dimension is contiguous: `first` .. `first + width` of it
template <typename F>
F factor_of(const Tensor& t, int64_t first = 0) {
  if (t.dim() != 4) throw Raise{PyExc_ValueError, "factor arrays are 4-D [b, l, r, x], got shape " + sizes_of(t)};
  if (t.size(3) > 1 && t.stride(3) != 1) throw Raise{PyExc_ValueError, "the last dimension of a factor array must be contiguous"};
  F f;
  f.ptr = reinterpret_cast<decltype(f.ptr)>(static_cast<char*>(t.data_ptr()) + first * t.element_size());
  f.stride_b = t.stride(0);
  f.stride_l = t.stride(1);
  f.stride_r = t.stride(2);
  return f;
}

bool is_shape(const Tensor& t, std::initializer_list<int64_t> want) { return t.sizes() == at::IntArrayRef(want); }

// int32 [batch, length], one row for all batch entries broadcast (tpa/tpa.py:144-163 vmaps with in_axes=None)
Tensor segment_ids(const Tensor& ids, int64_t batch, int64_t length) {
  if (!ids.defined()) return ids;
  Tensor t = ids.scalar_type() == at::kInt ? ids : ids.to(at::kInt);
  if (t.dim() == 1) t = t.unsqueeze(0).expand({batch, length});
  if (!is_shape(t, {batch, length}))
    throw Raise{PyExc_ValueError, "segment ids must have shape (" + std::to_string(batch) + ", " + std::to_string(length) + "), got " + sizes_of(t)};
  return t.contiguous();
}
Tensor lengths(const Tensor& len, int64_t batch) {
  if (!len.defined()) return len;
  Tensor t = len.scalar_type() == at::kInt ? len.contiguous() : len.to(at::kInt).contiguous();
  if (!is_shape(t, {batch})) throw Raise{PyExc_ValueError, "kv_lengths must have shape (" + std::to_string(batch) + ",), got " + sizes_of(t)};
  return t;
}
const int32_t* ids_ptr(const Tensor& t) { return t.defined() ? static_cast<const int32_t*>(t.data_ptr()) : nullptr; }
float* f32_ptr(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

Tensor bytes_on(const at::Device& device, size_t n) { return at::empty({(int64_t)n}, at::TensorOptions().dtype(at::kByte).device(device)); }
void* aligned(const Tensor& t, size_t to) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return reinterpret_cast<void*>((p + to - 1) / to * to);
}
void* stream_of(const at::Device& device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

// every operand on one device: a pointer of another would be read there, or not at all
void one_device(std::initializer_list<Tensor> tensors) {
  const Tensor* first = nullptr;
  for (const Tensor& t : tensors) {
    if (!t.defined()) continue;
    if (!first) first = &t;
    else if (t.device() != first->device())
      throw Raise{PyExc_ValueError, "operands on two devices: " + first->device().str() + " and " + t.device().str()};
  }
}
// a dual tensor need not ask for gradients, so an autograd node, which refuses a tangent, may never see it
void no_tangents(std::initializer_list<Tensor> tensors, const char* name) {
  for (const Tensor& t : tensors)
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
      throw Raise{PyExc_NotImplementedError, std::string(name) + " has no forward-mode derivative: an input carries a tangent"};
}
// The gradient of a leaf is accumulated on the stream that the leaf's node was made on.  While an eager graph of the leaf lives, that is not
// the stream that is being captured, and a backward pass in the capture would wait for the other one, which ends the process.
void no_node_from_outside_a_capture(std::initializer_list<Tensor> tensors, const char* name) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor& t : tensors) {
    if (!t.defined() || !t.is_leaf() || !t.requires_grad()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto of = node ? node->stream() : std::nullopt;
    if (of && *of != c10::hip::getCurrentHIPStream(t.device().index()).unwrap())
      throw Raise{PyExc_RuntimeError, std::string(name) + " is being captured into a graph while an eager graph of one of its inputs lives: delete what was computed from it first, or detach the input"};
  }
}
// a call wrote into `t`: a node that saved it notices
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
template <typename Args>
void take_workspace(const Tensor& ws, size_t alignment, Args& a) {
  if (!ws.is_contiguous()) throw Raise{PyExc_ValueError, "workspace must be contiguous"};
  const size_t bytes = ws.numel() * ws.element_size(), skip = static_cast<char*>(aligned(ws, alignment)) - static_cast<char*>(ws.data_ptr());
  a.workspace = aligned(ws, alignment);
  a.workspace_bytes = bytes > skip ? bytes - skip : 0;
}

// ------------------------------------------------------------------------------------------------ forward
struct FwdCall {
  Tensor qseg, kvseg, kvlen;
  double sm_scale = 1.0;
  int causal = 0, kernel = TPA_KERNEL_AUTO, causal_offset = 0, nomat = 0;
  bool return_lse = true, use_workspace = true;
};

// `a` holds the six factors and the sizes; allocates the outputs and the workspace and makes the call
std::pair<Tensor, Tensor> run_fwd(TpaFwdArgs& a, const FwdCall& c, const at::Device& device, at::ScalarType dtype) {
  a.dtype = dtype_code(dtype);
  const Tensor qseg = segment_ids(c.qseg, a.B, a.lq), kvseg = segment_ids(c.kvseg, a.B, a.lk);
  if (qseg.defined() != kvseg.defined()) throw Raise{PyExc_ValueError, "q_segment_ids and kv_segment_ids must be given together"};
  const Tensor kvlen = lengths(c.kvlen, a.B);
  const auto options = at::TensorOptions().device(device);
  Tensor o = at::empty({a.B, a.lq, a.H, a.dv}, options.dtype(dtype)), lse, ws;
  if (c.return_lse) lse = at::empty({a.B, a.H, a.lq}, options.dtype(at::kFloat));
  a.q_segment_ids = ids_ptr(qseg);
  a.kv_segment_ids = ids_ptr(kvseg);
  a.kv_lengths = ids_ptr(kvlen);
  a.o = o.data_ptr();
  a.lse = f32_ptr(lse);
  a.sm_scale = (float)c.sm_scale;
  a.causal = c.causal;
  a.kernel = c.kernel;
  a.causal_offset = c.causal_offset;
  a.nomat = c.nomat;
  // the workspace with which the library can pick its fastest kernel (nomat: the split partials, required)
  const size_t need = c.use_workspace || c.nomat ? lib.tpa_fwd_call_workspace_bytes(&a) : 0;
  if (need) {
    try {
      ws = bytes_on(device, need + 256);
    } catch (const c10::OutOfMemoryError&) {
      if (c.nomat) throw;  // otherwise it is optional: on a card too full for it the kernels that take none serve the call
    }
  }
  if (ws.defined()) {
    a.workspace = aligned(ws, 256);
    a.workspace_bytes = need;
  }
  check("tpa_fwd", lib.tpa_fwd(&a, stream_of(device)));
  return {o, lse};
}

void check_dtypes(const Tensor* t, const char* const* names, int n) {
  for (int i = 1; i < n; ++i)
    if (t[i].scalar_type() != t[0].scalar_type())
      throw Raise{PyExc_TypeError, std::string(names[i]) + " has dtype " + c10::toString(t[i].scalar_type()) + ", expected " + c10::toString(t[0].scalar_type())};
}

// q[b, lq, rq, h + dk], k[b, lk, rk, h + dk], v[b, lk, rk, h + dv] of one type: what the operator and its gradient take
void check_concatenated(const Tensor& q, const Tensor& k, const Tensor& v, int64_t h) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4) throw Raise{PyExc_ValueError, "q, k, v must be [b, l, r, h + d]"};
  // rank and length of the keys are read from v (tpa/tpa.py:474-475)
  expect(is_shape(k, {q.size(0), v.size(1), v.size(2), q.size(3)}), k);
  expect(v.size(0) == q.size(0), v);
  if (!(0 < h && h < q.size(3) && h < v.size(3)))
    throw Raise{PyExc_AssertionError, "num_heads = " + std::to_string(h) + ", " + sizes_of(q) + ", " + sizes_of(v)};
  const Tensor three[3] = {q, k, v};
  static const char* const names[3] = {"q", "k", "v"};
  check_dtypes(three, names, 3);
}

void unpack_six(PyObject* const* args, Tensor* t) {
  static const char* const names[6] = {"qa", "qb", "ka", "kb", "va", "vb"};
  for (int i = 0; i < 6; ++i) t[i] = THPVariable_Unpack(args[i]);
  check_dtypes(t, names, 6);
  for (int i = 0; i < 6; ++i)
    if (t[i].dim() != 4) throw Raise{PyExc_ValueError, "factor arrays are 4-D [b, l, r, x], got shape " + sizes_of(t[i])};
}

// the six factors and the sizes of a problem whose keys are not paged
template <typename Args>
void describe(const Tensor* t, Args& a) {
  a.B = (int)t[0].size(0); a.lq = (int)t[0].size(1); a.rq = (int)t[0].size(2); a.H = (int)t[0].size(3);
  a.lk = (int)t[5].size(1); a.rk = (int)t[5].size(2); a.dv = (int)t[5].size(3); a.dk = (int)t[1].size(3);
  // shape rules of tpa/tpa.py:474-475: k and v share length and rank, q and k share h + dk
  expect(is_shape(t[1], {a.B, a.lq, a.rq, a.dk}), t[1]);
  expect(is_shape(t[2], {a.B, a.lk, a.rk, a.H}), t[2]);
  expect(is_shape(t[3], {a.B, a.lk, a.rk, a.dk}), t[3]);
  expect(is_shape(t[4], {a.B, a.lk, a.rk, a.H}), t[4]);
  expect(t[5].size(0) == a.B, t[5]);
  a.qa = factor_of<TpaFactor>(t[0]); a.qb = factor_of<TpaFactor>(t[1]);
  a.ka = factor_of<TpaFactor>(t[2]); a.kb = factor_of<TpaFactor>(t[3]);
  a.va = factor_of<TpaFactor>(t[4]); a.vb = factor_of<TpaFactor>(t[5]);
}

PyObject* pair(std::pair<Tensor, Tensor>&& r) {
  PyObject* out = PyTuple_New(2);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(r.first)));
  if (r.second.defined()) {
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(r.second)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 1, Py_None);
  }
  return out;
}

// factors(qa, qb, ka, kb, va, vb, q_segment_ids, kv_segment_ids, kv_lengths, sm_scale, causal, kernel, return_lse,
//         use_workspace, causal_offset, nomat)
PyObject* factors(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("factors", n, 16);
  if (!gpu_tensors(args, 6) || !none_or_gpu(args[6]) || !none_or_gpu(args[7]) || !none_or_gpu(args[8])) Py_RETURN_NOTIMPLEMENTED;
  Tensor t[6];
  unpack_six(args, t);
  TpaFwdArgs a{};
  FwdCall c;
  c.qseg = tensor_or_none(args[6]); c.kvseg = tensor_or_none(args[7]); c.kvlen = tensor_or_none(args[8]);
  c.sm_scale = real(args[9]);
  c.causal = (int)integer(args[10]); c.kernel = (int)integer(args[11]);
  c.return_lse = integer(args[12]); c.use_workspace = integer(args[13]);
  c.causal_offset = (int)integer(args[14]); c.nomat = (int)integer(args[15]);
  describe(t, a);
  std::pair<Tensor, Tensor> r;
  {
    WithoutGil free;
    const c10::DeviceGuard guard(t[0].device());
    r = run_fwd(a, c, t[0].device(), t[0].scalar_type());
  }
  return pair(std::move(r));
  END_CALL
}

// ------------------------------------------------------------------------------------------------ decode
// the six factors and the sizes of a problem whose keys are a contiguous cache or, with `pages`, page pools; returns the table to hold on to
Tensor describe_cache(const Tensor* t, Tensor pages, TpaFwdArgs& a) {
  if (!pages.defined()) {
    describe(t, a);
  } else {
    // page pools [pages, page_size, rk, x]; the logical cache length is pages_per_seq * page_size
    a.B = (int)t[0].size(0); a.lq = (int)t[0].size(1); a.rq = (int)t[0].size(2); a.H = (int)t[0].size(3);
    a.rk = (int)t[5].size(2); a.dv = (int)t[5].size(3); a.dk = (int)t[1].size(3);
    const int64_t npages = t[5].size(0), page = t[5].size(1);
    if (pages.scalar_type() != at::kInt) pages = pages.to(at::kInt);
    pages = pages.contiguous();
    expect(pages.dim() == 2 && pages.size(0) == a.B, pages);
    expect(is_shape(t[1], {a.B, a.lq, a.rq, a.dk}), t[1]);
    expect(is_shape(t[3], {npages, page, a.rk, a.dk}), t[3]);
    expect(is_shape(t[2], {npages, page, a.rk, a.H}), t[2]);
    expect(is_shape(t[4], {npages, page, a.rk, a.H}), t[4]);
    a.page_table = ids_ptr(pages);
    a.page_size = (int)page;
    a.pages_per_seq = (int)pages.size(1);
    a.lk = a.pages_per_seq * a.page_size;
    a.qa = factor_of<TpaFactor>(t[0]); a.qb = factor_of<TpaFactor>(t[1]);
    a.ka = factor_of<TpaFactor>(t[2]); a.kb = factor_of<TpaFactor>(t[3]);
    a.va = factor_of<TpaFactor>(t[4]); a.vb = factor_of<TpaFactor>(t[5]);
  }
  return pages;
}

// decode(qa, qb, ka, kb, va, vb, kv_lengths, page_table, workspace, sm_scale, num_splits, kernel, causal, causal_offset)
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("decode", n, 14);
  if (!gpu_tensors(args, 6) || !none_or_gpu(args[6]) || !none_or_gpu(args[7]) || !none_or_gpu(args[8])) Py_RETURN_NOTIMPLEMENTED;
  Tensor t[6];
  unpack_six(args, t);
  TpaFwdArgs a{};
  Tensor ws = tensor_or_none(args[8]);
  const Tensor pages = describe_cache(t, tensor_or_none(args[7]), a);
  a.dtype = dtype_code(t[0].scalar_type());
  a.sm_scale = (float)real(args[9]);
  a.num_splits = (int)integer(args[10]);
  a.kernel = (int)integer(args[11]);
  a.causal = (int)integer(args[12]);
  a.causal_offset = (int)integer(args[13]);
  std::pair<Tensor, Tensor> r;
  {
    WithoutGil free;
    const at::Device device = t[0].device();
    const c10::DeviceGuard guard(device);
    const Tensor kvlen = lengths(tensor_or_none(args[6]), a.B);
    a.kv_lengths = ids_ptr(kvlen);
    const auto options = at::TensorOptions().device(device);
    if (!ws.defined()) ws = bytes_on(device, std::max<size_t>(lib.tpa_decode_call_workspace_bytes(&a), 16));
    r.first = at::empty({a.B, a.lq, a.H, a.dv}, options.dtype(t[0].scalar_type()));
    r.second = at::empty({a.B, a.H, a.lq}, options.dtype(at::kFloat));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws.numel() * ws.element_size();
    a.o = r.first.data_ptr();
    a.lse = f32_ptr(r.second);
    check("tpa_decode", lib.tpa_decode(&a, stream_of(device)));
  }
  return pair(std::move(r));
  END_CALL
}

// ------------------------------------------------------------------------------------------------ cache append
// append(x, w, rope_cos, rope_sin, ka, kb, va, vb, kv_lengths, positions, page_table, workspace, rank_q, kernel, use_workspace)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("append", n, 15);
  if (!gpu_tensors(args, 8)) Py_RETURN_NOTIMPLEMENTED;
  for (int i = 8; i < 12; ++i)
    if (!none_or_gpu(args[i])) Py_RETURN_NOTIMPLEMENTED;
  static const char* const names[6] = {"x", "w", "ka", "kb", "va", "vb"};
  Tensor t[6] = {THPVariable_Unpack(args[0]), THPVariable_Unpack(args[1]), THPVariable_Unpack(args[4]),
                 THPVariable_Unpack(args[5]), THPVariable_Unpack(args[6]), THPVariable_Unpack(args[7])};
  check_dtypes(t, names, 6);
  Tensor x = t[0], w = t[1], cos = THPVariable_Unpack(args[2]), sin = THPVariable_Unpack(args[3]);
  const Tensor &ka = t[2], &kb = t[3], &va = t[4], &vb = t[5];
  if (x.dim() != 3) throw Raise{PyExc_ValueError, "x is [b, n, d_model], got shape " + sizes_of(x)};
  TpaAppendArgs a{};
  a.B = (int)x.size(0); a.n = (int)x.size(1); a.d_model = (int)x.size(2);
  a.ka = factor_of<TpaFactor>(ka); a.kb = factor_of<TpaFactor>(kb); a.va = factor_of<TpaFactor>(va); a.vb = factor_of<TpaFactor>(vb);
  a.rk = (int)ka.size(2); a.H = (int)ka.size(3); a.D = (int)kb.size(3); a.rq = (int)integer(args[12]);
  a.dtype = dtype_code(x.scalar_type());
  a.kernel = (int)integer(args[13]);
  (void)integer(args[14]);  // use_workspace: no append kernel takes scratch memory any more
  expect(is_shape(w, {(int64_t)(a.rq + 2 * a.rk) * (a.H + a.D), a.d_model}), w);
  expect(kb.sizes().slice(0, 3) == ka.sizes().slice(0, 3) && va.sizes() == ka.sizes() && vb.sizes() == kb.sizes(), kb);
  expect(cos.sizes() == sin.sizes() && cos.dim() == 2 && cos.size(1) == a.D / 2, cos);
  a.rope_len = (int)cos.size(0);
  Tensor pages = tensor_or_none(args[10]), pos = tensor_or_none(args[9]), ws = tensor_or_none(args[11]), qa, qb, new_len;
  {
    WithoutGil free;
    const at::Device device = x.device();
    const c10::DeviceGuard guard(device);
    if (!pages.defined()) {
      expect(ka.size(0) == a.B, ka);
      a.cache_len = (int)ka.size(1);
    } else {
      if (pages.scalar_type() != at::kInt) pages = pages.to(at::kInt);
      pages = pages.contiguous();
      expect(pages.dim() == 2 && pages.size(0) == a.B, pages);
      a.page_table = ids_ptr(pages);
      a.page_size = (int)ka.size(1);
      a.pages_per_seq = (int)pages.size(1);
      a.cache_len = a.pages_per_seq * a.page_size;
    }
    const Tensor kvlen = lengths(tensor_or_none(args[8]), a.B);
    if (pos.defined()) {
      pos = pos.scalar_type() == at::kInt ? pos.contiguous() : pos.to(at::kInt).contiguous();
      expect(is_shape(pos, {a.B, a.n}), pos);
    }
    x = x.contiguous();
    w = w.contiguous();
    cos = cos.to(at::kFloat).contiguous();
    sin = sin.to(at::kFloat).contiguous();
    const auto options = at::TensorOptions().device(device);
    qa = at::empty({a.B, a.n, a.rq, a.H}, options.dtype(x.scalar_type()));
    qb = at::empty({a.B, a.n, a.rq, a.D}, options.dtype(x.scalar_type()));
    new_len = at::empty({a.B}, options.dtype(at::kInt));
    if (ws.defined()) {
      a.workspace = aligned(ws, 16);
      a.workspace_bytes = ws.numel() * ws.element_size() - (static_cast<char*>(a.workspace) - static_cast<char*>(ws.data_ptr()));
    }
    a.x = x.data_ptr(); a.w = w.data_ptr();
    a.rope_cos = f32_ptr(cos); a.rope_sin = f32_ptr(sin);
    a.positions = ids_ptr(pos); a.kv_lengths = ids_ptr(kvlen); a.new_kv_lengths = static_cast<int32_t*>(new_len.data_ptr());
    a.qa = factor_of<TpaFactor>(qa); a.qb = factor_of<TpaFactor>(qb);
    check("tpa_cache_append", lib.tpa_cache_append(&a, stream_of(device)));
  }
  PyObject* out = PyTuple_New(3);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(qa)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(qb)));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(new_len)));
  return out;
  END_CALL
}

// ------------------------------------------------------------------------------------------------ backward
// Gradients of the six factors into concatenated arrays dq, dk, dv of the inputs' type (tpa/tpa.py:960-962); `lse` is [b, h, lq].
struct BwdCall {
  Tensor q, k, v, qseg, kvseg, o, lse, d_o;
  int64_t heads = 0;
  double sm_scale = 1.0;
  int causal = 0, causal_offset = 0;
};

void run_bwd(const BwdCall& c, Tensor* grads) {
  const at::Device device = c.q.device();
  const c10::DeviceGuard guard(device);
  const at::ScalarType dtype = c.q.scalar_type();
  const int64_t h = c.heads;
  TpaBwdArgs a{};
  a.B = (int)c.q.size(0); a.lq = (int)c.q.size(1); a.rq = (int)c.q.size(2); a.H = (int)h; a.dk = (int)(c.q.size(3) - h);
  a.lk = (int)c.v.size(1); a.rk = (int)c.v.size(2); a.dv = (int)(c.v.size(3) - h);
  a.qa = factor_of<TpaFactor>(c.q); a.qb = factor_of<TpaFactor>(c.q, h);
  a.ka = factor_of<TpaFactor>(c.k); a.kb = factor_of<TpaFactor>(c.k, h);
  a.va = factor_of<TpaFactor>(c.v); a.vb = factor_of<TpaFactor>(c.v, h);
  a.dtype = dtype_code(dtype);
  const Tensor qseg = segment_ids(c.qseg, a.B, a.lq), kvseg = segment_ids(c.kvseg, a.B, a.lk);
  const Tensor o = c.o.to(dtype).contiguous(), d_o = c.d_o.to(dtype).contiguous(), lse = c.lse.to(at::kFloat).contiguous();
  expect(is_shape(o, {a.B, a.lq, a.H, a.dv}), o);
  expect(is_shape(d_o, {a.B, a.lq, a.H, a.dv}), d_o);
  expect(is_shape(lse, {a.B, a.H, a.lq}), lse);
  const Tensor* in[3] = {&c.q, &c.k, &c.v};
  for (int i = 0; i < 3; ++i) grads[i] = at::empty(in[i]->sizes(), at::TensorOptions().device(device).dtype(dtype));
  a.dqa = factor_of<TpaGrad>(grads[0]); a.dqb = factor_of<TpaGrad>(grads[0], h);
  a.dka = factor_of<TpaGrad>(grads[1]); a.dkb = factor_of<TpaGrad>(grads[1], h);
  a.dva = factor_of<TpaGrad>(grads[2]); a.dvb = factor_of<TpaGrad>(grads[2], h);
  a.q_segment_ids = ids_ptr(qseg);
  a.kv_segment_ids = ids_ptr(kvseg);
  a.o = o.data_ptr();
  a.lse = f32_ptr(lse);
  a.d_o = d_o.data_ptr();
  a.sm_scale = (float)c.sm_scale;
  a.causal = c.causal;
  a.causal_offset = c.causal_offset;
  a.grad_dtype = a.dtype;
  const size_t need = lib.tpa_bwd_workspace_bytes(a.B, a.lq, a.lk, a.H, a.dk, a.dv);
  const Tensor ws = bytes_on(device, need + 256);
  a.workspace = aligned(ws, 256);
  a.workspace_bytes = need;
  check("tpa_bwd", lib.tpa_bwd(&a, stream_of(device)));
}

// backward(q, k, v, q_segment_ids, kv_segment_ids, o, lse, do, num_heads, sm_scale, causal, causal_offset)
PyObject* backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("backward", n, 12);
  if (!gpu_tensors(args, 3) || !gpu_tensors(args + 5, 3) || !none_or_gpu(args[3]) || !none_or_gpu(args[4])) Py_RETURN_NOTIMPLEMENTED;
  BwdCall c;
  c.q = THPVariable_Unpack(args[0]); c.k = THPVariable_Unpack(args[1]); c.v = THPVariable_Unpack(args[2]);
  c.qseg = tensor_or_none(args[3]); c.kvseg = tensor_or_none(args[4]);
  c.o = THPVariable_Unpack(args[5]); c.lse = THPVariable_Unpack(args[6]); c.d_o = THPVariable_Unpack(args[7]);
  c.heads = integer(args[8]);
  check_concatenated(c.q, c.k, c.v, c.heads);
  c.sm_scale = real(args[9]);
  c.causal = (int)integer(args[10]); c.causal_offset = (int)integer(args[11]);
  Tensor grads[3];
  {
    WithoutGil free;
    const at::AutoGradMode no_grad(false);
    run_bwd(c, grads);
  }
  PyObject* out = PyTuple_New(3);
  if (!out) throw python_error();
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(std::move(grads[i])));
  return out;
  END_CALL
}

// ------------------------------------------------------------------------------------------------ the operator
// tpa() on concatenated q[b, lq, rq, h + dk], k[b, lk, rk, h + dk], v[b, lk, rk, h + dv]; the vjp registered for it is
// tpa/tpa.py:217's.
std::pair<Tensor, Tensor> run_concat(const Tensor& q, const Tensor& k, const Tensor& v, int64_t h, const FwdCall& c) {
  const c10::DeviceGuard guard(q.device());
  TpaFwdArgs a{};
  a.B = (int)q.size(0); a.lq = (int)q.size(1); a.rq = (int)q.size(2); a.H = (int)h; a.dk = (int)(q.size(3) - h);
  a.lk = (int)v.size(1); a.rk = (int)v.size(2); a.dv = (int)(v.size(3) - h);
  a.qa = factor_of<TpaFactor>(q); a.qb = factor_of<TpaFactor>(q, h);
  a.ka = factor_of<TpaFactor>(k); a.kb = factor_of<TpaFactor>(k, h);
  a.va = factor_of<TpaFactor>(v); a.vb = factor_of<TpaFactor>(v, h);
  return run_fwd(a, c, q.device(), q.scalar_type());
}

// writes that an array has seen; one made under inference mode counts none
int64_t writes_of(const Tensor& t) { return t.defined() && !t.is_inference() ? (int64_t)t._version() : -1; }

struct Operator : torch::autograd::Function<Operator> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                                                int64_t h, const FwdCall& c) {
    auto [o, lse] = run_concat(q, k, v, h, c);
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, o, lse});
    // segment ids stay where they are (hooks on what is saved see the floating-point tensors alone), with the count of their writes
    ctx->saved_data["call"] = c10::IValue(std::make_tuple(h, c.qseg, c.kvseg, c.sm_scale, (int64_t)c.causal, (int64_t)c.causal_offset, writes_of(c.qseg), writes_of(c.kvseg)));
    return {o, lse};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list d_out) {
    torch::autograd::variable_list out(5);
    if (!d_out[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const auto call = ctx->saved_data["call"].toTuple();
    const auto& e = call->elements();
    BwdCall b;
    b.q = saved[0]; b.k = saved[1]; b.v = saved[2]; b.o = saved[3]; b.lse = saved[4];
    b.d_o = d_out[0];
    b.heads = e[0].toInt();
    b.qseg = e[1].toTensor(); b.kvseg = e[2].toTensor();
    TORCH_CHECK(writes_of(b.qseg) == e[6].toInt() && writes_of(b.kvseg) == e[7].toInt(),
                "segment ids needed for the gradient computation of tpa have been modified by an inplace operation");
    b.sm_scale = e[3].toDouble();
    b.causal = (int)e[4].toInt(); b.causal_offset = (int)e[5].toInt();
    try {
      run_bwd(b, out.data());
    } catch (const CallFailed& f) {  // an engine thread: hand the Python exception to the thread that asked
      PyGILState_STATE gil = PyGILState_Ensure();
      set_python_error(f);
      python_error e2;
      e2.persist();
      PyGILState_Release(gil);
      throw e2;
    } catch (const Raise& f) {
      TORCH_CHECK(false, f.text);
    }
    return out;
  }
};

// tpa(q, k, v, q_segment_ids, kv_segment_ids, num_heads, sm_scale, causal, kernel, use_workspace, causal_offset, nomat)
PyObject* tpa(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("tpa", n, 12);
  if (!gpu_tensors(args, 3) || !none_or_gpu(args[3]) || !none_or_gpu(args[4])) Py_RETURN_NOTIMPLEMENTED;
  const Tensor q = THPVariable_Unpack(args[0]), k = THPVariable_Unpack(args[1]), v = THPVariable_Unpack(args[2]);
  const int64_t h = integer(args[5]);
  check_concatenated(q, k, v, h);
  // a dual tensor need not ask for gradients, so the autograd node below, which refuses a tangent, may never see it
  for (const Tensor* t : {&q, &k, &v})
    if (t->_fw_grad(/*level=*/0).defined())
      throw Raise{PyExc_NotImplementedError, "tpa has no forward-mode derivative: an input carries a tangent"};
  FwdCall c;
  c.qseg = tensor_or_none(args[3]); c.kvseg = tensor_or_none(args[4]);
  c.sm_scale = real(args[6]);
  c.causal = (int)integer(args[7]); c.kernel = (int)integer(args[8]);
  c.use_workspace = integer(args[9]);
  c.causal_offset = (int)integer(args[10]); c.nomat = (int)integer(args[11]);
  std::pair<Tensor, Tensor> r;
  {
    WithoutGil free;
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
      auto out = Operator::apply(q, k, v, h, c);
      r = {out[0], out[1]};
    } else {
      r = run_concat(q, k, v, h, c);
    }
  }
  return pair(std::move(r));
  END_CALL
}

// ------------------------------------------------------------------------------------------------ decode over a shared prefix
// decode_shared(qa, qb, ka, kb, va, vb, kv_lengths, page_table, workspace, prefix_length, sm_scale, kernel, causal, causal_offset)
PyObject* decode_shared(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("decode_shared", n, 14);
  if (!gpu_tensors(args, 6) || !none_or_gpu(args[6]) || !none_or_gpu(args[7]) || !none_or_gpu(args[8])) Py_RETURN_NOTIMPLEMENTED;
  Tensor t[6];
  unpack_six(args, t);
  TpaFwdArgs a{};
  Tensor ws = tensor_or_none(args[8]);
  one_device({t[0], t[1], t[2], t[3], t[4], t[5], tensor_or_none(args[6]), tensor_or_none(args[7]), ws});
  const int64_t prefix = integer(args[9]);
  a.sm_scale = (float)real(args[10]);
  a.kernel = (int)integer(args[11]);
  a.causal = (int)integer(args[12]);
  a.causal_offset = (int)integer(args[13]);
  std::pair<Tensor, Tensor> r;
  {
    WithoutGil free;
    const at::Device device = t[0].device();
    const c10::DeviceGuard guard(device);
    const Tensor pages = describe_cache(t, tensor_or_none(args[7]), a);
    a.dtype = dtype_code(t[0].scalar_type());
    if (prefix < 0 || prefix > a.lk)
      throw Raise{PyExc_ValueError, "prefix_length must be between 0 and the cache's " + std::to_string(a.lk) + " tokens, got " + std::to_string(prefix)};
    const Tensor kvlen = lengths(tensor_or_none(args[6]), a.B);
    a.kv_lengths = ids_ptr(kvlen);
    const auto options = at::TensorOptions().device(device);
    r.first = at::empty({a.B, a.lq, a.H, a.dv}, options.dtype(t[0].scalar_type()));
    r.second = at::empty({a.B, a.H, a.lq}, options.dtype(at::kFloat));
    if (r.first.numel() && a.lk) {  // nothing to launch for no rows
      if (!ws.defined()) ws = bytes_on(device, lib.tpa_decode_shared_workspace_bytes(&a, (int)prefix) + 256);
      take_workspace(ws, 256, a);
      a.o = r.first.data_ptr();
      a.lse = f32_ptr(r.second);
      check("tpa_decode_shared", lib.tpa_decode_shared(&a, (int)prefix, stream_of(device)));
    } else {
      r.first.fill_(NAN);
      r.second.fill_(-INFINITY);
    }
  }
  return pair(std::move(r));
  END_CALL
}

// ------------------------------------------------------------------------------------------------ page tables
PyObject* tuple_of(std::initializer_list<Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}
// as int32; what does not fit stays out of every range
Tensor ints(const Tensor& t) {
  if (!at::isIntegralType(t.scalar_type(), /*includeBool=*/false))
    throw Raise{PyExc_TypeError, std::string("lengths, pages, slots and positions are integers, got ") + c10::toString(t.scalar_type())};
  return (t.scalar_type() == at::kInt ? t : t.scalar_type() == at::kLong ? t.clamp(INT32_MIN, INT32_MAX).to(at::kInt) : t.to(at::kInt)).contiguous();
}

// page_tables(kv_lengths, new_tokens, free_pages, free_start, page_table, page_size, num_tokens)
PyObject* page_tables(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("page_tables", n, 7);
  if (!gpu_tensors(args, 3) || !none_or_gpu(args[3])) Py_RETURN_NOTIMPLEMENTED;
  if (!gpu_tensors(args + 4, 1)) throw Raise{PyExc_TypeError, "page_table is written in place: it must be a GPU tensor"};
  const Tensor table = THPVariable_Unpack(args[4]);
  Tensor len = THPVariable_Unpack(args[0]), fresh = THPVariable_Unpack(args[1]), pool = THPVariable_Unpack(args[2]), start = tensor_or_none(args[3]);
  one_device({len, fresh, pool, start, table});
  if (table.scalar_type() != at::kInt || table.dim() != 2 || !table.is_contiguous())
    throw Raise{PyExc_ValueError, "page_table is written in place: it must be a contiguous int32 [b, pages_per_seq] tensor"};
  const int64_t b = table.size(0), page = integer(args[5]), rows = integer(args[6]);
  if (!is_shape(len, {b})) throw Raise{PyExc_ValueError, "kv_lengths must have shape (" + std::to_string(b) + ",), got " + sizes_of(len)};
  if (!is_shape(fresh, {b})) throw Raise{PyExc_ValueError, "new_tokens must have shape (" + std::to_string(b) + ",), got " + sizes_of(fresh)};
  if (pool.dim() != 1) throw Raise{PyExc_ValueError, "free_pages is a list of pages, got shape " + sizes_of(pool)};
  if (start.defined() && start.numel() != 1) throw Raise{PyExc_ValueError, "free_start is one number, got shape " + sizes_of(start)};
  if (page < 1 || page > INT32_MAX) throw Raise{PyExc_ValueError, "page_size must be positive, got " + std::to_string(page)};
  if (rows < 0 || rows > INT32_MAX) throw Raise{PyExc_ValueError, "num_tokens must not be negative, got " + std::to_string(rows)};
  if (pool.numel() > INT32_MAX || b > INT32_MAX || table.size(1) > INT32_MAX) throw CallFailed{"tpa_page_tables", TPA_ERR_SHAPE};
  Tensor out[5];
  {
    WithoutGil free;
    const at::Device device = table.device();
    const c10::DeviceGuard guard(device);
    len = ints(len);
    fresh = ints(fresh);
    pool = ints(pool);
    if (start.defined()) start = ints(start);
    const auto options = at::TensorOptions().device(device).dtype(at::kInt);
    // one allocation: slots, positions and lengths of a step are read on this device, and each is a few kilobytes
    const int64_t sizes[5] = {rows, rows, b + 1, b, 1};
    int64_t at = 0, total = 0;
    for (int64_t s : sizes) total += (s + 63) / 64 * 64;
    const Tensor all = at::empty({total}, options);
    for (int i = 0; i < 5; ++i) {  // (narrow() takes longer than the kernel for five of them)
      out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
      out[i].unsafeGetTensorImpl()->set_storage_offset(at);
      out[i].unsafeGetTensorImpl()->set_sizes_contiguous({sizes[i]});
      at += (sizes[i] + 63) / 64 * 64;
    }
    if (b) {
      TpaPageTablesArgs a{};
      a.kv_lengths = ids_ptr(len); a.new_tokens = ids_ptr(fresh);
      a.page_table = static_cast<int32_t*>(table.data_ptr());
      a.free_pages = ids_ptr(pool); a.free_start = ids_ptr(start);
      int32_t* to[5];
      for (int i = 0; i < 5; ++i) to[i] = static_cast<int32_t*>(out[i].data_ptr());
      a.slots = to[0]; a.positions = to[1]; a.starts = to[2]; a.new_kv_lengths = to[3]; a.new_free_start = to[4];
      a.B = (int)b; a.pages_per_seq = (int)table.size(1); a.page_size = (int)page; a.num_free = (int)pool.numel(); a.num_tokens = (int)rows;
      check("tpa_page_tables", lib.tpa_page_tables(&a, stream_of(device)));
      written(table);
    } else {  // no requests: rows of padding, no page taken
      out[0].fill_(-1);
      out[1].zero_();
      out[2].zero_();
      if (start.defined()) out[4].copy_(start.view({1}).clamp(0, pool.numel()));
      else out[4].zero_();
    }
  }
  return tuple_of({out[0], out[1], out[2], out[3], out[4]});
  END_CALL
}

// ------------------------------------------------------------------------------------------------ norms and rotation
struct NormRope {  // what a call has beside q and k
  Tensor q_weight, k_weight, positions, cos, sin;
  int64_t heads = 0;
  std::vector<int64_t> sections;
  bool normalize = true;
  double eps = 0;
  int kernel = TPA_KERNEL_AUTO;
};

void check_norm_rope(const Tensor& q, const Tensor& k, NormRope& c) {
  if (q.dim() != 4 || k.dim() != 4) throw Raise{PyExc_ValueError, "q, k must be [b, l, r, h + d]"};
  expect(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3), k);
  if (!(0 < c.heads && c.heads < q.size(3))) throw Raise{PyExc_AssertionError, "num_heads = " + std::to_string(c.heads) + ", " + sizes_of(q)};
  const Tensor two[2] = {q, k};
  static const char* const names[2] = {"q", "k"};
  check_dtypes(two, names, 2);
  (void)dtype_code(q.scalar_type());
  const int64_t d = q.size(3) - c.heads;
  expect(c.cos.sizes() == c.sin.sizes() && c.cos.dim() == 2 && c.cos.size(1) == d / 2 && c.cos.size(0) <= INT32_MAX, c.cos);
  for (const Tensor* w : {&c.q_weight, &c.k_weight})
    if (w->defined()) {
      expect(is_shape(*w, {d}), *w);
      (void)dtype_code(w->scalar_type());
    }
  if (c.q_weight.defined() && c.k_weight.defined() && c.q_weight.scalar_type() != c.k_weight.scalar_type())
    throw Raise{PyExc_TypeError, std::string("k_weight has dtype ") + c10::toString(c.k_weight.scalar_type()) + ", expected " + c10::toString(c.q_weight.scalar_type())};
  if (c.sections.empty()) c.sections = {d / 2};
  int64_t sum = 0;
  for (int64_t s : c.sections) {
    if (s < 0) throw Raise{PyExc_ValueError, "sections must not be negative"};
    sum += s;
    if (sum > d / 2) throw Raise{PyExc_ValueError, "sections add up to more than the " + std::to_string(d / 2) + " pairs of a head"};
  }
  const int64_t axes = (int64_t)c.sections.size();
  if (axes > 4) throw Raise{PyExc_ValueError, "at most 4 axes, got " + std::to_string(axes)};
  if (c.positions.defined()) {
    const bool flat = axes == 1 && is_shape(c.positions, {q.size(0), q.size(1)});
    if (!flat && !is_shape(c.positions, {q.size(0), q.size(1), axes}))
      throw Raise{PyExc_ValueError, "positions must have shape (" + std::to_string(q.size(0)) + ", " + std::to_string(q.size(1)) +
                                        (axes == 1 ? ")" : ", " + std::to_string(axes) + ")") + ", got " + sizes_of(c.positions)};
  }
}
// contiguous arrays of the types that the kernels read
void settle(NormRope& c) {
  if (c.positions.defined()) c.positions = ints(c.positions);
  c.cos = c.cos.to(at::kFloat).contiguous();
  c.sin = c.sin.to(at::kFloat).contiguous();
  if (c.q_weight.defined()) c.q_weight = c.q_weight.contiguous();
  if (c.k_weight.defined()) c.k_weight = c.k_weight.contiguous();
}
template <typename Args>
void describe_norm_rope(const Tensor& q, const Tensor& k, const NormRope& c, Args& a) {
  const int64_t h = c.heads;
  a.qa = factor_of<TpaFactor>(q); a.qb = factor_of<TpaFactor>(q, h);
  a.ka = factor_of<TpaFactor>(k); a.kb = factor_of<TpaFactor>(k, h);
  a.positions = ids_ptr(c.positions); a.rope_cos = f32_ptr(c.cos); a.rope_sin = f32_ptr(c.sin);
  a.q_weight = c.q_weight.defined() ? c.q_weight.data_ptr() : nullptr;
  a.k_weight = c.k_weight.defined() ? c.k_weight.data_ptr() : nullptr;
  const Tensor& w = c.q_weight.defined() ? c.q_weight : c.k_weight;
  a.weight_dtype = w.defined() ? dtype_code(w.scalar_type()) : TPA_DTYPE_F32;
  a.n_axes = (int)c.sections.size();
  for (size_t i = 0; i < c.sections.size(); ++i) a.sections[i] = (int)c.sections[i];
  a.B = (int)q.size(0); a.l = (int)q.size(1); a.H = (int)h; a.D = (int)(q.size(3) - h); a.rq = (int)q.size(2); a.rk = (int)k.size(2);
  a.rope_len = (int)c.cos.size(0); a.dtype = dtype_code(q.scalar_type()); a.kernel = c.kernel;
  a.normalize = c.normalize; a.eps = (float)c.eps;
}
std::pair<Tensor, Tensor> run_norm_rope(const Tensor& q, const Tensor& k, const NormRope& c) {
  const c10::DeviceGuard guard(q.device());
  std::pair<Tensor, Tensor> r;
  r.first = at::empty(q.sizes(), q.options());
  r.second = at::empty(k.sizes(), k.options());
  if (!q.size(0) || !q.size(1)) return r;  // no tokens
  TpaNormRopeArgs a{};
  describe_norm_rope(q, k, c, a);
  a.qa_out = factor_of<TpaFactor>(r.first); a.qb_out = factor_of<TpaFactor>(r.first, c.heads);
  a.ka_out = factor_of<TpaFactor>(r.second); a.kb_out = factor_of<TpaFactor>(r.second, c.heads);
  check("tpa_norm_rope", lib.tpa_norm_rope(&a, stream_of(q.device())));
  return r;
}
// gradients of q, k, q_weight, k_weight; an output without a gradient gives its side none
void run_norm_rope_bwd(const Tensor& q, const Tensor& k, const NormRope& c, const Tensor& dq_out, const Tensor& dk_out, const bool (&weights)[2], Tensor* grads) {
  const c10::DeviceGuard guard(q.device());
  const Tensor in[2] = {q, k};
  Tensor d_out[2] = {dq_out, dk_out};
  const Tensor weight[2] = {c.q_weight, c.k_weight};
  for (int i = 0; i < 2; ++i) {
    if (!d_out[i].defined()) continue;
    expect(d_out[i].sizes() == in[i].sizes(), d_out[i]);
    d_out[i] = d_out[i].to(q.scalar_type()).contiguous();
    grads[i] = at::empty(in[i].sizes(), in[i].options());
    if (weights[i] && weight[i].defined()) grads[2 + i] = at::empty(weight[i].sizes(), weight[i].options());
  }
  if (!d_out[0].defined() && !d_out[1].defined()) return;
  if (!q.size(0) || !q.size(1)) {
    for (int i = 2; i < 4; ++i)
      if (grads[i].defined()) grads[i].zero_();
    return;
  }
  TpaNormRopeBwdArgs a{};
  describe_norm_rope(q, k, c, a);
  const int64_t h = c.heads;
  if (d_out[0].defined()) {
    a.dqa_out = factor_of<TpaFactor>(d_out[0]); a.dqb_out = factor_of<TpaFactor>(d_out[0], h);
    a.dqa = factor_of<TpaFactor>(grads[0]); a.dqb = factor_of<TpaFactor>(grads[0], h);
  }
  if (d_out[1].defined()) {
    a.dka_out = factor_of<TpaFactor>(d_out[1]); a.dkb_out = factor_of<TpaFactor>(d_out[1], h);
    a.dka = factor_of<TpaFactor>(grads[1]); a.dkb = factor_of<TpaFactor>(grads[1], h);
  }
  Tensor ws;
  if (grads[2].defined() || grads[3].defined()) {
    a.dq_weight = grads[2].defined() ? grads[2].data_ptr() : nullptr;
    a.dk_weight = grads[3].defined() ? grads[3].data_ptr() : nullptr;
    ws = bytes_on(q.device(), lib.tpa_norm_rope_bwd_workspace_bytes(a.B, a.l, a.D) + 256);
    take_workspace(ws, 256, a);
  }
  check("tpa_norm_rope_bwd", lib.tpa_norm_rope_bwd(&a, stream_of(q.device())));
}

struct NormRopeOperator : torch::autograd::Function<NormRopeOperator> {
  // (a weight that is not given is no argument of the node: an undefined tensor would be refused)
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const std::optional<Tensor>& q_weight,
                                                const std::optional<Tensor>& k_weight, const NormRope& c) {
    auto [yq, yk] = run_norm_rope(q, k, c);
    ctx->set_materialize_grads(false);
    // positions and tables too: the node notices where one of them is written again before the backward (one made under inference mode counts no
    // writes and cannot be saved: the node has a copy)
    auto kept = [](const Tensor& t) { return t.defined() && t.is_inference() ? t.clone() : t; };
    ctx->save_for_backward({q, k, q_weight.value_or(Tensor()), k_weight.value_or(Tensor()), kept(c.positions), kept(c.cos), kept(c.sin)});
    ctx->saved_data["call"] = c10::IValue(std::make_tuple(c.heads, c.sections, c.normalize, c.eps, (int64_t)c.kernel));
    return {yq, yk};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list d_out) {
    torch::autograd::variable_list out(5);
    TORCH_CHECK(!at::GradMode::is_enabled(), "tpa_norm_rope has no second derivative (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const auto call = ctx->saved_data["call"].toTuple();
    const auto& e = call->elements();
    NormRope c;
    c.q_weight = saved[2]; c.k_weight = saved[3]; c.positions = saved[4]; c.cos = saved[5]; c.sin = saved[6];
    c.heads = e[0].toInt(); c.sections = e[1].toIntVector(); c.normalize = e[2].toBool(); c.eps = e[3].toDouble(); c.kernel = (int)e[4].toInt();
    const bool weights[2] = {c.q_weight.defined() && ctx->needs_input_grad(2), c.k_weight.defined() && ctx->needs_input_grad(c.q_weight.defined() ? 3 : 2)};
    try {
      run_norm_rope_bwd(saved[0], saved[1], c, d_out[0], d_out[1], weights, out.data());
    } catch (const CallFailed& f) {  // an engine thread: hand the Python exception to the thread that asked
      PyGILState_STATE gil = PyGILState_Ensure();
      set_python_error(f);
      python_error e2;
      e2.persist();
      PyGILState_Release(gil);
      throw e2;
    } catch (const Raise& f) {
      TORCH_CHECK(false, f.text);
    }
    return out;
  }
};

std::vector<int64_t> numbers(PyObject* arg) {  // None or a sequence of integers
  std::vector<int64_t> out;
  if (arg == Py_None) return out;
  PyObject* seq = PySequence_Fast(arg, "sections must be a sequence of integers");
  if (!seq) throw python_error();
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq); ++i) {
    const long long v = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
    if (v == -1 && PyErr_Occurred()) {
      Py_DECREF(seq);
      throw python_error();
    }
    out.push_back(v);
  }
  Py_DECREF(seq);
  if (out.empty()) throw Raise{PyExc_ValueError, "sections must have an entry for each axis"};
  return out;
}
// the arguments behind the factors: rope_cos, rope_sin, q_weight, k_weight, positions, num_heads, sections, normalize, eps, kernel
NormRope norm_rope_call(PyObject* const* args) {
  NormRope c;
  c.cos = THPVariable_Unpack(args[0]); c.sin = THPVariable_Unpack(args[1]);
  c.q_weight = tensor_or_none(args[2]); c.k_weight = tensor_or_none(args[3]); c.positions = tensor_or_none(args[4]);
  c.heads = integer(args[5]);
  c.sections = numbers(args[6]);
  c.normalize = integer(args[7]);
  c.eps = real(args[8]);
  c.kernel = (int)integer(args[9]);
  return c;
}

// norm_rope(q, k, rope_cos, rope_sin, q_weight, k_weight, positions, num_heads, sections, normalize, eps, kernel)
PyObject* norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("norm_rope", n, 12);
  if (!gpu_tensors(args, 4) || !none_or_gpu(args[4]) || !none_or_gpu(args[5]) || !none_or_gpu(args[6])) Py_RETURN_NOTIMPLEMENTED;
  const Tensor q = THPVariable_Unpack(args[0]), k = THPVariable_Unpack(args[1]);
  NormRope c = norm_rope_call(args + 2);
  check_norm_rope(q, k, c);
  one_device({q, k, c.cos, c.sin, c.q_weight, c.k_weight, c.positions});
  no_tangents({q, k, c.q_weight, c.k_weight, c.cos, c.sin}, "tpa_norm_rope");
  if (at::GradMode::is_enabled() && (c.cos.requires_grad() || c.sin.requires_grad()))
    throw Raise{PyExc_NotImplementedError, "tpa_norm_rope has no gradient for rope_cos and rope_sin: detach them"};
  std::pair<Tensor, Tensor> r;
  {
    WithoutGil free;
    const c10::DeviceGuard guard(q.device());
    settle(c);
    auto asks = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
    if (at::GradMode::is_enabled() && (asks(q) || asks(k) || asks(c.q_weight) || asks(c.k_weight))) {
      no_node_from_outside_a_capture({q, k, c.q_weight, c.k_weight}, "tpa_norm_rope");
      auto given = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
      auto out = NormRopeOperator::apply(q, k, given(c.q_weight), given(c.k_weight), c);
      r = {out[0], out[1]};
    } else {
      r = run_norm_rope(q, k, c);
    }
  }
  return pair(std::move(r));
  END_CALL
}

// norm_rope_backward(q, k, dq_out, dk_out, rope_cos, rope_sin, q_weight, k_weight, positions, num_heads, sections, normalize, eps, kernel)
PyObject* norm_rope_backward(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("norm_rope_backward", n, 14);
  if (!gpu_tensors(args, 6) || !none_or_gpu(args[6]) || !none_or_gpu(args[7]) || !none_or_gpu(args[8])) Py_RETURN_NOTIMPLEMENTED;
  const Tensor q = THPVariable_Unpack(args[0]), k = THPVariable_Unpack(args[1]), dq_out = THPVariable_Unpack(args[2]), dk_out = THPVariable_Unpack(args[3]);
  NormRope c = norm_rope_call(args + 4);
  check_norm_rope(q, k, c);
  one_device({q, k, c.cos, c.sin, c.q_weight, c.k_weight, c.positions, dq_out, dk_out});
  Tensor grads[4];
  {
    WithoutGil free;
    const at::AutoGradMode no_grad(false);
    const c10::DeviceGuard guard(q.device());
    settle(c);
    run_norm_rope_bwd(q, k, c, dq_out, dk_out, {true, true}, grads);
  }
  PyObject* out = PyTuple_New(4);
  if (!out) throw python_error();
  for (int i = 0; i < 4; ++i) {
    if (!grads[i].defined()) Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, i, grads[i].defined() ? THPVariable_Wrap(std::move(grads[i])) : Py_None);
  }
  return out;
  END_CALL
}

// norm_rope_write(q, k, v, slots, rope_cos, rope_sin, q_weight, k_weight, positions, num_heads, sections, normalize, eps, kernel, ka, kb, va, vb)
PyObject* norm_rope_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("norm_rope_write", n, 18);
  if (!gpu_tensors(args, 6) || !none_or_gpu(args[6]) || !none_or_gpu(args[7]) || !none_or_gpu(args[8])) Py_RETURN_NOTIMPLEMENTED;
  if (!gpu_tensors(args + 14, 4)) throw Raise{PyExc_TypeError, "the cache is written in place: ka, kb, va, vb must be GPU tensors"};
  const Tensor q = THPVariable_Unpack(args[0]), k = THPVariable_Unpack(args[1]), v = THPVariable_Unpack(args[2]);
  Tensor slots = THPVariable_Unpack(args[3]);
  NormRope c = norm_rope_call(args + 4);
  check_norm_rope(q, k, c);
  const int64_t h = c.heads, d = q.size(3) - h, rk = k.size(2);
  expect(v.sizes() == k.sizes(), v);
  if (!is_shape(slots, {q.size(0), q.size(1)}))
    throw Raise{PyExc_ValueError, "slots must have shape (" + std::to_string(q.size(0)) + ", " + std::to_string(q.size(1)) + "), got " + sizes_of(slots)};
  static const char* const names[6] = {"q", "ka", "kb", "va", "vb", "v"};
  const Tensor t[6] = {q, THPVariable_Unpack(args[14]), THPVariable_Unpack(args[15]), THPVariable_Unpack(args[16]), THPVariable_Unpack(args[17]), v};
  check_dtypes(t, names, 6);
  one_device({q, k, v, c.cos, c.sin, c.q_weight, c.k_weight, c.positions, slots, t[1], t[2], t[3], t[4]});
  const Tensor& ka = t[1];
  if (ka.dim() != 4) throw Raise{PyExc_ValueError, "the cache's arrays are [pages, page_size, rank, x], got shape " + sizes_of(ka)};
  for (int i = 1; i < 5; ++i) expect(is_shape(t[i], {ka.size(0), ka.size(1), rk, i % 2 ? h : d}), t[i]);
  if (ka.size(0) * ka.size(1) > INT32_MAX) throw CallFailed{"tpa_norm_rope", TPA_ERR_SHAPE};
  Tensor yq;
  {
    WithoutGil free;
    const at::AutoGradMode no_grad(false);  // a cache is state: no gradient flows into it
    const c10::DeviceGuard guard(q.device());
    settle(c);
    slots = ints(slots);
    yq = at::empty(q.sizes(), q.options());
    if (q.size(0) && q.size(1)) {
      TpaNormRopeArgs a{};
      describe_norm_rope(q, k, c, a);
      a.qa_out = factor_of<TpaFactor>(yq); a.qb_out = factor_of<TpaFactor>(yq, h);
      a.va = factor_of<TpaFactor>(v); a.vb = factor_of<TpaFactor>(v, h);
      a.ka_out = factor_of<TpaFactor>(t[1]); a.kb_out = factor_of<TpaFactor>(t[2]);
      a.va_out = factor_of<TpaFactor>(t[3]); a.vb_out = factor_of<TpaFactor>(t[4]);
      a.slots = ids_ptr(slots);
      a.page_size = (int)ka.size(1);
      a.num_slots = (int)(ka.size(0) * ka.size(1));
      check("tpa_norm_rope", lib.tpa_norm_rope(&a, stream_of(q.device())));
      for (int i = 1; i < 5; ++i) written(t[i]);
    }
  }
  return THPVariable_Wrap(std::move(yq));
  END_CALL
}

// ------------------------------------------------------------------------------------------------ a cache in 4 bits
// A cache of rows [pages or batch entries, tokens, rk, bytes]; `bytes` = what H + D numbers take
void check_fp4_cache(const Tensor& t, const char* name, int64_t rk, int64_t h, int64_t d) {
  if (t.scalar_type() != at::kByte) throw Raise{PyExc_TypeError, std::string(name) + " holds rows of bytes (uint8), got " + c10::toString(t.scalar_type())};
  const int64_t bytes = h <= INT32_MAX && d <= INT32_MAX ? (int64_t)lib.tpa_fp4_row_bytes((int)h, (int)d) : 0;
  if (t.dim() != 4 || t.size(2) != rk || t.size(3) != bytes)
    throw Raise{PyExc_ValueError, std::string(name) + " must be [pages, page_size, " + std::to_string(rk) + ", " + std::to_string(bytes) + "] for " + std::to_string(h) + " heads of " +
                                      std::to_string(d) + ", got " + sizes_of(t)};
}
void fits_int(std::initializer_list<int64_t> sizes, const char* name) {
  for (int64_t s : sizes)
    if (s > INT32_MAX) throw CallFailed{name, TPA_ERR_SHAPE};
}
// what writing and reading have in common; false: nothing to do
bool describe_fp4_rows(const Tensor& k, const Tensor& v, const Tensor& kc, const Tensor& vc, const Tensor& slots, int64_t h, const char* name, TpaFp4RowsArgs& a) {
  expect(kc.sizes().slice(0, 3) == vc.sizes().slice(0, 3), vc);
  if (!is_shape(slots, {k.size(0), k.size(1)}))
    throw Raise{PyExc_ValueError, "slots must have shape (" + std::to_string(k.size(0)) + ", " + std::to_string(k.size(1)) + "), got " + sizes_of(slots)};
  fits_int({k.size(0), k.size(1), k.size(2), k.size(3), v.size(3), kc.size(0), kc.size(1)}, name);
  if (kc.size(0) && kc.size(1) > INT32_MAX / kc.size(0)) throw CallFailed{name, TPA_ERR_SHAPE};
  if (!k.size(0) || !k.size(1) || !k.size(2)) return false;
  a.ka = factor_of<TpaFactor>(k); a.kb = factor_of<TpaFactor>(k, h);
  a.va = factor_of<TpaFactor>(v); a.vb = factor_of<TpaFactor>(v, h);
  a.k_cache = factor_of<TpaFactor>(kc); a.v_cache = factor_of<TpaFactor>(vc);
  a.slots = ids_ptr(slots);
  a.page_size = std::max((int)kc.size(1), 1);
  a.num_slots = (int)(kc.size(0) * kc.size(1));
  a.B = (int)k.size(0); a.l = (int)k.size(1); a.rk = (int)k.size(2); a.H = (int)h; a.dk = (int)(k.size(3) - h); a.dv = (int)(v.size(3) - h);
  a.dtype = dtype_code(k.scalar_type());
  return true;
}

// cache_write_fp4(k, v, slots, k_cache, v_cache, num_heads)
PyObject* cache_write_fp4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("cache_write_fp4", n, 6);
  if (!gpu_tensors(args + 3, 2)) throw Raise{PyExc_TypeError, "the cache is written in place: k_cache and v_cache must be GPU tensors"};
  if (!gpu_tensors(args, 3)) Py_RETURN_NOTIMPLEMENTED;
  const Tensor k = THPVariable_Unpack(args[0]), v = THPVariable_Unpack(args[1]), kc = THPVariable_Unpack(args[3]), vc = THPVariable_Unpack(args[4]);
  Tensor slots = THPVariable_Unpack(args[2]);
  const int64_t h = integer(args[5]);
  one_device({k, v, slots, kc, vc});
  if (k.dim() != 4 || v.dim() != 4) throw Raise{PyExc_ValueError, "k, v must be [b, l, r, h + d]"};
  expect(v.sizes().slice(0, 3) == k.sizes().slice(0, 3), v);
  if (!(0 < h && h < k.size(3) && h < v.size(3))) throw Raise{PyExc_AssertionError, "num_heads = " + std::to_string(h) + ", " + sizes_of(k) + ", " + sizes_of(v)};
  const Tensor two[2] = {k, v};
  static const char* const names[2] = {"k", "v"};
  check_dtypes(two, names, 2);
  (void)dtype_code(k.scalar_type());
  check_fp4_cache(kc, "k_cache", k.size(2), h, k.size(3) - h);
  check_fp4_cache(vc, "v_cache", v.size(2), h, v.size(3) - h);
  {
    WithoutGil free;
    const c10::DeviceGuard guard(k.device());
    slots = ints(slots);
    TpaFp4RowsArgs a{};
    if (describe_fp4_rows(k, v, kc, vc, slots, h, "tpa_cache_write_fp4", a)) {
      check("tpa_cache_write_fp4", lib.tpa_cache_write_fp4(&a, stream_of(k.device())));
      written(kc);
      written(vc);
    }
  }
  Py_RETURN_NONE;
  END_CALL
}

// cache_read_fp4(k_cache, v_cache, slots, num_heads, head_dim, v_head_dim, bf16)
PyObject* cache_read_fp4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("cache_read_fp4", n, 7);
  if (!gpu_tensors(args, 3)) Py_RETURN_NOTIMPLEMENTED;
  const Tensor kc = THPVariable_Unpack(args[0]), vc = THPVariable_Unpack(args[1]);
  Tensor slots = THPVariable_Unpack(args[2]), k, v;
  const int64_t h = integer(args[3]), dk = integer(args[4]), dv = integer(args[5]);
  const at::ScalarType dtype = integer(args[6]) ? at::kBFloat16 : at::kFloat;
  one_device({kc, vc, slots});
  if (h <= 0 || dk <= 0 || dv <= 0) throw Raise{PyExc_ValueError, "num_heads and the head sizes must be positive"};
  if (kc.dim() != 4) throw Raise{PyExc_ValueError, "k_cache must be [pages, page_size, rk, bytes], got " + sizes_of(kc)};
  check_fp4_cache(kc, "k_cache", kc.size(2), h, dk);
  check_fp4_cache(vc, "v_cache", kc.size(2), h, dv);
  if (slots.dim() != 2) throw Raise{PyExc_ValueError, "slots must be [b, l], got " + sizes_of(slots)};
  {
    WithoutGil free;
    const c10::DeviceGuard guard(kc.device());
    slots = ints(slots);
    const auto options = at::TensorOptions().device(kc.device()).dtype(dtype);
    k = at::empty({slots.size(0), slots.size(1), kc.size(2), h + dk}, options);
    v = at::empty({slots.size(0), slots.size(1), kc.size(2), h + dv}, options);
    TpaFp4RowsArgs a{};
    if (describe_fp4_rows(k, v, kc, vc, slots, h, "tpa_cache_read_fp4", a)) check("tpa_cache_read_fp4", lib.tpa_cache_read_fp4(&a, stream_of(kc.device())));
  }
  return tuple_of({k, v});
  END_CALL
}

// decode_fp4(qa, qb, k_cache, v_cache, kv_lengths, page_table, workspace, sm_scale, kernel, causal, causal_offset, v_head_dim)
PyObject* decode_fp4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("decode_fp4", n, 12);
  if (!gpu_tensors(args, 4) || !none_or_gpu(args[4]) || !none_or_gpu(args[5]) || !none_or_gpu(args[6])) Py_RETURN_NOTIMPLEMENTED;
  const Tensor qa = THPVariable_Unpack(args[0]), qb = THPVariable_Unpack(args[1]), kc = THPVariable_Unpack(args[2]), vc = THPVariable_Unpack(args[3]);
  Tensor pages = tensor_or_none(args[5]), ws = tensor_or_none(args[6]);
  one_device({qa, qb, kc, vc, tensor_or_none(args[4]), pages, ws});
  TpaDecodeFp4Args a{};
  a.sm_scale = (float)real(args[7]);
  a.kernel = (int)integer(args[8]);
  a.causal = (int)integer(args[9]);
  a.causal_offset = (int)integer(args[10]);
  const int64_t given_dv = integer(args[11]);
  if (qa.dim() != 4 || qb.dim() != 4) throw Raise{PyExc_ValueError, "qa, qb must be [b, lq, rq, x], got " + sizes_of(qa) + ", " + sizes_of(qb)};
  expect(qb.sizes().slice(0, 3) == qa.sizes().slice(0, 3), qb);
  const Tensor two[2] = {qa, qb};
  static const char* const names[2] = {"qa", "qb"};
  check_dtypes(two, names, 2);
  a.dtype = dtype_code(qa.scalar_type());
  const int64_t h = qa.size(3), dk = qb.size(3), dv = given_dv == kNotGiven ? dk : given_dv;
  if (h <= 0 || dk <= 0 || dv <= 0 || qa.size(2) <= 0) throw CallFailed{"tpa_decode_fp4", TPA_ERR_SHAPE};
  if (kc.dim() != 4) throw Raise{PyExc_ValueError, "k_cache must be [pages, page_size, rk, bytes], got " + sizes_of(kc)};
  check_fp4_cache(kc, "k_cache", kc.size(2), h, dk);
  check_fp4_cache(vc, "v_cache", kc.size(2), h, dv);
  expect(kc.sizes().slice(0, 3) == vc.sizes().slice(0, 3), vc);
  fits_int({qa.size(0), qa.size(1), qa.size(2), h, dk, dv, kc.size(0), kc.size(1), kc.size(2)}, "tpa_decode_fp4");
  std::pair<Tensor, Tensor> r;
  {
    WithoutGil free;
    const at::Device device = qa.device();
    const c10::DeviceGuard guard(device);
    a.B = (int)qa.size(0); a.lq = (int)qa.size(1); a.rq = (int)qa.size(2); a.H = (int)h; a.dk = (int)dk; a.dv = (int)dv; a.rk = (int)kc.size(2);
    if (pages.defined()) {
      pages = ints(pages);
      expect(pages.dim() == 2 && pages.size(0) == a.B, pages);
      fits_int({pages.size(1), pages.size(1) * kc.size(1)}, "tpa_decode_fp4");
      a.page_table = ids_ptr(pages);
      a.page_size = (int)kc.size(1);
      a.pages_per_seq = (int)pages.size(1);
      a.num_pages = (int)kc.size(0);
      a.lk = a.page_size * a.pages_per_seq;
    } else {
      expect(kc.size(0) == a.B, kc);
      a.lk = (int)kc.size(1);
    }
    a.qa = factor_of<TpaFactor>(qa); a.qb = factor_of<TpaFactor>(qb);
    a.k_cache = factor_of<TpaFactor>(kc); a.v_cache = factor_of<TpaFactor>(vc);
    const Tensor kvlen = lengths(tensor_or_none(args[4]), a.B);
    a.kv_lengths = ids_ptr(kvlen);
    // output and logsumexp in one allocation
    const int64_t first = ((int64_t)a.B * a.lq * a.H * a.dv * qa.element_size() + 255) / 256 * 256;
    const Tensor all = bytes_on(device, first + (int64_t)4 * a.B * a.H * a.lq);
    auto part = [&](int64_t at, at::ScalarType type, std::initializer_list<int64_t> sizes) {
      Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(type));
      t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
      t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
      return t;
    };
    r.first = part(0, qa.scalar_type(), {a.B, a.lq, a.H, a.dv});
    r.second = part(first, at::kFloat, {a.B, a.H, a.lq});
    if (r.first.numel() && a.lk && kc.numel() && vc.numel()) {
      const size_t need = lib.tpa_decode_fp4_workspace_bytes(&a);
      if (!ws.defined() && need) ws = bytes_on(device, need + 256);
      if (ws.defined()) take_workspace(ws, 256, a);
      a.o = r.first.data_ptr();
      a.lse = f32_ptr(r.second);
      check("tpa_decode_fp4", lib.tpa_decode_fp4(&a, stream_of(device)));
    } else {  // no rows, or none that sees a key
      r.first.fill_(NAN);
      r.second.fill_(-INFINITY);
    }
  }
  return pair(std::move(r));
  END_CALL
}

// ------------------------------------------------------------------------------------------------ beams
// beam_select(logits, scores, finished, num_out, eos_token)
PyObject* beam_select(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("beam_select", n, 5);
  if (!gpu_tensors(args, 2) || !none_or_gpu(args[2])) Py_RETURN_NOTIMPLEMENTED;
  Tensor logits = THPVariable_Unpack(args[0]), scores = THPVariable_Unpack(args[1]), finished = tensor_or_none(args[2]), out[4];
  const int64_t given = integer(args[3]), eos = integer(args[4]);
  one_device({logits, scores, finished});
  if (logits.dim() != 3) throw Raise{PyExc_ValueError, "logits must be [b, beams, vocab], got " + sizes_of(logits)};
  const int64_t b = logits.size(0), beams = logits.size(1), vocab = logits.size(2), k = given == kNotGiven ? beams : given;
  const int dtype = dtype_code(logits.scalar_type());
  for (const Tensor* t : {&scores, &finished})
    if (t->defined() && !is_shape(*t, {b, beams}))
      throw Raise{PyExc_ValueError, std::string(t == &scores ? "scores" : "finished") + " must have shape (" + std::to_string(b) + ", " + std::to_string(beams) + "), got " + sizes_of(*t)};
  if (!at::isFloatingType(scores.scalar_type())) throw Raise{PyExc_TypeError, std::string("scores are floating-point numbers, got ") + c10::toString(scores.scalar_type())};
  if (finished.defined() && finished.scalar_type() != at::kBool) throw Raise{PyExc_TypeError, std::string("finished holds truth values, got ") + c10::toString(finished.scalar_type())};
  if (finished.defined() && eos < 0) throw Raise{PyExc_ValueError, "finished beams need an eos_token"};
  if (eos < -1 || eos >= vocab) throw Raise{PyExc_ValueError, "eos_token must be below the vocabulary's " + std::to_string(vocab) + ", got " + std::to_string(eos)};
  if (k < 1 || beams < 1 || vocab < 1 || k > beams * vocab)
    throw Raise{PyExc_ValueError, "num_out must be between 1 and beams * vocab, got " + std::to_string(k) + " of " + sizes_of(logits)};
  fits_int({b, beams, vocab, k}, "tpa_beam_select");
  {
    WithoutGil free;
    const at::Device device = logits.device();
    const c10::DeviceGuard guard(device);
    if (vocab > 1 && logits.stride(2) != 1) logits = logits.contiguous();
    if (scores.scalar_type() != at::kFloat) scores = scores.to(at::kFloat);
    scores = scores.contiguous();
    if (finished.defined()) finished = finished.contiguous();
    // one allocation for four small results, each at a multiple of 256 bytes
    const int64_t each = (b * k * 4 + 255) / 256 * 256;
    const Tensor all = bytes_on(device, 4 * each);
    const at::ScalarType types[4] = {at::kFloat, at::kInt, at::kInt, at::kBool};
    for (int i = 0; i < 4; ++i) {
      out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), c10::scalarTypeToTypeMeta(types[i]));
      out[i].unsafeGetTensorImpl()->set_storage_offset(i * each / (int64_t)c10::elementSize(types[i]));
      out[i].unsafeGetTensorImpl()->set_sizes_contiguous({b, k});
    }
    if (b) {
      TpaBeamSelectArgs a{};
      a.logits = logits.data_ptr();
      a.stride_b = logits.stride(0); a.stride_n = logits.stride(1);
      a.scores = f32_ptr(scores);
      a.finished = finished.defined() ? static_cast<const uint8_t*>(finished.data_ptr()) : nullptr;
      a.new_scores = f32_ptr(out[0]);
      a.parents = static_cast<int32_t*>(out[1].data_ptr());
      a.tokens = static_cast<int32_t*>(out[2].data_ptr());
      a.new_finished = static_cast<uint8_t*>(out[3].data_ptr());
      a.B = (int)b; a.beams = (int)beams; a.vocab = (int)vocab; a.num_out = (int)k; a.eos_token = (int)eos; a.dtype = dtype;
      const Tensor ws = bytes_on(device, lib.tpa_beam_select_workspace_bytes(a.B, a.beams, a.vocab, a.num_out, a.dtype) + 16);
      take_workspace(ws, 16, a);
      check("tpa_beam_select", lib.tpa_beam_select(&a, stream_of(device)));
    }
  }
  return tuple_of({out[0], out[1], out[2], out[3]});
  END_CALL
}

// ------------------------------------------------------------------------------------------------ pages between sequences
// The pools of a call: GPU tensors [num_pages, page_size, ..] whose pages have no gaps
std::vector<Tensor> pools_of(PyObject* arg) {
  PyObject* const list = PySequence_Fast(arg, "pools is a list of tensors");
  if (!list) throw python_error();
  std::vector<Tensor> pools;
  bool ok = true;
  for (Py_ssize_t i = 0; ok && i < PySequence_Fast_GET_SIZE(list); ++i) {
    PyObject* const item = PySequence_Fast_GET_ITEM(list, i);
    ok = gpu_tensors(&item, 1);
    if (ok) pools.push_back(THPVariable_Unpack(item));
  }
  Py_DECREF(list);
  if (!ok) throw Raise{PyExc_TypeError, "pages are moved in place: pools must be GPU tensors"};
  return pools;
}
std::vector<TpaPool> describe_pools(const std::vector<Tensor>& pools, int64_t num_pages, int64_t page_size) {
  std::vector<TpaPool> out;
  for (const Tensor& t : pools) {
    if (t.dim() < 2 || t.size(0) != num_pages || t.size(1) != page_size)
      throw Raise{PyExc_ValueError, "pools must be [" + std::to_string(num_pages) + ", " + std::to_string(page_size) + ", ..], got " + sizes_of(t)};
    if (!t.numel()) continue;  // nothing in a page
    int64_t each = 1;          // elements of a token, then of a page
    bool whole = true;
    for (int64_t d = t.dim() - 1; d >= 1; --d) {
      if (t.size(d) > 1 && t.stride(d) != each) whole = false;
      each *= t.size(d);
    }
    if (!whole || (num_pages > 1 && t.stride(0) < each)) throw Raise{PyExc_ValueError, "the pages of a pool must be contiguous and apart"};
    const int64_t e = t.element_size();
    out.push_back(TpaPool{t.data_ptr(), std::max(t.stride(0), each) * e, each / page_size * e});
  }
  return out;
}
// int32 results of the given sizes in one allocation
void allocate_ints(const at::Device& device, std::initializer_list<std::vector<int64_t>> shapes, Tensor* out) {
  int64_t at = 0, total = 0;
  auto room = [](const std::vector<int64_t>& s) {
    int64_t n = 1;
    for (int64_t x : s) n *= x;
    return (n + 63) / 64 * 64;
  };
  for (const auto& s : shapes) total += room(s);
  const Tensor all = at::empty({total}, at::TensorOptions().device(device).dtype(at::kInt));
  int i = 0;
  for (const auto& s : shapes) {
    out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    out[i].unsafeGetTensorImpl()->set_storage_offset(at);
    out[i++].unsafeGetTensorImpl()->set_sizes_contiguous(s);
    at += room(s);
  }
}
// what both calls take: a table, lengths, counts, a list of free pages and the place in it
struct PageState {
  Tensor table, len, shares, free, start;
  int64_t page_size = 0;
};
void check_page_state(const PageState& s, const char* name) {
  if (s.table.dim() != 2) throw Raise{PyExc_ValueError, "page_table must be [b, pages_per_seq], got " + sizes_of(s.table)};
  const int64_t b = s.table.size(0);
  if (!is_shape(s.len, {b})) throw Raise{PyExc_ValueError, "kv_lengths must have shape (" + std::to_string(b) + ",), got " + sizes_of(s.len)};
  if (s.shares.dim() != 1 || !s.shares.size(0)) throw Raise{PyExc_ValueError, "page_shares has a number for every page, got shape " + sizes_of(s.shares)};
  if (s.free.dim() != 1) throw Raise{PyExc_ValueError, "free_pages is a list of pages, got shape " + sizes_of(s.free)};
  if (s.start.defined() && s.start.numel() != 1) throw Raise{PyExc_ValueError, "free_start is one number, got shape " + sizes_of(s.start)};
  if (s.page_size < 1 || s.page_size > INT32_MAX) throw Raise{PyExc_ValueError, "page_size must be positive, got " + std::to_string(s.page_size)};
  if (!s.table.size(1)) throw Raise{PyExc_ValueError, "page_table must be [b, pages_per_seq], got " + sizes_of(s.table)};
  fits_int({b, s.table.size(1), s.shares.size(0), s.free.size(0)}, name);
}
void settle(PageState& s) {
  s.table = ints(s.table);
  s.len = ints(s.len);
  s.shares = ints(s.shares);
  s.free = ints(s.free);
  if (s.start.defined()) s.start = ints(s.start);
}
template <typename Args>
void describe_pages(const PageState& s, const std::vector<TpaPool>& pools, Args& a) {
  a.page_table = ids_ptr(s.table); a.kv_lengths = ids_ptr(s.len); a.page_shares = ids_ptr(s.shares); a.free_pages = ids_ptr(s.free); a.free_start = ids_ptr(s.start);
  a.pools = pools.data(); a.num_pools = (int)pools.size();
  a.B = (int)s.table.size(0); a.pages_per_seq = (int)s.table.size(1); a.page_size = (int)s.page_size;
  a.num_pages = (int)s.shares.size(0); a.num_free = (int)s.free.size(0);
}
int32_t* int_ptr(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// pages_fork(page_table, kv_lengths, parents, page_shares, free_pages, free_start, pools, page_size)
PyObject* pages_fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("pages_fork", n, 8);
  if (!gpu_tensors(args, 5) || !none_or_gpu(args[5])) Py_RETURN_NOTIMPLEMENTED;
  PageState s;
  s.table = THPVariable_Unpack(args[0]); s.len = THPVariable_Unpack(args[1]); s.shares = THPVariable_Unpack(args[3]); s.free = THPVariable_Unpack(args[4]);
  s.start = tensor_or_none(args[5]);
  Tensor parents = THPVariable_Unpack(args[2]), out[5];
  const std::vector<Tensor> pools = pools_of(args[6]);
  s.page_size = integer(args[7]);
  one_device({s.table, s.len, parents, s.shares, s.free, s.start});
  for (const Tensor& t : pools) one_device({s.table, t});
  check_page_state(s, "tpa_pages_fork");
  if (parents.dim() < 1) throw Raise{PyExc_ValueError, "parents has a number for every new sequence, got shape " + sizes_of(parents)};
  fits_int({parents.numel()}, "tpa_pages_fork");
  const std::vector<TpaPool> described = describe_pools(pools, s.shares.size(0), s.page_size);
  {
    WithoutGil free;
    const at::Device device = s.table.device();
    const c10::DeviceGuard guard(device);
    settle(s);
    parents = ints(parents);
    const int64_t m = parents.numel();
    allocate_ints(device, {{m, s.table.size(1)}, {m}, {s.shares.size(0)}, {s.free.size(0)}, {1}}, out);
    TpaPagesForkArgs a{};
    describe_pages(s, described, a);
    a.parents = ids_ptr(parents);
    a.M = (int)m;
    a.new_page_table = int_ptr(out[0]); a.new_kv_lengths = int_ptr(out[1]); a.new_page_shares = int_ptr(out[2]);
    a.new_free_pages = int_ptr(out[3]); a.new_free_start = int_ptr(out[4]);
    Tensor ws;
    if (const size_t need = lib.tpa_pages_workspace_bytes(a.B, a.M, a.num_pages, a.num_pools)) take_workspace(ws = bytes_on(device, need + 16), 16, a);
    check("tpa_pages_fork", lib.tpa_pages_fork(&a, stream_of(device)));
    for (const Tensor& t : pools) written(t);
  }
  return tuple_of({out[0], out[1], out[2], out[3], out[4]});
  END_CALL
}

// pages_compact(page_table, kv_lengths, page_shares, free_pages, free_start, pools, page_size)
PyObject* pages_compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
  BEGIN_CALL
  count("pages_compact", n, 7);
  if (!gpu_tensors(args, 4) || !none_or_gpu(args[4])) Py_RETURN_NOTIMPLEMENTED;
  PageState s;
  s.table = THPVariable_Unpack(args[0]); s.len = THPVariable_Unpack(args[1]); s.shares = THPVariable_Unpack(args[2]); s.free = THPVariable_Unpack(args[3]);
  s.start = tensor_or_none(args[4]);
  Tensor out[5];
  const std::vector<Tensor> pools = pools_of(args[5]);
  s.page_size = integer(args[6]);
  one_device({s.table, s.len, s.shares, s.free, s.start});
  for (const Tensor& t : pools) one_device({s.table, t});
  check_page_state(s, "tpa_pages_compact");
  const std::vector<TpaPool> described = describe_pools(pools, s.shares.size(0), s.page_size);
  {
    WithoutGil free;
    const at::Device device = s.table.device();
    const c10::DeviceGuard guard(device);
    settle(s);
    allocate_ints(device, {{s.table.size(0), s.table.size(1)}, {s.shares.size(0)}, {s.free.size(0)}, {1}, {s.shares.size(0)}}, out);
    TpaPagesCompactArgs a{};
    describe_pages(s, described, a);
    a.new_page_table = int_ptr(out[0]); a.new_page_shares = int_ptr(out[1]); a.new_free_pages = int_ptr(out[2]); a.new_free_start = int_ptr(out[3]);
    a.moved = int_ptr(out[4]);
    Tensor ws;
    if (const size_t need = lib.tpa_pages_workspace_bytes(a.B, 0, a.num_pages, a.num_pools)) take_workspace(ws = bytes_on(device, need + 16), 16, a);
    check("tpa_pages_compact", lib.tpa_pages_compact(&a, stream_of(device)));
    for (const Tensor& t : pools) written(t);
  }
  return tuple_of({out[0], out[1], out[2], out[3], out[4]});
  END_CALL
}

// ------------------------------------------------------------------------------------------------ module
// bind(path of libtpa_gfx950.so, TpaError)
PyObject* bind(PyObject*, PyObject* args) {
  const char* path;
  PyObject* cls;
  if (!PyArg_ParseTuple(args, "sO", &path, &cls)) return nullptr;
  void* h = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (!h) {
    PyErr_SetString(PyExc_RuntimeError, dlerror());
    return nullptr;
  }
#define X(name)                                                                           \
  lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(h, #name));                       \
  if (!lib.name) {                                                                        \
    PyErr_SetString(PyExc_RuntimeError, "the library does not export " #name);            \
    return nullptr;                                                                       \
  }
  TPA_CALLS(X)
#undef X
  Py_INCREF(cls);
  error_class = cls;
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(factors), FAST(decode), FAST(append), FAST(backward), FAST(tpa), FAST(decode_shared), FAST(page_tables),
                         FAST(norm_rope), FAST(norm_rope_backward), FAST(norm_rope_write),
                         FAST(cache_write_fp4), FAST(cache_read_fp4), FAST(decode_fp4), FAST(beam_select), FAST(pages_fork), FAST(pages_compact), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "tpa_host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_tpa_host_calls() { return PyModule_Create(&module); }

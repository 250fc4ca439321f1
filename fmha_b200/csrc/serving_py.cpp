// serving_py.cpp -- the Python side of the paged-cache calls (fmha_b200._serving,
// used by serving.py): checks the tensors, allocates outputs and workspace on
// torch's current stream, and calls the C ABI. A decode step makes these calls
// once per layer and the kernels of small batches take a few microseconds, so
// the host's time is what they cost: the same checks written in Python took 6 to
// 8 us a call, here about 1.
//
// Arguments come by position, in the order that serving.py passes them. The
// C entry points and the exception class are handed over once by bind().
#include <Python.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "../../include/fmha.h"

namespace {

using at::ScalarType;
using at::Tensor;

decltype(&fmha_rope_append) g_append;
decltype(&fmha_paged_decode) g_decode;
decltype(&fmha_paged_decode_workspace) g_workspace;
decltype(&fmha_prompt) g_prompt;
PyObject* g_error;  // FmhaError(status, what)

struct Refused {
  int status;
  std::string why;
};

[[noreturn]] void refuse(const std::string& why, int status = FMHA_ERR_INVALID_ARG) {
  throw Refused{status, why};
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Refused{-1, std::string(name) + " must be a tensor"};
  return THPVariable_Unpack(o);
}

double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Refused{-2, ""};
  return x;
}

bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw Refused{-2, ""};
  return x != 0;
}

int type_code(ScalarType t, const char* name) {
  if (t == at::kBFloat16) return FMHA_DTYPE_BF16;
  if (t == at::kHalf) return FMHA_DTYPE_FP16;
  refuse(std::string(name) + " must be bf16 or fp16", FMHA_ERR_UNSUPPORTED);
}

// A [tokens, heads, d] operand with adjacent heads; its token stride.
int64_t rows(const Tensor& t, const char* name, int64_t tokens, int64_t heads, int64_t d,
             ScalarType type, int device) {
  if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != d ||
      t.scalar_type() != type || !t.is_cuda() || t.get_device() != device)
    refuse(std::string(name) + " must be " + c10::toString(type) + " [" + std::to_string(tokens) +
           ", " + std::to_string(heads) + ", " + std::to_string(d) + "] on cuda:" +
           std::to_string(device));
  if ((t.stride(2) != 1 && d > 1) || (t.stride(1) != d && heads > 1))
    refuse(std::string(name) + "'s heads must be adjacent (strides (*, " + std::to_string(d) + ", 1))");
  return tokens > 1 ? t.stride(0) : heads * d;
}

const int32_t* ints(const Tensor& t, const char* name, int64_t n, int device) {
  if (t.dim() != 1 || t.size(0) != n || t.scalar_type() != at::kInt || !t.is_cuda() ||
      t.get_device() != device || (n > 1 && t.stride(0) != 1))
    refuse(std::string(name) + " must be " + std::to_string(n) + " adjacent int32 on cuda:" +
           std::to_string(device));
  return static_cast<const int32_t*>(t.data_ptr());
}

// The cache's struct; Hkv and the batch.
fmha_paged_cache_t pages(const Tensor& k, const Tensor& v, const Tensor& table,
                         const Tensor& seqlens, int64_t d, double k_scale, double v_scale,
                         int device, int64_t* hkv, int64_t* batch) {
  if (k.dim() != 4 || k.size(3) != d || v.sizes() != k.sizes())
    refuse("k_pages and v_pages must be [num_pages, Hkv, page_size, " + std::to_string(d) + "]");
  if (v.strides() != k.strides() || k.stride(3) != 1)
    refuse("k_pages and v_pages must have equal strides and adjacent elements");
  const ScalarType type = k.scalar_type();
  if (v.scalar_type() != type)
    refuse("k_pages and v_pages must have one type", FMHA_ERR_UNSUPPORTED);
  int code = FMHA_DTYPE_E4M3;
  if (type == at::kBFloat16) code = FMHA_DTYPE_BF16;
  else if (type == at::kHalf) code = FMHA_DTYPE_FP16;
  else if (type != at::kFloat8_e4m3fn)
    refuse("pages must be bf16, fp16 or float8_e4m3fn", FMHA_ERR_UNSUPPORTED);
  if (!k.is_cuda() || !v.is_cuda() || !table.is_cuda() || k.get_device() != device ||
      v.get_device() != device || table.get_device() != device)
    refuse("pages and block_table must be on cuda:" + std::to_string(device));
  if (table.dim() != 2 || table.scalar_type() != at::kInt ||
      (table.size(1) > 1 && table.stride(1) != 1))
    refuse("block_table must be int32 [batch, max_pages] with adjacent columns");
  if (k.size(0) > INT32_MAX || k.size(1) > INT32_MAX || k.size(2) > INT32_MAX ||
      table.size(0) > INT32_MAX || table.size(1) > INT32_MAX)
    refuse("a size beyond 2^31", FMHA_ERR_UNSUPPORTED);
  *hkv = k.size(1);
  *batch = table.size(0);
  fmha_paged_cache_t c;
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.block_table = static_cast<const int32_t*>(table.data_ptr());
  c.seqlens_kv = ints(seqlens, "seqlens_kv", *batch, device);
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.token_stride = k.stride(2);
  c.table_stride = table.stride(0);
  c.num_pages = (int32_t)k.size(0);
  c.page_size = (int32_t)k.size(2);
  c.max_pages = (int32_t)table.size(1);
  c.dtype = code;
  c.k_scale = (float)k_scale;
  c.v_scale = (float)v_scale;
  return c;
}

// q of a call: 3 dimensions on a CUDA device.
struct Query {
  const Tensor& q;
  int64_t tokens, heads, d;
  int device, code;
  ScalarType type;
  explicit Query(PyObject* o) : q(tensor(o, "q")) {
    if (!q.is_cuda()) refuse("q must be a CUDA tensor");
    if (q.dim() != 3) refuse("q must be [tokens, heads, head_dim]");
    tokens = q.size(0);
    heads = q.size(1);
    d = q.size(2);
    device = q.get_device();
    type = q.scalar_type();
    code = type_code(type, "q");
    if (tokens > INT32_MAX || heads > INT32_MAX || d > INT32_MAX)
      refuse("a size beyond 2^31", FMHA_ERR_UNSUPPORTED);
  }
};

fmha_stream_t stream_of(int device) {
  return reinterpret_cast<fmha_stream_t>(c10::cuda::getCurrentCUDAStream(device).stream());
}

// The output (given, or new), its type's code and its token stride.
Tensor output(const Query& Q, PyObject* o, PyObject* out_dtype, int* code, int64_t* stride) {
  ScalarType want = at::kHalf;
  if (out_dtype != Py_None) {
    if (!THPDtype_Check(out_dtype)) throw Refused{-1, "out_dtype must be a torch.dtype"};
    want = reinterpret_cast<THPDtype*>(out_dtype)->scalar_type;
  }
  if (o == Py_None) {
    *code = type_code(want, "out_dtype");
    *stride = Q.heads * Q.d;
    return at::empty({Q.tokens, Q.heads, Q.d}, Q.q.options().dtype(want));
  }
  const Tensor& t = tensor(o, "o");
  if (out_dtype != Py_None && t.scalar_type() != want)
    refuse(std::string("o must be ") + c10::toString(want));
  *code = type_code(t.scalar_type(), "o");
  *stride = rows(t, "o", Q.tokens, Q.heads, Q.d, t.scalar_type(), Q.device);
  return t;
}

float* lse_of(PyObject* o, const Query& Q) {
  if (o == Py_None) return nullptr;
  const Tensor& t = tensor(o, "lse");
  if (t.dim() != 2 || t.size(0) != Q.tokens || t.size(1) != Q.heads ||
      t.scalar_type() != at::kFloat || !t.is_cuda() || t.get_device() != Q.device ||
      !t.is_contiguous())
    refuse("lse must be contiguous fp32 [" + std::to_string(Q.tokens) + ", " +
           std::to_string(Q.heads) + "] on cuda:" + std::to_string(Q.device));
  return static_cast<float*>(t.data_ptr());
}

void done(fmha_status_t st) {
  if (st != FMHA_OK) refuse("", st);
}

// Runs `body`; a refusal becomes FmhaError(status, "what: why") or a TypeError.
template <class Body>
PyObject* call(const char* what, Py_ssize_t have, Py_ssize_t want, Body body) {
  if (have != want) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", what, want);
    return nullptr;
  }
  try {
    return body();
  } catch (const Refused& r) {
    if (r.status == -2) return nullptr;  // a Python error is set
    const std::string text = r.why.empty() ? std::string(what) : std::string(what) + ": " + r.why;
    if (r.status < 0) {
      PyErr_SetString(PyExc_TypeError, text.c_str());
      return nullptr;
    }
    PyObject* const e = PyObject_CallFunction(g_error, "is", r.status, text.c_str());
    if (e) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// (q, k, v, k_pages, v_pages, block_table, seqlens_kv, cos, sin, cu_seqlens_q,
//  interleaved, k_scale, v_scale, q_out, k_out, return_k)
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call("fmha_rope_append", n, 16, [&]() -> PyObject* {
    const Query Q(a[0]);
    const c10::cuda::CUDAGuard guard(Q.device);
    const Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
    fmha_rope_append_args_t A;
    int64_t hkv, batch;
    A.cache = pages(tensor(a[3], "k_pages"), tensor(a[4], "v_pages"), tensor(a[5], "block_table"),
                    tensor(a[6], "seqlens_kv"), Q.d, number(a[11]), number(a[12]), Q.device, &hkv,
                    &batch);
    A.q_stride = rows(Q.q, "q", Q.tokens, Q.heads, Q.d, Q.type, Q.device);
    A.k_stride = rows(k, "k", Q.tokens, hkv, Q.d, Q.type, Q.device);
    A.v_stride = rows(v, "v", Q.tokens, hkv, Q.d, Q.type, Q.device);
    A.cu_seqlens_q =
        a[9] == Py_None ? nullptr
                        : ints(tensor(a[9], "cu_seqlens_q"), "cu_seqlens_q", batch + 1, Q.device);
    A.cos_table = A.sin_table = nullptr;
    A.rotary_dim = A.max_position = 0;
    if ((a[7] == Py_None) != (a[8] == Py_None)) refuse("cos and sin go together");
    if (a[7] != Py_None) {
      const Tensor &c = tensor(a[7], "cos"), &s = tensor(a[8], "sin");
      for (const Tensor* t : {&c, &s})
        if (t->dim() != 2 || t->sizes() != c.sizes() || t->scalar_type() != at::kFloat ||
            !t->is_contiguous() || !t->is_cuda() || t->get_device() != Q.device ||
            t->size(0) > INT32_MAX || t->size(1) > 1024)
          refuse("cos and sin must be contiguous fp32 [max_position, rotary_dim/2]");
      A.cos_table = static_cast<const float*>(c.data_ptr());
      A.sin_table = static_cast<const float*>(s.data_ptr());
      A.max_position = (int32_t)c.size(0);
      A.rotary_dim = (int32_t)(2 * c.size(1));
    }
    Tensor q_out, k_out;
    A.q_out_stride = Q.heads * Q.d;
    if (a[13] == Py_None) {
      q_out = at::empty({Q.tokens, Q.heads, Q.d}, Q.q.options());
    } else {
      q_out = tensor(a[13], "q_out");
      A.q_out_stride = rows(q_out, "q_out", Q.tokens, Q.heads, Q.d, Q.type, Q.device);
    }
    A.k_out = nullptr;
    A.k_out_stride = hkv * Q.d;
    const bool with_k = a[14] != Py_None || truth(a[15]);
    if (a[14] != Py_None) {
      k_out = tensor(a[14], "k_out");
      A.k_out_stride = rows(k_out, "k_out", Q.tokens, hkv, Q.d, Q.type, Q.device);
    } else if (with_k) {
      k_out = at::empty({Q.tokens, hkv, Q.d}, Q.q.options());
    }
    if (with_k) A.k_out = k_out.data_ptr();
    A.q = Q.q.data_ptr();
    A.k = k.data_ptr();
    A.v = v.data_ptr();
    A.q_out = q_out.data_ptr();
    A.total_tokens = (int32_t)Q.tokens;
    A.batch = (int32_t)batch;
    A.num_heads_q = (int32_t)Q.heads;
    A.num_heads_kv = (int32_t)hkv;
    A.head_dim = (int32_t)Q.d;
    A.interleaved = truth(a[10]);
    A.dtype = Q.code;
    done(g_append(&A, stream_of(Q.device)));
    PyObject* const first = THPVariable_Wrap(std::move(q_out));
    if (!with_k) return first;
    PyObject* const second = THPVariable_Wrap(std::move(k_out));
    PyObject* const both = PyTuple_Pack(2, first, second);
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
  });
}

// (q, k_pages, v_pages, block_table, seqlens_kv, softmax_scale, k_scale, v_scale,
//  o, out_dtype, lse, workspace)
PyObject* paged_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call("fmha_paged_decode", n, 12, [&]() -> PyObject* {
    const Query Q(a[0]);
    const c10::cuda::CUDAGuard guard(Q.device);
    fmha_paged_decode_args_t A;
    int64_t hkv, batch;
    A.cache = pages(tensor(a[1], "k_pages"), tensor(a[2], "v_pages"), tensor(a[3], "block_table"),
                    tensor(a[4], "seqlens_kv"), Q.d, number(a[6]), number(a[7]), Q.device, &hkv,
                    &batch);
    if (batch != Q.tokens) refuse("q and block_table must have the same batch");
    A.q_stride = rows(Q.q, "q", Q.tokens, Q.heads, Q.d, Q.type, Q.device);
    Tensor o = output(Q, a[8], a[9], &A.o_dtype, &A.o_stride);
    A.lse = lse_of(a[10], Q);
    // Negative for heads that the call refuses: it says so itself.
    const int64_t need = g_workspace((int)Q.heads, (int)hkv, (int)Q.d,
                                     (int64_t)A.cache.max_pages * A.cache.page_size);
    Tensor scratch;
    A.workspace = nullptr;
    A.workspace_bytes = 0;
    if (a[11] != Py_None) {
      const Tensor& w = tensor(a[11], "workspace");
      if (!w.is_cuda() || w.get_device() != Q.device || !w.is_contiguous())
        refuse("workspace must be contiguous on cuda:" + std::to_string(Q.device));
      A.workspace = w.data_ptr();
      A.workspace_bytes = (int64_t)w.nbytes();
    } else if (need > 0) {
      scratch = at::empty({need}, Q.q.options().dtype(at::kByte));
      A.workspace = scratch.data_ptr();
      A.workspace_bytes = need;
    }
    A.q = Q.q.data_ptr();
    A.o = o.data_ptr();
    A.batch = (int32_t)batch;
    A.num_heads_q = (int32_t)Q.heads;
    A.num_heads_kv = (int32_t)hkv;
    A.head_dim = (int32_t)Q.d;
    A.dtype = Q.code;
    A.softmax_scale = (float)number(a[5]);
    done(g_decode(&A, stream_of(Q.device)));
    return THPVariable_Wrap(std::move(o));
  });
}

// (q, k, v, cu_seqlens_q, cu_seqlens_kv, causal, softmax_scale, o, out_dtype, lse)
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call("fmha_prompt", n, 10, [&]() -> PyObject* {
    const Query Q(a[0]);
    const c10::cuda::CUDAGuard guard(Q.device);
    const Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &cu = tensor(a[3], "cu_seqlens_q");
    if (k.dim() != 3 || k.size(0) > INT32_MAX || k.size(1) > INT32_MAX)
      refuse("k must be [tokens, heads, head_dim]");
    if (cu.dim() != 1 || cu.size(0) < 1 || cu.size(0) > INT32_MAX)
      refuse("cu_seqlens_q must be [batch + 1]");
    fmha_prompt_args_t A;
    const int64_t tk = k.size(0), hkv = k.size(1), batch = cu.size(0) - 1;
    A.q_stride = rows(Q.q, "q", Q.tokens, Q.heads, Q.d, Q.type, Q.device);
    A.k_stride = rows(k, "k", tk, hkv, Q.d, Q.type, Q.device);
    A.v_stride = rows(v, "v", tk, hkv, Q.d, Q.type, Q.device);
    A.cu_seqlens_q = ints(cu, "cu_seqlens_q", batch + 1, Q.device);
    A.cu_seqlens_kv =
        a[4] == Py_None ? nullptr
                        : ints(tensor(a[4], "cu_seqlens_kv"), "cu_seqlens_kv", batch + 1, Q.device);
    Tensor o = output(Q, a[7], a[8], &A.o_dtype, &A.o_stride);
    A.lse = lse_of(a[9], Q);
    A.q = Q.q.data_ptr();
    A.k = k.data_ptr();
    A.v = v.data_ptr();
    A.o = o.data_ptr();
    A.total_q = (int32_t)Q.tokens;
    A.total_kv = (int32_t)tk;
    A.batch = (int32_t)batch;
    A.num_heads_q = (int32_t)Q.heads;
    A.num_heads_kv = (int32_t)hkv;
    A.head_dim = (int32_t)Q.d;
    A.causal = truth(a[5]);
    A.dtype = Q.code;
    A.softmax_scale = (float)number(a[6]);
    done(g_prompt(&A, stream_of(Q.device)));
    return THPVariable_Wrap(std::move(o));
  });
}

// bind(FmhaError, addresses of fmha_rope_append, fmha_paged_decode,
//      fmha_paged_decode_workspace, fmha_prompt)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[4];
  PyObject* error;
  if (!PyArg_ParseTuple(args, "OKKKK", &error, &p[0], &p[1], &p[2], &p[3])) return nullptr;
  Py_INCREF(error);
  Py_XSETREF(g_error, error);
  g_append = reinterpret_cast<decltype(g_append)>(p[0]);
  g_decode = reinterpret_cast<decltype(g_decode)>(p[1]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(p[2]);
  g_prompt = reinterpret_cast<decltype(g_prompt)>(p[3]);
  Py_RETURN_NONE;
}

#define FMHA_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f))
PyMethodDef g_methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                           {"rope_append", FMHA_FAST(rope_append), METH_FASTCALL, nullptr},
                           {"paged_decode", FMHA_FAST(paged_decode), METH_FASTCALL, nullptr},
                           {"prompt", FMHA_FAST(prompt), METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&g_module); }

// Python binding of the paged-cache entry points (include/liteweight_b200.h):
// reads the tensors' types, shapes, strides and addresses, checks them,
// allocates the result and the scratch and makes the C call on the current
// stream. The same through ctypes costs 8 - 11 us of tensor attribute calls, as
// much as three of the calls' own launches; a decode step makes two such calls
// per layer. The C functions are found by the ctypes binding, which hands over
// their addresses (init).
//
// A refused argument raises AssertionError, a tensor that is not on a CUDA device
// RuntimeError. A status of the library other than LW_OK is returned as a number.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "liteweight_b200.h"

namespace {

decltype(&lw_qk_norm_rope) g_rope = nullptr;
decltype(&lw_paged_attention) g_attention = nullptr;
decltype(&lw_paged_attention_workspace_size) g_workspace = nullptr;

struct Refused {
  PyObject* type;
  std::string why;
};

void require(bool ok, const char* why) {
  if (!ok) throw Refused{PyExc_AssertionError, why};
}

// A tensor argument; an undefined tensor for None where that is allowed.
at::Tensor tensor(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return {};
  if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string(name) + " must be a tensor"};
  return THPVariable_Unpack(o);
}

long long whole(PyObject* o, const char* name) {
  PyObject* i = PyNumber_Index(o);
  if (!i) {
    PyErr_Clear();
    throw Refused{PyExc_TypeError, std::string(name) + " must be a whole number"};
  }
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(i, &over);
  Py_DECREF(i);
  return over > 0 ? LLONG_MAX : over < 0 ? LLONG_MIN : v;
}

double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Refused{PyExc_TypeError, std::string(name) + " must be a number"};
  }
  return v;
}

// All tensors (undefined ones aside) on one CUDA device, q's.
void same_device(std::initializer_list<const at::Tensor*> ts) {
  const at::Device dev = (*ts.begin())->device();
  for (const at::Tensor* t : ts) {
    if (!t->defined()) continue;
    if (!t->is_cuda())
      throw Refused{PyExc_RuntimeError,
                    "liteweight_b200 ops run on CUDA tensors only (no CPU fallback); got a tensor on " +
                        t->device().str()};
  }
  for (const at::Tensor* t : ts) require(!t->defined() || t->device() == dev, "all tensors must be on one device");
}

// The stride of a dimension; of one element (or none) it addresses nothing and may be any.
long long stride_of(const at::Tensor& t, int dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

lw_paged_cache cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens) {
  lw_paged_cache c = {};
  const auto dt = k.scalar_type();
  require((dt == at::kHalf || dt == at::kBFloat16) && v.scalar_type() == dt,
          "k_pages / v_pages: both float16 or both bfloat16");
  require(k.dim() == 4 && v.sizes() == k.sizes(), "k_pages / v_pages: [pages, kv heads, page, head_dim]");
  require(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt, "page_table and kv_lens are int32");
  require(table.dim() == 2 && lens.dim() == 1 && lens.size(0) == table.size(0),
          "page_table: [batch, width], kv_lens: [batch]");
  require((k.stride(3) == 1 && v.stride(3) == 1) || k.numel() == 0, "the pools' last dimension must be contiguous");
  require(table.stride(1) == 1 || table.size(1) <= 1, "page_table's rows must be contiguous");
  require(lens.stride(0) == 1 || lens.size(0) <= 1, "kv_lens must be contiguous");
  for (int64_t n : {k.size(0), k.size(1), k.size(2), k.size(3), table.size(0), table.size(1)})
    require(n <= INT_MAX, "sizes past 2^31 - 1 are not supported");
  c.k_pages = k.data_ptr();
  c.v_pages = v.data_ptr();
  for (int i = 0; i < 3; ++i) {
    c.k_strides[i] = stride_of(k, i);
    c.v_strides[i] = stride_of(v, i);
  }
  c.n_pages = (int)k.size(0);
  c.n_kv_heads = (int)k.size(1);
  c.page_size = (int)k.size(2);
  c.head_dim = (int)k.size(3);
  c.dtype = dt == at::kHalf ? LW_DTYPE_F16 : LW_DTYPE_BF16;
  c.batch = (int)table.size(0);
  c.page_table = static_cast<const int*>(table.data_ptr());
  c.table_stride = stride_of(table, 0);
  c.table_width = (int)table.size(1);
  c.kv_lens = static_cast<const int*>(lens.data_ptr());
  return c;
}

// (token, head) strides of a [tokens, heads, head_dim] tensor of the cache's type.
void rows(const at::Tensor& t, const at::Tensor& like, long long (&strides)[2], const char* why) {
  require(t.scalar_type() == like.scalar_type() && t.dim() == 3 && t.size(2) == like.size(3) &&
              (t.stride(2) == 1 || t.numel() == 0) && t.size(0) <= INT_MAX && t.size(1) <= INT_MAX,
          why);
  strides[0] = stride_of(t, 0);
  strides[1] = stride_of(t, 1);
}

const int* offsets(const at::Tensor& off, int batch, int64_t tokens) {
  if (!off.defined()) {
    require(tokens == batch, "one new token per sequence: as many rows as sequences");
    return nullptr;
  }
  require(off.scalar_type() == at::kInt && off.dim() == 1 && off.size(0) == (int64_t)batch + 1 &&
              (off.stride(0) == 1 || off.size(0) <= 1),
          "q_offsets: int32 [batch + 1], contiguous");
  return static_cast<const int*>(off.data_ptr());
}

template <typename Args>
int call(int (*fn)(const Args*, lw_stream_t), const Args& args, c10::DeviceIndex dev) {
  const auto stream = reinterpret_cast<lw_stream_t>(c10::cuda::getCurrentCUDAStream(dev).stream());
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = fn(&args, stream);
  Py_END_ALLOW_THREADS
  return status;
}

template <typename Body>
PyObject* guarded(Body body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.why.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope(q, k, v, cos, sin, k_pages, v_pages, page_table, kv_lens, q_offsets, q_weight, k_weight, eps, out)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require(n == 14 && g_rope, "qk_norm_rope: 14 arguments, after init");
    const at::Tensor q = tensor(a[0], "q"), k = tensor(a[1], "k"), v = tensor(a[2], "v"), cos = tensor(a[3], "cos"),
                     sin = tensor(a[4], "sin"), kp = tensor(a[5], "k_pages"), vp = tensor(a[6], "v_pages"),
                     table = tensor(a[7], "page_table"), lens = tensor(a[8], "kv_lens"),
                     off = tensor(a[9], "q_offsets", true), qw = tensor(a[10], "q_weight", true),
                     kw = tensor(a[11], "k_weight", true);
    at::Tensor out = tensor(a[13], "out", true);
    lw_qk_norm_rope_args p = {};
    p.cache = cache(kp, vp, table, lens);
    const auto dt = kp.scalar_type();
    const int64_t hd = kp.size(3);
    rows(q, kp, p.q_strides, "q: [tokens, q heads, head_dim] in the cache's type, its last dimension contiguous");
    rows(k, kp, p.k_strides, "k: [tokens, kv heads, head_dim] in the cache's type, its last dimension contiguous");
    rows(v, kp, p.v_strides, "v: [tokens, kv heads, head_dim] in the cache's type, its last dimension contiguous");
    require(k.size(0) == q.size(0) && k.size(1) == kp.size(1) && v.sizes() == k.sizes(),
            "k and v: [tokens, kv heads, head_dim]");
    require(cos.dim() == 2 && cos.size(1) == hd && sin.sizes() == cos.sizes(), "cos / sin: [positions, head_dim]");
    require((cos.scalar_type() == dt || cos.scalar_type() == at::kFloat) && sin.scalar_type() == cos.scalar_type(),
            "cos / sin: float32 or the cache's type");
    require(stride_of(cos, 0) == stride_of(sin, 0) && ((cos.stride(1) == 1 && sin.stride(1) == 1) || cos.numel() == 0) &&
                cos.size(0) <= INT_MAX,
            "cos / sin: rows contiguous, strides alike");
    require(qw.defined() == kw.defined(), "norm weights for both queries and keys, or for neither");
    for (const at::Tensor* w : {&qw, &kw})
      require(!w->defined() || (w->scalar_type() == dt && w->dim() == 1 && w->size(0) == hd && w->stride(0) == 1),
              "norm weights: [head_dim] in the cache's type");
    p.q_offsets = offsets(off, p.cache.batch, q.size(0));
    p.eps = (float)number(a[12], "eps");
    require(!out.defined() || out.sizes() == q.sizes(), "out must have q's shape");
    if (out.defined()) rows(out, kp, p.out_strides, "out: q's type, its last dimension contiguous");
    same_device({&q, &k, &v, &cos, &sin, &kp, &vp, &table, &lens, &off, &qw, &kw, &out});
    const c10::cuda::CUDAGuard guard(q.device());
    p.zero_tail = !out.defined();
    if (!out.defined()) {
      out = at::empty(q.sizes(), q.options());
      p.out_strides[0] = out.stride(0), p.out_strides[1] = out.stride(1);
    }
    p.q = q.data_ptr();
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.q_out = out.data_ptr();
    p.tokens = (int)q.size(0);
    p.n_q_heads = (int)q.size(1);
    p.rope_cos = cos.data_ptr();
    p.rope_sin = sin.data_ptr();
    p.rope_stride = stride_of(cos, 0);
    p.rope_dtype = cos.scalar_type() == at::kFloat ? LW_DTYPE_F32 : p.cache.dtype;
    p.rope_rows = (int)cos.size(0);
    p.q_weight = qw.defined() ? qw.data_ptr() : nullptr;
    p.k_weight = kw.defined() ? kw.data_ptr() : nullptr;
    p.pdl = 1;
    const int status = call(g_rope, p, q.get_device());
    return status ? PyLong_FromLong(status) : THPVariable_Wrap(out);
  });
}

// attention(q, k_pages, v_pages, page_table, kv_lens, q_offsets, window, sinks, scale, out)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require(n == 10 && g_attention, "attention: 10 arguments, after init");
    const at::Tensor q = tensor(a[0], "q"), kp = tensor(a[1], "k_pages"), vp = tensor(a[2], "v_pages"),
                     table = tensor(a[3], "page_table"), lens = tensor(a[4], "kv_lens"),
                     off = tensor(a[5], "q_offsets", true);
    at::Tensor out = tensor(a[9], "out", true);
    lw_paged_attention_args p = {};
    p.cache = cache(kp, vp, table, lens);
    rows(q, kp, p.q_strides, "q: [tokens, q heads, head_dim] in the cache's type, its last dimension contiguous");
    require(kp.size(1) > 0 && q.size(1) % kp.size(1) == 0, "q heads must be a multiple of the kv heads");
    if (a[6] != Py_None) {
      const long long window = whole(a[6], "window");
      require(window >= 1, "window: at least 1, or None");
      p.window = (int)std::min<long long>(window, INT_MAX);
    }
    const long long sinks = whole(a[7], "sinks");
    require(sinks >= 0, "sinks: at least 0");
    p.sinks = (int)std::min<long long>(sinks, INT_MAX);
    p.scale = a[8] == Py_None ? (float)(1.0 / std::sqrt((double)kp.size(3))) : (float)number(a[8], "scale");
    p.q_offsets = offsets(off, p.cache.batch, q.size(0));
    require(!out.defined() || out.sizes() == q.sizes(), "out must have q's shape");
    if (out.defined()) rows(out, kp, p.out_strides, "out: q's type, its last dimension contiguous");
    same_device({&q, &kp, &vp, &table, &lens, &off, &out});
    const c10::cuda::CUDAGuard guard(q.device());
    p.zero_tail = !out.defined();
    if (!out.defined()) {
      out = at::empty(q.sizes(), q.options());
      p.out_strides[0] = out.stride(0), p.out_strides[1] = out.stride(1);
    }
    p.q = q.data_ptr();
    p.out = out.data_ptr();
    p.tokens = (int)q.size(0);
    p.n_q_heads = (int)q.size(1);
    p.pdl = 1;
    // scratch of this call alone: calls on other streams or in other graphs never share it
    at::Tensor scratch;
    if (const size_t need = g_workspace(&p)) {
      scratch = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      p.workspace = scratch.data_ptr();
      p.workspace_bytes = need;
    }
    const int status = call(g_attention, p, q.get_device());
    return status ? PyLong_FromLong(status) : THPVariable_Wrap(out);
  });
}

// init(address of lw_abi_version, of lw_struct_size, of lw_qk_norm_rope, of lw_paged_attention,
// of lw_paged_attention_workspace_size). Refuses a library of another version or with other structs.
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    require(n == 5, "init: 5 addresses");
    const int version = reinterpret_cast<decltype(&lw_abi_version)>(whole(args[0], "address"))();
    const auto size = reinterpret_cast<decltype(&lw_struct_size)>(whole(args[1], "address"));
    if (version != LW_ABI_VERSION || size(5) != sizeof(lw_paged_cache) || size(6) != sizeof(lw_qk_norm_rope_args) ||
        size(7) != sizeof(lw_paged_attention_args))
      throw Refused{PyExc_RuntimeError, "lw_bind.so was built for version " + std::to_string(LW_ABI_VERSION) +
                                            " of the library and got version " + std::to_string(version) +
                                            " or other structs; build both with `python -m liteweight_b200.build`"};
    PyObject* const* a = args + 2;
    g_rope = reinterpret_cast<decltype(g_rope)>(whole(a[0], "address"));
    g_attention = reinterpret_cast<decltype(g_attention)>(whole(a[1], "address"));
    g_workspace = reinterpret_cast<decltype(g_workspace)>(whole(a[2], "address"));
    Py_RETURN_NONE;
  });
}

PyMethodDef methods[] = {
    {"init", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(init)), METH_FASTCALL, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(qk_norm_rope)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "lw_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lw_bind(void) { return PyModule_Create(&module); }

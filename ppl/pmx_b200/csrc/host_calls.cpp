// The regular case of the attention block's operators without Python in between.
//
// A decode step launches kernels that run for 2 to 10 us; checking arguments, allocating results and packing
// the argument struct in Python takes about as long again.  These functions do that for calls in which nothing needs
// converting -- tensors on the current CUDA device, index arrays dense and 64 bits wide, views that the kernels
// read in place, no gradient and no tangent asked for, no export under way -- and call the C ABI (include/pmx_moe.h).  For any other
// call they return None, and the operators in torch_function/dynamic_batching check, convert and raise as they would
// without this file.  They do run without it: it is used where it was built for the torch and the Python at hand (built_for).
// A failed call comes back as its status.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <cstring>

#include "../../../include/pmx_moe.h"

namespace {

decltype(&pmx_rotary_embedding) g_rotary = nullptr;
decltype(&pmx_prompt_attention) g_prompt = nullptr;
decltype(&pmx_tree_cache_attention) g_tree = nullptr;
decltype(&pmx_compact_cache) g_compact = nullptr;
decltype(&pmx_attention_workspace_bytes) g_workspace = nullptr;

// One call's arguments; `regular` turns false at the first one that the general path has to look at.
struct Call {
  PyObject* const* args;
  bool regular = true;
  int device = -1;
  bool grad = c10::GradMode::is_enabled();

  const at::Tensor* tensor(int i, bool optional = false) {
    PyObject* o = args[i];
    if (o == Py_None) {
      if (!optional) regular = false;
      return nullptr;
    }
    if (!THPVariable_CheckExact(o)) {
      regular = false;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || (grad && t.requires_grad()) || t._fw_grad(0).defined()) {
      regular = false;
      return nullptr;
    }
    if (device < 0) device = t.get_device();
    if (t.get_device() != device) regular = false;
    return &t;
  }
  // int64, dense, of `count` entries (-1: any)
  const at::Tensor* index(int i, int64_t count, bool optional = false) {
    const at::Tensor* t = tensor(i, optional);
    if (t && (t->scalar_type() != at::kLong || !t->is_contiguous() || (count >= 0 && t->numel() != count))) regular = false;
    return t;
  }
  // [rows, heads, dim] in place, as the kernels read it
  const at::Tensor* heads(int i, int64_t heads, int64_t dim, at::ScalarType type, bool aligned) {
    const at::Tensor* t = tensor(i);
    if (!t || !regular) return nullptr;
    if (t->dim() != 3 || t->size(1) != heads || t->size(2) != dim || t->scalar_type() != type || t->stride(2) != 1 ||
        t->numel() == 0)
      regular = false;
    else if (aligned) {
      const int64_t a = t->stride(0), b = t->stride(1);
      if ((a | b) * (int64_t)t->element_size() % 16 || a <= 0 || b <= 0 || reinterpret_cast<uintptr_t>(t->data_ptr()) % 16)
        regular = false;
    }
    return t;
  }
  int64_t number(int i) {
    if (!PyLong_CheckExact(args[i])) {
      regular = false;
      return 0;
    }
    const int64_t v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      regular = false;
    }
    return v;
  }
  double real(int i) {
    if (!PyFloat_CheckExact(args[i])) {
      regular = false;
      return 0.0;
    }
    return PyFloat_AS_DOUBLE(args[i]);
  }
  bool ready() const {
    return regular && device >= 0 && c10::cuda::current_device() == device && !torch::jit::tracer::isTracing();
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
};

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return PMX_DTYPE_F16;
    case at::kBFloat16: return PMX_DTYPE_BF16;
    case at::kFloat: return PMX_DTYPE_F32;
    default: return -1;
  }
}
template <typename T>
T* ptr(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
at::Tensor dense_like(const at::Tensor& t) {
  return at::empty(t.sizes(), t.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
}
PyObject* none() { Py_RETURN_NONE; }

// no C++ exception leaves for the interpreter: each becomes the one that torch raises for it (running out of memory is
// torch.OutOfMemoryError)
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  return F(args, n);
  END_HANDLE_TH_ERRORS
}

// cache [5 dimensions] in one of the four layouts -> strides and sizes, or false
bool cache_layout(const at::Tensor& c, int64_t layout, int64_t layers, int64_t* rows, int64_t* heads, int64_t* row, int64_t* layer,
                  int64_t* kv, int64_t* head) {
  if (c.dim() != 5 || !c.is_contiguous() || layout < 0 || layout > 3 || c.numel() == 0) return false;
  // where (row, layer, kv, head) stand in each layout
  static const int at[4][4] = {{0, 1, 2, 3}, {1, 0, 2, 3}, {2, 0, 1, 3}, {3, 0, 1, 2}};
  const int* p = at[layout];
  if (c.size(p[2]) != 2 || c.size(p[1]) != layers) return false;
  *rows = c.size(p[0]); *heads = c.size(p[3]);
  *row = c.stride(p[0]); *layer = c.stride(p[1]); *kv = c.stride(p[2]); *head = c.stride(p[3]);
  return true;
}

// rotary(query, key | None, query weight | None, key weight | None, eps, seqstarts | None, start_pos | None, position_ids | None,
//        rotary_dim, interleaved, address of the frequencies, factor)
PyObject* rotary(PyObject* const* args, Py_ssize_t n) {
  if (n != 12 || !g_rotary) return none();
  Call c{args};
  const at::Tensor* q = c.tensor(0);
  if (!q || !c.regular || q->dim() != 3) return none();
  const int64_t T = q->size(0), D = q->size(2);
  const auto type = q->scalar_type();
  q = c.heads(0, q->size(1), D, type, false);
  const at::Tensor* k = nullptr;
  if (args[1] != Py_None) {
    k = c.tensor(1);
    if (!k || !c.regular || k->dim() != 3 || k->size(0) != T) return none();
    k = c.heads(1, k->size(1), D, type, false);
  }
  const at::Tensor* qw = c.tensor(2, true);
  const at::Tensor* kw = c.tensor(3, true);
  for (const at::Tensor* w : {qw, kw})
    if (w && (w->dim() != 1 || w->size(0) != D || w->scalar_type() != type || !w->is_contiguous())) return none();
  if ((qw != nullptr) != (kw != nullptr) || (qw && !k)) return none();
  const at::Tensor* ids = c.index(7, T, true);
  const at::Tensor *starts = nullptr, *past = nullptr;
  if (!ids) {
    starts = c.index(5, -1);
    past = c.index(6, starts ? starts->numel() - 1 : 0);
    if (!starts || starts->numel() < 2) return none();
  }
  const int64_t r = c.number(8);
  pmx_rotary_args a{};
  a.interleaved = c.number(9);
  a.frequencies = reinterpret_cast<const double*>(c.number(10));
  a.eps = c.real(4);
  a.factor = c.real(11);
  a.dtype = dtype_code(type);
  if (!c.ready() || a.dtype < 0 || r > D || r <= 0) return none();
  const at::Tensor qo = dense_like(*q);
  at::Tensor ko;
  if (k) ko = dense_like(*k);
  a.query = q->data_ptr(); a.key = ptr<void>(k);
  a.query_norm_weight = ptr<void>(qw); a.key_norm_weight = ptr<void>(kw);
  a.query_out = qo.data_ptr(); a.key_out = k ? ko.data_ptr() : nullptr;
  a.seqstarts = ptr<int64_t>(starts); a.start_pos = ptr<int64_t>(past); a.position_ids = ptr<int64_t>(ids);
  a.tokens = T; a.sequences = starts ? starts->numel() - 1 : 0;
  a.num_heads = q->size(1); a.num_kv_heads = k ? k->size(1) : 0; a.head_dim = D;
  a.q_token_stride = q->stride(0); a.q_head_stride = q->stride(1);
  a.k_token_stride = k ? k->stride(0) : 0; a.k_head_stride = k ? k->stride(1) : 0;
  a.rotary_dim = r;
  const int st = g_rotary(&a, c.stream());
  if (st) return PyLong_FromLong(st);
  PyObject* pair = PyTuple_New(2);
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(qo));
  PyTuple_SET_ITEM(pair, 1, k ? THPVariable_Wrap(ko) : none());
  return pair;
}

// prompt(query, key, value, seqstarts, kvstarts, max_seqlen, max_kvlen, num_heads, head_dim, is_causal, num_kv_heads, scale, cap,
//        alibi_slopes | None, prefix_lens | None)
PyObject* prompt(PyObject* const* args, Py_ssize_t n) {
  if (n != 15 || !g_prompt) return none();
  Call c{args};
  pmx_prompt_attention_args a{};
  a.num_heads = c.number(7);
  a.head_dim = c.number(8);
  a.num_kv_heads = c.number(10);
  const at::Tensor* q = c.tensor(0);
  if (!q || !c.regular) return none();
  const auto type = q->scalar_type();
  if (a.num_kv_heads == 0) a.num_kv_heads = a.num_heads;
  q = c.heads(0, a.num_heads, a.head_dim, type, true);
  const at::Tensor* k = c.heads(1, a.num_kv_heads, a.head_dim, type, true);
  const at::Tensor* v = c.heads(2, a.num_kv_heads, a.head_dim, type, true);
  if (!q || !k || !v || k->size(0) != v->size(0)) return none();
  const at::Tensor* starts = c.index(3, -1);
  if (!starts || starts->numel() < 2) return none();
  a.sequences = starts->numel() - 1;
  const at::Tensor* kv = c.index(4, a.sequences + 1);
  const at::Tensor* slopes = c.tensor(13, true);
  const at::Tensor* prefix = c.index(14, a.sequences, true);
  a.max_seqlen = c.number(5);
  a.max_kvlen = c.number(6);
  a.is_causal = args[9] == Py_True;
  a.scale = args[11] == Py_None ? 1.0 / std::sqrt((double)a.head_dim) : c.real(11);
  a.logit_cap = c.real(12);
  a.dtype = dtype_code(type);
  if (!c.ready() || a.dtype < 0 || a.max_seqlen <= 0 || a.max_kvlen <= 0 || (args[9] != Py_True && args[9] != Py_False) ||
      !(a.scale > 0.0) || std::isinf(a.scale) || !(a.logit_cap >= 0.0) || std::isinf(a.logit_cap) ||
      a.num_heads % a.num_kv_heads ||
      (slopes && (slopes->scalar_type() != at::kFloat || slopes->dim() != 1 || slopes->size(0) != a.num_heads || !slopes->is_contiguous())))
    return none();
  a.tokens = q->size(0); a.keys = k->size(0);
  const at::Tensor out = dense_like(*q);
  a.workspace_bytes = (int64_t)g_workspace(a.tokens, (int32_t)a.sequences, (int32_t)a.num_heads, (int32_t)a.num_kv_heads,
                                           (int32_t)a.head_dim, a.max_seqlen, a.max_kvlen, (int32_t)a.dtype);
  at::Tensor ws;
  if (a.workspace_bytes) ws = at::empty({a.workspace_bytes}, q->options().dtype(at::kByte));
  a.query = q->data_ptr(); a.key = k->data_ptr(); a.value = v->data_ptr();
  a.seqstarts = ptr<int64_t>(starts); a.kvstarts = ptr<int64_t>(kv); a.prefix_lens = ptr<int64_t>(prefix);
  a.alibi_slopes = ptr<float>(slopes);
  a.out = out.data_ptr(); a.workspace = a.workspace_bytes ? ws.data_ptr() : nullptr;
  a.q_token_stride = q->stride(0); a.q_head_stride = q->stride(1);
  a.k_token_stride = k->stride(0); a.k_head_stride = k->stride(1);
  a.v_token_stride = v->stride(0); a.v_head_stride = v->stride(1);
  const int st = g_prompt(&a, c.stream());
  return st ? PyLong_FromLong(st) : THPVariable_Wrap(out);
}

// tree(query, current_key, current_value, seqstarts, cachestarts, start_pos, tree_mask, max_seqlen, max_kvlen, cache, num_heads,
//      head_dim, num_kv_heads, num_layer, layer_idx, cache_layout, scale, cap)
PyObject* tree(PyObject* const* args, Py_ssize_t n) {
  if (n != 18 || !g_tree) return none();
  Call c{args};
  pmx_tree_attention_args a{};
  a.num_heads = c.number(10);
  a.head_dim = c.number(11);
  a.num_kv_heads = c.number(12);
  const at::Tensor* q = c.tensor(0);
  const at::Tensor* cache = c.tensor(9);
  if (!q || !cache || !c.regular) return none();
  const auto type = q->scalar_type();
  if (a.num_kv_heads == 0) a.num_kv_heads = a.num_heads;
  q = c.heads(0, a.num_heads, a.head_dim, type, true);
  const at::Tensor* k = c.heads(1, a.num_kv_heads, a.head_dim, type, true);
  const at::Tensor* v = c.heads(2, a.num_kv_heads, a.head_dim, type, true);
  if (!q || !k || !v || k->size(0) != q->size(0) || v->size(0) != q->size(0)) return none();
  a.tokens = q->size(0);
  const at::Tensor* starts = c.index(3, -1);
  if (!starts || starts->numel() < 2) return none();
  a.sequences = starts->numel() - 1;
  const at::Tensor* first = c.index(4, a.sequences);
  const at::Tensor* past = c.index(5, a.sequences);
  const at::Tensor* mask = c.index(6, a.tokens);
  a.max_seqlen = c.number(7);
  a.max_kvlen = c.number(8);
  const int64_t layers = c.number(13), layer = c.number(14), layout = c.number(15);
  int64_t cache_heads, layer_stride;
  if (!c.regular || cache->scalar_type() != type || cache->dim() != 5 || cache->size(4) != a.head_dim ||
      !cache_layout(*cache, layout, layers, &a.cache_rows, &cache_heads, &a.row_stride, &layer_stride, &a.kv_stride, &a.head_stride) ||
      cache_heads != a.num_kv_heads || layer < 0 || layer >= layers)
    return none();
  a.layer_offset = layer * layer_stride;
  a.scale = args[16] == Py_None ? 1.0 / std::sqrt((double)a.head_dim) : c.real(16);
  a.logit_cap = c.real(17);
  a.dtype = dtype_code(type);
  if (!c.ready() || a.dtype < 0 || a.max_seqlen <= 0 || a.max_kvlen <= 0 || !(a.scale > 0.0) || std::isinf(a.scale) ||
      !(a.logit_cap >= 0.0) || std::isinf(a.logit_cap) || a.num_heads % a.num_kv_heads)
    return none();
  const at::Tensor out = dense_like(*q);
  a.workspace_bytes = (int64_t)g_workspace(a.tokens, (int32_t)a.sequences, (int32_t)a.num_heads, (int32_t)a.num_kv_heads,
                                           (int32_t)a.head_dim, a.max_seqlen, a.max_kvlen, (int32_t)a.dtype);
  at::Tensor ws;
  if (a.workspace_bytes) ws = at::empty({a.workspace_bytes}, q->options().dtype(at::kByte));
  a.query = q->data_ptr(); a.current_key = k->data_ptr(); a.current_value = v->data_ptr();
  a.cache = cache->data_ptr();
  a.seqstarts = ptr<int64_t>(starts); a.cachestarts = ptr<int64_t>(first); a.start_pos = ptr<int64_t>(past);
  a.tree_mask = ptr<int64_t>(mask);
  a.out = out.data_ptr(); a.workspace = a.workspace_bytes ? ws.data_ptr() : nullptr;
  a.q_token_stride = q->stride(0); a.q_head_stride = q->stride(1);
  a.k_token_stride = k->stride(0); a.k_head_stride = k->stride(1);
  a.v_token_stride = v->stride(0); a.v_head_stride = v->stride(1);
  const int st = g_tree(&a, c.stream());
  return st ? PyLong_FromLong(st) : THPVariable_Wrap(out);
}

// compact(cache, cachestarts, start_pos, accept_starts, accept_index, max_accept, num_layer, cache_layout) -> status
PyObject* compact(PyObject* const* args, Py_ssize_t n) {
  if (n != 8 || !g_compact) return none();
  Call c{args};
  const at::Tensor* cache = c.tensor(0);
  const at::Tensor* starts = c.index(3, -1);
  if (!cache || !starts || starts->numel() < 2) return none();
  pmx_compact_cache_args a{};
  a.sequences = starts->numel() - 1;
  const at::Tensor* first = c.index(1, a.sequences);
  const at::Tensor* past = c.index(2, a.sequences);
  const at::Tensor* picks = c.index(4, -1);
  a.max_accept = c.number(5);
  a.num_layers = c.number(6);
  const int64_t layout = c.number(7);
  a.dtype = dtype_code(cache->scalar_type());
  if (!c.ready() || a.dtype < 0 || a.max_accept <= 0 || a.max_accept > 64 || picks->numel() == 0 ||
      !cache_layout(*cache, layout, a.num_layers, &a.cache_rows, &a.num_kv_heads, &a.row_stride, &a.layer_stride, &a.kv_stride, &a.head_stride))
    return none();
  a.head_dim = cache->size(4);
  a.cache = cache->data_ptr();
  a.cachestarts = ptr<int64_t>(first); a.start_pos = ptr<int64_t>(past);
  a.accept_starts = ptr<int64_t>(starts); a.accept_index = ptr<int64_t>(picks);
  a.index_count = picks->numel();
  return PyLong_FromLong(g_compact(&a, c.stream()));
}

// bind(addresses of pmx_rotary_embedding, pmx_prompt_attention, pmx_tree_cache_attention, pmx_compact_cache,
//      pmx_attention_workspace_bytes): the entry points of the library that the package has loaded
PyObject* bind(PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind: five addresses");
    return nullptr;
  }
  void* at[5];
  for (int i = 0; i < 5; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_rotary = reinterpret_cast<decltype(g_rotary)>(at[0]);
  g_prompt = reinterpret_cast<decltype(g_prompt)>(at[1]);
  g_tree = reinterpret_cast<decltype(g_tree)>(at[2]);
  g_compact = reinterpret_cast<decltype(g_compact)>(at[3]);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(at[4]);
  Py_RETURN_NONE;
}

#define PMX_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<name>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {PMX_METHOD(rotary), PMX_METHOD(prompt), PMX_METHOD(tree), PMX_METHOD(compact), PMX_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host_calls(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", PMX_BUILT_FOR)) Py_CLEAR(m);
  return m;
}

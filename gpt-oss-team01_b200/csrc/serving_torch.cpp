// The serving operators on torch tensors, as a Python module: checks of the tensors, outputs and scratch from torch's
// allocator, the call of the C ABI on the current stream of the tensors' device.  It is compiled because these calls run for
// as little as 2 us on the GPU: from Python, reading types, shapes and addresses of ten tensors and filling in the argument
// structure took 5 to 8 us a call.  The C functions come in as addresses from whichever build of the library is loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/gptoss_b200.h"

namespace {

PyObject *g_error = nullptr;  // GptossError(code, message)
decltype(&gptoss_tree_attention) f_tree;
decltype(&gptoss_tree_attention_workspace) f_tree_workspace;
decltype(&gptoss_cache_commit) f_commit;
decltype(&gptoss_lora_apply) f_lora;
decltype(&gptoss_lora_workspace) f_lora_workspace;
decltype(&gptoss_expert_choice) f_choice;
decltype(&gptoss_serving_last_error) f_last_error;

struct Refused {
  int code;
  std::string message;
};
struct Raised {};  // a Python exception is set already

[[noreturn]] void bad(std::string message) { throw Refused{GPTOSS_ERR_BAD_ARG, std::move(message)}; }

struct NoGil {
  PyThreadState *state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// o as a tensor of that type and number of dimensions on cuda device `dev` (-1: any).  The operators have no backward pass: as
// torch's own operators without one refuse it, a tensor that asks for its gradient is refused, not silently left without.
const at::Tensor &view(PyObject *o, const char *name, at::ScalarType type, int64_t ndim, int dev) {
  if (THPVariable_Check(o)) {
    const at::Tensor &t = THPVariable_Unpack(o);
    if (t.requires_grad() && c10::GradMode::is_enabled())
      bad(std::string(name) + " requires a gradient, which the serving operators do not give: detach it, or call under torch.no_grad()");
    if (t.layout() == at::kStrided && t.scalar_type() == type && t.dim() == ndim && t.is_cuda() && (dev < 0 || t.get_device() == dev)) return t;
  }
  bad(std::string(name) + " must be a " + at::toString(type) + " tensor of " + std::to_string(ndim) + " dimensions on " +
      (dev < 0 ? "a cuda device" : "cuda:" + std::to_string(dev)));
}
const at::Tensor &dense(PyObject *o, const char *name, at::ScalarType type, int64_t ndim, int dev) {
  const at::Tensor &t = view(o, name, type, ndim, dev);
  if (!t.is_contiguous()) bad(std::string(name) + " must be contiguous");
  return t;
}
// address of an optional vector of n entries (at_least: or more)
template <typename T>
const T *vector_or_null(PyObject *o, const char *name, at::ScalarType type, int dev, int64_t n, bool at_least = false) {
  if (o == Py_None) return nullptr;
  const at::Tensor &t = dense(o, name, type, 1, dev);
  if (at_least ? t.size(0) < n : t.size(0) != n) bad(std::string(name) + " needs " + std::to_string(n) + " entries");
  return static_cast<const T *>(t.const_data_ptr());
}
int small(int64_t v, const char *name) {
  if (v < -2147483647 || v > 2147483647) bad(std::string(name) + " does not fit in 32 bits");
  return (int)v;
}
int integer(PyObject *o, const char *name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return small(v, name);
}
float number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return (float)v;
}
void check(int rc) {
  if (rc) throw Refused{rc, f_last_error()};
}

// A tensor of the caller's that the call has written: its version counts up, so that a graph that saved it notices.
void written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// body(args) with C++ exceptions turned into Python's
template <typename F>
PyObject *guarded(Py_ssize_t n_args, Py_ssize_t want, F body) {
  try {
    if (n_args != want) {
      PyErr_Format(PyExc_TypeError, "%zd arguments instead of %zd", n_args, want);
      return nullptr;
    }
    return body();
  } catch (const Raised &) {
  } catch (const Refused &r) {
    if (PyObject *e = PyObject_CallFunction(g_error, "is", r.code, r.message.c_str())) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
  } catch (const c10::OutOfMemoryError &e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// (q, k_cache, v_cache, offsets, ctx_len, mask, depth, max_nodes, max_ctx, sinks, cache_rows, window, scale, out)
PyObject *tree_attention(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
  return guarded(n_args, 14, [&] {
    const at::Tensor &q = view(o[0], "q", at::kBFloat16, 3, -1);
    const int dev = q.get_device();
    const at::Tensor &k = dense(o[1], "k_cache", at::kBFloat16, 4, dev), &v = dense(o[2], "v_cache", at::kBFloat16, 4, dev);
    const at::Tensor &offsets = dense(o[3], "offsets", at::kInt, 1, dev), &ctx = dense(o[4], "ctx_len", at::kInt, 1, dev),
                     &mask = dense(o[5], "mask", at::kInt, 2, dev);
    const int64_t n_tokens = q.size(0), nq = q.size(1), hd = q.size(2), n_seqs = ctx.size(0);
    if (q.stride(2) != 1 || (q.stride(1) != hd && nq > 1)) bad("q: heads of a token must be contiguous");
    if (v.sizes() != k.sizes() || k.size(3) != hd) bad("k_cache and v_cache must have the same shape and q's head_dim");
    if (offsets.size(0) != n_seqs + 1 || mask.size(0) < n_tokens) bad("offsets needs one more entry than ctx_len, mask a row per token");
    gptoss_tree_attention_args a{};
    a.depth = vector_or_null<int>(o[6], "depth", at::kInt, dev, n_tokens, true);
    a.sinks = vector_or_null<float>(o[9], "sinks", at::kFloat, dev, nq);
    a.rows = vector_or_null<int>(o[10], "cache_rows", at::kInt, dev, n_seqs);
    a.max_nodes = integer(o[7], "max_nodes"), a.max_ctx = integer(o[8], "max_ctx"), a.window = integer(o[11], "window");
    a.scale = o[12] == Py_None ? (float)(1.0 / std::sqrt((double)hd)) : number(o[12]);
    const bool given = o[13] != Py_None;
    at::Tensor out;
    if (given) {
      out = view(o[13], "out", at::kBFloat16, 3, dev);
      if (out.sizes() != q.sizes() || out.stride(2) != 1 || (out.stride(1) != hd && nq > 1)) bad("out must have q's shape and contiguous heads");
    }
    a.q = q.const_data_ptr(), a.k_cache = k.const_data_ptr(), a.v_cache = v.const_data_ptr();
    a.offsets = static_cast<const int *>(offsets.const_data_ptr()), a.ctx_len = static_cast<const int *>(ctx.const_data_ptr());
    a.mask = static_cast<const int *>(mask.const_data_ptr());
    a.q_stride = n_tokens > 1 ? q.stride(0) : nq * hd;
    a.n_tokens = small(n_tokens, "n_tokens"), a.n_seqs = small(n_seqs, "n_seqs"), a.mask_words = small(mask.size(1), "mask_words");
    a.cache_rows = small(k.size(0), "cache rows"), a.n_kv_heads = small(k.size(1), "n_kv_heads"), a.max_seq = small(k.size(2), "max_seq");
    a.n_q_heads = small(nq, "n_q_heads"), a.head_dim = small(hd, "head_dim");
    {
      NoGil no_gil;
      const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
      if (!given) out = at::empty(q.sizes(), q.options());
      a.out = out.mutable_data_ptr(), a.out_stride = n_tokens > 1 ? out.stride(0) : nq * hd;
      a.workspace_bytes = f_tree_workspace(&a);
      at::Tensor work;
      if (a.workspace_bytes) {
        work = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
        a.workspace = work.mutable_data_ptr();
      }
      check(f_tree(&a, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()));
    }
    if (given) written(out);
    return given ? Py_NewRef(o[13]) : THPVariable_Wrap(std::move(out));
  });
}

// (k_cache, v_cache, ctx_len, offsets, path, max_path, cache_rows)
PyObject *cache_commit(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
  return guarded(n_args, 7, [&] {
    const int64_t ndim = THPVariable_Check(o[0]) && THPVariable_Unpack(o[0]).dim() == 4 ? 4 : 5;
    const at::Tensor &k = dense(o[0], "k_cache", at::kBFloat16, ndim, -1);
    const int dev = k.get_device();
    const at::Tensor &v = dense(o[1], "v_cache", at::kBFloat16, ndim, dev), &ctx = dense(o[2], "ctx_len", at::kInt, 1, dev),
                     &offsets = dense(o[3], "offsets", at::kInt, 1, dev), &path = dense(o[4], "path", at::kInt, 1, dev);
    if (v.sizes() != k.sizes()) bad("k_cache and v_cache must have the same shape");
    const int64_t n_seqs = ctx.size(0);
    if (offsets.size(0) != n_seqs + 1) bad("offsets needs one more entry than ctx_len");
    const int *rows = vector_or_null<int>(o[6], "cache_rows", at::kInt, dev, n_seqs);
    const int max_path = integer(o[5], "max_path");
    const int layers = ndim == 4 ? 1 : small(k.size(0), "layers"), cache_rows = small(k.size(-4), "cache rows"),
              nkv = small(k.size(-3), "n_kv_heads"), max_seq = small(k.size(-2), "max_seq"), hd = small(k.size(-1), "head_dim"),
              n_path = small(path.size(0), "path");
    {
      NoGil no_gil;
      const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
      check(f_commit(k.mutable_data_ptr(), v.mutable_data_ptr(), layers, cache_rows, nkv, max_seq, hd, small(n_seqs, "n_seqs"), rows,
                     static_cast<const int *>(ctx.const_data_ptr()), static_cast<const int *>(offsets.const_data_ptr()),
                     static_cast<const int *>(path.const_data_ptr()), n_path, max_path,
                     c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()));
    }
    written(k), written(v);
    Py_RETURN_NONE;
  });
}

// (x, a, b, ids, y, scale, out)
PyObject *lora_apply(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
  return guarded(n_args, 7, [&] {
    const at::Tensor &x = view(o[0], "x", at::kBFloat16, 2, -1);
    const int dev = x.get_device();
    const at::Tensor &a = dense(o[1], "a", at::kBFloat16, 3, dev), &b = dense(o[2], "b", at::kBFloat16, 3, dev),
                     &ids = dense(o[3], "ids", at::kInt, 1, dev), &y = view(o[4], "y", at::kFloat, 2, dev);
    PyObject *const result = o[6] == Py_None ? o[4] : o[6];
    const at::Tensor &out = view(result, "out", at::kFloat, 2, dev);
    const int64_t T = x.size(0), K = x.size(1), n = a.size(0), rank = a.size(1), n_out = b.size(1);
    if (a.size(2) != K || b.size(0) != n || b.size(2) != rank) bad("a must be [n_adapters, rank, K] and b [n_adapters, n_out, rank]");
    if (y.size(0) != T || y.size(1) != n_out || out.sizes() != y.sizes() || y.stride(1) != 1 || out.stride(1) != 1)
      bad("y and out must be [T, n_out] with contiguous rows");
    if (ids.size(0) != T || x.stride(1) != 1) bad("ids needs an entry per token, x contiguous rows");
    gptoss_lora_args g{};
    g.scale = vector_or_null<float>(o[5], "scale", at::kFloat, dev, n);
    g.x = x.const_data_ptr(), g.a = a.const_data_ptr(), g.b = b.const_data_ptr();
    g.ids = static_cast<const int *>(ids.const_data_ptr());
    g.y = static_cast<const float *>(y.const_data_ptr()), g.out = static_cast<float *>(out.mutable_data_ptr());
    g.x_stride = T > 1 ? x.stride(0) : K, g.y_stride = T > 1 ? y.stride(0) : n_out, g.out_stride = T > 1 ? out.stride(0) : n_out;
    g.T = small(T, "T"), g.K = small(K, "K"), g.n_out = small(n_out, "n_out"), g.rank = small(rank, "rank"),
    g.n_adapters = small(n, "n_adapters");
    {
      NoGil no_gil;
      const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
      g.workspace_bytes = f_lora_workspace(&g);
      at::Tensor work;
      if (g.workspace_bytes) {
        work = at::empty({(int64_t)g.workspace_bytes}, x.options().dtype(at::kByte));
        g.workspace = work.mutable_data_ptr();
      }
      check(f_lora(&g, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()));
    }
    written(out);
    return Py_NewRef(result);
  });
}

// (logits, top_k, scoring, bias, n_groups, topk_groups, group_top, renormalize, weight_scale)
PyObject *route_experts(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
  return guarded(n_args, 9, [&] {
    const at::Tensor &logits = view(o[0], "logits", at::kFloat, 2, -1);
    const int dev = logits.get_device();
    const int64_t T = logits.size(0), E = logits.size(1);
    if (logits.stride(1) != 1 && E > 1) bad("logits must have contiguous rows");
    gptoss_expert_choice_args a{};
    a.k = integer(o[1], "top_k"), a.scoring = integer(o[2], "scoring");
    a.bias = vector_or_null<float>(o[3], "bias", at::kFloat, dev, E);
    a.n_groups = integer(o[4], "n_groups"), a.topk_groups = integer(o[5], "topk_groups"), a.group_top = integer(o[6], "group_top");
    const int renormalize = PyObject_IsTrue(o[7]);
    if (renormalize < 0) throw Raised{};
    a.renormalize = renormalize, a.weight_scale = number(o[8]);
    if (a.k < 1 || a.k > 8) bad("top_k must be 1..8");
    a.logits = static_cast<const float *>(logits.const_data_ptr());
    a.stride = T > 1 ? logits.stride(0) : E;
    a.T = small(T, "T"), a.E = small(E, "E");
    at::Tensor w, ids;
    {
      NoGil no_gil;
      const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
      w = at::empty({T, a.k}, logits.options()), ids = at::empty({T, a.k}, logits.options().dtype(at::kInt));
      a.topk_w = static_cast<float *>(w.mutable_data_ptr()), a.topk_i = static_cast<int *>(ids.mutable_data_ptr());
      check(f_choice(&a, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream()));
    }
    PyObject *pw = THPVariable_Wrap(std::move(w)), *pi = pw ? THPVariable_Wrap(std::move(ids)) : nullptr;
    PyObject *pair = pi ? PyTuple_Pack(2, pw, pi) : nullptr;
    Py_XDECREF(pw), Py_XDECREF(pi);
    return pair;
  });
}

// (error class, addresses of the C functions in the order below)
PyObject *bind(PyObject *, PyObject *const *o, Py_ssize_t n_args) {
  return guarded(n_args, 8, [&] {
    void *p[7];
    for (int i = 0; i < 7; ++i)
      if (!(p[i] = PyLong_AsVoidPtr(o[i + 1]))) throw Raised{};
    f_tree = reinterpret_cast<decltype(f_tree)>(p[0]), f_tree_workspace = reinterpret_cast<decltype(f_tree_workspace)>(p[1]);
    f_commit = reinterpret_cast<decltype(f_commit)>(p[2]);
    f_lora = reinterpret_cast<decltype(f_lora)>(p[3]), f_lora_workspace = reinterpret_cast<decltype(f_lora_workspace)>(p[4]);
    f_choice = reinterpret_cast<decltype(f_choice)>(p[5]), f_last_error = reinterpret_cast<decltype(f_last_error)>(p[6]);
    Py_XSETREF(g_error, Py_NewRef(o[0]));
    Py_RETURN_NONE;
  });
}

PyMethodDef g_methods[] = {{"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
                           {"cache_commit", (PyCFunction)(void (*)(void))cache_commit, METH_FASTCALL, nullptr},
                           {"lora_apply", (PyCFunction)(void (*)(void))lora_apply, METH_FASTCALL, nullptr},
                           {"route_experts", (PyCFunction)(void (*)(void))route_experts, METH_FASTCALL, nullptr},
                           {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_serving_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving_torch(void) { return PyModule_Create(&g_module); }

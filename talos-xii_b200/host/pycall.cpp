// Native call path of the Python binding: one CPython function per status-returning entry point of the C ABI, its argument
// conversion generated by the compiler from the header's own declaration.
//
// A small call through ctypes spends 0.7 to 1.2 us converting a dozen arguments, which is a quarter of what launching its
// kernel costs; here the conversion takes 0.1 to 0.2 us.  Only the plain argument forms are converted (int, float, None and
// ctypes.c_void_p handles); any other form (byref, arrays, wrong types or counts) is handed to the ctypes
// function of the same name, so what is accepted and what is raised stays the same.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <tuple>
#include <type_traits>
#include <utility>

#include "../../include/talos_b200.h"
#include "../../include/talos_b200_ppo.h"
#include "../../include/talos_b200_lm.h"

namespace {

PyObject* g_error = nullptr;         // TalosError(status, message)
PyObject* g_handle_type = nullptr;   // ctypes.c_void_p
PyObject* g_fallback = nullptr;      // {name: ctypes function}
PyObject* g_value = nullptr;         // "value"

bool get(PyObject* o, void*& v) {
  if (o == Py_None) { v = nullptr; return true; }
  if (PyLong_CheckExact(o)) { v = PyLong_AsVoidPtr(o); if (v == nullptr && PyErr_Occurred()) { PyErr_Clear(); return false; } return true; }
  if ((PyObject*)Py_TYPE(o) != g_handle_type) return false;
  PyObject* x = PyObject_GetAttr(o, g_value);
  if (!x) { PyErr_Clear(); return false; }
  const bool ok = x == Py_None || PyLong_CheckExact(x);
  v = ok && x != Py_None ? PyLong_AsVoidPtr(x) : nullptr;
  Py_DECREF(x);
  return ok;
}
bool get_int(PyObject* o, long long& v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0;
}
bool get_float(PyObject* o, double& v) {
  if (PyFloat_CheckExact(o)) { v = PyFloat_AS_DOUBLE(o); return true; }
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
  return true;
}
template <typename T> bool convert(PyObject* o, T& v) {
  if constexpr (std::is_pointer_v<T>) { void* p; if (!get(o, p)) return false; v = (T)p; return true; }
  else if constexpr (std::is_floating_point_v<T>) { double d; if (!get_float(o, d)) return false; v = (T)d; return true; }
  else { long long i; if (!get_int(o, i)) return false; v = (T)i; return true; }
}

PyObject* fall_back(const char* name, PyObject* const* args, Py_ssize_t n) {
  PyObject* f = g_fallback ? PyDict_GetItemString(g_fallback, name) : nullptr;      // borrowed
  if (!f) { PyErr_Format(PyExc_TypeError, "%s: unsupported argument", name); return nullptr; }
  return PyObject_Vectorcall(f, args, (size_t)n, nullptr);
}
PyObject* raise_status(talos_status st) {
  if (!g_error) { PyErr_Format(PyExc_RuntimeError, "talos status %d: %s", (int)st, talos_last_error_string()); return nullptr; }
  PyObject* e = PyObject_CallFunction(g_error, "is", (int)st, talos_last_error_string());
  if (e) { PyErr_SetObject(g_error, e); Py_DECREF(e); }
  return nullptr;
}

template <typename... A, size_t... I>
PyObject* call(talos_status (*fn)(A...), const char* name, PyObject* const* args, Py_ssize_t n, std::index_sequence<I...>) {
  std::tuple<A...> v;
  if (n != (Py_ssize_t)sizeof...(A) || !(convert(args[I], std::get<I>(v)) && ...)) return fall_back(name, args, n);
  talos_status st;
  Py_BEGIN_ALLOW_THREADS
  st = fn(std::get<I>(v)...);
  Py_END_ALLOW_THREADS
  if (st != TALOS_OK) return raise_status(st);
  Py_RETURN_NONE;
}
template <typename... A>
PyObject* call(talos_status (*fn)(A...), const char* name, PyObject* const* args, Py_ssize_t n) { return call(fn, name, args, n, std::index_sequence_for<A...>{}); }

#define TALOS_FUNCTIONS(X)                                                                                                                     \
  X(talos_ctx_create) X(talos_ctx_destroy) X(talos_ctx_synchronize) X(talos_ctx_set_stream) X(talos_ctx_reserve_workspace)                    \
  X(talos_debug_set_device_status) X(talos_debug_gemm_stall) X(talos_malloc) X(talos_free) X(talos_ctx_trim) X(talos_ctx_memory_stats)         \
  X(talos_ctx_timeline_begin) X(talos_ctx_timeline_end) X(talos_memset_zero) X(talos_copy_from_host) X(talos_copy_to_host) X(talos_copy_device) \
  X(talos_upload_f64) X(talos_download_f64) X(talos_gemm) X(talos_gemm_batched) X(talos_linear_fwd) X(talos_linear_bwd) X(talos_bias_add)      \
  X(talos_colsum) X(talos_colsum_noalloc) X(talos_axpy) X(talos_dot) X(talos_vector_fma) X(talos_vector_scale) X(talos_softmax_exp_sum)        \
  X(talos_rmsnorm_fwd) X(talos_rmsnorm_bwd) X(talos_rope_table) X(talos_rope) X(talos_softmax_fwd) X(talos_softmax_bwd) X(talos_attention_fwd) \
  X(talos_attention_bwd) X(talos_gae) X(talos_normalize_slice) X(talos_dueling_combine_fwd) X(talos_dueling_combine_bwd) X(talos_dqn_target)   \
  X(talos_dqn_loss_fwd_bwd) X(talos_soft_update) X(talos_mla_decode_step) X(talos_decode_advance) X(talos_transpose) X(talos_concat_last)      \
  X(talos_layernorm_fwd) X(talos_layernorm_bwd) X(talos_dropout_fwd) X(talos_dropout_bwd) X(talos_dropout_add_layernorm_fwd)                     \
  X(talos_dropout_add_layernorm_bwd) X(talos_policy_loss_fwd_bwd) X(talos_attention_lse_fwd) X(talos_attention_lse_bwd)                          \
  X(talos_split_last) X(talos_last_token) X(talos_eltwise_unary) X(talos_eltwise_unary_bwd) X(talos_eltwise_binary) X(talos_eltwise_binary_bwd) \
  X(talos_reduce_sum) X(talos_fill_from_scalar) X(talos_ppo_loss_fwd_bwd) X(talos_adam_step) X(talos_adam_step_global_clip)                    \
  X(talos_rng_uniform_host) X(talos_rng_normal_host) X(talos_rng_bounded_host) X(talos_lcg_rand_host) X(talos_comm_unique_id)                  \
  X(talos_comm_init) X(talos_comm_destroy) X(talos_comm_allreduce_sum) X(talos_debug_comm_stall) X(talos_ppo_create) X(talos_ppo_destroy)      \
  X(talos_ppo_param_count) X(talos_ppo_set_params_host) X(talos_ppo_get_params_host) X(talos_ppo_get_grads_host) X(talos_ppo_reset_optimizer)  \
  X(talos_ppo_set_lr) X(talos_ppo_forward) X(talos_ppo_log_prob) X(talos_ppo_step) X(talos_ppo_update) X(talos_ppo_update_host)                \
  X(talos_ppo_last_loss)

#define TALOS_DEFINE(f) PyObject* py_##f(PyObject*, PyObject* const* args, Py_ssize_t n) { return call(f, #f, args, n); }
TALOS_FUNCTIONS(TALOS_DEFINE)

// setup(TalosError, ctypes.c_void_p, {name: ctypes function})
PyObject* py_setup(PyObject*, PyObject* args) {
  PyObject *error, *handle, *fallback;
  if (!PyArg_ParseTuple(args, "OOO!", &error, &handle, &PyDict_Type, &fallback)) return nullptr;
  Py_INCREF(error); Py_INCREF(handle); Py_INCREF(fallback);
  Py_XSETREF(g_error, error); Py_XSETREF(g_handle_type, handle); Py_XSETREF(g_fallback, fallback);
  Py_RETURN_NONE;
}

#define TALOS_ENTRY(f) {#f, (PyCFunction)(void (*)(void))py_##f, METH_FASTCALL, nullptr},
PyMethodDef methods[] = {TALOS_FUNCTIONS(TALOS_ENTRY){"setup", py_setup, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pycall(void) {
  g_value = PyUnicode_InternFromString("value");
  return g_value ? PyModule_Create(&module) : nullptr;
}

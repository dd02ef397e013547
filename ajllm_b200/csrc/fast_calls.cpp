// The serving operators' ordinary call, from tensors to launch, as a Python extension.
//
// A small call of these operators runs for 3 to 7 us on the device, and checking its arguments attribute by attribute,
// allocating and packing took Python 5 to 9 us. Here the same checks are field reads. What they find wanting, and whatever
// is not an ordinary CUDA call (CPU tensors, another device than the current one, strides that need a copy, a given `out`
// of two of the three, subclasses), makes these functions return None: ops/serving.py then takes the same call through its
// own checks, which name what is wrong. Nothing is computed here, and nothing kept between calls.
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "serving_args.h"

namespace {

using Entry = int (*)(const void*);
Entry batch_maps_entry = nullptr, shared_prefix_entry = nullptr, process_logits_entry = nullptr;
const char* (*last_error)() = nullptr;

const at::Tensor* tensor(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// a contiguous tensor of this type, device and shape
bool plain(const at::Tensor* t, at::ScalarType type, int device, at::IntArrayRef shape) {
  return t != nullptr && t->layout() == at::kStrided && t->is_cuda() && t->get_device() == device && t->scalar_type() == type &&
         t->sizes() == shape && t->is_contiguous();
}

// an int in [least, most]
bool whole(PyObject* o, long long least, long long most, long long& value) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  value = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0 && value >= least && value <= most;
}

// the entry's status, without the GIL (a launch may wait for room in the queue)
int run(Entry entry, const void* args) {
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = entry(args);
  Py_END_ALLOW_THREADS
  return status;
}

PyObject* failed(const char* name, int status) {
  const char* detail = last_error != nullptr ? last_error() : nullptr;
  PyErr_Format(PyExc_RuntimeError, "%s failed with status %d: %s", name, status, detail != nullptr ? detail : "");
  return nullptr;
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

at::TensorOptions on(int device, at::ScalarType type) {
  return at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)device));
}

// (block_ids, block_counts, cached_lens, q_lens, total_tokens, max_blocks, block_size, pad_block, out or None)
// -> True when out was written, a tuple of the five results, or None
PyObject* fast_batch_maps(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 9 || batch_maps_entry == nullptr) Py_RETURN_NONE;
  const at::Tensor *ids = tensor(a[0]), *counts = tensor(a[1]), *cached = tensor(a[2]), *q_lens = tensor(a[3]);
  long long total, width, block, pad;
  if (ids == nullptr || counts == nullptr || !ids->is_cuda() || ids->dim() != 1 || counts->dim() != 1 ||
      !whole(a[4], 0, (1 << 30) - 1, total) || !whole(a[5], 1, INT_MAX, width) || !whole(a[6], 1, INT_MAX, block) ||
      !whole(a[7], 0, INT_MAX, pad))
    Py_RETURN_NONE;
  const int device = ids->get_device();
  const int64_t n = counts->size(0), n_ids = ids->size(0);
  if (device != c10::cuda::current_device() || n > 16384 || n_ids >= (1 << 30) || !plain(ids, at::kInt, device, {n_ids}) ||
      !plain(counts, at::kInt, device, {n}) || !plain(cached, at::kInt, device, {n}) || !plain(q_lens, at::kInt, device, {n}))
    Py_RETURN_NONE;
  const at::Tensor* out[5];
  at::Tensor made[5];
  const bool given = a[8] != Py_None;
  if (given) {
    if (!PyTuple_Check(a[8]) || PyTuple_GET_SIZE(a[8]) != 5) Py_RETURN_NONE;
    for (int i = 0; i < 5; ++i) out[i] = tensor(PyTuple_GET_ITEM(a[8], i));
    if (!plain(out[0], at::kInt, device, {n, width}) || !plain(out[1], at::kInt, device, {total}) ||
        !plain(out[2], at::kLong, device, {total}) || !plain(out[3], at::kInt, device, {n + 1}) || !plain(out[4], at::kInt, device, {n}))
      Py_RETURN_NONE;
  } else {
    made[0] = at::empty({n, width}, on(device, at::kInt));
    made[1] = at::empty({total}, on(device, at::kInt));
    made[2] = at::empty({total}, on(device, at::kLong));
    made[3] = at::empty({n + 1}, on(device, at::kInt));
    made[4] = at::empty({n}, on(device, at::kInt));
    for (int i = 0; i < 5; ++i) out[i] = &made[i];
  }
  BatchMapsArgs args;
  args.size = sizeof(args);
  args.ids = ids->data_ptr(); args.counts = counts->data_ptr(); args.cached = cached->data_ptr(); args.q_lens = q_lens->data_ptr();
  args.n_ids = (int)n_ids; args.seqs = (int)n; args.total = (int)total; args.width = (int)width;
  args.block_size = (int)block; args.pad = (int)pad;
  args.tables = out[0]->data_ptr(); args.positions = out[1]->data_ptr(); args.slots = out[2]->data_ptr();
  args.q_start = out[3]->data_ptr(); args.context = out[4]->data_ptr();
  args.stream = stream_of(device);
  if (const int status = run(batch_maps_entry, &args)) return failed("ajb_batch_maps", status);
  if (given) Py_RETURN_TRUE;
  PyObject* result = PyTuple_New(5);
  if (result == nullptr) return nullptr;
  for (int i = 0; i < 5; ++i) {
    PyObject* item = THPVariable_Wrap(made[i]);
    if (item == nullptr) { Py_DECREF(result); return nullptr; }
    PyTuple_SET_ITEM(result, i, item);
  }
  return result;
  END_HANDLE_TH_ERRORS
}

// (q, key_cache, value_cache, block_tables, context_lens, prefix_len, q_len, scale or None, max_context or None, prefix_plan)
// -> the result, or None
PyObject* fast_shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 10 || shared_prefix_entry == nullptr) Py_RETURN_NONE;
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *tables = tensor(a[3]), *context = tensor(a[4]);
  long long prefix, q_len;
  if (q == nullptr || k == nullptr || tables == nullptr || !q->is_cuda() || q->dim() != 3 || k->dim() != 4 || tables->dim() != 2 ||
      !whole(a[5], 0, INT_MAX, prefix) || !whole(a[6], 1, INT_MAX, q_len))
    Py_RETURN_NONE;
  const int device = q->get_device();
  const int64_t total = q->size(0), heads = q->size(1), hd = q->size(2), blocks = k->size(0), block = k->size(1), kv_heads = k->size(2),
                n = tables->size(0), max_blocks = tables->size(1);
  if (device != c10::cuda::current_device() || total == 0 || total != n * q_len || k->size(3) != hd || kv_heads < 1 || heads < 1 ||
      heads % kv_heads != 0 || blocks < 1 || block < 1 || max_blocks < 1 || prefix > max_blocks * block ||
      std::max({total * heads, blocks, block, max_blocks * block, heads, hd}) > (1 << 30) ||
      !plain(q, at::kBFloat16, device, q->sizes()) || !plain(k, at::kBFloat16, device, k->sizes()) ||
      !plain(v, at::kBFloat16, device, k->sizes()) || !plain(tables, at::kInt, device, tables->sizes()) ||
      !plain(context, at::kInt, device, {n}) || reinterpret_cast<uintptr_t>(q->data_ptr()) % 16 != 0)
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt((double)hd);
  if (a[7] != Py_None) {
    if (!PyFloat_CheckExact(a[7])) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(a[7]);
    if (!(scale >= 1e-30 && scale <= 1e3)) Py_RETURN_NONE;
  }
  const long long shared = prefix / block * block, room = max_blocks * block;
  long long behind = room - shared;
  if (a[8] != Py_None) {
    long long bound;
    if (!whole(a[8], LLONG_MIN, LLONG_MAX, bound)) Py_RETURN_NONE;
    // in whole tiles of 128 keys, like ops/serving.py: contexts that grow by a token per step keep their plan for 128 steps
    behind = (std::max(0ll, std::min(bound, room) - shared) + 127) / 128 * 128;
  }
  PyObject* plan = PyObject_CallFunction(a[9], "LLLLLLLL", (long long)n, q_len, (long long)(heads / kv_heads), (long long)kv_heads,
                                         (long long)hd, shared, behind, (long long)(a[8] != Py_None));
  if (plan == nullptr) return nullptr;
  int tokens, prefix_splits, splits, parts;
  const bool understood = PyArg_ParseTuple(plan, "iiii", &tokens, &prefix_splits, &splits, &parts);
  Py_DECREF(plan);
  if (!understood) return nullptr;
  const int64_t count = total * heads * parts;          // fp32 parts: un-normalised outputs, then (reference maximum, sum) pairs
  at::Tensor out = at::empty(q->sizes(), on(device, at::kBFloat16));
  at::Tensor workspace = at::empty({count * (hd + 2)}, on(device, at::kFloat));
  float* part_o = workspace.data_ptr<float>();
  SharedPrefixArgs args;
  args.size = sizeof(args);
  args.q = q->data_ptr(); args.k_cache = k->data_ptr(); args.v_cache = v->data_ptr(); args.block_tables = tables->data_ptr();
  args.context_lens = context->data_ptr(); args.out = out.data_ptr(); args.q_pitch = heads * hd;
  args.num_seqs = (int)n; args.num_blocks = (int)blocks; args.block_size = (int)block; args.max_blocks = (int)max_blocks;
  args.heads = (int)heads; args.kv_heads = (int)kv_heads; args.head_dim = (int)hd; args.q_len = (int)q_len; args.shared = (int)shared;
  args.scale = (float)scale; args.prefix_tokens = tokens; args.prefix_splits = prefix_splits; args.suffix_splits = splits;
  args.parts = parts; args.part_o = part_o; args.part_ml = part_o + count * hd; args.stream = stream_of(device);
  if (const int status = run(shared_prefix_entry, &args)) return failed("ajb_shared_prefix_attention", status);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (logits, history, prompt_lens, history_lens, repetition, presence, frequency, bias_ids, bias_values, token_mask) -> the
// result, or None
PyObject* fast_process_logits(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  if (n_args != 10 || process_logits_entry == nullptr) Py_RETURN_NONE;
  const at::Tensor* logits = tensor(a[0]);
  if (logits == nullptr || !logits->is_cuda() || logits->layout() != at::kStrided || logits->dim() != 2) Py_RETURN_NONE;
  const int device = logits->get_device();
  const at::ScalarType type = logits->scalar_type();
  const int64_t rows = logits->size(0), vocab = logits->size(1);
  if (device != c10::cuda::current_device() || (type != at::kBFloat16 && type != at::kFloat) || vocab < 1 || vocab > (1 << 30) ||
      rows > INT_MAX || logits->stride(1) != 1)
    Py_RETURN_NONE;
  // null for None; `wanted` says whether a tensor that is there is as it has to be
  bool wanted = true;
  auto optional = [&](PyObject* o, at::ScalarType t, at::IntArrayRef shape) -> void* {
    if (o == Py_None) return nullptr;
    const at::Tensor* x = tensor(o);
    if (!plain(x, t, device, shape)) { wanted = false; return nullptr; }
    return x->data_ptr();
  };
  ProcessLogitsArgs args;
  args.size = sizeof(args);
  int64_t width = 0, biases = 0;
  if (a[1] != Py_None) {
    const at::Tensor* history = tensor(a[1]);
    if (history == nullptr || history->dim() != 2 || a[2] == Py_None || a[3] == Py_None) Py_RETURN_NONE;
    width = history->size(1);
  } else {
    for (int i = 2; i < 7; ++i)
      if (a[i] != Py_None) Py_RETURN_NONE;
  }
  if ((a[7] == Py_None) != (a[8] == Py_None)) Py_RETURN_NONE;
  if (a[7] != Py_None) {
    const at::Tensor* ids = tensor(a[7]);
    if (ids == nullptr || ids->dim() != 2) Py_RETURN_NONE;
    biases = ids->size(1);
  }
  if (width > INT_MAX || biases > INT_MAX) Py_RETURN_NONE;
  args.history = optional(a[1], at::kInt, {rows, width});
  args.prompt_lens = optional(a[2], at::kInt, {rows});
  args.history_lens = optional(a[3], at::kInt, {rows});
  args.repetition = optional(a[4], at::kFloat, {rows});
  args.presence = optional(a[5], at::kFloat, {rows});
  args.frequency = optional(a[6], at::kFloat, {rows});
  args.bias_ids = optional(a[7], at::kInt, {rows, biases});
  args.bias_values = optional(a[8], at::kFloat, {rows, biases});
  args.mask_pitch = (vocab + 31) / 32;
  args.mask = optional(a[9], at::kInt, {rows, args.mask_pitch});
  if (!wanted) Py_RETURN_NONE;
  at::Tensor out = at::empty({rows, vocab}, on(device, at::kFloat));
  args.logits = logits->data_ptr(); args.dtype = type == at::kFloat ? 1 : 0; args.in_pitch = logits->stride(0);
  args.out = out.data_ptr(); args.rows = (int)rows; args.vocab = (int)vocab;
  if (width == 0) args.history = nullptr;
  args.history_pitch = width; args.history_width = (int)width; args.biases = (int)biases;
  args.stream = stream_of(device);
  if (const int status = run(process_logits_entry, &args)) return failed("ajb_process_logits", status);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// addresses of ajb_batch_maps, ajb_shared_prefix_attention, ajb_process_logits and ajb_last_error in the kernel library
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long at[4];
  if (!PyArg_ParseTuple(args, "KKKK", &at[0], &at[1], &at[2], &at[3])) return nullptr;
  batch_maps_entry = reinterpret_cast<Entry>(at[0]);
  shared_prefix_entry = reinterpret_cast<Entry>(at[1]);
  process_logits_entry = reinterpret_cast<Entry>(at[2]);
  last_error = reinterpret_cast<const char* (*)()>(at[3]);
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction as_method(F* f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"batch_maps", as_method(fast_batch_maps), METH_FASTCALL, nullptr},
    {"shared_prefix_attention", as_method(fast_shared_prefix_attention), METH_FASTCALL, nullptr},
    {"process_logits", as_method(fast_process_logits), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "fast_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fast_calls() { return PyModule_Create(&module); }

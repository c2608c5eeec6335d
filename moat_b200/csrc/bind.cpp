// The Python side of the drafted-decoding entry points (moat_b200/tree.py, evict.py): tests of
// the tensors, results, workspaces and the C call in one step. In Python, with some 70 tensor
// attributes to read, the same took 12 to 19 us of host time per call, more than most of the kernels.
//
// Every function returns its result, a status of the C call (an int), or None where an argument does
// not fit; which one and why, a slower pass in Python finds out.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <vector>

#include "moat_b200.h"

namespace {

// From the CUDA library, which moat_b200/_lib.py loads: set_entry_points hands their addresses over.
decltype(&mb_tree_attn) tree_attn;
decltype(&mb_tree_attn_workspace_size) tree_attn_workspace_size;
decltype(&mb_tree_accept) tree_accept;
decltype(&mb_cache_evict) cache_evict;
decltype(&mb_cache_evict_workspace_size) cache_evict_workspace_size;

using at::IntArrayRef;
using at::ScalarType;
using at::Tensor;

// A tensor argument; null if it is none.
const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// What the call takes must all lie on one device.
struct Device {
  int index = -1;
  bool add(const Tensor* x) {
    if (!x || !x->is_cuda()) return false;
    if (index < 0) index = x->get_device();
    return x->get_device() == index;
  }
  template <class... Rest>
  bool add(const Tensor* x, Rest... rest) {
    return add(x) && add(rest...);
  }
};

// A contiguous tensor of one dtype and shape.
bool plain(const Tensor* x, ScalarType type, IntArrayRef shape) {
  return x->scalar_type() == type && x->sizes() == shape && x->is_contiguous();
}

// The device error word: the kernels do 32-bit atomics on its first element.
bool error_word(const Tensor* x) { return x->scalar_type() == at::kInt && x->numel() > 0; }

bool unit_stride(const Tensor* x) { return x->stride(-1) == 1 || x->size(-1) == 1; }

// Every element has a place of its own as far as broadcast axes go: what is written by several CTAs
// must not share addresses.
bool no_broadcast(const Tensor* x) {
  for (int64_t u = 0; u < x->dim(); ++u)
    if (x->stride(u) == 0 && x->size(u) > 1) return false;
  return true;
}

bool small(IntArrayRef sizes) {
  for (int64_t n : sizes)
    if (n > INT_MAX) return false;
  return true;
}

template <class T>
T* address(const Tensor* x) {
  return x ? static_cast<T*>(x->data_ptr()) : nullptr;
}

Tensor make(IntArrayRef shape, ScalarType type, int device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, device)));
}

// A contiguous tensor in another's memory.
Tensor part_of(const Tensor& x, int64_t offset, IntArrayRef shape) {
  Tensor part = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(x.storage()), x.key_set(), x.dtype());
  part.unsafeGetTensorImpl()->set_storage_offset(offset);
  part.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  return part;
}

// Scratch of one call, from torch's allocator on the current device and stream: it goes back when
// the call has been enqueued, and whatever gets it next on that stream comes after. The kernels
// expect no initial contents. A call that is captured takes it from its graph's pool, so that
// graphs share none.
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

// Runs `body`; a C++ exception becomes torch's Python error for it (out of memory is its own).
template <class Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (...) {
    if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

PyObject* borrowed(PyObject* o) {
  Py_INCREF(o);
  return o;
}

PyObject* none() { return borrowed(Py_None); }

PyObject* tuple(std::initializer_list<PyObject*> items) {
  PyObject* t = PyTuple_New(items.size());
  Py_ssize_t i = 0;
  for (PyObject* x : items) PyTuple_SET_ITEM(t, i++, x);
  return t;
}

// q, k_cache, v_cache, lens, k_draft, v_draft, masks, scale, out, scores, scores_out, draft_scores, dev_err
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 13) return none();
  return guarded([&]() -> PyObject* {
    const Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *lens = tensor(args[3]),
                 *kd = tensor(args[4]), *vd = tensor(args[5]), *masks = tensor(args[6]);
    Device dev;
    if (!dev.add(q, k, v, lens, kd, vd, masks) || q->dim() != 4 || k->dim() != 4 || kd->dim() != 4) return none();
    const int64_t T = q->size(0), m = q->size(1), H = q->size(2), d = q->size(3), Hkv = k->size(1), Lmax = k->size(2);
    const ScalarType type = q->scalar_type();
    if (m < 1 || m > 64 || T < 1 || Hkv < 1 || H < 1 || H % Hkv || d < 1 || d > 256 || !small(q->sizes()) ||
        !small(k->sizes()) || k->sizes() != IntArrayRef{T, Hkv, Lmax, d} || v->sizes() != k->sizes() ||
        kd->sizes() != IntArrayRef{T, m, Hkv, d} || vd->sizes() != kd->sizes() ||
        (type != at::kHalf && type != at::kBFloat16) || k->scalar_type() != type || v->scalar_type() != type ||
        kd->scalar_type() != type || vd->scalar_type() != type || !unit_stride(q) || !unit_stride(k) ||
        !unit_stride(v) || !unit_stride(kd) || !unit_stride(vd) || !plain(lens, at::kInt, {T}) ||
        !(masks->dim() == 1 ? plain(masks, at::kLong, {m}) : plain(masks, at::kLong, {T, m})))
      return none();
    Tensor made[2];
    const Tensor* out = args[8] == Py_None ? &(made[0] = make(q->sizes(), type, dev.index)) : tensor(args[8]);
    if (!dev.add(out) || out->sizes() != q->sizes() || out->scalar_type() != type || !unit_stride(out) ||
        !no_broadcast(out))
      return none();
    const Tensor *scores = nullptr, *scores_out = nullptr, *draft_scores = nullptr, *err = nullptr;
    if (args[9] != Py_None) {
      scores = tensor(args[9]);
      scores_out = args[10] == Py_None ? scores : tensor(args[10]);
      draft_scores = args[11] == Py_None ? &(made[1] = make({T, Hkv, m}, at::kFloat, dev.index)) : tensor(args[11]);
      if (!dev.add(scores, scores_out, draft_scores) || !plain(scores, at::kFloat, {T, Hkv, Lmax}) ||
          !plain(scores_out, at::kFloat, {T, Hkv, Lmax}) || !plain(draft_scores, at::kFloat, {T, Hkv, m}))
        return none();
      if (out->data_ptr() == q->data_ptr()) return none();  // the weights read q after the outputs are there
    } else if (args[10] != Py_None || args[11] != Py_None) {
      return none();
    }
    if (args[12] != Py_None && (!dev.add(err = tensor(args[12])) || !error_word(err))) return none();
    double scale = 1.0 / std::sqrt(static_cast<double>(d));
    if (args[7] != Py_None) {
      scale = PyFloat_AsDouble(args[7]);
      if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    }
    if (!std::isfinite(static_cast<float>(scale))) {
      PyErr_SetString(PyExc_ValueError, "scale must be finite");
      return nullptr;
    }
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != dev.index) guard.set_index(dev.index);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index).stream();
    const size_t bytes = tree_attn_workspace_size(T, m, H, Hkv, Lmax, d, scores != nullptr);
    const c10::DataPtr space = scratch(bytes);
    mb_tree_attn_args a;
    a.q = address<uint16_t>(q);
    a.k_cache = address<uint16_t>(k);
    a.v_cache = address<uint16_t>(v);
    a.lens = address<int32_t>(lens);
    a.k_draft = address<uint16_t>(kd);
    a.v_draft = address<uint16_t>(vd);
    a.masks = address<int64_t>(masks);
    a.out = address<uint16_t>(out);
    a.scores = address<float>(scores);
    a.scores_out = address<float>(scores_out);
    a.draft_scores = address<float>(draft_scores);
    a.workspace = space.get();
    a.workspace_bytes = bytes;
    a.dev_err = address<uint32_t>(err);
    const Tensor* strided[6] = {q, k, v, kd, vd, out};
    for (int i = 0; i < 6; ++i)
      for (int u = 0; u < 3; ++u) a.strides[3 * i + u] = strided[i]->stride(u);
    a.shared_masks = masks->dim() == 1;
    a.is_bf16 = type == at::kBFloat16;
    a.T = T;
    a.m = m;
    a.H = H;
    a.Hkv = Hkv;
    a.Lmax = Lmax;
    a.d = d;
    a.scale = static_cast<float>(scale);
    const int rc = tree_attn(&a, stream);
    if (rc != MB_OK) return PyLong_FromLong(rc);
    PyObject* o = args[8] == Py_None ? THPVariable_Wrap(*out) : borrowed(args[8]);
    if (!scores) return o;
    return tuple({o, borrowed(args[10] == Py_None ? args[9] : args[10]),
                  args[11] == Py_None ? THPVariable_Wrap(*draft_scores) : borrowed(args[11])});
  });
}

// [layers, T, Hkv, Lmax, d] with or without the first axis.
struct Cache {
  int64_t layers, T, Hkv, Lmax, d;
  int lead;  // axes before T
  bool read(const Tensor* k, const Tensor* v) {
    lead = static_cast<int>(k->dim()) - 4;
    if (lead < 0 || lead > 1 || k->numel() == 0 || !small(k->sizes()) || v->sizes() != k->sizes() ||
        v->scalar_type() != k->scalar_type() || k->element_size() != 2 || !unit_stride(k) || !unit_stride(v) ||
        !no_broadcast(k) || !no_broadcast(v))  // its rows are written
      return false;
    layers = lead ? k->size(0) : 1;
    T = k->size(lead);
    Hkv = k->size(lead + 1);
    Lmax = k->size(lead + 2);
    d = k->size(lead + 3);
    return true;
  }
  // strides by (layer, trace, head or node, row or head); without a layer axis its is not used
  void strides(const Tensor* x, int64_t* to) const {
    to[0] = lead ? x->stride(0) : 0;
    for (int u = 0; u < 3; ++u) to[1 + u] = x->stride(lead + u);
  }
};

// tokens, parents, target, lens, next_pos, k_cache, v_cache, k_draft, v_draft, scores, draft_scores, positions, dev_err
PyObject* accept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 13) return none();
  return guarded([&]() -> PyObject* {
    const Tensor *tokens = tensor(args[0]), *parents = tensor(args[1]), *target = tensor(args[2]),
                 *lens = tensor(args[3]), *next_pos = tensor(args[4]), *k = tensor(args[5]), *v = tensor(args[6]),
                 *kd = tensor(args[7]), *vd = tensor(args[8]);
    Device dev;
    Cache c;
    if (!dev.add(k, v, kd, vd, tokens, parents, target, lens, next_pos) || !c.read(k, v) || kd->dim() != k->dim())
      return none();
    const int64_t m = kd->size(c.lead + 1);
    const ScalarType type = k->scalar_type();
    std::vector<int64_t> shape(k->sizes().begin(), k->sizes().end());  // of the drafts, then of scores
    shape[c.lead + 1] = m;
    shape[c.lead + 2] = c.Hkv;
    if (m < 1 || m > 64 || kd->sizes() != IntArrayRef(shape) || vd->sizes() != kd->sizes() ||
        kd->scalar_type() != type || vd->scalar_type() != type || !unit_stride(kd) || !unit_stride(vd) ||
        !plain(tokens, at::kInt, {c.T, m}) || !plain(target, at::kInt, {c.T, m}) || !plain(lens, at::kInt, {c.T}) ||
        !plain(next_pos, at::kInt, {c.T}) ||
        !(parents->dim() == 1 ? plain(parents, at::kInt, {m}) : plain(parents, at::kInt, {c.T, m})))
      return none();
    const Tensor *scores = nullptr, *draft_scores = nullptr, *positions = nullptr, *err = nullptr;
    const IntArrayRef rows = k->sizes().slice(0, c.lead + 3);
    if ((args[9] == Py_None) != (args[10] == Py_None)) return none();
    if (args[9] != Py_None) {
      scores = tensor(args[9]);
      draft_scores = tensor(args[10]);
      shape.assign(rows.begin(), rows.end());
      shape.back() = m;
      if (!dev.add(scores, draft_scores) || !plain(scores, at::kFloat, rows) ||
          !plain(draft_scores, at::kFloat, shape))
        return none();
    }
    if (args[11] != Py_None && (!dev.add(positions = tensor(args[11])) || !plain(positions, at::kInt, rows)))
      return none();
    if (args[12] != Py_None && (!dev.add(err = tensor(args[12])) || !error_word(err))) return none();
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != dev.index) guard.set_index(dev.index);
    const Tensor all = make({c.T * (m + 4)}, at::kInt, dev.index);  // one allocation for the five results
    const Tensor counts = part_of(all, 0, {c.T}), next_ids = part_of(all, c.T, {c.T}),
                 new_lens = part_of(all, 2 * c.T, {c.T}), new_pos = part_of(all, 3 * c.T, {c.T}),
                 path = part_of(all, 4 * c.T, {c.T, m});
    mb_tree_accept_args a;
    a.tokens = address<int32_t>(tokens);
    a.parents = address<int32_t>(parents);
    a.target = address<int32_t>(target);
    a.lens = address<int32_t>(lens);
    a.next_pos = address<int32_t>(next_pos);
    a.k_cache = address<uint16_t>(k);
    a.v_cache = address<uint16_t>(v);
    a.k_draft = address<uint16_t>(kd);
    a.v_draft = address<uint16_t>(vd);
    a.scores = address<float>(scores);
    a.draft_scores = address<float>(draft_scores);
    a.positions = address<int32_t>(positions);
    a.path = address<int32_t>(&path);
    a.counts = address<int32_t>(&counts);
    a.next_ids = address<int32_t>(&next_ids);
    a.lens_out = address<int32_t>(&new_lens);
    a.pos_out = address<int32_t>(&new_pos);
    a.dev_err = address<uint32_t>(err);
    c.strides(k, a.strides);
    c.strides(v, a.strides + 4);
    c.strides(kd, a.strides + 8);
    c.strides(vd, a.strides + 12);
    a.shared_parents = parents->dim() == 1;
    a.layers = c.layers;
    a.T = c.T;
    a.m = m;
    a.Hkv = c.Hkv;
    a.Lmax = c.Lmax;
    a.d = c.d;
    const int rc = tree_accept(&a, c10::cuda::getCurrentCUDAStream(dev.index).stream());
    if (rc != MB_OK) return PyLong_FromLong(rc);
    return tuple({THPVariable_Wrap(path), THPVariable_Wrap(counts), THPVariable_Wrap(next_ids),
                  THPVariable_Wrap(new_lens), THPVariable_Wrap(new_pos)});
  });
}

// k_cache, v_cache, scores, positions, lens, next_pos, scores_out, positions_out, budget, recent, sinks
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11) return none();
  return guarded([&]() -> PyObject* {
    const Tensor *k = tensor(args[0]), *v = tensor(args[1]), *scores = tensor(args[2]), *positions = tensor(args[3]),
                 *lens = tensor(args[4]), *next_pos = tensor(args[5]), *scores_out = tensor(args[6]),
                 *positions_out = tensor(args[7]);
    Device dev;
    Cache c;
    if (!dev.add(k, v, scores, positions, lens, next_pos, scores_out, positions_out) || !c.read(k, v)) return none();
    const IntArrayRef rows = k->sizes().slice(0, c.lead + 3);
    if (!plain(scores, at::kFloat, rows) || !plain(scores_out, at::kFloat, rows) ||
        !plain(positions, at::kInt, rows) || !plain(positions_out, at::kInt, rows) || !plain(lens, at::kInt, {c.T}) ||
        !plain(next_pos, at::kInt, {c.T}))
      return none();
    int64_t number[3];  // budget, recent, sinks
    for (int i = 0; i < 3; ++i) {
      number[i] = PyLong_AsLongLong(args[8 + i]);
      if (number[i] == -1 && PyErr_Occurred()) return nullptr;
      if (number[i] > INT_MAX || number[i] < INT_MIN) number[i] = -1;
    }
    if (number[0] < 1 || number[1] < 0 || number[2] < 0 || number[1] + number[2] > number[0]) {
      PyErr_SetString(PyExc_ValueError, "budget must be positive and hold the recent rows and the sinks");
      return nullptr;
    }
    if ((scores->data_ptr() == scores_out->data_ptr()) != (positions->data_ptr() == positions_out->data_ptr())) {
      PyErr_SetString(PyExc_ValueError, "scores and positions are both updated in place, or neither");
      return nullptr;
    }
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != dev.index) guard.set_index(dev.index);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index).stream();
    const Tensor new_lens = make({c.T}, at::kInt, dev.index);
    const size_t bytes =
        cache_evict_workspace_size(c.layers, c.T, c.Hkv, c.Lmax, static_cast<int>(number[0]));
    const c10::DataPtr space = scratch(bytes);
    mb_cache_evict_args a;
    a.k_cache = address<uint16_t>(k);
    a.v_cache = address<uint16_t>(v);
    a.scores = address<float>(scores);
    a.positions = address<int32_t>(positions);
    a.scores_out = address<float>(scores_out);
    a.positions_out = address<int32_t>(positions_out);
    a.lens = address<int32_t>(lens);
    a.next_pos = address<int32_t>(next_pos);
    a.lens_out = address<int32_t>(&new_lens);
    a.workspace = space.get();
    a.workspace_bytes = bytes;
    c.strides(k, a.strides);
    c.strides(v, a.strides + 4);
    a.layers = c.layers;
    a.T = c.T;
    a.Hkv = c.Hkv;
    a.Lmax = c.Lmax;
    a.d = c.d;
    a.budget = static_cast<int>(number[0]);
    a.recent = static_cast<int>(number[1]);
    a.sinks = static_cast<int>(number[2]);
    const int rc = cache_evict(&a, stream);
    if (rc != MB_OK) return PyLong_FromLong(rc);
    return tuple({borrowed(args[6]), borrowed(args[7]), THPVariable_Wrap(new_lens)});
  });
}

// addresses of mb_tree_attn, its workspace size, mb_tree_accept, mb_cache_evict, its workspace size
PyObject* set_entry_points(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) return none();
  void* p[5];
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  tree_attn = reinterpret_cast<decltype(tree_attn)>(p[0]);
  tree_attn_workspace_size = reinterpret_cast<decltype(tree_attn_workspace_size)>(p[1]);
  tree_accept = reinterpret_cast<decltype(tree_accept)>(p[2]);
  cache_evict = reinterpret_cast<decltype(cache_evict)>(p[3]);
  cache_evict_workspace_size = reinterpret_cast<decltype(cache_evict_workspace_size)>(p[4]);
  return none();
}

PyMethodDef methods[] = {
    {"set_entry_points", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_entry_points)), METH_FASTCALL,
     nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {"accept", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(accept)), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(evict)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "moat_bind", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_moat_bind() { return PyModule_Create(&module); }

// The host side of the calls that are short on the GPU, natively: checks,
// allocations and launches of one call without a round trip through Python for
// each of them.
//
// A 17 x 5120 x 5120 linear keeps the GPU busy for 11 us, while the Python wrappers
// of its two kernels (argument checks, four allocations, two ctypes calls) take 24 us
// of host time; here it takes 10.  The adapter linear: 16 us of GPU time at 256 x 1536
// x 4608, 34 us of host time in the wrappers, 11 here.  Each function here takes
// the tensors of a call, and either runs the whole of it on the tensor's current
// stream or returns None without having enqueued anything that the caller sees:
// every other layout, type, device or error goes on to the Python wrappers, which
// decide and report as before.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "../../include/vflash_amd.h"

namespace {

// The tensor behind a plain torch.Tensor or torch.nn.Parameter, else null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  // A tensor with a pending sign (torch._neg_view) is not what its memory holds.
  return t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() ? &t : nullptr;
}

bool gfx950(c10::DeviceIndex index) {
  const char* arch = at::cuda::getDeviceProperties(index)->gcnArchName;
  return std::strncmp(arch, "gfx950", 6) == 0 && (arch[6] == 0 || arch[6] == ':');
}

// The operands of a W8A8 linear in the layout the kernels take without a copy.
struct Linear {
  const at::Tensor *x, *w, *sw, *b;
  int64_t m, n, k, m_pad;
};

bool linear_ok(PyObject* const* a, Linear& l) {
  l.x = plain(a[0]);
  l.w = plain(a[1]);
  l.sw = plain(a[2]);
  l.b = a[3] == Py_None ? nullptr : plain(a[3]);
  if (!l.x || !l.w || !l.sw || (a[3] != Py_None && !l.b)) return false;
  if (l.x->scalar_type() != at::kBFloat16 || l.w->scalar_type() != at::kFloat8_e4m3fn ||
      l.sw->scalar_type() != at::kFloat)
    return false;
  if (l.x->dim() < 1 || l.w->dim() != 2 || !l.x->is_contiguous() || !l.sw->is_contiguous()) return false;
  l.n = l.w->size(0);
  l.k = l.w->size(1);
  if (l.n < 1 || l.k < 16 || l.k % 16 || l.x->size(-1) != l.k || l.x->numel() == 0) return false;
  if (l.w->stride(1) != 1 || l.sw->dim() != 2 || l.sw->size(0) != l.n || l.sw->size(1) != 1) return false;
  const c10::Device d = l.x->device();
  if (l.w->device() != d || l.sw->device() != d) return false;
  if (l.b && (l.b->dim() != 1 || l.b->size(0) != l.n || l.b->scalar_type() != at::kBFloat16 ||
              l.b->device() != d || !l.b->is_contiguous()))
    return false;
  l.m = l.x->numel() / l.k;
  l.m_pad = (l.m + 15) / 16 * 16;
  return gfx950(d.index());
}

// Other Python threads run while this one allocates and launches.
struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

at::Tensor output(const Linear& l) {
  c10::SmallVector<int64_t, 5> shape(l.x->sizes().begin(), l.x->sizes().end());
  shape.back() = l.n;
  return at::empty(shape, l.x->options().requires_grad(false));
}

// w8a8_linear(value, weight, scale, bias): quantize the rows, then the GEMM.
PyObject* w8a8_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Linear l;
  if (nargs != 4 || !linear_ok(a, l)) Py_RETURN_NONE;
  at::Tensor out;
  int status;
  {
    const NoGil nogil;
    // Two allocations: with the scales right behind the codes (a whole number of
    // megabytes away) the 4096x3072x3072 linear took 43.8 us instead of 42.9.
    const at::Tensor code_rows = at::empty({l.m_pad, l.k}, l.x->options().dtype(at::kByte));
    const at::Tensor row_scales = at::empty({l.m_pad}, l.x->options().dtype(at::kFloat));
    out = output(l);
    uint8_t* codes = static_cast<uint8_t*>(code_rows.data_ptr());
    float* scales = static_cast<float*>(row_scales.data_ptr());
    void* stream = c10::hip::getCurrentHIPStream(l.x->device().index()).stream();
    status = vflash_quantize_rows_e4m3(l.x->data_ptr(), l.m, l.k, l.k, codes, scales, l.m_pad, stream);
    if (status == VFLASH_OK)
      status = vflash_fp8_linear(codes, scales, l.k, l.w->data_ptr(),
                                 static_cast<float*>(l.sw->data_ptr()), l.w->stride(0), l.m, l.n, l.k,
                                 l.b ? l.b->data_ptr() : nullptr, out.data_ptr(), l.n, stream);
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// w8a8_linear_lora(value, weight, scale, bias, down, up, scaling, strength): codes
// and t = bf16(x . down^T) in one launch, then the GEMM with the merged adapter.
PyObject* w8a8_linear_lora(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Linear l;
  if (nargs != 8 || !linear_ok(a, l)) Py_RETURN_NONE;
  const at::Tensor *down = plain(a[4]), *up = plain(a[5]);
  if (!down || !up || down->dim() != 2 || up->dim() != 2) Py_RETURN_NONE;
  const int64_t rank = down->size(0), ldt = (rank + 15) / 16 * 16;
  // Ranks that are a multiple of 8 need no padding of the rows of `up`.
  if (rank < 8 || rank > 128 || rank % 8 || down->size(1) != l.k || up->size(0) != l.n ||
      up->size(1) != rank)
    Py_RETURN_NONE;
  if (down->scalar_type() != at::kBFloat16 || up->scalar_type() != at::kBFloat16 ||
      !down->is_contiguous() || !up->is_contiguous() || down->device() != l.x->device() ||
      up->device() != l.x->device())
    Py_RETURN_NONE;
  const double scaling = PyFloat_AsDouble(a[6]), strength = PyFloat_AsDouble(a[7]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  at::Tensor out;
  int status;
  {
    const NoGil nogil;
    const at::Tensor code_rows = at::empty({l.m_pad, l.k}, l.x->options().dtype(at::kByte));
    const at::Tensor row_scales = at::empty({l.m_pad}, l.x->options().dtype(at::kFloat));
    const at::Tensor t_rows = at::empty({l.m, ldt}, l.x->options());
    out = output(l);
    uint8_t* codes = static_cast<uint8_t*>(code_rows.data_ptr());
    float* scales = static_cast<float*>(row_scales.data_ptr());
    void* t = t_rows.data_ptr();
    void* stream = c10::hip::getCurrentHIPStream(l.x->device().index()).stream();
    status = vflash_quantize_rows_lora_e4m3(l.x->data_ptr(), l.m, l.k, l.k, codes, scales, l.m_pad,
                                            down->data_ptr(), rank, t, ldt, stream);
    if (status == VFLASH_OK)
      status = vflash_fp8_linear_lora(codes, scales, l.k, l.w->data_ptr(),
                                      static_cast<float*>(l.sw->data_ptr()), l.w->stride(0), l.m, l.n,
                                      l.k, l.b ? l.b->data_ptr() : nullptr, t, ldt, up->data_ptr(),
                                      rank, rank, (float)scaling, (float)strength, out.data_ptr(), l.n,
                                      stream);
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// A gradient or a forward-mode tangent to carry: the wrappers refuse both.
bool records(const at::Tensor& t) {
  return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// nvfp4_w16_linear(values, packed, scales, alpha, bias): the weight-only NVFP4 linear.
PyObject* nvfp4_w16_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) Py_RETURN_NONE;
  const at::Tensor *x = plain(a[0]), *w = plain(a[1]), *ws = plain(a[2]), *alpha = plain(a[3]);
  const at::Tensor* b = a[4] == Py_None ? nullptr : plain(a[4]);
  if (!x || !w || !ws || !alpha || (a[4] != Py_None && !b)) Py_RETURN_NONE;
  if (records(*x) || (b && b->_fw_grad(0).defined())) Py_RETURN_NONE;
  const bool f16 = x->scalar_type() == at::kHalf;
  if ((!f16 && x->scalar_type() != at::kBFloat16) || w->scalar_type() != at::kByte || ws->scalar_type() != at::kByte ||
      alpha->scalar_type() != at::kFloat || alpha->numel() != 1)
    Py_RETURN_NONE;
  if (x->dim() < 1 || !x->is_contiguous() || w->dim() != 2 || !w->is_contiguous() || !ws->is_contiguous() || x->numel() == 0)
    Py_RETURN_NONE;
  const int64_t n = w->size(0), k = 2 * w->size(1);
  if (x->size(-1) != k || ws->dim() != 2 || ws->size(0) != n || ws->size(1) != k / 16) Py_RETURN_NONE;
  const c10::Device d = x->device();
  if (w->device() != d || ws->device() != d || alpha->device() != d || !gfx950(d.index())) Py_RETURN_NONE;
  if (b && (b->dim() != 1 || b->size(0) != n || b->scalar_type() != at::kBFloat16 || b->device() != d || !b->is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor out;
  int status;
  {
    const NoGil nogil;
    c10::SmallVector<int64_t, 5> shape(x->sizes().begin(), x->sizes().end());
    shape.back() = n;
    out = at::empty(shape, x->options().dtype(at::kBFloat16).requires_grad(false));
    // Alignments and limits are the entry's to refuse.
    status = vflash_nvfp4_w16_linear(x->data_ptr(), f16, k, w->data_ptr(), ws->data_ptr(),
                                     static_cast<float*>(alpha->data_ptr()), x->numel() / k, n, k,
                                     b ? b->data_ptr() : nullptr, out.data_ptr(), n,
                                     c10::hip::getCurrentHIPStream(d.index()).stream());
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// The offsets or lengths of `count` sequences (any number where it is negative).
const int64_t* indices(const at::Tensor* t, c10::Device d, int64_t count) {
  if (!t || t->scalar_type() != at::kLong || t->dim() != 1 || !t->is_contiguous() || t->device() != d ||
      (count >= 0 && t->numel() != count))
    return nullptr;
  return static_cast<const int64_t*>(t->data_ptr());
}

// packed_attention(q, k, v, q_offsets, k_offsets, k_lengths, causal, scale): with a causal of True
// or False and a scale of None or a float.
PyObject* packed_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 8 || !PyBool_Check(a[6]) || (a[7] != Py_None && !PyFloat_CheckExact(a[7]))) Py_RETURN_NONE;
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *qo = plain(a[3]), *ko = plain(a[4]);
  const at::Tensor* kl = a[5] == Py_None ? nullptr : plain(a[5]);
  if (!q || !k || !v || !qo || !ko || (a[5] != Py_None && !kl)) Py_RETURN_NONE;
  if (records(*q) || records(*k) || records(*v)) Py_RETURN_NONE;
  const auto type = q->scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || k->scalar_type() != type || v->scalar_type() != type) Py_RETURN_NONE;
  if (q->dim() != 3 || k->dim() != 3 || k->sizes() != v->sizes() || q->size(2) != k->size(2)) Py_RETURN_NONE;
  const c10::Device d = q->device();
  if (k->device() != d || v->device() != d || !gfx950(d.index()) || qo->numel() < 1) Py_RETURN_NONE;
  for (const at::Tensor* t : {q, k, v})
    if (t->stride(2) != 1 || !aligned16(*t)) Py_RETURN_NONE;
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2), keys = k->size(0), key_heads = k->size(1);
  const int64_t batch = qo->numel() - 1;
  const int64_t *q_offsets = indices(qo, d, -1), *k_offsets = indices(ko, d, kl ? batch : batch + 1);
  const int64_t* k_lengths = kl ? indices(kl, d, batch) : nullptr;
  if (!q_offsets || !k_offsets || (kl && !k_lengths) || tokens == 0) Py_RETURN_NONE;
  const int64_t bytes = vflash_packed_attention_workspace(tokens, keys, batch, heads, key_heads, dim);
  if (bytes < 0) Py_RETURN_NONE;
  const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)dim) : PyFloat_AS_DOUBLE(a[7]);
  const bool causal = a[6] == Py_True;
  at::Tensor out;
  int status;
  {
    const NoGil nogil;
    out = at::empty({tokens, heads, dim}, q->options().requires_grad(false));
    const at::Tensor workspace = bytes ? at::empty({bytes}, q->options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
    status = vflash_packed_attention(
        q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(),
        v->stride(0), v->stride(1), type == at::kHalf, tokens, keys, heads, key_heads, dim, q_offsets, k_offsets,
        k_lengths, batch, causal, (float)scale, out.data_ptr(), heads * dim, dim, bytes ? workspace.data_ptr() : nullptr,
        bytes, c10::hip::getCurrentHIPStream(d.index()).stream());
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// Tells autograd, which may have saved it, that the tensor has other values now.
void written(const at::Tensor* t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// A [rows, heads, dim] operand as the kernels of the heads take it, with nothing to record.
bool heads_ok(const at::Tensor* t, const at::Tensor& like) {
  return t->dim() == 3 && t->size(1) >= 1 && t->size(2) == like.size(2) && t->scalar_type() == like.scalar_type() &&
         t->device() == like.device() && t->stride(2) == 1 && t->stride(0) % 8 == 0 && t->stride(1) % 8 == 0 &&
         t->stride(0) < (int64_t(1) << 23) && aligned16(*t) && !records(*t);
}
bool half(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

// phases, axis, axes, interleaved, magnitude as vflash_amd.rotary.Rotary keeps them, and positions.
struct Turns {
  const int64_t *phases = nullptr, *axis = nullptr, *positions = nullptr;
  int64_t pairs = 0, axes = 1;
  int interleaved = 0;
  double magnitude = 1.0;
};
bool turns_ok(PyObject* positions, PyObject* const* a, int64_t tokens, int64_t dim, c10::Device d, Turns& r) {
  const at::Tensor *phases = plain(a[0]), *axis = a[1] == Py_None ? nullptr : plain(a[1]);
  const at::Tensor* at = positions == Py_None ? nullptr : plain(positions);
  if (!phases || (a[1] != Py_None && !axis) || (positions != Py_None && !at)) return false;
  if (!PyLong_CheckExact(a[2]) || !PyBool_Check(a[3]) || !PyFloat_CheckExact(a[4])) return false;
  r.axes = PyLong_AsLongLong(a[2]);
  r.interleaved = a[3] == Py_True;
  r.magnitude = PyFloat_AS_DOUBLE(a[4]);
  r.pairs = phases->numel();
  r.phases = indices(phases, d, -1);
  r.axis = indices(axis, d, r.pairs);
  if (!r.phases || (axis && !r.axis) || 2 * r.pairs > dim || r.axes < 1 || r.axes > 64) return false;
  if (!at) return r.axes == 1;
  if (at->scalar_type() != at::kLong || !at->is_contiguous() || at->device() != d || at->dim() < 1 || at->size(0) != tokens)
    return false;
  if (at->dim() > 2 || (at->dim() == 2 ? at->size(1) != r.axes : r.axes != 1)) return false;
  r.positions = static_cast<const int64_t*>(at->data_ptr());
  return true;
}

// rotate(q, k, positions, phases, axis, axes, interleaved, magnitude)
PyObject* rotate(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 8 || a[2] == Py_None) Py_RETURN_NONE;
  const at::Tensor *q = plain(a[0]), *k = a[1] == Py_None ? nullptr : plain(a[1]);
  if (!q || (a[1] != Py_None && !k) || q->dim() != 3 || !half(*q) || !heads_ok(q, *q) || (k && !heads_ok(k, *q)))
    Py_RETURN_NONE;
  const c10::Device d = q->device();
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2);
  Turns r;
  if (!gfx950(d.index()) || tokens == 0 || (k && k->size(0) != tokens) || !turns_ok(a[2], a + 3, tokens, dim, d, r))
    Py_RETURN_NONE;
  at::Tensor q_out, k_out;
  int status;
  {
    const NoGil nogil;
    q_out = at::empty({tokens, heads, dim}, q->options().requires_grad(false));
    if (k) k_out = at::empty({tokens, k->size(1), dim}, q->options().requires_grad(false));
    status = vflash_rotate(q->data_ptr(), q->stride(0), q->stride(1), k ? k->data_ptr() : nullptr, k ? k->stride(0) : 0,
                           k ? k->stride(1) : 0, q->scalar_type() == at::kHalf, tokens, heads, k ? k->size(1) : 0, dim,
                           reinterpret_cast<const uint64_t*>(r.phases), r.axis, r.pairs, r.interleaved, (float)r.magnitude,
                           r.positions, r.axes, q_out.data_ptr(), k ? k_out.data_ptr() : nullptr,
                           c10::hip::getCurrentHIPStream(d.index()).stream());
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  PyObject* both = PyTuple_New(2);
  if (!both) return nullptr;
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(std::move(q_out)));
  if (k) PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(std::move(k_out)));
  else PyTuple_SET_ITEM(both, 1, Py_NewRef(Py_None));
  return both;
  END_HANDLE_TH_ERRORS
}

// A paged cache (as vflash_amd.paged.PagedCache checks it), its table, lengths and the offsets of the tokens.
struct Pages {
  const at::Tensor *values, *scales = nullptr;
  const int64_t *table, *lengths, *offsets = nullptr;
  int64_t batch, width;
};
bool pages_ok(PyObject* values, PyObject* scales, PyObject* table, PyObject* lengths, PyObject* offsets,
              const at::Tensor& like, Pages& c) {
  c.values = plain(values);
  c.scales = scales == Py_None ? nullptr : plain(scales);
  const at::Tensor *t = plain(table), *l = plain(lengths), *o = offsets == Py_None ? nullptr : plain(offsets);
  if (!c.values || (scales != Py_None && !c.scales) || !t || !l || (offsets != Py_None && !o)) return false;
  const c10::Device d = like.device();
  if (c.values->dim() != 5 || c.values->device() != d || c.values->size(0) < 1 || c.values->size(4) != like.size(2))
    return false;
  if (!c.scales && c.values->scalar_type() != like.scalar_type()) return false;
  if (t->scalar_type() != at::kLong || t->dim() != 2 || t->size(0) < 1 || t->size(1) < 1 || !t->is_contiguous() || t->device() != d)
    return false;
  c.batch = t->size(0);
  c.width = t->size(1);
  c.table = static_cast<const int64_t*>(t->data_ptr());
  c.lengths = indices(l, d, c.batch);
  c.offsets = indices(o, d, c.batch + 1);
  return c.lengths && (!o || c.offsets) && (o || like.size(0) == c.batch) && gfx950(d.index());
}

// paged_append(q, k, v, values, scales, table, lengths, q_offsets, positions, phases, axis, axes, interleaved,
// magnitude): q rotated; without q, True.
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 14) Py_RETURN_NONE;
  const at::Tensor *q = a[0] == Py_None ? nullptr : plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
  if ((a[0] != Py_None && !q) || !k || !v || k->dim() != 3 || !half(*k) || !heads_ok(k, *k) || !heads_ok(v, *k) ||
      v->sizes() != k->sizes() || (q && (!heads_ok(q, *k) || q->size(0) != k->size(0))))
    Py_RETURN_NONE;
  const c10::Device d = k->device();
  const int64_t tokens = k->size(0), key_heads = k->size(1), dim = k->size(2);
  Pages c;
  Turns r;
  if (tokens == 0 || !pages_ok(a[3], a[4], a[5], a[6], a[7], *k, c) || c.values->size(2) != key_heads) Py_RETURN_NONE;
  const bool turns = a[9] != Py_None;
  if (turns ? !turns_ok(a[8], a + 9, tokens, dim, d, r) : (q || a[8] != Py_None)) Py_RETURN_NONE;
  at::Tensor q_out;
  int status;
  {
    const NoGil nogil;
    if (q) q_out = at::empty({tokens, q->size(1), dim}, q->options().requires_grad(false));
    status = vflash_paged_append(
        q ? q->data_ptr() : nullptr, q ? q->stride(0) : 0, q ? q->stride(1) : 0, k->data_ptr(), k->stride(0), k->stride(1),
        v->data_ptr(), v->stride(0), v->stride(1), k->scalar_type() == at::kHalf, tokens, q ? q->size(1) : 0, key_heads, dim,
        c.offsets, reinterpret_cast<const uint64_t*>(r.phases), r.axis, r.pairs, r.interleaved, (float)r.magnitude,
        r.positions, r.axes, c.values->data_ptr(), c.scales ? static_cast<float*>(c.scales->data_ptr()) : nullptr,
        c.values->size(0), c.values->size(3), c.table, c.width, c.lengths, c.batch, q ? q_out.data_ptr() : nullptr,
        c10::hip::getCurrentHIPStream(d.index()).stream());
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  written(c.values);
  written(c.scales);
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(q_out));
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, values, scales, table, lengths, q_offsets, scale)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || (a[6] != Py_None && !PyFloat_CheckExact(a[6]))) Py_RETURN_NONE;
  const at::Tensor* q = plain(a[0]);
  if (!q || q->dim() != 3 || !half(*q) || !heads_ok(q, *q)) Py_RETURN_NONE;
  Pages c;
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2);
  if (tokens == 0 || !pages_ok(a[1], a[2], a[3], a[4], a[5], *q, c)) Py_RETURN_NONE;
  const int64_t key_heads = c.values->size(2), page = c.values->size(3);
  const int64_t bytes = vflash_paged_attention_workspace(tokens, c.batch, heads, key_heads, dim, page, c.width, c.scales != nullptr);
  if (bytes < 0) Py_RETURN_NONE;
  const double scale = a[6] == Py_None ? 1.0 / std::sqrt((double)dim) : PyFloat_AS_DOUBLE(a[6]);
  at::Tensor out;
  int status;
  {
    const NoGil nogil;
    out = at::empty({tokens, heads, dim}, q->options().requires_grad(false));
    const at::Tensor workspace = bytes ? at::empty({bytes}, q->options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
    status = vflash_paged_attention(
        q->data_ptr(), q->stride(0), q->stride(1), q->scalar_type() == at::kHalf, tokens, heads, key_heads, dim, c.offsets,
        c.values->data_ptr(), c.scales ? static_cast<const float*>(c.scales->data_ptr()) : nullptr, c.values->size(0), page,
        c.table, c.width, c.lengths, c.batch, (float)scale, out.data_ptr(), heads * dim, dim,
        bytes ? workspace.data_ptr() : nullptr, bytes, c10::hip::getCurrentHIPStream(q->device().index()).stream());
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// request_adapters(base, x, down, up, scaling, ranks, widths, index, inplace), the stacks as
// vflash_amd.adapters.RequestAdapters checks them; contiguous rows.
PyObject* request_adapters(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 9 || !PyTuple_CheckExact(a[6]) || !PyBool_Check(a[8])) Py_RETURN_NONE;
  const at::Tensor *base = plain(a[0]), *x = plain(a[1]), *down = plain(a[2]), *up = plain(a[3]);
  const at::Tensor *scaling = plain(a[4]), *ranks = plain(a[5]), *index = plain(a[7]);
  if (!base || !x || !down || !up || !scaling || !ranks || !index || !half(*base) || records(*base) || records(*x)) Py_RETURN_NONE;
  const c10::Device d = base->device();
  for (const at::Tensor* t : {x, down, up, scaling, ranks, index})
    if (t->device() != d) Py_RETURN_NONE;
  const auto type = base->scalar_type();
  if (x->scalar_type() != type || down->scalar_type() != type || down->dim() != 3 || up->dim() != 3) Py_RETURN_NONE;
  const int64_t k = down->size(2), n = up->size(1), width = up->size(2), branches = PyTuple_GET_SIZE(a[6]);
  if (x->dim() < 1 || base->dim() != x->dim() || x->size(-1) != k || base->size(-1) != n || !x->is_contiguous() ||
      !base->is_contiguous() || !aligned16(*x) || !aligned16(*base) || x->numel() == 0 || branches < 1 || branches > 3)
    Py_RETURN_NONE;
  const int64_t rows = x->numel() / k;
  if (x->sizes().slice(0, x->dim() - 1) != base->sizes().slice(0, x->dim() - 1)) Py_RETURN_NONE;
  if (index->scalar_type() != at::kLong || index->numel() != rows || !index->is_contiguous() || !gfx950(d.index())) Py_RETURN_NONE;
  int64_t widths[3];
  for (int64_t b = 0; b < branches; ++b) {
    widths[b] = PyLong_AsLongLong(PyTuple_GET_ITEM(a[6], b));
    if (PyErr_Occurred()) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
  }
  const int64_t bytes = vflash_request_adapters_workspace(rows, k, widths, branches, down->size(0), width);
  if (bytes < 0) Py_RETURN_NONE;
  at::Tensor out;
  int status;
  {
    const NoGil nogil;
    out = a[8] == Py_True ? *base : at::empty(base->sizes(), base->options().requires_grad(false));
    const at::Tensor workspace = at::empty({bytes}, base->options().dtype(at::kByte).requires_grad(false));
    status = vflash_request_adapters(base->data_ptr(), n, x->data_ptr(), k, type == at::kHalf, rows, k, widths, branches,
                                     down->data_ptr(), up->data_ptr(), static_cast<const float*>(scaling->data_ptr()),
                                     static_cast<const int32_t*>(ranks->data_ptr()), down->size(0), width,
                                     static_cast<const int64_t*>(index->data_ptr()), out.data_ptr(), n,
                                     workspace.data_ptr(), bytes, c10::hip::getCurrentHIPStream(d.index()).stream());
  }
  if (status != VFLASH_OK) Py_RETURN_NONE;
  if (a[8] == Py_True) {
    written(base);
    return Py_NewRef(a[0]);
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"w8a8_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(w8a8_linear)),
     METH_FASTCALL, nullptr},
    {"w8a8_linear_lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(w8a8_linear_lora)),
     METH_FASTCALL, nullptr},
    {"nvfp4_w16_linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(nvfp4_w16_linear)),
     METH_FASTCALL, nullptr},
    {"packed_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(packed_attention)),
     METH_FASTCALL, nullptr},
    {"rotate", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rotate)), METH_FASTCALL, nullptr},
    {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged_append)), METH_FASTCALL, nullptr},
    {"paged_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(paged_attention)), METH_FASTCALL, nullptr},
    {"request_adapters", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(request_adapters)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host(void) { return PyModule_Create(&kModule); }

// Native front end of the Python ops (oxide_paged_kv/_native, a CPython module): checks the tensors,
// allocates outputs and workspaces through torch's allocator and calls the C ABI, for
// the calls of a serving step.  ops.py calls these first; each returns
//   * the op's result,
//   * None when some argument is not of the plain form handled here (a subclass, another
//     dtype or layout, a keyword's other forms): ops.py's general code then runs and
//     raises or handles it,
//   * False when the library recorded an error (ops.py raises it).
//
// Why: a step of a small batch is bound by these calls.  Through ctypes a decode call
// spent 7 of its 13.8 us on attribute reads, argument conversion and torch's stream
// object, around 4.5 us of launches; a layer's three calls 33 us for 16 us of kernels.
//
// The library's entry points are bound by address (bind), so that the functions called
// are those of the library _lib.py loaded.  The GIL is released around library calls.
#include <Python.h>

#include <ATen/Functions.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <initializer_list>

#include "oxide_paged_kv.h"

namespace {

decltype(&paged_decode_attention) g_decode = nullptr;
decltype(&paged_decode_attention_append) g_decode_append = nullptr;
decltype(&paged_decode_attention_workspace_size) g_decode_ws = nullptr;
decltype(&paged_prefill_attention_workspace) g_prefill_paged = nullptr;
decltype(&varlen_prefill_attention_workspace) g_prefill_varlen = nullptr;
decltype(&prefill_attention_workspace_size) g_prefill_ws = nullptr;
decltype(&qk_norm_rope_and_cache) g_prologue = nullptr;
decltype(&build_decode_metadata_device) g_metadata = nullptr;
decltype(&qk_norm_mrope_and_cache) g_mrope = nullptr;
decltype(&build_step_metadata_device) g_step_metadata = nullptr;
decltype(&linear_attention_decode) g_linear_decode = nullptr;
decltype(&linear_attention_prefill) g_linear_prefill = nullptr;
decltype(&linear_attention_prefill_workspace_size) g_linear_ws = nullptr;
decltype(&oxide_last_error) g_last_error = nullptr;

// A plain torch tensor on the device, contiguous.
const at::Tensor* device_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() ? &t : nullptr;
}
bool bits32(const at::Tensor& t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32; }
int dtype_code(const at::Tensor& t) {
  return t.scalar_type() == at::kHalf ? OXIDE_DTYPE_F16 : t.scalar_type() == at::kBFloat16 ? OXIDE_DTYPE_BF16 : -1;
}
void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
bool as_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0;
}
bool as_double(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}
// window_left: None = -1, else an int of 32 bits.
bool as_window(PyObject* o, int32_t* v) {
  int64_t x = -1;
  if (o != Py_None && (!as_int(o, &x) || x < INT32_MIN || x > INT32_MAX)) return false;
  *v = static_cast<int32_t>(x);
  return true;
}
// An optional device tensor: false when it is neither None nor one.
bool optional_tensor(PyObject* o, const at::Tensor** t) {
  *t = nullptr;
  return o == Py_None || (*t = device_tensor(o)) != nullptr;
}
void* data(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

PyObject* result(at::Tensor t) {
  if (g_last_error() != OXIDE_OK) Py_RETURN_FALSE;
  return THPVariable_Wrap(std::move(t));
}
at::Tensor bytes_like(const at::Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// decode(q, k_cache, v_cache, cu_seqlens_k, block_table, max_seqlen_k, softmax_scale,
//        window_left, page_block_size, out, workspace, append)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || !g_decode) Py_RETURN_NONE;
  const at::Tensor *q = device_tensor(a[0]), *k = device_tensor(a[1]), *v = device_tensor(a[2]),
                   *cu = device_tensor(a[3]), *table = device_tensor(a[4]), *out = nullptr, *ws = nullptr;
  int64_t max_k = 0, page = 0;
  double scale = 0;
  int32_t window = -1;
  if (!q || !k || !v || !cu || !table || !as_int(a[5], &max_k) || !as_double(a[6], &scale) ||
      !as_window(a[7], &window) || !as_int(a[8], &page) || !optional_tensor(a[9], &out) ||
      !optional_tensor(a[10], &ws))
    Py_RETURN_NONE;
  const int code = dtype_code(*q);
  if (code < 0 || q->dim() != 3 || k->dim() != 4 || k->sizes() != v->sizes() || k->size(3) != q->size(2) ||
      k->size(1) != page || table->dim() != 2 || table->scalar_type() != at::kInt || !bits32(*cu) ||
      k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type())
    Py_RETURN_NONE;
  const int64_t B = q->size(0), Hq = q->size(1), D = q->size(2), NB = k->size(0), Hkv = k->size(2);
  const at::Tensor *key = nullptr, *value = nullptr, *slots = nullptr;
  if (a[11] != Py_None) {
    if (!PyTuple_CheckExact(a[11]) || PyTuple_GET_SIZE(a[11]) != 3) Py_RETURN_NONE;
    key = device_tensor(PyTuple_GET_ITEM(a[11], 0));
    value = device_tensor(PyTuple_GET_ITEM(a[11], 1));
    slots = device_tensor(PyTuple_GET_ITEM(a[11], 2));
    if (!key || !value || !slots || key->sizes() != at::IntArrayRef({B, Hkv, D}) || value->sizes() != key->sizes() ||
        slots->scalar_type() != at::kLong)
      Py_RETURN_NONE;
  }
  at::Tensor o = out ? *out : at::empty_like(*q);
  const int64_t need = static_cast<int64_t>(g_decode_ws(B, Hq, Hkv, D, max_k));
  at::Tensor w = ws && static_cast<int64_t>(ws->nbytes()) >= need ? *ws : bytes_like(*q, need > 0 ? need : 1);
  void* s = stream_of(*q);
  void *po = o.data_ptr(), *pq = q->data_ptr(), *pk = k->data_ptr(), *pv = v->data_ptr(), *pw = w.data_ptr();
  const uint32_t* pc = static_cast<const uint32_t*>(cu->data_ptr());
  const int32_t* pt = static_cast<const int32_t*>(table->data_ptr());
  const int64_t width = table->size(1);
  const size_t wbytes = w.nbytes();
  void *pkey = data(key), *pvalue = data(value);
  const int64_t* pslots = static_cast<const int64_t*>(data(slots));
  Py_BEGIN_ALLOW_THREADS;
  if (key)
    g_decode_append(po, pq, pkey, pvalue, pslots, pk, pv, pc, pt, width, NB, B, Hq, Hkv, D, page, max_k, window,
                    static_cast<float>(scale), pw, wbytes, code, s);
  else
    g_decode(po, pq, pk, pv, pc, pt, width, NB, B, Hq, Hkv, D, page, max_k, window, static_cast<float>(scale), pw,
             wbytes, code, s);
  Py_END_ALLOW_THREADS;
  return result(std::move(o));
  END_HANDLE_TH_ERRORS
}

// prefill(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale,
//         block_table, window_left, out)
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !g_prefill_paged) Py_RETURN_NONE;
  const at::Tensor *q = device_tensor(a[0]), *k = device_tensor(a[1]), *v = device_tensor(a[2]),
                   *cq = device_tensor(a[3]), *ck = device_tensor(a[4]), *table = nullptr, *out = nullptr;
  int64_t max_q = 0, max_k = 0;
  double scale = 0;
  int32_t window = -1;
  if (!q || !k || !v || !cq || !ck || !as_int(a[5], &max_q) || !as_int(a[6], &max_k) || !as_double(a[7], &scale) ||
      !optional_tensor(a[8], &table) || !as_window(a[9], &window) || !optional_tensor(a[10], &out))
    Py_RETURN_NONE;
  const int code = dtype_code(*q);
  const int64_t kd = table ? 4 : 3;
  if (code < 0 || q->dim() != 3 || k->dim() != kd || k->sizes() != v->sizes() || k->size(kd - 1) != q->size(2) ||
      !bits32(*cq) || !bits32(*ck) || cq->dim() != 1 || cq->numel() < 1 || ck->sizes() != cq->sizes() ||
      k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
      (table && (table->dim() != 2 || table->scalar_type() != at::kInt)))
    Py_RETURN_NONE;
  const int64_t B = cq->size(0) - 1, Hq = q->size(1), D = q->size(2), Hkv = k->size(kd - 2);
  at::Tensor o = out ? *out : at::empty_like(*q);
  size_t need = g_prefill_ws(B, Hq, Hkv, D, max_q, max_k, window);
  at::Tensor w;
  try {
    if (need > 0) w = bytes_like(*q, static_cast<int64_t>(need));
  } catch (const c10::OutOfMemoryError&) {  // it attends without one
    need = 0;
  }
  void* s = stream_of(*q);
  void *po = o.data_ptr(), *pq = q->data_ptr(), *pk = k->data_ptr(), *pv = v->data_ptr();
  void* pw = need > 0 ? w.data_ptr() : nullptr;
  const uint32_t* pcq = static_cast<const uint32_t*>(cq->data_ptr());
  const uint32_t* pck = static_cast<const uint32_t*>(ck->data_ptr());
  const int32_t* pt = static_cast<const int32_t*>(data(table));
  const int64_t width = table ? table->size(1) : 0, rows = k->size(0), page = table ? k->size(1) : 1;
  Py_BEGIN_ALLOW_THREADS;
  if (table)
    g_prefill_paged(po, pq, pk, pv, pcq, pck, pt, width, rows, B, Hq, Hkv, D, page, max_q, max_k, window,
                    static_cast<float>(scale), pw, need, code, s);
  else
    g_prefill_varlen(po, pq, pk, pv, pcq, pck, rows, B, Hq, Hkv, D, max_q, max_k, window, static_cast<float>(scale),
                     pw, need, code, s);
  Py_END_ALLOW_THREADS;
  return result(std::move(o));
  END_HANDLE_TH_ERRORS
}

// prologue(qkv, num_heads, num_kv_heads, q_norm_weight, k_norm_weight, eps, cos_sin_cache,
//          positions, key_cache, value_cache, slot_mapping, q_out)
PyObject* prologue(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12 || !g_prologue) Py_RETURN_NONE;
  const at::Tensor *qkv = device_tensor(a[0]), *qw = nullptr, *kw = nullptr, *rope = device_tensor(a[6]),
                   *pos = device_tensor(a[7]), *kc = nullptr, *vc = nullptr, *slots = nullptr, *out = nullptr;
  int64_t Hq = 0, Hkv = 0;
  double eps = 0;
  if (!qkv || !rope || !pos || !as_int(a[1], &Hq) || !as_int(a[2], &Hkv) || !optional_tensor(a[3], &qw) ||
      !optional_tensor(a[4], &kw) || !as_double(a[5], &eps) || !optional_tensor(a[8], &kc) ||
      !optional_tensor(a[9], &vc) || !optional_tensor(a[10], &slots) || !optional_tensor(a[11], &out))
    Py_RETURN_NONE;
  const int code = dtype_code(*qkv);
  if (code < 0 || qkv->dim() != 2 || qkv->stride(1) != 1 || rope->dim() != 2 || rope->scalar_type() != at::kFloat ||
      pos->scalar_type() != at::kInt || (slots && slots->scalar_type() != at::kLong) || Hq < 0 || Hkv < 0)
    Py_RETURN_NONE;
  const int64_t T = qkv->size(0), D = rope->size(1);
  if (out && (out->sizes() != at::IntArrayRef({T, Hq, D}) || out->scalar_type() != qkv->scalar_type() ||
              out->device() != qkv->device()))
    Py_RETURN_NONE;
  at::Tensor o = out ? *out : at::empty({T, Hq, D}, qkv->options());
  void* s = stream_of(*qkv);
  void *po = o.data_ptr(), *px = qkv->data_ptr(), *pqw = data(qw), *pkw = data(kw), *pkc = data(kc), *pvc = data(vc);
  const float* pr = static_cast<const float*>(rope->data_ptr());
  const int32_t* pp = static_cast<const int32_t*>(pos->data_ptr());
  const int64_t* ps = static_cast<const int64_t*>(data(slots));
  const int64_t stride = qkv->stride(0), max_position = rope->size(0);
  Py_BEGIN_ALLOW_THREADS;
  g_prologue(po, nullptr, px, stride, pqw, pkw, eps, pr, max_position, pp, pkc, pvc, ps, T, Hq, Hkv, D, code, s);
  Py_END_ALLOW_THREADS;
  return result(std::move(o));
  END_HANDLE_TH_ERRORS
}

// metadata(context_lens, block_table, block_size) -> (cu_seqlens_k, slot_mapping)
PyObject* metadata(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3 || !g_metadata) Py_RETURN_NONE;
  const at::Tensor *lens = device_tensor(a[0]), *table = device_tensor(a[1]);
  int64_t page = 0;
  if (!lens || !table || !as_int(a[2], &page) || !bits32(*lens) || lens->dim() != 1 || lens->numel() < 1 ||
      table->dim() != 2 || table->numel() < 1 || table->scalar_type() != at::kInt)
    Py_RETURN_NONE;
  const int64_t B = lens->size(0), width = table->size(1);
  at::Tensor cu = at::empty({B + 1}, lens->options().dtype(at::kInt));
  at::Tensor slots = at::empty({B}, lens->options().dtype(at::kLong));
  void* s = stream_of(*lens);
  const uint32_t* pl = static_cast<const uint32_t*>(lens->data_ptr());
  const int32_t* pt = static_cast<const int32_t*>(table->data_ptr());
  uint32_t* pc = static_cast<uint32_t*>(cu.data_ptr());
  int64_t* ps = static_cast<int64_t*>(slots.data_ptr());
  Py_BEGIN_ALLOW_THREADS;
  g_metadata(pl, pt, width, B, page, pc, ps, s);
  Py_END_ALLOW_THREADS;
  if (g_last_error() != OXIDE_OK) Py_RETURN_FALSE;
  PyObject* c = THPVariable_Wrap(std::move(cu));
  PyObject* m = THPVariable_Wrap(std::move(slots));
  PyObject* both = c && m ? PyTuple_Pack(2, c, m) : nullptr;
  Py_XDECREF(c);
  Py_XDECREF(m);
  return both;
  END_HANDLE_TH_ERRORS
}

bool same_device(const at::Tensor& t, std::initializer_list<const at::Tensor*> others) {
  for (const at::Tensor* o : others)
    if (o && o->device() != t.device()) return false;
  return true;
}
// A plain torch tensor [T, H, D] on the device whose rows are contiguous, any row stride.
const at::Tensor* rows_tensor(PyObject* o, int64_t* stride) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.dim() != 3) return nullptr;
  const int64_t T = t.size(0), H = t.size(1), D = t.size(2);
  if ((D > 1 && t.stride(2) != 1) || (H > 1 && t.stride(1) != D)) return nullptr;
  *stride = T > 1 ? t.stride(0) : H * D;
  return &t;
}

// A tensor of `type` and `sizes` at a byte offset of a buffer, sharing its storage: an
// allocation (or a view through the dispatcher) costs 0.6 us on the host, this 0.1.
at::Tensor part_of(const at::Tensor& buffer, int64_t offset, at::ScalarType type, at::IntArrayRef sizes) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(),
                                                          c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  t.unsafeGetTensorImpl()->set_storage_offset(offset / static_cast<int64_t>(c10::elementSize(type)));
  return t;
}

// step_metadata(context_lens, query_lens, block_table, free_blocks, num_tokens, block_size,
//               position_offsets, num_axes)
//   -> (cu_seqlens_q, cu_seqlens_k, slot_mapping, positions, cu_new_blocks)
PyObject* step_metadata(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !g_step_metadata) Py_RETURN_NONE;
  const at::Tensor *ctx = device_tensor(a[0]), *query = device_tensor(a[1]), *table = device_tensor(a[2]),
                   *free_list = nullptr, *offsets = nullptr;
  int64_t rows = 0, page = 0, axes = 0;
  if (!ctx || !query || !table || !optional_tensor(a[3], &free_list) || !as_int(a[4], &rows) || !as_int(a[5], &page) ||
      !optional_tensor(a[6], &offsets) || (a[7] != Py_None && (!as_int(a[7], &axes) || axes < 1 || axes > 4)))
    Py_RETURN_NONE;
  if (!bits32(*ctx) || !bits32(*query) || ctx->dim() != 1 || query->sizes() != ctx->sizes() || table->dim() != 2 ||
      table->size(0) != ctx->size(0) || table->scalar_type() != at::kInt || rows < 0 ||
      (free_list && (free_list->scalar_type() != at::kInt || free_list->dim() != 1)) ||
      (offsets && (offsets->scalar_type() != at::kInt || offsets->sizes() != ctx->sizes())) ||
      !same_device(*ctx, {query, table, free_list, offsets}))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(ctx->device());
  const int64_t B = ctx->size(0), width = table->size(1), free_n = free_list ? free_list->size(0) : 0;
  // One allocation: slots, positions and the three prefix sums, at multiples of 256 bytes.
  auto up = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
  const int64_t at_pos = up(rows * 8), at_cu = at_pos + up(rows * 4 * (axes ? axes : 1)), cu_bytes = up((B + 1) * 4);
  const at::Tensor buffer = bytes_like(*ctx, at_cu + 3 * cu_bytes);
  at::Tensor slots = part_of(buffer, 0, at::kLong, {rows});
  at::Tensor pos = axes ? part_of(buffer, at_pos, at::kInt, {axes, rows}) : part_of(buffer, at_pos, at::kInt, {rows});
  at::Tensor cu_q = part_of(buffer, at_cu, at::kInt, {B + 1}), cu_k = part_of(buffer, at_cu + cu_bytes, at::kInt, {B + 1}),
             cu_new = part_of(buffer, at_cu + 2 * cu_bytes, at::kInt, {B + 1});
  void* s = stream_of(*ctx);
  const uint32_t* pc = static_cast<const uint32_t*>(ctx->data_ptr());
  const uint32_t* pq = static_cast<const uint32_t*>(query->data_ptr());
  const int32_t *po = static_cast<const int32_t*>(data(offsets)), *pf = static_cast<const int32_t*>(data(free_list));
  int32_t *pt = static_cast<int32_t*>(table->data_ptr()), *pp = static_cast<int32_t*>(pos.data_ptr());
  uint32_t *pcq = static_cast<uint32_t*>(cu_q.data_ptr()), *pck = static_cast<uint32_t*>(cu_k.data_ptr()),
           *pcn = static_cast<uint32_t*>(cu_new.data_ptr());
  int64_t* ps = static_cast<int64_t*>(slots.data_ptr());
  Py_BEGIN_ALLOW_THREADS;
  g_step_metadata(pc, pq, po, pt, width, pf, free_n, B, page, rows, axes ? axes : 1, pcq, pck, pcn, ps, pp, s);
  Py_END_ALLOW_THREADS;
  if (g_last_error() != OXIDE_OK) Py_RETURN_FALSE;
  PyObject* r = PyTuple_New(5);
  if (!r) return nullptr;
  at::Tensor* made[] = {&cu_q, &cu_k, &slots, &pos, &cu_new};
  for (int i = 0; i < 5; ++i) {
    PyObject* o = THPVariable_Wrap(std::move(*made[i]));
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, o);
  }
  return r;
  END_HANDLE_TH_ERRORS
}

// mrope(qkv, num_heads, num_kv_heads, q_norm_weight, k_norm_weight, eps, cos_sin_cache, positions,
//       sections, key_cache, value_cache, slot_mapping, interleaved, q_out)
PyObject* mrope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14 || !g_mrope) Py_RETURN_NONE;
  const at::Tensor *qkv = device_tensor(a[0]), *qw = nullptr, *kw = nullptr, *rope = device_tensor(a[6]),
                   *pos = device_tensor(a[7]), *kc = nullptr, *vc = nullptr, *slots = nullptr, *out = nullptr;
  int64_t Hq = 0, Hkv = 0;
  double eps = 0;
  if (!qkv || !rope || !pos || !as_int(a[1], &Hq) || !as_int(a[2], &Hkv) || !optional_tensor(a[3], &qw) ||
      !optional_tensor(a[4], &kw) || !as_double(a[5], &eps) || !PyTuple_CheckExact(a[8]) ||
      !optional_tensor(a[9], &kc) || !optional_tensor(a[10], &vc) || !optional_tensor(a[11], &slots) ||
      !PyBool_Check(a[12]) || !optional_tensor(a[13], &out))
    Py_RETURN_NONE;
  const int64_t axes = PyTuple_GET_SIZE(a[8]);
  int32_t sections[4] = {0, 0, 0, 0};
  if (axes < 1 || axes > 4) Py_RETURN_NONE;
  for (int64_t i = 0; i < axes; ++i) {
    int64_t x = 0;
    if (!as_int(PyTuple_GET_ITEM(a[8], i), &x) || x < 0 || x > INT32_MAX) Py_RETURN_NONE;
    sections[i] = static_cast<int32_t>(x);
  }
  const int code = dtype_code(*qkv);
  if (code < 0 || qkv->dim() != 2 || rope->dim() != 2 || rope->scalar_type() != at::kFloat || Hq < 1 || Hkv < 1 ||
      Hq > 4096 || Hkv > 4096)
    Py_RETURN_NONE;
  const int64_t T = qkv->size(0), D = rope->size(1);
  auto like_qkv = [&](const at::Tensor* t, at::IntArrayRef sizes) {
    return t->sizes() == sizes && t->scalar_type() == qkv->scalar_type();
  };
  if (qkv->size(1) < (Hq + 2 * Hkv) * D || pos->scalar_type() != at::kInt || pos->sizes() != at::IntArrayRef({axes, T}) ||
      (qw && !like_qkv(qw, {D})) || (kw && !like_qkv(kw, {D})) || (out && !like_qkv(out, {T, Hq, D})) ||
      !same_device(*qkv, {qw, kw, rope, pos, kc, vc, slots, out}))
    Py_RETURN_NONE;
  if (slots ? !kc || !vc || kc->dim() != 4 || kc->sizes() != vc->sizes() || kc->size(2) != Hkv || kc->size(3) != D ||
                  kc->scalar_type() != qkv->scalar_type() || vc->scalar_type() != qkv->scalar_type() ||
                  slots->scalar_type() != at::kLong || slots->sizes() != at::IntArrayRef({T})
            : kc || vc)
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(qkv->device());
  at::Tensor o = out ? *out : at::empty({T, Hq, D}, qkv->options());
  void* s = stream_of(*qkv);
  void *po = o.data_ptr(), *px = qkv->data_ptr(), *pqw = data(qw), *pkw = data(kw), *pkc = data(kc), *pvc = data(vc);
  const float* pr = static_cast<const float*>(rope->data_ptr());
  const int32_t* pp = static_cast<const int32_t*>(pos->data_ptr());
  const int64_t* ps = static_cast<const int64_t*>(data(slots));
  const int64_t stride = qkv->size(1), max_position = rope->size(0), rows = slots ? kc->size(0) * kc->size(1) : 0;
  const int dealt = a[12] == Py_True;
  Py_BEGIN_ALLOW_THREADS;
  g_mrope(po, nullptr, px, stride, pqw, pkw, eps, pr, max_position, pp, axes, sections, dealt, pkc, pvc, rows, ps, T,
          Hq, Hkv, D, code, s);
  Py_END_ALLOW_THREADS;
  return result(std::move(o));
  END_HANDLE_TH_ERRORS
}

// The tensors of a linear attention call, checked as ops._check_linear does.
struct Linear {
  const at::Tensor *q, *k, *v, *decay, *state, *slots, *out;
  int64_t sq, sk, sv, T, Hq, Hkv, D;
  int code;
};
bool as_linear(PyObject* const* a, PyObject* out, Linear* x) {
  x->q = rows_tensor(a[0], &x->sq);
  x->k = rows_tensor(a[1], &x->sk);
  x->v = rows_tensor(a[2], &x->sv);
  x->decay = device_tensor(a[3]);
  x->state = device_tensor(a[4]);
  x->slots = device_tensor(a[5]);
  if (!x->q || !x->k || !x->v || !x->decay || !x->state || !x->slots || !optional_tensor(out, &x->out)) return false;
  x->T = x->q->size(0), x->Hq = x->q->size(1), x->D = x->q->size(2), x->Hkv = x->k->size(1);
  x->code = dtype_code(*x->q);
  return x->code >= 0 && x->k->size(0) == x->T && x->k->size(2) == x->D && x->v->sizes() == x->k->sizes() &&
         x->Hkv > 0 && x->Hq % x->Hkv == 0 && x->k->scalar_type() == x->q->scalar_type() &&
         x->v->scalar_type() == x->q->scalar_type() && x->decay->scalar_type() == at::kFloat &&
         x->decay->sizes() == at::IntArrayRef({x->Hkv}) && x->state->scalar_type() == at::kFloat &&
         x->state->dim() == 4 && x->state->size(1) == x->Hkv && x->state->size(2) == x->D &&
         x->state->size(3) == x->D && x->slots->scalar_type() == at::kInt && x->slots->dim() == 1 &&
         (!x->out || (x->out->sizes() == x->q->sizes() && x->out->scalar_type() == x->q->scalar_type())) &&
         same_device(*x->q, {x->k, x->v, x->decay, x->state, x->slots, x->out});
}

// linear_decode(q, k, v, log_decay, state, state_slots, scale, out)
PyObject* linear_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Linear x;
  double scale = 0;
  if (n != 8 || !g_linear_decode || !as_double(a[6], &scale) || !as_linear(a, a[7], &x) || x.slots->size(0) != x.T)
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(x.q->device());
  at::Tensor o = x.out ? *x.out : at::empty({x.T, x.Hq, x.D}, x.q->options());
  void* s = stream_of(*x.q);
  void *po = o.data_ptr(), *pq = x.q->data_ptr(), *pk = x.k->data_ptr(), *pv = x.v->data_ptr();
  const float* pd = static_cast<const float*>(x.decay->data_ptr());
  float* pst = static_cast<float*>(x.state->data_ptr());
  const int32_t* psl = static_cast<const int32_t*>(x.slots->data_ptr());
  const int64_t num_slots = x.state->size(0);
  Py_BEGIN_ALLOW_THREADS;
  g_linear_decode(po, pq, pk, pv, x.sq, x.sk, x.sv, pd, pst, psl, num_slots, x.T, x.Hq, x.Hkv, x.D,
                  static_cast<float>(scale), x.code, s);
  Py_END_ALLOW_THREADS;
  return result(std::move(o));
  END_HANDLE_TH_ERRORS
}

// linear_prefill(q, k, v, log_decay, state, state_slots, cu_seqlens_q, max_seqlen_q, scale,
//                context_lens, out, workspace)
PyObject* linear_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Linear x;
  double scale = 0;
  int64_t max_q = 0;
  const at::Tensor *cu = nullptr, *ctx = nullptr, *ws = nullptr;
  if (n != 12 || !g_linear_prefill || !(cu = device_tensor(a[6])) || !as_int(a[7], &max_q) ||
      !as_double(a[8], &scale) || !optional_tensor(a[9], &ctx) || !as_linear(a, a[10], &x) ||
      !optional_tensor(a[11], &ws))
    Py_RETURN_NONE;
  const int64_t B = cu->numel() - 1;
  if (!bits32(*cu) || cu->dim() != 1 || B < 0 || x.slots->size(0) != B ||
      (ctx && (!bits32(*ctx) || ctx->sizes() != at::IntArrayRef({B}))) || !same_device(*x.q, {cu, ctx, ws}))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(x.q->device());
  at::Tensor o = x.out ? *x.out : at::empty({x.T, x.Hq, x.D}, x.q->options());
  at::Tensor w;
  if (ws) {
    w = *ws;
  } else if (const size_t need = g_linear_ws(x.T, B, x.Hq, x.Hkv, x.D, max_q)) {
    try {
      w = bytes_like(*x.q, static_cast<int64_t>(need));
    } catch (const c10::OutOfMemoryError&) {  // it works without one
    }
  }
  void* s = stream_of(*x.q);
  void *po = o.data_ptr(), *pq = x.q->data_ptr(), *pk = x.k->data_ptr(), *pv = x.v->data_ptr();
  const float* pd = static_cast<const float*>(x.decay->data_ptr());
  float* pst = static_cast<float*>(x.state->data_ptr());
  const int32_t* psl = static_cast<const int32_t*>(x.slots->data_ptr());
  const uint32_t *pcu = static_cast<const uint32_t*>(cu->data_ptr()), *pctx = static_cast<const uint32_t*>(data(ctx));
  const int64_t num_slots = x.state->size(0);
  void* pw = w.defined() ? w.data_ptr() : nullptr;
  const size_t wbytes = w.defined() ? w.nbytes() : 0;
  Py_BEGIN_ALLOW_THREADS;
  g_linear_prefill(po, pq, pk, pv, x.sq, x.sk, x.sv, pd, pst, psl, pctx, pcu, num_slots, x.T, B, x.Hq, x.Hkv, x.D,
                   max_q, static_cast<float>(scale), pw, wbytes, x.code, s);
  Py_END_ALLOW_THREADS;
  return result(std::move(o));
  END_HANDLE_TH_ERRORS
}

// bind(name, address): the library's function of that name; names not used here are
// accepted.
PyObject* bind(PyObject*, PyObject* args) {
  const char* name = nullptr;
  unsigned long long addr = 0;
  if (!PyArg_ParseTuple(args, "sK", &name, &addr)) return nullptr;
  void* p = reinterpret_cast<void*>(static_cast<uintptr_t>(addr));
#define OXIDE_BIND(var, fn) \
  if (std::strcmp(name, #fn) == 0) var = reinterpret_cast<decltype(&fn)>(p);
  OXIDE_BIND(g_decode, paged_decode_attention)
  OXIDE_BIND(g_decode_append, paged_decode_attention_append)
  OXIDE_BIND(g_decode_ws, paged_decode_attention_workspace_size)
  OXIDE_BIND(g_prefill_paged, paged_prefill_attention_workspace)
  OXIDE_BIND(g_prefill_varlen, varlen_prefill_attention_workspace)
  OXIDE_BIND(g_prefill_ws, prefill_attention_workspace_size)
  OXIDE_BIND(g_prologue, qk_norm_rope_and_cache)
  OXIDE_BIND(g_metadata, build_decode_metadata_device)
  OXIDE_BIND(g_mrope, qk_norm_mrope_and_cache)
  OXIDE_BIND(g_step_metadata, build_step_metadata_device)
  OXIDE_BIND(g_linear_decode, linear_attention_decode)
  OXIDE_BIND(g_linear_prefill, linear_attention_prefill)
  OXIDE_BIND(g_linear_ws, linear_attention_prefill_workspace_size)
  OXIDE_BIND(g_last_error, oxide_last_error)
#undef OXIDE_BIND
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef fast(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef kMethods[] = {fast<decode>("decode"),     fast<prefill>("prefill"),
                          fast<prologue>("prologue"), fast<metadata>("metadata"),
                          fast<mrope>("mrope"),       fast<step_metadata>("step_metadata"),
                          fast<linear_decode>("linear_decode"), fast<linear_prefill>("linear_prefill"),
                          {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() {
  PyObject* m = PyModule_Create(&kModule);
  // The torch whose headers it was built against; _lib.py uses it with no other.
  if (m && PyModule_AddStringConstant(m, "torch_version", OXIDE_TORCH_VERSION) < 0) Py_CLEAR(m);
  return m;
}

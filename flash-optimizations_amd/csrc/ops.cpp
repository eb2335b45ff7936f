// Argument checks and launches of the 4-bit and index operators, the tree attention and
// the slot maps, for remnant/mx4.py, index.py, tree.py and slots.py (module remnant_ops).
// Small calls are bound by the host: a launch takes 3.2 us, and the same checks in Python,
// with ctypes, took 4 to 8 more (a call of a window list 8.2 us, 6.1 here; the slot map of a step 10.0 and 6.3;
// a decode of one launch with window rows 12.4 and 6.8, of two launches 14.6 and 9.3).
// Shape and type mistakes raise ValueError before anything is launched (TypeError where a
// tensor or a number is something else altogether); work goes to the current stream of the
// tensors' device.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>

#include "remnant_mi355x.h"

namespace {

using at::Tensor;

// The C entry points of the loaded library and what is needed of Python, from setup().
struct {
  decltype(&rm_mx4_store_rows_ratio) store;
  decltype(&rm_mx4_gather_bf16) gather;
  decltype(&rm_mx4_sparse_decode_workspace) plan;
  decltype(&rm_mx4_sparse_decode_fwd) decode;
  decltype(&rm_append_slots_after) append;
  decltype(&rm_window_slots) window;
  decltype(&rm_index_store_rows) index_store;
  decltype(&rm_index_gather_bf16) index_gather;
  decltype(&rm_index_scores) scores;
  decltype(&rm_index_topk) topk;
  decltype(&rm_tree_decode_workspace) tree_plan;
  decltype(&rm_tree_decode_fwd) tree;
  PyObject* pool_type;    // LatentPool
  PyObject* get_stream;   // device index -> raw current stream
  PyObject* check;        // (status, name): raises
  PyObject* native_pages; // Native pool argument -> page tensor
  PyObject *fmt, *buffer; // attribute names
} lib;

constexpr int64_t kInt32 = (int64_t)1 << 31;
constexpr const char* kRatio = "ratio must be a positive int";

// ---- arguments ----

// A tensor whose memory holds its values in the plain way.
const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  const Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK_VALUE(t.layout() == at::kStrided && !t.is_conj() && !t.is_neg(), name,
                    " must be a strided tensor, not a conjugated or negated view");
  return t;
}
// None: no tensor.
const Tensor* maybe(PyObject* o, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, name);
}
const int32_t* i32(const Tensor* t) { return t ? (const int32_t*)t->const_data_ptr() : nullptr; }
const int32_t* i32(const Tensor& t) { return i32(&t); }
int32_t* i32_out(const Tensor& t) { return (int32_t*)t.mutable_data_ptr(); }

// An int (no bool, no other number) in [lo, hi).
int64_t integer(PyObject* o, int64_t lo, int64_t hi, const char* message) {
  int over = 0;
  const int64_t v = PyLong_CheckExact(o) ? PyLong_AsLongLongAndOverflow(o, &over) : lo - 1;
  TORCH_CHECK_VALUE(over == 0 && v >= lo && v < hi, message);
  return v;
}
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return (float)v;
}
void vector(const Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n &&
                        t.is_contiguous(),
                    name, " must be a contiguous int32 vector of ", n, " entries");
}

// Raises unless all of the tensors (null left out) live on one GPU; its index.
template <class... T>
c10::Device one_device(const Tensor& first, const T*... others) {
  const c10::Device device = first.device();
  TORCH_CHECK_VALUE(device.is_cuda(), "tensors must live on the GPU");
  TORCH_CHECK_VALUE(((!others || others->device() == device) && ...),
                    "tensors must live on the same GPU");
  return device;
}

template <class F, class... A>
void launch(c10::Device device, const char* name, F entry, A... args) {
  const c10::DeviceGuard guard(device);
  PyObject* const index = PyLong_FromLong(device.index());
  PyObject* const stream = index ? PyObject_CallOneArg(lib.get_stream, index) : nullptr;
  Py_XDECREF(index);
  if (!stream) throw python_error();
  void* const raw = PyLong_AsVoidPtr(stream);
  Py_DECREF(stream);
  if (!raw && PyErr_Occurred()) throw python_error();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = entry(args..., raw);
  Py_END_ALLOW_THREADS
  if (status == RM_OK) return;
  PyObject* const r = PyObject_CallFunction(lib.check, "is", status, name);
  Py_XDECREF(r);
  if (!r) throw python_error();
}

bool is_pool(PyObject* o) {
  if ((PyObject*)Py_TYPE(o) == lib.pool_type) return true;
  const int r = PyObject_IsInstance(o, lib.pool_type);
  if (r < 0) throw python_error();
  return r != 0;
}
// New reference to a LatentPool's attribute.
THPObjectPtr attribute(PyObject* pool, PyObject* name) {
  THPObjectPtr r(PyObject_GetAttr(pool, name));
  if (!r) throw python_error();
  return r;
}
bool has_format(PyObject* pool, const char* fmt) {
  THPObjectPtr r = attribute(pool, lib.fmt);
  return PyUnicode_Check(r.get()) && PyUnicode_CompareWithASCIIString(r.get(), fmt) == 0;
}

// The pages of a layer of a pool argument: a LatentPool or a uint8 page tensor.
struct Pages {
  Tensor buffer;
  uint8_t* at;
  int64_t pages;
};
// A record format whose pools the operators here take whole.
struct Format {
  const char* name;   // of LatentPool
  const char* title;
  int64_t page_bytes, dim;
};
constexpr Format kMx4{"mx4", "4-bit (mx4)", RM_MX4_PAGE_BYTES, RM_HEAD_DIM};
constexpr Format kIndex{"index", "index", RM_INDEX_PAGE_BYTES, RM_INDEX_DIM};
constexpr Format kNative{"native", "Native", RM_NATIVE_PAGE_BYTES, RM_HEAD_DIM};

Pages pages_of(PyObject* pool, PyObject* layer_id, const Format& f, const char* name = "pool") {
  if (THPVariable_Check(pool)) {
    const Tensor& t = tensor(pool, name);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kByte && t.dim() == 2 &&
                          t.size(1) == f.page_bytes && t.is_contiguous(),
                      name, " must be a contiguous uint8 [pages, ", f.page_bytes, "] tensor");
    return {t, (uint8_t*)t.mutable_data_ptr(), t.size(0)};
  }
  TORCH_CHECK_VALUE(is_pool(pool), name, " must be a LatentPool or a uint8 page tensor");
  TORCH_CHECK_VALUE(has_format(pool, f.name), "this operator takes a ", f.title, " pool");
  THPObjectPtr o = attribute(pool, lib.buffer);
  const Tensor& t = tensor(o.get(), "pool.buffer");
  TORCH_CHECK_VALUE(t.scalar_type() == at::kByte && t.dim() == 3 &&
                        t.size(2) == f.page_bytes && t.is_contiguous(),
                    "a pool's buffer is uint8 [layers, pages, ", f.page_bytes, "]");
  const int64_t layer =
      layer_id == Py_None ? 0 : integer(layer_id, 0, t.size(0), "layer_id out of range");
  return {t, (uint8_t*)t.mutable_data_ptr() + layer * t.stride(0), t.size(1)};
}
Pages native_pages(PyObject* pool) {
  if (!THPVariable_Check(pool) && is_pool(pool) && has_format(pool, "native")) {
    THPObjectPtr o = attribute(pool, lib.buffer);
    const Tensor& t = tensor(o.get(), "pool.buffer");
    if (t.dim() == 3 && t.size(2) == RM_NATIVE_PAGE_BYTES && t.is_contiguous())
      return {t, (uint8_t*)t.mutable_data_ptr(), t.size(1)};
  }
  THPObjectPtr o(PyObject_CallOneArg(lib.native_pages, pool));
  if (!o) throw python_error();
  const Tensor& t = tensor(o.get(), "swa_pool");
  return {t, (uint8_t*)t.mutable_data_ptr(), t.size(0)};
}

struct Table {
  const Tensor& t;
  int64_t batch, width, stride;
};
Table slot_table(PyObject* o, const char* name = "block_table") {
  const Tensor& t = tensor(o, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 2 &&
                        (t.size(1) <= 1 || t.stride(1) == 1 || t.numel() == 0),
                    name, " must be int32 [batch, max_blocks] with unit inner stride");
  const int64_t batch = t.size(0), width = t.size(1);
  TORCH_CHECK_VALUE(batch <= 1 || t.stride(0) >= width, name, " rows must not overlap");
  return {t, batch, width, std::max(t.stride(0), width)};
}

PyObject* none() { Py_RETURN_NONE; }
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// ---- operators: positional arguments in the order of the Python functions' ----

#define ARGUMENTS(n) \
  TORCH_CHECK_TYPE(count == n, "expected ", n, " arguments, not ", count)

// x, weight, eps, loc, positions, freqs_cis, pool, layer_id, ratio
template <class F>
PyObject* store_rows(PyObject* const* v, Py_ssize_t count, const Format& format, const char* name,
                     F entry) {
  HANDLE_TH_ERRORS
  ARGUMENTS(9);
  const Pages pool = pages_of(v[6], v[7], format);
  const Tensor &x = tensor(v[0], "x"), &weight = tensor(v[1], "weight"), &loc = tensor(v[3], "loc");
  TORCH_CHECK_VALUE(x.dim() == 2 && x.size(1) == format.dim && x.stride(1) == 1, "x must be [rows, ",
                    format.dim, "] with unit inner stride");
  const bool bf16 = x.scalar_type() == at::kBFloat16;
  TORCH_CHECK_VALUE(bf16 || x.scalar_type() == at::kFloat, "x must be float32 or bfloat16");
  const int64_t rows = x.size(0);
  TORCH_CHECK_VALUE(loc.scalar_type() == at::kInt && loc.dim() == 1 && loc.size(0) == rows &&
                        loc.is_contiguous(),
                    "loc must be a contiguous int32 [rows] tensor");
  TORCH_CHECK_VALUE(weight.scalar_type() == at::kFloat && weight.dim() == 1 &&
                        weight.size(0) == format.dim && weight.is_contiguous(),
                    "weight must be a contiguous float32 [", format.dim, "] tensor");
  const float eps = number(v[2]);
  const int64_t ratio = integer(v[8], 1, kInt32, kRatio);
  const Tensor* const freqs = maybe(v[5], "freqs_cis");
  const Tensor* const positions = freqs ? maybe(v[4], "positions") : nullptr;
  int64_t freq_rows = 0;
  if (freqs) {
    TORCH_CHECK_VALUE(freqs->scalar_type() == at::kComplexFloat && freqs->is_contiguous(),
                      "freqs_cis must be a contiguous complex64 tensor");
    TORCH_CHECK_VALUE(positions && positions->scalar_type() == at::kInt &&
                          positions->dim() == 1 && positions->size(0) == rows &&
                          positions->is_contiguous(),
                      "positions must be a contiguous int32 [rows] tensor when freqs_cis is given");
    freq_rows = freqs->numel() / ((RM_HEAD_DIM - RM_NOPE_DIM) / 2);
  }
  if (rows == 0 || (freqs && freq_rows == 0)) return none();
  // (one row has no distance to a next one: whatever the tensor says)
  launch(one_device(x, &weight, &loc, positions, freqs, &pool.buffer), name, entry,
         x.const_data_ptr(), bf16 ? (int)RM_BF16 : (int)RM_F32, rows > 1 ? x.stride(0) : format.dim,
         (const float*)weight.const_data_ptr(), eps, i32(loc), i32(positions),
         freqs ? (const float*)freqs->const_data_ptr() : nullptr, freq_rows, ratio, rows, pool.at,
         pool.pages);
  return none();
  END_HANDLE_TH_ERRORS
}
PyObject* store(PyObject*, PyObject* const* v, Py_ssize_t count) {
  return store_rows(v, count, kMx4, "rm_mx4_store_rows_ratio", lib.store);
}
PyObject* index_store(PyObject*, PyObject* const* v, Py_ssize_t count) {
  return store_rows(v, count, kIndex, "rm_index_store_rows", lib.index_store);
}

// pool, slots, lengths, output, layer_id -> output
template <class F>
PyObject* gather_rows(PyObject* const* v, Py_ssize_t count, const Format& format, const char* name,
                      F entry) {
  HANDLE_TH_ERRORS
  ARGUMENTS(5);
  const Pages pool = pages_of(v[0], v[4], format);
  const Tensor& slots = tensor(v[1], "slots");
  TORCH_CHECK_VALUE(slots.scalar_type() == at::kInt && slots.dim() == 2,
                    "slots must be int32 [queries, k]");
  const int64_t queries = slots.size(0), k = slots.size(1), rows = queries * k;
  const Tensor* const lengths = maybe(v[2], "lengths");
  TORCH_CHECK_VALUE(!lengths || (lengths->scalar_type() == at::kInt && lengths->dim() == 1 &&
                                 lengths->size(0) == queries),
                    "lengths must be int32 [queries]");
  Tensor output = v[3] == Py_None
                      ? at::empty({rows, format.dim}, slots.options().dtype(at::kBFloat16))
                      : tensor(v[3], "output");
  TORCH_CHECK_VALUE(output.scalar_type() == at::kBFloat16 && output.dim() == 2 &&
                        output.size(1) == format.dim && output.is_contiguous(),
                    "output must be a contiguous bfloat16 [rows, ", format.dim, "] tensor");
  TORCH_CHECK_VALUE(output.size(0) >= rows, "output has fewer rows than queries * k");
  if (rows > 0)
    launch(one_device(pool.buffer, &slots, lengths, &output), name, entry,
           (const uint8_t*)pool.at, pool.pages, i32(slots), slots.stride(0), slots.stride(1),
           i32(lengths), lengths ? lengths->stride(0) : 0, queries, k,
           (uint16_t*)output.mutable_data_ptr());
  return v[3] == Py_None ? THPVariable_Wrap(std::move(output)) : same(v[3]);
  END_HANDLE_TH_ERRORS
}
PyObject* gather(PyObject*, PyObject* const* v, Py_ssize_t count) {
  return gather_rows(v, count, kMx4, "rm_mx4_gather_bf16", lib.gather);
}
PyObject* index_gather(PyObject*, PyObject* const* v, Py_ssize_t count) {
  return gather_rows(v, count, kIndex, "rm_index_gather_bf16", lib.index_gather);
}

// q, pool, block_table, indices, seqlens, topk_length, sink, softmax_scale, out, lse,
// workspace, layer_id, swa_pool, swa_indices, swa_lengths -> (out, lse)
PyObject* decode(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  ARGUMENTS(15);
  const Pages pool = pages_of(v[1], v[11], kMx4);
  const Tensor &q = tensor(v[0], "q"), &table = tensor(v[2], "block_table"),
               &indices = tensor(v[3], "indices");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == RM_HEAD_DIM &&
                        q.scalar_type() == at::kBFloat16 && q.is_contiguous(),
                    "q must be a contiguous bfloat16 [batch, q_len, heads, 512] tensor");
  const int64_t batch = q.size(0), q_len = q.size(1), heads = q.size(2), tokens = batch * q_len;
  TORCH_CHECK_VALUE(indices.scalar_type() == at::kInt && indices.dim() == 3 &&
                        indices.size(0) == batch && indices.size(1) == q_len &&
                        indices.is_contiguous(),
                    "indices must be a contiguous int32 [batch, q_len, topk] tensor");
  const int64_t topk = indices.size(2);
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 &&
                        table.size(0) == batch && table.stride(1) == 1,
                    "block_table must be int32 [batch, max_blocks] with unit inner stride");
  const int64_t max_blocks = table.size(1);
  // a single request's table may be a broadcast view (stride 0 in dim 0)
  const int64_t bt_stride = batch > 1 ? table.stride(0) : std::max(table.stride(0), max_blocks);
  const Tensor *const seqlens = maybe(v[4], "seqlens"), *const lengths = maybe(v[5], "topk_length"),
               *const sink = maybe(v[6], "sink");
  TORCH_CHECK_VALUE(!seqlens || (seqlens->scalar_type() == at::kInt && seqlens->numel() == batch &&
                                 seqlens->is_contiguous()),
                    "seqlens must be a contiguous int32 tensor of ", batch, " entries");
  TORCH_CHECK_VALUE(!lengths || (lengths->scalar_type() == at::kInt && lengths->numel() == tokens &&
                                 lengths->is_contiguous()),
                    "topk_length must be a contiguous int32 tensor of ", tokens, " entries");
  TORCH_CHECK_VALUE(!sink || (sink->scalar_type() == at::kFloat && sink->dim() == 1 &&
                              sink->size(0) == heads && sink->is_contiguous()),
                    "sink must be a contiguous float32 [heads] tensor");
  const float scale = v[7] == Py_None ? 0.04419417382415922f : number(v[7]);  // 1 / sqrt(512)
  Tensor out = v[8] == Py_None ? at::empty(q.sizes(), q.options()) : tensor(v[8], "out");
  Tensor lse = v[9] == Py_None
                   ? at::empty({batch, q_len, heads}, q.options().dtype(at::kFloat))
                   : tensor(v[9], "lse");
  TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16 &&
                        out.is_contiguous(),
                    "out must be a contiguous bfloat16 tensor shaped like q");
  TORCH_CHECK_VALUE(lse.sizes() == q.sizes().slice(0, 3) && lse.scalar_type() == at::kFloat &&
                        lse.is_contiguous(),
                    "lse must be a contiguous float32 [batch, q_len, heads] tensor");
  Pages swa{};
  const Tensor *swa_indices = nullptr, *swa_lengths = nullptr;
  int64_t width = 0;
  if (v[12] != Py_None || v[13] != Py_None) {
    TORCH_CHECK_VALUE(v[12] != Py_None && v[13] != Py_None,
                      "swa_pool and swa_indices are given together");
    swa = native_pages(v[12]);
    swa_indices = &tensor(v[13], "swa_indices");
    swa_lengths = maybe(v[14], "swa_lengths");
    TORCH_CHECK_VALUE(swa_indices->scalar_type() == at::kInt && swa_indices->dim() == 3 &&
                          swa_indices->size(0) == batch && swa_indices->size(1) == q_len &&
                          swa_indices->is_contiguous(),
                      "swa_indices must be a contiguous int32 [batch, q_len, W] tensor");
    width = swa_indices->size(2);
    TORCH_CHECK_VALUE(width <= 512, "at most 512 window rows per token");
    TORCH_CHECK_VALUE(!swa_lengths ||
                          (swa_lengths->scalar_type() == at::kInt &&
                           swa_lengths->numel() == tokens && swa_lengths->is_contiguous()),
                      "swa_lengths must be a contiguous int32 tensor of ", tokens, " entries");
  }
  const Tensor* workspace = maybe(v[10], "workspace");
  TORCH_CHECK_VALUE(!workspace ||
                        (workspace->scalar_type() == at::kByte && workspace->is_contiguous()),
                    "workspace must be a contiguous uint8 tensor on the GPU");
  if (tokens * heads > 0) {
    size_t need = 0;
    Tensor own;
    // (sizes it refuses, the launch refuses too)
    if (lib.plan(tokens, heads, topk, width, nullptr, &need) == RM_OK && need > 0 &&
        (!workspace || (size_t)workspace->numel() < need)) {
      own = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      workspace = &own;
    }
    launch(one_device(q, &pool.buffer, &table, &indices, seqlens, lengths, sink, &out, &lse,
                      swa_indices ? &swa.buffer : nullptr, swa_indices, swa_lengths, workspace),
           "rm_mx4_sparse_decode_fwd", lib.decode, (const uint16_t*)q.const_data_ptr(), batch,
           q_len, heads, (const uint8_t*)pool.at, pool.pages, i32(table), bt_stride, max_blocks,
           i32(seqlens), i32(indices), topk, i32(lengths), (const uint8_t*)swa.at, swa.pages,
           i32(swa_indices), width, i32(swa_lengths),
           sink ? (const float*)sink->const_data_ptr() : nullptr, scale,
           (uint16_t*)out.mutable_data_ptr(), (float*)lse.mutable_data_ptr(),
           workspace ? workspace->mutable_data_ptr() : nullptr,
           workspace ? (size_t)workspace->numel() : (size_t)0);
  }
  THPObjectPtr o(v[8] == Py_None ? THPVariable_Wrap(std::move(out)) : same(v[8]));
  THPObjectPtr l(v[9] == Py_None ? THPVariable_Wrap(std::move(lse)) : same(v[9]));
  if (!o || !l) throw python_error();
  return PyTuple_Pack(2, o.get(), l.get());
  END_HANDLE_TH_ERRORS
}

// block_table, old_lengths, new_lengths, free_pages, ratio, rows, out, taken -> the five
// outputs
PyObject* append(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  ARGUMENTS(8);
  const Table table = slot_table(v[0]);
  const int64_t batch = table.batch;
  TORCH_CHECK_VALUE(batch <= RM_MAX_SLOT_BATCH, "at most ", RM_MAX_SLOT_BATCH, " requests a call");
  const int64_t ratio = integer(v[4], 1, kInt32, kRatio);
  const Tensor &before = tensor(v[1], "old_lengths"), &after = tensor(v[2], "new_lengths"),
               &free = tensor(v[3], "free_pages");
  vector(before, batch, "old_lengths");
  vector(after, batch, "new_lengths");
  TORCH_CHECK_VALUE(free.scalar_type() == at::kInt && free.dim() == 1 && free.is_contiguous(),
                    "free_pages must be a contiguous int32 vector");
  const Tensor* const taken = maybe(v[7], "taken");
  if (taken) vector(*taken, 1, "taken");
  static const char* const names[5] = {"loc", "positions", "row_starts", "seqlens", "pages_taken"};
  Tensor made[5];
  const Tensor* out[5];
  int64_t rows = -1;
  if (v[5] != Py_None || v[6] == Py_None)
    rows = integer(v[5], 0, kInt32, "rows must be an int, the capacity of the row lists");
  if (v[6] == Py_None) {
    const int64_t sizes[5] = {rows, rows, batch + 1, batch, 1};
    for (int i = 0; i < 5; ++i) {
      made[i] = at::empty({sizes[i]}, table.t.options());
      out[i] = &made[i];
    }
  } else {
    TORCH_CHECK_VALUE(PyTuple_Check(v[6]) && PyTuple_GET_SIZE(v[6]) == 5,
                      "out must be a SlotMap or five tensors");
    for (int i = 0; i < 5; ++i) out[i] = &tensor(PyTuple_GET_ITEM(v[6], i), names[i]);
    if (rows < 0) rows = out[0]->dim() == 1 ? out[0]->size(0) : 0;
    const int64_t sizes[5] = {rows, rows, batch + 1, batch, 1};
    for (int i = 0; i < 5; ++i) vector(*out[i], sizes[i], names[i]);
  }
  launch(one_device(table.t, &before, &after, &free, taken, out[0], out[1], out[2], out[3], out[4]),
         "rm_append_slots_after", lib.append, i32_out(table.t), table.stride, table.width, i32(before),
         i32(after), batch, ratio, i32(free), free.size(0), i32(taken), rows, i32_out(*out[0]),
         i32_out(*out[1]), i32_out(*out[2]), i32_out(*out[3]), i32_out(*out[4]));
  if (v[6] != Py_None) return same(v[6]);
  THPObjectPtr r(PyTuple_New(5));
  if (!r) throw python_error();
  for (int i = 0; i < 5; ++i) {
    PyObject* const t = THPVariable_Wrap(std::move(made[i]));
    if (!t) throw python_error();
    PyTuple_SET_ITEM(r.get(), i, t);
  }
  return r.release();
  END_HANDLE_TH_ERRORS
}

// block_table, lengths, q_len, window, first, out -> (slots, counts)
PyObject* window(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  ARGUMENTS(6);
  const Table table = slot_table(v[0]);
  constexpr const char* kSizes = "q_len, window and first must be non-negative ints";
  const int64_t q_len = integer(v[2], 0, kInt32, kSizes), window = integer(v[3], 0, kInt32, kSizes),
                first = integer(v[4], 0, kInt32, kSizes);
  const Tensor& lengths = tensor(v[1], "lengths");
  vector(lengths, table.batch, "lengths");
  const int64_t width = first + window, tokens = table.batch * q_len;
  Tensor slots, counts;
  if (v[5] == Py_None) {
    slots = at::empty({table.batch, q_len, width}, table.t.options());
    counts = at::empty({tokens}, table.t.options());
  } else {
    THPObjectPtr pair(PySequence_Tuple(v[5]));
    if (!pair) throw python_error();
    TORCH_CHECK_VALUE(PyTuple_GET_SIZE(pair.get()) == 2, "out must be two tensors");
    slots = tensor(PyTuple_GET_ITEM(pair.get(), 0), "slots");
    counts = tensor(PyTuple_GET_ITEM(pair.get(), 1), "counts");
    TORCH_CHECK_VALUE(slots.scalar_type() == at::kInt && slots.dim() == 3 &&
                          slots.size(0) == table.batch && slots.size(1) == q_len &&
                          slots.size(2) == width && slots.is_contiguous(),
                      "slots must be a contiguous int32 [", table.batch, ", ", q_len, ", ", width,
                      "] tensor");
    vector(counts, tokens, "counts");
  }
  if (tokens > 0)
    launch(one_device(table.t, &lengths, &slots, &counts), "rm_window_slots", lib.window,
           i32(table.t), table.stride, table.width, i32(lengths), table.batch, q_len, window, first,
           i32_out(slots), i32_out(counts));
  THPObjectPtr s(THPVariable_Wrap(std::move(slots))), c(THPVariable_Wrap(std::move(counts)));
  if (!s || !c) throw python_error();
  return PyTuple_Pack(2, s.get(), c.get());
  END_HANDLE_TH_ERRORS
}

// q, weights, pool, block_table, lengths, out, layer_id -> out
PyObject* scores(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  ARGUMENTS(7);
  const Pages pool = pages_of(v[2], v[6], kIndex);
  const Tensor &q = tensor(v[0], "q"), &weights = tensor(v[1], "weights"),
               &lengths = tensor(v[4], "lengths");
  const Table table = slot_table(v[3]);
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == RM_INDEX_DIM &&
                        q.scalar_type() == at::kBFloat16 && q.is_contiguous(),
                    "q must be a contiguous bfloat16 [batch, q_len, heads, 128] tensor");
  const int64_t batch = q.size(0), q_len = q.size(1), heads = q.size(2), tokens = batch * q_len;
  TORCH_CHECK_VALUE(heads <= RM_MAX_INDEX_HEADS, "at most ", RM_MAX_INDEX_HEADS, " heads");
  TORCH_CHECK_VALUE(weights.sizes() == q.sizes().slice(0, 3) && weights.scalar_type() == at::kFloat &&
                        weights.is_contiguous(),
                    "weights must be a contiguous float32 [batch, q_len, heads] tensor");
  TORCH_CHECK_VALUE(table.batch == batch, "block_table must have a row for each request");
  TORCH_CHECK_VALUE(lengths.scalar_type() == at::kInt && lengths.numel() == tokens &&
                        lengths.is_contiguous(),
                    "lengths must be a contiguous int32 tensor of ", tokens, " entries");
  Tensor out = v[5] == Py_None ? at::empty({batch, q_len, table.width * RM_PAGE_RECORDS},
                                           q.options().dtype(at::kFloat))
                               : tensor(v[5], "out");
  TORCH_CHECK_VALUE(out.dim() == 3 && out.size(0) == batch && out.size(1) == q_len &&
                        out.scalar_type() == at::kFloat && out.is_contiguous(),
                    "out must be a contiguous float32 [batch, q_len, records] tensor");
  if (tokens > 0 && out.size(2) > 0)
    launch(one_device(q, &weights, &pool.buffer, &table.t, &lengths, &out), "rm_index_scores",
           lib.scores, (const uint16_t*)q.const_data_ptr(), batch, q_len, heads,
           (const float*)weights.const_data_ptr(), (const uint8_t*)pool.at, pool.pages,
           i32(table.t), table.stride, table.width, i32(lengths), out.size(2),
           (float*)out.mutable_data_ptr());
  return v[5] == Py_None ? THPVariable_Wrap(std::move(out)) : same(v[5]);
  END_HANDLE_TH_ERRORS
}

// scores, lengths, k, out -> (indices, counts)
PyObject* topk(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  ARGUMENTS(4);
  const Tensor& scores = tensor(v[0], "scores");
  TORCH_CHECK_VALUE(scores.scalar_type() == at::kFloat && (scores.dim() == 2 || scores.dim() == 3),
                    "scores must be float32 [rows, records] or [batch, q_len, records]");
  const int64_t width = scores.size(-1), outer = scores.dim() == 3 ? scores.size(0) : 1,
                inner = scores.size(-2), rows = outer * inner;
  // rows at one distance from each other
  const int64_t stride = inner > 1 ? scores.stride(-2) : outer > 1 ? scores.stride(0) : width;
  TORCH_CHECK_VALUE(scores.numel() == 0 ||
                        ((width == 1 || scores.stride(-1) == 1) && (rows == 1 || stride >= width) &&
                         (outer == 1 || inner == 1 || scores.stride(0) == inner * stride)),
                    "scores must have unit inner stride and rows at one distance");
  const int64_t k = integer(v[2], 0, (int64_t)RM_MAX_INDEX_WIDTH + 1, "k must be an int of 0 to 2^20");
  TORCH_CHECK_VALUE(width <= RM_MAX_INDEX_WIDTH, "at most 2^20 records a row");
  const Tensor* const lengths = maybe(v[1], "lengths");
  TORCH_CHECK_VALUE(!lengths || (lengths->scalar_type() == at::kInt && lengths->numel() == rows &&
                                 lengths->is_contiguous()),
                    "lengths must be a contiguous int32 tensor of ", rows, " entries");
  Tensor indices, counts;
  at::DimVector shape(scores.sizes().begin(), scores.sizes().end());
  shape.back() = k;
  if (v[3] == Py_None) {
    const auto options = scores.options().dtype(at::kInt);
    indices = at::empty(shape, options);
    counts = at::empty({rows}, options);
  } else {
    THPObjectPtr pair(PySequence_Tuple(v[3]));
    if (!pair) throw python_error();
    TORCH_CHECK_VALUE(PyTuple_GET_SIZE(pair.get()) == 2, "out must be two tensors");
    indices = tensor(PyTuple_GET_ITEM(pair.get(), 0), "indices");
    counts = tensor(PyTuple_GET_ITEM(pair.get(), 1), "counts");
    TORCH_CHECK_VALUE(indices.scalar_type() == at::kInt && indices.sizes() == shape &&
                          indices.is_contiguous(),
                      "indices must be a contiguous int32 tensor shaped like scores, with ", k,
                      " entries a row");
    vector(counts, rows, "counts");
  }
  if (rows > 0)
    launch(one_device(scores, lengths, &indices, &counts), "rm_index_topk", lib.topk,
           (const float*)scores.const_data_ptr(), stride, i32(lengths), rows, width, k,
           i32_out(indices), i32_out(counts));
  THPObjectPtr i(THPVariable_Wrap(std::move(indices))), c(THPVariable_Wrap(std::move(counts)));
  if (!i || !c) throw python_error();
  return PyTuple_Pack(2, i.get(), c.get());
  END_HANDLE_TH_ERRORS
}

// q, pool, block_table, lengths, parents, window, history_pool, history_table,
// history_lengths, sink, softmax_scale, out, lse, workspace, layer_id, history_layer_id ->
// (out, lse)
PyObject* tree(PyObject*, PyObject* const* v, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  ARGUMENTS(16);
  const Pages pool = pages_of(v[1], v[14], kNative);
  const Tensor &q = tensor(v[0], "q"), &lengths = tensor(v[3], "lengths"),
               &parents = tensor(v[4], "parents");
  const Table table = slot_table(v[2]);
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == RM_HEAD_DIM &&
                        q.scalar_type() == at::kBFloat16 && q.is_contiguous(),
                    "q must be a contiguous bfloat16 [batch, nodes, heads, 512] tensor");
  const int64_t batch = q.size(0), nodes = q.size(1), heads = q.size(2);
  TORCH_CHECK_VALUE(nodes <= RM_MAX_TREE_NODES, "at most ", RM_MAX_TREE_NODES, " nodes a tree");
  TORCH_CHECK_VALUE(table.batch == batch, "block_table must have a row for each request");
  vector(lengths, batch, "lengths");
  TORCH_CHECK_VALUE(parents.scalar_type() == at::kInt && parents.dim() == 2 &&
                        parents.size(0) == batch && parents.size(1) == nodes &&
                        parents.is_contiguous(),
                    "parents must be a contiguous int32 [batch, nodes] tensor");
  const int64_t window =
      v[5] == Py_None ? 0 : integer(v[5], 1, kInt32, "window must be a positive int");
  Pages past{};
  const Tensor* past_lengths = nullptr;
  const Tensor* past_table = nullptr;
  int64_t past_blocks = 0, past_stride = 0;
  if (v[6] != Py_None || v[7] != Py_None || v[8] != Py_None) {
    TORCH_CHECK_VALUE(v[6] != Py_None && v[7] != Py_None && v[8] != Py_None,
                      "history_pool, history_table and history_lengths are given together");
    past = pages_of(v[6], v[15], kNative, "history_pool");
    const Table t = slot_table(v[7], "history_table");
    TORCH_CHECK_VALUE(t.batch == batch, "history_table must have a row for each request");
    past_lengths = &tensor(v[8], "history_lengths");
    vector(*past_lengths, batch, "history_lengths");
    past_table = &t.t;
    past_blocks = t.width;
    past_stride = t.stride;
  }
  const Tensor* const sink = maybe(v[9], "sink");
  TORCH_CHECK_VALUE(!sink || (sink->scalar_type() == at::kFloat && sink->dim() == 1 &&
                              sink->size(0) == heads && sink->is_contiguous()),
                    "sink must be a contiguous float32 [heads] tensor");
  const float scale = v[10] == Py_None ? 0.04419417382415922f : number(v[10]);  // 1 / sqrt(512)
  Tensor out = v[11] == Py_None ? at::empty(q.sizes(), q.options()) : tensor(v[11], "out");
  Tensor lse = v[12] == Py_None
                   ? at::empty({batch, nodes, heads}, q.options().dtype(at::kFloat))
                   : tensor(v[12], "lse");
  TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.scalar_type() == at::kBFloat16 &&
                        out.is_contiguous(),
                    "out must be a contiguous bfloat16 tensor shaped like q");
  TORCH_CHECK_VALUE(lse.sizes() == q.sizes().slice(0, 3) && lse.scalar_type() == at::kFloat &&
                        lse.is_contiguous(),
                    "lse must be a contiguous float32 [batch, nodes, heads] tensor");
  const Tensor* workspace = maybe(v[13], "workspace");
  TORCH_CHECK_VALUE(!workspace ||
                        (workspace->scalar_type() == at::kByte && workspace->is_contiguous()),
                    "workspace must be a contiguous uint8 tensor on the GPU");
  if (q.numel() > 0) {
    size_t need = 0;
    Tensor own;
    // (sizes it refuses, the launch refuses too)
    if (lib.tree_plan(batch, nodes, heads, table.width, window, past_blocks, nullptr, &need) == RM_OK &&
        need > 0 && (!workspace || (size_t)workspace->numel() < need)) {
      own = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
      workspace = &own;
    }
    launch(one_device(q, &pool.buffer, &table.t, &lengths, &parents,
                      past_lengths ? &past.buffer : nullptr, past_table, past_lengths, sink, &out,
                      &lse, workspace),
           "rm_tree_decode_fwd", lib.tree, (const uint16_t*)q.const_data_ptr(), batch, nodes, heads,
           (const uint8_t*)pool.at, pool.pages, i32(table.t), table.stride, table.width,
           i32(lengths), i32(parents), window, (const uint8_t*)past.at, past.pages, i32(past_table),
           past_stride, past_blocks, i32(past_lengths),
           sink ? (const float*)sink->const_data_ptr() : nullptr, scale,
           (uint16_t*)out.mutable_data_ptr(), (float*)lse.mutable_data_ptr(),
           workspace ? workspace->mutable_data_ptr() : nullptr,
           workspace ? (size_t)workspace->numel() : (size_t)0);
  }
  THPObjectPtr o(v[11] == Py_None ? THPVariable_Wrap(std::move(out)) : same(v[11]));
  THPObjectPtr s(v[12] == Py_None ? THPVariable_Wrap(std::move(lse)) : same(v[12]));
  if (!o || !s) throw python_error();
  return PyTuple_Pack(2, o.get(), s.get());
  END_HANDLE_TH_ERRORS
}

// (entry points' addresses in the order of `lib`), LatentPool, get_stream, check, native_pages
PyObject* setup(PyObject*, PyObject* args) {
  constexpr int kEntries = 12;
  PyObject *entries, *pool_type, *get_stream, *check, *pages;
  if (!PyArg_ParseTuple(args, "O!OOOO", &PyTuple_Type, &entries, &pool_type, &get_stream, &check,
                        &pages))
    return nullptr;
  void* at[kEntries];
  if (PyTuple_GET_SIZE(entries) != kEntries) {
    PyErr_SetString(PyExc_ValueError, "entry points missing");
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i) {
    at[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(entries, i));
    if (!at[i] && PyErr_Occurred()) return nullptr;
  }
  lib.store = (decltype(lib.store))at[0];
  lib.gather = (decltype(lib.gather))at[1];
  lib.plan = (decltype(lib.plan))at[2];
  lib.decode = (decltype(lib.decode))at[3];
  lib.append = (decltype(lib.append))at[4];
  lib.window = (decltype(lib.window))at[5];
  lib.index_store = (decltype(lib.index_store))at[6];
  lib.index_gather = (decltype(lib.index_gather))at[7];
  lib.scores = (decltype(lib.scores))at[8];
  lib.topk = (decltype(lib.topk))at[9];
  lib.tree_plan = (decltype(lib.tree_plan))at[10];
  lib.tree = (decltype(lib.tree))at[11];
  lib.pool_type = same(pool_type);
  lib.get_stream = same(get_stream);
  lib.check = same(check);
  lib.native_pages = same(pages);
  lib.fmt = PyUnicode_InternFromString("fmt");
  lib.buffer = PyUnicode_InternFromString("buffer");
  return none();
}

#define FAST(f) \
  { #f, (PyCFunction)(void*)f, METH_FASTCALL, nullptr }
PyMethodDef methods[] = {FAST(store),        FAST(gather), FAST(decode), FAST(append),
                         FAST(window),       FAST(index_store),
                         FAST(index_gather), FAST(scores), FAST(topk),   FAST(tree),
                         {"setup", setup, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "remnant_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_remnant_ops() { return PyModule_Create(&module); }

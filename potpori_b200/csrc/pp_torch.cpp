// potpori_b200._paged: the paged operators on torch tensors. Checks of types, shapes, strides and
// devices, the outputs and work buffers from torch's allocator, the current stream, and one call of
// the C ABI each (include/potpori_b200.h). A small call's kernel runs for 3 to 4 us; checked and called
// from Python the same call cost its caller 11 to 18 us, from here about half.
// potpori_b200/paged.py has the classes that users see.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <optional>
#include <string>

#include "../../include/potpori_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void raise(int status, const std::string& message) {
  static py::handle error = py::object(py::module_::import("potpori_b200._lib").attr("PPError")).release();
  py::object e = error(status, message);
  PyErr_SetObject(error.ptr(), e.ptr());
  throw py::error_already_set();
}
[[noreturn]] void refuse(const std::string& message) { raise(PP_E_INVALID, message); }

void check(pp_status st, const char* what) {
  if (st == PP_OK) return;
  char buf[1024];
  buf[0] = 0;
  pp_last_error(nullptr, buf, sizeof buf);
  raise(st, std::string(what) + ": " + buf);
}

uint32_t dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PP_F32;
    case at::kBFloat16: return PP_BF16;
    case at::kHalf: return PP_F16;
    default: return 3;
  }
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

// Address of a contiguous tensor of this type and shape on device `index`.
void* pointer(const char* name, const Tensor& t, int64_t index, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || !t.is_cuda() || t.get_device() != index || t.sizes() != shape || !t.is_contiguous())
    refuse(std::string(name) + ": a contiguous " + c10::toString(type) + " tensor of shape " + shape_text(shape) +
           " on cuda:" + std::to_string(index) + " expected, got " + c10::toString(t.scalar_type()) + " " +
           shape_text(t.sizes()) + " on " + t.device().str());
  return t.data_ptr();
}
void* pointer(const char* name, const OptTensor& t, int64_t index, at::ScalarType type, at::IntArrayRef shape) {
  return t ? pointer(name, *t, index, type, shape) : nullptr;
}

void* stream_of(int64_t index) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream(); }

at::TensorOptions on(int64_t index, at::ScalarType type) {
  return at::TensorOptions().device(at::Device(at::kCUDA, (c10::DeviceIndex)index)).dtype(type);
}

struct Batch {
  Tensor page_table, lengths, cu_rows;
  pp_paged_batch c = {};
  int64_t index = -1;
  bool bounded;

  Batch(Tensor table, Tensor len, Tensor cu, int64_t max_rows, std::optional<int64_t> max_length)
      : page_table(std::move(table)), lengths(std::move(len)), cu_rows(std::move(cu)), bounded(max_length.has_value()) {
    if (page_table.dim() != 2 || page_table.size(1) == 0) refuse("page_table: [batch, pages] expected");
    if (!page_table.is_cuda()) refuse("the batch's tensors must be on a CUDA device");
    if (max_rows < 0 || max_rows > INT32_MAX || (bounded && (*max_length < 0 || *max_length > INT32_MAX)))
      refuse("max_rows and max_length must be within 0..2^31 - 1");
    index = page_table.get_device();
    const int64_t n = page_table.size(0), stride = page_table.size(1);
    if (n > INT32_MAX || stride > INT32_MAX) refuse("page_table too large");
    c.batch = (uint32_t)n;
    c.max_rows = (uint32_t)max_rows;
    c.max_len = bounded ? (uint32_t)*max_length : 0;
    c.table_stride = (uint32_t)stride;
    c.cu_rows = (const int32_t*)pointer("cu_rows", cu_rows, index, at::kInt, {n + 1});
    c.kv_len = (const int32_t*)pointer("lengths", lengths, index, at::kInt, {n});
    c.page_table = (const int32_t*)pointer("page_table", page_table, index, at::kInt, {n, stride});
  }
};

struct Cache {
  Tensor k, v, err;
  pp_paged_cache c = {};
  int64_t index;
  at::ScalarType type;

  // Checked by the Python class: k and v alike, on one CUDA device.
  Cache(Tensor k_, Tensor v_, Tensor err_, bool rows_first) : k(std::move(k_)), v(std::move(v_)), err(std::move(err_)) {
    const int row = rows_first ? -3 : -2, head = rows_first ? -2 : -3;
    for (int64_t n : k.sizes())
      if (n > INT32_MAX) refuse("cache sizes out of range");
    index = k.get_device();
    type = k.scalar_type();
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    c.dtype = dtype_of(type);
    c.layers = k.dim() == 5 ? (uint32_t)k.size(0) : 1;
    c.n_pages = (uint32_t)k.size(-4);
    c.page_size = (uint32_t)k.size(row);
    c.n_kv_heads = (uint32_t)k.size(head);
    c.head_dim = (uint32_t)k.size(-1);
    c.layer_stride = k.dim() == 5 ? k.stride(0) : 0;
    c.page_stride = k.stride(-4);
    c.row_stride = k.stride(row);
    c.head_stride = k.stride(head);
    c.cuda_device = (int32_t)index;
  }

  uint32_t* err_word() const { return (uint32_t*)err.data_ptr(); }
  pp_paged_batch batch_of(const Batch& b, int64_t rows) const {
    if (b.index != index)
      refuse("the batch is on cuda:" + std::to_string(b.index) + ", the cache on cuda:" + std::to_string(index));
    pp_paged_batch d = b.c;
    if (rows > INT32_MAX) refuse("rows out of range");
    d.rows = (uint32_t)rows;
    if (!b.bounded) {
      const uint64_t most = (uint64_t)d.table_stride * c.page_size;
      d.max_len = most < 0x7fffffffu ? (uint32_t)most : 0x7fffffffu;
    }
    return d;
  }
  // Row stride of t, [rows, heads, dim] with the heads of a row adjacent.
  int64_t rows_of(const char* name, const Tensor& t, int64_t rows, int64_t heads, at::ScalarType want) const {
    const int64_t dim = c.head_dim;
    if (t.dim() != 3 || t.size(0) != rows || t.size(1) != heads || t.size(2) != dim || t.scalar_type() != want ||
        !t.is_cuda() || t.get_device() != index)
      refuse(std::string(name) + ": " + c10::toString(want) + " " + shape_text({rows, heads, dim}) + " on cuda:" +
             std::to_string(index) + " expected, got " + c10::toString(t.scalar_type()) + " " + shape_text(t.sizes()) +
             " on " + t.device().str());
    if (t.stride(2) != 1 || (heads > 1 && t.stride(1) != dim))
      refuse(std::string(name) + ": the heads of a row must be adjacent");
    return t.stride(0);
  }
  void check_layer(int64_t layer) const {
    if (layer < 0 || layer >= (int64_t)c.layers) refuse("layer outside the cache");
  }

  OptTensor append(const Batch& batch, const Tensor& kn, const Tensor& vn, const OptTensor& q, const OptTensor& inv_freq,
                   const OptTensor& positions, const OptTensor& q_norm, const OptTensor& k_norm, double eps,
                   bool interleaved, int64_t layer, OptTensor out) const {
    const int64_t rows = kn.dim() ? kn.size(0) : 0;
    const at::ScalarType t = kn.scalar_type();
    pp_append_rows a = {};
    a.dtype = dtype_of(t);
    if (a.dtype > PP_F16) refuse("k, v and q must be float32, bfloat16 or float16");
    a.k_stride = rows_of("k", kn, rows, c.n_kv_heads, t);
    a.v_stride = rows_of("v", vn, rows, c.n_kv_heads, t);
    a.k = kn.data_ptr();
    a.v = vn.data_ptr();
    if (q) {
      const int64_t heads = q->dim() == 3 ? q->size(1) : 0, dim = c.head_dim;
      a.q_stride = rows_of("q", *q, rows, heads, t);
      if (heads > INT32_MAX) refuse("q: too many heads");
      a.q = q->data_ptr();
      a.n_heads = (uint32_t)heads;
      if (!out) out = at::empty({rows, heads, dim}, on(index, type));
      a.q_out = pointer("out", *out, index, type, {rows, heads, dim});
    } else if (out) {
      refuse("out without q");
    }
    if (inv_freq) {
      a.rotary_dim = (uint32_t)(2 * inv_freq->numel());
      a.inv_freq = (const double*)pointer("inv_freq", *inv_freq, index, at::kDouble, {inv_freq->numel()});
    }
    const int64_t dim = c.head_dim;
    a.q_norm = (const float*)pointer("q_norm", q_norm, index, at::kFloat, {dim});
    a.k_norm = (const float*)pointer("k_norm", k_norm, index, at::kFloat, {dim});
    a.positions = (const int32_t*)pointer("positions", positions, index, at::kInt, {rows});
    a.eps = (float)eps;
    a.interleaved = interleaved;
    check_layer(layer);
    a.layer = (uint32_t)layer;
    if (rows) {
      const pp_paged_batch b = batch_of(batch, rows);
      check(pp_paged_append(&c, &b, &a, err_word(), stream_of(index)), "append");
    }
    return out;
  }

  Tensor tree_attention(const Batch& batch, const Tensor& q, const OptTensor& mask, std::optional<double> scale,
                        int64_t layer, OptTensor out, const OptTensor& lse) const {
    if (q.dim() != 3) refuse("q: [rows, heads, dim] expected");
    const int64_t rows = q.size(0), heads = q.size(1), dim = c.head_dim;
    pp_tree_query a = {};
    a.q_stride = rows_of("q", q, rows, heads, type);
    if (heads > INT32_MAX) refuse("q: too many heads");
    a.q = q.data_ptr();
    if (!out) out = at::empty({rows, heads, dim}, on(index, type));
    a.out = pointer("out", *out, index, type, {rows, heads, dim});
    a.lse = (float*)pointer("lse", lse, index, at::kFloat, {rows, heads});
    a.n_heads = (uint32_t)heads;
    check_layer(layer);
    a.layer = (uint32_t)layer;
    if (mask) {
      const int64_t words = mask->dim() == 2 ? mask->size(1) : 0;
      if (rows && words == 0) refuse("mask: [rows, words] int32 expected");
      a.mask = (const uint32_t*)pointer("mask", *mask, index, at::kInt, {rows, words});
      a.mask_words = (uint32_t)(words < INT32_MAX ? words : INT32_MAX);
    }
    a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)dim));
    if (rows) {
      const pp_paged_batch b = batch_of(batch, rows);
      const uint64_t need = pp_tree_attention_work_bytes(&c, &b, a.n_heads);
      if (!need) check(PP_E_INVALID, "tree_attention");
      const Tensor work = at::empty({(int64_t)need}, on(index, at::kByte));
      check(pp_tree_attention(&c, &b, &a, work.data_ptr(), need, err_word(), stream_of(index)), "tree_attention");
    }
    return *out;
  }

  py::tuple tree_commit(const Batch& batch, const Tensor& tokens, const Tensor& parents, const Tensor& picks) const {
    if (tokens.dim() != 1) refuse("tokens: [rows] expected");
    const int64_t n = batch.c.batch, rows = tokens.size(0), width = batch.c.max_rows ? batch.c.max_rows : 1;
    // A batch without rows has no arrays: any valid pointer stands in.
    auto ints = [&](const char* name, const Tensor& t) -> const int32_t* {
      void* p = pointer(name, t, index, at::kInt, {rows});
      return (const int32_t*)(p ? p : err_word());
    };
    const int32_t *tp = ints("tokens", tokens), *pp = ints("parents", parents), *kp = ints("picks", picks);
    const at::TensorOptions o = on(index, at::kInt);
    const Tensor path = at::empty({n, width}, o), rest = at::empty({3, n}, o);
    int32_t* r = (int32_t*)rest.data_ptr();
    const pp_paged_batch b = batch_of(batch, rows);
    check(pp_tree_commit(&c, &b, tp, pp, kp, (int32_t*)path.data_ptr(), (uint32_t)width, r, r + n, r + 2 * n, err_word(),
                         stream_of(index)),
          "tree_commit");
    return py::make_tuple(path, rest.select(0, 0), rest.select(0, 1), rest.select(0, 2));
  }

  py::tuple beam_reorder(const Tensor& table, const Tensor& lengths, const Tensor& beams, const Tensor& spare) const {
    if (table.dim() != 3 || beams.dim() != 2)
      refuse("page_table: [groups, beams, pages] and beams: [groups, new beams] expected");
    const int64_t g = table.size(0), old = table.size(1), stride = table.size(2), next = beams.size(1);
    if (g > INT32_MAX || old > INT32_MAX || stride > INT32_MAX || next > INT32_MAX) refuse("page_table too large");
    auto ints = [&](const char* name, const Tensor& t, at::IntArrayRef shape) {
      return (const int32_t*)pointer(name, t, index, at::kInt, shape);
    };
    const int32_t *tp = ints("page_table", table, {g, old, stride}), *lp = ints("lengths", lengths, {g, old}),
                  *bp = ints("beams", beams, {g, next}), *sp = ints("spare", spare, {g, next});
    const at::TensorOptions o = on(index, at::kInt);
    const Tensor moved = at::empty({g, next, stride}, o), rest = at::empty({2, g, next}, o);
    int32_t* r = (int32_t*)rest.data_ptr();
    check(pp_beam_reorder(&c, tp, lp, (uint32_t)g, (uint32_t)old, (uint32_t)next, (uint32_t)stride, bp, sp,
                          (int32_t*)moved.data_ptr(), r, r + g * next, err_word(), stream_of(index)),
          "beam_reorder");
    return py::make_tuple(moved, rest.select(0, 0), rest.select(0, 1));
  }
};

py::tuple beam_select(const Tensor& logits, const Tensor& scores, int64_t k, const OptTensor& finished, int64_t pad,
                      const OptTensor& err) {
  const uint32_t t = dtype_of(logits.scalar_type());
  if (logits.dim() != 3 || t > PP_F16 || !logits.is_cuda())
    refuse("logits: [groups, beams, vocab] float32, bfloat16 or float16 on a CUDA device expected");
  const int64_t index = logits.get_device(), g = logits.size(0), w = logits.size(1), vocab = logits.size(2);
  if ((vocab > 1 && logits.stride(2) != 1) || (g > 1 && w > 1 && logits.stride(0) != w * logits.stride(1)))
    refuse("logits: contiguous rows, evenly spaced, expected");
  if (g > INT32_MAX || w > INT32_MAX || vocab > INT32_MAX || k < 1 || k > INT32_MAX) refuse("sizes or k out of range");
  const int64_t row = w > 1 ? logits.stride(1) : g > 1 ? logits.stride(0) : vocab;
  const float* sp = (const float*)pointer("scores", scores, index, at::kFloat, {g, w});
  const uint8_t* fp = nullptr;
  if (finished)
    fp = (const uint8_t*)pointer("finished", *finished, index,
                                 finished->scalar_type() == at::kByte ? at::kByte : at::kBool, {g, w});
  uint32_t* ep = (uint32_t*)pointer("err", err, index, at::kInt, {1});
  const uint64_t need = pp_beam_select_work_bytes((uint32_t)g, (uint32_t)w, (uint32_t)vocab, (uint32_t)k);
  if (need > (1ull << 36)) refuse("sizes or k out of range");
  const Tensor work = at::empty({(int64_t)(need ? need : 16)}, on(index, at::kByte));
  const Tensor best = at::empty({g, k}, on(index, at::kFloat)), picks = at::empty({2, g, k}, on(index, at::kInt));
  int32_t* p = (int32_t*)picks.data_ptr();
  check(pp_beam_select(logits.data_ptr(), (pp_dtype)t, row, sp, fp, (int32_t)pad, (uint32_t)g, (uint32_t)w,
                       (uint32_t)vocab, (uint32_t)k, (float*)best.data_ptr(), p, p + g * k, work.data_ptr(), need, ep,
                       (int32_t)index, stream_of(index)),
        "beam_select");
  return py::make_tuple(best, picks.select(0, 0), picks.select(0, 1));
}

}  // namespace

PYBIND11_MODULE(_paged, m) {
  const auto none = py::none();
  py::class_<Batch>(m, "Batch")
      .def(py::init<Tensor, Tensor, Tensor, int64_t, std::optional<int64_t>>(), py::arg("page_table"),
           py::arg("lengths"), py::arg("cu_rows"), py::arg("max_rows"), py::arg("max_length") = none)
      .def_readonly("page_table", &Batch::page_table)
      .def_readonly("lengths", &Batch::lengths)
      .def_readonly("cu_rows", &Batch::cu_rows);
  py::class_<Cache>(m, "Cache")
      .def(py::init<Tensor, Tensor, Tensor, bool>())
      .def_readonly("k", &Cache::k)
      .def_readonly("v", &Cache::v)
      .def_readonly("err", &Cache::err)
      .def("append", &Cache::append, py::arg("batch"), py::arg("k"), py::arg("v"), py::arg("q") = none,
           py::arg("inv_freq") = none, py::arg("positions") = none, py::arg("q_norm") = none, py::arg("k_norm") = none,
           py::arg("eps") = 1e-6, py::arg("interleaved") = false, py::arg("layer") = 0, py::arg("out") = none,
           "Write the rows k, v [rows, kv_heads, dim] into the pages of their positions, k normed and rotated on "
           "the way; returns q [rows, heads, dim] normed and rotated likewise in the cache's type (None without q). "
           "inv_freq [rotary_dim / 2] float64 radians per position.")
      .def("tree_attention", &Cache::tree_attention, py::arg("batch"), py::arg("q"), py::arg("mask") = none,
           py::arg("scale") = none, py::arg("layer") = 0, py::arg("out") = none, py::arg("lse") = none,
           "Attention of q [rows, heads, dim] (the cache's type) over the cache. Row i of a sequence sees its "
           "context and the nodes j whose bit j % 32 of mask[row, j // 32] (int32 words) is set; without a mask the "
           "rows are a chain. scale defaults to dim ** -0.5. lse, optional: [rows, heads] float32, receives the log "
           "of the softmax's sum.")
      .def("tree_commit", &Cache::tree_commit, py::arg("batch"), py::arg("tokens"), py::arg("parents"),
           py::arg("picks"),
           "Accept every tree's longest path that the target's picks follow and move its K/V rows, in every layer, "
           "to the front of the tree's. tokens, parents, picks: [rows] int32. Returns (path [batch, max_rows], "
           "accepted, correction, lengths), int32.")
      .def("beam_reorder", &Cache::beam_reorder, py::arg("page_table"), py::arg("lengths"), py::arg("beams"),
           py::arg("spare"),
           "States of new beams j continuing old beams beams[g, j]: (page table [groups, new, pages], lengths "
           "[groups, new], taken [groups, new]). Full pages are shared; a part-full last page stays with its first "
           "child and is copied, every layer, into page spare[g, j] for each other (taken[g, j] = 1).");
  m.def("beam_select", &beam_select, py::arg("logits"), py::arg("scores"), py::arg("k"), py::arg("finished") = none,
        py::arg("pad") = 0, py::arg("err") = none,
        "The k best continuations of every group of beams: logits [groups, beams, vocab], scores [groups, beams] "
        "float32 running log-probabilities (-inf: not in use), finished [groups, beams] bool or uint8 (such a beam "
        "goes on only as token `pad`, its score unchanged). Returns scores float32, beams int32, tokens int32, each "
        "[groups, k], best first, ties to the lower beam and token; -inf, -1, -1 where candidates run out. err: int32 "
        "[1], gets value 2 where a beam was left out for a NaN or +inf.");
}

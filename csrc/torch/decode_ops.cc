// Calls of the decode-step operators (quantizing store, tree attention, constrained logits) on torch
// tensors: the checks of arguments, the allocation of results and workspaces and the launch, on the
// first tensor's device and that device's current stream. Decode calls are short, and in Python the
// checks alone took 8 of a call's 16 us. This module is built against torch; the kernels stay in the
// engine's extension (which needs no torch) and are called through the addresses it gives out.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "kernels/decode_ops.cuh"

namespace py = pybind11;

namespace {

struct Launchers {
  decltype(&foa::kv_store) kv_store = nullptr;
  decltype(&foa::tree_attention) tree_attention = nullptr;
  decltype(&foa::tree_attention_split) tree_attention_split = nullptr;
  decltype(&foa::process_logits) process_logits = nullptr;
  decltype(&foa::logits_slices) logits_slices = nullptr;
} run;

[[noreturn]] void refuse(const std::string& why) { throw py::value_error(why); }

// A tensor's address, type, device, sizes and strides.
struct View {
  static constexpr int kDims = 5;
  uint64_t ptr = 0;
  at::ScalarType dtype = at::ScalarType::Undefined;
  int device = -1, dim = 0;
  long size[kDims] = {}, stride[kDims] = {};

  explicit View(py::handle t, const char* what) {
    if (!THPVariable_Check(t.ptr())) throw py::type_error(std::string(what) + " must be a torch tensor");
    const at::Tensor& x = THPVariable_Unpack(t.ptr());
    if (x.layout() != at::kStrided) refuse(std::string(what) + " must be a strided tensor");
    dtype = x.scalar_type();
    device = x.is_cuda() ? x.get_device() : -1;
    dim = (int)x.dim();
    for (int i = 0; i < dim && i < kDims; ++i) {
      size[i] = x.size(i);
      stride[i] = x.stride(i);
    }
    ptr = reinterpret_cast<uint64_t>(x.data_ptr());
  }
  bool is(std::initializer_list<long> shape) const {
    if (dim != (int)shape.size()) return false;
    int i = 0;
    for (long n : shape)
      if (size[i++] != n) return false;
    return true;
  }
  bool contiguous() const {
    long want = 1;
    for (int i = dim - 1; i >= 0; --i) {
      if (size[i] == 0) return true;
      if (size[i] != 1 && stride[i] != want) return false;
      want *= size[i];
    }
    return true;
  }
};

// A call's device: that of its first tensor, which the others have to share.
struct Place {
  int device;
  explicit Place(const View& first) : device(first.device) {}
  void with(const View& t) const {
    if (t.device != device) refuse(device < 0 || t.device < 0 ? "the operands must be CUDA tensors" : "the operands must be on one CUDA device");
  }
  void check() const {
    if (device < 0) refuse("the operands must be CUDA tensors");
  }
};

at::Tensor allocate(at::ScalarType dtype, int device, std::initializer_list<int64_t> shape) {
  return at::empty(shape, at::TensorOptions().dtype(dtype).device(at::kCUDA, (c10::DeviceIndex)device));
}
uint64_t address(const at::Tensor& t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }
py::object wrap(at::Tensor t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t))); }
cudaStream_t stream_of(int device) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream(); }

void check(int rc, const char* what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + " launch rejected: code " + std::to_string(rc));
}

std::string list(std::initializer_list<long> shape) {
  std::string s = "[";
  for (long n : shape) s += (s.size() > 1 ? ", " : "") + std::to_string(n);
  return s + "]";
}

void ints(const View& t, std::initializer_list<long> shape, const char* name) {
  if (t.dtype != at::kInt || !t.is(shape) || !t.contiguous())
    refuse(std::string(name) + " must be a contiguous int32 tensor of shape " + list(shape));
}

// BF16 [rows, heads, d] whose rows are packed, each row 16-byte aligned.
void heads(const View& t, const char* name) {
  const std::string n(name);
  if (t.dtype != at::kBFloat16 || t.dim != 3) refuse(n + " must be BF16 [rows, heads, head_dim]");
  if ((t.stride[2] != 1 && t.size[2] != 1) || (t.stride[1] != t.size[2] && t.size[1] != 1))
    refuse(n + " must have its heads packed in each row");
  if (t.size[0] > 1 && (t.stride[0] < t.size[1] * t.size[2] || t.stride[0] % 8 != 0))
    refuse(n + " must have rows a multiple of 8 elements apart");
  if (t.ptr % 16 != 0) refuse(n + " must be 16-byte aligned");
}

// Quantized pages of heads of d. (A QuantizedCache checks them too when it is made, but its fields can
// be set to other ones later.)
void quantized_pages(const View& t, long d) {
  if ((d != 64 && d != 128) || t.dtype != at::kByte || t.dim != 4 || t.size[1] != 2 ||
      t.size[3] != foa::quantized_page_bytes((int)d) || !t.contiguous() || t.ptr % 16 != 0)
    refuse("quantized pages must be contiguous uint8 [blocks, 2, kv_heads, 16 * head_dim + 64] for a head_dim of 64 or 128, 16-byte aligned");
}

// The layer's pages: quantized ones when head_dim > 0.
void pages(const View& t, int quantized_dim, long kv_heads, long d, const char* what) {
  if (quantized_dim > 0) {
    quantized_pages(t, quantized_dim);
    if (quantized_dim != d || t.size[2] != kv_heads) refuse("the cache has other heads");
  } else if (t.dtype != at::kBFloat16 || t.dim != 5 || t.size[1] != 2 || t.size[2] != kv_heads || t.size[3] != 16 ||
             t.size[4] != d || !t.contiguous() || t.ptr % 16 != 0) {
    refuse(what);
  }
}

// Two tensors of as many rows of `width` bytes (elements of `size` bytes) are the same one or share
// nothing: rows are read while others are written.
void same_or_apart(const View& a, const View& b, long width, long size, const char* what) {
  const long rows = a.size[0], as = rows > 1 ? a.stride[0] * size : width, bs = rows > 1 ? b.stride[0] * size : width;
  if (rows == 0 || (a.ptr == b.ptr && as == bs)) return;
  if (a.ptr + (rows - 1) * as + width <= b.ptr || b.ptr + (rows - 1) * bs + width <= a.ptr) return;
  // Side by side in the rows of one tensor.
  const long shift = (((long)(b.ptr - a.ptr)) % as + as) % as;
  if (as != bs || shift < width || shift + width > as) refuse(what);
}

template <class T>
T* at(uint64_t p) {
  return reinterpret_cast<T*>(p);
}

py::object kv_store(py::handle qkv, long q_heads, long kv_heads, long d, py::handle q_norm, py::handle k_norm, float eps,
                    py::handle positions, py::handle inv_freq, float attention_factor, py::handle cache, int quantized_dim,
                    py::handle slots, long rotary_dim, bool interleaved, uint64_t status) {
  const View x(qkv, "qkv");
  if (x.dtype != at::kBFloat16 || x.dim != 2 || x.size[1] != (q_heads + 2 * kv_heads) * d)
    refuse("qkv must be BF16 [rows, (q_heads + 2 * kv_heads) * head_dim]");
  if (kv_heads < 1 || q_heads < 0 || kv_heads > 1 << 16 || q_heads > 1 << 16 || (d != 64 && d != 128))
    refuse("head_dim must be 64 or 128, with at least one key/value head");
  const long rows = x.size[0];
  if (x.stride[1] != 1 || (rows > 1 && (x.stride[0] < x.size[1] || x.stride[0] % 8 != 0)) || x.ptr % 16 != 0)
    refuse("qkv must have unit column stride and 16-byte aligned rows");
  if (rotary_dim % 16 != 0 || rotary_dim < 16 || rotary_dim > d) refuse("rotary_dim must be a multiple of 16, at most head_dim");
  if (q_norm.is_none() != k_norm.is_none()) refuse("q_norm and k_norm come together");
  Place place(x);
  foa::KvStore a;
  if (!q_norm.is_none()) {
    const View w[2] = {View(q_norm, "q_norm"), View(k_norm, "k_norm")};
    for (const View& v : w) {
      if (v.dtype != at::kBFloat16 || !v.is({d}) || !v.contiguous() || v.ptr % 16 != 0)
        refuse("norm weights must be contiguous BF16 [head_dim], 16-byte aligned");
      place.with(v);
    }
    a.q_norm = at<const __nv_bfloat16>(w[0].ptr);
    a.k_norm = at<const __nv_bfloat16>(w[1].ptr);
  }
  const View pos(positions, "positions"), slot(slots, "slots"), freq(inv_freq, "inv_freq"), c(cache, "cache");
  ints(pos, {rows}, "positions");
  ints(slot, {rows}, "slots");
  if (freq.dtype != at::kFloat || !freq.is({rotary_dim / 2}) || !freq.contiguous())
    refuse("inv_freq must be a contiguous FP32 tensor of rotary_dim / 2 frequencies");
  pages(c, quantized_dim, kv_heads, d, "the cache must be contiguous BF16 [blocks, 2, kv_heads, 16, head_dim]");
  for (const View* v : {&pos, &slot, &freq, &c}) place.with(*v);
  place.check();
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)place.device);
  at::Tensor q = allocate(at::kBFloat16, place.device, {rows, q_heads, d});
  a.qkv = at<const __nv_bfloat16>(x.ptr);
  a.ld_qkv = rows > 1 ? x.stride[0] : x.size[1];
  if (rows > 1L << 30) refuse("qkv has more than 2^30 rows");
  a.rows = (int)rows;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)d;
  a.eps = eps;
  a.positions = at<const int32_t>(pos.ptr);
  a.inv_freq = at<const float>(freq.ptr);
  a.attention_factor = attention_factor;
  a.rotary_dim = (int)rotary_dim;
  a.interleaved = interleaved ? 1 : 0;
  a.q_out = at<__nv_bfloat16>(address(q));
  a.cache = at<void>(c.ptr);
  a.quantized = quantized_dim > 0 ? 1 : 0;
  a.slots = at<const int32_t>(slot.ptr);
  a.cache_slots = c.size[0] * 16;
  a.status = at<int>(status);
  int rc;
  {
    py::gil_scoped_release nogil;
    rc = run.kv_store(a, stream_of(place.device));
  }
  check(rc, "kv_store");
  return wrap(std::move(q));
}

py::object tree_attention(py::handle q, py::handle cache, int quantized_dim, py::handle table, py::handle segments,
                          long kv_heads, long max_keys, long max_len, py::handle mask, py::handle scale, py::handle split,
                          py::handle out, uint64_t status) {
  const View x(q, "q");
  heads(x, "q");
  const long rows = x.size[0], q_heads = x.size[1], d = x.size[2];
  if ((d != 64 && d != 128) || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0)
    refuse("head_dim must be 64 or 128, with query heads a multiple of the key/value heads");
  const View c(cache, "cache"), seg(segments, "segments"), tab(table, "table");
  pages(c, quantized_dim, kv_heads, d, "the cache must be contiguous BF16 [blocks, 2, kv_heads, 16, d], or a QuantizedCache");
  const long n = seg.dim > 0 ? seg.size[0] : 0;
  ints(seg, {n, 5}, "segments");
  ints(tab, {tab.dim == 1 ? tab.size[0] : 0}, "table");
  if (max_keys < 1 || max_len < 1 || max_keys > 1L << 30 || max_len > 1L << 24)
    refuse("max_keys must be in [1, 2^30] and max_len in [1, 2^24]");
  if (rows > 1L << 30 || n > 1L << 30 || q_heads > 65535) refuse("q has too many rows or heads");
  long width = 0;
  if (!split.is_none()) {
    width = py::cast<long>(split);
    if (width < 16 || width % 16 != 0 || width > 1L << 30) refuse("keys_per_split must be a positive multiple of 16");
  }
  Place place(x);
  for (const View* v : {&c, &seg, &tab}) place.with(*v);
  foa::TreeAttention a;
  if (!mask.is_none()) {
    const View m(mask, "mask");
    const long words = m.dim == 2 ? m.size[1] : 0;
    ints(m, {rows, words}, "mask");
    if (words < 1 || words > 1L << 20) refuse("mask must have a word for every 32 appended rows");
    place.with(m);
    a.mask = at<const uint32_t>(m.ptr);
    a.mask_words = (int)words;
  }
  py::object o;
  if (!out.is_none()) {
    const View y(out, "out");
    heads(y, "out");
    if (!y.is({rows, q_heads, d})) refuse("out must have the shape of q");
    same_or_apart(x, y, q_heads * d * 2, 2, "out must be q itself or not overlap it");
    place.with(y);
    o = py::reinterpret_borrow<py::object>(out);
    a.o = at<__nv_bfloat16>(y.ptr);
    a.ld_o = rows > 1 ? y.stride[0] : q_heads * d;
  }
  const float s = scale.is_none() ? (d == 64 ? 0.125f : 0.08838834764831845f) : py::cast<float>(scale);
  if (!std::isfinite(s)) refuse("scale must be finite in FP32");
  place.check();
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)place.device);
  if (out.is_none()) {
    at::Tensor made = allocate(at::kBFloat16, place.device, {rows, q_heads, d});
    a.o = at<__nv_bfloat16>(address(made));
    o = wrap(std::move(made));
    a.ld_o = q_heads * d;
  }
  if (n == 0 || rows == 0) return o;
  a.quantized = quantized_dim > 0 ? 1 : 0;
  if (width == 0)
    width = run.tree_attention_split((int)n, (int)q_heads, (int)kv_heads, (int)d, a.quantized, (int)max_keys, (int)max_len);
  const long splits = (max_keys + width - 1) / width;
  at::Tensor work;
  if (splits > 1) {
    const long need = rows * q_heads * splits;
    work = allocate(at::kFloat, place.device, {need * (d + 2)});
    const uint64_t w = address(work);
    a.partial_o = at<float>(w);
    a.partial_ml = at<float2>(w + (uint64_t)need * d * 4);
    a.partial_capacity = (size_t)need;
  }
  a.q = at<const __nv_bfloat16>(x.ptr);
  a.ld_q = rows > 1 ? x.stride[0] : q_heads * d;
  a.rows = (int)rows;
  a.cache = at<const void>(c.ptr);
  a.cache_blocks = c.size[0];
  a.table = at<const int32_t>(tab.ptr);
  a.table_len = tab.size[0];
  a.segments = at<const foa::Segment>(seg.ptr);
  a.num_segments = (int)n;
  a.q_heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)d;
  a.scale = s;
  a.max_keys = (int)max_keys;
  a.max_len = (int)max_len;
  a.keys_per_split = (int)width;
  a.status = at<int>(status);
  int rc;
  {
    py::gil_scoped_release nogil;
    rc = run.tree_attention(a, stream_of(place.device));
  }
  check(rc, "tree_attention");
  return o;
}

// Views of quantized pages: the rows' codes, and their scales.
py::object codes(py::handle pages, long d) {
  quantized_pages(View(pages, "pages"), d);
  const at::Tensor& x = THPVariable_Unpack(pages.ptr());
  const int64_t page = x.size(3), heads = x.size(2) * page;
  return wrap(x.as_strided({x.size(0), 2, x.size(2), 16, d}, {2 * heads, heads, page, d, 1}));
}
py::object scales(py::handle pages, long d) {
  quantized_pages(View(pages, "pages"), d);
  const at::Tensor& x = THPVariable_Unpack(pages.ptr());
  return wrap(x.slice(3, 16 * d).view(at::kFloat));
}

// (tokens, ..., starts): row r's tokens are tokens[starts[r] .. starts[r + 1]).
foa::TokenLists token_lists(py::handle lists, long rows, const char* name, const Place& place) {
  foa::TokenLists l;
  if (lists.is_none()) return l;
  py::sequence s = py::reinterpret_borrow<py::sequence>(lists);
  const size_t n = py::len(s);
  if (n < 2) refuse(std::string(name) + " must be (tokens, starts)");
  const py::object t = s[0], f = s[n - 1];
  const View tokens(t, name), starts(f, name);
  const std::string what(name);
  ints(tokens, {tokens.dim == 1 ? tokens.size[0] : 0}, (what + " tokens").c_str());
  ints(starts, {rows + 1}, (what + " starts").c_str());
  if (tokens.size[0] > 1L << 30) refuse(what + " holds more than 2^30 tokens");
  place.with(tokens);
  place.with(starts);
  // (An empty list still has starts to read; the address stands for "given".)
  l.tokens = at<const int32_t>(tokens.size[0] > 0 ? tokens.ptr : starts.ptr);
  l.starts = at<const int32_t>(starts.ptr);
  l.count = (int)tokens.size[0];
  return l;
}

py::object process_logits(py::handle logits, py::handle prompt, py::handle output, py::handle repetition,
                          py::handle frequency, py::handle presence, py::handle bias, py::handle allowed, py::handle out,
                          uint64_t status) {
  const View x(logits, "logits");
  if (x.dim != 2 || (x.dtype != at::kFloat && x.dtype != at::kBFloat16)) refuse("logits must be FP32 or BF16 [rows, vocab]");
  const long rows = x.size[0], vocab = x.size[1];
  if (vocab < 1 || vocab > 1L << 30 || rows > 1L << 24) refuse("logits must have 1 to 2^30 columns and at most 2^24 rows");
  if ((x.stride[1] != 1 && vocab != 1) || (rows > 1 && x.stride[0] < vocab)) refuse("logits must have unit column stride");
  Place place(x);
  foa::LogitsArgs a;
  a.prompt = token_lists(prompt, rows, "prompt", place);
  a.output = token_lists(output, rows, "output", place);
  a.bias = token_lists(bias, rows, "bias", place);
  if (!bias.is_none()) {
    py::sequence s = py::reinterpret_borrow<py::sequence>(bias);
    if (py::len(s) != 3) refuse("bias must be (tokens, FP32 values, starts)");
    const py::object given = s[1];
    const View v(given, "bias values");
    if (v.dtype != at::kFloat || !v.is({a.bias.count}) || !v.contiguous()) refuse("bias must be (tokens, FP32 values, starts)");
    place.with(v);
    a.bias_values = at<const float>(v.ptr);
  }
  auto per_row = [&](py::handle t, const char* name) -> const float* {
    if (t.is_none()) return nullptr;
    const View v(t, name);
    if (v.dtype != at::kFloat || !v.is({rows}) || !v.contiguous())
      refuse(std::string(name) + " must be a contiguous FP32 tensor of one value a row");
    place.with(v);
    return at<const float>(v.ptr);
  };
  a.repetition = per_row(repetition, "repetition");
  a.frequency = per_row(frequency, "frequency");
  a.presence = per_row(presence, "presence");
  if (!allowed.is_none()) {
    const View v(allowed, "allowed");
    if (v.dtype != at::kInt || v.dim != 2 || v.size[0] != rows || v.size[1] < (vocab + 31) / 32 ||
        (v.stride[1] != 1 && v.size[1] != 1) || (rows > 1 && v.stride[0] < 0))
      refuse("allowed must be int32 [rows, at least vocab / 32] with unit column stride");
    place.with(v);
    a.allowed = at<const uint32_t>(v.ptr);
    a.ld_allowed = v.stride[0];
  }
  if (!out.is_none()) {
    const View v(out, "out");
    if (v.dtype != x.dtype || !v.is({rows, vocab}) || (v.stride[1] != 1 && vocab != 1) || (rows > 1 && v.stride[0] < vocab))
      refuse("out must have the logits' shape and type, and unit column stride");
    const long size = x.dtype == at::kFloat ? 4 : 2;
    same_or_apart(x, v, vocab * size, size, "out must be the logits themselves or not overlap them");
    place.with(v);
    a.out = at<void>(v.ptr);
    a.ldo = v.stride[0];
  }
  place.check();
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)place.device);
  at::Tensor index = allocate(at::kInt, place.device, {rows}), value = allocate(at::kFloat, place.device, {rows});
  if (rows == 0) return py::make_tuple(wrap(std::move(index)), wrap(std::move(value)));
  at::Tensor partial;
  const long slices = run.logits_slices((int)vocab);
  if (slices > 1) {
    partial = allocate(at::kFloat, place.device, {rows * slices * 2});
    a.partial = at<float2>(address(partial));
    a.partial_count = (size_t)(rows * slices);
  }
  a.logits = at<const void>(x.ptr);
  a.half = x.dtype == at::kBFloat16 ? 1 : 0;
  a.ld = x.stride[0];
  a.rows = (int)rows;
  a.vocab = (int)vocab;
  a.index = at<int32_t>(address(index));
  a.value = at<float>(address(value));
  a.status = at<int>(status);
  int rc;
  {
    py::gil_scoped_release nogil;
    rc = run.process_logits(a, stream_of(place.device));
  }
  check(rc, "process_logits");
  return py::make_tuple(wrap(std::move(index)), wrap(std::move(value)));
}

}  // namespace

PYBIND11_MODULE(_calls, m) {
  m.doc() = "Calls of the decode-step operators on torch tensors.";
  m.def("connect", [](uint64_t kv_store, uint64_t tree_attention, uint64_t tree_attention_split, uint64_t process_logits,
                      uint64_t logits_slices) {
    run.kv_store = reinterpret_cast<decltype(run.kv_store)>(kv_store);
    run.tree_attention = reinterpret_cast<decltype(run.tree_attention)>(tree_attention);
    run.tree_attention_split = reinterpret_cast<decltype(run.tree_attention_split)>(tree_attention_split);
    run.process_logits = reinterpret_cast<decltype(run.process_logits)>(process_logits);
    run.logits_slices = reinterpret_cast<decltype(run.logits_slices)>(logits_slices);
  });
  m.def("codes", &codes);
  m.def("scales", &scales);
  m.def("kv_store", &kv_store);
  m.def("tree_attention", &tree_attention);
  m.def("process_logits", &process_logits);
}

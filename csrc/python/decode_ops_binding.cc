// Raw launchers of the decode-step operators (quantizing store, tree attention, constrained logits):
// tensors cross as device addresses and strides, launches as a CUDA stream handle. The arguments are
// positional only in these three (a call's host time counts), in the order of the structs' fields.
#include <pybind11/pybind11.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "kernels/decode_ops.cuh"

namespace py = pybind11;

namespace {

template <class T>
T* at(uint64_t p) {
  return reinterpret_cast<T*>(p);
}

void check(int rc, const char* what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + " launch rejected: code " + std::to_string(rc));
}

}  // namespace

void bind_decode_ops(py::module_& m) {
  m.def("kv_store", [](uint64_t qkv, long ld_qkv, int rows, int q_heads, int kv_heads, int head_dim, uint64_t q_norm,
                       uint64_t k_norm, float eps, uint64_t positions, uint64_t inv_freq, float attention_factor,
                       int rotary_dim, bool interleaved, uint64_t q_out, uint64_t cache, bool quantized, uint64_t slots,
                       long cache_slots, uint64_t status, uint64_t stream) {
    foa::KvStore a;
    a.qkv = at<const __nv_bfloat16>(qkv);
    a.ld_qkv = ld_qkv;
    a.rows = rows;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.q_norm = at<const __nv_bfloat16>(q_norm);
    a.k_norm = at<const __nv_bfloat16>(k_norm);
    a.eps = eps;
    a.positions = at<const int32_t>(positions);
    a.inv_freq = at<const float>(inv_freq);
    a.attention_factor = attention_factor;
    a.rotary_dim = rotary_dim;
    a.interleaved = interleaved ? 1 : 0;
    a.q_out = at<__nv_bfloat16>(q_out);
    a.cache = at<void>(cache);
    a.quantized = quantized ? 1 : 0;
    a.slots = at<const int32_t>(slots);
    a.cache_slots = cache_slots;
    a.status = at<int>(status);
    check(foa::kv_store(a, at<CUstream_st>(stream)), "kv_store");
  }, py::call_guard<py::gil_scoped_release>());
  m.def("tree_attention_split", &foa::tree_attention_split);
  m.def("tree_attention", [](uint64_t q, long ld_q, uint64_t o, long ld_o, int rows, uint64_t cache, bool quantized,
                             long cache_blocks, uint64_t table, long table_len, uint64_t segments, int num_segments,
                             int q_heads, int kv_heads, int head_dim, float scale, uint64_t mask, int mask_words,
                             int max_keys, int max_len, int keys_per_split, uint64_t partial_o, uint64_t partial_ml,
                             size_t capacity, uint64_t status, uint64_t stream) {
    foa::TreeAttention a;
    a.q = at<const __nv_bfloat16>(q);
    a.ld_q = ld_q;
    a.o = at<__nv_bfloat16>(o);
    a.ld_o = ld_o;
    a.rows = rows;
    a.cache = at<const void>(cache);
    a.quantized = quantized ? 1 : 0;
    a.cache_blocks = cache_blocks;
    a.table = at<const int32_t>(table);
    a.table_len = table_len;
    a.segments = at<const foa::Segment>(segments);
    a.num_segments = num_segments;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.head_dim = head_dim;
    a.scale = scale;
    a.mask = at<const uint32_t>(mask);
    a.mask_words = mask_words;
    a.max_keys = max_keys;
    a.max_len = max_len;
    a.keys_per_split = keys_per_split;
    a.partial_o = at<float>(partial_o);
    a.partial_ml = at<float2>(partial_ml);
    a.partial_capacity = capacity;
    a.status = at<int>(status);
    check(foa::tree_attention(a, at<CUstream_st>(stream)), "tree_attention");
  }, py::call_guard<py::gil_scoped_release>());
  m.def("logits_slices", &foa::logits_slices);
  m.def("process_logits", [](uint64_t logits, long ld, uint64_t out, long ldo, bool half, int rows, int vocab,
                             uint64_t prompt, uint64_t prompt_starts, int prompt_count, uint64_t output,
                             uint64_t output_starts, int output_count, uint64_t bias, uint64_t bias_starts,
                             int bias_count, uint64_t bias_values, uint64_t repetition, uint64_t frequency,
                             uint64_t presence, uint64_t allowed, long ld_allowed, uint64_t index, uint64_t value,
                             uint64_t partial, size_t partial_count, uint64_t status, uint64_t stream) {
    foa::LogitsArgs a;
    a.logits = at<const void>(logits);
    a.out = at<void>(out);
    a.half = half ? 1 : 0;
    a.ld = ld;
    a.ldo = ldo;
    a.rows = rows;
    a.vocab = vocab;
    a.prompt = {at<const int32_t>(prompt), at<const int32_t>(prompt_starts), prompt_count};
    a.output = {at<const int32_t>(output), at<const int32_t>(output_starts), output_count};
    a.bias = {at<const int32_t>(bias), at<const int32_t>(bias_starts), bias_count};
    a.bias_values = at<const float>(bias_values);
    a.repetition = at<const float>(repetition);
    a.frequency = at<const float>(frequency);
    a.presence = at<const float>(presence);
    a.allowed = at<const uint32_t>(allowed);
    a.ld_allowed = ld_allowed;
    a.index = at<int32_t>(index);
    a.value = at<float>(value);
    a.partial = at<float2>(partial);
    a.partial_count = partial_count;
    a.status = at<int>(status);
    check(foa::process_logits(a, at<CUstream_st>(stream)), "process_logits");
  }, py::call_guard<py::gil_scoped_release>());
}

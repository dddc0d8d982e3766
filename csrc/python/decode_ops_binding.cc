// The addresses of the decode-step operators' launchers, for the module that calls them on torch
// tensors (csrc/torch), and how attention cuts a history into parts.
#include <pybind11/pybind11.h>

#include <cstdint>

#include "kernels/decode_ops.cuh"
#include "kernels/tree_split.cuh"

namespace py = pybind11;

void bind_decode_ops(py::module_& m) {
  m.def("decode_launchers", [] {
    auto at = [](auto* f) { return reinterpret_cast<uint64_t>(f); };
    return py::make_tuple(at(&foa::kv_store), at(&foa::tree_attention), at(&foa::tree_attention_split),
                          at(&foa::process_logits), at(&foa::logits_slices));
  });
  m.def("history_parts", [](int keys, int keys_per_split, bool even) {
    if (keys < 1 || keys > 1 << 30 || keys_per_split < 16 || keys_per_split > 1 << 30)
      throw py::value_error("keys must be in [1, 2^30] and keys_per_split in [16, 2^30]");
    const foa::Parts parts(keys, keys_per_split, even);
    return py::make_tuple(parts.width, parts.count);
  });
}

// The addresses of the decode-step operators' launchers, for the module that calls them on torch
// tensors (csrc/torch).
#include <pybind11/pybind11.h>

#include <cstdint>

#include "kernels/decode_ops.cuh"

namespace py = pybind11;

void bind_decode_ops(py::module_& m) {
  m.def("decode_launchers", [] {
    auto at = [](auto* f) { return reinterpret_cast<uint64_t>(f); };
    return py::make_tuple(at(&foa::kv_store), at(&foa::tree_attention), at(&foa::tree_attention_split),
                          at(&foa::process_logits), at(&foa::logits_slices));
  });
}

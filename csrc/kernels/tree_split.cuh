// The parts of one history: keys_per_split keys each (mma.sync form), or as few as that allows and
// equally long in whole 128-key tiles (tcgen05 form, which holds an SM alone: a CTA with a short rest
// costs its set-up). A row's parts follow from its own keys and the given width alone.
#pragma once

#ifdef __CUDACC__
#define FOA_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define FOA_HOST_DEVICE inline
#endif

namespace foa {

struct Parts {
  int width, count;  // keys of a part (at most the given width), parts
  FOA_HOST_DEVICE Parts(int keys, int keys_per_split, bool even)
      : width(keys_per_split), count((keys + keys_per_split - 1) / keys_per_split) {
    if (!even || count == 1 || keys_per_split % 128 != 0) return;
    const int tiles = (keys + 127) / 128, each = (tiles + count - 1) / count;
    width = 128 * each;
    count = (tiles + each - 1) / each;
  }
};

}  // namespace foa

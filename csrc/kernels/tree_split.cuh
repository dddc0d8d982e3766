// The parts of one history: keys_per_split keys each (mma.sync form), or as few as that allows and
// equally long in whole 128-key tiles (tcgen05 form, which holds an SM alone: a CTA with a short rest
// costs its set-up). A row's parts follow from its own keys and the given width alone.
#pragma once

namespace foa {

struct Parts {
  int width, count;  // keys of a part (at most the given width), parts
  __device__ __forceinline__ Parts(int keys, int keys_per_split, bool even) : width(keys_per_split) {
    count = (keys + keys_per_split - 1) / keys_per_split;
    if (!even || count == 1 || keys_per_split % 128 != 0 || keys >= 1 << 22) return;
    // At least keys / count, rounded up to tiles (the quotient is off by less than one).
    width = ((int)__fdividef((float)keys, (float)count) + 128) / 128 * 128;
    if (width > keys_per_split) width = keys_per_split;
    while ((count - 1) * width >= keys) --count;
  }
};

}  // namespace foa

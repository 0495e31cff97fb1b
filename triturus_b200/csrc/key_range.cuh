// Ranges of 32-bit keys that radix selection narrows down, 256 bins at a time; plain C++, so that it can be checked without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TB200_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TB200_HOST_DEVICE inline
#endif

namespace tb200 {

struct KeyRange {
  uint32_t lo, hi;  // both in it

  // Bins are of 2^shift() keys, at most 256 of them: 24, 16, 8 and 0 at the most in four rounds, the last of which leaves one key.
  TB200_HOST_DEVICE int shift() const {
    uint32_t d = (hi - lo) >> 8;  // the number of its digits
    int s = 0;
    for (int part = 16; part > 0; part /= 2) {
      const int more = d >> part != 0 ? part : 0;
      s += more;
      d >>= more;
    }
    return s + static_cast<int>(d);
  }
  // Bin `b` of those counted from lo upwards, or from hi downwards.  What is left of the range bounds the bin's other end: a sum or difference
  // with the bin's width leaves 32 bits near the ends of the keys.
  TB200_HOST_DEVICE KeyRange bin_upwards(uint32_t b, int s) const {
    const uint32_t first = lo + (b << s), width = (1u << s) - 1u;
    return {first, hi - first < width ? hi : first + width};
  }
  TB200_HOST_DEVICE KeyRange bin_downwards(uint32_t b, int s) const {
    const uint32_t last = hi - (b << s), width = (1u << s) - 1u;
    return {last - lo < width ? lo : last - width, last};
  }
};
constexpr int kKeyRounds = 4;

}  // namespace tb200

// Division by a number that the host knows; plain C++, so that it can be checked without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define TB200_DIVISOR_DEVICE __host__ __device__ __forceinline__
#else
#define TB200_DIVISOR_DEVICE inline
#endif

namespace tb200 {

// Quotients of numbers from 0 to 2^31 - 1 by a positive one, without the instructions of a division (four of which cost a tile of a matrix
// product 800 cycles): with 2^shift >= d, n / d = (n + floor(n m / 2^32)) / 2^shift for m = floor(2^32 (2^shift - d) / d) + 1.
struct Divisor {
  uint32_t mul, shift;
  Divisor() = default;
  explicit Divisor(int divisor) : mul(0), shift(0) {
    const uint64_t d = static_cast<uint32_t>(divisor);
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  TB200_DIVISOR_DEVICE int operator()(int n) const {
    const uint32_t u = static_cast<uint32_t>(n);
    return static_cast<int>((static_cast<uint32_t>((static_cast<uint64_t>(u) * mul) >> 32) + u) >> shift);
  }
};

}  // namespace tb200

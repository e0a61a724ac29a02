// Equal shares of a line of units: the integer arithmetic of the paged
// attention kernels, in plain C++ so that it also compiles without CUDA.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define Q6W_SHARE __host__ __device__ __forceinline__
#else
#define Q6W_SHARE inline
#endif

namespace q6w {
namespace paged {

// a b / c, in 32 bits when the product and the divisor fit (a 64-bit division is a long subroutine).
Q6W_SHARE int64_t muldiv(int64_t a, int64_t b, int64_t c) {
  const int64_t p = a * b;
  return ((p | c) >> 32) == 0 ? (int64_t)((uint32_t)p / (uint32_t)c) : p / c;
}

// Worker w holds units [w units / workers, (w + 1) units / workers): the one that
// holds `unit`.  (The dividend is at least `units`: if it fits 32 bits, so does the divisor.)
Q6W_SHARE int64_t owner_of(int64_t unit, int64_t units, int64_t workers) {
  const int64_t p = (unit + 1) * workers + units - 1;
  return ((p >> 32) == 0 ? (int64_t)((uint32_t)p / (uint32_t)units) : p / units) - 1;
}

}  // namespace paged
}  // namespace q6w

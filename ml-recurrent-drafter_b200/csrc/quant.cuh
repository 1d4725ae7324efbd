// What the kernels of a cache in codes of 8 or 4 bits, and of products of 8-bit integers, share.  A row's parameters are 32 bits: the bf16 pattern of its scale below, its
// zero (0 .. 255) above; see cache_quant.cu for what they mean.
#pragma once
#include <atomic>
#include <type_traits>

#include "rd_common.cuh"

namespace rd_quant {

constexpr uint32_t kNanScale = 0x7fffu;  // scale of a row that held NaN or infinities

__device__ __forceinline__ float param_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ uint32_t param_zero(uint32_t p) { return p >> 16; }
// an integer below 2^23 as fp32: exact, two instructions of the full rate
__device__ __forceinline__ float code_as_float(uint32_t c) { return __uint_as_float(0x4b000000u | c) - 8388608.f; }

// max / min that pass NaN on
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// rint(x / scale) for a scale of 8 significant bits and |x / scale| < 2^22 (256 for Bits8), as the bits of 12582912 + it: subtract kRintBias for
// the integer.
// x of up to 24 bits: q = x r is within two units of the quotient; what is left, x - q scale, has few bits and is exact, so the second step
// gives the quotient rounded once but for an error of 2^-46: quotients half way between two integers come out exactly, and others are
// further from half way than half a unit (cache_quant.cu), by 2^-9 of it at least.
// x of 8 bits (Bits8): a quotient that is not half way is 2^-9 or more away from there, for then 2 x - (2 k + 1) scale is at least the last place of
// the scale; x r is off by 2^-15 at most, and rounded to a multiple of 2^-10, which adding 1.5 2^13 does, it is half way where the quotient is.
// The compiler's division takes some ten instructions and was what the quantising kernels spent their time on (20235 tokens of 8
// heads: 63 us, 40 with four, now two for bf16).
template <bool Bits8>
struct Divider {
  float scale, inverse;
  bool fast;  // neither the inverse nor what is left leaves fp32's normal range
  __device__ __forceinline__ explicit Divider(float s) : scale(s), inverse(1.f / s), fast(s >= 0x1p-100f && s <= 0x1p100f) {}
  __device__ __forceinline__ uint32_t rint_bits(float x) const {
    if (!fast) return __float_as_uint(x / scale + 12582912.f);
    if constexpr (Bits8) return __float_as_uint(fmaf(x, inverse, 12288.f) + (12582912.f - 12288.f));
    float q = x * inverse;
    q = fmaf(fmaf(-q, scale, x), inverse, q);
    return __float_as_uint(q + 12582912.f);
  }
};
constexpr uint32_t kRintBias = 0x4b400000u;

// Lets a kernel have its dynamic shared memory on the current device, and as many CTAs on an SM as fit into that; once for each.  (Without the
// second attribute two CTAs of 99 KB were never placed on one SM.)
template <auto Kernel>
bool allow_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return true;
  cudaError_t err = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess) err = cudaFuncSetAttribute(Kernel, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared);
  if (err != cudaSuccess) {
    rd_set_last_cuda_error((int)err);
    return false;
  }
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
inline int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && v > 0 ? v : 148;
  }();
  return n;
}

}  // namespace rd_quant

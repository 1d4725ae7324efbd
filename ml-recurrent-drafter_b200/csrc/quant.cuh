// What the kernels of a cache in codes of 8 or 4 bits share.  A row's parameters are 32 bits: the bf16 pattern of its scale below, its
// zero (0 .. 255) above; see cache_quant.cu for what they mean.
#pragma once
#include <type_traits>

#include "rd_common.cuh"

namespace rd_quant {

constexpr uint32_t kNanScale = 0x7fffu;  // scale of a row that held NaN or infinities

__device__ __forceinline__ float param_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ uint32_t param_zero(uint32_t p) { return p >> 16; }
// an integer below 2^23 as fp32: exact, two instructions of the full rate
__device__ __forceinline__ float code_as_float(uint32_t c) { return __uint_as_float(0x4b000000u | c) - 8388608.f; }

}  // namespace rd_quant

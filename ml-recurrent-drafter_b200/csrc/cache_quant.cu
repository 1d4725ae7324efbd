// A key/value cache held in codes of 8 or 4 bits: quantising rows as they are written, reading them back.
//
// A row (one token's key or value of one head, hd features x) with Q = 2^bits - 1, low = min(0, min x), high = max(0, max x):
//   scale = bf16((high - low) / Q),  zero = rint(-low / scale),  code = rint(x / scale) + zero,  both cut to 0 .. Q;
// a code stands for scale * (code - zero).  Rows with NaN or infinities, or whose range passes fp32's, get a scale of NaN.
// The scale has 8 significant bits, so that fp32's division gives the codes of exact arithmetic: a value half way between two codes,
// scale * (k + 1/2), has at most 17 significant bits and lies on the grid of the fp32 numbers around it, hence x is such a value or at
// least a unit of its last place away from it, and a quotient that far away does not round to k + 1/2.
#include "quant.cuh"

namespace {

using namespace rd_quant;

constexpr int kThreads = 256;
constexpr int kVec = 8;  // features of a lane

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + 4);
  }
}

// One row by `lanes` lanes (a power of two), 8 features each; lanes past hd hold zeros, which change no range.
template <int BITS>
__device__ __forceinline__ void quantise_row(const float* x, int lanes, bool mine, bool first, uint8_t* codes, uint32_t* param) {
  constexpr float kQ = (float)((1 << BITS) - 1);
  float low = 0.f, high = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    low = fminf(low, x[i]);
    high = fmaxf(high, x[i]);
    odd |= !(fabsf(x[i]) <= 3.402823466e38f);
  }
  if (odd) high = INFINITY;
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const float range = high - low;
  __nv_bfloat16 s = __float2bfloat16_rn(range / kQ);
  const bool fine = range <= 3.402823466e38f;
  const float scale = __bfloat162float(s);
  const bool some = fine && scale > 0.f;
  const float zero = some ? fminf(rintf(-low / scale), kQ) : 0.f;
  uint32_t c[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) c[i] = some ? (uint32_t)fminf(fmaxf(rintf(x[i] / scale) + zero, 0.f), kQ) : 0u;
  if (mine) {
    if constexpr (BITS == 4) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) w |= c[i] << (4 * i);
      *reinterpret_cast<uint32_t*>(codes) = w;
    } else {
      uint2 w = make_uint2(0u, 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) w.x |= c[i] << (8 * i), w.y |= c[4 + i] << (8 * i);
      *reinterpret_cast<uint2*>(codes) = w;
    }
  }
  if (first) *param = (uint32_t)(fine ? __bfloat16_as_ushort(s) : (unsigned short)kNanScale) | ((uint32_t)zero << 16);
}

struct Planes {
  uint8_t *k_codes, *v_codes;
  uint32_t *k_params, *v_params;
};

// A unit is one head of one token, its key and its value.  Bound by memory: hd values read and hd * BITS / 8 + 4 bytes written for
// each of the two.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) cache_quant_append_kernel(const T* k, const T* v, int64_t tok_stride, int64_t head_stride, Planes to,
                                                                      const int32_t* tok_row, const int32_t* tok_slot, int m_max,
                                                                      const int32_t* m_dev, int B, int nkv, int hd, int max_len, int lanes) {
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int64_t units = (int64_t)rd::live_rows(m_dev, m_max) * nkv;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
  const int part = threadIdx.x & (lanes - 1), d = part * kVec;
  bool live = unit < units;
  const int64_t t = live ? unit / nkv : 0;
  const int head = (int)(unit - t * nkv);
  int row = 0, slot = 0;
  if (live) {
    row = tok_row[t];
    slot = tok_slot[t];
    live = row >= 0 && row < B && slot >= 0 && slot < max_len;
  }
  const bool mine = live && d < hd;
  float xk[kVec] = {}, xv[kVec] = {};
  if (mine) {
    const int64_t from = t * tok_stride + head * head_stride + d;
    load8(k + from, xk);
    load8(v + from, xv);
  }
  const int64_t at = ((int64_t)row * nkv + head) * max_len + slot;  // row of the planes
  const int64_t byte = at * (hd * BITS / 8) + d * BITS / 8;
  quantise_row<BITS>(xk, lanes, mine, live && part == 0, to.k_codes + byte, to.k_params + at);
  quantise_row<BITS>(xv, lanes, mine, live && part == 0, to.v_codes + byte, to.v_params + at);
}

// Eight codes as the values that they stand for.
template <int BITS>
__device__ __forceinline__ void values8(const uint8_t* codes, uint32_t param, float* x) {
  const float scale = param_scale(param), zero = (float)param_zero(param);
  if constexpr (BITS == 4) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = scale * (code_as_float((w >> (4 * i)) & 15u) - zero);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(codes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = scale * (code_as_float((w.x >> (8 * i)) & 255u) - zero);
      x[4 + i] = scale * (code_as_float((w.y >> (8 * i)) & 255u) - zero);
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 2) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  } else {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
    *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(x + 4);
  }
}

constexpr int kReadRows = 4;  // rows of a thread

// grid: x = blocks of rows, y = heads of all batch rows, keys first, then values
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) cache_quant_read_kernel(Planes from, const int32_t* begin, const int32_t* length, int nkv, int hd,
                                                                    int max_len, T* k_out, T* v_out, int out_len, int chains) {
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  for (int64_t y = blockIdx.y; y < 2 * (int64_t)chains; y += gridDim.y) {
    const bool value = y >= chains;
    const int64_t chain = value ? y - chains : y;
    const int b = (int)(chain / nkv);
    const int first = begin[b];
    // rows outside the cache or the output do not exist
    const int n = min(min(length[b], out_len), max_len - max(first, 0));
    const uint8_t* codes = value ? from.v_codes : from.k_codes;
    const uint32_t* params = value ? from.v_params : from.k_params;
    T* out = (value ? v_out : k_out) + chain * out_len * hd;
    const int vecs = hd / kVec;
    const int64_t work = (int64_t)n * vecs, step = (int64_t)gridDim.x * kThreads;
    if (first < 0) continue;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < work; i += step) {
      const int64_t j = i / vecs;
      const int d = (int)(i - j * vecs) * kVec;
      const int64_t at = chain * max_len + first + j;
      float x[kVec];
      values8<BITS>(codes + at * (hd * BITS / 8) + d * BITS / 8, params[at], x);
      store8(out + j * hd + d, x);
    }
  }
}

// The accepted path of a draft: slot base_len[b] + unpacker[b, seq, j] moves to base_len[b] + j.  A thread moves its own columns, row
// after row, so that no barrier is needed between the rows.  grid: x = heads, y = batch rows, z = planes
__global__ void __launch_bounds__(kThreads / 2) cache_quant_commit_kernel(uint8_t* codes, uint32_t* params, int B, int nkv, int max_len, int row_words,
                                                                     const int32_t* kv_begin, const int32_t* base_len, const int32_t* unpacker, int W,
                                                                     int Lb, const int32_t* n_accepted, const int32_t* seq_in_beam) {
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int b = blockIdx.y;
  const int32_t* u = unpacker + ((int64_t)b * W + seq_in_beam[b]) * Lb;
  const int64_t first = (((int64_t)blockIdx.z * B + b) * nkv + blockIdx.x) * max_len + kv_begin[b] + base_len[b];
  const int n = n_accepted[b], w = threadIdx.x;
  if (w > row_words) return;
  uint32_t* rows = w < row_words ? reinterpret_cast<uint32_t*>(codes) + first * row_words + w : params + first;
  const int64_t step = w < row_words ? row_words : 1;
  for (int j = 0; j <= n && j < Lb; ++j)
    if (u[j] != j) rows[j * step] = rows[u[j] * step];
}

int check_layout(int bits, int B, int nkv, int hd, int max_len) {
  RD_REQUIRE(bits == 4 || bits == 8, RD_ERR_UNSUPPORTED);
  RD_REQUIRE(B >= 0 && nkv >= 1 && max_len >= 1, RD_ERR_ARG);
  RD_REQUIRE(hd >= 8 && hd <= 256 && hd % 8 == 0, RD_ERR_SIZE);
  return RD_OK;
}

}  // namespace

extern "C" int rd_cache_quant_append(int dtype, int bits, const void* k, const void* v, int64_t tok_stride, int64_t head_stride,
                                     uint8_t* k_codes, void* k_params, uint8_t* v_codes, void* v_params, const int32_t* tok_row,
                                     const int32_t* tok_slot, int m_max, const int32_t* m_dev, int B, int nkv, int hd, int max_len,
                                     void* stream) {
  RD_REQUIRE(dtype == RD_F32 || dtype == RD_BF16, RD_ERR_DTYPE);
  int rc = check_layout(bits, B, nkv, hd, max_len);
  if (rc != RD_OK) return rc;
  RD_REQUIRE(m_max >= 0 && tok_stride >= 0 && head_stride >= 0, RD_ERR_ARG);
  if (m_max == 0 || B == 0) return RD_OK;
  RD_REQUIRE(k && v && k_codes && k_params && v_codes && v_params && tok_row && tok_slot, RD_ERR_ARG);
  const int esz = dtype == RD_BF16 ? 2 : 4;
  RD_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (tok_stride * esz) % 16 == 0 && (head_stride * esz) % 16 == 0, RD_ERR_ALIGN);
  RD_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0, RD_ERR_ALIGN);
  int lanes = 1;
  while (lanes * kVec < hd) lanes *= 2;
  const int64_t blocks = ((int64_t)m_max * nkv * lanes + kThreads - 1) / kThreads;
  RD_REQUIRE(blocks <= 0x7fffffff, RD_ERR_SIZE);
  const Planes to{k_codes, v_codes, (uint32_t*)k_params, (uint32_t*)v_params};
  cudaError_t err;
  auto run = [&](auto kern, auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    err = rd::launch_chained(kern, dim3((unsigned)blocks), dim3(kThreads), 0, (cudaStream_t)stream, 1, (const T*)k, (const T*)v, tok_stride, head_stride, to,
                             tok_row, tok_slot, m_max, m_dev, B, nkv, hd, max_len, lanes);
  };
  if (dtype == RD_BF16) bits == 4 ? run(cache_quant_append_kernel<__nv_bfloat16, 4>, (__nv_bfloat16*)nullptr) : run(cache_quant_append_kernel<__nv_bfloat16, 8>, (__nv_bfloat16*)nullptr);
  else bits == 4 ? run(cache_quant_append_kernel<float, 4>, (float*)nullptr) : run(cache_quant_append_kernel<float, 8>, (float*)nullptr);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

extern "C" int rd_cache_quant_read(int dtype, int bits, const uint8_t* k_codes, const void* k_params, const uint8_t* v_codes, const void* v_params,
                                   const int32_t* begin, const int32_t* length, int B, int nkv, int hd, int max_len, void* k_out, void* v_out,
                                   int out_len, void* stream) {
  RD_REQUIRE(dtype == RD_F32 || dtype == RD_BF16, RD_ERR_DTYPE);
  int rc = check_layout(bits, B, nkv, hd, max_len);
  if (rc != RD_OK) return rc;
  RD_REQUIRE(out_len >= 0, RD_ERR_ARG);
  if (B == 0 || out_len == 0) return RD_OK;
  RD_REQUIRE(k_codes && k_params && v_codes && v_params && begin && length && k_out && v_out, RD_ERR_ARG);
  RD_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
             RD_ERR_ALIGN);
  const int64_t chains = (int64_t)B * nkv;
  RD_REQUIRE(chains <= 0x3fffffff, RD_ERR_SIZE);
  const int64_t vecs = (int64_t)out_len * (hd / kVec);
  const unsigned gx = (unsigned)((vecs + kThreads * kReadRows - 1) / (kThreads * kReadRows));
  const unsigned gy = (unsigned)(2 * chains < 65535 ? 2 * chains : 65535);
  const Planes from{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params};
  cudaError_t err;
  auto run = [&](auto kern, auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    err = rd::launch_chained(kern, dim3(gx, gy), dim3(kThreads), 0, (cudaStream_t)stream, 1, from, begin, length, nkv, hd, max_len, (T*)k_out, (T*)v_out, out_len,
                             (int)chains);
  };
  if (dtype == RD_BF16) bits == 4 ? run(cache_quant_read_kernel<__nv_bfloat16, 4>, (__nv_bfloat16*)nullptr) : run(cache_quant_read_kernel<__nv_bfloat16, 8>, (__nv_bfloat16*)nullptr);
  else bits == 4 ? run(cache_quant_read_kernel<float, 4>, (float*)nullptr) : run(cache_quant_read_kernel<float, 8>, (float*)nullptr);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

extern "C" int rd_cache_quant_commit(int bits, uint8_t* codes, void* params, int planes, int B, int nkv, int max_len, int hd,
                                     const int32_t* kv_begin, const int32_t* base_len, const int32_t* unpacker, int W, int Lb,
                                     const int32_t* n_accepted, const int32_t* seq_in_beam, void* stream) {
  const int rc = check_layout(bits, B, nkv, hd, max_len);
  if (rc != RD_OK) return rc;
  RD_REQUIRE(codes && params && kv_begin && base_len && unpacker && n_accepted && seq_in_beam, RD_ERR_ARG);
  RD_REQUIRE(B >= 1 && B <= 65535 && planes >= 1 && planes <= 65535 && W >= 1 && Lb >= 1, RD_ERR_SIZE);
  RD_REQUIRE((((uintptr_t)codes | (uintptr_t)params) & 15) == 0, RD_ERR_ALIGN);
  const int words = hd * bits / 32;  // at most 64, and one thread more for the parameters
  static_assert(256 / 4 + 1 <= kThreads / 2, "one column a thread");
  cudaError_t err = rd::launch_chained(cache_quant_commit_kernel, dim3(nkv, B, planes), dim3(kThreads / 2), 0, (cudaStream_t)stream, 1, codes, (uint32_t*)params,
                                       B, nkv, max_len, words, kv_begin, base_len, unpacker, W, Lb, n_accepted, seq_in_beam);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

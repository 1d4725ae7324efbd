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

__device__ __forceinline__ uint32_t max_nan2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ uint32_t min_nan2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// A lane's VEC features of a row, as they lie
template <typename T, int VEC>
struct Piece {
  static constexpr int kWords = VEC * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(w + i) = *reinterpret_cast<const uint4*>(p + i * 4 / sizeof(T));
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
  }
  // widens [low, high]; NaN stays
  __device__ __forceinline__ void range(float& low, float& high) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) low = min_nan(low, value(i)), high = max_nan(high, value(i));
    } else {
      uint32_t l = 0, h = 0;
#pragma unroll
      for (int i = 0; i < kWords; ++i) l = min_nan2(l, w[i]), h = max_nan2(h, w[i]);
      low = min_nan(low, min_nan(__uint_as_float(l << 16), __uint_as_float(l & 0xffff0000u)));
      high = max_nan(high, max_nan(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)));
    }
  }
};

// One row by `lanes` lanes (a power of two); lanes past hd hold zeros, which change no range.
template <int BITS, typename T, int VEC>
__device__ __forceinline__ void quantise_row(const Piece<T, VEC>& x, int lanes, bool mine, bool first, uint8_t* codes, uint32_t* param) {
  constexpr int kQ = (1 << BITS) - 1;
  float low = 0.f, high = 0.f;
  x.range(low, high);
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const float range = high - low;
  const bool fine = range <= 3.402823466e38f;  // not so for NaN either
  const __nv_bfloat16 s = __float2bfloat16_rn(range / (float)kQ);
  const float scale = __bfloat162float(s);
  const bool some = fine && scale > 0.f;
  const Divider<sizeof(T) == 2> by(some ? scale : 1.f);
  const int zero = some ? min((int)(by.rint_bits(-low) - kRintBias), kQ) : 0;
  uint32_t w[VEC * BITS / 32];
#pragma unroll
  for (int i = 0; i < VEC * BITS / 32; ++i) w[i] = 0;
  if (some) {
    const int shift = zero - (int)kRintBias;
#pragma unroll
    for (int i = 0; i < VEC; ++i)  // cut to 0 .. Q, added up by multiplications
      w[i * BITS / 32] += (uint32_t)__vimin_s32_relu((int)by.rint_bits(x.value(i)) + shift, kQ) * (1u << (i * BITS % 32));
  }
  if (mine) {
    if constexpr (VEC * BITS == 32) *reinterpret_cast<uint32_t*>(codes) = w[0];
    else if constexpr (VEC * BITS == 64) *reinterpret_cast<uint2*>(codes) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(codes) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (first) *param = (fine ? (uint32_t)__bfloat16_as_ushort(s) : kNanScale) | ((uint32_t)zero << 16);
}

struct Planes {
  uint8_t *k_codes, *v_codes;
  uint32_t *k_params, *v_params;
};

// A unit is one head of one token, its key and its value, by hd / VEC lanes (rounded up to a power of two).  Bound by memory for fp32 rows (20235 tokens of
// 8 heads of 128 at 8 bits: 38 us, 5.5 TB/s) and by instructions for bf16 ones (31.5 us, 4.0 TB/s; at 4 bits 30; issue slots 74 %, the integer pipe 60, memory
// 34): two a quotient, one for its cut, one to put its code in place.  CTAs that go through several units each with the next one's rows under way: 63 to 125 us instead of 57, appended and read.
template <typename T, int BITS, int VEC>
__global__ void __launch_bounds__(kThreads) cache_quant_append_kernel(const T* k, const T* v, int64_t tok_stride, int64_t head_stride, Planes to,
                                                                      const int32_t* tok_row, const int32_t* tok_slot, int m_max,
                                                                      const int32_t* m_dev, int B, int nkv, int hd, int max_len, int lanes) {
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const uint32_t units = (uint32_t)rd::live_rows(m_dev, m_max) * (uint32_t)nkv;
  const uint32_t unit = blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const int part = threadIdx.x & (lanes - 1), d = part * VEC;
  bool live = unit < units;
  const uint32_t t = live ? unit / (uint32_t)nkv : 0;
  const int head = live ? (int)(unit - t * nkv) : 0;
  const bool mine = live && d < hd;
  Piece<T, VEC> xk, xv;
  xk.clear();
  xv.clear();
  if (mine) {
    const int64_t from = (int64_t)t * tok_stride + head * head_stride + d;
    xk.load(k + from);
    xv.load(v + from);
  }
  int row = 0, slot = 0;
  if (live) {
    row = tok_row[t];
    slot = tok_slot[t];
    live = row >= 0 && row < B && slot >= 0 && slot < max_len;
  }
  const int64_t at = ((int64_t)row * nkv + head) * max_len + slot;  // row of the planes
  const int64_t byte = at * (hd * BITS / 8) + d * BITS / 8;
  quantise_row<BITS>(xk, lanes, mine && live, live && part == 0, to.k_codes + byte, to.k_params + at);
  quantise_row<BITS>(xv, lanes, mine && live, live && part == 0, to.v_codes + byte, to.v_params + at);
}

constexpr int kReadThreads = 128, kReadRows = 4;  // a step: kReadRows rows of a thread, all asked for before the first is written
constexpr int kReadSteps = 16;                    // at most, of a CTA

// grid: x = blocks of rows, y = heads of all batch rows, keys first, then values.  A lane has 16 bytes of the output.  A CTA goes through its steps with
// the codes of the next under way while it writes one: 71321 tokens of 32 heads of 128 features at 4 bits take 310 us with a CTA for each step of 128
// rows and 243 with this (6.1 TB/s); 8192 + 12043 tokens of 8 heads, appended and read, 63 and 54.
template <typename T, int BITS>
__global__ void __launch_bounds__(kReadThreads) cache_quant_read_kernel(Planes from, const int32_t* begin, const int32_t* length, int nkv, int hd,
                                                                        int max_len, T* k_out, T* v_out, int out_len, int chains, int lanes) {
  constexpr int VEC = 16 / (int)sizeof(T);
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int rows = kReadThreads / lanes, part = threadIdx.x & (lanes - 1), d = part * VEC;
  const int row_bytes = hd * BITS / 8;
  if (d >= hd) return;
  for (int64_t y = blockIdx.y; y < 2 * (int64_t)chains; y += gridDim.y) {
    const bool value = y >= chains;
    const int64_t chain = value ? y - chains : y;
    const int b = (int)((uint32_t)chain / (uint32_t)nkv);
    const int first = begin[b];
    // rows outside the cache or the output do not exist
    const int n = first < 0 ? 0 : min(min(length[b], out_len), max_len - first);
    const uint8_t* codes = (value ? from.v_codes : from.k_codes) + (chain * max_len + first) * row_bytes + d * BITS / 8;
    const uint32_t* params = (value ? from.v_params : from.k_params) + chain * max_len + first;
    T* out = (value ? v_out : k_out) + chain * out_len * hd + d;
    uint32_t w[2][kReadRows][2], p[2][kReadRows];
    auto ask = [&](auto set, int64_t j0) {
      constexpr int S = decltype(set)::value;
#pragma unroll
      for (int i = 0; i < kReadRows; ++i) {
        const int64_t j = j0 + i * rows;
        if (j >= n) continue;
        const uint8_t* c = codes + j * row_bytes;
        if constexpr (VEC * BITS == 16) w[S][i][0] = *reinterpret_cast<const uint16_t*>(c);
        else w[S][i][0] = *reinterpret_cast<const uint32_t*>(c);
        if constexpr (VEC * BITS == 64) w[S][i][1] = *reinterpret_cast<const uint32_t*>(c + 4);
        p[S][i] = params[j];
      }
    };
    auto put = [&](auto set, int64_t j0) {
      constexpr int S = decltype(set)::value;
#pragma unroll
      for (int i = 0; i < kReadRows; ++i) {
        const int64_t j = j0 + i * rows;
        if (j >= n) continue;
        const float scale = param_scale(p[S][i]), zero = 8388608.f + (float)param_zero(p[S][i]);
        float x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const uint32_t c = (w[S][i][e * BITS / 32] >> (e * BITS % 32)) & ((1u << BITS) - 1);
          x[e] = scale * (__uint_as_float(0x4b000000u | c) - zero);  // both sums exact
        }
        if constexpr (sizeof(T) == 2) {
          __nv_bfloat162 h[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
          *reinterpret_cast<uint4*>(out + j * hd) = *reinterpret_cast<const uint4*>(h);
        } else {
          *reinterpret_cast<float4*>(out + j * hd) = *reinterpret_cast<const float4*>(x);
        }
      }
    };
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    const int64_t step = (int64_t)gridDim.x * rows * kReadRows;
    int64_t j = (int64_t)blockIdx.x * rows * kReadRows + threadIdx.x / lanes;
    ask(Even(), j);
    for (; j < n; j += 2 * step) {
      ask(Odd(), j + step);
      put(Even(), j);
      ask(Even(), j + 2 * step);
      put(Odd(), j + step);
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
  const int seq = seq_in_beam[b];
  const int64_t slot0 = (int64_t)kv_begin[b] + base_len[b];
  if (seq < 0 || seq >= W || slot0 < 0) return;
  const int32_t* u = unpacker + ((int64_t)b * W + seq) * Lb;
  const int64_t first = (((int64_t)blockIdx.z * B + b) * nkv + blockIdx.x) * max_len + slot0, places = max_len - slot0;  // slots outside the cache do not exist
  const int n = n_accepted[b], w = threadIdx.x;
  if (w > row_words) return;
  uint32_t* rows = w < row_words ? reinterpret_cast<uint32_t*>(codes) + first * row_words + w : params + first;
  const int64_t step = w < row_words ? row_words : 1;
  for (int j = 0; j <= n && j < Lb; ++j)
    if (u[j] > j && u[j] < places) rows[j * step] = rows[u[j] * step];
}

int check_layout(int bits, int B, int nkv, int hd, int max_len) {
  RD_REQUIRE(bits == 4 || bits == 8, RD_ERR_UNSUPPORTED);
  RD_REQUIRE(B >= 0 && nkv >= 1 && max_len >= 1, RD_ERR_ARG);
  RD_REQUIRE(hd >= 8 && hd <= 256 && hd % 8 == 0, RD_ERR_SIZE);
  return RD_OK;
}

}  // namespace

extern "C" int rd_cache_quant_append(const rd_cache_quant_append_desc* desc, void* stream) {
  RD_REQUIRE(desc, RD_ERR_ARG);
  const auto [k, v, tok_stride, head_stride, k_codes, k_params, v_codes, v_params, tok_row, tok_slot, m_dev, dtype, bits, m_max, B, nkv, hd, max_len] = *desc;
  RD_REQUIRE(dtype == RD_F32 || dtype == RD_BF16, RD_ERR_DTYPE);
  int rc = check_layout(bits, B, nkv, hd, max_len);
  if (rc != RD_OK) return rc;
  RD_REQUIRE(m_max >= 0 && tok_stride >= 0 && head_stride >= 0, RD_ERR_ARG);
  if (m_max == 0 || B == 0) return RD_OK;
  RD_REQUIRE(k && v && k_codes && k_params && v_codes && v_params && tok_row && tok_slot, RD_ERR_ARG);
  const int esz = dtype == RD_BF16 ? 2 : 4;
  RD_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && (tok_stride * esz) % 16 == 0 && (head_stride * esz) % 16 == 0, RD_ERR_ALIGN);
  RD_REQUIRE((((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0, RD_ERR_ALIGN);
  const int vec = hd % 16 == 0 ? 16 : 8;
  int lanes = 1;
  while (lanes * vec < hd) lanes *= 2;
  RD_REQUIRE((int64_t)m_max * nkv <= 0x7fffffff - kThreads, RD_ERR_SIZE);
  const int64_t blocks = ((int64_t)m_max * nkv + kThreads / lanes - 1) / (kThreads / lanes);
  const Planes to{k_codes, v_codes, (uint32_t*)k_params, (uint32_t*)v_params};
  cudaError_t err;
  auto run = [&](auto kern, auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    err = rd::launch_chained(kern, dim3((unsigned)blocks), dim3(kThreads), 0, (cudaStream_t)stream, 1, (const T*)k, (const T*)v, tok_stride, head_stride, to,
                             tok_row, tok_slot, m_max, m_dev, B, nkv, hd, max_len, lanes);
  };
  auto pick = [&](auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    if (vec == 16) bits == 4 ? run(cache_quant_append_kernel<T, 4, 16>, zero) : run(cache_quant_append_kernel<T, 8, 16>, zero);
    else bits == 4 ? run(cache_quant_append_kernel<T, 4, 8>, zero) : run(cache_quant_append_kernel<T, 8, 8>, zero);
  };
  if (dtype == RD_BF16) pick((__nv_bfloat16*)nullptr);
  else pick((float*)nullptr);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

extern "C" int rd_cache_quant_read(const rd_cache_quant_read_desc* desc, void* stream) {
  RD_REQUIRE(desc, RD_ERR_ARG);
  const auto [k_codes, k_params, v_codes, v_params, begin, length, k_out, v_out, dtype, bits, B, nkv, hd, max_len, out_len] = *desc;
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
  int lanes = 1;
  while (lanes * (dtype == RD_BF16 ? 8 : 4) < hd) lanes *= 2;
  const int rows = kReadThreads / lanes * kReadRows;
  const int64_t gy = 2 * chains < 65535 ? 2 * chains : 65535, all = ((int64_t)out_len + rows - 1) / rows;  // steps of a chain
  // as many steps to a CTA as leave sixteen CTAs for each SM
  int64_t steps = all * gy / (16 * rd_quant::sm_count());
  steps = steps < 1 ? 1 : steps > kReadSteps ? kReadSteps : steps;
  const int64_t gx = (all + steps - 1) / steps;
  const Planes from{(uint8_t*)k_codes, (uint8_t*)v_codes, (uint32_t*)k_params, (uint32_t*)v_params};
  cudaError_t err;
  auto run = [&](auto kern, auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    err = rd::launch_chained(kern, dim3((unsigned)gx, (unsigned)gy), dim3(kReadThreads), 0, (cudaStream_t)stream, 1, from, begin, length, nkv, hd, max_len, (T*)k_out, (T*)v_out, out_len,
                             (int)chains, lanes);
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

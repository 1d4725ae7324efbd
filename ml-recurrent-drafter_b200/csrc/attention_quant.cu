// Attention over a key/value cache held in codes of 8 or 4 bits (cache_quant.cu): softmax(scale Q K^T) V with
// K = scale_k (code - zero_k), V likewise, a scale and a zero for each token of a head.
//
// attention_quant_rows_kernel: one CTA per (new token, head).  A warp
// takes 32 keys at a time, a key each for the scores, then all of them together for the values, a lane some features; running
// maximum and sum in fp32.  The score is scale_k (q . code - zero_k sum q), the value's weight p scale_v.
#include "quant.cuh"

namespace {

using namespace rd_quant;

constexpr int kWarps = 4;
constexpr int kMaxHd = 256;

struct Args {
  const void* q;
  int64_t ldq;
  const uint8_t *k_codes, *v_codes;
  const uint32_t *k_params, *v_params;
  void* out;
  const int32_t *row_start, *kv_begin, *base_len;
  int m_max, B, nh, nkv, hd, max_len, max_new, max_kv, mode;
  const uint32_t* tree_mask;
  int mask_words;
  float scale;
};

// Keys of a batch row: those before `base` are seen by all of its new tokens, n_new more among themselves.
struct Row {
  int start, n_new, first, base, end;  // end: base + n_new, cut to the cache
};
__device__ __forceinline__ Row row_of(const Args& a, int b) {
  Row r;
  r.start = a.row_start[b];
  r.n_new = min(a.row_start[b + 1] - r.start, a.max_new);
  r.first = max(a.kv_begin[b], 0);
  r.base = max(a.base_len[b], 0);
  if (r.start < 0 || r.start + r.n_new > a.m_max) r.n_new = 0;
  // what the caller bounded it by, whatever the row says: workspaces are sized by it
  r.end = min(min(r.base + r.n_new, a.max_len - r.first), a.max_kv);
  return r;
}
// does new token i of a row see its key j (j >= base)?
__device__ __forceinline__ bool sees(const Args& a, const Row& r, int i, int j) {
  const int jn = j - r.base;
  if (a.mode == RD_ATTN_CAUSAL) return jn <= i;
  return (jn >> 5) < a.mask_words && ((a.tree_mask[(int64_t)(r.start + i) * a.mask_words + (jn >> 5)] >> (jn & 31)) & 1u);
}

template <typename T, int BITS>
__global__ void __launch_bounds__(kWarps * 32) attention_quant_rows_kernel(const Args a) {
  __shared__ float q[kMaxHd], o[kWarps][kMaxHd], stats[kWarps][2];
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Row r = row_of(a, b);
  if (i >= r.n_new) return;
  const int hd = a.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* from = (const T*)a.q + (int64_t)(r.start + i) * a.ldq + (int64_t)h * hd;
  for (int d = threadIdx.x; d < hd; d += kWarps * 32) q[d] = rd::Num<T>::to_f(from[d]);
  __syncthreads();
  float q_sum = 0.f;
  for (int d = lane; d < hd; d += 32) q_sum += q[d];
  q_sum = rd::warp_sum(q_sum);
  const int64_t plane = ((int64_t)b * a.nkv + h / (a.nh / a.nkv)) * a.max_len + r.first;
  const int row_bytes = hd * BITS / 8;
  constexpr int kPer = 8 / BITS;  // codes of a byte
  float m = -INFINITY, l = 0.f, acc[kMaxHd / 32] = {};
  for (int j0 = warp * 32; j0 < r.end; j0 += kWarps * 32) {
    const int j = j0 + lane;
    const bool seen = j < r.end && (j < r.base || sees(a, r, i, j));
    float s = -INFINITY, sv = 0.f, zv = 0.f;
    if (seen) {
      const uint32_t pk = a.k_params[plane + j], pv = a.v_params[plane + j];
      const uint8_t* k = a.k_codes + (plane + j) * row_bytes;
      float dot = 0.f;
      for (int w = 0; w < row_bytes / 4; ++w) {
        const uint32_t u = reinterpret_cast<const uint32_t*>(k)[w];
#pragma unroll
        for (int e = 0; e < 4 * kPer; ++e) dot = fmaf(q[w * 4 * kPer + e], code_as_float((u >> (BITS * e)) & ((1u << BITS) - 1)), dot);
      }
      s = (dot - (float)param_zero(pk) * q_sum) * param_scale(pk) * a.scale;
      sv = param_scale(pv);
      zv = (float)param_zero(pv);
    }
    const bool any_nan = __any_sync(0xffffffffu, s != s);
    const float top = any_nan ? __int_as_float(0x7fffffff) : fmaxf(m, rd::warp_max(s));
    if (top == -INFINITY) continue;
    const float keep = m == -INFINITY ? 0.f : expf(m - top);
    const float p = seen ? expf(s - top) : 0.f;
    l = l * keep + rd::warp_sum(p);
    m = top;
    const float pw = seen ? p * sv : 0.f;
#pragma unroll
    for (int c = 0; c < kMaxHd / 32; ++c) acc[c] *= keep;
    const int n = min(32, r.end - j0);
    for (int x = 0; x < n; ++x) {
      const float w = __shfl_sync(0xffffffffu, pw, x), z = __shfl_sync(0xffffffffu, zv, x);
      if (w == 0.f) continue;
      const uint8_t* v = a.v_codes + (plane + j0 + x) * row_bytes;
#pragma unroll
      for (int c = 0; c < kMaxHd / 32; ++c) {
        const int d = c * 32 + lane;
        if (d < hd) acc[c] = fmaf(w, code_as_float((v[d / kPer] >> (BITS * (d % kPer))) & ((1u << BITS) - 1)) - z, acc[c]);
      }
    }
  }
  if (lane == 0) stats[warp][0] = m, stats[warp][1] = l;
#pragma unroll
  for (int c = 0; c < kMaxHd / 32; ++c) o[warp][c * 32 + lane] = acc[c];
  __syncthreads();
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, stats[w][0]), nan |= stats[w][0] != stats[w][0];
  float sum = 0.f, f[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    f[w] = stats[w][0] == -INFINITY ? 0.f : expf(stats[w][0] - top);
    sum += stats[w][1] * f[w];
  }
  const float inv = nan ? __int_as_float(0x7fffffff) : sum > 0.f ? 1.f / sum : (sum != sum ? sum : 0.f);
  T* to = (T*)a.out + ((int64_t)(r.start + i) * a.nh + h) * hd;
  for (int d = threadIdx.x; d < hd; d += kWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += o[w][d] * f[w];
    to[d] = rd::Num<T>::from_f(v * inv);
  }
}

}  // namespace

extern "C" int64_t rd_attention_quant_workspace_bytes(int dtype, int bits, int m_max, int B, int nh, int nkv, int hd, int max_new, int max_kv) {
  if ((dtype != RD_F32 && dtype != RD_BF16) || (bits != 4 && bits != 8) || m_max < 0 || B < 0 || nh < 1 || nkv < 1 || hd < 1 || max_new < 0 || max_kv < 0) return RD_ERR_ARG;
  if (nh % nkv != 0 || B == 0 || m_max == 0 || max_new == 0) return 0;
  return 0;
}

extern "C" int rd_attention_quant(int dtype, int bits, const void* q, int64_t ldq, const uint8_t* k_codes, const void* k_params, const uint8_t* v_codes,
                                  const void* v_params, void* out, const int32_t* row_start, const int32_t* kv_begin, const int32_t* base_len, int m_max,
                                  int B, int nh, int nkv, int hd, int max_len, int max_new, int max_kv, int mode, const uint32_t* tree_mask,
                                  int mask_words, float scale, void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  RD_REQUIRE(dtype == RD_F32 || dtype == RD_BF16, RD_ERR_DTYPE);
  RD_REQUIRE(bits == 4 || bits == 8, RD_ERR_UNSUPPORTED);
  RD_REQUIRE(mode == RD_ATTN_CAUSAL || mode == RD_ATTN_TREE, RD_ERR_UNSUPPORTED);
  RD_REQUIRE(m_max >= 0 && B >= 0 && nh >= 1 && nkv >= 1 && nh % nkv == 0 && max_new >= 0 && max_kv >= 0, RD_ERR_ARG);
  RD_REQUIRE(hd >= 8 && hd <= kMaxHd && hd % 8 == 0, RD_ERR_SIZE);
  RD_REQUIRE(max_len >= 1 && max_len % 16 == 0, RD_ERR_SIZE);
  RD_REQUIRE(nh <= 65535 && B <= 65535, RD_ERR_SIZE);
  if (m_max == 0 || B == 0 || max_new == 0) return RD_OK;
  RD_REQUIRE(q && k_codes && k_params && v_codes && v_params && out && row_start && kv_begin && base_len, RD_ERR_ARG);
  RD_REQUIRE(ldq >= (int64_t)nh * hd && scale > 0.f && scale <= 3.402823466e38f, RD_ERR_ARG);
  RD_REQUIRE(mode != RD_ATTN_TREE || (tree_mask && mask_words >= 1), RD_ERR_ARG);
  RD_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_params | (uintptr_t)v_params) & 15) == 0, RD_ERR_ALIGN);
  RD_REQUIRE((ldq * (dtype == RD_BF16 ? 2 : 4)) % 16 == 0, RD_ERR_ALIGN);
  const Args a{q, ldq, k_codes, v_codes, (const uint32_t*)k_params, (const uint32_t*)v_params, out, row_start, kv_begin, base_len, m_max, B, nh, nkv, hd,
               max_len, max_new, max_kv, mode, tree_mask, mask_words, scale};
  const int64_t need = rd_attention_quant_workspace_bytes(dtype, bits, m_max, B, nh, nkv, hd, max_new, max_kv);
  RD_REQUIRE(need <= workspace_bytes, RD_ERR_CAPACITY);
  RD_REQUIRE(need == 0 || workspace, RD_ERR_ARG);
  RD_REQUIRE(need == 0 || ((uintptr_t)workspace & 15) == 0, RD_ERR_ALIGN);
  (void)status;
  const dim3 grid(max_new, nh, B);
  cudaError_t err;
  auto run = [&](auto kern) { err = rd::launch_chained(kern, grid, dim3(kWarps * 32), 0, (cudaStream_t)stream, 1, a); };
  if (dtype == RD_BF16) bits == 4 ? run(attention_quant_rows_kernel<__nv_bfloat16, 4>) : run(attention_quant_rows_kernel<__nv_bfloat16, 8>);
  else bits == 4 ? run(attention_quant_rows_kernel<float, 4>) : run(attention_quant_rows_kernel<float, 8>);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

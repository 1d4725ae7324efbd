// Attention over a key/value cache held in codes of 8 or 4 bits (cache_quant.cu): softmax(scale Q K^T) V with
// K = scale_k (code - zero_k), V likewise, a scale and a zero for each token of a head.
//
// attention_quant_rows_kernel: one CTA per (new token, head), for 32-bit queries and heads that the other kernels do not have.  A warp
// takes 32 keys at a time, a lane one or two words of a row's codes; running maximum and sum in fp32, a lane a key.  The score is scale_k (q . code - zero_k
// sum q), the value's weight p scale_v.  Bound by its instructions (unpacking, and the sums over lanes): eight rows of 4096 keys, 32 heads on 8 of 128
// features, fp32 queries take 322 us at 8 bits and 181 at 4 on one B200; one row of 300 keys, 8 heads of 64, 12 us.  Keys are never cut, and the
// query heads of a group unpack the same codes each: one row of 131072 keys takes 6.9 ms, a prompt of 512 tokens 1.1.
#include <cuda_fp16.h>

#include "quant.cuh"
#include "umma.cuh"

namespace {

using namespace rd_quant;

constexpr int kWarps = 8;
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

// W: words of codes that a lane holds of a row; `lanes` lanes (a power of two) hold a row, 32 / lanes rows at a time.
template <typename T, int BITS, int W>
__global__ void __launch_bounds__(kWarps * 32) attention_quant_rows_kernel(const Args a, int lanes) {
  constexpr int kPer = 32 / BITS, kBatch = 8;  // codes of a word; loads of a lane that are on their way together
  __shared__ float o[kWarps][kMaxHd], stats[kWarps][2];
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const Row r = row_of(a, b);
  if (i >= r.n_new) return;
  const int hd = a.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int words = hd / kPer, part = lane & (lanes - 1), at_once = 32 / lanes, group = lane / lanes;
  const T* from = (const T*)a.q + (int64_t)(r.start + i) * a.ldq + (int64_t)h * hd;
  float q[W][kPer], q_sum = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      q[w][e] = part + 32 * w < words ? rd::Num<T>::to_f(from[(part + 32 * w) * kPer + e]) : 0.f;
      q_sum += q[w][e];
    }
  for (int x = lanes >> 1; x > 0; x >>= 1) q_sum += __shfl_xor_sync(0xffffffffu, q_sum, x);
  const int64_t plane = ((int64_t)b * a.nkv + h / (a.nh / a.nkv)) * a.max_len + r.first;
  // words of keys (or values) s * at_once + group of 32 from j0 on, s from s0 on
  auto load = [&](const uint8_t* codes, int j0, int s0, uint32_t (&u)[kBatch][W]) {
#pragma unroll
    for (int x = 0; x < kBatch; ++x) {
      const int j = j0 + (s0 + x) * at_once + group;
#pragma unroll
      for (int w = 0; w < W; ++w)
        u[x][w] = s0 + x < lanes && j < r.end && part + 32 * w < words ? reinterpret_cast<const uint32_t*>(codes + (plane + j) * (hd * BITS / 8))[part + 32 * w] : 0u;
    }
  };
  float m = -INFINITY, l = 0.f, acc[W][kPer] = {};
  for (int j0 = warp * 32; j0 < r.end; j0 += kWarps * 32) {
    const int j = j0 + lane;
    const bool seen = j < r.end && (j < r.base || sees(a, r, i, j));
    const uint32_t pk = seen ? a.k_params[plane + j] : 0u, pv = seen ? a.v_params[plane + j] : 0u;
    float mine = 0.f;  // q . codes of key j
    uint32_t u[kBatch][W];
    for (int s0 = 0; s0 < lanes; s0 += kBatch) {
      load(a.k_codes, j0, s0, u);
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        float dot = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int e = 0; e < kPer; ++e) dot = fmaf(q[w][e], code_as_float((u[x][w] >> (BITS * e)) & ((1u << BITS) - 1)), dot);
        for (int y = lanes >> 1; y > 0; y >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, y);
        dot = __shfl_sync(0xffffffffu, dot, (lane & (at_once - 1)) * lanes);
        if (lane / at_once == s0 + x) mine = dot;
      }
    }
    const float s = seen ? (mine - (float)param_zero(pk) * q_sum) * param_scale(pk) * a.scale : -INFINITY;
    load(a.v_codes, j0, 0, u);  // under way while the weights are formed
    const bool any_nan = __any_sync(0xffffffffu, s != s);
    const float top = any_nan ? __int_as_float(0x7fffffff) : fmaxf(m, rd::warp_max(s));
    if (top == -INFINITY) continue;
    const float keep = m == -INFINITY ? 0.f : expf(m - top);
    const float p = seen ? expf(s - top) : 0.f;
    l = l * keep + rd::warp_sum(p);
    m = top;
    const float pw = seen ? p * param_scale(pv) : 0.f, zv = (float)param_zero(pv);
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[w][e] *= keep;
    for (int s0 = 0; s0 < lanes; s0 += kBatch) {
      if (s0 > 0) load(a.v_codes, j0, s0, u);
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const int key = (s0 + x) * at_once + group;  // past 31 where lanes < kBatch: nothing
        const float weight = __shfl_sync(0xffffffffu, pw, key & 31), zero = __shfl_sync(0xffffffffu, zv, key & 31);
        if (key > 31) continue;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
          for (int e = 0; e < kPer; ++e) acc[w][e] = fmaf(weight, code_as_float((u[x][w] >> (BITS * e)) & ((1u << BITS) - 1)) - zero, acc[w][e]);
      }
    }
  }
#pragma unroll
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      for (int x = lanes; x < 32; x <<= 1) acc[w][e] += __shfl_xor_sync(0xffffffffu, acc[w][e], x);
      if (group == 0 && part + 32 * w < words) o[warp][(part + 32 * w) * kPer + e] = acc[w][e];
    }
  if (lane == 0) stats[warp][0] = m, stats[warp][1] = l;
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

#include "attention_quant_few.cuh"
#include "attention_quant_many.cuh"

// The few-rows kernel serves 16-bit queries of heads of 64 or 128 features whose group has at most kFewRows rows.
struct FewPlan {
  int rows;          // of an item: 8 or 16; 0: not for this call
  int keys, slots;   // of a tile; CTAs at most
  int64_t items;     // bound of their number
};
FewPlan few_plan(int dtype, int bits, int B, int nh, int nkv, int hd, int max_new, int max_kv) {
  FewPlan p{0, 0, 0, 0};
  const int64_t rows = (int64_t)max_new * (nh / nkv);
  if (dtype != RD_BF16 || (hd != 64 && hd != 128) || rows > kFewRows) return p;
  p.rows = rows <= 8 ? 8 : 16;
  p.keys = kTileBytes * 8 / (hd * bits);
  p.slots = rd_quant::sm_count() * (p.rows == 8 ? 2 : 1);
  const int64_t tiles = ((int64_t)max_kv + p.keys - 1) / p.keys + 1, chains = (int64_t)B * nkv;  // one more: rows begin inside a tile
  const int64_t all = chains * ((tiles + kFewWarps - 1) / kFewWarps);
  p.items = all < chains + 4 * p.slots ? all : chains + 4 * p.slots;
  return p;
}
// chains that no call cuts need no workspace
bool few_cut(const FewPlan& p, int B, int nkv) { return p.items > (int64_t)B * nkv; }

template <int HD, int BITS, int NT>
int launch_few(const Args& a, const FewPlan& p, void* workspace, int32_t* status, cudaStream_t s) {
  constexpr auto kernel = attention_quant_few_kernel<HD, BITS, NT>;
  using Sm = FewSmem<HD, BITS, NT>;
  RD_REQUIRE(rd_quant::allow_smem<kernel>(Sm::kBytes), RD_ERR_LAUNCH);
  CUtensorMap mk, mv;
  const int64_t lines = (int64_t)a.B * a.nkv * a.max_len * (HD * BITS / 8) / 128;
  RD_REQUIRE(lines <= 0x7fffffff, RD_ERR_SIZE);
  RD_REQUIRE(rd_umma::make_byte_map(&mk, a.k_codes, lines, 128, 128, kTileBytes / 128) && rd_umma::make_byte_map(&mv, a.v_codes, lines, 128, 128, kTileBytes / 128),
             RD_ERR_ARG);
  const bool cut = few_cut(p, a.B, a.nkv);
  int* header = (int*)workspace;
  float* partial = cut ? (float*)((uint8_t*)workspace + kFewHeader) : nullptr;
  const unsigned grid = (unsigned)(p.items < p.slots ? p.items : p.slots);
  cudaError_t err = rd::launch_chained(kernel, dim3(grid), dim3(kFewThreads), Sm::kBytes, s, 1, mk, mv, a, partial, p.slots, cut ? header : nullptr, status);
  RD_CHECK_CHAINED(err);
  if (!cut) return RD_OK;
  err = rd::launch_chained(attention_quant_merge_kernel<HD, Shape<HD, BITS>::kKeys>, dim3((unsigned)(a.nkv * p.rows), (unsigned)a.B), dim3(256), 0, s, 1, a, (const float*)partial,
                           (const int*)header, p.rows);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

// The many-rows kernel serves the other 16-bit calls of such heads.
struct ManyPlan {
  bool here;
  int tiles;    // of 128 query rows to a CTA
  int n_split;
};
ManyPlan many_plan(int dtype, int B, int nh, int nkv, int hd, int max_new, int max_kv) {
  const int64_t rows = (int64_t)max_new * (nh / nkv), chains = (int64_t)B * nkv;
  ManyPlan p{dtype == RD_BF16 && (hd == 64 || hd == 128) && rows > kFewRows, 1, 1};
  if (!p.here) return p;
  // Two tiles that share their keys cost 0.7 to 0.85 of two that do not, if both are there and such pairs fill the SMs.  Where the bound is one of several
  // rows' it is taken for half as much again as most have: eight draft trees of 64 to 140 query rows take 38 us in such pairs and 32 without.
  if (chains * ((rows + 2 * kManyRows - 1) / (2 * kManyRows)) >= rd_quant::sm_count() && rows > (B == 1 ? kManyRows : kManyRows * 3 / 2)) p.tiles = 2;
  // Shares of the keys where the query tiles leave CTAs idle: enough to fill two to an SM, each of at least four tiles of keys.
  const int64_t ctas = chains * ((rows + p.tiles * kManyRows - 1) / (p.tiles * kManyRows)), slots = 2 * rd_quant::sm_count() / p.tiles;
  const int64_t key_tiles = ((int64_t)max_kv + kManyKeys - 1) / kManyKeys, by_fill = 2 * ctas < slots ? slots / ctas : 1, by_length = key_tiles / 4;
  int64_t n = by_fill < by_length ? by_fill : by_length;
  // Of several rows one may be much longer than the others, which is not known here: then shares that would fill the SMs one and a half times, of at
  // least twelve tiles, where rows have as many new tokens as the longest on average; a multiple of those above, so that rows that are alike take
  // whole rounds.  This pays where rows differ and costs where they do not (one B200, 32 heads on 8 of 128, 8 bits, us, with these shares against only those
  // that fill the SMs): 11 to 147 new tokens on 2 to 2554 49 : 93, 5 to 147 on 30 to 6000 85 : 197, 64 and 200 on 4000 and 100 53 : 84; but 4 x 128 on 3968 in
  // four shares 106, in two 89 (in three 125: two rounds of a third), 2 x 128 on 8000 110 : 88, 8 x 128 on 3872 139 either way.
  if (B > 1) {
    int64_t expected = chains * rows / (p.tiles * kManyRows);
    expected = expected < chains ? chains : expected;
    const int64_t by_spread = 3 * slots / (2 * expected), most = key_tiles / 12, spread = by_spread < most ? by_spread : most;
    const int64_t rounded = (spread + by_fill - 1) / by_fill * by_fill;
    if (n < spread && rounded <= most) n = rounded;
  }
  n = n < kManyMaxSplit ? n : kManyMaxSplit;
  p.n_split = n > 1 ? (int)n : 1;
  return p;
}

template <int HD, int BITS, int QT>
int launch_many(const Args& a, const ManyPlan& p, void* workspace, int32_t* status, cudaStream_t s) {
  constexpr auto kernel = attention_quant_many_kernel<HD, BITS, QT>;
  using L = Many<HD, QT>;
  RD_REQUIRE(rd_quant::allow_smem<kernel>(L::kBytes), RD_ERR_LAUNCH);
  const int64_t tiles = ((int64_t)a.max_new * (a.nh / a.nkv) + QT * kManyRows - 1) / (QT * kManyRows), items = tiles * p.n_split * a.nkv * a.B;
  RD_REQUIRE(items <= 0x7fffffff, RD_ERR_SIZE);
  const int64_t grid = items <= rd_quant::sm_count() ? items : (items + L::kParts - 1) / L::kParts;
  cudaError_t err = rd::launch_chained(kernel, dim3((unsigned)grid), dim3(L::kThreads), L::kBytes, s, 1, a, (float*)workspace, (int)tiles, p.n_split,
                                       (unsigned)items, status);
  RD_CHECK_CHAINED(err);
  if (p.n_split == 1) return RD_OK;
  err = rd::launch_chained(attention_quant_merge_shares_kernel<HD>, dim3((unsigned)(((int64_t)a.max_new * a.nh + 7) / 8), a.B), dim3(256), 0, s, 1, a,
                           (const float*)workspace, p.n_split);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}
template <int HD, int BITS>
int launch_many(const Args& a, const ManyPlan& p, void* workspace, int32_t* status, cudaStream_t s) {
  return p.tiles == 2 ? launch_many<HD, BITS, 2>(a, p, workspace, status, s) : launch_many<HD, BITS, 1>(a, p, workspace, status, s);
}

}  // namespace

extern "C" int64_t rd_attention_quant_workspace_bytes(int dtype, int bits, int m_max, int B, int nh, int nkv, int hd, int max_new, int max_kv) {
  if ((dtype != RD_F32 && dtype != RD_BF16) || (bits != 4 && bits != 8) || m_max < 0 || B < 0 || nh < 1 || nkv < 1 || hd < 1 || max_new < 0 || max_kv < 0) return RD_ERR_ARG;
  if (nh % nkv != 0 || B == 0 || m_max == 0 || max_new == 0) return 0;
  const FewPlan p = few_plan(dtype, bits, B, nh, nkv, hd, max_new, max_kv);
  if (p.rows && few_cut(p, B, nkv)) return kFewHeader + p.items * few_item_floats(hd, p.rows) * 4;
  const ManyPlan q = many_plan(dtype, B, nh, nkv, hd, max_new, max_kv);
  if (q.here && q.n_split > 1) return (int64_t)m_max * nh * q.n_split * (hd == 64 ? kShareFloats<64> : kShareFloats<128>) * 4;
  return 0;
}

extern "C" int rd_attention_quant(const rd_attention_quant_desc* desc, void* stream) {
  RD_REQUIRE(desc, RD_ERR_ARG);
  const auto [q, ldq, k_codes, k_params, v_codes, v_params, out, row_start, kv_begin, base_len, tree_mask, workspace, workspace_bytes, status, dtype, bits, m_max,
              B, nh, nkv, hd, max_len, max_new, max_kv, mode, mask_words, scale] = *desc;
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
  const FewPlan few = few_plan(dtype, bits, B, nh, nkv, hd, max_new, max_kv);
  if (few.rows != 0 && max_kv > 0) {
    cudaStream_t s = (cudaStream_t)stream;
    if (hd == 128) {
      if (bits == 4) return few.rows == 8 ? launch_few<128, 4, 1>(a, few, workspace, status, s) : launch_few<128, 4, 2>(a, few, workspace, status, s);
      return few.rows == 8 ? launch_few<128, 8, 1>(a, few, workspace, status, s) : launch_few<128, 8, 2>(a, few, workspace, status, s);
    }
    if (bits == 4) return few.rows == 8 ? launch_few<64, 4, 1>(a, few, workspace, status, s) : launch_few<64, 4, 2>(a, few, workspace, status, s);
    return few.rows == 8 ? launch_few<64, 8, 1>(a, few, workspace, status, s) : launch_few<64, 8, 2>(a, few, workspace, status, s);
  }
  const ManyPlan many = many_plan(dtype, B, nh, nkv, hd, max_new, max_kv);
  if (many.here && max_kv > 0) {
    cudaStream_t s = (cudaStream_t)stream;
    if (hd == 128) return bits == 4 ? launch_many<128, 4>(a, many, workspace, status, s) : launch_many<128, 8>(a, many, workspace, status, s);
    return bits == 4 ? launch_many<64, 4>(a, many, workspace, status, s) : launch_many<64, 8>(a, many, workspace, status, s);
  }
  const dim3 grid(max_new, nh, B);
  cudaError_t err;
  const int words = hd * bits / 32;
  int lanes = 1;
  while (lanes < words && lanes < 32) lanes *= 2;
  auto run = [&](auto kern) { err = rd::launch_chained(kern, grid, dim3(kWarps * 32), 0, (cudaStream_t)stream, 1, a, lanes); };
  auto pick = [&](auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    if (bits == 4) run(attention_quant_rows_kernel<T, 4, 1>);
    else words <= 32 ? run(attention_quant_rows_kernel<T, 8, 1>) : run(attention_quant_rows_kernel<T, 8, 2>);
  };
  if (dtype == RD_BF16) pick((__nv_bfloat16*)nullptr);
  else pick((float*)nullptr);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

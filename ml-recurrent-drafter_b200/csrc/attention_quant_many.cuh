// Attention over a cache in codes for many query rows to a key/value head (packed drafts, prompts), on the 5th-generation tensor cores:
// included by attention_quant.cu.
//
// One CTA serves 128 query rows of one (batch row, key/value head): row R is head R % group of new token R / group, so that the codes of a
// tile are unpacked once for all heads of a group.
//   warps 0-3  the queries, scaled by a power of two to fp16, into shared memory; then softmax: a thread owns a row (= TMEM lane), S times
//              its keys' scales, running maximum (moved only when exceeded by 2^6) and sum, weights W = p scale_v / r 2^8 as fp16 to TMEM;
//   warps 4-7  unpacking: codes minus their zeros as fp16 (exact: 1024 + code is one masking instruction, minus 1024 + zero) into
//              swizzled shared-memory tiles of 64 keys, two stages each for K and V; scales of keys and values beside them.  r, a power
//              of two, is the largest value scale of the tiles so far;
//   warp 8     issues S = Q K^T (both from shared memory) and O += W V (W from TMEM, V as an MN-major operand).
// Features lie in the order in which the masks deliver them (within 8 of 4 bits: 0 4 1 5 2 6 3 7, within 4 of 8 bits: 0 2 1 3); the queries
// take the same order, the output undoes it.  Two CTAs on an SM overlap each other's waits.
// With n_split > 1 a CTA walks its share of the tiles and leaves its sums for attention_quant_merge_shares_kernel.
//
// Every wait is bounded; on give-up the kernel records a code in *status, frees its TMEM and returns.

constexpr int kManyRows = 128, kManyKeys = 64, kManyThreads = 288;
constexpr int kManyMaxSplit = 16;
constexpr float kManySlack = 6.f;      // log2 units that a tile's maximum may exceed the running one
constexpr uint32_t kColS = 0, kColP = 64, kColO = 128;  // TMEM: S 64 fp32 columns, W two buffers of 32, O HD

template <int HD>
struct ManySmem {
  static constexpr int kQ = kManyRows * HD * 2, kTile = kManyKeys * HD * 2;
  static constexpr int kVectors = 4 * kManyKeys * 4 * 2 + 4 * 4;  // scales of keys and values of four tiles, and r of each
  static constexpr int kBytes = 1024 + kQ + 4 * kTile + kVectors + kManyRows * 4 + 32 * 8;
  static constexpr uint32_t kTmemCols = 256;
};

__device__ __forceinline__ bool mbar_wait_or(uint64_t* bar, uint32_t parity, volatile int* stop) {
  if (rd_umma::mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    if (rd_umma::mbar_try(bar, parity)) return true;
    if (*stop || clock64() - t0 > (1ll << 31)) return false;
  }
}
// by all lanes of a warp, the same answer for all
__device__ __forceinline__ bool warp_wait_or(uint64_t* bar, uint32_t parity, volatile int* stop) {
  return __all_sync(0xffffffffu, mbar_wait_or(bar, parity, stop));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(rd_umma::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// fp16 operands, fp32 accumulator, M = 128
__device__ __forceinline__ uint32_t idesc_fp16(int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Eight codes (4 bits: one word; 8 bits: two) minus zero as fp16; z2: 1024 + zero in both halves.
template <int BITS>
__device__ __forceinline__ uint4 unpack8(const uint32_t* w, uint32_t z2) {
  uint4 u;
  if constexpr (BITS == 4) {
    u.x = sub_f16x2((w[0] & 0x000f000fu) | 0x64006400u, z2);
    u.y = sub_f16x2(((w[0] >> 4) & 0x000f000fu) | 0x64006400u, z2);
    u.z = sub_f16x2(((w[0] >> 8) & 0x000f000fu) | 0x64006400u, z2);
    u.w = sub_f16x2(((w[0] >> 12) & 0x000f000fu) | 0x64006400u, z2);
  } else {
    u.x = sub_f16x2((w[0] & 0x00ff00ffu) | 0x64006400u, z2);
    u.y = sub_f16x2(((w[0] >> 8) & 0x00ff00ffu) | 0x64006400u, z2);
    u.z = sub_f16x2((w[1] & 0x00ff00ffu) | 0x64006400u, z2);
    u.w = sub_f16x2(((w[1] >> 8) & 0x00ff00ffu) | 0x64006400u, z2);
  }
  return u;
}
// where feature k of 8 lies among them
template <int BITS>
__device__ __forceinline__ constexpr int order8(int k) {
  return BITS == 4 ? (k < 4 ? 2 * k : 2 * (k - 4) + 1) : (k & 4) + ((k & 1) * 2 + ((k >> 1) & 1));
}

template <int HD, int BITS>
__global__ void __launch_bounds__(kManyThreads, 2)
    attention_quant_many_kernel(const Args a, float* partial, int n_split, int32_t* status) {
  using Sm = ManySmem<HD>;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;
  uint8_t* sK = smem + Sm::kQ;
  uint8_t* sV = sK + 2 * Sm::kTile;
  float* k_scale = reinterpret_cast<float*>(sV + 2 * Sm::kTile);  // [4][64]
  float* v_scale = k_scale + 4 * kManyKeys;                       // [4][64], over r, times 2^8
  float* refs = v_scale + 4 * kManyKeys;                          // [4]
  float* units = refs + 4;                                        // [128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(units + kManyRows);
  uint64_t *q_full = bars, *k_full = bars + 1, *v_full = bars + 3, *s_full = bars + 5, *o_full = bars + 7, *p_full = bars + 9, *s_empty = bars + 11;
  uint64_t* scales_full = bars + 12;  // [4]: the scales of a tile are there; a tile's place is written again only when the softmax is done with it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int group = a.nh / a.nkv;
  // in causal calls later tiles see more keys: they start first
  const bool late_first = a.mode == RD_ATTN_CAUSAL && n_split == 1 && gridDim.x > 1;
  const int linear = (int)(blockIdx.x + gridDim.x * blockIdx.y);
  const int bx = late_first ? (int)gridDim.x - 1 - linear / (int)gridDim.y : (int)blockIdx.x;
  const int hk = late_first ? linear % (int)gridDim.y : (int)blockIdx.y;
  const int b = blockIdx.z, split = bx % n_split, q0 = bx / n_split * kManyRows;
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const Row r = row_of(a, b);
  const int rows = r.n_new * group;
  if (q0 >= rows) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first_token = q0 / group, last_token = (min(q0 + kManyRows, rows) - 1) / group;
  const int kv_end = a.mode == RD_ATTN_CAUSAL ? min(r.end, r.base + last_token + 1) : r.end;
  const int all_tiles = (max(kv_end, 0) + kManyKeys - 1) / kManyKeys;
  const int per_split = (all_tiles + n_split - 1) / n_split;
  const int t_begin = split * per_split, n_tiles = max(0, min(per_split, all_tiles - t_begin));
  if (threadIdx.x == 0) {
    rd_umma::mbar_init(q_full, 4);
    for (int s = 0; s < 2; ++s) {
      rd_umma::mbar_init(&k_full[s], 4);
      rd_umma::mbar_init(&v_full[s], 4);
      rd_umma::mbar_init(&s_full[s], 1);
      rd_umma::mbar_init(&o_full[s], 1);
      rd_umma::mbar_init(&p_full[s], 4);
    }
    for (int s = 0; s < 4; ++s) rd_umma::mbar_init(&scales_full[s], 4);
    rd_umma::mbar_init(s_empty, 4);
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) rd_umma::tmem_alloc(tmem_slot, Sm::kTmemCols);
  rd_umma::fence_before();
  __syncthreads();
  rd_umma::fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  int site = 0;

  if (warp >= 4 && warp < 8) {
    // ---------------- unpacking ----------------
    constexpr int kBytes = HD * BITS / 16;  // a thread's half of a key: 16, 32 or 64 bytes
    constexpr int kLoads = kBytes / 16, kChunks = HD / 16, kWordsOf8 = BITS / 4;
    const int tid = threadIdx.x - 128, key = tid & 63, half = tid >> 6;
    const int64_t plane = ((int64_t)b * a.nkv + hk) * a.max_len + r.first;
    uint4 kc[kLoads], vc[kLoads];
    uint32_t kp = 0, vp = 0, vq = 0;
    // Keys past the last one stand for zeros.  Each half is asked for as soon as the registers of the tile before are free.
    auto request_k = [&](int t) {
      const int j0 = (t_begin + t) * kManyKeys, j = j0 + key, other = j0 + (key ^ 32);
      const bool there = j < kv_end;
      const uint8_t* k = a.k_codes + (plane + j) * (HD * BITS / 8) + half * kBytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) kc[i] = there ? reinterpret_cast<const uint4*>(k)[i] : make_uint4(0u, 0u, 0u, 0u);
      kp = there ? a.k_params[plane + j] : 0u;
      vp = there ? a.v_params[plane + j] : 0u;
      vq = other < kv_end ? a.v_params[plane + other] : 0u;  // with vp: every warp knows all 64 scales of the values
    };
    auto request_v = [&](int t) {
      const int j = (t_begin + t) * kManyKeys + key;
      const uint8_t* v = a.v_codes + (plane + j) * (HD * BITS / 8) + half * kBytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) vc[i] = j < kv_end ? reinterpret_cast<const uint4*>(v)[i] : make_uint4(0u, 0u, 0u, 0u);
    };
    auto store = [&](uint8_t* tile, const uint4* c, uint32_t param) {
      const uint32_t z2 = (0x6400u + param_zero(param)) * 0x10001u;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int chunk = half * kChunks + i;
        *reinterpret_cast<uint4*>(tile + (chunk >> 3) * (kManyKeys * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4)) =
            unpack8<BITS>(reinterpret_cast<const uint32_t*>(c) + i * kWordsOf8, z2);
      }
    };
    uint32_t top = 0;  // exponent bits of r: at least 2^-100
    if (n_tiles > 0) {
      request_k(0);
      request_v(0);
    }
    for (int t = 0; t < n_tiles; ++t) {
      if (t >= 2 && !warp_wait_or(&s_full[t & 1], ((t - 2) >> 1) & 1, stop)) {
        ok = false, site = 1;
        break;
      }
      store(sK + (t & 1) * Sm::kTile, kc, kp);
      // scales are never negative; NaN counts as none
      const float v0 = param_scale(vp), v1 = param_scale(vq);
      const uint32_t bits = max(v0 == v0 ? __float_as_uint(v0) : 0u, v1 == v1 ? __float_as_uint(v1) : 0u);
      top = max(max(top, 27u << 23), __reduce_max_sync(0xffffffffu, bits) & 0x7f800000u);
      if (half == 0) {
        k_scale[(t & 3) * kManyKeys + key] = param_scale(kp);
        v_scale[(t & 3) * kManyKeys + key] = v0 * __uint_as_float((262u << 23) - top);  // 2^8 / r
        if (key == 0) refs[t & 3] = __uint_as_float(top);
      }
      const uint32_t vz = vp;
      if (t + 1 < n_tiles) request_k(t + 1);
      rd_umma::fence_async_proxy();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&scales_full[t & 3]);
        mbar_arrive(&k_full[t & 1]);
      }
      if (t >= 2 && !warp_wait_or(&o_full[t & 1], ((t - 2) >> 1) & 1, stop)) {
        ok = false, site = 2;
        break;
      }
      store(sV + (t & 1) * Sm::kTile, vc, vz);
      if (t + 1 < n_tiles) request_v(t + 1);
      rd_umma::fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[t & 1]);
    }
  } else if (warp == 8) {
    // ---------------- products ----------------
    if (rd::elect_one()) {
      const uint32_t idesc_qk = idesc_fp16(kManyKeys, false), idesc_pv = idesc_fp16(HD, true);
      auto issue_qk = [&](int t) {
        const uint32_t k = rd_umma::smem_u32(sK + (t & 1) * Sm::kTile), q = rd_umma::smem_u32(sQ);
#pragma unroll
        for (int kd = 0; kd < HD / 16; ++kd)
          rd_umma::mma_ss(tmem + kColS, rd_umma::desc_k_major(q + (kd >> 2) * (kManyRows * 128) + (kd & 3) * 32),
                          rd_umma::desc_k_major(k + (kd >> 2) * (kManyKeys * 128) + (kd & 3) * 32), idesc_qk, kd != 0);
        rd_umma::commit(&s_full[t & 1]);
      };
      ok = mbar_wait_or(q_full, 0, stop);
      if (ok && n_tiles > 0) {
        ok = mbar_wait_or(&k_full[0], 0, stop);
        if (ok) {
          rd_umma::fence_after();
          issue_qk(0);
        }
      }
      for (int t = 0; ok && t < n_tiles; ++t) {
        if (t + 1 < n_tiles) {
          ok = mbar_wait_or(&k_full[(t + 1) & 1], ((t + 1) >> 1) & 1, stop) && mbar_wait_or(s_empty, t & 1, stop);
          if (!ok) break;
          rd_umma::fence_after();
          issue_qk(t + 1);
        }
        ok = mbar_wait_or(&p_full[t & 1], (t >> 1) & 1, stop) && mbar_wait_or(&v_full[t & 1], (t >> 1) & 1, stop);
        if (!ok) break;
        rd_umma::fence_after();
        const uint32_t v = rd_umma::smem_u32(sV + (t & 1) * Sm::kTile);
#pragma unroll
        for (int ks = 0; ks < kManyKeys / 16; ++ks)
          mma_ts(tmem + kColO, tmem + kColP + (t & 1) * 32 + ks * 8, rd_umma::desc_mn_major(v + ks * 2048, kManyKeys * 128), idesc_pv, (t | ks) != 0);
        rd_umma::commit(&o_full[t & 1]);
      }
      if (!ok) site = 3;
    }
    __syncwarp();
  } else {
    // ---------------- queries: eight lanes a row ----------------
    {
      const int part = lane & 7;
      constexpr int kPart = HD / 8;  // features of a lane: 8 or 16
#pragma unroll 2
      for (int i = 0; i < 8; ++i) {
        const int row = warp * 32 + i * 4 + (lane >> 3), R = q0 + row;
        const bool live = R < rows;
        const __nv_bfloat16* src =
            (const __nv_bfloat16*)a.q + (int64_t)(r.start + (live ? R / group : 0)) * a.ldq + (hk * group + (live ? R % group : 0)) * HD + part * kPart;
        float x[kPart];
#pragma unroll
        for (int c = 0; c < kPart / 8; ++c) {
          const uint4 u = live ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0u, 0u, 0u, 0u);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) x[8 * c + 2 * e] = __uint_as_float(w[e] << 16), x[8 * c + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < kPart; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // the row's largest to [2^14, 2^15): see the few-rows kernel
        const int e2 = most > 0.f && most < INFINITY ? (int)(__float_as_uint(most) >> 23) : 141;
        const int up = 141 - e2, h1 = up / 2, h2 = up - h1;
        const float f1 = __uint_as_float((uint32_t)(127 + h1) << 23), f2 = __uint_as_float((uint32_t)(127 + h2) << 23);
#pragma unroll
        for (int c = 0; c < kPart / 8; ++c) {
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[order8<BITS>(k)] = x[8 * c + k] * f1 * f2;
          const int chunk = part * (kPart / 8) + c;
          *reinterpret_cast<uint4*>(sQ + (chunk >> 3) * (kManyRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) =
              make_uint4(pack_f16(y[0], y[1]), pack_f16(y[2], y[3]), pack_f16(y[4], y[5]), pack_f16(y[6], y[7]));
        }
        if (part == 0)
          units[row] = a.scale * 1.44269504f * __uint_as_float((uint32_t)(127 - h1) << 23) * __uint_as_float((uint32_t)(127 - h2) << 23);
      }
      rd_umma::fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // ---------------- softmax: a thread a row ----------------
    const int row = warp * 32 + lane, R = q0 + row;
    const bool live = R < rows;
    const int token = live ? R / group : 0;
    const float unit = units[row];  // its own warp's
    const uint32_t taddr = tmem + ((uint32_t)(warp * 32) << 16);
    const int all_see = a.mode == RD_ATTN_CAUSAL ? min(kv_end, r.base + first_token + 1) : min(kv_end, r.base);
    float m_run = -INFINITY, l_run = 0.f, ref = 0.f;
    for (int t = 0; t < n_tiles; ++t) {
      if (!warp_wait_or(&scales_full[t & 3], (t >> 2) & 1, stop) || !warp_wait_or(&s_full[t & 1], (t >> 1) & 1, stop)) {
        ok = false, site = 4;
        break;
      }
      rd_umma::fence_after();
      const int j0 = (t_begin + t) * kManyKeys;
      const bool whole = j0 + kManyKeys <= all_see;
      uint64_t vis = ~0ull;
      if (!whole) {
        const int off = j0 - r.base, first = max(off, 0);  // first: the tile's first new token
        uint64_t nb;
        if (a.mode == RD_ATTN_CAUSAL) {
          const int n = token - first + 1;
          nb = n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1ull;
        } else {
          const uint32_t* mask = a.tree_mask + (int64_t)(r.start + token) * a.mask_words;
          const int w = first >> 5, sh = first & 31;
          const uint64_t lo = w < a.mask_words ? mask[w] : 0u, mid = w + 1 < a.mask_words ? mask[w + 1] : 0u, hi = w + 2 < a.mask_words ? mask[w + 2] : 0u;
          nb = ((lo | (mid << 32)) >> sh) | (sh ? hi << (64 - sh) : 0ull);
        }
        vis = off >= 0 ? nb : off <= -64 ? ~0ull : (nb << -off) | ((1ull << -off) - 1ull);
        const int n_in = kv_end - j0;
        if (n_in < 64) vis &= (1ull << max(n_in, 0)) - 1ull;
        if (!live) vis = 0;
      }
      const float4* ks = reinterpret_cast<const float4*>(k_scale + (t & 3) * kManyKeys);
      const float4* vs = reinterpret_cast<const float4*>(v_scale + (t & 3) * kManyKeys);
      const float ref_t = refs[t & 3];
      float mx = -INFINITY;
      // S is read twice, a half at a time: 64 scores and their weights at once would not fit the registers of two CTAs
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float s[32];
        rd_umma::tmem_ld32(taddr + kColS + 32 * hf, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 f = ks[8 * hf + i];
          s[4 * i] *= f.x, s[4 * i + 1] *= f.y, s[4 * i + 2] *= f.z, s[4 * i + 3] *= f.w;
        }
        if (!whole) {
          const uint32_t v = (uint32_t)(vis >> (32 * hf));
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((v >> i) & 1)) s[i] = -INFINITY;
        }
        float part[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int i = 4; i < 32; ++i) part[i & 3] = fmaxf(part[i & 3], s[i]);
        mx = fmaxf(mx, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
      }
      const float mx2 = mx * unit;
      const bool moved = mx2 > m_run + kManySlack;  // also for the first visible key
      const float m_new = moved ? mx2 : m_run;
      const float alpha = m_run == -INFINITY ? 0.f : ex2(m_run - m_new);
      float keep = moved && m_run != -INFINITY ? alpha : 1.f;
      l_run *= moved ? alpha : 1.f;
      m_run = m_new;
      if (ref_t != ref) {
        if (t > 0) keep *= ref / ref_t;
        ref = ref_t;
      }
      if (__any_sync(0xffffffffu, t > 0 && keep != 1.f)) {
        // O has to be quiet while it is brought to the new maximum or r
        if (!warp_wait_or(&o_full[(t - 1) & 1], ((t - 1) >> 1) & 1, stop)) {
          ok = false, site = 5;
          break;
        }
        rd_umma::fence_after();
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          float x[32];
          rd_umma::tmem_ld32(taddr + kColO + c * 32, x);
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] *= keep;
          rd_umma::tmem_st32(taddr + kColO + c * 32, x);
        }
      }
      const float off = m_run == -INFINITY ? 0.f : -m_run;
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float s[32];
        rd_umma::tmem_ld32(taddr + kColS + 32 * hf, s);
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 f = ks[8 * hf + i];
          s[4 * i] *= f.x, s[4 * i + 1] *= f.y, s[4 * i + 2] *= f.z, s[4 * i + 3] *= f.w;
        }
        const uint32_t v = (uint32_t)(vis >> (32 * hf));
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[i] = ex2(fmaf(s[i], unit, off));
          if (!whole && !((v >> i) & 1)) s[i] = 0.f;
          if (i & 1) sum1 += s[i];
          else sum0 += s[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 f = vs[8 * hf + i];
          float y[4] = {s[4 * i] * f.x, s[4 * i + 1] * f.y, s[4 * i + 2] * f.z, s[4 * i + 3] * f.w};
          if (!whole) {  // a hidden value counts for nothing, NaN or not
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!((v >> (4 * i + e)) & 1)) y[e] = 0.f;
          }
          w[2 * i] = pack_f16(y[0], y[1]);
          w[2 * i + 1] = pack_f16(y[2], y[3]);
        }
        asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
                taddr + kColP + (t & 1) * 32 + 16 * hf),
            "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]), "r"(w[11]),
            "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
            : "memory");
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      l_run += sum0 + sum1;
      rd_umma::fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(s_empty);
        mbar_arrive(&p_full[t & 1]);
      }
    }
    if (ok && n_tiles > 0) {
      ok = warp_wait_or(&o_full[(n_tiles - 1) & 1], ((n_tiles - 1) >> 1) & 1, stop);
      if (!ok) site = 6;
    }
    if (ok) {
      rd_umma::fence_after();
      const int64_t at = (int64_t)(r.start + token) * a.nh + hk * group + (live ? R % group : 0);
      float* to = partial + (at * n_split + split) * (HD + 2);
      const float f = n_split > 1 ? ref * 0x1p-8f : (l_run == 0.f ? 0.f : ref * 0x1p-8f / l_run);
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float x[32], y[32];
        if (n_tiles > 0) {
          rd_umma::tmem_ld32(taddr + kColO + c * 32, x);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = f == 0.f ? 0.f : x[(i & 24) + order8<BITS>(i & 7)] * f;
        if (!live) continue;
        if (n_split > 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i) *reinterpret_cast<float2*>(to + c * 32 + 2 * i) = make_float2(y[2 * i], y[2 * i + 1]);
        } else {
          uint4* dst = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + at * HD + c * 32);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            __nv_bfloat162 h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(y[8 * i + 2 * e], y[8 * i + 2 * e + 1]);
            dst[i] = *reinterpret_cast<uint4*>(h);
          }
        }
      }
      if (n_split > 1 && live) to[HD] = m_run, to[HD + 1] = l_run;
    }
  }
  if (!ok && atomicCAS((int*)stop, 0, 1) == 0 && status) atomicExch(status, 420 + site);
  rd_umma::fence_before();
  __syncthreads();
  if (warp == 8) {
    rd_umma::fence_after();
    rd_umma::tmem_dealloc(tmem, Sm::kTmemCols);
  }
}

// Sums the shares: a warp for each (new token, head).
template <int HD>
__global__ void __launch_bounds__(256) attention_quant_merge_shares_kernel(const Args a, const float* partial, int n_split) {
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, token = (int)(unit / a.nh);
  const int b = blockIdx.y;
  const Row r = row_of(a, b);
  if (token >= r.n_new) return;
  const int64_t at = (int64_t)r.start * a.nh + unit;
  const float* p = partial + at * n_split * (HD + 2);
  const float mine = lane < n_split ? p[lane * (HD + 2) + HD] : -INFINITY;
  const float top = rd::warp_max(mine);
  float sum = 0.f, v[HD / 32] = {};
#pragma unroll 4
  for (int c = 0; c < n_split; ++c) {
    const float* x = p + c * (HD + 2);
    const float mc = x[HD], f = mc == -INFINITY ? 0.f : ex2(mc - top);
    sum += f * x[HD + 1];
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) v[k] += f == 0.f ? 0.f : f * x[k * 32 + lane];
  }
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) ((__nv_bfloat16*)a.out)[at * HD + k * 32 + lane] = __float2bfloat16_rn(sum == 0.f ? 0.f : v[k] / sum);
}

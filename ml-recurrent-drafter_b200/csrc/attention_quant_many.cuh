// Attention over a cache in codes for many query rows to a key/value head (packed drafts, prompts), on the 5th-generation tensor cores:
// included by attention_quant.cu.
//
// One part of a CTA serves QT tiles of 128 query rows of one (batch row, key/value head): row R is head R % group of new token R / group, so that the codes of
// a tile of keys are unpacked once for all of them.
//   4 QT warps  the queries, scaled by a power of two to fp16, into shared memory; then softmax: a thread owns a row (= TMEM lane), running
//               maximum and sum, weights W = 2^7 p as fp16 to TMEM;
//   4 warps     unpacking: codes minus their zeros (exact: 1024 + code is one masking instruction, minus 1024 + zero) times their scales
//               over a power of two, fp16, into swizzled shared-memory tiles of 64 keys, two or four stages each for K and V.  For keys that power
//               is of the tile and goes into the scores' unit; for values it is r, that of the largest scale so far;
//   QT warps    issue S = Q K^T (both from shared memory) and O += W V (W from TMEM, V as an MN-major operand).
// Keys, values and weights are thus rounded to fp16's 11 bits, each by at most 2^-11 of itself, an eighth of what a bf16 cache costs.  With the
// scales left to the softmax instead (codes alone are exact) its 64 x 128 scores cost four instructions for two where they now take
// two and a half, which bounded the kernel: a tile of 256 rows 2560 cycles.
// S has two buffers, W of a tile takes the place of its S: QK of the next two tiles run under the softmax of this one.  A tile is read from TMEM once,
// 32 scores at a time, and weighted by the maximum so far; only where the sum of the weights turns out too large the tile's maximum is
// looked for and the tile weighted again.
// Features lie in the order in which the masks deliver them (within 8 of 4 bits: 0 4 1 5 2 6 3 7, within 4 of 8 bits: 0 2 1 3); the queries
// take the same order, the output undoes it.  QT = 2 unpacks half as often; with QT = 1 an SM works at two of these at once all the same.
// With n_split > 1 a CTA walks its share of the tiles and leaves its sums for attention_quant_merge_shares_kernel.
//
// Measured on one B200: 2048 new tokens on 6144 before, 32 heads on 8 of 128, 8 bits, 302 us, 0.82 PFLOP/s (bf16 products of the library reach 1.64): a step of 256
// rows and 64 keys takes some 2350 cycles, of which the tensor cores are busy for 42 % (products 1024 wide, with their operands' way through shared memory
// 1280), exponentials for 42, shared memory for 71, and the last of 1.7 rounds of tiles leaves SMs idle.  Eight draft trees of 64 to 140 tokens on some 400, 32
// heads, 4 bits: 31 us, ten steps of 1.3 us each, the way to the first of them and out of the last.  Tried and slower: tiles of 128 keys with one buffer of
// scores (418 us), two tiles of rows taking turns (367); no different: scores of the next tile read before this one's weights are stored, 64 columns a load.
//
// Every wait is bounded; on give-up the kernel records a code in *status, frees its TMEM and returns.

constexpr int kManyRows = 128, kManyKeys = 64;
constexpr int kManyMaxSplit = 16;
template <int HD>
constexpr int kShareFloats = HD + 4;  // of a share of a row: O, then maximum and sum; 16-byte pieces
constexpr float kWeightBits = 7.f;        // weights are 2^7 p
constexpr float kMostWeights = 32768.f;   // of a tile of a row: none is more, and fp16 holds it

// A CTA is kParts of what the head of this file describes: one of two tiles, or two of one tile that share nothing but the SM.  (The driver places
// one CTA on an SM where a kernel uses tensor memory, whatever its registers and shared memory.)
template <int HD, int QT>
struct Many {
  static constexpr int kParts = QT == 1 ? 2 : 1;
  static constexpr int kTiles = QT * kParts;
  static constexpr int kUnpack = 4 * kTiles, kIssue = kUnpack + 4 * kParts;  // first warps of these roles; softmax first: its warps' lanes in TMEM
  static constexpr int kThreads = (kIssue + kTiles) * 32;
  static constexpr int kStages = QT == 1 ? 2 : 4;  // of unpacked keys, and of values
  static constexpr int kQ = kManyRows * HD * 2, kTile = kManyKeys * HD * 2;  // bytes
  static constexpr int kBars = 256;
  static constexpr int kVectors = 8 * 4 * 4;                                // of eight tiles: r, the keys' power of two, which values are NaN
  static constexpr int kPart = (QT * kQ + 2 * kStages * kTile + kVectors + QT * kManyRows * 4 + kBars + 1023) / 1024 * 1024;
  static constexpr int kBytes = 1024 + kParts * kPart;
  // TMEM of a tile of rows: two buffers of 64 columns for S, then W; O
  static constexpr uint32_t kColS = 0, kColO = 128, kCols = 256;
  static constexpr uint32_t kTmem = kTiles * kCols;
};

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
using F2 = unsigned long long;  // two fp32 numbers
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ void unpack2(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
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
// Sixteen columns of this thread's lane; there only after tmem_have16() of the same registers, which waits for all loads before it.
__device__ __forceinline__ void tmem_ask16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_have16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
  tmem_ask16(taddr, r);
  tmem_have16(r);
}
// complete only after a wait::st
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// fp16 operands, fp32 accumulator, M = 128
__device__ __forceinline__ uint32_t idesc_fp16(int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// Eight codes (4 bits: one word; 8 bits: two) minus zero, times a scale, as fp16; z2: 1024 + zero in both halves.
template <int BITS>
__device__ __forceinline__ uint4 unpack8(const uint32_t* w, uint32_t z2, uint32_t s2) {
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
  u.x = mul_f16x2(u.x, s2), u.y = mul_f16x2(u.y, s2), u.z = mul_f16x2(u.z, s2), u.w = mul_f16x2(u.w, s2);
  return u;
}
// where feature k of 8 lies among them
template <int BITS>
__device__ __forceinline__ constexpr int order8(int k) {
  return BITS == 4 ? (k < 4 ? 2 * k : 2 * (k - 4) + 1) : (k & 4) + ((k & 1) * 2 + ((k >> 1) & 1));
}

template <int HD, int BITS, int QT>
__global__ void __launch_bounds__(Many<HD, QT>::kThreads, 1)
    attention_quant_many_kernel(const Args a, float* partial, int n_row_tiles, int n_split, unsigned n_items, int32_t* status) {
  using L = Many<HD, QT>;
  constexpr int kUnpack = L::kUnpack, kIssue = L::kIssue;
  extern __shared__ uint8_t raw[];
  __shared__ uint32_t tmem_slot;
  __shared__ int stop_flag;
  volatile int* stop = &stop_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = L::kParts == 1 ? 0 : warp < kUnpack ? warp >> 2 : warp < kIssue ? (warp - kUnpack) >> 2 : warp - kIssue;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023) + part * L::kPart;
  uint8_t* sQ = smem;
  uint8_t* sK = smem + QT * L::kQ;
  constexpr int kSt = L::kStages;
  uint8_t* sV = sK + kSt * L::kTile;
  // entries of eight tiles: what their values are multiples of, and their keys; which of their values are NaN.  The place of a tile's is
  // written again when the softmax is done with it.
  float* entries = reinterpret_cast<float*>(sV + kSt * L::kTile);  // [8][4]
  float* units = entries + 32;                                     // [QT][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(units + QT * kManyRows);
  uint64_t *k_full = bars, *v_full = k_full + kSt, *k_empty = v_full + kSt, *v_empty = k_empty + kSt;
  uint64_t* q_full = v_empty + kSt;       // [QT]
  uint64_t* s_full = q_full + QT;         // [QT][2]
  uint64_t* p_full = s_full + 2 * QT;     // [QT][2]
  uint64_t* o_full = p_full + 2 * QT;     // [QT][2]
  static_assert((4 * kSt + 7 * QT) * 8 <= L::kBars, "barriers");

  const int group = a.nh / a.nkv;
  // Which tile of which head of which row, and which share of its keys.  In causal calls later tiles see more keys: they start first.
  const int n_tiles_all = n_row_tiles * n_split;
  const unsigned index = gridDim.x < n_items ? blockIdx.x * L::kParts + part : blockIdx.x;
  const bool none = index >= n_items || (gridDim.x >= n_items && part > 0);
  const int b = none ? 0 : index / ((unsigned)n_tiles_all * a.nkv), in_row = none ? 0 : index % ((unsigned)n_tiles_all * a.nkv);
  const bool late_first = a.mode == RD_ATTN_CAUSAL && n_split == 1;
  const int hk = in_row % a.nkv, bx = late_first ? n_tiles_all - 1 - in_row / a.nkv : in_row / a.nkv;
  const int split = bx % n_split, q0 = bx / n_split * (QT * kManyRows);
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const Row r = row_of(a, b);
  const int rows = none ? 0 : r.n_new * group;
  if (!__syncthreads_or(q0 < rows)) return;
  const bool here = q0 < rows;
  const int n_q = !here ? 0 : QT == 1 ? 1 : min(QT, (rows - q0 + kManyRows - 1) / kManyRows);  // tiles of rows that there are
  const int first_token = q0 / group, last_token = (min(q0 + QT * kManyRows, rows) - 1) / group;
  const int kv_end = a.mode == RD_ATTN_CAUSAL ? min(r.end, r.base + last_token + 1) : r.end;
  const int all_tiles = (max(kv_end, 0) + kManyKeys - 1) / kManyKeys;
  const int per_split = (all_tiles + n_split - 1) / n_split;
  const int t_begin = split * per_split, n_tiles = here ? max(0, min(per_split, all_tiles - t_begin)) : 0;
  if (here && lane == 0 && warp == part * 4) {
    for (int s = 0; s < QT; ++s) rd_umma::mbar_init(&q_full[s], 4);
    for (int s = 0; s < kSt; ++s) {
      rd_umma::mbar_init(&k_full[s], 4);
      rd_umma::mbar_init(&v_full[s], 4);
      rd_umma::mbar_init(&k_empty[s], n_q);
      rd_umma::mbar_init(&v_empty[s], n_q);
    }
    for (int s = 0; s < 2 * QT; ++s) {
      rd_umma::mbar_init(&s_full[s], 2);  // the product, and its issuer, who has seen the tile's entries
      rd_umma::mbar_init(&p_full[s], 4);
      rd_umma::mbar_init(&o_full[s], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) *stop = 0;
  if (warp == kIssue) rd_umma::tmem_alloc(&tmem_slot, L::kTmem);
  rd_umma::fence_before();
  __syncthreads();
  rd_umma::fence_after();
  const uint32_t tmem = tmem_slot + part * L::kCols;
  bool ok = true;
  int site = 0;

  if (warp >= kUnpack && warp < kIssue) {
    // ---------------- unpacking ----------------
    constexpr int kBytes = HD * BITS / 16;  // a thread's half of a key: 16, 32 or 64 bytes
    constexpr int kLoads = kBytes / 16, kChunks = HD / 16, kWordsOf8 = BITS / 4;
    const int tid = (threadIdx.x - kUnpack * 32) & 127, key = tid & 63, half = tid >> 6;
    const int64_t plane = ((int64_t)b * a.nkv + hk) * a.max_len + r.first;
    // With two tiles under way, what a tile's codes are asked into is free when the tile two before has been stored, so that a trip to memory has the
    // time of a whole tile (2048 rows of 8192 keys: 313 us with one, 305 with two).  QT = 1 has no registers for that.
    constexpr int kDeep = QT;
    uint4 kc[kDeep][kLoads], vc[kDeep][kLoads];
    uint32_t kp[kDeep] = {}, kq[kDeep] = {}, vp[kDeep] = {}, vq[kDeep] = {};
    // Keys past the last one stand for zeros.
    auto request_k = [&](int t, auto set) {
      constexpr int S = decltype(set)::value;
      const int j0 = (t_begin + t) * kManyKeys, j = j0 + key, other = j0 + (key ^ 32);
      const bool there = t < n_tiles && j < kv_end;
      const uint8_t* k = a.k_codes + (plane + j) * (HD * BITS / 8) + half * kBytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) kc[S][i] = there ? reinterpret_cast<const uint4*>(k)[i] : make_uint4(0u, 0u, 0u, 0u);
      kp[S] = there ? a.k_params[plane + j] : 0u;
      vp[S] = there ? a.v_params[plane + j] : 0u;
      // with kp, vp: every warp knows all 64 scales
      kq[S] = t < n_tiles && other < kv_end ? a.k_params[plane + other] : 0u;
      vq[S] = t < n_tiles && other < kv_end ? a.v_params[plane + other] : 0u;
    };
    auto request_v = [&](int t, auto set) {
      constexpr int S = decltype(set)::value;
      const int j = (t_begin + t) * kManyKeys + key;
      const bool there = t < n_tiles && j < kv_end;
      const uint8_t* v = a.v_codes + (plane + j) * (HD * BITS / 8) + half * kBytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) vc[S][i] = there ? reinterpret_cast<const uint4*>(v)[i] : make_uint4(0u, 0u, 0u, 0u);
    };
    auto store = [&](uint8_t* tile, const uint4* c, uint32_t param, float scale) {
      const uint32_t z2 = (0x6400u + param_zero(param)) * 0x10001u, s2 = pack_f16(scale, scale);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int chunk = half * kChunks + i;
        *reinterpret_cast<uint4*>(tile + (chunk >> 3) * (kManyKeys * 128) + key * 128 + (((chunk & 7) ^ (key & 7)) << 4)) =
            unpack8<BITS>(reinterpret_cast<const uint32_t*>(c) + i * kWordsOf8, z2, s2);
      }
    };
    // The exponent bits of the largest of a warp's scales, at least 2^-100; scales are never negative, NaN counts as none.
    auto largest = [&](uint32_t p, uint32_t q) {
      const float x = param_scale(p), y = param_scale(q);
      const uint32_t bits = max(x == x ? __float_as_uint(x) : 0u, y == y ? __float_as_uint(y) : 0u);
      return max(27u << 23, __reduce_max_sync(0xffffffffu, bits) & 0x7f800000u);
    };
    // Scales are taken over 2^-kUp of that power of two: below 2 before, the products with codes stay below fp16's 2^16
    constexpr uint32_t kUp = BITS == 4 ? 10 : 6;
    uint32_t top = 0;
    auto unpack = [&](int t, auto set) {
      constexpr int S = decltype(set)::value;
      const int st = t % kSt;
      if (t >= kSt && !rd_umma::warp_wait(&k_empty[st], (t / kSt - 1) & 1, stop)) {
        ok = false, site = 1;
        return;
      }
      const uint32_t k_top = largest(kp[S], kq[S]);
      store(sK + st * L::kTile, kc[S], kp[S], param_scale(kp[S]) * __uint_as_float(((254 + kUp) << 23) - k_top));
      top = max(top, largest(vp[S], vq[S]));
      float v = param_scale(vp[S]);
      const uint32_t nan = __ballot_sync(0xffffffffu, v != v);
      v = v != v ? 0.f : v * __uint_as_float(((254 + kUp) << 23) - top);
      // QK of tile t - kSt is done: it was issued when the softmax was through with tile t - kSt - 2, so that this place, tile t - 8's, is free
      static_assert(kSt + 2 <= 8, "entries of eight tiles");
      if (half == 0 && lane == 0) {
        float* e = entries + (t & 7) * 4;
        e[2 + (key >> 5)] = __uint_as_float(nan);
        if (key == 0) e[0] = __uint_as_float(top - (kUp << 23)), e[1] = __uint_as_float(k_top - (kUp << 23));
      }
      const uint32_t vz = vp[S];
      request_k(t + kDeep, set);
      rd_umma::fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[st]);
      if (t >= kSt && !rd_umma::warp_wait(&v_empty[st], (t / kSt - 1) & 1, stop)) {
        ok = false, site = 2;
        return;
      }
      store(sV + st * L::kTile, vc[S], vz, v);
      request_v(t + kDeep, set);
      rd_umma::fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
    };
    using First = std::integral_constant<int, 0>;
    using Last = std::integral_constant<int, kDeep - 1>;
    request_k(0, First());
    request_v(0, First());
    if (kDeep == 2) {
      request_k(1, Last());
      request_v(1, Last());
    }
    for (int t = 0; ok && t < n_tiles; t += 2) {
      unpack(t, First());
      if (ok && t + 1 < n_tiles) unpack(t + 1, Last());
    }
  } else if (warp >= kIssue) {
    // ---------------- products: a warp for each tile of rows, so that neither waits for the other's softmax ----------------
    const int x = L::kParts == 1 ? warp - kIssue : 0;
    if (x < n_q && rd::elect_one()) {
      const uint32_t idesc_qk = idesc_fp16(kManyKeys, false), idesc_pv = idesc_fp16(HD, true);
      const uint32_t q = rd_umma::smem_u32(sQ + x * L::kQ), base = tmem + x * L::kCols;
      // S of tile t: its buffer held W of tile t - 2, whose product has been issued before; products run in that order
      auto scores = [&](int t) {
        const int st = t % kSt;
        if (!rd_umma::wait_or(&k_full[st], (t / kSt) & 1, stop)) return false;
        rd_umma::fence_after();
        const uint32_t k = rd_umma::smem_u32(sK + st * L::kTile);
#pragma unroll
        for (int kd = 0; kd < HD / 16; ++kd)
          rd_umma::mma_ss(base + L::kColS + (t & 1) * 64, rd_umma::desc_k_major(q + (kd >> 2) * (kManyRows * 128) + (kd & 3) * 32),
                          rd_umma::desc_k_major(k + (kd >> 2) * (kManyKeys * 128) + (kd & 3) * 32), idesc_qk, kd != 0);
        mbar_arrive(&s_full[2 * x + (t & 1)]);
        rd_umma::commit(&s_full[2 * x + (t & 1)]);
        rd_umma::commit(&k_empty[st]);
        return true;
      };
      ok = rd_umma::wait_or(&q_full[x], 0, stop);
      for (int t = 0; ok && t < 2 && t < n_tiles; ++t) ok = scores(t);
      for (int t = 0; ok && t < n_tiles; ++t) {
        const int st = t % kSt;
        ok = rd_umma::wait_or(&p_full[2 * x + (t & 1)], (t >> 1) & 1, stop) && rd_umma::wait_or(&v_full[st], (t / kSt) & 1, stop);
        if (!ok) break;
        rd_umma::fence_after();
        const uint32_t v = rd_umma::smem_u32(sV + st * L::kTile);
#pragma unroll
        for (int ks = 0; ks < kManyKeys / 16; ++ks)
          mma_ts(base + L::kColO, base + L::kColS + (t & 1) * 64 + ks * 8, rd_umma::desc_mn_major(v + ks * 2048, kManyKeys * 128), idesc_pv, (t | ks) != 0);
        rd_umma::commit(&o_full[2 * x + (t & 1)]);
        rd_umma::commit(&v_empty[st]);
        if (t + 2 < n_tiles) ok = scores(t + 2);
      }
      if (!ok) site = 3;
    }
    __syncwarp();
  } else if ((L::kParts == 1 ? warp >> 2 : 0) < n_q) {
    const int tile = L::kParts == 1 ? warp >> 2 : 0, quarter = warp & 3;
    uint8_t* myQ = sQ + tile * L::kQ;
    const int row = quarter * 32 + lane, R = q0 + tile * kManyRows + row;
    const bool live = R < rows;
    const int token = live ? R / group : 0, head = hk * group + (live ? R % group : 0);
    // ---------------- queries: eight lanes a row; bf16 goes where fp16 is to stand, and is converted there by who brought it ----------------
    {
      constexpr int kPart = HD / 8;  // features of a lane: 8 or 16
      const int eighth = lane & 7;
      const int64_t mine = (int64_t)(r.start + token) * a.ldq + head * HD;
      auto place = [&](int i, int c) {
        const int of = quarter * 32 + i * 4 + (lane >> 3), chunk = eighth * (kPart / 8) + c;
        return myQ + (chunk >> 3) * (kManyRows * 128) + of * 128 + (((chunk & 7) ^ (of & 7)) << 4);
      };
#pragma unroll 2
      for (int i = 0; i < 8; ++i) {
        const int64_t from = __shfl_sync(0xffffffffu, mine, i * 4 + (lane >> 3));
        const int there = __shfl_sync(0xffffffffu, live ? 16 : 0, i * 4 + (lane >> 3));  // bytes; zeros for the others
#pragma unroll
        for (int c = 0; c < kPart / 8; ++c)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(rd_umma::smem_u32(place(i, c))),
                       "l"((const __nv_bfloat16*)a.q + from + eighth * kPart + c * 8), "r"(there)
                       : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
      for (int i = 0; i < 8; ++i) {
        float x[kPart], most = 0.f;
#pragma unroll
        for (int c = 0; c < kPart / 8; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(place(i, c));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) x[8 * c + 2 * e] = __uint_as_float(w[e] << 16), x[8 * c + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
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
          *reinterpret_cast<uint4*>(place(i, c)) = make_uint4(pack_f16(y[0], y[1]), pack_f16(y[2], y[3]), pack_f16(y[4], y[5]), pack_f16(y[6], y[7]));
        }
        if (eighth == 0)
          units[tile * kManyRows + quarter * 32 + i * 4 + (lane >> 3)] =
              a.scale * 1.44269504f * __uint_as_float((uint32_t)(127 - h1) << 23) * __uint_as_float((uint32_t)(127 - h2) << 23);
      }
      rd_umma::fence_async_proxy();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[tile]);
    }
    // ---------------- softmax: a thread a row ----------------
    const float unit = units[tile * kManyRows + row];  // its own warp's
    const uint32_t taddr = tmem + tile * L::kCols + ((uint32_t)(quarter * 32) << 16);
    const int all_see = a.mode == RD_ATTN_CAUSAL ? min(kv_end, r.base + first_token + 1) : min(kv_end, r.base);
    float m_run = -INFINITY, l_run = 0.f, ref = 0.f;
    // A tile's weights (packed, 32 words) at the maximum m, scores in units of u; returns their sum.  odd: keys whose values are NaN.
    auto weigh = [&](auto whole, int t, uint64_t vis, uint64_t odd, float m, float u, uint32_t* w) {
      constexpr bool WHOLE = decltype(whole)::value;
      const float off = m == -INFINITY ? 0.f : kWeightBits - m;
      const F2 unit2 = pack2(u, u), off2 = pack2(off, off);
      F2 sum = 0;
      // sixteen scores are on their way while sixteen are weighted
      uint32_t s[2][16];
      const uint32_t from = taddr + L::kColS + (t & 1) * 64;
      tmem_ask16(from, s[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t* y = s[c & 1];
        tmem_have16(y);
        if (c < 3) tmem_ask16(from + 16 * (c + 1), s[(c + 1) & 1]);
        const uint32_t v = (uint32_t)(vis >> (16 * c)), o = (uint32_t)(odd >> (16 * c));
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          float x0, x1;
          unpack2(fma2(pack2(__uint_as_float(y[i]), __uint_as_float(y[i + 1])), unit2, off2), x0, x1);
          x0 = ex2(x0), x1 = ex2(x1);
          if (!WHOLE) {
            if (!((v >> i) & 1)) x0 = 0.f;
            if (!((v >> (i + 1)) & 1)) x1 = 0.f;
          }
          sum = add2(sum, pack2(x0, x1));
          if (!WHOLE) {
            if ((v & o) >> i & 1) x0 = __int_as_float(0x7fffffff);
            if ((v & o) >> (i + 1) & 1) x1 = __int_as_float(0x7fffffff);
          }
          w[8 * c + i / 2] = pack_f16(x0, x1);
        }
      }
      float s0, s1;
      unpack2(sum, s0, s1);
      return s0 + s1;
    };
    // the largest score that a row sees
    auto largest = [&](int t, uint64_t vis) {
      float top = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t x[16];
        tmem_ld16(taddr + L::kColS + (t & 1) * 64 + 16 * c, x);
        const uint32_t v = (uint32_t)(vis >> (16 * c));
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, (v >> i) & 1 ? __uint_as_float(x[i]) : -INFINITY);
      }
      return top;
    };
    for (int t = 0; t < n_tiles; ++t) {
      if (!rd_umma::warp_wait(&s_full[2 * tile + (t & 1)], (t >> 1) & 1, stop)) {
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
      const float4 entry = *reinterpret_cast<const float4*>(entries + (t & 7) * 4);
      const float ref_t = entry.x, u = unit * entry.y;
      const uint64_t odd = (uint64_t)__float_as_uint(entry.z) | (uint64_t)__float_as_uint(entry.w) << 32;
      uint32_t w[32];
      float sum;
#pragma unroll 1
      for (bool again = false;; again = true) {
        sum = whole && odd == 0 ? weigh(std::true_type(), t, vis, odd, m_run, u, w) : weigh(std::false_type(), t, vis, odd, m_run, u, w);
        // seldom: the first keys that a row sees, weights too large, a larger r.  At the tile's own maximum 64 weights come to 2^13 at most.
        const bool low = m_run == -INFINITY || sum > kMostWeights;
        if (again || !__any_sync(0xffffffffu, low || ref_t != ref)) break;
        const float top = largest(t, vis) * u;
        float keep = ref / ref_t;  // what O is to be multiplied with
        if (low && top > m_run) {
          const float alpha = m_run == -INFINITY ? 0.f : ex2(m_run - top);
          l_run *= alpha;
          if (m_run != -INFINITY) keep *= alpha;
          m_run = top;
        }
        ref = ref_t;
        if (t == 0) continue;
        // O has to be quiet
        if (!rd_umma::warp_wait(&o_full[2 * tile + ((t - 1) & 1)], ((t - 1) >> 1) & 1, stop)) {
          ok = false, site = 5;
          break;
        }
        rd_umma::fence_after();
#pragma unroll 1
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t x[16];
          tmem_ld16(taddr + L::kColO + c * 16, x);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * keep);
          tmem_st16(taddr + L::kColO + c * 16, x);
        }
      }
      if (!ok) break;
      l_run += sum;
      tmem_st16(taddr + L::kColS + (t & 1) * 64, w);
      tmem_st16(taddr + L::kColS + (t & 1) * 64 + 16, w + 16);
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      rd_umma::fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * tile + (t & 1)]);
    }
    if (ok && n_tiles > 0) {
      ok = rd_umma::warp_wait(&o_full[2 * tile + ((n_tiles - 1) & 1)], ((n_tiles - 1) >> 1) & 1, stop);
      if (!ok) site = 6;
    }
    if (ok) {
      rd_umma::fence_after();
      const int64_t at = (int64_t)(r.start + token) * a.nh + head;
      float* to = partial + (at * n_split + split) * kShareFloats<HD>;
      const float f = n_split > 1 ? ref : (l_run == 0.f ? 0.f : ref / l_run);  // the weights' 2^7 is in O and in l
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        float x[32], y[32];
        if (n_tiles > 0) {
          rd_umma::tmem_ld32(taddr + L::kColO + c * 32, x);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) y[i] = f == 0.f ? 0.f : x[(i & 24) + order8<BITS>(i & 7)] * f;
        if (!live) continue;
        if (n_split > 1) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<float4*>(to + c * 32 + 4 * i) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
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
  if (*stop)
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // products in flight read and write shared memory and TMEM
  if (warp == kIssue) {
    rd_umma::fence_after();
    rd_umma::tmem_dealloc(tmem_slot, L::kTmem);
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
  const float* p = partial + at * n_split * kShareFloats<HD>;
  const float mine = lane < n_split ? p[lane * kShareFloats<HD> + HD] : -INFINITY;
  const float top = rd::warp_max(mine);
  float sum = 0.f, v[HD / 32] = {};
#pragma unroll 4
  for (int c = 0; c < n_split; ++c) {
    const float* x = p + c * kShareFloats<HD>;
    const float mc = x[HD], f = mc == -INFINITY ? 0.f : ex2(mc - top);
    sum += f * x[HD + 1];
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) v[k] += f == 0.f ? 0.f : f * x[k * 32 + lane];
  }
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) ((__nv_bfloat16*)a.out)[at * HD + k * 32 + lane] = __float2bfloat16_rn(sum == 0.f ? 0.f : v[k] / sum);
}

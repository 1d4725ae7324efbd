// Attention over a cache in codes for few query rows to a key/value head (a decode step: the query heads of a group times the new tokens
// of a row, up to 16): included by attention_quant.cu.
//
// Such a call is bound by the bytes of the codes.  A warp takes a tile of keys at a time (2 KB of key codes, 2 KB of value codes, brought by TMA into
// a ring of its own) and multiplies it on the warp-level tensor cores, codes as they lie: a code in the low bits of a 16-bit word is
// the fp16 number code * 2^-24, a code four bits higher 16 times that, so two of them are formed by one masking instruction.  (tcgen05 would want
// the operands in shared memory or TMEM: writing the unpacked codes there costs more than these products, 8 columns wide.)
//   S^T = K Q^T   A: 16 keys x 16 features of codes, B: 8 query rows, scaled by a power of two to fp16 (bf16's 8 bits fit) and, where the codes
//                 are 16 times too large, by 1/16.  score = scale_k (S - zero_k sum q).
//   O^T += V^T W  A: 16 features x 16 keys of codes, B: W = p scale_v / r 2^14 in fp16, where r is the largest value scale so far: weights
//                 keep fp16's 11 bits down to 2^-28 of the largest.  What the zeros come to, sum W zero, is one number for a row of
//                 queries and is taken off its features every eight tiles: until then O's fp32 holds at most some 2000 codes too much.
//                 Codes of 4 bits are all taken four bits up here: the tensor core cuts a sum some 24 bits below what its factors' exponents allow for,
//                 and with factors of code * 2^-24 that was 2^-19 of the largest value, moved that is 2^-23, as for codes of 8 bits.  Each
//                 of the n keys is cut there: where one key has nearly all the weight and a value near 0, the others' part is off by up to n 2^-24 of the
//                 largest value (22 keys against one of weight 0.99995: 6 10^-7 of it).
// The accumulators' layouts fit: a lane holds the same query columns in S^T and in O^T, so the running maximum and sum need no
// exchange but the maximum's over the 8 lanes of a column, and only where some lane's exceeds it; the weights become a B operand by
// movmatrix.
// Shared memory lies in TMA's 128-byte swizzle, and the 16 keys of a product are taken in an order (Shape::key) in which both the reads of K
// (16 bytes of 8 keys) and of V (4 to 16 bytes of 4 keys) touch every bank once.
//
// Work is cut on the device, where the rows' lengths are known: chains (row, key/value head) in chunks of equal length.
//
// Measured on one B200: 16 rows of 105000 keys in all, 32 heads of 128 features with keys of their own, 8 bits, 138 us, 5.4 TB/s of codes (a copy reaches
// 6.6): schedulers issue in 57 % of the cycles, the vector pipes are busy for 47, memory for 69.  One row of 131072 keys, 8 heads of 4 bits, four query heads
// each: 42 us, 3.4 TB/s, of which some 8 until the first products and 3 for the sum of the chunks.  One row of 1001 keys: 9.6 us, trips to memory one
// after another (lengths, codes, queries, chunks) and two launches.

constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewStages = 3;
constexpr int kTileBytes = 2048;  // of key codes, and of value codes
constexpr int kFewRows = 16;      // query rows at most

template <int HD, int BITS>
struct Shape {
  static constexpr int kRowBytes = HD * BITS / 8;
  static constexpr int kKeys = kTileBytes / kRowBytes;  // of a tile: 16, 32 or 64
  static constexpr int kWords = kRowBytes / 16;         // 32-bit words of a key that a lane holds for S^T
  static constexpr int kPer = 32 / BITS;                // codes of a word
  static constexpr int kSteps = HD / 16;                // products along the features
  static constexpr int kStage = 2 * kTileBytes + 2 * 64 * 4;  // codes, then the parameters of up to 64 keys and values
  // the key of a sub-tile of 16 whose scores are row i of a product
  static __device__ __forceinline__ int key(int i) {
    const int i0 = i & 1, i1 = (i >> 1) & 1, i2 = (i >> 2) & 1, i3 = i >> 3;
    if constexpr (kRowBytes == 128) return i0 | (i1 << 1) | ((i2 ^ i0) << 2) | (i3 << 3);
    else if constexpr (kRowBytes == 64) return i0 | (i3 << 1) | (i1 << 2) | (i2 << 3);
    else return i0 | (i1 << 1) | (i3 << 2) | (i2 << 3);
  }
  // byte `at` of key `k` of a tile, in the swizzled tile
  static __device__ __forceinline__ uint32_t place(int k, int at) {
    const uint32_t b = k * kRowBytes + at;
    return b ^ ((b >> 3) & 0x70);
  }
  // the place of a byte of sub-tile u from its tile's first byte (a multiple of 1024) and its place in sub-tile 0
  static __device__ __forceinline__ uint32_t in_sub(uint32_t tile, uint32_t at, int u) {
    const uint32_t b = tile + at + u * 16 * kRowBytes;
    return kRowBytes == 32 && (u & 1) ? b ^ 64 : b;  // 512 bytes on, the swizzle's third bit is another
  }
  // first feature of word w of a lane with t = lane % 4
  static __device__ __forceinline__ int feature(int t, int w) {
    if constexpr (kWords == 8) return (w >> 2) * 64 + t * 16 + (w & 3) * 4;
    else return t * (HD / 4) + w * kPer;
  }
};

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t x;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at) : "memory");
  return x;
}
__device__ __forceinline__ void lds64(uint32_t at, uint32_t* x) { asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(at) : "memory"); }
__device__ __forceinline__ void lds128(uint32_t at, uint32_t* x) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(rd_umma::smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(rd_umma::smem_u32(bar))
               : "memory");
}

// Rounds of row b: its tiles (at multiples of KEYS slots) over the warps of a CTA; one where there are new tokens and no keys, for the zeros that they get.
template <int KEYS>
__device__ __forceinline__ int rounds_of(const Args& a, int b) {
  const Row r = row_of(a, b);
  if (r.n_new <= 0) return 0;
  if (r.end <= 0) return 1;
  const int tiles = (int)((uint32_t)(r.first + r.end + KEYS - 1) / KEYS - (uint32_t)r.first / KEYS);
  return (tiles + kFewWarps - 1) / kFewWarps;
}
// All rows' rounds, those of the first kListed rows in shared memory: the choice below asks for them again and again.  (Reading the rows' lengths anew
// each time cost a call of one row 2.6 us, one of 131072 keys 5.)
constexpr int kListed = 512;
template <int KEYS>
struct Rounds {
  const Args& a;
  const int* listed;
  __device__ __forceinline__ int operator()(int b) const { return b < kListed ? listed[b] : rounds_of<KEYS>(a, b); }
};
__device__ __forceinline__ int chunks_of(int rounds, int chunk) { return (int)((uint32_t)(rounds + chunk - 1) / (uint32_t)chunk); }
// Items of all rows at this chunk; one warp.
template <typename R>
__device__ __forceinline__ int count_items(const Args& a, const R& rounds, int chunk) {
  int n = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) n += chunks_of(rounds(b), chunk);
  return rd::warp_sum_i(n) * a.nkv;
}
// The chunk of a launch of `slots` CTAs; one warp, the same answer in every CTA.  One item to a CTA if that fills them evenly: the smallest chunk that
// leaves no more items than CTAs is at most 1.25 times what an even share would be.  Otherwise four items to a CTA, one after another.
template <typename R>
__device__ __forceinline__ int choose_chunk(const Args& a, const R& rounds, int slots) {
  int total = 0, most = 0;
  for (int b = threadIdx.x & 31; b < a.B; b += 32) {
    const int r = rounds(b);
    total += r;
    most = max(most, r);
  }
  total = rd::warp_sum_i(total);
  most = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
  if (most == 0) return 1;
  const int64_t work = (int64_t)total * a.nkv;
  int lo = (int)max((work + slots - 1) / slots, (int64_t)1);  // a chunk in [lo, hi] is looked for
  if (lo >= most) return most;
  int hi = min(most, lo + lo / 4);
  if (count_items(a, rounds, hi) > slots) return (int)max((work + 4 * slots - 1) / (4 * slots), (int64_t)1);
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (count_items(a, rounds, mid) <= slots) hi = mid;
    else lo = mid + 1;
  }
  return hi;
}
struct Item {
  int b, head, index, of;  // row, key/value head, chunk of the chain, chunks of the chain
};
// Item i; one warp, all lanes the same answer.  b = -1: there are fewer.  The heads of a chunk come one after another.
template <typename R>
__device__ __forceinline__ Item find_item(const Args& a, const R& rounds, int chunk, int i) {
  Item it{-1, 0, 0, 0};
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int chunks = b0 + lane < a.B ? chunks_of(rounds(b0 + lane), chunk) : 0;
    int sum = chunks * a.nkv;
    const int mine = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + sum > i);
    if (past != 0) {
      const int who = __ffs(past) - 1;
      const int start = before + __shfl_sync(0xffffffffu, sum - mine, who);
      it.of = __shfl_sync(0xffffffffu, chunks, who);
      it.b = b0 + who;
      it.index = (int)((uint32_t)(i - start) / (uint32_t)a.nkv);
      it.head = (i - start) - it.index * a.nkv;
      return it;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return it;
}

// The workspace: a header of one int (the chunk), then for every item its rows' unnormalised outputs, maxima (base 2) and sums.
constexpr int kFewHeader = 256;
__host__ __device__ constexpr int64_t few_item_floats(int hd, int rows) { return (int64_t)rows * (hd + 2); }

template <int HD, int BITS, int NT>
struct FewSmem {
  static constexpr int kRing = kFewWarps * kFewStages * Shape<HD, BITS>::kStage;
  static constexpr int kMerge = kFewWarps * 8 * NT * (HD + 4) * 4;  // outputs, then maxima and sums, of all warps
  static constexpr int kBytes = 1024 + (kRing > kMerge ? kRing : kMerge) + kFewWarps * kFewStages * 8 + 16;
};

template <int HD, int BITS, int NT>
__global__ void __launch_bounds__(kFewThreads, NT == 1 ? 2 : 1)
    attention_quant_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Args a, float* partial, int slots,
                               int* header, int32_t* status) {
  using S = Shape<HD, BITS>;
  constexpr int kKeys = S::kKeys, kSub = kKeys / 16, kMT = HD / 16;
  constexpr int kRows = 8 * NT;
  extern __shared__ uint8_t raw[];
  __shared__ int listed[kListed];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  using Sm = FewSmem<HD, BITS, NT>;
  constexpr int kData = Sm::kRing > Sm::kMerge ? Sm::kRing : Sm::kMerge;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kData);
  volatile int* gave_up = reinterpret_cast<volatile int*>(bars + kFewWarps * kFewStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* full = bars + warp * kFewStages;
  // tiles of all warps first (their swizzle wants 1024 bytes of alignment), then the parameters
  uint8_t* codes = smem + warp * kFewStages * 2 * kTileBytes;
  uint32_t* params = reinterpret_cast<uint32_t*>(smem + kFewWarps * kFewStages * 2 * kTileBytes) + warp * kFewStages * 128;
  rd::pdl_launch_dependents();
  if (threadIdx.x == 0) *gave_up = 0;
  if (lane == 0) {
    for (int s = 0; s < kFewStages; ++s) rd_umma::mbar_init(&full[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  rd::pdl_wait();
  for (int b = threadIdx.x; b < a.B && b < kListed; b += kFewThreads) listed[b] = rounds_of<kKeys>(a, b);
  __syncthreads();
  const Rounds<kKeys> rounds{a, listed};
  const int chunk = choose_chunk(a, rounds, slots);
  if (blockIdx.x == 0 && threadIdx.x == 0 && header != nullptr) *header = chunk;
  const int group = a.nh / a.nkv;
  const int64_t plane_rows = (int64_t)a.B * a.nkv * a.max_len;
  // where a lane reads: key codes of rows g and g + 8 of a product, value codes of rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9, parameters of the former
  const uint32_t codes_u32 = rd_umma::smem_u32(codes), params_u32 = rd_umma::smem_u32(params);
  uint32_t k_at[2], v_at[4], p_at[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) k_at[x] = S::place(S::key(g + 8 * x), t * (S::kWords == 2 ? 8 : 16)), p_at[x] = 4 * S::key(g + 8 * x);
#pragma unroll
  for (int x = 0; x < 4; ++x) v_at[x] = S::place(S::key(2 * t + (x & 1) + 8 * (x >> 1)), g * (S::kRowBytes / 8));
  uint32_t used = 0;  // tiles that this warp has waited for so far: stage and phase
  bool ok = true;
  for (int item = blockIdx.x; ok; item += gridDim.x) {
    const Item it = find_item(a, rounds, chunk, item);
    if (it.b < 0) break;
    const Row r = row_of(a, it.b);
    const int64_t chain = (int64_t)it.b * a.nkv + it.head;
    const int64_t slot0 = chain * a.max_len;  // row of the planes
    const int tile_first = r.first / kKeys, tile_end = (r.first + r.end + kKeys - 1) / kKeys;
    const int from = tile_first + it.index * chunk * kFewWarps, to = min(tile_end, from + chunk * kFewWarps);
    const int mine = from + warp < to ? (to - from - warp + kFewWarps - 1) / kFewWarps : 0;
    auto load = [&](int i) {  // tile i of this warp, one lane
      const uint32_t stage = (used + i) % kFewStages;
      const int64_t row = slot0 + (int64_t)(from + warp + i * kFewWarps) * kKeys;
      const uint32_t n = (uint32_t)min((int64_t)kKeys, plane_rows - row) * 4;
      rd_umma::mbar_expect_tx(&full[stage], 2 * kTileBytes + 2 * n);
      const int line = (int)(row / (128 / S::kRowBytes));
      rd_umma::tma_load_2d(codes + stage * 2 * kTileBytes, &map_k, &full[stage], 0, line);
      rd_umma::tma_load_2d(codes + stage * 2 * kTileBytes + kTileBytes, &map_v, &full[stage], 0, line);
      bulk_load(params + stage * 128, a.k_params + row, n, &full[stage]);
      bulk_load(params + stage * 128 + 64, a.v_params + row, n, &full[stage]);
    };
    if (rd::elect_one())
      for (int i = 0; i < kFewStages && i < mine; ++i) load(i);
    __syncwarp();

    // the queries: row n * 8 + g is head (row % group) of new token row / group; a lane holds its share of the features
    const int rows = r.n_new * group;
    uint32_t q[NT][S::kSteps][2];
    float q_sum[NT][2], unit[NT][2];  // of the columns 2 t, 2 t + 1 of a block of rows: 2^-24 sum q, and what a score is to be multiplied with
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = n * 8 + g;
      float x[HD / 4];
      const bool live = row < rows;
      const __nv_bfloat16* src = (const __nv_bfloat16*)a.q + (int64_t)(r.start + (live ? row / group : 0)) * a.ldq + (it.head * group + (live ? row % group : 0)) * HD;
#pragma unroll
      for (int w = 0; w < S::kWords; ++w) {
        const int d = S::feature(t, w);
#pragma unroll
        for (int e = 0; e < S::kPer; e += 4) {
          const uint2 u = live ? *reinterpret_cast<const uint2*>(src + d + e) : make_uint2(0u, 0u);
          x[w * S::kPer + e] = __uint_as_float(u.x << 16), x[w * S::kPer + e + 1] = __uint_as_float(u.x & 0xffff0000u);
          x[w * S::kPer + e + 2] = __uint_as_float(u.y << 16), x[w * S::kPer + e + 3] = __uint_as_float(u.y & 0xffff0000u);
        }
      }
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 4; ++i) top = fmaxf(top, fabsf(x[i]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row's largest to [2^14, 2^15): what is below 2^-38 of it is lost.  2^(141 - e) and its inverse, in two factors each, because e
      // runs over all of fp32's exponents.
      const int e = top > 0.f && top < INFINITY ? (int)(__float_as_uint(top) >> 23) : 141;
      const int up = 141 - e, h1 = up / 2, h2 = up - h1;
      const float f1 = __uint_as_float((uint32_t)(127 + h1) << 23), f2 = __uint_as_float((uint32_t)(127 + h2) << 23);
      const float i1 = __uint_as_float((uint32_t)(127 - h1) << 23), i2 = __uint_as_float((uint32_t)(127 - h2) << 23);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < S::kWords; ++w) {
        float* y = x + w * S::kPer;
#pragma unroll
        for (int i = 0; i < S::kPer; ++i) y[i] = y[i] * f1 * f2;
        if constexpr (BITS == 4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // codes i and i + 4 of a word share a register; those of odd i are 16 times too large
            const float f = (i & 1) ? 0.0625f : 1.f;
            const uint32_t u = pack_f16(y[i] * f, y[i + 4] * f);
            q[n][2 * w + i / 2][i & 1] = u;
            sum += (__half2float(__ushort_as_half((unsigned short)u)) + __half2float(__ushort_as_half((unsigned short)(u >> 16)))) / f;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t u = pack_f16(y[i], y[i + 2]);
            q[n][w][i] = u;
            sum += __half2float(__ushort_as_half((unsigned short)u)) + __half2float(__ushort_as_half((unsigned short)(u >> 16)));
          }
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // log2(e) scale 2^24 / the queries' factor: scores in base 2
      const float back = a.scale * 1.44269504f * 16777216.f * i1 * i2;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        q_sum[n][c] = __shfl_sync(0xffffffffu, sum, 4 * (2 * t + c)) * 0x1p-24f;
        unit[n][c] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + c));
      }
    }

    float o[NT][kMT][4], m[NT][2], l[NT][2], z[NT][2], ref = 0.f, inv_ref = 0.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < kMT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = z[n][0] = z[n][1] = 0.f;
    }
    // O holds sums of codes; their zeros' part, the same for all features of a row, is taken off here
    auto centre = [&]() {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          f[c] = z[n][c];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) f[c] += __shfl_xor_sync(0xffffffffu, f[c], x);
          f[c] *= BITS == 4 ? 0x1p-20f : 0x1p-24f;
          z[n][c] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < kMT; ++k) {
          o[n][k][0] -= f[0], o[n][k][1] -= f[1], o[n][k][2] -= f[0], o[n][k][3] -= f[1];
        }
      }
    };
    // One tile; kt: its codes in shared memory, pt: its parameters.  WHOLE: every row sees every key.
    auto tile = [&](auto whole, uint32_t kt, uint32_t pt, int j0) {
      constexpr bool WHOLE = decltype(whole)::value;
      float s[NT][kSub][4], sv[kSub][2], zv[kSub][2], most = 0.f, mx[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        uint32_t w[2][S::kWords];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t at = S::in_sub(kt, k_at[x], u);
          if constexpr (S::kWords == 2) lds64(at, w[x]);
          else lds128(at, w[x]);
          if constexpr (S::kWords == 8) lds128(at ^ 64, w[x] + 4);
        }
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
        for (int y = 0; y < S::kWords; ++y) {
          if constexpr (BITS == 4) {
            const uint32_t b0 = w[0][y] >> 8, b1 = w[1][y] >> 8;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_f16(acc[n], w[0][y] & 0x000f000fu, w[1][y] & 0x000f000fu, w[0][y] & 0x00f000f0u, w[1][y] & 0x00f000f0u, q[n][2 * y][0], q[n][2 * y][1]);
              mma_f16(acc[n], b0 & 0x000f000fu, b1 & 0x000f000fu, b0 & 0x00f000f0u, b1 & 0x00f000f0u, q[n][2 * y + 1][0], q[n][2 * y + 1][1]);
            }
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_f16(acc[n], w[0][y] & 0x00ff00ffu, w[1][y] & 0x00ff00ffu, __byte_perm(w[0][y], 0, 0x4341), __byte_perm(w[1][y], 0, 0x4341), q[n][y][0], q[n][y][1]);
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t at = pt + p_at[x] + u * 64;
          const uint32_t pk = lds32(at), pv = lds32(at + 256);
          const float sk = param_scale(pk), zk = code_as_float(param_zero(pk));
          sv[u][x] = param_scale(pv);
          zv[u][x] = code_as_float(param_zero(pv));
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) s[n][u][2 * x + c] = fmaf(-zk, q_sum[n][c], acc[n][2 * x + c]) * sk;
          if constexpr (!WHOLE) {
            const int j = j0 + u * 16 + S::key(g + 8 * x);
            const bool there = j >= 0 && j < r.end;
            if (!there) sv[u][x] = zv[u][x] = 0.f;  // whatever lies there
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int row = n * 8 + 2 * t + c;
                if (!(there && row < rows && (j < r.base || sees(a, r, row / group, j)))) s[n][u][2 * x + c] = -INFINITY;
              }
          }
          most = fmaxf(most, sv[u][x]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mx[n][0] = fmaxf(mx[n][0], s[n][u][2 * x]), mx[n][1] = fmaxf(mx[n][1], s[n][u][2 * x + 1]);
        }
      }
      bool more = most > ref;
#pragma unroll
      for (int n = 0; n < NT; ++n) more |= mx[n][0] > m[n][0] || mx[n][1] > m[n][1];
      if (__any_sync(0xffffffffu, more)) {
        // a larger maximum or a larger value scale: what has been summed so far is brought to it
        float top = fmaxf(most, ref);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        // not below 2^-112, so that its inverse stays finite; at that the weights of a value whose scale is 2^-126 are still p
        top = fmaxf(top, 0x1p-112f);
        const float back = ref / top;
        ref = top;
        inv_ref = 16384.f / ref;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(mx[n][c], m[n][c]);
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, y));
            f[c] = m[n][c] == -INFINITY ? 0.f : ex2((m[n][c] - x) * unit[n][c]);
            m[n][c] = x;
            l[n][c] *= f[c];
            f[c] *= back;
            z[n][c] *= f[c];
          }
#pragma unroll
          for (int k = 0; k < kMT; ++k) o[n][k][0] *= f[0], o[n][k][1] *= f[1], o[n][k][2] *= f[0], o[n][k][3] *= f[1];
        }
      }
      float off[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) off[n][c] = m[n][c] == -INFINITY ? 0.f : -m[n][c] * unit[n][c];
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        constexpr int kVWords = S::kRowBytes / 32;  // words of a key that a lane holds: features g * HD / 8 ..
        uint32_t w[4][kVWords], b[NT][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t at = S::in_sub(kt + kTileBytes, v_at[x], u);
          if constexpr (kVWords == 1) w[x][0] = lds32(at);
          else if constexpr (kVWords == 2) lds64(at, w[x]);
          else lds128(at, w[x]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float f = sv[u][x] * inv_ref;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float p0 = ex2(fmaf(s[n][u][2 * x], unit[n][0], off[n][0])), p1 = ex2(fmaf(s[n][u][2 * x + 1], unit[n][1], off[n][1]));
            l[n][0] += p0;
            l[n][1] += p1;
            float w0 = p0 * f, w1 = p1 * f;
            if constexpr (!WHOLE) w0 = p0 == 0.f ? 0.f : w0, w1 = p1 == 0.f ? 0.f : w1;  // a hidden value counts for nothing, NaN or not
            const uint32_t h = pack_f16(w0, w1);
            z[n][0] = fmaf(__low2float(*reinterpret_cast<const __half2*>(&h)), zv[u][x], z[n][0]);  // the weights as the products have them
            z[n][1] = fmaf(__high2float(*reinterpret_cast<const __half2*>(&h)), zv[u][x], z[n][1]);
            b[n][x] = transpose8x8(h);
          }
        }
        // the values of the keys whose weights this lane's B registers hold: rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int y = 0; y < kVWords; ++y) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // two bytes of each of two keys: four features of 4 bits, or two of 8
            const uint32_t c0 = __byte_perm(w[0][y], w[1][y], half ? 0x7632 : 0x5410), c1 = __byte_perm(w[2][y], w[3][y], half ? 0x7632 : 0x5410);
            if constexpr (BITS == 4) {
              const uint32_t e0 = c0 << 4, e1 = c1 << 4, f0 = c0 >> 4, f1 = c1 >> 4, h0 = c0 >> 8, h1 = c1 >> 8;
              constexpr uint32_t kMask = 0x00f000f0u;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma_f16(o[n][4 * y + 2 * half], e0 & kMask, c0 & kMask, e1 & kMask, c1 & kMask, b[n][0], b[n][1]);
                mma_f16(o[n][4 * y + 2 * half + 1], f0 & kMask, h0 & kMask, f1 & kMask, h1 & kMask, b[n][0], b[n][1]);
              }
            } else {
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma_f16(o[n][2 * y + half], c0 & 0x00ff00ffu, __byte_perm(c0, 0, 0x4341), c1 & 0x00ff00ffu, __byte_perm(c1, 0, 0x4341), b[n][0], b[n][1]);
            }
          }
        }
      }
    };
#pragma unroll 1
    for (int i = 0; i < mine; ++i) {
      const uint32_t stage = (used + i) % kFewStages;
      if (!__all_sync(0xffffffffu, rd_umma::mbar_wait(&full[stage], ((used + i) / kFewStages) & 1))) {
        ok = false;
        break;
      }
      const int j0 = (from + warp + i * kFewWarps) * kKeys - r.first;  // key of the tile's first slot
      const uint32_t kt = codes_u32 + stage * 2 * kTileBytes, pt = params_u32 + stage * 512;
      if (j0 >= 0 && j0 + kKeys <= min(r.base, r.end)) tile(std::true_type(), kt, pt, j0);
      else tile(std::false_type(), kt, pt, j0);
      __syncwarp();  // every lane has read its part of the stage
      if (i + kFewStages < mine && rd::elect_one()) load(i + kFewStages);
      __syncwarp();
      // often enough that the sums of codes stay near those of the values that they stand for
      if ((i & 7) == 7) centre();
    }
    centre();
    used += mine;
    if (!ok) *gave_up = 1;

    // The warps' results meet in shared memory, where the rings were: no copy is under way any more.
    __syncthreads();
    if (*gave_up) {
      ok = false;
      break;
    }
    float* so = reinterpret_cast<float*>(smem);                       // [warp][row][HD + 2]: a row's stride shifts the banks
    float* ss = so + kFewWarps * kRows * (HD + 2);                    // [warp][row][2]
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[n][c];
#pragma unroll
        for (int o2 = 4; o2 < 32; o2 <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o2);
        const int row = n * 8 + 2 * t + c;
        constexpr float kBack = BITS == 4 ? 64.f : 1024.f;  // the codes' 2^20 or 2^24 over the weights' 2^14
        float* dst = so + (warp * kRows + row) * (HD + 2);
#pragma unroll
        for (int k = 0; k < kMT; ++k) {
          dst[g * (HD / 8) + 2 * k] = o[n][k][c] * kBack * ref;
          dst[g * (HD / 8) + 2 * k + 1] = o[n][k][2 + c] * kBack * ref;
        }
        if (g == 0) {
          ss[(warp * kRows + row) * 2] = m[n][c] == -INFINITY ? -INFINITY : m[n][c] * unit[n][c];
          ss[(warp * kRows + row) * 2 + 1] = sum;
        }
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < min(rows, kRows) * HD; x += kFewThreads) {
      const int row = x / HD, d = x - row * HD;
      float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, ss[(w * kRows + row) * 2]);
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float mw = ss[(w * kRows + row) * 2];
        const float f = mw == -INFINITY ? 0.f : ex2(mw - top);
        sum += f * ss[(w * kRows + row) * 2 + 1];
        v += mw == -INFINITY ? 0.f : f * so[(w * kRows + row) * (HD + 2) + d];
      }
      if (it.of == 1) {
        const int64_t at = ((int64_t)(r.start + row / group) * a.nh + it.head * group + row % group) * HD + d;
        ((__nv_bfloat16*)a.out)[at] = __float2bfloat16_rn(sum == 0.f ? 0.f : v / sum);
      } else {
        float* dst = partial + item * few_item_floats(HD, kRows) + row * (HD + 2);
        dst[d] = v;
        if (d == 0) dst[HD] = top, dst[HD + 1] = sum;
      }
    }
    __syncthreads();
    // The next item's copies go where generic writes have just been
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
  if (!ok) {
    if (status && threadIdx.x == 0) atomicExch(status, 41);
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land
  }
}

// Sums the chunks of the chains that have several.  A CTA for each query row of each chain, its warps a share of the chunks each: a trip to
// memory for every eight chunks.
template <int HD, int KEYS>
__global__ void __launch_bounds__(256) attention_quant_merge_kernel(const Args a, const float* partial, const int* header, int item_rows) {
  __shared__ float vs[8][HD], sums[8][2];
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = a.nh / a.nkv;
  const int head = blockIdx.x / item_rows, row = blockIdx.x - head * item_rows;
  const int chunk = *reinterpret_cast<const volatile int*>(header);
  const Row r = row_of(a, b);
  if (row >= r.n_new * group) return;
  const int n = chunks_of(rounds_of<KEYS>(a, b), chunk);
  if (n <= 1) return;
  int before = 0;
  for (int x = lane; x < b; x += 32) before += chunks_of(rounds_of<KEYS>(a, x), chunk);
  before = rd::warp_sum_i(before) * a.nkv;
  const int64_t step = few_item_floats(HD, item_rows) * a.nkv;
  const float* p = partial + (before + head) * few_item_floats(HD, item_rows) + row * (HD + 2);
  float top = -INFINITY, sum = 0.f, v[HD / 32] = {};
#pragma unroll 4
  for (int c = warp; c < n; c += 8) {
    const float* x = p + c * step;
    const float mc = x[HD], lc = x[HD + 1];
    float y[HD / 32];
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) y[k] = x[k * 32 + lane];
    const float t = fmaxf(top, mc);
    const float f = top == -INFINITY ? 0.f : ex2(top - t), fc = mc == -INFINITY ? 0.f : ex2(mc - t);
    top = t;
    sum = sum * f + lc * fc;
#pragma unroll
    for (int k = 0; k < HD / 32; ++k) v[k] = v[k] * f + (mc == -INFINITY ? 0.f : y[k] * fc);
  }
#pragma unroll
  for (int k = 0; k < HD / 32; ++k) vs[warp][k * 32 + lane] = v[k];
  if (lane == 0) sums[warp][0] = top, sums[warp][1] = sum;
  __syncthreads();
  if (threadIdx.x >= HD) return;
  float all = -INFINITY, total = 0.f, out = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) all = fmaxf(all, sums[w][0]);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float f = sums[w][0] == -INFINITY ? 0.f : ex2(sums[w][0] - all);
    total += sums[w][1] * f;
    out += f == 0.f ? 0.f : vs[w][threadIdx.x] * f;
  }
  ((__nv_bfloat16*)a.out)[((int64_t)(r.start + row / group) * a.nh + head * group + row % group) * HD + threadIdx.x] = __float2bfloat16_rn(total == 0.f ? 0.f : out / total);
}

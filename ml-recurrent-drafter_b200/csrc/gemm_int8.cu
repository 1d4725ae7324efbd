// Products of matrices held in 8-bit integers with a scale for each row: C[t, n] = sA[t] sW[n] sum_k A[t, k] W[n, k], and the quantiser of
// their rows.  A row x of K values: scale = bf16(max |x| / 127) in fp32, code = rint(x / scale) cut to -127 .. 127; the scale's 8 significant
// bits make fp32's division give the codes of exact arithmetic (cache_quant.cu has the argument).  The sums are integers and exact.
#include <atomic>
#include <type_traits>

#include "quant.cuh"
#include "umma.cuh"

namespace {


// One block a row, 8 values of a thread at a time; rows of up to kQuantHeld * 8 * THREADS values stay in registers between the maximum and the
// codes, what is longer is read again.  A few rows are bound by a trip to memory: these have blocks of 1024 threads (one row of 4096 values 2.0 us, 110
// of 11008 2.6).  Many are bound by how little is asked for at once: what is held, as fp32, takes 89 registers a thread, so that two blocks are on an SM (4095 of
// 4096 values 19.5 us, 2.6 TB/s: issue slots 40 %, memory 14, warps wait for their loads).  VEC: rows on 16-byte boundaries, K a multiple of 8.

template <bool Bits8>
__device__ __forceinline__ uint32_t int8_code(float x, const rd_quant::Divider<Bits8>& by) {
  return (uint32_t)min(max((int)(by.rint_bits(x) - rd_quant::kRintBias), -127), 127) & 0xffu;
}
template <typename T, bool VEC>
__device__ __forceinline__ void load_row8(const T* row, int i, int K, float* x) {
  if constexpr (VEC && sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + i);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  } else if constexpr (VEC) {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(row + i);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(row + i + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = i + e < K ? rd::Num<T>::to_f(row[i + e]) : 0.f;
  }
}

template <typename T, bool VEC, int THREADS>
__global__ void __launch_bounds__(THREADS) quant_rows_kernel(const T* x, int64_t ldx, int8_t* codes, int64_t ld_codes, float* scales, int m_max,
                                                                   const int32_t* m_dev, int K) {
  constexpr int kQuantHeld = THREADS == 1024 ? 2 : 6;
  __shared__ float red[THREADS / 32];
  rd::pdl_wait();
  rd::pdl_launch_dependents();  // after the wait: a product that follows may read what was complete before this kernel began
  const int t = blockIdx.x;
  if (t >= rd::live_rows(m_dev, m_max)) return;
  const T* row = x + (int64_t)t * ldx;
  int8_t* to = codes + (int64_t)t * ld_codes;
  constexpr int kStep = THREADS * 8;
  const int first = threadIdx.x * 8;
  float held[kQuantHeld][8], top = 0.f;
  auto look = [&](const float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = rd_quant::max_nan(top, fabsf(v[e]));
  };
#pragma unroll
  for (int j = 0; j < kQuantHeld; ++j)
    if (first + j * kStep < K) load_row8<T, VEC>(row, first + j * kStep, K, held[j]);
#pragma unroll
  for (int j = 0; j < kQuantHeld; ++j)
    if (first + j * kStep < K) look(held[j]);
  for (int i = first + kQuantHeld * kStep; i < K; i += kStep) {
    float v[8];
    load_row8<T, VEC>(row, i, K, v);
    look(v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = rd_quant::max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) top = rd_quant::max_nan(top, red[i]);
  const bool fine = top <= 3.402823466e38f;  // not so for NaN either
  const float scale = __bfloat162float(__float2bfloat16_rn(top / 127.f));
  const bool some = fine && scale > 0.f;
  const rd_quant::Divider<sizeof(T) == 2> by(some ? scale : 1.f);
  if (threadIdx.x == 0) scales[t] = fine ? scale : __int_as_float(0x7fffffff);
  auto put = [&](int i, const float* v) {
    uint2 w = make_uint2(0u, 0u);
    if (some && v != nullptr) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w.x |= int8_code(v[e], by) << (8 * e), w.y |= int8_code(v[4 + e], by) << (8 * e);
    }
    *reinterpret_cast<uint2*>(to + i) = w;
  };
  // columns past K: codes of zeros; ld_codes is a multiple of 16
#pragma unroll
  for (int j = 0; j < kQuantHeld; ++j)
    if (first + j * kStep < ld_codes) put(first + j * kStep, first + j * kStep < K ? held[j] : nullptr);
  for (int64_t i = first + kQuantHeld * kStep; i < ld_codes; i += kStep) {
    float v[8];
    if (i < K) load_row8<T, VEC>(row, (int)i, K, v);
    put((int)i, i < K ? v : nullptr);
  }
}

struct Int8Args {
  const int8_t* A;
  int64_t lda;
  const float* a_scales;
  const int8_t* W;
  int64_t ldw;
  const float* w_scales;
  void* C;
  int64_t ldc;
  const void* R;
  int64_t ldr;
  int m_max;
  const int32_t* m_dev;
  int N, K;
};

constexpr int kBlock = 128;  // bytes of K in a block: a row of a swizzled tile
constexpr int kMmaK = 32;    // of one product
constexpr int kEpiWarps = 4;

// 8-bit signed operands, 32-bit integer accumulator, both K-major
__host__ __device__ constexpr uint32_t int8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int PAIR>
__device__ __forceinline__ void mma_int8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32i(uint32_t taddr, int* v) {
  float f[32];
  rd_umma::tmem_ld32(taddr, f);
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __float_as_int(f[i]);
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// all threads of the cluster's CTAs, each warp where it stands
__device__ __forceinline__ void cluster_sync_part() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the same place of shared memory in another CTA of the cluster
__device__ __forceinline__ uint32_t of_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(rd_umma::smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void ld_cluster(uint32_t at, int* x) {
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at) : "memory");
}
template <typename OutT>
__device__ __forceinline__ float gated(float gate, float up) {
  return (sizeof(OutT) == 2 ? rd::silu_f(gate) : rd::silu_exact(gate)) * up;
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Few tokens (up to kFewTokens): bound by the weight's bytes, and with more tokens by theirs, which every CTA reads from L2.  A CTA owns `slab` rows
// of the weight, a share of K and all tokens; the weight rows ride the products' M, the tokens their N.  The CTAs of a slab are a
// cluster: their sums, integers, meet in shared memory, and each finishes a part of the tokens.  In a chain that begins with the
// row quantiser the first ring of weights is asked for before the codes of the tokens are there (`early`: the quantiser starts its
// successors only when all before it is complete).  On one B200, quantiser included: one token x 12288 x 4096 13.7 us (3.7 TB/s of weights, some 3 us of them
// before the first block of the tokens, 2 after the last product), 110 x 4096 x 11008 with a residual 19.3 us, 32000 x 4096 27.9 us (4.7 TB/s).
constexpr int kFewTokens = 256, kMostShares = 8;
constexpr int kFewRing = 200 * 1024, kFewStagesMost = 16, kFewThreads = 192;
constexpr int kFewSmem = 1024 + kFewRing + 16 * 1024 /* a product reads 128 rows from a slab's first */ + 512;
struct FewShape {
  int slab, shares, tokens, blocks, stages, tmem_cols, early;  // slab: a multiple of 8; tokens: of m_max, a multiple of 16; blocks of K a stage
};

template <typename OutT, int EPI>
__global__ void __launch_bounds__(kFewThreads)
    int8_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const Int8Args a, const FewShape sh, int32_t* status) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kFewRing + 16 * 1024);
  uint64_t* empty = full + kFewStagesMost;
  uint64_t* acc_full = empty + kFewStagesMost;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = blockIdx.x % sh.shares, row0 = blockIdx.x / sh.shares * sh.slab;
  const int w_bytes = sh.slab * kBlock, a_bytes = sh.tokens * kBlock, stage_bytes = sh.blocks * (w_bytes + a_bytes);
  const int all_blocks = (a.K + kBlock - 1) / kBlock, block0 = share * all_blocks / sh.shares, k_blocks = (share + 1) * all_blocks / sh.shares - block0;
  const int steps = (k_blocks + sh.blocks - 1) / sh.blocks;
  rd::pdl_launch_dependents();
  if (warp == 0 && rd::elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
    for (int s = 0; s < kFewStagesMost; ++s) {
      rd_umma::mbar_init(&full[s], 2);
      rd_umma::mbar_init(&empty[s], 1);
    }
    rd_umma::mbar_init(acc_full, 1);
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) rd_umma::tmem_alloc(tmem_slot, sh.tmem_cols);
  rd_umma::fence_before();
  __syncthreads();
  rd_umma::fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  int site = 0;
  if (warp == 0) {
    if (rd::elect_one()) {
      // blocks of a step: weights, then tokens; blocks past K are not loaded and not multiplied
      auto load = [&](int step, bool weights) {
        const int s = step % sh.stages, n = min(sh.blocks, k_blocks - step * sh.blocks);
        uint8_t* to = smem + s * stage_bytes + (weights ? 0 : sh.blocks * w_bytes);
        rd_umma::mbar_expect_tx(&full[s], n * (weights ? w_bytes : a_bytes));
        for (int i = 0; i < n; ++i)
          rd_umma::tma_load_2d(to + i * (weights ? w_bytes : a_bytes), weights ? &map_w : &map_a, &full[s], (block0 + step * sh.blocks + i) * kBlock, weights ? row0 : 0);
      };
      const int ahead = min(steps, sh.stages);
      if (!sh.early) rd::pdl_wait();
      for (int i = 0; i < ahead; ++i) load(i, true);
      if (sh.early) rd::pdl_wait();
      for (int i = 0; i < ahead; ++i) load(i, false);
      for (int i = ahead; i < steps; ++i) {
        if (!rd_umma::wait_or(&empty[i % sh.stages], (i / sh.stages - 1) & 1, stop)) {
          ok = false, site = 1;
          break;
        }
        load(i, true);
        load(i, false);
      }
    }
  } else if (warp == 1) {
    if (rd::elect_one()) {
      rd::pdl_wait();
      const int M = rd::live_rows(a.m_dev, a.m_max);
      const uint32_t idesc = int8_idesc(128, max(16, (M + 15) / 16 * 16));
      for (int i = 0; i < steps; ++i) {
        const int s = i % sh.stages, n = min(sh.blocks, k_blocks - i * sh.blocks);
        if (!rd_umma::wait_or(&full[s], (i / sh.stages) & 1, stop)) {
          ok = false, site = 2;
          break;
        }
        rd_umma::fence_after();
        const uint32_t w = rd_umma::smem_u32(smem + s * stage_bytes), t = w + sh.blocks * w_bytes;
        for (int b = 0; b < n; ++b) {
          const uint64_t dw = rd_umma::desc_k_major(w + b * w_bytes), dt = rd_umma::desc_k_major(t + b * a_bytes);
#pragma unroll
          for (int k = 0; k < kBlock / kMmaK; ++k) mma_int8<0>(tmem, dw + 2 * k, dt + 2 * k, idesc, i | b | k);
        }
        rd_umma::commit(&empty[s]);
      }
      if (ok) rd_umma::commit(acc_full);
    }
  } else {
    rd::pdl_wait();
    const int M = rd::live_rows(a.m_dev, a.m_max), quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int each = (M + sh.shares - 1) / sh.shares, t_end = min(M, (share + 1) * each);
    const int f = row0 + lane * 4;
    const bool mine = lane * 4 < sh.slab && f < a.N;  // rows of the product past the slab are the next slab's
    constexpr bool kGated = EPI == RD_EPI_SWIGLU;
    constexpr int kOut = kGated ? 2 : 4;
    const int col = kGated ? f / 2 : f, wide = kGated ? a.N / 2 : a.N;
    const bool vec = col + kOut <= wide && ((uintptr_t)a.C % (kOut * sizeof(OutT))) == 0 && a.ldc % kOut == 0 &&
                     (EPI != RD_EPI_RES || (((uintptr_t)a.R % (kOut * sizeof(OutT))) == 0 && a.ldr % kOut == 0));
    if (EPI == RD_EPI_RES && mine)  // on their way from memory to L2 meanwhile
      for (int t = share * each + quarter; t < t_end; t += 4)
        asm volatile("prefetch.global.L2 [%0];" ::"l"((const OutT*)a.R + (int64_t)t * a.ldr + min(col, wide - 1)) : "memory");
    ok = rd_umma::warp_wait(acc_full, 0, stop);
    if (!ok) site = 3;
    rd_umma::fence_after();
    // Sums go to shared memory, [token][128 features], where the ring was; then a warp takes a token at a time, a lane four features.  Short
    // loops: code that an SM has not run since the last kernel costs a trip to L2 for every stretch of it (an epilogue unrolled over
    // 32 tokens took 4 us for one).
    int* sums = reinterpret_cast<int*>(smem);
    for (int c = 0; ok && row - lane < sh.slab && c < M; c += 32) {
      int v[32];
      tmem_ld32i(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
#pragma unroll
      for (int i = 0; i < 32; ++i) sums[(c + i) * 128 + row] = v[i];
    }
    if (sh.shares > 1) cluster_sync_part();
    else asm volatile("bar.sync 1, 128;" ::: "memory");
    const int t1 = ok ? t_end : 0;
    float sw[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) sw[e] = mine && f + e < a.N ? a.w_scales[f + e] : 0.f;
    using Vec = std::conditional_t<kOut * sizeof(OutT) == 16, uint4, std::conditional_t<kOut * sizeof(OutT) == 8, uint2, uint32_t>>;
#pragma unroll 2
    for (int t = share * each + quarter; t < t1; t += 4) {
      const float sa = a.a_scales[t];
      OutT r[kOut];
      if (EPI == RD_EPI_RES && mine) {
        const OutT* from = (const OutT*)a.R + (int64_t)t * a.ldr + col;
        if (vec) {
          *reinterpret_cast<Vec*>(r) = *reinterpret_cast<const Vec*>(from);
        } else {
#pragma unroll
          for (int e = 0; e < kOut; ++e) r[e] = col + e < wide ? from[e] : rd::Num<OutT>::from_f(0.f);
        }
      }
      int v[4] = {};
      for (int s = 0; s < sh.shares; ++s) {
        int x[4];
        ld_cluster(of_rank(sums + t * 128 + lane * 4, sh.shares > 1 ? s : (int)cluster_rank()), x);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += x[e];
      }
      if (!mine) continue;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (float)v[e] * (sa * sw[e]);
      OutT out[kOut];
      if constexpr (kGated) {
        out[0] = rd::Num<OutT>::from_f(gated<OutT>(y[0], y[1]));
        out[1] = rd::Num<OutT>::from_f(gated<OutT>(y[2], y[3]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = rd::Num<OutT>::from_f(EPI == RD_EPI_RES ? y[e] + rd::Num<OutT>::to_f(r[e]) : y[e]);
      }
      OutT* to = (OutT*)a.C + (int64_t)t * a.ldc + col;
      if (vec) {
        *reinterpret_cast<Vec*>(to) = *reinterpret_cast<const Vec*>(out);
      } else {
#pragma unroll
        for (int e = 0; e < kOut; ++e)
          if (col + e < wide) to[e] = out[e];
      }
    }
  }
  __syncwarp();
  if (sh.shares > 1) {
    if (warp < 2) cluster_sync_part();  // the epilogue warps have met the others' above
    cluster_sync_part();                // no CTA leaves while its sums are read
  }
  if (!ok && atomicCAS((int*)stop, 0, 1) == 0 && status) atomicExch(status, 510 + site);
  __syncwarp();
  rd_umma::fence_before();
  __syncthreads();
  if (*stop)
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land
  if (warp == 1) {
    rd_umma::fence_after();
    rd_umma::tmem_dealloc(tmem, sh.tmem_cols);
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Many tokens: bound by the tensor cores and by the operands' way from L2.  Persistent, CTAs in clusters of two that share products of 256
// tokens (the products' M, 128 to a CTA) x `width` features (their N; each CTA stages half of them):
//   warp 0     loads of both operands, six stages of a block of K each; both CTAs' loads complete on the leader's barrier;
//   warp 1     of the leader: issues the products into one of two accumulators;
//   warps 2-5  epilogue, a token to a lane: scales, gate; 32 output features at a time through shared memory, from where rows go out
//              (and residual rows come in) in 16-byte pieces of consecutive addresses.
// 4095 tokens x 22016 x 4096 with a gate on one B200: 199 us, 3.7 POP/s, the tensor cores busy for 95 % of the cycles.
constexpr int kManyStages = 6, kManyThreads = 192, kTileTokens = 256, kMostWidth = 256;
struct ManySmem {
  static constexpr int kTokens = 128 * kBlock, kFeatures = kMostWidth / 2 * kBlock;
  static constexpr int kScratch = kEpiWarps * 32 * 32 * 4, kScales = 2 * kMostWidth * 4;
  static constexpr int kBytes = 1024 + kManyStages * (kTokens + kFeatures) + kScratch + kScales + 256;
};
struct ManyMaps {
  CUtensorMap a, w;
};
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(rd_umma::smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void commit_both(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(rd_umma::smem_u32(bar)), "h"((uint16_t)3)
               : "memory");
}

template <typename OutT, int EPI>
__global__ void __launch_bounds__(kManyThreads, 1)
    int8_many_kernel(const __grid_constant__ ManyMaps maps, const Int8Args a, int width, int32_t* status) {
  using L = ManySmem;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sW = sA + kManyStages * L::kTokens;
  float* scratch = reinterpret_cast<float*>(sW + kManyStages * L::kFeatures);
  float* s_scale = scratch + kEpiWarps * 32 * 32;  // [2][256]: the weight scales of a tile
  uint64_t* full = reinterpret_cast<uint64_t*>(s_scale + 2 * kMostWidth);
  uint64_t* empty = full + kManyStages;
  uint64_t* acc_full = empty + kManyStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* stop = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  rd::pdl_launch_dependents();
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.w) : "memory");
    for (int s = 0; s < kManyStages; ++s) {
      rd_umma::mbar_init(&full[s], 1);
      rd_umma::mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      rd_umma::mbar_init(&acc_full[i], 1);
      rd_umma::mbar_init(&acc_empty[i], 2 * kEpiWarps);
    }
    *stop = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(rd_umma::smem_u32(tmem_slot)), "r"(2 * kMostWidth) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  rd_umma::fence_before();
  __syncthreads();
  cluster_sync_part();
  rd_umma::fence_after();
  const uint32_t tmem = *tmem_slot;
  rd::pdl_wait();
  const int M = rd::live_rows(a.m_dev, a.m_max);
  const int t_tiles = (M + kTileTokens - 1) / kTileTokens, f_tiles = (a.N + width - 1) / width, tiles = t_tiles * f_tiles;
  const int k_blocks = (a.K + kBlock - 1) / kBlock;
  bool ok = true;
  int site = 0;
  // tiles that run at the same time share features: those are read from memory once, the tokens lie in L2
  if (warp == 0) {
    if (rd::elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int tile = pair; ok && tile < tiles; tile += n_pairs) {
        const int t0 = tile % t_tiles * kTileTokens + (int)rank * 128, f0 = tile / t_tiles * width + (int)rank * (width / 2);
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!rd_umma::wait_or(&empty[stage], phase ^ 1, stop)) {
            ok = false, site = 1;
            break;
          }
          const uint32_t bar = of_rank(&full[stage], 0);
          if (rank == 0) rd_umma::mbar_expect_tx(&full[stage], 2 * (L::kTokens + width / 2 * kBlock));
          load_pair(sA + stage * L::kTokens, &maps.a, bar, kb * kBlock, t0);
          load_pair(sW + stage * L::kFeatures, &maps.w, bar, kb * kBlock, f0);
          if (++stage == kManyStages) stage = 0, phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && rd::elect_one()) {
      const uint32_t idesc = int8_idesc(256, width);
      int stage = 0, local = 0;
      uint32_t phase = 0;
      for (int tile = pair; ok && tile < tiles; tile += n_pairs, ++local) {
        const int acc = local & 1;
        if (!rd_umma::wait_or(&acc_empty[acc], ((local >> 1) & 1) ^ 1, stop)) {
          ok = false, site = 2;
          break;
        }
        rd_umma::fence_after();
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!rd_umma::wait_or(&full[stage], phase, stop)) {
            ok = false, site = 3;
            break;
          }
          rd_umma::fence_after();
          const uint64_t da = rd_umma::desc_k_major(rd_umma::smem_u32(sA + stage * L::kTokens)), dw = rd_umma::desc_k_major(rd_umma::smem_u32(sW + stage * L::kFeatures));
#pragma unroll
          for (int k = 0; k < kBlock / kMmaK; ++k) mma_int8<1>(tmem + acc * kMostWidth, da + 2 * k, dw + 2 * k, idesc, kb | k);
          commit_both(&empty[stage]);
          if (++stage == kManyStages) stage = 0, phase ^= 1;
        }
        if (ok) commit_both(&acc_full[acc]);
      }
    }
  } else {
    const int quarter = warp & 3;
    float* scr = scratch + (warp - 2) * 32 * 32;
    constexpr bool kGated = EPI == RD_EPI_SWIGLU;
    constexpr int kEach = 16 / (int)sizeof(OutT), kLanes = 32 / kEach, kRowsAtOnce = 32 / kLanes;  // values of a 16-byte piece; lanes of a row of 32 outputs
    const bool vec = ((uintptr_t)a.C % 16 == 0) && (a.ldc * sizeof(OutT)) % 16 == 0 && (EPI != RD_EPI_RES || ((uintptr_t)a.R % 16 == 0 && (a.ldr * sizeof(OutT)) % 16 == 0));
    const int wide = kGated ? a.N / 2 : a.N;
    int local = 0;
    for (int tile = pair; tile < tiles; tile += n_pairs, ++local) {
      const int t0 = tile % t_tiles * kTileTokens + (int)rank * 128 + quarter * 32, f0 = tile / t_tiles * width;
      float* sw = s_scale + (local & 1) * kMostWidth;
      for (int i = threadIdx.x - 64; i < width; i += kEpiWarps * 32) sw[i] = f0 + i < a.N ? a.w_scales[f0 + i] : 0.f;
      const float sa = t0 + lane < M ? a.a_scales[t0 + lane] : 0.f;
      const int acc = local & 1;
      // the scales are there for all four warps, and they leave together
      if (!rd::epilogue_agrees(rd_umma::warp_wait(&acc_full[acc], (local >> 1) & 1, stop))) {
        ok = false, site = 4;
        break;
      }
      rd_umma::fence_after();
      const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + acc * kMostWidth;
      for (int c = 0; c < width; c += kGated ? 64 : 32) {
        const int o0 = kGated ? (f0 + c) >> 1 : f0 + c;  // first of 32 outputs
        if (o0 >= wide) break;
        __syncwarp();
#pragma unroll
        for (int half = 0; half < (kGated ? 2 : 1); ++half) {
          int v[32];
          tmem_ld32i(taddr + c + 32 * half, v);
          float y[32];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 s = *reinterpret_cast<const float4*>(sw + c + 32 * half + i);
            y[i] = (float)v[i] * (sa * s.x), y[i + 1] = (float)v[i + 1] * (sa * s.y), y[i + 2] = (float)v[i + 2] * (sa * s.z), y[i + 3] = (float)v[i + 3] * (sa * s.w);
          }
          if (kGated) {
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = gated<OutT>(y[2 * i], y[2 * i + 1]);
          }
#pragma unroll
          for (int i = 0; i < (kGated ? 4 : 8); ++i) {
            const int piece = (half * 4 + i) ^ (lane & 7);
            *reinterpret_cast<float4*>(scr + lane * 32 + piece * 4) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          }
        }
        __syncwarp();
        if (vec && o0 + 32 <= wide) {
          const int part = lane % kLanes * kEach;
#pragma unroll
          for (int i = 0; i < 32; i += kRowsAtOnce) {
            const int row = i + lane / kLanes;
            float x[kEach];
#pragma unroll
            for (int e = 0; e < kEach; e += 4) *reinterpret_cast<float4*>(x + e) = *reinterpret_cast<const float4*>(scr + row * 32 + ((((part + e) >> 2) ^ (row & 7)) << 2));
            if (t0 + row >= M) continue;
            if (EPI == RD_EPI_RES) {
              OutT r[kEach];
              *reinterpret_cast<uint4*>(r) = *reinterpret_cast<const uint4*>((const OutT*)a.R + (int64_t)(t0 + row) * a.ldr + o0 + part);
#pragma unroll
              for (int e = 0; e < kEach; ++e) x[e] += rd::Num<OutT>::to_f(r[e]);
            }
            OutT out[kEach];
#pragma unroll
            for (int e = 0; e < kEach; ++e) out[e] = rd::Num<OutT>::from_f(x[e]);
            *reinterpret_cast<uint4*>((OutT*)a.C + (int64_t)(t0 + row) * a.ldc + o0 + part) = *reinterpret_cast<const uint4*>(out);
          }
        } else {
          for (int row = 0; row < 32 && t0 + row < M; ++row) {
            if (o0 + lane >= wide) continue;
            float x = scr[row * 32 + (((lane >> 2) ^ (row & 7)) << 2) + (lane & 3)];
            if (EPI == RD_EPI_RES) x += rd::Num<OutT>::to_f(((const OutT*)a.R)[(int64_t)(t0 + row) * a.ldr + o0 + lane]);
            ((OutT*)a.C)[(int64_t)(t0 + row) * a.ldc + o0 + lane] = rd::Num<OutT>::from_f(x);
          }
        }
      }
      rd_umma::fence_before();
      __syncwarp();
      if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(of_rank(&acc_empty[acc], 0)) : "memory");
    }
  }
  if (!ok && atomicCAS((int*)stop, 0, 1) == 0 && status) atomicExch(status, 520 + site);
  __syncwarp();
  rd_umma::fence_before();
  __syncthreads();
  if (*stop)
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);  // copies in flight land
  cluster_sync_part();  // the peer signals and reads no more
  if (warp == 1) {
    rd_umma::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kMostWidth) : "memory");
  }
}

// How many CTAs of a kernel, one on an SM, run at the same time in clusters of `shares`; asked once for each size of cluster.
template <auto Kernel>
int64_t resident_ctas(int shares, int threads, int smem) {
  static std::atomic<int> known[kMostShares + 1] = {};
  std::atomic<int>& here = known[shares];
  int n = here.load(std::memory_order_relaxed);
  if (n == 0) {
    if (shares == 1) {
      n = rd_quant::sm_count();
    } else {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(shares);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = shares;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, Kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();
        clusters = 0;
      }
      n = clusters > 0 ? clusters * shares : 1;
    }
    here.store(n, std::memory_order_relaxed);
  }
  return n;
}

// What a call costs with either kernel: rows of 128 bytes that an SM brings in, and for few tokens those that the sums come to in shared memory.
struct ManyShape {
  int width;
  int64_t cost, tiles;
};
ManyShape many_shape(const Int8Args& a) {
  // features of a tile: the width with which the rounds of tiles take least, a tile of w features counting w + 64
  const int64_t pairs = rd_quant::sm_count() / 2, t_tiles = (a.m_max + kTileTokens - 1) / kTileTokens;
  ManyShape sh{kMostWidth, 0, 0};
  int64_t best = INT64_MAX;
  for (int w = kMostWidth; w >= 64; w -= 64) {
    const int64_t tiles = t_tiles * ((a.N + w - 1) / w), rounds = (tiles + pairs - 1) / pairs;
    if (rounds * (w + 64) < best) best = rounds * (w + 64), sh = ManyShape{w, rounds * (128 + w / 2) * ((a.K + kBlock - 1) / kBlock), tiles};
  }
  return sh;
}
// cost INT64_MAX: not for this call
template <auto kernel>
int64_t few_shape(const Int8Args& a, FewShape& sh) {
  sh.tokens = (a.m_max + 15) / 16 * 16;
  if (sh.tokens > kFewTokens) return INT64_MAX;
  // Weight rows of a CTA and shares of K: those with which an SM has the fewest bytes to bring in, all CTAs at the same time.  Fewer shares where
  // that is the same.
  const int sms = rd_quant::sm_count(), k_blocks = (a.K + kBlock - 1) / kBlock;
  static_assert(kFewTokens * 512 <= kFewRing, "the sums");
  int64_t best = INT64_MAX;
  for (int shares = 1; shares <= kMostShares && shares <= k_blocks; ++shares) {
    const int64_t most = resident_ctas<kernel>(shares, kFewThreads, kFewSmem);
    for (int slab = 128; slab >= 16; slab -= 8) {
      const int64_t ctas = (int64_t)((a.N + slab - 1) / slab) * shares;
      if (ctas > most) break;
      const int64_t cost = (slab + sh.tokens) * ((k_blocks + shares - 1) / shares) + 8 * sh.tokens;
      if (cost < best) best = cost, sh.slab = slab, sh.shares = shares;
    }
  }
  if (best == INT64_MAX) {  // more slabs than run at the same time
    if (sh.tokens > 128) return best;
    sh.slab = 128, sh.shares = 1;
    best = ((a.N + 127) / 128 + sms - 1) / sms * ((128 + sh.tokens) * (int64_t)k_blocks + 8 * sh.tokens);
  }
  // four blocks of K a stage, 512 consecutive bytes of each row, where at least four such stages fit
  const int block = (sh.slab + sh.tokens) * kBlock;
  sh.blocks = 16 * block <= kFewRing ? 4 : 8 * block <= kFewRing ? 2 : 1;
  sh.stages = kFewRing / (sh.blocks * block);
  if (sh.stages > kFewStagesMost) sh.stages = kFewStagesMost;
  sh.tmem_cols = 32;
  while (sh.tmem_cols < sh.tokens) sh.tmem_cols *= 2;
  sh.early = 0;
  return best;
}

template <typename OutT, int EPI>
int launch_few(const Int8Args& a, const FewShape& sh, int32_t* status, cudaStream_t s) {
  constexpr auto kernel = int8_few_kernel<OutT, EPI>;
  const int slabs = (a.N + sh.slab - 1) / sh.slab;
  CUtensorMap ma, mw;
  RD_REQUIRE(rd_umma::make_byte_map(&ma, a.A, a.m_max, a.K, a.lda, sh.tokens) && rd_umma::make_byte_map(&mw, a.W, a.N, a.K, a.ldw, sh.slab), RD_ERR_ARG);
  cudaError_t err = rd::launch_chained(kernel, dim3((unsigned)(slabs * sh.shares)), dim3(kFewThreads), kFewSmem, s, sh.shares, ma, mw, a, sh, status);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

template <typename OutT, int EPI>
int launch_many(const Int8Args& a, const ManyShape& sh, int32_t* status, cudaStream_t s) {
  constexpr auto kernel = int8_many_kernel<OutT, EPI>;
  RD_REQUIRE(rd_quant::allow_smem<kernel>(ManySmem::kBytes), RD_ERR_LAUNCH);
  ManyMaps maps;
  RD_REQUIRE(rd_umma::make_byte_map(&maps.a, a.A, a.m_max, a.K, a.lda, 128) && rd_umma::make_byte_map(&maps.w, a.W, a.N, a.K, a.ldw, sh.width / 2), RD_ERR_ARG);
  RD_REQUIRE(sh.tiles <= 0x7fffffff, RD_ERR_SIZE);
  const int64_t pairs = rd_quant::sm_count() / 2;
  const unsigned grid = 2 * (unsigned)(sh.tiles < pairs ? sh.tiles : pairs);
  cudaError_t err = rd::launch_chained(kernel, dim3(grid), dim3(kManyThreads), ManySmem::kBytes, s, 2, maps, a, sh.width, status);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

int check_rows(int dtype, const void* x, int64_t ldx, const int8_t* codes, int64_t ld_codes, const float* scales, int m_max, int K) {
  RD_REQUIRE(dtype == RD_F32 || dtype == RD_BF16, RD_ERR_DTYPE);
  RD_REQUIRE(m_max >= 0 && K >= 1 && ldx >= 0 && ld_codes >= K, RD_ERR_ARG);
  if (m_max == 0) return RD_OK;
  RD_REQUIRE(x && codes && scales, RD_ERR_ARG);
  RD_REQUIRE(((uintptr_t)x & (dtype == RD_BF16 ? 1 : 3)) == 0, RD_ERR_ALIGN);
  RD_REQUIRE(((uintptr_t)codes & 15) == 0 && ld_codes % 16 == 0 && ((uintptr_t)scales & 3) == 0, RD_ERR_ALIGN);
  return RD_OK;
}

int check_product(int out_dtype, const Int8Args& a, int epilogue) {
  RD_REQUIRE(out_dtype == RD_F32 || out_dtype == RD_BF16, RD_ERR_DTYPE);
  RD_REQUIRE(epilogue == RD_EPI_NONE || epilogue == RD_EPI_RES || epilogue == RD_EPI_SWIGLU, RD_ERR_UNSUPPORTED);
  RD_REQUIRE(a.m_max >= 0 && a.N >= 1 && a.K >= 1, RD_ERR_ARG);
  // a sum of K products of at most 127^2 has to fit 31 bits
  RD_REQUIRE(a.K <= 131072 && a.K % 16 == 0, RD_ERR_SIZE);
  RD_REQUIRE(epilogue != RD_EPI_SWIGLU || a.N % 2 == 0, RD_ERR_SIZE);
  if (a.m_max == 0) return RD_OK;
  RD_REQUIRE(a.A && a.a_scales && a.W && a.w_scales && a.C && (epilogue != RD_EPI_RES || a.R), RD_ERR_ARG);
  RD_REQUIRE(a.lda >= a.K && a.ldw >= a.K && a.ldc >= (epilogue == RD_EPI_SWIGLU ? a.N / 2 : a.N) && (epilogue != RD_EPI_RES || a.ldr >= a.N), RD_ERR_ARG);
  RD_REQUIRE((((uintptr_t)a.A | (uintptr_t)a.W) & 15) == 0 && a.lda % 16 == 0 && a.ldw % 16 == 0, RD_ERR_ALIGN);
  RD_REQUIRE(((uintptr_t)a.C & (out_dtype == RD_BF16 ? 1 : 3)) == 0 && ((uintptr_t)a.R & (out_dtype == RD_BF16 ? 1 : 3)) == 0, RD_ERR_ALIGN);
  return RD_OK;
}

int quant_rows(int dtype, const void* x, int64_t ldx, int8_t* codes, int64_t ld_codes, float* scales, int m_max, const int32_t* m_dev, int K, cudaStream_t s) {
  cudaError_t err;
  const bool vec = K % 8 == 0 && ((uintptr_t)x & 15) == 0 && (ldx * (dtype == RD_BF16 ? 2 : 4)) % 16 == 0;
  const bool wide = m_max <= rd_quant::sm_count() && K > 2048;  // a block an SM: the row's latency is the kernel's
  auto run = [&](auto kern, int threads, auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    err = rd::launch_chained(kern, dim3(m_max), dim3(threads), 0, s, 1, (const T*)x, ldx, codes, ld_codes, scales, m_max, m_dev, K);
  };
  auto pick = [&](auto* zero) {
    using T = std::remove_pointer_t<decltype(zero)>;
    if (wide) vec ? run(quant_rows_kernel<T, true, 1024>, 1024, zero) : run(quant_rows_kernel<T, false, 1024>, 1024, zero);
    else vec ? run(quant_rows_kernel<T, true, 256>, 256, zero) : run(quant_rows_kernel<T, false, 256>, 256, zero);
  };
  if (dtype == RD_BF16) pick((__nv_bfloat16*)nullptr);
  else pick((float*)nullptr);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

template <typename OutT, int EPI>
int product_of(const Int8Args& a, bool early, int32_t* status, cudaStream_t s) {
  // The kernel for few tokens up to 32 of them, and where it is expected to be sooner done.  Times fit 4.6 us + 1.45 ns x cost for many tokens, 5.5 us + 2.05 ns
  // x cost for few within a tenth (one B200, row quantiser included, us, few against many: 12288 x 4096 features, 40 tokens 16 : 18, 110 tokens 21 : 18, 256
  // tokens 33 : 19; 22016 x 4096, 16 tokens 27 : 32, 110 tokens 41 : 27; 4096 x 11008, 110 tokens 18 : 24, 256 tokens 24 : 25; 2048 x 2048, 64 tokens 7.8 : 7.3).
  FewShape few;
  const ManyShape many = many_shape(a);
  constexpr auto few_kernel = int8_few_kernel<OutT, EPI>;
  RD_REQUIRE(rd_quant::allow_smem<few_kernel>(kFewSmem), RD_ERR_LAUNCH);
  const int64_t cost = few_shape<few_kernel>(a, few);
  if (cost == INT64_MAX || (a.m_max > 32 && 10 * (cost + 450) > 7 * many.cost)) return launch_many<OutT, EPI>(a, many, status, s);
  few.early = early;
  return launch_few<OutT, EPI>(a, few, status, s);
}
template <typename OutT>
int product_as(const Int8Args& a, int epilogue, bool early, int32_t* status, cudaStream_t s) {
  if (epilogue == RD_EPI_NONE) return product_of<OutT, RD_EPI_NONE>(a, early, status, s);
  if (epilogue == RD_EPI_RES) return product_of<OutT, RD_EPI_RES>(a, early, status, s);
  return product_of<OutT, RD_EPI_SWIGLU>(a, early, status, s);
}
int product(int out_dtype, const Int8Args& a, int epilogue, bool early, int32_t* status, cudaStream_t s) {
  return out_dtype == RD_F32 ? product_as<float>(a, epilogue, early, status, s) : product_as<__nv_bfloat16>(a, epilogue, early, status, s);
}

}  // namespace

extern "C" int rd_quant_rows(int dtype, const void* x, int64_t ldx, int8_t* codes, int64_t ld_codes, float* scales, int m_max, const int32_t* m_dev,
                             int K, void* stream) {
  const int rc = check_rows(dtype, x, ldx, codes, ld_codes, scales, m_max, K);
  if (rc != RD_OK || m_max == 0) return rc;
  return quant_rows(dtype, x, ldx, codes, ld_codes, scales, m_max, m_dev, K, (cudaStream_t)stream);
}

extern "C" int rd_gemm_int8(int out_dtype, const int8_t* A, int64_t lda, const float* a_scales, const int8_t* W, int64_t ldw, const float* w_scales,
                            void* C, int64_t ldc, const void* R, int64_t ldr, int m_max, const int32_t* m_dev, int N, int K, int epilogue,
                            int32_t* status, void* stream) {
  const Int8Args a{A, lda, a_scales, W, ldw, w_scales, C, ldc, R, ldr, m_max, m_dev, N, K};
  const int rc = check_product(out_dtype, a, epilogue);
  if (rc != RD_OK || m_max == 0) return rc;
  return product(out_dtype, a, epilogue, false, status, (cudaStream_t)stream);
}

extern "C" int rd_linear_int8(const rd_linear_int8_desc* d, void* stream) {
  RD_REQUIRE(d, RD_ERR_ARG);
  int rc = check_rows(d->dtype, d->x, d->ldx, d->codes, d->ld_codes, d->scales, d->m_max, d->K);
  if (rc != RD_OK) return rc;
  const Int8Args a{d->codes, d->ld_codes, d->scales, d->W, d->ldw, d->w_scales, d->C, d->ldc, d->R, d->ldr, d->m_max, d->m_dev, d->N, (d->K + 15) / 16 * 16};
  rc = check_product(d->out_dtype, a, d->epilogue);
  if (rc != RD_OK || d->m_max == 0) return rc;
  rc = quant_rows(d->dtype, d->x, d->ldx, d->codes, d->ld_codes, d->scales, d->m_max, d->m_dev, d->K, (cudaStream_t)stream);
  return rc != RD_OK ? rc : product(d->out_dtype, a, d->epilogue, true, d->status, (cudaStream_t)stream);
}

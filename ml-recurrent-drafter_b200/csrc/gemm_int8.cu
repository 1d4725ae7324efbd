// Products of matrices held in 8-bit integers with a scale for each row: C[t, n] = sA[t] sW[n] sum_k A[t, k] W[n, k], and the quantiser of
// their rows.  A row x of K values: scale = bf16(max |x| / 127) in fp32, code = rint(x / scale) cut to -127 .. 127; the scale's 8 significant
// bits make fp32's division give the codes of exact arithmetic (cache_quant.cu has the argument).  The sums are integers and exact.
#include "rd_common.cuh"

namespace {

constexpr int kQuantThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quant_rows_kernel(const T* x, int64_t ldx, int8_t* codes, int64_t ld_codes, float* scales, int m_max,
                                                                   const int32_t* m_dev, int K) {
  __shared__ float red[kQuantThreads / 32];
  rd::pdl_wait();
  rd::pdl_launch_dependents();
  const int t = blockIdx.x;
  if (t >= rd::live_rows(m_dev, m_max)) return;
  const T* row = x + (int64_t)t * ldx;
  int8_t* to = codes + (int64_t)t * ld_codes;
  float top = 0.f;
  bool odd = false;
  for (int i = threadIdx.x; i < K; i += kQuantThreads) {
    const float v = fabsf(rd::Num<T>::to_f(row[i]));
    odd |= !(v <= 3.402823466e38f);
    top = fmaxf(top, v);
  }
  if (odd) top = INFINITY;
  top = rd::warp_max(top);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = red[0];
#pragma unroll
  for (int i = 1; i < kQuantThreads / 32; ++i) top = fmaxf(top, red[i]);
  const bool fine = top <= 3.402823466e38f;
  const float scale = __bfloat162float(__float2bfloat16_rn(top / 127.f));
  const bool some = fine && scale > 0.f;
  if (threadIdx.x == 0) scales[t] = fine ? scale : __int_as_float(0x7fffffff);
  for (int i = threadIdx.x; i < ld_codes; i += kQuantThreads)
    to[i] = some && i < K ? (int8_t)fminf(fmaxf(rintf(rd::Num<T>::to_f(row[i]) / scale), -127.f), 127.f) : (int8_t)0;
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

constexpr int BM = 64, BN = 64, BK = 16;  // BK: words of 4

template <typename OutT, int EPI>
__global__ void __launch_bounds__(256) gemm_int8_kernel(const Int8Args a) {
  __shared__ int As[BK][BM + 4], Ws[BK][BN + 4];
  rd::pdl_launch_dependents();
  rd::pdl_wait();
  const int M = rd::live_rows(a.m_dev, a.m_max);
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  if (m0 >= M) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int lr = threadIdx.x >> 2, lk = (threadIdx.x & 3) * 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 4 * BK) {
    const int k = k0 + 4 * lk;
    int4 u = make_int4(0, 0, 0, 0), w = u;
    if (k < a.K && m0 + lr < M) u = *reinterpret_cast<const int4*>(a.A + (int64_t)(m0 + lr) * a.lda + k);
    if (k < a.K && n0 + lr < a.N) w = *reinterpret_cast<const int4*>(a.W + (int64_t)(n0 + lr) * a.ldw + k);
    As[lk][lr] = u.x, As[lk + 1][lr] = u.y, As[lk + 2][lr] = u.z, As[lk + 3][lr] = u.w;
    Ws[lk][lr] = w.x, Ws[lk + 1][lr] = w.y, Ws[lk + 2][lr] = w.z, Ws[lk + 3][lr] = w.w;
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < BK; ++kk)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(As[kk][ty * 4 + i], Ws[kk][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty * 4 + i;
    if (m >= M) continue;
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      v[j] = n < a.N ? (float)acc[i][j] * (a.a_scales[m] * a.w_scales[n]) : 0.f;
    }
    OutT* C = (OutT*)a.C + (int64_t)m * a.ldc;
    if (EPI == RD_EPI_SWIGLU) {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        const int n = n0 + tx * 4 + j;
        if (n + 1 < a.N) C[n / 2] = rd::Num<OutT>::from_f(rd::silu_exact(v[j]) * v[j + 1]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx * 4 + j;
        if (n >= a.N) continue;
        if (EPI == RD_EPI_RES) v[j] += rd::Num<OutT>::to_f(((const OutT*)a.R)[(int64_t)m * a.ldr + n]);
        C[n] = rd::Num<OutT>::from_f(v[j]);
      }
    }
  }
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
  if (dtype == RD_BF16)
    err = rd::launch_chained(quant_rows_kernel<__nv_bfloat16>, dim3(m_max), dim3(kQuantThreads), 0, s, 1, (const __nv_bfloat16*)x, ldx, codes, ld_codes, scales,
                             m_max, m_dev, K);
  else
    err = rd::launch_chained(quant_rows_kernel<float>, dim3(m_max), dim3(kQuantThreads), 0, s, 1, (const float*)x, ldx, codes, ld_codes, scales, m_max, m_dev, K);
  RD_CHECK_CHAINED(err);
  return RD_OK;
}

int product(int out_dtype, const Int8Args& a, int epilogue, cudaStream_t s) {
  const dim3 grid((a.N + BN - 1) / BN, (a.m_max + BM - 1) / BM);
  cudaError_t err;
  auto run = [&](auto kern) { err = rd::launch_chained(kern, grid, dim3(256), 0, s, 1, a); };
  const bool f32 = out_dtype == RD_F32;
  if (epilogue == RD_EPI_NONE) f32 ? run(gemm_int8_kernel<float, RD_EPI_NONE>) : run(gemm_int8_kernel<__nv_bfloat16, RD_EPI_NONE>);
  else if (epilogue == RD_EPI_RES) f32 ? run(gemm_int8_kernel<float, RD_EPI_RES>) : run(gemm_int8_kernel<__nv_bfloat16, RD_EPI_RES>);
  else f32 ? run(gemm_int8_kernel<float, RD_EPI_SWIGLU>) : run(gemm_int8_kernel<__nv_bfloat16, RD_EPI_SWIGLU>);
  RD_CHECK_CHAINED(err);
  return RD_OK;
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
  (void)status;
  const Int8Args a{A, lda, a_scales, W, ldw, w_scales, C, ldc, R, ldr, m_max, m_dev, N, K};
  const int rc = check_product(out_dtype, a, epilogue);
  if (rc != RD_OK || m_max == 0) return rc;
  return product(out_dtype, a, epilogue, (cudaStream_t)stream);
}

extern "C" int rd_linear_int8(int dtype, const void* x, int64_t ldx, int8_t* codes, int64_t ld_codes, float* scales, const int8_t* W, int64_t ldw,
                              const float* w_scales, int out_dtype, void* C, int64_t ldc, const void* R, int64_t ldr, int m_max, const int32_t* m_dev,
                              int N, int K, int epilogue, int32_t* status, void* stream) {
  (void)status;
  int rc = check_rows(dtype, x, ldx, codes, ld_codes, scales, m_max, K);
  if (rc != RD_OK) return rc;
  const Int8Args a{codes, ld_codes, scales, W, ldw, w_scales, C, ldc, R, ldr, m_max, m_dev, N, (K + 15) / 16 * 16};
  rc = check_product(out_dtype, a, epilogue);
  if (rc != RD_OK || m_max == 0) return rc;
  rc = quant_rows(dtype, x, ldx, codes, ld_codes, scales, m_max, m_dev, K, (cudaStream_t)stream);
  return rc != RD_OK ? rc : product(out_dtype, a, epilogue, (cudaStream_t)stream);
}

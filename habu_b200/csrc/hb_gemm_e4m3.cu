// Product of two e4m3 matrices with one fp32 scale per 128 values (hb_matmul_scaled).
//
//   C[m, n] = epilogue( sum over k-blocks of 128:  a_scale[m, kb] * b_scale[n / 128, kb] * sum_k A[m, k] B[n, k] )
//
// This is the plain kernel: a 64 x 64 tile per CTA, operands widened to fp32 in shared memory, the
// sum of one k-block kept apart from the running sum so that the scales are applied once per block.
#include <cuda_fp8.h>
#include <string.h>

#include <new>

#include "hb_internal.h"
#include "hb_ptx.cuh"

namespace {

constexpr int KB = 128;          // k per scale

struct ScaledArgs {
  const uint8_t* A;              // [M, lda]
  const uint8_t* B;              // [N, ldb]
  const float* sa;               // strides sa_m, sa_k
  const float* sb;               // strides sb_n, sb_k
  __nv_bfloat16* C;
  const __nv_bfloat16* R;        // residual or null
  int64_t M, N, K, lda, ldb, ldc, ldr, sa_m, sa_k, sb_n, sb_k;
  int epilogue;
  int b_is_weights;
};

__device__ __forceinline__ float gelu_erf(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f)); }
__device__ __forceinline__ float silu(float x) { return x / (1.0f + __expf(-x)); }

__device__ __forceinline__ float from_e4m3(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

constexpr int T = 64, TK = 32;

__global__ void __launch_bounds__(256) hb_matmul_scaled_plain_kernel(const ScaledArgs p) {
  __shared__ float a[TK][T + 1], b[TK][T + 1];
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * T, n0 = static_cast<int64_t>(blockIdx.x) * T;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;       // 4 x 4 outputs: rows ty * 4 + i, columns tx * 4 + j
  float acc[4][4] = {};
  for (int64_t kb = 0; kb * KB < p.K; ++kb) {
    float part[4][4] = {};
    for (int k0 = 0; k0 < KB; k0 += TK) {
      for (int i = threadIdx.x; i < T * TK; i += 256) {
        const int r = i / TK, kk = i % TK;
        const int64_t k = kb * KB + k0 + kk;
        a[kk][r] = m0 + r < p.M && k < p.K ? from_e4m3(p.A[(m0 + r) * p.lda + k]) : 0.f;
        b[kk][r] = n0 + r < p.N && k < p.K ? from_e4m3(p.B[(n0 + r) * p.ldb + k]) : 0.f;
      }
      __syncthreads();
      for (int kk = 0; kk < TK; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) part[i][j] += a[kk][ty * 4 + i] * b[kk][tx * 4 + j];
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
        if (m < p.M && n < p.N) acc[i][j] += part[i][j] * (p.sa[m * p.sa_m + kb * p.sa_k] * p.sb[n / KB * p.sb_n + kb * p.sb_k]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty * 4 + i;
    if (m >= p.M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n >= p.N) continue;
      if (p.epilogue == HB_EPI_SWIGLU) {
        if (!(j & 1)) p.C[m * p.ldc + n / 2] = __float2bfloat16_rn(silu(acc[i][j]) * acc[i][j + 1]);
        continue;
      }
      float v = acc[i][j];
      if (p.epilogue == HB_EPI_GELU) v = gelu_erf(v);
      if (p.epilogue == HB_EPI_RESIDUAL) v += __bfloat162float(p.R[m * p.ldr + n]);
      p.C[m * p.ldc + n] = __float2bfloat16_rn(v);
    }
  }
}

hb_status decode(hb_ctx* ctx, const hb_tensor* A, const hb_tensor* sa, const hb_tensor* B, const hb_tensor* sb,
                 const hb_tensor* C, const hb_matmul_opts* opts, ScaledArgs* g) {
  const char* op = "matmul_scaled";
  if (!A || !sa || !B || !sb || !C) return hb_fail(ctx, HB_ERR_INVALID, "%s: null tensor", op);
  if (A->rank != 2 || B->rank != 2 || C->rank != 2) return hb_fail(ctx, HB_ERR_INVALID, "%s: tensors must have rank 2", op);
  if (!A->ptr || !B->ptr || !C->ptr) return hb_fail(ctx, HB_ERR_INVALID, "%s: null data pointer", op);
  if (A->dtype != HB_E4M3 || B->dtype != HB_E4M3) return hb_fail(ctx, HB_ERR_INVALID, "%s: A and B must be e4m3", op);
  if (C->dtype != HB_BF16) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: C must be bf16", op);
  const int64_t M = A->shape[0], K = A->shape[1], N = B->shape[1];
  const int epi = opts ? (opts->epilogue & 0xff) : HB_EPI_NONE;
  if (epi > HB_EPI_RESIDUAL || (opts && (opts->epilogue & ~(0xff | HB_MATMUL_WEIGHTS_B))))
    return hb_fail(ctx, HB_ERR_INVALID, "%s: unknown epilogue %d", op, opts->epilogue);
  if (opts && opts->config_id != -1) return hb_fail(ctx, HB_ERR_INVALID, "%s: config_id must be -1", op);
  if (M <= 0 || N <= 0 || K <= 0) return hb_fail(ctx, HB_ERR_INVALID, "%s: empty dimension", op);
  if (M > INT32_MAX - 1024 || N > INT32_MAX - 1024 || K > INT32_MAX - 1024)
    return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: dimension too large", op);
  if (B->shape[0] != K)
    return hb_fail(ctx, HB_ERR_INVALID, "%s: inner dimensions differ (A is %lld x %lld, B is %lld x %lld)", op, (long long)M,
                   (long long)K, (long long)B->shape[0], (long long)N);
  if (epi == HB_EPI_SWIGLU && (N & 1)) return hb_fail(ctx, HB_ERR_INVALID, "%s: swiglu epilogue needs an even N", op);
  const int64_t NC = epi == HB_EPI_SWIGLU ? N / 2 : N;
  if (C->shape[0] != M || C->shape[1] != NC) return hb_fail(ctx, HB_ERR_INVALID, "%s: C must be %lld x %lld", op, (long long)M, (long long)NC);
  if (A->stride[1] != 1 && K > 1) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: A must be row-major", op);
  if (B->stride[0] != 1 && K > 1) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: B must be contiguous along K", op);
  if (C->stride[1] != 1 && NC > 1) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: C must be row-major", op);
  if ((M > 1 && (A->stride[0] < K || C->stride[0] < NC)) || (N > 1 && B->stride[1] < K))
    return hb_fail(ctx, HB_ERR_INVALID, "%s: row stride smaller than the width", op);
  // TMA needs 16-byte aligned bases and row pitches.  A pitch that no second row uses is free.
  memset(g, 0, sizeof(*g));
  g->lda = M > 1 ? A->stride[0] : (K + 15) / 16 * 16;
  g->ldb = N > 1 ? B->stride[1] : (K + 15) / 16 * 16;
  if ((reinterpret_cast<uintptr_t>(A->ptr) | reinterpret_cast<uintptr_t>(B->ptr) | (uintptr_t)g->lda | (uintptr_t)g->ldb) & 15)
    return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: A and B need 16-byte aligned bases and row pitches that are multiples of 16", op);
  if (reinterpret_cast<uintptr_t>(C->ptr) & 1) return hb_fail(ctx, HB_ERR_INVALID, "%s: misaligned pointer", op);
  hb_status st = hb_check_scales(ctx, op, sa, M, (K + KB - 1) / KB);
  if (st == HB_OK) st = hb_check_scales(ctx, op, sb, (K + KB - 1) / KB, (N + KB - 1) / KB);
  if (st != HB_OK) return st;
  g->A = static_cast<const uint8_t*>(A->ptr); g->B = static_cast<const uint8_t*>(B->ptr);
  g->sa = static_cast<const float*>(sa->ptr); g->sb = static_cast<const float*>(sb->ptr);
  g->C = static_cast<__nv_bfloat16*>(C->ptr);
  g->M = M; g->N = N; g->K = K;
  g->ldc = M > 1 ? C->stride[0] : NC;
  g->sa_m = sa->stride[0]; g->sa_k = sa->stride[1];
  g->sb_k = sb->stride[0]; g->sb_n = sb->stride[1];
  g->epilogue = epi;
  g->b_is_weights = opts && (opts->epilogue & HB_MATMUL_WEIGHTS_B) ? 1 : 0;
  if (epi == HB_EPI_RESIDUAL) {
    if (!opts->residual) return hb_fail(ctx, HB_ERR_INVALID, "%s: residual epilogue without a residual", op);
    g->R = static_cast<const __nv_bfloat16*>(opts->residual);
    g->ldr = opts->residual_ld ? opts->residual_ld : N;
    if (g->ldr < N && M > 1) return hb_fail(ctx, HB_ERR_INVALID, "%s: residual row stride smaller than its width", op);
    if (reinterpret_cast<uintptr_t>(g->R) & 1) return hb_fail(ctx, HB_ERR_INVALID, "%s: misaligned pointer", op);
  }
  return HB_OK;
}

hb_status matmul_scaled(hb_ctx* ctx, const hb_tensor* A, const hb_tensor* sa, const hb_tensor* B, const hb_tensor* sb,
                        const hb_tensor* C, const hb_matmul_opts* opts) {
  ScaledArgs g;
  const hb_status st = decode(ctx, A, sa, B, sb, C, opts, &g);
  if (st != HB_OK) return st;
  hb_device_guard guard(ctx);
  const dim3 grid((unsigned)((g.N + T - 1) / T), (unsigned)((g.M + T - 1) / T));
  if (grid.y > 65535) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "matmul_scaled: too many rows");
  hb_matmul_scaled_plain_kernel<<<grid, 256, 0, ctx->stream>>>(g);
  ctx->launches++;
  return hb_check_cuda(ctx, cudaGetLastError(), "matmul_scaled launch");
}

}  // namespace

extern "C" hb_status hb_matmul_scaled(hb_ctx* ctx, const hb_tensor* A, const hb_tensor* a_scale, const hb_tensor* B,
                                      const hb_tensor* b_scale, hb_tensor* C, const hb_matmul_opts* opts) {
  if (!ctx) return HB_ERR_INVALID;
  try {
    return matmul_scaled(ctx, A, a_scale, B, b_scale, C, opts);
  } catch (...) {
    return HB_ERR_NOMEM;
  }
}

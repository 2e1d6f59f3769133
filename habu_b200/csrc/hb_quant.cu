// Quantisation to e4m3 with one fp32 scale per 128 values: plain, behind RMSNorm (with the
// residual's addition) and behind SwiGLU.  These kernels produce the operands of
// hb_matmul_scaled; each reads its input once, keeps it in registers while the maximum of a
// group is formed, and writes one byte per value plus four bytes per 128.
//
//   scale = max(max|y| / 448, 2^-126)     q = e4m3(y / scale)
//
// The floor keeps the scale normal and its reciprocal finite, so that a group of zeros (or of
// values so small that 1 / scale would overflow) needs no case of its own.  y / scale is formed as
// y * (1 / scale): 2^-23 off at most, against the 2^-4 of the rounding to e4m3 that follows.
// fmaxf drops NaNs, so a NaN does not spread over its group: its own product is NaN and converts
// to the e4m3 NaN.
#include <cuda_fp8.h>
#include <math.h>

#include <new>

#include "hb_internal.h"

namespace {

constexpr int QG = 128;                   // values per scale
constexpr float Q_TOP = 448.0f;           // largest e4m3 value
constexpr float Q_FLOOR = 1.17549435e-38f;   // 2^-126

#define HB_LAUNCH_DEPENDENTS() asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory")

__device__ __forceinline__ float2 bf2_to_f2(uint32_t v) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
}
__device__ __forceinline__ uint32_t f2_to_bf2(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Maximum over the 16 lanes that hold a group (8 values each); every lane of the warp takes part.
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float scale_of(float amax) { return fmaxf(amax / Q_TOP, Q_FLOOR); }

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
  float m = fabsf(y[0]);
#pragma unroll
  for (int k = 1; k < 8; ++k) m = fmaxf(m, fabsf(y[k]));
  return m;
}
// Eight values to eight e4m3 bytes (to nearest even; beyond 448 saturates, NaN stays NaN).
__device__ __forceinline__ uint2 pack8(const float (&y)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * h] * inv, y[4 * h + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * h + 2] * inv, y[4 * h + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | hi << 16;
  }
  return make_uint2(w[0], w[1]);
}

// ------------------------------------------------------------------ RMSNorm
// One CTA per row, the row in registers, as in hb_rmsnorm: VEC 16-byte vectors per thread.
// Sixteen neighbouring threads hold the 128 values of a group, so its maximum is four shuffles.
constexpr int RMS_THREADS = 256;
constexpr int RMS_MAX_VEC = 8;

struct NormParams {
  const __nv_bfloat16* x;
  const uint4* gain;
  __nv_bfloat16* residual;     // or null
  uint8_t* q;
  float* scale;
  int64_t ldx, ldr, ldq, ss0, ss1;
  int cols8;
  float inv_cols, eps;
};

template <int VEC>
__global__ void __launch_bounds__(RMS_THREADS) rmsnorm_quant_kernel(const NormParams p) {
  __shared__ float red[RMS_THREADS / 32];
  HB_LAUNCH_DEPENDENTS();
  const int64_t row = blockIdx.x;
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + row * p.ldx);
  uint4* rr = p.residual ? reinterpret_cast<uint4*>(p.residual + row * p.ldr) : nullptr;
  float v[VEC][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int c = threadIdx.x + i * RMS_THREADS;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[i][k] = 0.f;
    if (c < p.cols8) {
      const uint4 a = xr[c];
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
      uint32_t rw[4] = {0, 0, 0, 0};
      if (rr) { const uint4 r = rr[c]; rw[0] = r.x; rw[1] = r.y; rw[2] = r.z; rw[3] = r.w; }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 f = bf2_to_f2(aw[k]);
        if (rr) {
          const float2 g = bf2_to_f2(rw[k]);
          // the updated residual is what gets normalised, after its own bf16 rounding
          rw[k] = f2_to_bf2(f.x + g.x, f.y + g.y);
          f = bf2_to_f2(rw[k]);
        }
        v[i][2 * k] = f.x;
        v[i][2 * k + 1] = f.y;
        ss += f.x * f.x + f.y * f.y;
      }
      if (rr) rr[c] = make_uint4(rw[0], rw[1], rw[2], rw[3]);
    }
  }
  ss = warp_sum(ss);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int w = 0; w < RMS_THREADS / 32; ++w) tot += red[w];
  const float inv_rms = rsqrtf(tot * p.inv_cols + p.eps);
  uint8_t* qr = p.q + row * p.ldq;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const int c = threadIdx.x + i * RMS_THREADS;
    if (c < p.cols8) {
      const uint4 g = __ldg(p.gain + c);
      const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 gf = bf2_to_f2(gw[k]);
        v[i][2 * k] *= inv_rms * gf.x;
        v[i][2 * k + 1] *= inv_rms * gf.y;
      }
    }
    const float s = scale_of(group_max(abs_max8(v[i])));
    if (c < p.cols8) {
      *reinterpret_cast<uint2*>(qr + c * 8) = pack8(v[i], 1.0f / s);
      if ((threadIdx.x & 15) == 0) p.scale[row * p.ss0 + (c >> 4) * p.ss1] = s;
    }
  }
}

// ------------------------------------------------------------------ rows of a matrix, and SwiGLU
enum { SRC_BF16 = 0, SRC_F32 = 1, SRC_SWIGLU = 2 };

struct RowParams {
  const void* x;
  uint8_t* q;
  float* scale;
  int64_t rows;
  int64_t ldx, ldq, ss0, ss1;
  int cols;                    // columns of q (SwiGLU: half the columns of x)
};

// v / (1 + exp(-v)): approximate exponential and division (2 ulp each); for v far below zero the
// denominator is infinite and the quotient -0.
__device__ __forceinline__ float silu_f(float v) { return __fdividef(v, 1.0f + __expf(-v)); }

// Eight values of `row` that belong to thread c of the row.  VEC: the consecutive columns 8 c .. 8 c + 7
// in whole 16-byte vectors.  Otherwise (odd widths, pitches or addresses) columns 16 apart inside the
// same group of 128, so that neighbouring threads still read neighbouring elements.
__device__ __forceinline__ int loose_col(int c, int k) { return (c >> 4) * QG + (c & 15) + 16 * k; }
template <int SRC, bool VEC>
__device__ __forceinline__ void load8(const RowParams& p, int64_t row, int c, float (&y)[8]) {
  if constexpr (SRC == SRC_SWIGLU) {
    const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(p.x) + row * p.ldx + c * 8;
    const uint4 g = *reinterpret_cast<const uint4*>(base), u = *reinterpret_cast<const uint4*>(base + p.cols);
    const uint32_t gw[4] = {g.x, g.y, g.z, g.w}, uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = bf2_to_f2(gw[k]), b = bf2_to_f2(uw[k]);
      y[2 * k] = silu_f(a.x) * b.x;
      y[2 * k + 1] = silu_f(a.y) * b.y;
    }
  } else if constexpr (SRC == SRC_BF16) {
    const __nv_bfloat16* row_ptr = static_cast<const __nv_bfloat16*>(p.x) + row * p.ldx;
    if constexpr (VEC) {
      const uint4 g = *reinterpret_cast<const uint4*>(row_ptr + c * 8);
      const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 a = bf2_to_f2(gw[k]);
        y[2 * k] = a.x;
        y[2 * k + 1] = a.y;
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = loose_col(c, k) < p.cols ? __bfloat162float(row_ptr[loose_col(c, k)]) : 0.f;
    }
  } else {
    const float* row_ptr = static_cast<const float*>(p.x) + row * p.ldx;
    if constexpr (VEC) {
      const float4 a = reinterpret_cast<const float4*>(row_ptr + c * 8)[0], b = reinterpret_cast<const float4*>(row_ptr + c * 8)[1];
      y[0] = a.x; y[1] = a.y; y[2] = a.z; y[3] = a.w;
      y[4] = b.x; y[5] = b.y; y[6] = b.z; y[7] = b.w;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = loose_col(c, k) < p.cols ? row_ptr[loose_col(c, k)] : 0.f;
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void store8(const RowParams& p, int64_t row, int c, const float (&y)[8], float inv) {
  uint8_t* dst = p.q + row * p.ldq;
  const uint2 w = pack8(y, inv);
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(dst + c * 8) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (loose_col(c, k) < p.cols) dst[loose_col(c, k)] = static_cast<uint8_t>((k < 4 ? w.x : w.y) >> 8 * (k & 3));
  }
}

// blockDim = (columns / 8 covered at once, rows): every run of 16 threads in x is one group.
template <int SRC, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(const RowParams p) {
  HB_LAUNCH_DEPENDENTS();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  const bool live = row < p.rows && (VEC ? c * 8 : loose_col(c, 0)) < p.cols;
  float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) load8<SRC, VEC>(p, row, c, y);
  const float s = scale_of(group_max(abs_max8(y)));
  if (live) {
    store8<VEC>(p, row, c, y, 1.0f / s);
    if ((threadIdx.x & 15) == 0) p.scale[row * p.ss0 + (c >> 4) * p.ss1] = s;
  }
}

// ------------------------------------------------------------------ 128 x 128 blocks
// One CTA per block, 64 values per thread in registers: 16 threads span the 128 columns, 16 rows
// are read at a time.
template <int SRC, bool VEC>
__global__ void __launch_bounds__(256) quant_blocks_kernel(const RowParams p) {
  __shared__ float red[8];
  HB_LAUNCH_DEPENDENTS();
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * QG + (threadIdx.x >> 4);
  const int c = blockIdx.y * (QG / 8) + (threadIdx.x & 15);
  const bool live = (VEC ? c * 8 : loose_col(c, 0)) < p.cols;
  float y[8][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) y[i][k] = 0.f;
    if (row0 + 16 * i < p.rows && live) load8<SRC, VEC>(p, row0 + 16 * i, c, y[i]);
    m = fmaxf(m, abs_max8(y[i]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  const float s = scale_of(m), inv = 1.0f / s;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (row0 + 16 * i < p.rows && live) store8<VEC>(p, row0 + 16 * i, c, y[i], inv);
  if (threadIdx.x == 0) p.scale[blockIdx.x * p.ss0 + blockIdx.y * p.ss1] = s;
}

bool aligned(const void* ptr, int64_t pitch_bytes, int n) {
  return ((reinterpret_cast<uintptr_t>(ptr) | static_cast<uintptr_t>(pitch_bytes)) & (n - 1)) == 0;
}

// Rank-2 input with contiguous rows.
hb_status check_rows(hb_ctx* ctx, const char* op, const char* what, const hb_tensor* t, int64_t rows, int64_t cols) {
  if (t->rank != 2) return hb_fail(ctx, HB_ERR_INVALID, "%s: %s must have rank 2", op, what);
  if (!t->ptr) return hb_fail(ctx, HB_ERR_INVALID, "%s: null data pointer (%s)", op, what);
  if (t->shape[0] <= 0 || t->shape[1] <= 0) return hb_fail(ctx, HB_ERR_INVALID, "%s: empty dimension", op);
  if (t->shape[0] != rows || t->shape[1] != cols)
    return hb_fail(ctx, HB_ERR_INVALID, "%s: %s must be %lld x %lld", op, what, (long long)rows, (long long)cols);
  if (t->stride[1] != 1 && cols > 1) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: rows of %s must be contiguous", op, what);
  if (t->stride[0] < cols && rows > 1) return hb_fail(ctx, HB_ERR_INVALID, "%s: row stride of %s smaller than its width", op, what);
  return HB_OK;
}

// The (q, scale) pair an operator writes.
hb_status check_pair(hb_ctx* ctx, const char* op, const hb_tensor* q, const hb_tensor* s, int64_t rows, int64_t cols, int block_rows) {
  if (!q || !s) return hb_fail(ctx, HB_ERR_INVALID, "%s: null tensor", op);
  if (rows > INT32_MAX || cols > INT32_MAX - QG) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: dimension exceeds 2^31-1", op);
  if (q->dtype != HB_E4M3) return hb_fail(ctx, HB_ERR_INVALID, "%s: the quantised output must be e4m3", op);
  hb_status st = check_rows(ctx, op, "the quantised output", q, rows, cols);
  if (st != HB_OK) return st;
  return hb_check_scales(ctx, op, s, (rows + block_rows - 1) / block_rows, (cols + QG - 1) / QG);
}

int pow2_up(int64_t v, int lo, int hi) {
  int p = lo;
  while (p < hi && p < v) p *= 2;
  return p;
}

template <int SRC, bool VEC>
hb_status launch_rows(hb_ctx* ctx, const RowParams& p, const char* what) {
  const int64_t vecs = VEC ? p.cols / 8 : (int64_t)(p.cols + QG - 1) / QG * 16;
  const int tx = pow2_up(vecs, 16, 256), ty = 256 / tx;
  const dim3 grid((unsigned)((p.rows + ty - 1) / ty), (unsigned)((vecs + tx - 1) / tx));
  if (grid.y > 65535) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: too many columns", what);
  const cudaError_t e = hb_launch_dependent(quant_rows_kernel<SRC, VEC>, grid, dim3(tx, ty), 0, ctx->stream, p);
  if (e != cudaSuccess) { cudaGetLastError(); return hb_check_cuda(ctx, e, what); }
  ctx->launches++;
  return HB_OK;
}
template <int SRC, bool VEC>
hb_status launch_blocks(hb_ctx* ctx, const RowParams& p, const char* what) {
  const dim3 grid((unsigned)((p.rows + QG - 1) / QG), (unsigned)((p.cols + QG - 1) / QG));
  if (grid.y > 65535) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: too many columns", what);
  const cudaError_t e = hb_launch_dependent(quant_blocks_kernel<SRC, VEC>, grid, dim3(256), 0, ctx->stream, p);
  if (e != cudaSuccess) { cudaGetLastError(); return hb_check_cuda(ctx, e, what); }
  ctx->launches++;
  return HB_OK;
}

hb_status quantize(hb_ctx* ctx, const hb_tensor* x, hb_tensor* q, hb_tensor* scale, int block_rows) {
  const char* op = "quantize";
  if (!x) return hb_fail(ctx, HB_ERR_INVALID, "%s: null tensor", op);
  if (block_rows != 1 && block_rows != QG) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: block_rows must be 1 or 128", op);
  if (x->dtype != HB_BF16 && x->dtype != HB_F32) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: dtype %d is not supported", op, x->dtype);
  hb_status st = check_rows(ctx, op, "x", x, x->shape[0], x->shape[1]);
  if (st != HB_OK) return st;
  const int64_t rows = x->shape[0], cols = x->shape[1];
  if ((st = check_pair(ctx, op, q, scale, rows, cols, block_rows)) != HB_OK) return st;
  const int es = x->dtype == HB_BF16 ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(x->ptr) & (es - 1)) return hb_fail(ctx, HB_ERR_INVALID, "%s: misaligned pointer", op);
  RowParams p = {x->ptr, static_cast<uint8_t*>(q->ptr), static_cast<float*>(scale->ptr), rows, x->stride[0], q->stride[0],
                 scale->stride[0], scale->stride[1], (int)cols};
  // whole 16-byte vectors wherever every row starts on one and ends on one
  const bool vec = cols % 8 == 0 && aligned(x->ptr, x->stride[0] * es, 16) && aligned(q->ptr, q->stride[0], 8);
  hb_device_guard guard(ctx);
#define HB_Q_LAUNCH(F)                                                                                          \
  (x->dtype == HB_BF16 ? (vec ? F<SRC_BF16, true>(ctx, p, op) : F<SRC_BF16, false>(ctx, p, op))                 \
                       : (vec ? F<SRC_F32, true>(ctx, p, op) : F<SRC_F32, false>(ctx, p, op)))
  return block_rows == 1 ? HB_Q_LAUNCH(launch_rows) : HB_Q_LAUNCH(launch_blocks);
#undef HB_Q_LAUNCH
}

hb_status swiglu_quant(hb_ctx* ctx, const hb_tensor* x, hb_tensor* q, hb_tensor* scale) {
  const char* op = "swiglu_quant";
  if (!x) return hb_fail(ctx, HB_ERR_INVALID, "%s: null tensor", op);
  if (x->dtype != HB_BF16) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: dtype %d is not supported", op, x->dtype);
  hb_status st = check_rows(ctx, op, "x", x, x->shape[0], x->shape[1]);
  if (st != HB_OK) return st;
  const int64_t rows = x->shape[0], half = x->shape[1] / 2;
  if (x->shape[1] % 16) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: half width must be a multiple of 8", op);
  if ((st = check_pair(ctx, op, q, scale, rows, half, 1)) != HB_OK) return st;
  if (!aligned(x->ptr, x->stride[0] * 2, 16) || !aligned(q->ptr, q->stride[0], 8))
    return hb_fail(ctx, HB_ERR_INVALID, "%s: rows of x must be 16-byte aligned and rows of the output 8-byte aligned", op);
  RowParams p = {x->ptr, static_cast<uint8_t*>(q->ptr), static_cast<float*>(scale->ptr), rows, x->stride[0], q->stride[0],
                 scale->stride[0], scale->stride[1], (int)half};
  hb_device_guard guard(ctx);
  return launch_rows<SRC_SWIGLU, true>(ctx, p, op);
}

hb_status rmsnorm_quant(hb_ctx* ctx, const hb_tensor* x, const void* gain, hb_tensor* q, hb_tensor* scale, hb_tensor* res, float eps) {
  const char* op = "rmsnorm_quant";
  if (!x || !gain) return hb_fail(ctx, HB_ERR_INVALID, "%s: null tensor", op);
  if (x->dtype != HB_BF16 || (res && res->dtype != HB_BF16))
    return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: x and the residual must be bf16", op);
  hb_status st = check_rows(ctx, op, "x", x, x->shape[0], x->shape[1]);
  if (st != HB_OK) return st;
  const int64_t rows = x->shape[0], cols = x->shape[1];
  if (cols % 8 || cols > RMS_THREADS * RMS_MAX_VEC * 8)
    return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: cols must be a multiple of 8 and at most %d", op, RMS_THREADS * RMS_MAX_VEC * 8);
  if (res && (st = check_rows(ctx, op, "the residual", res, rows, cols)) != HB_OK) return st;
  if ((st = check_pair(ctx, op, q, scale, rows, cols, 1)) != HB_OK) return st;
  if (!aligned(x->ptr, x->stride[0] * 2, 16) || !aligned(gain, 0, 16) || (res && !aligned(res->ptr, res->stride[0] * 2, 16)) ||
      !aligned(q->ptr, q->stride[0], 8))
    return hb_fail(ctx, HB_ERR_INVALID,
                   "%s: gain and rows of x and the residual must be 16-byte aligned, rows of the output 8-byte aligned", op);
  NormParams p = {static_cast<const __nv_bfloat16*>(x->ptr), static_cast<const uint4*>(gain),
                  res ? static_cast<__nv_bfloat16*>(res->ptr) : nullptr, static_cast<uint8_t*>(q->ptr),
                  static_cast<float*>(scale->ptr), x->stride[0], res ? res->stride[0] : 0, q->stride[0], scale->stride[0],
                  scale->stride[1], (int)(cols / 8), 1.0f / (float)cols, eps};
  hb_device_guard guard(ctx);
  const int vec = (int)((cols / 8 + RMS_THREADS - 1) / RMS_THREADS);
  void (*kern)(NormParams) = vec <= 1 ? rmsnorm_quant_kernel<1> : vec <= 2 ? rmsnorm_quant_kernel<2>
                             : vec <= 4 ? rmsnorm_quant_kernel<4> : rmsnorm_quant_kernel<RMS_MAX_VEC>;
  const cudaError_t e = hb_launch_dependent(kern, dim3((unsigned)rows), dim3(RMS_THREADS), 0, ctx->stream, p);
  if (e != cudaSuccess) { cudaGetLastError(); return hb_check_cuda(ctx, e, op); }
  ctx->launches++;
  return HB_OK;
}

}  // namespace

hb_status hb_check_scales(hb_ctx* ctx, const char* op, const hb_tensor* s, int64_t d0, int64_t d1) {
  if (s->rank != 2 || s->dtype != HB_F32) return hb_fail(ctx, HB_ERR_INVALID, "%s: scales must be an fp32 matrix", op);
  if (!s->ptr) return hb_fail(ctx, HB_ERR_INVALID, "%s: null data pointer (scales)", op);
  if (s->shape[0] != d0 || s->shape[1] != d1)
    return hb_fail(ctx, HB_ERR_INVALID, "%s: scales must be %lld x %lld", op, (long long)d0, (long long)d1);
  if (reinterpret_cast<uintptr_t>(s->ptr) & 3) return hb_fail(ctx, HB_ERR_INVALID, "%s: misaligned pointer (scales)", op);
  const int64_t a = s->stride[0], b = s->stride[1];
  const bool own_place = (d0 == 1 || a > 0) && (d1 == 1 || b > 0) &&
                         (d0 == 1 || d1 == 1 || a >= (d1 - 1) * b + 1 || b >= (d0 - 1) * a + 1);
  if (!own_place) return hb_fail(ctx, HB_ERR_INVALID, "%s: scale strides overlap", op);
  return HB_OK;
}

// No C++ exception (the error text allocates) leaves a C entry point.
extern "C" hb_status hb_quantize(hb_ctx* ctx, const hb_tensor* x, hb_tensor* q, hb_tensor* scale, int32_t block_rows) {
  if (!ctx) return HB_ERR_INVALID;
  try {
    return quantize(ctx, x, q, scale, block_rows);
  } catch (...) {
    return HB_ERR_NOMEM;
  }
}
extern "C" hb_status hb_rmsnorm_quant(hb_ctx* ctx, const hb_tensor* x, const void* gain, hb_tensor* q, hb_tensor* scale,
                                      hb_tensor* residual_inout, float eps) {
  if (!ctx) return HB_ERR_INVALID;
  try {
    return rmsnorm_quant(ctx, x, gain, q, scale, residual_inout, eps);
  } catch (...) {
    return HB_ERR_NOMEM;
  }
}
extern "C" hb_status hb_swiglu_quant(hb_ctx* ctx, const hb_tensor* x, hb_tensor* q, hb_tensor* scale) {
  if (!ctx) return HB_ERR_INVALID;
  try {
    return swiglu_quant(ctx, x, q, scale);
  } catch (...) {
    return HB_ERR_NOMEM;
  }
}

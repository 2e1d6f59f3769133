// Quantisation to e4m3 with one fp32 scale per 128 values: plain, behind RMSNorm (with the
// residual's addition) and behind SwiGLU.  These kernels produce the operands of
// hb_matmul_scaled; each reads its input once, keeps it in registers while the maximum of a
// group is formed, and writes one byte per value plus four bytes per 128.
//
//   scale = max(max|y| / 448, 2^-126)     q = e4m3(y / scale)
//
// The floor keeps the scale normal and its reciprocal finite, so that a group of zeros (or of
// values so small that 1 / scale would overflow) needs no case of its own.
// fmaxf drops NaNs, so a NaN does not spread over its group: its own product is NaN and converts
// to the e4m3 NaN.
#include <cuda_fp8.h>
#include <math.h>

#include <atomic>
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
// Two fp32 products, and two multiply-adds, in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\tmul.rn.f32x2 %0, x, y;\n\t}"
      : "=l"(d) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%1, %2};\n\tmov.b64 y, {%3, %4};\n\tmov.b64 z, {%5, %6};\n\tfma.rn.f32x2 %0, x, y, z;\n\t}"
      : "=l"(d) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}
__device__ __forceinline__ uint32_t lane_id() {
  uint32_t l;
  asm("mov.u32 %0, %%laneid;" : "=r"(l));
  return l;
}
// Maximum over the 16 lanes that hold a group (8 values each); every lane of the warp takes part.  The values
// are not negative, so that their bits are in the same order and a reduction of each half-warp's does it.
__device__ __forceinline__ float group_max(float v) {
  const bool upper = lane_id() & 16;
  const uint32_t bits = __float_as_uint(v);
  const uint32_t lo = __reduce_max_sync(0xffffffffu, upper ? 0u : bits), hi = __reduce_max_sync(0xffffffffu, upper ? bits : 0u);
  return __uint_as_float(upper ? hi : lo);
}
// What a group with maximum `top` is stored with: its scale, and the factor that takes a value to q's
// range, q = e4m3(y * to_q).  The factor is 448 / top to within a rounding (the reciprocal of the scale, 1
// ulp, and one correction: a division each for the scale and its inverse would be a fifth of the
// instructions of these kernels), at most 2^126, which is where the scale meets its floor.  No argument
// of the reciprocal is subnormal or has a subnormal result.
struct Scale {
  float s, to_q;
  float rest;                                                  // 448 / top - to_q, for round_exactly
};
__device__ __forceinline__ Scale finite_scale_of(float top) {
  const float s = fmaxf(top * (1.0f / Q_TOP), Q_FLOOR);        // 2^-23 off at most
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  const float to_q = fminf(fmaf(fmaf(-top, r, Q_TOP) * (1.0f / Q_TOP), r, r), 1.0f / Q_FLOOR);
  return {s, to_q, to_q < 1.0f / Q_FLOOR ? fmaf(-top, to_q, Q_TOP) * (1.0f / Q_TOP) * r : 0.0f};
}
// ... and a factor of 0 behind an infinity.
__device__ __forceinline__ Scale scale_of(float top) {
  Scale z = finite_scale_of(top);
  if (!(top < INFINITY)) z.to_q = 0.0f;
  return z;
}

__device__ __forceinline__ float abs_max8(const float (&y)[8]) {
  float m = 0.f;                                // NaNs drop out, eight of them too
#pragma unroll
  for (int k = 0; k < 8; k += 2) asm("max.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(fabsf(y[k])), "f"(fabsf(y[k + 1])));
  return m;
}
// p = fl(y * to_q) is off by two units in its last place at most, which matters where a value half-way between
// two e4m3 values (at most five significant bits) lies that near: there p is taken to the side of it that
// y * 448 / top is on, which the product's own error and the factor's tell.
__device__ __forceinline__ float round_exactly(float p, float y, const Scale& z) {
  const uint32_t u = __float_as_uint(p) + 2, half = u & 0xFFF80000u;
  if ((u & 0x7FFFFu) > 4 || half << 1 == 0 || !(fabsf(p) < INFINITY)) return p;
  const float t = __uint_as_float(half), off = (p - t) + fmaf(y, z.rest, fmaf(y, z.to_q, -p));
  return off == 0.0f ? t : __uint_as_float((off > 0.0f) == (t > 0.0f) ? half + 1 : half - 1);
}
// Eight values to eight e4m3 bytes (to nearest even; beyond 448 saturates, NaN stays NaN).  EXACT: as if y / scale
// had been rounded once; for fp32 inputs, whose only rounding this is (one value in ten million differs; rows of
// 8192 x 4096 26.3 us for 25.9, blocks as before).
template <bool EXACT = false>
__device__ __forceinline__ uint2 pack8(const float (&y)[8], const Scale& z) {
  float p[8];
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const float2 v = mul2(make_float2(y[k], y[k + 1]), make_float2(z.to_q, z.to_q));
    p[k] = v.x;
    p[k + 1] = v.y;
  }
  if constexpr (EXACT) {
    // From 2^-6 on half-way points end in a one and nineteen zeros (a group's largest value, 448, does not);
    // below, in fewer digits.
    uint32_t near = 0xFFFFFFFFu;
    float small = INFINITY;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const uint32_t up = (2u - 0x80000u) << 12;
      near = min(near, min((__float_as_uint(p[k]) << 12) + up, (__float_as_uint(p[k + 1]) << 12) + up));
      small = fminf(small, fminf(fabsf(p[k]), fabsf(p[k + 1])));
    }
    if (near <= 4u << 12 || small < 0x1p-6f) {
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = round_exactly(p[k], y[k], z);
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(p[4 * h], p[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(p[4 * h + 2], p[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | hi << 16;
  }
  return make_uint2(w[0], w[1]);
}

// ------------------------------------------------------------------ RMSNorm
// `tpr` threads take a row (a power of two from 16 on), each VEC 16-byte vectors of it at fixed columns;
// a CTA takes blockDim / tpr rows at a time and goes on to the next ones: it is persistent, and a thread's
// vectors of the next rows are on their way to its own places in shared memory while it works on these.
// With h = x * gain, y = h * r and max|y| = max|h| * r for the row's r = rsqrt(..): y / scale = h * 448 / max|h|
// does not depend on the row's statistic.  So a vector is done with at once and no row stays in registers;
// the scales come behind, for BATCH rows at a time: one barrier, and one thread per group adds up the
// row's sum (a barrier per row, with one warp at the scales and the others waiting for it, was a tenth
// slower).  Where y / scale is not that (the scale meets its floor, r or a maximum is not finite), that
// thread forms the group's q again, from y.
// Bound by HBM with the residual: 8192 x 4096 37.8 us (6.2 TB/s, 95 % of a copy).  Without it 20.0 us
// (5.0 TB/s), bound by its instructions (118 per warp and 256 values; 69 % of the issue slots taken);
// 16 x 4096 2.1 us.  With y in registers until the statistic was there and q formed from it: 37.9 and 26.5 us.
constexpr int RMS_MAX_COLS = 16384;

struct NormParams {
  const __nv_bfloat16* x;
  const uint4* gain;
  __nv_bfloat16* residual;     // or null
  uint8_t* q;
  float* scale;
  uint32_t rows;               // row numbers in 32 bits, offsets in 64: one wide multiply-add each
  uint64_t ldx, ldr, ldq, ss0, ss1;
  uint32_t cols8, tpr;
  float inv_cols, eps;
};

// Own places of a thread: STAGES rows ahead, x and the residual, and the gain where it is not in registers.
template <int VEC, bool RES, int THREADS>
struct NormLayout {
  static constexpr int STAGES = 2;
  static constexpr int BATCH = 4;                                   // rows of a thread between two barriers
  static constexpr bool GAIN_IN_REGS = VEC <= 2;
  static constexpr int PER_STAGE = (RES ? 2 : 1) * VEC * THREADS;   // 16-byte places
  static constexpr int BYTES = 16 * (STAGES * PER_STAGE + (GAIN_IN_REGS ? 0 : VEC * THREADS));
};

template <int VEC, bool RES, int THREADS>
__global__ void __launch_bounds__(THREADS) rmsnorm_quant_kernel(const NormParams p) {
  using L = NormLayout<VEC, RES, THREADS>;
  extern __shared__ uint4 places[];
  constexpr uint32_t BATCH = L::BATCH, SLOTS = THREADS / 16 * VEC;
  static_assert(BATCH * SLOTS <= THREADS, "one thread per group of a batch");
  __shared__ float red[2][BATCH][THREADS / 16], tops[2][BATCH][SLOTS];
  const uint32_t tpr = p.tpr, warps = tpr > 32 ? tpr / 32 : 1;           // warps that share a row
  const uint32_t t = threadIdx.x & (tpr - 1);                       // thread of the row
  const uint32_t sub_row = threadIdx.x / tpr, per_step = THREADS / tpr;
  const uint32_t groups = (p.cols8 + 15) >> 4, row_slots = (tpr >> 4) * VEC;
  uint4* const mine = places + threadIdx.x;
  const uint32_t mine_at = static_cast<uint32_t>(__cvta_generic_to_shared(mine));
  HB_LAUNCH_DEPENDENTS();
  auto request = [&](uint32_t row, int stage) {
    if (row < p.rows) {
      const uint4* xr = reinterpret_cast<const uint4*>(p.x + row * p.ldx) + t;
      const uint4* rr = reinterpret_cast<const uint4*>(p.residual + row * p.ldr) + t;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (t + i * tpr < p.cols8) {
          const uint32_t at = mine_at + (stage * L::PER_STAGE + i * THREADS) * 16;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(xr + i * tpr) : "memory");
          if (RES) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + VEC * THREADS * 16), "l"(rr + i * tpr) : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  uint32_t row = blockIdx.x * per_step + sub_row;
  const uint32_t step = gridDim.x * per_step;
#pragma unroll
  for (int s = 0; s < L::STAGES; ++s) request(row + s * step, s);
  float2 gain[L::GAIN_IN_REGS ? VEC : 1][4];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    const uint4 g = p.gain[min(t + i * tpr, p.cols8 - 1)];   // (a plain load: the kernel in front may have written it)
    if constexpr (L::GAIN_IN_REGS) {
      const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) gain[i][k] = bf2_to_f2(gw[k]);
    } else {
      mine[L::STAGES * L::PER_STAGE + i * THREADS] = g;
    }
  }
  int buf = 0, stage = 0;
  for (uint32_t base = row - sub_row; base < p.rows; base += BATCH * step, buf ^= 1) {   // every thread of the CTA takes every step
#pragma unroll 1
    for (uint32_t j = 0; j < BATCH && base + j * step < p.rows; ++j, row += step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 1) : "memory");
      const uint4* now = mine + stage * L::PER_STAGE;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const bool in = t + i * tpr < p.cols8;                        // (elsewhere the place holds anything)
        const uint4 xv = now[i * THREADS];
        uint32_t w[4] = {xv.x, xv.y, xv.z, xv.w};
        if constexpr (RES) {
          // the updated residual is what gets normalised, after its own bf16 rounding
          const uint4 rv = now[(VEC + i) * THREADS];
          const uint32_t r[4] = {rv.x, rv.y, rv.z, rv.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = bf2_to_f2(w[k]), g = bf2_to_f2(r[k]);
            w[k] = f2_to_bf2(f.x + g.x, f.y + g.y);
          }
          if (in && row < p.rows) reinterpret_cast<uint4*>(p.residual + row * p.ldr)[t + i * tpr] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        uint4 gv = {};
        if constexpr (!L::GAIN_IN_REGS) gv = mine[L::STAGES * L::PER_STAGE + i * THREADS];
        const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
        float2 part = make_float2(0.f, 0.f);
        float h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = bf2_to_f2(w[k]);
          part = fma2(f, f, part);
          const float2 y = mul2(f, L::GAIN_IN_REGS ? gain[L::GAIN_IN_REGS ? i : 0][k] : bf2_to_f2(gw[k]));
          h[2 * k] = y.x;
          h[2 * k + 1] = y.y;
        }
        if (in) ss += part.x + part.y;
        const float top = group_max(in ? abs_max8(h) : 0.f);
        if ((t & 15) == 0) tops[buf][j][sub_row * row_slots + (t + i * tpr) / 16] = top;
        const uint2 q = pack8(h, finite_scale_of(top));
        if (in && row < p.rows) reinterpret_cast<uint2*>(p.q + row * p.ldq)[t + i * tpr] = q;
      }
      request(row + L::STAGES * step, stage);
      if (++stage == L::STAGES) stage = 0;
      for (uint32_t o = (tpr < 32 ? tpr : 32) / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if ((t & 31) == 0) red[buf][j][tpr < 32 ? sub_row : threadIdx.x >> 5] = ss;
    }
    __syncthreads();                                                // the other buffers are rewritten behind the next one
    const uint32_t j = threadIdx.x / SLOTS, slot = threadIdx.x % SLOTS, sub = slot / row_slots, g = slot % row_slots;
    const uint32_t at = base + j * step + sub;
    if (j < BATCH && g < groups && at < p.rows) {
      float ss = 0.f;
      for (uint32_t w = 0; w < warps; ++w) ss += red[buf][j][sub * warps + w];
      const float inv_rms = rsqrtf(ss * p.inv_cols + p.eps), top = tops[buf][j][slot];
      Scale z = finite_scale_of(top * inv_rms);
      if (!(top >= Q_TOP * Q_FLOOR && z.s > Q_FLOOR && z.s < INFINITY) && !(top == 0.f && inv_rms < INFINITY)) {
        z = scale_of(top * inv_rms);
        const __nv_bfloat16* v = (RES ? p.residual + at * p.ldr : p.x + at * p.ldx) + g * QG;
        const __nv_bfloat16* gain = reinterpret_cast<const __nv_bfloat16*>(p.gain) + g * QG;
        uint8_t* q = p.q + at * p.ldq + g * QG;
#pragma unroll 1
        for (uint32_t k = 0; k < min(uint32_t{QG}, p.cols8 * 8 - g * QG); ++k)
          q[k] = __nv_cvt_float_to_fp8(__bfloat162float(v[k]) * __bfloat162float(gain[k]) * inv_rms * z.to_q, __NV_SATFINITE, __NV_E4M3);
      }
      p.scale[at * p.ss0 + g * p.ss1] = z.s;
    }
  }
}

// ------------------------------------------------------------------ rows of a matrix, and SwiGLU
enum { SRC_BF16 = 0, SRC_F32 = 1, SRC_SWIGLU = 2 };

struct RowParams {
  const void* x;
  uint8_t* q;
  float* scale;
  uint32_t rows;
  uint64_t ldx, ldq, ss0, ss1;
  int cols;                    // columns of q (SwiGLU: half the columns of x)
};

// v / (1 + exp(-v)): approximate exponential and division, 2^-21 off at most for |v| < 20 (the accurate
// ones took SwiGLU of 8192 x 14336 from 97 to 149 us); far below zero the denominator is infinite and the
// quotient -0.
__device__ __forceinline__ float silu_f(float v) { return __fdividef(v, 1.0f + __expf(-v)); }

// Eight values of `row` that belong to thread c of the row.  VEC: the consecutive columns 8 c .. 8 c + 7
// in whole 16-byte vectors.  Otherwise (odd widths, pitches or addresses) columns 16 apart inside the
// same group of 128, so that neighbouring threads still read neighbouring elements.
__device__ __forceinline__ int loose_col(int c, int k) { return (c >> 4) * QG + (c & 15) + 16 * k; }
// load() only requests; widen() is where the thread first waits.  Rows and columns past the edge
// repeat the last ones, so that no load hides behind a branch; the caller drops what it does not own.
template <int SRC, bool VEC>
struct Values {
  uint4 a, b;                  // VEC: the 16-byte vectors (b: the up half, or the second four fp32 values)
  float f[8];                  // otherwise
  __device__ __forceinline__ void load(const RowParams& p, uint32_t row, int c) {
    if constexpr (SRC == SRC_SWIGLU) {
      const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(p.x) + row * p.ldx + c * 8;
      a = *reinterpret_cast<const uint4*>(base);
      b = *reinterpret_cast<const uint4*>(base + p.cols);
    } else if constexpr (SRC == SRC_BF16) {
      const __nv_bfloat16* base = static_cast<const __nv_bfloat16*>(p.x) + row * p.ldx;
      if constexpr (VEC) {
        a = *reinterpret_cast<const uint4*>(base + c * 8);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = __bfloat162float(base[min(loose_col(c, k), p.cols - 1)]);
      }
    } else {
      const float* base = static_cast<const float*>(p.x) + row * p.ldx;
      if constexpr (VEC) {
        a = reinterpret_cast<const uint4*>(base + c * 8)[0];
        b = reinterpret_cast<const uint4*>(base + c * 8)[1];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = base[min(loose_col(c, k), p.cols - 1)];
      }
    }
  }
  __device__ __forceinline__ void widen(float (&y)[8]) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = f[k];     // repeats of the last column do not change a maximum
    } else if constexpr (SRC == SRC_F32) {
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = __uint_as_float(w[k]);
    } else {
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = bf2_to_f2(aw[k]);
        y[2 * k] = v.x;
        y[2 * k + 1] = v.y;
      }
      if constexpr (SRC == SRC_SWIGLU) {
        const uint32_t bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 u = bf2_to_f2(bw[k]);
          y[2 * k] = silu_f(y[2 * k]) * u.x;
          y[2 * k + 1] = silu_f(y[2 * k + 1]) * u.y;
        }
      }
    }
  }
};

template <bool VEC, bool EXACT>
__device__ __forceinline__ void store8(const RowParams& p, uint32_t row, int c, const float (&y)[8], const Scale& z) {
  uint8_t* dst = p.q + row * p.ldq;
  const uint2 w = pack8<EXACT>(y, z);
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(dst + c * 8) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (loose_col(c, k) < p.cols) dst[loose_col(c, k)] = static_cast<uint8_t>((k < 4 ? w.x : w.y) >> 8 * (k & 3));
  }
}

// blockDim = (columns / 8 covered at once, rows): every run of 16 threads in x is one group.  A thread takes
// the same columns of UNROLL rows, all of them requested before the first is used.  Bound by HBM: with one
// 16-byte load per thread 8192 x 4096 bf16 took 21.7 us, with two 17.1, three 16.4 (6.2 TB/s), four 18.7, eight
// 19.1; fp32 26.0 us with three (6.5 TB/s); SwiGLU 8192 x 14336 94 us (6.2 TB/s).  Rows that allow no 16-byte
// vectors (8192 x 4001): 25.7 us.
constexpr int ROWS_MANY = 3;
template <int SRC, bool VEC, int UNROLL>
__global__ void __launch_bounds__(256) quant_rows_kernel(const RowParams p) {
  HB_LAUNCH_DEPENDENTS();
  const uint32_t row0 = blockIdx.x * blockDim.y * UNROLL + threadIdx.y;
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  const bool mine = (VEC ? c * 8 : loose_col(c, 0)) < p.cols;
  const int c_load = mine ? c : 0;
  Values<SRC, VEC> v[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) v[i].load(p, min(row0 + i * blockDim.y, p.rows - 1), c_load);
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    const uint32_t row = row0 + i * blockDim.y;
    float y[8];
    v[i].widen(y);
    const Scale z = scale_of(group_max(mine ? abs_max8(y) : 0.f));
    if (mine && row < p.rows) {
      store8<VEC, SRC == SRC_F32>(p, row, c, y, z);
      if ((threadIdx.x & 15) == 0) p.scale[row * p.ss0 + (c >> 4) * p.ss1] = z.s;
    }
  }
}

// ------------------------------------------------------------------ 128 x 128 blocks
// One CTA per block, 64 values per thread in registers: 16 threads span the 128 columns, 16 rows
// are read at a time.  Bound by HBM: 28672 x 4096 from fp32 94 us (6.2 TB/s), from bf16 57 us (6.2 TB/s; 65 us
// with two CTAs per SM instead of three).
template <int SRC, bool VEC>
__global__ void __launch_bounds__(256, VEC ? 3 : 2) quant_blocks_kernel(const RowParams p) {
  __shared__ float red[8];
  HB_LAUNCH_DEPENDENTS();
  const uint32_t row0 = blockIdx.x * QG + (threadIdx.x >> 4);
  const int c = blockIdx.y * (QG / 8) + (threadIdx.x & 15);
  const bool live = (VEC ? c * 8 : loose_col(c, 0)) < p.cols;
  const int c_load = live ? c : 0;
  Values<SRC, VEC> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i].load(p, min(row0 + 16 * i, p.rows - 1), c_load);
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float y[8];
    v[i].widen(y);
    if (live && row0 + 16 * i < p.rows) m = fmaxf(m, abs_max8(y));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  const Scale z = scale_of(m);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (row0 + 16 * i < p.rows && live) {
      float y[8];
      v[i].widen(y);
      store8<VEC, SRC == SRC_F32>(p, row0 + 16 * i, c, y, z);
    }
  if (threadIdx.x == 0) p.scale[blockIdx.x * p.ss0 + blockIdx.y * p.ss1] = z.s;
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
  const int64_t across = (vecs + tx - 1) / tx;
  if (across > 65535) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: too many columns", what);
  // several rows per thread once there is work for every SM with that
  const bool many = (p.rows + ROWS_MANY * ty - 1) / (ROWS_MANY * ty) * across >= 4 * ctx->sm_count;
  const int rows = many ? ROWS_MANY * ty : ty;
  const dim3 grid((unsigned)((p.rows + rows - 1) / rows), (unsigned)across);
  const cudaError_t e = hb_launch_dependent(many ? quant_rows_kernel<SRC, VEC, ROWS_MANY> : quant_rows_kernel<SRC, VEC, 1>, grid, dim3(tx, ty),
                                            0, ctx->stream, p);
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
  RowParams p = {x->ptr, static_cast<uint8_t*>(q->ptr), static_cast<float*>(scale->ptr), (uint32_t)rows, (uint64_t)x->stride[0], (uint64_t)q->stride[0],
                 (uint64_t)scale->stride[0], (uint64_t)scale->stride[1], (int)cols};
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
  RowParams p = {x->ptr, static_cast<uint8_t*>(q->ptr), static_cast<float*>(scale->ptr), (uint32_t)rows, (uint64_t)x->stride[0], (uint64_t)q->stride[0],
                 (uint64_t)scale->stride[0], (uint64_t)scale->stride[1], (int)half};
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
  if (cols % 8 || cols > RMS_MAX_COLS)
    return hb_fail(ctx, HB_ERR_UNSUPPORTED, "%s: cols must be a multiple of 8 and at most %d", op, RMS_MAX_COLS);
  if (res && (st = check_rows(ctx, op, "the residual", res, rows, cols)) != HB_OK) return st;
  if ((st = check_pair(ctx, op, q, scale, rows, cols, 1)) != HB_OK) return st;
  if (!aligned(x->ptr, x->stride[0] * 2, 16) || !aligned(gain, 0, 16) || (res && !aligned(res->ptr, res->stride[0] * 2, 16)) ||
      !aligned(q->ptr, q->stride[0], 8))
    return hb_fail(ctx, HB_ERR_INVALID,
                   "%s: gain and rows of x and the residual must be 16-byte aligned, rows of the output 8-byte aligned", op);
  const int cols8 = (int)(cols / 8);
  // 16-byte vectors per thread, and threads
  const int vec = cols8 <= 16 ? 1 : cols8 <= 512 ? 2 : 4;
  const int tpr = pow2_up((cols8 + vec - 1) / vec, 16, 512);
  const int threads = tpr > 256 ? tpr : 256;
  NormParams p = {static_cast<const __nv_bfloat16*>(x->ptr), static_cast<const uint4*>(gain),
                  res ? static_cast<__nv_bfloat16*>(res->ptr) : nullptr, static_cast<uint8_t*>(q->ptr),
                  static_cast<float*>(scale->ptr), (uint32_t)rows, (uint64_t)x->stride[0], (uint64_t)(res ? res->stride[0] : 0),
                  (uint64_t)q->stride[0], (uint64_t)scale->stride[0], (uint64_t)scale->stride[1], (uint32_t)cols8, (uint32_t)tpr,
                  1.0f / (float)cols, eps};
  hb_device_guard guard(ctx);
  int variant, bytes;
  void (*kern)(NormParams);
#define HB_NORM_PICK(I, VEC, T)                                                                             \
  (variant = I, bytes = res ? NormLayout<VEC, true, T>::BYTES : NormLayout<VEC, false, T>::BYTES,           \
   kern = res ? rmsnorm_quant_kernel<VEC, true, T> : rmsnorm_quant_kernel<VEC, false, T>)
  if (vec == 1) HB_NORM_PICK(0, 1, 256);
  else if (vec == 2) HB_NORM_PICK(1, 2, 256);
  else if (threads == 256) HB_NORM_PICK(2, 4, 256);
  else HB_NORM_PICK(3, 4, 512);
#undef HB_NORM_PICK
  static std::atomic<int> resident[64][4][2];                       // CTAs per SM, by device and variant
  std::atomic<int>& known = resident[ctx->device & 63][variant][res ? 1 : 0];
  int per_sm = known.load(std::memory_order_acquire);
  if (!per_sm) {
    HB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    HB_CUDA(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, bytes));
    if (per_sm < 1) per_sm = 1;
    known.store(per_sm, std::memory_order_release);
  }
  const int64_t steps = (rows + threads / tpr - 1) / (threads / tpr);
  // With the residual two CTAs per SM keep enough in flight; with more, reads and writes disturb each other:
  // 8192 x 4096 37.8 us with two, 47.4 with three, 44.3 with four, 16384 x 512 11.4, 13.0 and 11.3.  Without it
  // 22.6, 20.7 and 20.9 us, and 7.6, 9.1 and 7.0.
  const int ctas = per_sm < (res ? 2 : 4) ? per_sm : (res ? 2 : 4);
  const int64_t most = (int64_t)ctx->sm_count * ctas;
  const cudaError_t e = hb_launch_dependent(kern, dim3((unsigned)(steps < most ? steps : most)), dim3(threads), bytes, ctx->stream, p);
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

// Product of two e4m3 matrices with one fp32 scale per 128 values (hb_matmul_scaled).
//
//   C[m, n] = epilogue( sum over k-blocks of 128:  a_scale[m, kb] * b_scale[n / 128, kb] * sum_k A[m, k] B[n, k] )
//
// The tensor cores sum one k-block (four tcgen05.mma of K = 32) into a slot of tensor memory; the
// scales differ from block to block, so the running sum cannot stay there.  Eight warps take each
// finished slot into registers and add it, times a_scale * b_scale, to fp32 accumulators that they
// hold for the whole tile: one packed multiply-add per two outputs and k-block.  One tensor-memory
// lane is one row of the tile and a warp's columns lie inside one 128-wide block of B, so the
// factor is one register per thread and k-block.  The slots (two of 256 columns, or four) let the
// tensor cores work on the next k-blocks meanwhile.
//
// Warp roles: warp 0 loads (TMA, 128-byte rows of one k-block, 128-byte swizzle), warp 1 issues the
// MMAs, warps 4..11 take the sums and write the tile.  The accumulators need more registers than
// an even share, so the first four warps hand some of theirs over (setmaxnreg; the shares add up to
// what the launch holds).
// Algorithmic traffic per launch: M*K + N*K + 2*M*N bytes and the scales; work 2*M*N*K flop at the
// 8-bit tensor rate (twice that of bf16).
//
// What bounds a large product is the board's power limit, which settles the clock at 1.25 to 1.5 GHz, and
// at that clock the way of a slot from the tensor cores through the sums and back: a k-block of the
// 256 x 256 tile takes about 750 clocks, its MMAs 512.  8192 x 4096 x 14336: 400 us in a burst, 467 sustained
// (2.06 PFLOP/s); 8192 x 28672 x 4096 with SwiGLU 947 us sustained; the same with one scale for all of A and
// one for B, in a library, 378 and 781 us sustained.  Measured and not taken: slots of 128 columns (each MMA
// then reads A again: 535 us where this took 509), two buffers of 32 columns behind each other (they do not
// fit the registers: 560), sums of sixteen columns at a time (472).
#include <math.h>
#include <string.h>

#include <atomic>
#include <new>

#include "hb_internal.h"
#include "hb_ptx.cuh"

namespace {

using namespace hb;

constexpr int KB = 128;          // k per scale, and bytes of a row that one ring stage holds
constexpr int UMMA_K = 32;
constexpr int TILE_THREADS = 384;
constexpr int EPI_WARP0 = 4, EPI_WARPS = 8;
constexpr int REGS_LAUNCH = 168, REGS_FEW = 40, REGS_MANY = 232;   // per thread, multiples of 8
static_assert(REGS_FEW + 2 * REGS_MANY <= 3 * REGS_LAUNCH && TILE_THREADS * REGS_LAUNCH <= 65536, "register split");

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

struct TileParams {
  const float* sa;
  const float* sb;
  __nv_bfloat16* C;
  const __nv_bfloat16* R;
  int64_t ldc, ldr, sa_m, sa_k, sb_n, sb_k;
  int M, N, num_kb, nblocks;     // nblocks: 128-wide blocks of B
  int tiles_m, tiles_n, raster_group;
  int tma_store;
  int split;                     // CTAs that share a tile's k-blocks
  int32_t* status;
};

// Output staging: each epilogue warp owns four buffers of 32 rows x 32 bf16 columns (64-byte rows,
// 64-byte swizzle: the 16-byte piece c of row r sits at piece c ^ ((r >> 1) & 3)), enough for its
// share of a tile, so that one proxy fence covers all of a tile's stores.
constexpr int STAGE_BUF_BYTES = 32 * 64;
constexpr int STAGE_BUFS = 4;
constexpr int STAGE_BYTES = EPI_WARPS * STAGE_BUFS * STAGE_BUF_BYTES;

constexpr int SPLIT_MAX = 4;       // CTAs that may share a tile's k-blocks (its sums travel in pieces of sixteen columns)
// PAIR: two CTAs share a tile of 256 rows.  SPLIT: a cluster of CTAs shares the k-blocks of one tile.
enum { TILE_ONE = 0, TILE_PAIR = 1, TILE_SPLIT = 2 };

template <int KIND, int BN, int STAGES>
struct TileLayout {
  static constexpr bool PAIR = KIND == TILE_PAIR;
  static constexpr int BM = PAIR ? 256 : 128;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;      // rows of B that one CTA loads
  static constexpr int A_BYTES = 128 * KB;
  static constexpr int B_BYTES = B_ROWS * KB;
  static constexpr int SLOTS = 512 / BN;
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = OFF_A + STAGES * A_BYTES;
  static constexpr int OFF_STAGE = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_BAR = OFF_STAGE + STAGE_BYTES;
  static constexpr int NUM_BARS = 2 * STAGES + 2 * SLOTS + 2 * EPI_WARPS;   // full, empty, tfull, tempty, xready, xfull
  static constexpr int OFF_TMEM_PTR = OFF_BAR + NUM_BARS * 8;
  static constexpr int OFF_ABORT = OFF_TMEM_PTR + 4;
  static constexpr int TOTAL = OFF_ABORT + 4;
  static constexpr int DYN_BYTES = TOTAL + 1024;         // slack for 1024-byte alignment
  static_assert(DYN_BYTES <= 227 * 1024, "ring does not fit shared memory");
};

// approximate exponential and division, 2 ulp each; far below zero the denominator is infinite and the quotient -0
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// kind::f8f6f4, both operands e4m3 (format 0) and K-major, fp32 sums:
//   [4,6) D format (1 = f32)   [17,23) N >> 3   [24,29) M >> 4
constexpr uint32_t umma_idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// Shared-memory descriptor of a K-major tile with 128-byte rows and 128-byte swizzle (as
// umma_desc_k_sw128), in two words: the low one carries the address and moves by plain addition.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr) { return ((smem_addr & 0x3FFFFu) >> 4) | (1u << 16); }
// One step of K = 32 (number STEP of a k-block; the first overwrites D).
#define HB_UMMA(GROUP, D, A_LO, B_LO, STEP)                                                                               \
  asm volatile(                                                                                                           \
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t" \
      "tcgen05.mma.cta_group::" #GROUP ".kind::f8f6f4 [%0], da, db, %4, p;\n\t}\n" ::"r"(D),                              \
      "r"((A_LO) + (STEP) * (UMMA_K >> 4)), "r"((B_LO) + (STEP) * (UMMA_K >> 4)), "r"(DESC_HI), "r"(idesc), "n"((STEP) > 0)   \
      : "memory")
static_assert(KB / UMMA_K == 4, "four steps");
// One k-block.  Executed by a whole converged warp -- one thread issues -- so that the operands stay in uniform
// registers; a loop inside a one-thread branch has to move every operand there and took some 500 clocks per
// k-block.
template <int CTA_GROUP>
__device__ __forceinline__ void umma_kblock(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  if constexpr (CTA_GROUP == 1) {
    HB_UMMA(1, d, a_lo, b_lo, 0); HB_UMMA(1, d, a_lo, b_lo, 1); HB_UMMA(1, d, a_lo, b_lo, 2); HB_UMMA(1, d, a_lo, b_lo, 3);
  } else {
    HB_UMMA(2, d, a_lo, b_lo, 0); HB_UMMA(2, d, a_lo, b_lo, 1); HB_UMMA(2, d, a_lo, b_lo, 2); HB_UMMA(2, d, a_lo, b_lo, 3);
  }
}
// Two k-blocks for two slots, their steps in turn: with as few columns as A has rows there, an MMA waits longer
// for the one before it on the same sums than it takes.
__device__ __forceinline__ void umma_two(uint32_t d0, uint32_t a0, uint32_t b0, uint32_t d1, uint32_t a1, uint32_t b1, uint32_t idesc) {
  HB_UMMA(1, d0, a0, b0, 0); HB_UMMA(1, d1, a1, b1, 0);
  HB_UMMA(1, d0, a0, b0, 1); HB_UMMA(1, d1, a1, b1, 1);
  HB_UMMA(1, d0, a0, b0, 2); HB_UMMA(1, d1, a1, b1, 2);
  HB_UMMA(1, d0, a0, b0, 3); HB_UMMA(1, d1, a1, b1, 3);
}
#undef HB_UMMA
// Two sums at once: acc += t * f.  Volatile like the tensor-memory load and the wait for it, so that it stays behind both.
__device__ __forceinline__ void fma2(uint64_t& acc, uint32_t t0, uint32_t t1, uint64_t f) {
  asm volatile("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, t, %3, %0;\n\t}" : "+l"(acc) : "r"(t0), "r"(t1), "l"(f));
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
// x Phi(x) = max(x, 0) - b erfc(sqrt(2) b) with b = |x| / 2, where nothing cancels.  -log2 erfc(sqrt(2) b) is smooth
// and nearly a parabola: a polynomial of degree 8 without a constant (least squares, the weights moved
// towards the largest error) and one exponential give erfc to 2^-17 of itself for |x| < 5.2, 2^-14 up to 6 and 2^-5
// beyond, where the product is below 1e-8; the rounding to bf16 takes up to 2^-8.  Two values at a time.  With
// 0.5 x (1 + erff(x / sqrt(2))) 3766 x 22616 x 384 took 163 us, so it takes 96 (59 without an epilogue).
__device__ __forceinline__ void gelu2(float& x, float& y) {
  constexpr float Q[8] = {-2.30247927f, -1.83368206f, -0.432660699f, 0.137890294f, -0.0313005634f, 0.00462997565f, -0.000390943867f, 1.40522461e-05f};
  const float hx = 0.5f * x, hy = 0.5f * y;
  const float bx = fminf(fabsf(hx), 8.0f), by = fminf(fabsf(hy), 8.0f);    // from there on erfc is 0
  const uint64_t b = pack2(bx, by);
  uint64_t q = pack2(Q[7], Q[7]);
#pragma unroll
  for (int k = 6; k >= 0; --k) asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(q) : "l"(b), "l"(pack2(Q[k], Q[k])));
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(q) : "l"(b));
  float2 e = unpack2(q);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
  x = fmaf(-bx, e.x, hx + fabsf(hx));
  y = fmaf(-by, e.y, hy + fabsf(hy));
}

__device__ __forceinline__ void tile_coords(int tile, const TileParams& p, int& tm, int& tn) {
  // N is swept inside groups of M-tiles, so that CTAs that run together share rows of A and B in L2
  const int per_group = p.raster_group * p.tiles_n;
  const int group = tile / per_group;
  const int first_m = group * p.raster_group;
  const int rows = min(p.raster_group, p.tiles_m - first_m);
  const int in_group = tile - group * per_group;
  tm = first_m + in_group % rows;
  tn = in_group / rows;
}

// ---- blocks of 32 rows x COLS bf16 columns in a warp's staging buffer.  COLS = 32: 64-byte rows, the
// 16-byte piece c of row r at piece c ^ ((r >> 1) & 3), which is TMA's 64-byte swizzle; COLS = 16: plain
// 32-byte rows.
template <int COLS>
__device__ __forceinline__ uint32_t piece_at(uint32_t buf, int r, int c) {
  return buf + r * (2 * COLS) + ((COLS == 32 ? c ^ ((r >> 1) & 3) : c) << 4);
}
// This lane's row (row number `lane`) of a block: COLS fp32 values, rounded once.
template <int COLS>
__device__ __forceinline__ void put_row(uint32_t buf, int lane, const float* f) {
#pragma unroll
  for (int c = 0; c < COLS / 8; ++c)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at<COLS>(buf, lane, c)), "r"(pack_bf16x2(f[8 * c], f[8 * c + 1])),
                 "r"(pack_bf16x2(f[8 * c + 2], f[8 * c + 3])), "r"(pack_bf16x2(f[8 * c + 4], f[8 * c + 5])),
                 "r"(pack_bf16x2(f[8 * c + 6], f[8 * c + 7]))
                 : "memory");
}
// ... and the same read back and added (the residual).
template <int COLS>
__device__ __forceinline__ void add_row(uint32_t buf, int lane, float* f) {
#pragma unroll
  for (int c = 0; c < COLS / 8; ++c) {
    uint32_t w[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(piece_at<COLS>(buf, lane, c)) : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[8 * c + 2 * j] += __uint_as_float(w[j] << 16);
      f[8 * c + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
    }
  }
}
// A matrix in memory, row-major bf16; `width` bytes of it (16, 4 or 2) can be moved at once, by its base
// and pitch.
struct Rows {
  uintptr_t base;
  int64_t pitch;               // bytes
  int rows, cols, width;
};
__device__ __forceinline__ Rows rows_of(const void* ptr, int64_t ld, int rows, int cols) {
  const uintptr_t base = reinterpret_cast<uintptr_t>(ptr), both = base | static_cast<uintptr_t>(ld * 2);
  return {base, ld * 2, rows, cols, (both & 15) == 0 ? 16 : (both & 3) == 0 ? 4 : 2};
}
// Copies the block at (row0, col0) between memory and a staging buffer, whole warp: neighbouring lanes
// take neighbouring pieces of a row, so that every instruction moves contiguous bytes.  What lies
// outside the matrix is not touched.  A row per lane, as the accumulators lie, would touch 32 lines for
// 64 bytes: 3647 x 1420 x 298 took 69 us that way.
template <int WIDTH>
struct Piece;
template <>
struct Piece<16> { using T = uint4; };
template <>
struct Piece<4> { using T = uint32_t; };
template <>
struct Piece<2> { using T = uint16_t; };
__device__ __forceinline__ void ld_shared(uint32_t at, uint4& v) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
}
__device__ __forceinline__ void ld_shared(uint32_t at, uint32_t& v) { asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory"); }
__device__ __forceinline__ void ld_shared(uint32_t at, uint16_t& v) { asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at) : "memory"); }
__device__ __forceinline__ void st_shared(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t at, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void st_shared(uint32_t at, uint16_t v) { asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"(v) : "memory"); }

template <int COLS, bool STORE, int WIDTH>
__device__ __forceinline__ void move_pieces(const Rows& m, uint32_t buf, int lane, int row0, int col0) {
  using T = typename Piece<WIDTH>::T;
  constexpr int PER_ROW = 2 * COLS / WIDTH, ROWS = 32 / PER_ROW;    // lanes per row, rows per step
  constexpr int STEPS = 32 / ROWS, BATCH = STEPS < 8 ? STEPS : 8;   // steps whose loads go out together
  const int in_row = lane % PER_ROW * WIDTH, col = col0 + in_row / 2;
  const bool whole = col + WIDTH / 2 <= m.cols;
  const int left = whole ? m.rows - row0 : 0;                       // rows of the block that exist
  const char* mem = reinterpret_cast<const char*>(m.base) + (row0 + lane / PER_ROW) * m.pitch + 2 * static_cast<int64_t>(col);
  const int64_t step = ROWS * m.pitch;
#pragma unroll 1
  for (int s0 = 0; s0 < STEPS; s0 += BATCH) {
    T v[BATCH] = {};
    const int r0 = s0 * ROWS + lane / PER_ROW;
    const char* at = mem;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int r = r0 + i * ROWS;
      if constexpr (STORE) ld_shared(piece_at<COLS>(buf, r, in_row >> 4) + (in_row & 15), v[i]);
      else if (r < left) v[i] = *reinterpret_cast<const T*>(at);
      at += step;
    }
    at = mem;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int r = r0 + i * ROWS;
      if constexpr (!STORE) st_shared(piece_at<COLS>(buf, r, in_row >> 4) + (in_row & 15), v[i]);
      else if (r < left) *reinterpret_cast<T*>(const_cast<char*>(at)) = v[i];
      at += step;
    }
    mem = at;
  }
  if (WIDTH > 2 && !whole && col < m.cols) {         // the rows end inside this lane's piece
    for (int r = lane / PER_ROW; r < 32 && row0 + r < m.rows; r += ROWS)
      for (int j = 0; j < WIDTH / 2 && col + j < m.cols; ++j) {
        const uint32_t at = piece_at<COLS>(buf, r, in_row >> 4) + (in_row & 15) + 2 * j;
        uint16_t* mem = reinterpret_cast<uint16_t*>(m.base + (row0 + r) * m.pitch + 2 * static_cast<int64_t>(col + j));
        uint16_t v;
        if constexpr (STORE) {
          ld_shared(at, v);
          *mem = v;
        } else {
          v = *mem;
          st_shared(at, v);
        }
      }
  }
}
template <int COLS, bool STORE>
__device__ __forceinline__ void move_block(const Rows& m, uint32_t buf, int lane, int row0, int col0) {
  if (m.width == 16) move_pieces<COLS, STORE, 16>(m, buf, lane, row0, col0);
  else if (m.width == 4) move_pieces<COLS, STORE, 4>(m, buf, lane, row0, col0);
  else move_pieces<COLS, STORE, 2>(m, buf, lane, row0, col0);
}

// The accumulators of one thread (row `row0 + lane`, HALF columns from col0 on) -> C: rounded once into
// the warp's staging buffers, and from there by TMA (whole lines, clipped at the matrix edge) or, where
// C's base, pitch or width allow no tensor map, by the warp.  The epilogue is a template argument here
// and in the kernels: this code runs once per tile, and what it takes is mostly the fetching of its
// instructions.
template <int EPI, int HALF>
__device__ __forceinline__ void write_half(const TileParams& p, const CUtensorMap* tmC, uint32_t stage, int lane, int row0,
                                           int col0, const uint64_t (&acc)[HALF / 2]) {
  if (p.tma_store) {
    if (lane == 0) tma_store_wait_read<0>();     // the last tile's stores have read the buffers
    __syncwarp();
  }
  constexpr bool swiglu = EPI == HB_EPI_SWIGLU;
  constexpr int BLOCKS = swiglu ? HALF / 64 : HALF / 32;
  const int first = swiglu ? col0 >> 1 : col0, ncols = swiglu ? p.N >> 1 : p.N;
  if constexpr (EPI == HB_EPI_RESIDUAL) {
    const Rows r = rows_of(p.R, p.ldr, p.M, p.N);
    for (int c = 0; c < BLOCKS; ++c) move_block<32, false>(r, stage + c * STAGE_BUF_BYTES, lane, row0, first + c * 32);
    __syncwarp();
  }
#pragma unroll
  for (int c = 0; c < BLOCKS; ++c) {
    const uint32_t buf = stage + c * STAGE_BUF_BYTES;
    float f[32];
    if constexpr (swiglu) {                        // columns interleave (gate, up): 64 sums give 32 outputs
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float2 gu = unpack2(acc[c * 32 + j]);
        f[j] = silu(gu.x) * gu.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 v = unpack2(acc[c * 16 + j]);
        f[2 * j] = v.x;
        f[2 * j + 1] = v.y;
      }
    }
    if constexpr (EPI == HB_EPI_GELU) {
#pragma unroll
      for (int j = 0; j < 32; j += 2) gelu2(f[j], f[j + 1]);
    }
    if constexpr (EPI == HB_EPI_RESIDUAL) add_row<32>(buf, lane, f);
    put_row<32>(buf, lane, f);
  }
  if (p.tma_store) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && row0 < p.M) {
      for (int c = 0; c < BLOCKS; ++c)
        if (first + c * 32 < ncols) tma_store_2d(tmC, stage + c * STAGE_BUF_BYTES, first + c * 32, row0);
      tma_store_commit();
    }
  } else {
    __syncwarp();
    const Rows out = rows_of(p.C, p.ldc, p.M, ncols);
    for (int c = 0; c < BLOCKS; ++c) move_block<32, true>(out, stage + c * STAGE_BUF_BYTES, lane, row0, first + c * 32);
    __syncwarp();                                  // the buffers are rewritten by the next tile
  }
}

__device__ __forceinline__ void report_timeout(int32_t* status, int what) {
  if (status) { atomicCAS(status, 0, HB_ERR_TIMEOUT); status[1] = HB_KTAG_SCALED; status[2] = what; }
}

// Arrive on / wait for a barrier when the data it stands for crossed between CTAs of the cluster.
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t bar_cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_wait_acquire_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < HB_SPIN_LIMIT; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}\n"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 1023u) == 1023u && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_v4(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Sixteen finished sums of row `row0 + lane` from column col0 on -> C, by way of the warp's staging buffer
// (a tile that is split is one of few, and its output small: no TMA).
template <int EPI>
__device__ __forceinline__ void put16(const TileParams& p, uint32_t stage, int lane, int row0, int col0, float (&f)[16]) {
  constexpr bool swiglu = EPI == HB_EPI_SWIGLU;
  __syncwarp();                                    // the buffer may still be read for the last piece
  if constexpr (swiglu) {                          // columns interleave (gate, up): eight outputs
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = silu(f[2 * j]) * f[2 * j + 1];
  }
  if constexpr (EPI == HB_EPI_GELU) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) gelu2(f[j], f[j + 1]);
  }
  const int first = swiglu ? col0 >> 1 : col0, ncols = swiglu ? p.N >> 1 : p.N;
  if constexpr (EPI == HB_EPI_RESIDUAL) {
    move_block<16, false>(rows_of(p.R, p.ldr, p.M, p.N), stage, lane, row0, first);
    __syncwarp();
    add_row<16>(stage, lane, f);
  }
  put_row<16>(stage, lane, f);
  __syncwarp();
  move_block<16, true>(rows_of(p.C, p.ldc, p.M, swiglu ? min(ncols, first + 8) : ncols), stage, lane, row0, first);
}

template <int KIND, int BN, int STAGES, int EPI>
__device__ __forceinline__ void scaled_tile_body(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmC,
                                                 const TileParams& p) {
  using L = TileLayout<KIND, BN, STAGES>;
  constexpr bool PAIR = KIND == TILE_PAIR, SPLIT = KIND == TILE_SPLIT;
  constexpr int GROUP = PAIR ? 2 : 1;             // CTAs that one MMA spans
  constexpr int HALF = BN / 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sA = smem_base + L::OFF_A;
  const uint32_t sB = smem_base + L::OFF_B;
  const uint32_t bar_full = smem_base + L::OFF_BAR;
  const uint32_t bar_empty = bar_full + STAGES * 8;
  const uint32_t bar_tfull = bar_empty + STAGES * 8;
  const uint32_t bar_tempty = bar_tfull + L::SLOTS * 8;
  const uint32_t bar_xready = bar_tempty + L::SLOTS * 8;
  const uint32_t bar_xfull = bar_xready + EPI_WARPS * 8;
  volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem + L::OFF_TMEM_PTR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_ABORT);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;
  // CTA, pair or cluster; a split tile has a cluster of its own, whose CTAs take a contiguous share of
  // the k-blocks each (never none: there are at least as many)
  const int together = SPLIT ? p.split : GROUP;
  const int unit = blockIdx.x / together;
  const int num_units = gridDim.x / together;
  const int part = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  const int kb_begin = SPLIT ? static_cast<int>(static_cast<int64_t>(p.num_kb) * part / p.split) : 0;
  const int kb_end = SPLIT ? static_cast<int>(static_cast<int64_t>(p.num_kb) * (part + 1) / p.split) : p.num_kb;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + s * 8, GROUP);
      mbar_init(bar_empty + s * 8, 1);
    }
    for (int a = 0; a < L::SLOTS; ++a) {
      mbar_init(bar_tfull + a * 8, 1);
      mbar_init(bar_tempty + a * 8, EPI_WARPS * GROUP);
    }
    if constexpr (SPLIT)
      for (int w = 0; w < EPI_WARPS; ++w) {
        mbar_init(bar_xready + w * 8, p.split);
        mbar_init(bar_xfull + w * 8, p.split);
      }
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc<GROUP>(smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)), L::TMEM_COLS);
    tmem_relinquish<GROUP>();
  }
  tc_fence_before();
  if constexpr (KIND != TILE_ONE) cluster_sync(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr_smem;
  grid_dependency_wait();
  grid_launch_dependents();

  const int num_tiles = p.tiles_m * p.tiles_n;
  if (warp < EPI_WARP0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
    if (warp == 0) {
      // ---------------------------------------------------------- TMA producer
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = unit; tile < num_tiles && ok; tile += num_units) {
        int tm, tn;
        tile_coords(tile, p, tm, tn);
        const int m0 = tm * L::BM + rank * 128, n0 = tn * BN + rank * L::B_ROWS;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          if (!mbar_wait(bar_empty + s * 8, phase ^ 1, abort_flag)) { ok = false; break; }
          if (elect_one()) {
            if constexpr (PAIR) {
              const uint32_t full_leader = mapa(bar_full + s * 8, 0);
              if (rank == 0) mbar_arrive_expect_tx(bar_full + s * 8, L::A_BYTES + L::B_BYTES);
              else mbar_arrive_expect_tx_cluster(full_leader, L::A_BYTES + L::B_BYTES);
              tma_load_2d_pair(sA + s * L::A_BYTES, &tmA, full_leader, kb * KB, m0);
              tma_load_2d_pair(sB + s * L::B_BYTES, &tmB, full_leader, kb * KB, n0);
            } else {
              mbar_arrive_expect_tx(bar_full + s * 8, L::A_BYTES + L::B_BYTES);
              tma_load_2d(sA + s * L::A_BYTES, &tmA, bar_full + s * 8, kb * KB, m0);
              tma_load_2d(sB + s * L::B_BYTES, &tmB, bar_full + s * 8, kb * KB, n0);
            }
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; phase ^= 1; }
        }
      }
      if (!ok && lane == 0) report_timeout(p.status, 1);
    } else if (warp == 1 && rank == 0) {
      // ---------------------------------------------------------- MMA issuer (of a pair: the leader)
      constexpr uint32_t idesc = umma_idesc_e4m3(L::BM, BN);
      const uint32_t a_lo = desc_lo(sA), b_lo = desc_lo(sB);
      int s = 0, slot = 0;
      uint32_t phase = 0, slot_phase = 0;
      bool ok = true;
      for (int tile = unit; tile < num_tiles && ok; tile += num_units) {
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          // the data first: a slot is what comes late, and each wait costs about a hundred clocks
          if (!mbar_wait_spin(bar_full + s * 8, phase, abort_flag) || !mbar_wait_spin(bar_tempty + slot * 8, slot_phase ^ 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            umma_kblock<GROUP>(tmem_base + slot * BN, a_lo + s * (L::A_BYTES >> 4), b_lo + s * (L::B_BYTES >> 4), idesc);
            if constexpr (PAIR) {
              umma_commit_pair_mcast(bar_tfull + slot * 8, 3);
              umma_commit_pair_mcast(bar_empty + s * 8, 3);
            } else {
              umma_commit<1>(bar_tfull + slot * 8);
              umma_commit<1>(bar_empty + s * 8);
            }
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; phase ^= 1; }
          if (++slot == L::SLOTS) { slot = 0; slot_phase ^= 1; }
        }
      }
      if (!ok && lane == 0) report_timeout(p.status, 2);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
    // ------------------------------------------------------------ sums (warps 4..11)
    const int q = warp & 3;                          // tensor-memory lanes this warp may read
    const int h = (warp - EPI_WARP0) >> 2;                   // half of the tile's columns
    const uint32_t stage_mine = smem_base + L::OFF_STAGE + (warp - EPI_WARP0) * STAGE_BUFS * STAGE_BUF_BYTES;
    const uint32_t t_mine = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + h * HALF;
    uint32_t tempty = bar_tempty;
    if constexpr (PAIR) tempty = mapa(bar_tempty, 0);
    int slot = 0;
    uint32_t slot_phase = 0;
    bool ok = true;
    // scales of this thread's row and columns in `tile`; rows and blocks past the edge repeat the last
    // one: their sums are zero and are not stored
    const float *sa = nullptr, *sb = nullptr;
    float fa = 0.f, fb = 0.f;
    auto first_scales = [&](int tile) {
      int tm, tn;
      tile_coords(tile, p, tm, tn);
      sa = p.sa + min(tm * L::BM + rank * 128 + q * 32 + lane, p.M - 1) * p.sa_m;
      sb = p.sb + min((tn * BN + h * HALF) / KB, p.nblocks - 1) * p.sb_n;
      fa = sa[kb_begin * p.sa_k];
      fb = sb[kb_begin * p.sb_k];
    };
    if (unit < num_tiles) first_scales(unit);
    for (int tile = unit; tile < num_tiles && ok; tile += num_units) {
      uint64_t acc[HALF / 2];
#pragma unroll
      for (int j = 0; j < HALF / 2; ++j) acc[j] = 0;
      for (int kb = kb_begin; kb < kb_end; ++kb) {
        const uint64_t f = pack2(fa * fb, fa * fb);
        if (kb + 1 < kb_end) {                       // the next block's scales arrive under this block's sums
          fa = sa[(kb + 1) * p.sa_k];
          fb = sb[(kb + 1) * p.sb_k];
        }
        if (!mbar_wait(bar_tfull + slot * 8, slot_phase, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t t = t_mine + slot * BN;
        // sixty-four columns at a time: the other warp of the scheduler adds while this one's are on their way
        uint32_t v[64];
#pragma unroll
        for (int c = 0; c < HALF / 64; ++c) {
          tmem_ld_32x64(t + c * 64, v);
          tmem_wait_ld();
          if (c + 1 == HALF / 64) {                  // everything is in registers: the slot is free
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) mbar_arrive_cluster(tempty + slot * 8);
              else mbar_arrive(tempty + slot * 8);
            }
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) fma2(acc[c * 32 + j], v[2 * j], v[2 * j + 1], f);
        }
        if (++slot == L::SLOTS) { slot = 0; slot_phase ^= 1; }
      }
      int tm, tn;
      tile_coords(tile, p, tm, tn);
      const int row0 = tm * L::BM + rank * 128 + q * 32, col0 = tn * BN + h * HALF;
      if (tile + num_units < num_tiles) first_scales(tile + num_units);   // arrive under this tile's output
      if constexpr (SPLIT) {
            // The CTAs add their sums up: a warp's columns go, sixteen at a time, to the CTA that writes them,
        // into its ring -- which is free once its own last k-block is done (xready) -- and are added
        // there in k order.  Warp w of a CTA deals with warps w alone.
        static_assert(HALF == 64, "four pieces of sixteen columns");
        constexpr int PIECE = 32 * 16 * 4;             // bytes of 32 rows x 16 columns
        const int w = warp - EPI_WARP0, S = p.split;
        auto first_piece = [&](int c) { return 4 * c / S; };
        if (!ok) break;
        if (lane < S) mbar_arrive_release_cluster(mapa(bar_xready + w * 8, lane));
        ok = mbar_wait_acquire_cluster(bar_xready + w * 8, 0, abort_flag);
        if (!ok) break;
        int to = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          while (c >= first_piece(to + 1)) ++to;
          const uint32_t dst = mapa(smem_base + (((c - first_piece(to)) * S + part) * EPI_WARPS + w) * PIECE + lane * 16, to);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 x = unpack2(acc[c * 8 + 2 * j]), y = unpack2(acc[c * 8 + 2 * j + 1]);
            st_cluster_v4(dst + j * 512, make_float4(x.x, x.y, y.x, y.y));
          }
        }
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        __syncwarp();
        if (lane < S) mbar_arrive_release_cluster(mapa(bar_xfull + w * 8, lane));
        ok = mbar_wait_acquire_cluster(bar_xfull + w * 8, 0, abort_flag);
        if (!ok) break;
        for (int c = first_piece(part); c < first_piece(part + 1); ++c) {
          float f[16] = {};
          for (int from = 0; from < S; ++from) {
            const uint8_t* src = smem + (((c - first_piece(part)) * S + from) * EPI_WARPS + w) * PIECE + lane * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 v = *reinterpret_cast<const float4*>(src + j * 512);
              f[4 * j] += v.x; f[4 * j + 1] += v.y; f[4 * j + 2] += v.z; f[4 * j + 3] += v.w;
            }
          }
          put16<EPI>(p, stage_mine, lane, row0, col0 + c * 16, f);
        }
      } else {
        if (ok) write_half<EPI, HALF>(p, &tmC, stage_mine, lane, row0, col0, acc);
      }
    }
    if (p.tma_store && lane == 0) tma_store_wait<0>();   // the staged blocks have left shared memory and landed
    if (!ok && lane == 0) report_timeout(p.status, 3);
  }

  // ---------------------------------------------------------------- teardown
  // of a pair, neither CTA may leave while its partner can still signal its barriers or read its
  // shared memory
  tc_fence_before();
  if constexpr (KIND != TILE_ONE) cluster_sync(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<GROUP>(tmem_base, L::TMEM_COLS);
  }
}

template <int BN, int STAGES, int EPI>
__global__ void __launch_bounds__(TILE_THREADS, 1)
hb_matmul_scaled_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ CUtensorMap tmC, const __grid_constant__ TileParams p) {
  scaled_tile_body<TILE_ONE, BN, STAGES, EPI>(tmA, tmB, tmC, p);
}
template <int BN, int STAGES, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TILE_THREADS, 1)
hb_matmul_scaled_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                             const __grid_constant__ CUtensorMap tmC, const __grid_constant__ TileParams p) {
  scaled_tile_body<TILE_PAIR, BN, STAGES, EPI>(tmA, tmB, tmC, p);
}
template <int BN, int STAGES, int EPI>
__global__ void __launch_bounds__(TILE_THREADS, 1)
hb_matmul_scaled_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                              const __grid_constant__ CUtensorMap tmC, const __grid_constant__ TileParams p) {
  scaled_tile_body<TILE_SPLIT, BN, STAGES, EPI>(tmA, tmB, tmC, p);
}

hb_status make_maps(hb_ctx* ctx, const ScaledArgs& g, int b_rows, CUtensorMap* tmA, CUtensorMap* tmB, CUtensorMap* tmC, int* tma_store) {
  uint64_t dims[2] = {(uint64_t)g.K, (uint64_t)g.M}, pitch[1] = {(uint64_t)g.lda};
  uint32_t box[2] = {KB, 128};
  hb_status st = hb_make_tensor_map(ctx, tmA, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, g.A, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != HB_OK) return st;
  dims[1] = (uint64_t)g.N; pitch[0] = (uint64_t)g.ldb; box[1] = (uint32_t)b_rows;
  if ((st = hb_make_tensor_map(ctx, tmB, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, g.B, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B)) != HB_OK) return st;
  *tmC = *tmA;
  const bool one_row = g.M == 1;                 // its pitch is never used
  const int64_t cols = g.epilogue == HB_EPI_SWIGLU ? g.N / 2 : g.N;
  // TMA clips a store at whole 16-byte pieces: a row that ends inside one would be written to the
  // piece's end (measured: a single-column store put seven zeros behind it)
  *tma_store = (cols & 7) == 0 && (one_row || (g.ldc & 7) == 0) && (reinterpret_cast<uintptr_t>(g.C) & 15) == 0;
  if (*tma_store) {
    dims[0] = (uint64_t)cols; dims[1] = (uint64_t)g.M; pitch[0] = (uint64_t)(one_row ? cols : g.ldc) * 2;
    box[0] = 32; box[1] = 32;
    st = hb_make_tensor_map(ctx, tmC, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g.C, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_64B);
  }
  return st;
}

template <int KIND, int BN, int STAGES, int EPI>
hb_status launch_tile_epi(hb_ctx* ctx, const ScaledArgs& g, int split) {
  using L = TileLayout<KIND, BN, STAGES>;
  constexpr bool PAIR = L::PAIR;
  void (*kern)(const CUtensorMap, const CUtensorMap, const CUtensorMap, const TileParams);
  if constexpr (PAIR) kern = hb_matmul_scaled_pair_kernel<BN, STAGES, EPI>;
  else if constexpr (KIND == TILE_SPLIT) kern = hb_matmul_scaled_split_kernel<BN, STAGES, EPI>;
  else kern = hb_matmul_scaled_kernel<BN, STAGES, EPI>;
  // persistent CTAs (or pairs) that can run at once; of pairs the occupancy query knows, because not
  // every SM has a neighbour to pair with
  static std::atomic<int> resident[64];
  if (!resident[ctx->device & 63].load(std::memory_order_acquire)) {
    HB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN_BYTES));
    int n = ctx->sm_count;
    if constexpr (PAIR) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(ctx->sm_count & ~1u);
      cfg.blockDim = dim3(TILE_THREADS);
      cfg.dynamicSmemBytes = L::DYN_BYTES;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) { cudaGetLastError(); n = ctx->sm_count / 2 - 8; }
    }
    resident[ctx->device & 63] = n;
  }
  CUtensorMap tmA, tmB, tmC;
  TileParams p;
  memset(&p, 0, sizeof(p));
  const hb_status st = make_maps(ctx, g, L::B_ROWS, &tmA, &tmB, &tmC, &p.tma_store);
  if (st != HB_OK) return st;
  p.sa = g.sa; p.sb = g.sb; p.C = g.C; p.R = g.R;
  p.ldc = g.ldc; p.ldr = g.ldr;
  p.sa_m = g.sa_m; p.sa_k = g.sa_k; p.sb_n = g.sb_n; p.sb_k = g.sb_k;
  p.M = (int)g.M; p.N = (int)g.N;
  p.num_kb = (int)((g.K + KB - 1) / KB);
  p.nblocks = (int)((g.N + KB - 1) / KB);
  const int64_t tiles_m = (g.M + L::BM - 1) / L::BM, tiles_n = (g.N + BN - 1) / BN;
  if (tiles_m * tiles_n > INT32_MAX / 2) return hb_fail(ctx, HB_ERR_UNSUPPORTED, "matmul_scaled: problem too large");
  p.tiles_m = (int)tiles_m; p.tiles_n = (int)tiles_n;
  p.raster_group = 8;
  p.status = ctx->d_status;
  const int tiles = p.tiles_m * p.tiles_n, most = resident[ctx->device & 63];
  p.split = split;
  cudaError_t e;
  if constexpr (KIND == TILE_SPLIT) {              // one tile per cluster, not persistent: the ring ends as the exchange
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles * split);
    cfg.blockDim = dim3(TILE_THREADS);
    cfg.dynamicSmemBytes = L::DYN_BYTES;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmC, p);
  } else {
    const unsigned ctas = (PAIR ? 2 : 1) * (unsigned)(tiles < most ? tiles : most);
    e = hb_launch_dependent(kern, dim3(ctas), dim3(TILE_THREADS), L::DYN_BYTES, ctx->stream, tmA, tmB, tmC, p);
  }
  if (e != cudaSuccess) { cudaGetLastError(); return hb_check_cuda(ctx, e, "matmul_scaled launch"); }
  ctx->launches++;
  return HB_OK;
}

// ------------------------------------------------------------------------------------
// Few rows (M <= 64): bound by reading B once.  The operands change places -- a slab of 128 rows of B
// is the M side of the MMA, the rows of A, padded to 16, 32 or 64 by TMA's zero fill, its N side.
// A CTA, or a cluster of S, owns whole slabs; a cluster cuts their (slab, k-block) units into S contiguous
// ranges of the same length, one per CTA, so that its SMs stream the same number of bytes.  A finished
// k-block goes to one of eight tensor-memory slots; a thread holds one column of C (one row of the slab) for
// all rows of A, and the factors a_scale * b_scale of a k-block come through shared memory from a warp
// that runs ahead.  Where a range starts inside a slab, its sums go to the CTA that started the slab, over
// distributed shared memory, as the first thing that a CTA finishes; the starter comes to that slab
// last, finds them there and adds them in k order: the same bits every run, nothing waits in
// practice, and there is no scratch and no counter in global memory that launches could share.
// With HB_MATMUL_WEIGHTS_B a CTA fills its ring with B before the kernel in front has finished
// (programmatic dependent launch); what depends on that kernel comes after the wait.
// 16 x 28672 x 4096 22.6 us, 16 x 128256 x 4096 79.1 us (6.6 TB/s, as fast as a copy), 1 x 6144 x 4096 8.0 us,
// 64 x 28672 x 4096 30.4 us: the stream itself runs at 6 to 7 TB/s, and about five microseconds of a
// launch are not it (start, the first bytes, the last sums; a second CTA on the SM would cover them, but
// of kernels that allocate tensor memory the occupancy query admits one).  A unit's MMAs take 0.25 us, as
// long for a lower slab.  Measured and not taken: equal units for all CTAs and partial sums in global memory
// (28 us for 16 x 28672 x 4096); slabs of as many rows as give every CTA the same (no gain, above 10 us for
// 1 x 6144 x 4096); A loaded by a warp of its own, and scales fetched further ahead (no change).
// ------------------------------------------------------------------------------------
constexpr int FEW_MAX_M = 64;
constexpr int FEW_THREADS = 224;                 // TMA, MMA, four warps of sums, factors
constexpr int FEW_SLOTS = 8;
constexpr int SLAB = 128;

struct FewParams {
  const float* sa;
  const float* sb;
  __nv_bfloat16* C;
  const __nv_bfloat16* R;
  int64_t ldc, ldr, sa_m, sa_k, sb_n, sb_k;
  int M, N, num_kb, slabs;
  int cluster;                 // CTAs per cluster
  int epilogue, b_is_weights;
  int32_t* status;
};

template <int MP>
struct FewLayout {
  static constexpr int A_BYTES = MP * KB, B_BYTES = SLAB * KB;
  // Units that share a barrier.  Two for few columns: their MMAs run in turn (below), and the sums wait once
  // for both.  With 64 it is slower (64 x 28672 x 4096 33.5 us, one by one 31.5).
  static constexpr int GROUP = MP <= 32 ? 2 : 1, GROUPS = FEW_SLOTS / GROUP;
  static constexpr int MAX_CLUSTER = MP <= 16 ? 6 : 4;                    // the sums received have to fit beside the ring
  static constexpr uint32_t TMEM_COLS = FEW_SLOTS * MP;                   // 128, 256 or 512
  static constexpr int F_BYTES = FEW_SLOTS * MP * 4;                      // factors: [slot][MP] fp32
  static constexpr int X_BYTES = (MAX_CLUSTER - 1) * MP * SLAB * 4;   // sums received: [sender][row of A][128] fp32
  static constexpr int W_BYTES = 16 * SLAB * 4;                           // sixteen rows on their way out
  static constexpr int STAGES = (227 * 1024 - 4096 - F_BYTES - X_BYTES - W_BYTES) / (A_BYTES + B_BYTES);
  static constexpr int OFF_B = 0;
  static constexpr int OFF_A = OFF_B + STAGES * B_BYTES;
  static constexpr int OFF_F = OFF_A + STAGES * A_BYTES;
  static constexpr int OFF_X = OFF_F + F_BYTES;
  static constexpr int OFF_W = OFF_X + X_BYTES;
  static constexpr int OFF_BAR = OFF_W + W_BYTES;      // full, empty per stage; tfull, tempty per group; xfull per warp
  static constexpr int OFF_TMEM_PTR = OFF_BAR + (2 * STAGES + 2 * GROUPS + 4) * 8;
  static constexpr int OFF_ABORT = OFF_TMEM_PTR + 4;
  static constexpr int DYN_BYTES = OFF_ABORT + 4 + 1024;
  static_assert(DYN_BYTES <= 227 * 1024 && STAGES >= 4, "ring does not fit shared memory");
};

template <int MP>
__global__ void __launch_bounds__(FEW_THREADS, 1)
hb_matmul_scaled_few_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                            const __grid_constant__ FewParams p) {
  using L = FewLayout<MP>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sB = smem_base + L::OFF_B, sA = smem_base + L::OFF_A;
  float* factors = reinterpret_cast<float*>(smem + L::OFF_F);
  const uint32_t bar_full = smem_base + L::OFF_BAR;
  const uint32_t bar_empty = bar_full + L::STAGES * 8;
  const uint32_t bar_tfull = bar_empty + L::STAGES * 8;
  const uint32_t bar_tempty = bar_tfull + L::GROUPS * 8;
  const uint32_t bar_xfull = bar_tempty + L::GROUPS * 8;
  volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem + L::OFF_TMEM_PTR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_ABORT);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = p.cluster;
  const int rank = static_cast<int>(cluster_ctarank());
  // the cluster's slabs are first_slab, first_slab + step, ...; unit u of the cluster is k-block u % num_kb
  // of its slab number u / num_kb; this CTA has the units [u_begin, u_end), never none: a cluster has a
  // slab, and S is at most num_kb
  const int first_slab = blockIdx.x / S, step = gridDim.x / S;
  const int64_t all = static_cast<int64_t>((p.slabs - first_slab + step - 1) / step) * p.num_kb;
  auto begin_of = [&](int c) { return all * c / S; };
  auto owner_of = [&](int64_t u) { return static_cast<int>(((u + 1) * S - 1) / all); };   // CTA of unit u
  const int64_t u_begin = begin_of(rank), u_end = begin_of(rank + 1);
  const int64_t units = u_end - u_begin;
  const int slab0 = first_slab + static_cast<int>(u_begin / p.num_kb) * step, kb0 = static_cast<int>(u_begin % p.num_kb);
  // CTAs that send this one their part of the slab that it starts last
  const int64_t last_start = (u_end - 1) / p.num_kb * p.num_kb;
  const int senders = last_start >= u_begin ? owner_of(last_start + p.num_kb - 1) - rank : 0;

  // units that fill the ring, and the loader warp's next unit
  const int fill = static_cast<int>(min(units, static_cast<int64_t>(L::STAGES)));
  int load_slab = slab0, load_kb = kb0;
  auto next_load = [&] {
    if (++load_kb == p.num_kb) { load_kb = 0; load_slab += step; }
  };
  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&tmB);
      tma_prefetch_desc(&tmA);
      *abort_flag = 0;
      for (int s = 0; s < L::STAGES; ++s) {
        mbar_init(bar_full + s * 8, 1);
        mbar_init(bar_empty + s * 8, 1);
      }
      for (int a = 0; a < L::GROUPS; ++a) {
        mbar_init(bar_tfull + a * 8, 2);         // the sums of the MMA, and the factors
        mbar_init(bar_tempty + a * 8, 4);
      }
      for (int w = 0; w < 4; ++w) mbar_init(bar_xfull + w * 8, max(senders, 1));
      mbar_fence_init();
      fence_proxy_async_smem();
    }
    __syncwarp();
    cluster_arrive();           // the partners may use these barriers
    // ring fill: B at once -- it needs neither the cluster nor tensor memory nor, being weights, the kernel in
    // front; A comes from the MMA warp, so that it does not queue behind all of B.  (After the cluster's barrier
    // and with A behind it 1 x 4096 x 4096 took 7.05 us, so it takes 6.73.)
    for (int i = 0; i < fill; ++i) {
      if (elect_one()) {
        mbar_arrive_expect_tx(bar_full + i * 8, L::A_BYTES + L::B_BYTES);
        tma_load_2d(sB + i * L::B_BYTES, &tmB, bar_full + i * 8, load_kb * KB, load_slab * SLAB);
      }
      next_load();
    }
    __syncwarp();
    cluster_wait();
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)), L::TMEM_COLS);
    tmem_relinquish<1>();
  }
  if (warp != 0) {
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
  }
  const uint32_t tmem_base = *tmem_ptr_smem;
  grid_launch_dependents();     // the next kernel on the stream may begin its own prologue

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    bool ok = true;
    grid_dependency_wait();
    int s = fill == L::STAGES ? 0 : fill;
    uint32_t phase = fill == L::STAGES ? 1 : 0;
    for (int64_t u = fill; u < units; ++u) {
      if (!mbar_wait(bar_empty + s * 8, phase ^ 1, abort_flag)) { ok = false; break; }
      if (elect_one()) {
        mbar_arrive_expect_tx(bar_full + s * 8, L::A_BYTES + L::B_BYTES);
        tma_load_2d(sB + s * L::B_BYTES, &tmB, bar_full + s * 8, load_kb * KB, load_slab * SLAB);
        tma_load_2d(sA + s * L::A_BYTES, &tmA, bar_full + s * 8, load_kb * KB, 0);
      }
      __syncwarp();
      next_load();
      if (++s == L::STAGES) { s = 0; phase ^= 1; }
    }
    if (!ok && lane == 0) report_timeout(p.status, 11);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    grid_dependency_wait();
    for (int i = 0, kb = kb0; i < fill; ++i) {
      if (elect_one()) tma_load_2d(sA + i * L::A_BYTES, &tmA, bar_full + i * 8, kb * KB, 0);
      if (++kb == p.num_kb) kb = 0;
    }
    __syncwarp();
    constexpr uint32_t idesc = umma_idesc_e4m3(SLAB, MP);
    const uint32_t a_lo = desc_lo(sA), b_lo = desc_lo(sB);
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = 0; u < units; u += L::GROUP) {
      const int slot = u % FEW_SLOTS, group = slot / L::GROUP;
      const bool both = L::GROUP == 2 && u + 1 < units;
      const int s2 = s + 1 == L::STAGES ? 0 : s + 1;         // the next stage
      const uint32_t phase2 = s2 ? phase : phase ^ 1;
      if (!mbar_wait(bar_tempty + group * 8, (u / FEW_SLOTS & 1) ^ 1, abort_flag) || !mbar_wait(bar_full + s * 8, phase, abort_flag) ||
          (both && !mbar_wait(bar_full + s2 * 8, phase2, abort_flag))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + slot * MP, a0 = b_lo + s * (L::B_BYTES >> 4), b0 = a_lo + s * (L::A_BYTES >> 4);
      const uint32_t a1 = b_lo + s2 * (L::B_BYTES >> 4), b1 = a_lo + s2 * (L::A_BYTES >> 4);
      if (elect_one()) {
        if (both) {
          umma_two(d, a0, b0, d + MP, a1, b1, idesc);
          umma_commit<1>(bar_empty + s * 8);
          umma_commit<1>(bar_empty + s2 * 8);
        } else {
          umma_kblock<1>(d, a0, b0, idesc);
          umma_commit<1>(bar_empty + s * 8);
        }
        umma_commit<1>(bar_tfull + group * 8);
      }
      __syncwarp();
      s = s2;
      phase = phase2;
      if (both) {
        if (++s == L::STAGES) { s = 0; phase ^= 1; }
      }
    }
    if (!ok && lane == 0) report_timeout(p.status, 12);
  } else if (warp == 6) {
    // ---------------------------------------------------------------- factors a_scale * b_scale
    // Eight units' scales are fetched at a time (units past the end repeat the last one), the next
    // eight under the hand-over of these; the scales of a weight matrix do not wait for the kernel
    // in front.
    constexpr int PER = (MP + 31) / 32, AHEAD = FEW_SLOTS;
    float fa[AHEAD][PER], fb[AHEAD];
    int slab = slab0, kb = kb0;                  // of the next unit to fetch
    int64_t left = units;
    auto next = [&] {
      if (--left <= 0) return;
      if (++kb == p.num_kb) { kb = 0; slab += step; }
    };
    auto fetch_a = [&](float (&x)[PER], int at) {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = p.sa[min(lane + 32 * i, p.M - 1) * p.sa_m + at * p.sa_k];
    };
    int first_kb[AHEAD];
    if (!p.b_is_weights) grid_dependency_wait();
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      fb[j] = p.sb[slab * p.sb_n + kb * p.sb_k];
      first_kb[j] = kb;
      next();
    }
    grid_dependency_wait();
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) fetch_a(fa[j], first_kb[j]);
    uint32_t slot_phase = 0;
    bool ok = true;
    for (int u = 0; u < units && ok; u += AHEAD, slot_phase ^= 1) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (u + j < units && ok) {
          if (j % L::GROUP == 0) ok = mbar_wait(bar_tempty + j / L::GROUP * 8, slot_phase ^ 1, abort_flag);
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < MP) factors[j * MP + lane + 32 * i] = fa[j][i] * fb[j];
          if (j % L::GROUP == L::GROUP - 1 || u + j + 1 == units) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_tfull + j / L::GROUP * 8);
          }
          fb[j] = p.sb[slab * p.sb_n + kb * p.sb_k];
          fetch_a(fa[j], kb);
          next();
        }
      }
    }
    if (!ok && lane == 0) report_timeout(p.status, 14);
  } else {
    // ---------------------------------------------------------------- sums (warps 2..5)
    const int q = warp & 3;
    const int r = q * 32 + lane;                 // row of the slab = output column slab * 128 + r
    const uint32_t t_mine = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const uint32_t x_mine = smem_base + L::OFF_X + r * 4;
    const float* x_local = reinterpret_cast<const float*>(smem + L::OFF_X) + r;
    float* w_local = reinterpret_cast<float*>(smem + L::OFF_W) + r;
    bool ok = true;
    grid_dependency_wait();                      // C may still be in use by the kernel in front
    int slab = slab0, kb = kb0;
    for (int64_t u = u_begin; u < u_end; slab += step, kb = 0) {
      const int nkb = static_cast<int>(min(u_end - u, static_cast<int64_t>(p.num_kb - kb)));
      uint64_t acc[MP / 2];
#pragma unroll
      for (int i = 0; i < MP / 2; ++i) acc[i] = 0;
      // a group's two slots at once where both belong to this slab
      for (int i = 0; i < nkb;) {
        const int at = static_cast<int>(u - u_begin) + i, slot = at % FEW_SLOTS;
        const bool both = L::GROUP == 2 && slot % 2 == 0 && i + 1 < nkb;
        ok = mbar_wait(bar_tfull + slot / L::GROUP * 8, at / FEW_SLOTS & 1, abort_flag);
        if (!ok) break;
        tc_fence_after();
        auto add = [&](const uint32_t (&v)[MP / 16][16], int which) {
          const float4* f4 = reinterpret_cast<const float4*>(factors + which * MP);
#pragma unroll
          for (int c = 0; c < MP / 4; ++c) {
            const float4 f = f4[c];
            const uint32_t* t = &v[c / 4][c % 4 * 4];
            fma2(acc[2 * c], t[0], t[1], pack2(f.x, f.y));
            fma2(acc[2 * c + 1], t[2], t[3], pack2(f.z, f.w));
          }
        };
        uint32_t v[MP / 16][16];
#pragma unroll
        for (int c = 0; c < MP / 16; ++c) tmem_ld_32x16(t_mine + slot * MP + c * 16, v[c]);
        if (both) {
          uint32_t w[MP / 16][16];
#pragma unroll
          for (int c = 0; c < MP / 16; ++c) tmem_ld_32x16(t_mine + (slot + 1) * MP + c * 16, w[c]);
          tmem_wait_ld();
          add(v, slot);
          add(w, slot + 1);
        } else {
          tmem_wait_ld();
          add(v, slot);
        }
        i += both ? 2 : 1;
        if (both || slot % L::GROUP == L::GROUP - 1) {   // the group's sums and factors are in registers
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_tempty + slot / L::GROUP * 8);
        }
      }
      if (!ok) break;
      if (kb > 0) {
        // the slab was started by another CTA: send the sums there; warp q hears from warps q alone
        const int starter = owner_of(u - kb);
        const uint32_t dst = mapa(x_mine + (rank - starter - 1) * (MP * SLAB * 4), starter);
#pragma unroll
        for (int m = 0; m < MP; ++m) {
          const float2 two = unpack2(acc[m / 2]);
          if (m < p.M) st_cluster_f32(dst + m * (SLAB * 4), m & 1 ? two.y : two.x);
        }
        asm volatile("fence.acq_rel.cluster;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_release_cluster(mapa(bar_xfull + q * 8, starter));
        u += nkb;
        continue;
      }
      if (nkb < p.num_kb) {
        ok = mbar_wait_acquire_cluster(bar_xfull + q * 8, 0, abort_flag);
        if (!ok) break;
      }
      u += nkb;
      const int from = nkb < p.num_kb ? senders : 0;
      const int n = slab * SLAB + r;
      // sixteen rows at a time through shared memory (each thread its own column), so that the
      // epilogue is a short loop: unrolled over the accumulators it would not fit the instruction cache
#pragma unroll
      for (int c16 = 0; c16 < MP; c16 += 16) {
        if (c16 >= p.M) break;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 two = unpack2(acc[(c16 + i) / 2]);
          w_local[i * SLAB] = i & 1 ? two.y : two.x;
        }
        for (int i = 0; i < 16 && c16 + i < p.M; i += 4) {
          float v[4];                             // rows past the last are read (from this buffer) and not used
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = w_local[(i + j) * SLAB];
          for (int c = 0; c < from; ++c)          // in k order
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += x_local[(c * MP + c16 + i + j) * SLAB];
          const int rows = min(4, p.M - c16 - i);
          if (p.epilogue == HB_EPI_SWIGLU) {      // columns interleave (gate, up): two neighbouring lanes
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = silu(v[j]) * __shfl_down_sync(0xffffffffu, v[j], 1);
          } else if (p.epilogue == HB_EPI_GELU) {
#pragma unroll
            for (int j = 0; j < 4; j += 2) gelu2(v[j], v[j + 1]);
          } else if (p.epilogue == HB_EPI_RESIDUAL) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < rows && n < p.N) v[j] += __bfloat162float(p.R[(c16 + i + j) * p.ldr + n]);
          }
          const bool mine = n < p.N && !(p.epilogue == HB_EPI_SWIGLU && (r & 1));
          __nv_bfloat16* dst = p.C + (c16 + i) * p.ldc + (p.epilogue == HB_EPI_SWIGLU ? n >> 1 : n);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < rows && mine) dst[j * p.ldc] = __float2bfloat16_rn(v[j]);
        }
      }
    }
    if (!ok && lane == 0) report_timeout(p.status, 13);
  }

  // no CTA may leave while a partner can still write to its shared memory (leaving one by one was also slower
  // behind each other, 16 x 28672 x 4096 32.7 for 24.0 us: the next launch's clusters then find SMs in pieces)
  tc_fence_before();
  if (S > 1) cluster_sync(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, L::TMEM_COLS);
  }
}

template <int MP>
hb_status launch_few(hb_ctx* ctx, const ScaledArgs& g) {
  using L = FewLayout<MP>;
  auto kern = hb_matmul_scaled_few_kernel<MP>;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(FEW_THREADS);
  cfg.dynamicSmemBytes = L::DYN_BYTES;
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  // clusters of S CTAs that can run at once, one CTA per SM
  static std::atomic<int> resident[64][L::MAX_CLUSTER + 1];       // (that of one CTA is set last)
  std::atomic<int>* most = resident[ctx->device & 63];
  if (!most[1].load(std::memory_order_acquire)) {
    HB_CUDA(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::DYN_BYTES));
    for (int c = L::MAX_CLUSTER; c >= 1; --c) {
      attr[0].val.clusterDim.x = c;
      cfg.gridDim = dim3(ctx->sm_count / c * c);
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
      n = n < ctx->sm_count / c ? n : ctx->sm_count / c;
      most[c].store(c == 1 && n < 1 ? ctx->sm_count : n, std::memory_order_release);
    }
  }
  CUtensorMap tmA, tmB;
  uint64_t dims[2] = {(uint64_t)g.K, (uint64_t)g.M}, pitch[1] = {(uint64_t)g.lda};
  uint32_t box[2] = {KB, MP};
  hb_status st = hb_make_tensor_map(ctx, &tmA, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, g.A, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != HB_OK) return st;
  dims[1] = (uint64_t)g.N; pitch[0] = (uint64_t)g.ldb; box[1] = SLAB;
  if ((st = hb_make_tensor_map(ctx, &tmB, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, g.B, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B)) != HB_OK) return st;
  FewParams p;
  memset(&p, 0, sizeof(p));
  p.sa = g.sa; p.sb = g.sb; p.C = g.C; p.R = g.R;
  p.ldc = g.ldc; p.ldr = g.ldr;
  p.sa_m = g.sa_m; p.sa_k = g.sa_k; p.sb_n = g.sb_n; p.sb_k = g.sb_k;
  p.M = (int)g.M; p.N = (int)g.N;
  p.num_kb = (int)((g.K + KB - 1) / KB);
  p.slabs = (int)((g.N + SLAB - 1) / SLAB);
  p.epilogue = g.epilogue;
  p.b_is_weights = g.b_is_weights;
  p.status = ctx->d_status;
  // CTAs of a cluster, by the longer of two times in microseconds: the busiest CTA's units at the rate of their
  // MMAs, and the bytes at the rate of HBM, which takes about 120 CTAs.  Measured (M = 16, K = 4096; clusters of 1, 2, 3,
  // 4, 6):  2048 columns 10.8 / 7.9 / 7.1 / 6.3 / 6.8     6144: 11.0 / 9.1 / 10.6 / 9.1 / 9.2
  //   12288: 13.0 / 12.1 / 13.0 / 13.3 / 13.3   20480: 22.2 / 19.7 / 18.6 / 18.1 / 18.4   28672: 22.6 / 22.6 / 23.1 / 22.6 / 22.8
  //   4096, K = 14336: 32.1 / 19.1 / 16.0 / 14.6 / 15.1; the choice is 1.6 % off the best on average, 9 % at most
  const double unit = MP <= 32 ? 0.23 : 0.30, bytes = (double)(g.N + g.M) * g.K / 6.5e6;
  double best = 0;
  for (int c = 1; c <= L::MAX_CLUSTER && c <= p.num_kb; ++c) {
    const int at_once = most[c], clusters = p.slabs < at_once ? p.slabs : at_once;
    if (clusters < 1) continue;
    const double units = (double)((p.slabs + clusters - 1) / clusters) * p.num_kb / c, share = clusters * c / 120.0;
    const double stream = share < 1 ? bytes / share : bytes, cost = units * unit > stream ? units * unit : stream;
    if (p.cluster == 0 || cost < best) { best = cost; p.cluster = c; }
  }
  const int at_once = most[p.cluster], clusters = p.slabs < at_once ? p.slabs : at_once;
  attr[0].val.clusterDim.x = p.cluster;
  cfg.gridDim = dim3((unsigned)(clusters * p.cluster));
  cfg.numAttrs = g.b_is_weights ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tmA, tmB, p);
  if (e != cudaSuccess) { cudaGetLastError(); return hb_check_cuda(ctx, e, "matmul_scaled launch"); }
  ctx->launches++;
  return HB_OK;
}

template <int KIND, int BN, int STAGES>
hb_status launch_tile(hb_ctx* ctx, const ScaledArgs& g, int split = 1) {
  switch (g.epilogue) {
    case HB_EPI_GELU: return launch_tile_epi<KIND, BN, STAGES, HB_EPI_GELU>(ctx, g, split);
    case HB_EPI_SWIGLU: return launch_tile_epi<KIND, BN, STAGES, HB_EPI_SWIGLU>(ctx, g, split);
    case HB_EPI_RESIDUAL: return launch_tile_epi<KIND, BN, STAGES, HB_EPI_RESIDUAL>(ctx, g, split);
    default: return launch_tile_epi<KIND, BN, STAGES, HB_EPI_NONE>(ctx, g, split);
  }
}

hb_status launch(hb_ctx* ctx, const ScaledArgs& g) {
  if (g.M <= FEW_MAX_M)
    return g.M <= 16 ? launch_few<16>(ctx, g) : g.M <= 32 ? launch_few<32>(ctx, g) : launch_few<64>(ctx, g);
  // The form that takes the least time, in microseconds: a fixed part and a k-block's time per wave of
  // tiles.  Measured (K = 4096; 256 x 256 pair, 256 x 128 pair, 128 x 256, split 2, split 4):
  //   128 x 4096: 18.0 / 14.2 / 20.0 / 11.6 / 10.8      128 x 28672: 33.5 / 41.3 / 25.8 / 54 / 80
  //   512 x 4096: 17.4 / 13.7 / 19.6 / 25.8 / 43.9      4096 x 4096: 65 / 81 / 70 / - / -
  //   128 x 4096, K = 14336: 46.7 / 35.0 / 55.5 / 26.1 / 19.5
  const double kblocks = (double)((g.K + KB - 1) / KB);
  const auto waves = [&](int64_t bm, int64_t bn, int64_t at_once) {
    const int64_t tiles = (g.M + bm - 1) / bm * ((g.N + bn - 1) / bn);
    return (double)((tiles + at_once - 1) / at_once);
  };
  const double pair_wide = 5.5 + 0.42 * kblocks * waves(256, 256, ctx->sm_count / 2),
               pair_narrow = 3.6 + 0.30 * kblocks * waves(256, 128, ctx->sm_count / 2),
               one = 5.0 + 0.47 * kblocks * waves(128, 256, ctx->sm_count);
  int split = 0;
  double best = pair_wide < pair_narrow ? pair_wide : pair_narrow;
  if (one < best) best = one;
  for (int c = 2; c <= SPLIT_MAX && c <= kblocks; ++c) {
    // clusters of c find room on most of the SMs only (148 SMs: 74, 45, 33)
    const double t = 5.0 + 1.3 * c + 0.325 * ceil(kblocks / c) * waves(128, 128, ctx->sm_count * 9 / 10 / c);
    if (t < best) { best = t; split = c; }
  }
  if (split) return launch_tile<TILE_SPLIT, 128, 4>(ctx, g, split);
  if (best == pair_wide) return launch_tile<TILE_PAIR, 256, 5>(ctx, g);
  if (best == pair_narrow) return launch_tile<TILE_PAIR, 128, 6>(ctx, g);
  return launch_tile<TILE_ONE, 256, 3>(ctx, g);
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
  return launch(ctx, g);
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

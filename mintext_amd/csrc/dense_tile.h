// One output tile of a matrix product C = A B on the 16-bit matrix cores (gfx950), in registers, and its
// way out through LDS: the loop that linear.hip and muon.hip build their kernels from.
//
// WM x WN waves, each with TM x TN accumulator blocks of v_mfma_f32_32x32x16; the reduction runs in stages of
// 32 elements through an NST-deep LDS ring that global_load_lds_dwordx4 fills NST - 1 stages ahead (no staging
// registers).  Either operand may have its reduction contiguous in memory ("rows": A [m][k], B [n][k]) or
// strided ("cols": A [k][m], B [k][n]); the latter is turned by ds_read_b64_tr_b16.  LDS layouts of a stage:
//   rows: 64 bytes a row, 16-byte chunk c of row r at chunk c ^ ((r >> 2) & 3)
//   cols: one line a reduction element, chunk c of element k at chunk c ^ 4 (k & 3) (64 columns: c ^ 2 (k & 2))
// with which neither the loads' writes nor the fragment reads conflict.
//
// A 256 x 256 tile keeps 256 accumulators a lane and one workgroup a CU; what bounds it is the matrix cores at the clock that the
// power limit leaves: 1.2 PFLOP/s in bf16 and f16, as a large library product.  128 x 128 tiles, two workgroups a CU, read
// twice as much LDS for a product and take 1.4 times as long for the same work, but fill the chip with fewer.
//
// Bounds: rows (or columns, which come in chunks of 8) past the operand's last re-read the last one, so no load
// leaves the operand and what they give is never stored.  TAIL: the reduction may end inside a stage; what is
// past its end re-reads valid elements, which are zeroed in both operands' fragments.
// TWO: each operand is the sum of two planes, hi + lo; a stage's three products hi hi, hi lo and lo hi follow
// each other as three ring stages, so the loop is the same and the last factor, lo lo, 2^-22 of the
// result in f16, is left out.
#pragma once
#include "common.h"
#include "lds_dma.h"
#include <type_traits>

namespace mtx {
namespace dense {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;

struct Bf16 {
  typedef __bf16 elem;
  typedef __attribute__((ext_vector_type(8))) __bf16 x8;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
struct F16 {
  typedef _Float16 elem;
  typedef __attribute__((ext_vector_type(8))) _Float16 x8;
  static __device__ __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

constexpr int BKS = 32;  // reduction elements per ring stage

// One operand of a tile: `p[0]` at the tile's first row (or column) of reduction element 0, uniform; `p[1]` the lo
// plane of it; `ld` its row stride in elements; `left` the rows (rows) or columns (cols) from there that exist.
// `missing` (cols, TAIL, below 8): lines at the reduction's end that this operand does not have and that the product leaves out;
// what the other operand has there can be read.
struct Operand {
  const void* p[2];
  int64_t ld;
  int left;
  int missing = 0;
};

// A pointer that is the same in every lane, in scalar registers whatever the compiler can prove.
__device__ __forceinline__ const char* uniform(const void* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const char*)((uint64_t)lo | ((uint64_t)hi << 32));
}

// Eight values to consecutive elements on a 16-byte boundary, rounded to nearest even by the conversion instructions.
__device__ __forceinline__ void store8(float* p, const float v[8]) { st8(p, 0, v); }
__device__ __forceinline__ void store8(uint16_t* p, const float v[8]) {
  typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
  *(bf16x8*)p = bf16x8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3],
                       (__bf16)v[4], (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]};
}

// Diagonal matrices that are multiplied in beside the product: C += D B + A D', D = diag(row), D' = diag(col), for operands
// whose reduction index is the output's row (D) or column (D') index.  Where a stage's reduction elements are a block's
// own rows (columns), one more MFMA takes that 32 x 32 block of D in A's place (D' in B's), made in registers: what
// an f16 matrix lost of its f32 diagonal joins the product with no access to memory.
// CONST: D = (hi + lo) I instead, for both planes of B.
struct Diagonal {
  const float *row, *col;  // of the whole matrices, or nullptr
  float hi, lo;            // CONST
  int m0, n0, m, n;        // the tile's first row and column; rows and columns of C that exist
};
enum { DIAG_NONE = 0, DIAG_VECTORS = 1, DIAG_CONST = 2 };

__device__ __forceinline__ int row_off(int r, int c) { return r * 64 + ((c ^ ((r >> 2) & 3)) << 4); }
// what chunks of line k of a cols operand are turned by: lines of 64 columns take turns with the next but one
template <int COLS>
__device__ __forceinline__ int col_turn(int k) { return COLS == 64 ? (k & 2) << 1 : (k & 3) << 2; }
template <int COLS>
__device__ __forceinline__ int col_off(int k, int c) { return k * (COLS * 2) + ((c ^ col_turn<COLS>(k)) << 4); }

// PART > 0: every PART stages make a sum of their own, for results whose rounding counts (logits around 10 of 1324 products
// are 2.0e-7 off with 4, 5.7e-7 with one sum).
template <class F, int TM_, int TN_, int WM_, int WN_, int NST_, bool A_COLS, bool B_COLS, bool TAIL = false,
          bool TWO = false, int DIAG = DIAG_NONE, int PART = 0>
struct Tile {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, NST = NST_, PD = NST - 1;
  static constexpr bool cols = A_COLS, b_cols = B_COLS;
  static constexpr int NW = WM * WN, NT = NW * 64, BM = 32 * TM * WM, BN = 32 * TN * WN;
  static constexpr int A_BYTES = BM * BKS * 2, B_BYTES = BN * BKS * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int LDS_BYTES = NST * STAGE;
  static constexpr int A_INSTR = A_BYTES / 1024 / NW, B_INSTR = B_BYTES / 1024 / NW, LPS = A_INSTR + B_INSTR;
  static_assert(A_BYTES % (1024 * NW) == 0 && B_BYTES % (1024 * NW) == 0, "whole load instructions per wave");
  static_assert(PD >= 3, "a stage's fragments are read from half a stage ahead");
  static_assert(!(TAIL && TWO), "two planes come padded");
  typedef typename F::x8 x8;

  static __device__ __forceinline__ int slot(int k) { return (NST & (NST - 1)) == 0 ? (k & (NST - 1)) : k % NST; }

  // byte offset of what lane `lane` of load instruction `i` of wave `wave` reads, from the operand's pointer at the
  // stage's first reduction element; `kleft`: reduction elements that exist from there (TAIL)
  template <bool COLS, int INSTR, int W>
  static __device__ __forceinline__ uint32_t source(const Operand& o, int i, int wave, int lane, int kleft) {
    const int seg = wave * INSTR + i;
    if constexpr (COLS) {
      constexpr int CH = W / 8, PER = 64 / CH;  // chunks per line, lines per instruction
      const int k = seg * PER + lane / CH, c = (lane % CH) ^ col_turn<W>(k);
      return (uint32_t)min(k, kleft - 1) * (uint32_t)(o.ld * 2) + (uint32_t)min(c * 8, o.left - 8) * 2u;
    } else {
      const int r = seg * 16 + (lane >> 2), c = (lane & 3) ^ ((r >> 2) & 3);
      return (uint32_t)min(r, o.left - 1) * (uint32_t)(o.ld * 2) + (uint32_t)min(c * 8, kleft - 8) * 2u;
    }
  }

  // acc = the product over reduction elements [0, K) (K > 0; without TAIL a multiple of 32, with it a multiple of 8
  // where an operand has it contiguous).  Ends with no load in flight, but the waves not in step.
  static __device__ __forceinline__ void product(const Operand& a, const Operand& b, int K, char* lds,
                                                 f32x16 (&acc)[TM][TN], const Diagonal* dg = nullptr) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / WN, wn = wave % WN;
    const int nk1 = (K + BKS - 1) / BKS, nk = TWO ? 3 * nk1 : nk1;
    const int tail = K - (nk1 - 1) * BKS, a_tail = tail - (A_COLS ? a.missing : 0), b_tail = tail - (B_COLS ? b.missing : 0);
    const int both_tail = min(a_tail, b_tail);  // what lies behind it is masked: a last line read again, times 0, may be no number
    uint32_t aoff[A_INSTR], boff[B_INSTR], atail[TAIL ? A_INSTR : 1], btail[TAIL ? B_INSTR : 1];
#pragma unroll
    for (int i = 0; i < A_INSTR; ++i) {
      aoff[i] = source<A_COLS, A_INSTR, BM>(a, i, wave, lane, TAIL && nk1 == 1 ? a_tail : BKS);
      if constexpr (TAIL) atail[i] = source<A_COLS, A_INSTR, BM>(a, i, wave, lane, a_tail);
    }
#pragma unroll
    for (int i = 0; i < B_INSTR; ++i) {
      boff[i] = source<B_COLS, B_INSTR, BN>(b, i, wave, lane, TAIL && nk1 == 1 ? b_tail : BKS);
      if constexpr (TAIL) btail[i] = source<B_COLS, B_INSTR, BN>(b, i, wave, lane, b_tail);
    }
    const int64_t a_step = A_COLS ? a.ld * (BKS * 2) : BKS * 2, b_step = B_COLS ? b.ld * (BKS * 2) : BKS * 2;
    const uint32_t lds_base = lds_addr(lds);
    const uint32_t wave_u = (uint32_t)__builtin_amdgcn_readfirstlane(wave);
    // The stage that is loaded next; stages past the end re-read the last one into a slot that is no longer read.
    const char* const planes_a[2] = {uniform(a.p[0]), uniform(a.p[TWO ? 1 : 0])};
    const char* const planes_b[2] = {uniform(b.p[0]), uniform(b.p[TWO ? 1 : 0])};
    const char *pa = planes_a[0], *pb = planes_b[0];
    int64_t at_a = 0, at_b = 0;  // TWO: byte offset of the reduction element in either plane
    int next = 0, part = 0;
    bool last = nk == 1;
    auto advance = [&]() {
      if (next + 1 >= nk) return;
      ++next;
      last = next + 1 == nk;
      if constexpr (TWO) {
        if (++part == 3) {
          part = 0;
          at_a += a_step;
          at_b += b_step;
        }
        pa = (part == 2 ? planes_a[1] : planes_a[0]) + at_a;
        pb = (part == 1 ? planes_b[1] : planes_b[0]) + at_b;
      } else {
        pa += a_step;
        pb += b_step;
      }
    };
    // load instruction d of the next stage, into the slot of stage kt
    auto issue = [&](int kt, int d) {
      const uint32_t st = lds_base + (uint32_t)(slot(kt) * STAGE);
      if (d < A_INSTR) {
        gload_lds16_s(pa, TAIL && last ? atail[TAIL ? d : 0] : aoff[d], st + (wave_u * A_INSTR + d) * 1024u);
      } else {
        const int i = d - A_INSTR;
        gload_lds16_s(pb, TAIL && last ? btail[TAIL ? i : 0] : boff[i],
                      st + (uint32_t)A_BYTES + (wave_u * B_INSTR + i) * 1024u);
      }
    };

    x8 fa[2][TM], fb[2][TN];
    const int frow = lane & 31, fhalf = lane >> 5;
    // eight reduction elements kk * 16 + 8 (lane / 32) .. of row or column x0 + lane % 32
    auto fragment = [&](const char* region, auto cols, auto width, int x0, int kk) -> x8 {
      if constexpr (decltype(cols)::value) {
        constexpr int W = decltype(width)::value;
        const int n = x0 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3), k = kk * 16 + 8 * fhalf + ((lane & 15) >> 2);
        const s16x4 both[2] = {
            __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(region + col_off<W>(k, n >> 3) + (n & 7) * 2)),
            __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(region + col_off<W>(k + 4, n >> 3) + (n & 7) * 2))};
        return __builtin_bit_cast(x8, both);
      } else {
        return *(const x8*)(region + row_off(x0 + frow, kk * 2 + fhalf));
      }
    };
    // fragment r of a substep: r < TM is A block r, else B block r - TM
    auto read = [&](int kt, int kk, int buf, int r) {
      const char* st = lds + slot(kt) * STAGE;
      if (r < TM)
        fa[buf][r] = fragment(st, std::bool_constant<A_COLS>(), std::integral_constant<int, BM>(),
                              wm * (TM * 32) + r * 32, kk);
      else
        fb[buf][r - TM] = fragment(st + A_BYTES, std::bool_constant<B_COLS>(), std::integral_constant<int, BN>(),
                                   wn * (TN * 32) + (r - TM) * 32, kk);
    };
    auto mask = [&](int buf, int kk) {
      const int nv = min(max(both_tail - kk * 16 - 8 * fhalf, 0), 8);
      u32x4 m;
#pragma unroll
      for (int d = 0; d < 4; ++d) m[d] = (2 * d + 1 < nv) ? 0xFFFFFFFFu : ((2 * d < nv) ? 0xFFFFu : 0u);
#pragma unroll
      for (int i = 0; i < TM; ++i) fa[buf][i] = __builtin_bit_cast(x8, __builtin_bit_cast(u32x4, fa[buf][i]) & m);
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[buf][j] = __builtin_bit_cast(x8, __builtin_bit_cast(u32x4, fb[buf][j]) & m);
    };

#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;
    f32x16 sum[PART > 0 ? TM : 1][PART > 0 ? TN : 1];
    if constexpr (PART > 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) sum[i][j] = acc[i][j];
    }

    // the lane's elements of the diagonals: row or column lane % 32 of each block
    float drow[DIAG == DIAG_VECTORS ? TM : 1], dcol[DIAG == DIAG_VECTORS ? TN : 1];
    const int row0 = DIAG ? __builtin_amdgcn_readfirstlane(dg->m0 + wm * (TM * 32)) : 0;
    const int col0 = DIAG ? __builtin_amdgcn_readfirstlane(dg->n0 + wn * (TN * 32)) : 0;
    bool has_row = DIAG == DIAG_CONST, has_col = false;
    if constexpr (DIAG == DIAG_VECTORS) {
      has_row = dg->row != nullptr;
      has_col = dg->col != nullptr;
      if (has_row) {
#pragma unroll
        for (int i = 0; i < TM; ++i) drow[i] = row0 + i * 32 + frow < dg->m ? dg->row[row0 + i * 32 + frow] : 0.0f;
      }
      if (has_col) {
#pragma unroll
        for (int j = 0; j < TN; ++j) dcol[j] = col0 + j * 32 + frow < dg->n ? dg->col[col0 + j * 32 + frow] : 0.0f;
      }
    }
    // substep `sub` of the 32 x 32 diagonal block with v in the lane's row
    auto diagonal = [&](float v, int sub) -> x8 {
      const typename F::elem e = (typename F::elem)v;
      const int at = frow - sub * 16 - 8 * fhalf;
      x8 d;
#pragma unroll
      for (int q = 0; q < 8; ++q) d[q] = q == at ? e : (typename F::elem)0.0f;
      return d;
    };
    // Behind a stage's products and before the barrier that lets its slot go: the fragments are read again, so that the
    // loop's own registers and order stay as they are (with the terms among the products those took a quarter longer).
    auto diagonals = [&](int kt) {
      const int part = TWO ? kt % 3 : 0, k = (TWO ? kt / 3 : kt) * BKS;
      const char* st = lds + slot(kt) * STAGE;
      auto frag_a = [&](int i, int sub) {
        return fragment(st, std::bool_constant<A_COLS>(), std::integral_constant<int, BM>(), wm * (TM * 32) + i * 32, sub);
      };
      auto frag_b = [&](int j, int sub) {
        return fragment(st + A_BYTES, std::bool_constant<B_COLS>(), std::integral_constant<int, BN>(),
                        wn * (TN * 32) + j * 32, sub);
      };
      if (DIAG == DIAG_CONST ? part == 2 : part != 0) return;
      if (has_row && k >= row0 && k < row0 + TM * 32) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (k != row0 + i * 32) continue;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            const x8 d = diagonal(DIAG == DIAG_CONST ? dg->hi : drow[DIAG == DIAG_CONST ? 0 : i], sub);
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = F::mfma(frag_b(j, sub), d, acc[i][j]);
            if (DIAG == DIAG_CONST && part == 0) {
              const x8 lo = diagonal(dg->lo, sub);
#pragma unroll
              for (int j = 0; j < TN; ++j) acc[i][j] = F::mfma(frag_b(j, sub), lo, acc[i][j]);
            }
          }
        }
      }
      if (DIAG == DIAG_VECTORS && has_col && k >= col0 && k < col0 + TN * 32) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          if (k != col0 + j * 32) continue;
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            const x8 d = diagonal(dcol[DIAG == DIAG_VECTORS ? j : 0], sub);
#pragma unroll
            for (int i = 0; i < TM; ++i) acc[i][j] = F::mfma(d, frag_a(i, sub), acc[i][j]);
          }
        }
      }
    };

    // prologue: stages 0 .. PD-1 in flight, stages 0 and 1 landed and visible
#pragma unroll
    for (int s = 0; s < PD; ++s) {
#pragma unroll
      for (int d = 0; d < LPS; ++d) issue(s, d);
      advance();
    }
    __builtin_amdgcn_s_waitcnt(MTX_VMCNT(LPS * (PD - 2)));
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TM + TN; ++r) read(0, 0, 0, r);
    // A stage is 2 x S slots in a fixed order: one MFMA, one fragment read of the other buffer, and the stage's
    // ring loads spread evenly, so that a SIMD's MFMA pipe is not held up by a burst of loads.
    constexpr int S = TM * TN;
    auto half = [&](auto which, int kt) {
      constexpr int sub = decltype(which)::value;
      if (TAIL && kt == nk - 1 && both_tail < BKS) mask(sub, sub);
#pragma unroll
      for (int qq = 0; qq < S; ++qq) {
        const int i = qq / TN, j = qq % TN;
        __builtin_amdgcn_sched_barrier(0);
        acc[i][j] = F::mfma(fb[sub][j], fa[sub][i], acc[i][j]);
        // a substep with fewer MFMAs than fragments reads the rest in its last slot
#pragma unroll
        for (int r = 0; r < TM + TN; ++r) {
          if (min(r, S - 1) != qq) continue;
          if (sub == 0) read(kt, 1, 1, r);
          else read(kt + 1, 0, 0, r);  // visible since the last barrier (last stage: not used)
        }
#pragma unroll
        for (int d = 0; d < LPS; ++d)
          if ((d * 2 * S) / LPS == sub * S + qq) issue(kt + PD, d);
      }
    };
    for (int kt = 0; kt < nk; ++kt) {
      half(std::integral_constant<int, 0>(), kt);
      half(std::integral_constant<int, 1>(), kt);
      advance();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (DIAG != DIAG_NONE) diagonals(kt);
      if constexpr (PART > 0) {
        if (kt % PART == PART - 1 || kt == nk - 1) {
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
              for (int v = 0; v < 16; ++v) {
                sum[i][j][v] += acc[i][j][v];
                acc[i][j][v] = 0.0f;
              }
        }
      }
      // Stage kt + 2 landed before the barrier makes it visible.  A bare s_barrier: the slot refilled next held
      // stage kt, whose fragments this iteration's MFMAs consumed.
      __builtin_amdgcn_s_waitcnt(MTX_VMCNT(LPS * (PD - 2)));
      __builtin_amdgcn_s_barrier();
    }
    __builtin_amdgcn_s_waitcnt(MTX_VMCNT(0));  // no ring load may land after the ring is reused
    if constexpr (PART > 0) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = sum[i][j];
    }
  }

  // ---- the tile's way out: acc[i][j][4g+q] of lane l is C[32 i + l % 32][32 j + 8 g + 4 (l / 32) + q] of the wave's
  // part.  Each wave puts 32 rows at a time into LDS of its own (f32, 16-byte chunk c of row r at c ^ (r % chunks))
  // and takes them back as eight consecutive columns a lane, whole lines a row.
  static constexpr int OUT_BYTES = 32 * TN * 32 * 4;  // of a wave
  static __device__ __forceinline__ char* out_lds(char* lds) { return lds + (threadIdx.x >> 6) * OUT_BYTES; }
  static __device__ __forceinline__ void put(const f32x16 (&acc)[TN], char* mine) {
    const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(mine + row * (TN * 128) + (((j * 8 + 2 * g + h) ^ (row & (TN * 8 - 1))) << 4)) =
            f32x4{acc[j][4 * g], acc[j][4 * g + 1], acc[j][4 * g + 2], acc[j][4 * g + 3]};
    __builtin_amdgcn_s_waitcnt(MTX_LGKMCNT0);
    asm volatile("" ::: "memory");
  }
  // The same for results in 16 bits: 32 rows of TN * 64 bytes, 16-byte chunk c of row r at c ^ (r % chunks).
  static constexpr int OUT16_BYTES = 32 * TN * 64;  // of a wave and plane
  static __device__ __forceinline__ int out16_off(int r, int c) { return r * (TN * 64) + ((c ^ (r & (TN * 4 - 1))) << 4); }
  static __device__ __forceinline__ s16x4 out16_tr(const char* mine, int r, int c) {  // four rows from r of column ..
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(mine + out16_off(r, c >> 3) + (c & 7) * 2));
  }
  static constexpr int OUT_STEPS = TN * 2;  // of 64 lanes x 8 columns; a lane's columns are the same in each
  static_assert(64 % (TN * 4) == 0, "whole rows a step");
  static __device__ __forceinline__ int out_row(int it) { return (it * 64 + (threadIdx.x & 63)) / (TN * 4); }
  static __device__ __forceinline__ int out_col(int it) { return (it * 64 + (threadIdx.x & 63)) % (TN * 4) * 8; }
  static __device__ __forceinline__ void get(const char* mine, int it, float v[8]) {
    const int row = out_row(it), c = out_col(it) >> 2;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 x = *(const f32x4*)(mine + row * (TN * 128) + (((c + h) ^ (row & (TN * 8 - 1))) << 4));
#pragma unroll
      for (int q = 0; q < 4; ++q) v[4 * h + q] = x[q];
    }
  }
};

// Workgroup `pid` of a launch of `total` tiles (grid: tiles_grid(total)): consecutive tiles go to one XCD, which
// keeps what they share in its L2.  -1: none.
__device__ __forceinline__ int tile_of(int pid, int total) {
  const int per = (total + 7) >> 3, t = (pid & 7) * per + (pid >> 3);
  return t < total && (pid >> 3) < per ? t : -1;
}
inline int64_t tiles_grid(int64_t total) { return (total + 7) / 8 * 8; }

}  // namespace dense
}  // namespace mtx

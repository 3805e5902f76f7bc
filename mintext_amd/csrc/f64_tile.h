// One output tile of a matrix product in f64 on the f64 matrix cores (gfx950): the tile loop of the float64 form of
// newton_schulz.
//
// BT x BT outputs, four waves of (BT / 2) x (BT / 2) in blocks of v_mfma_f64_16x16x4_f64, stages of KS reduction elements
// through one LDS buffer with the next stage's operands loaded into registers meanwhile.  Both operands are kept as [k][x]
// in LDS: two lines of BT + 16 values lie 32 banks apart and the next pair is shifted by two values, so that neither the
// fragments' reads (two lines of 16 values in half a wave) nor the writes of an operand whose reduction is contiguous in
// memory (16 lines) meet on a bank.  Any size and alignment: single values are loaded, those past the end are zeros.
// Large products are bound by the matrix cores: X <- Q X and its products of 12 x 768 x 640 run at 42 TFLOP/s, as a loop of
// these instructions alone does.  Stages of twice as many elements take 3 to 12 % longer, of four times up to 20 %.
#pragma once
#include "common.h"

namespace mtx {
namespace f64mm {

typedef __attribute__((ext_vector_type(4))) double f64x4;
constexpr int NT = 256;

// Element (x, k) of an operand is at p[x * ld + k] (reduction contiguous) or p[k * ld + x]; `left`: how many x exist.
struct Operand {
  const double* p;
  int64_t ld;
  int left;
};

template <int BT, int KS>
struct Tile {
  static constexpr int TB = BT / 32, LD = BT + 16, LDS = 2 * KS * LD, N = BT * KS / NT;  // LDS: in doubles

  static __device__ __forceinline__ int at(int k, int x) { return k * LD + x + 2 * ((k >> 1) & 7); }
  template <bool KC>
  static __device__ __forceinline__ void load(double (&v)[N], const Operand& o, int k0, int K) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int q = threadIdx.x + u * NT, k = k0 + (KC ? q % KS : q / BT), x = KC ? q / KS : q % BT;
      v[u] = x < o.left && k < K ? o.p[KC ? x * o.ld + k : k * o.ld + x] : 0.0;
    }
  }
  template <bool KC>
  static __device__ __forceinline__ void store(const double (&v)[N], double* to) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int q = threadIdx.x + u * NT;
      to[at(KC ? q % KS : q / BT, KC ? q / KS : q % BT)] = v[u];
    }
  }
  // acc[i][j][r] of lane l: row 16 i + l / 16 + 4 r, column 16 j + l % 16 of the wave's part.  A_KC, B_KC: the operand's
  // reduction is contiguous in memory.
  template <bool A_KC, bool B_KC>
  static __device__ __forceinline__ void product(const Operand& a, const Operand& b, int K, double* lds,
                                                 f64x4 (&acc)[TB][TB]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double *as = lds, *bs = lds + KS * LD;
    const int k = lane >> 4, xa = (wave >> 1) * (TB * 16) + (lane & 15), xb = (wave & 1) * (TB * 16) + (lane & 15);
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j) acc[i][j] = f64x4{0.0, 0.0, 0.0, 0.0};
    double va[N], vb[N];
    load<A_KC>(va, a, 0, K);
    load<B_KC>(vb, b, 0, K);
    for (int k0 = 0; k0 < K; k0 += KS) {
      store<A_KC>(va, as);
      store<B_KC>(vb, bs);
      __syncthreads();
      if (k0 + KS < K) {
        load<A_KC>(va, a, k0 + KS, K);
        load<B_KC>(vb, b, k0 + KS, K);
      }
#pragma unroll
      for (int kk = 0; kk < KS; kk += 4) {
        double x[TB], y[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
          x[i] = as[at(kk + k, xa + i * 16)];
          y[i] = bs[at(kk + k, xb + i * 16)];
        }
#pragma unroll
        for (int i = 0; i < TB; ++i)
#pragma unroll
          for (int j = 0; j < TB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(x[i], y[j], acc[i][j], 0, 0, 0);
      }
      __syncthreads();
    }
  }
  // f(row, column, value) for each of the lane's outputs
  template <typename F>
  static __device__ __forceinline__ void each(const f64x4 (&acc)[TB][TB], F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          f((wave >> 1) * (TB * 16) + i * 16 + (lane >> 4) + 4 * r, (wave & 1) * (TB * 16) + j * 16 + (lane & 15), acc[i][j][r]);
  }
};

}  // namespace f64mm
}  // namespace mtx

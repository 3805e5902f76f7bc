// Dense product with its epilogue, out = act(x w + bias) + residual, and the parts of its gradient.
//
// The bias, the activation, the residual and, for training, the copy of z = x w + bias that the gradient needs
// are applied to the f32 sums on their way out, so that z costs at most one write and the rest no
// pass of their own.  bf16 with rows of whole 16-byte chunks runs on the 16-bit matrix cores (dense_tile.h), in tiles of
// 256 x 256 or, where those are few, 256 x 128 or 128 x 128, and up to 64 rows on a kernel that streams w;
// everything else on f32 matrix-core tiles (f32_tile.h), which for bf16 at other widths is 7 to 16 times slower (4096 x
// 2048 x 50257 12.5 ms, 50264 columns 0.78; 1 x 2048 x 50257 295 us, 46; 4093 x 2047 x 7167 1805 us, 2048 x 7168 112).
#include "common.h"
#include "dense_tile.h"
#include "f32_tile.h"
#include <algorithm>

namespace mtx {
namespace lin {

enum { FWD = 0, DX = 1, DW = 2 };

struct Args {
  const void* a;         // FWD: x [M][K]; DX: dz [M][N]; DW: x [M][K]
  const void* b;         // FWD: w [K][N]; DX: w [K][N]; DW: dz [M][N]
  void* out;             // [rows][cols]
  const void* bias;      // [cols] or nullptr
  const void* residual;  // [rows][cols] or nullptr
  void* pre;             // [rows][cols]: z, or nullptr
  int act;
  int rows, cols, red;   // of the product
  int pieces;            // the reduction is split over so many workgroups; more than one: f32 sums to `part`
  float* part;           // [pieces][rows][cols]
};

// The activations.  -inf gives NaN in all but ReLU (0 x inf), as the formulas do.
__device__ __forceinline__ float activate(float z, int act) {
  switch (act) {
    case MTX_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays
    case MTX_ACT_SILU: return silu_f32(z);
    case MTX_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case MTX_ACT_GELU_TANH:  // 0.5 (1 + tanh u) = 1 / (1 + exp(-2 u))
      return z / (1.0f + expf(-1.5957691216057308f * (z + 0.044715f * z * z * z)));
    default: return z;
  }
}
// The same for results in bf16, with the hardware's exp2 and reciprocal: in the 256-row tiles' way out the exact
// functions took a fifth of the products' time.  erfc(x) = P(1 / (1 + 0.3275911 x)) exp(-x^2) is Abramowitz and Stegun's
// 7.1.26, |error| <= 1.5e-7.
__device__ __forceinline__ float activate_fast(float z, int act) {
  switch (act) {
    case MTX_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case MTX_ACT_SILU: return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    case MTX_ACT_GELU: {
      const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.0f + 0.3275911f * x);
      const float p = t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
      const float c = p * __expf(-x * x);  // erfc(|z| / sqrt 2)
      return 0.5f * z * (z < 0.0f ? c : 2.0f - c);
    }
    case MTX_ACT_GELU_TANH:
      return z * __builtin_amdgcn_rcpf(1.0f + __expf(-1.5957691216057308f * (z + 0.044715f * z * z * z)));
    default: return z;
  }
}
__device__ __forceinline__ float activation_slope(float z, int act) {
  switch (act) {
    case MTX_ACT_RELU: return z > 0.0f ? 1.0f : (z <= 0.0f ? 0.0f : z);
    case MTX_ACT_SILU: {
      const float s = 1.0f / (1.0f + expf(-z));
      return s * (1.0f + z * (1.0f - s));
    }
    case MTX_ACT_GELU:
      return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * 0.3989422804014327f * expf(-0.5f * z * z);
    case MTX_ACT_GELU_TANH: {
      if (fabsf(z) > 30.0f) return z > 0.0f ? 1.0f : 0.0f;  // z^3 would overflow
      const float s = 1.0f / (1.0f + expf(-1.5957691216057308f * (z + 0.044715f * z * z * z)));
      return s + z * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * z * z);
    }
    default: return 1.0f;
  }
}

// ---- any size and alignment: 64 x 64 tiles, products and sums in f32 --------------------------------------
// Small products are bound by the length of one tile's chain of stages, hence the split (plan()); large ones by the f32
// matrix cores: 1000 x 2000 x 1000 takes 51 us, 79 TFLOP/s of 154, 8192 x 4096 x 14336 8.3 ms, 116.
template <typename T, int MODE, int VEC>
__global__ __launch_bounds__(f32mm::NT) void f32_kernel(Args p) {
  using namespace f32mm;
  __shared__ __attribute__((aligned(16))) float as[TILE], bs[TILE];
  const int64_t r0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int64_t rows = p.rows, cols = p.cols;
  const T *A = (const T*)p.a, *B = (const T*)p.b;
  const int stages = (p.red + KS - 1) / KS, piece = blockIdx.z;
  const int64_t kb = (int64_t)piece * stages / p.pieces * KS;
  const int64_t red = min((int64_t)(piece + 1) * stages / p.pieces * KS, (int64_t)p.red);  // of this piece: [kb, red)
  auto at_a = [&](int r, int c, int s) -> const T* {
    if (MODE == DW) {
      const int64_t k = kb + (int64_t)s * KS + r, m = r0 + c;
      return k < red && m < rows ? A + k * rows + m : nullptr;
    }
    const int64_t m = r0 + r, k = kb + (int64_t)s * KS + c;
    return m < rows && k < red ? A + m * p.red + k : nullptr;
  };
  auto at_b = [&](int r, int c, int s) -> const T* {
    if (MODE == DX) {
      const int64_t n = n0 + r, k = kb + (int64_t)s * KS + c;
      return n < cols && k < red ? B + n * p.red + k : nullptr;
    }
    const int64_t k = kb + (int64_t)s * KS + r, n = n0 + c;
    return k < red && n < cols ? B + k * cols + n : nullptr;
  };
  f32x16 acc;
  mainloop<T, MODE == DW, MODE != DX, VEC>(acc, (int)(red - kb), as, bs, at_a, at_b, A, B);
  const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) >> 1, wn = (threadIdx.x >> 6) & 1;
  const int64_t n = n0 + wn * 32 + (lane & 31);
  if (n >= cols) return;
  const float bias = p.bias ? gld<T>((const T*)p.bias, n) : 0.0f;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int64_t r = r0 + wm * 32 + 8 * (v / 4) + 4 * (lane >> 5) + v % 4;
    if (r >= rows) continue;
    if (p.pieces > 1) {
      p.part[((int64_t)piece * rows + r) * cols + n] = acc[v];
      continue;
    }
    const float z = acc[v] + bias;
    if (p.pre) gst<T>((T*)p.pre, r * cols + n, z);
    float y = activate(z, p.act);
    if (p.residual) y += gld<T>((const T*)p.residual, r * cols + n);
    gst<T>((T*)p.out, r * cols + n, y);
  }
}

// ---- bf16, rows of whole 16-byte chunks: tiles of the 16-bit matrix cores -----------------------------------------
using dense::Operand;
template <int MODE, bool TAIL> using Big = dense::Tile<dense::Bf16, 4, 4, 2, 2, 4, MODE == DW, MODE != DX, TAIL>;
template <int MODE, bool TAIL> using Mid = dense::Tile<dense::Bf16, 4, 2, 2, 2, 4, MODE == DW, MODE != DX, TAIL>;
template <int MODE, bool TAIL> using Small = dense::Tile<dense::Bf16, 2, 2, 2, 2, 4, MODE == DW, MODE != DX, TAIL>;

// z = v + bias, out = act(z) + residual for eight columns; `bias` and `residual` are those eight of them
__device__ __forceinline__ void finish8(const Args& p, int act, int64_t at, float v[8], const float bias[8],
                                        const uint16_t* residual) {
  if (p.bias) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += bias[q];
  }
  if (p.pre) dense::store8((uint16_t*)p.pre + at, v);
  if (act != MTX_ACT_NONE) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate_fast(v[q], act);
  }
  if (p.residual) {
    float b[8];
    ld8(residual, 0, b);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += b[q];
  }
  dense::store8((uint16_t*)p.out + at, v);
}
__device__ __forceinline__ void finish8(const Args& p, int r, int c, float v[8]) {
  const int64_t at = (int64_t)r * p.cols + c;
  float bias[8];
  if (p.bias) ld8((const uint16_t*)p.bias, c, bias);
  finish8(p, p.act, at, v, bias, (const uint16_t*)p.residual + at);
}

// Bound by the matrix cores in large products: 8192 x 4096 x 14336 in 780 to 800 us, 1.2 PFLOP/s, which is what a plain
// library product of the size reaches (813 us); 4093 x 2048 x 7168 in 111 (137 with z and a residual), its gradients in 129
// to 134 and 115 to 119.  Of few
// tiles it is the length of a tile's reduction that counts, which plan() splits.
// Tiles go row by row within groups of kGroup rows of tiles, so that neighbours share both operands' strips in L2
// (8192 x 4096 x 14336: 805 us without groups, 778 in groups of 4, 783 of 8, 790 of 16).
constexpr int kGroup = 8;
template <class T, int MODE, int ACT>
__global__ __launch_bounds__(T::NT, T::LDS_BYTES > 80 * 1024 ? 1 : 2) void tile_kernel(Args p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS_BYTES];
  const int nm = (p.rows + T::BM - 1) / T::BM, nn = (p.cols + T::BN - 1) / T::BN;
  const int id = dense::tile_of(blockIdx.x, nm * nn * p.pieces);
  if (id < 0) return;
  const int t = id / p.pieces, piece = id % p.pieces, stages = (p.red + dense::BKS - 1) / dense::BKS;
  const int k0 = (int)((int64_t)piece * stages / p.pieces) * dense::BKS;
  const int k1 = min((int)((int64_t)(piece + 1) * stages / p.pieces) * dense::BKS, p.red);
  const int g = t / (kGroup * nn), gs = min(kGroup, nm - g * kGroup), in = t - g * kGroup * nn;
  const int m0 = (g * kGroup + in % gs) * T::BM, n0 = in / gs * T::BN;
  const uint16_t *a = (const uint16_t*)p.a, *b = (const uint16_t*)p.b;
  const uint16_t* pa = MODE == DW ? a + (int64_t)k0 * p.rows + m0 : a + (int64_t)m0 * p.red + k0;
  const uint16_t* pb = MODE == DX ? b + (int64_t)n0 * p.red + k0 : b + (int64_t)k0 * p.cols + n0;
  const Operand oa{{pa, pa}, MODE == DW ? p.rows : p.red, p.rows - m0};
  const Operand ob{{pb, pb}, MODE == DX ? p.red : p.cols, p.cols - n0};
  dense::f32x16 acc[T::TM][T::TN];
  T::product(oa, ob, k1 - k0, lds, acc);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  char* mine = T::out_lds(lds);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), c = n0 + (wave % T::WN) * (T::TN * 32) + T::out_col(0);
  if (T::BM == 128 && p.pieces > 1) {
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
      T::put(acc[i], mine);
#pragma unroll
      for (int it = 0; it < T::OUT_STEPS; ++it) {
        const int r = wr + i * 32 + T::out_row(it);
        float v[8];
        T::get(mine, it, v);
        if (r < p.rows && c < p.cols) st8(p.part + ((int64_t)piece * p.rows + r) * p.cols + c, 0, v);
      }
    }
    return;
  }
  float bias[8];
  if (p.bias) ld8((const uint16_t*)p.bias, min(c, p.cols - 8), bias);
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    // the residuals of 32 rows are on their way while the rows go through LDS
    dense::u32x4 res[T::OUT_STEPS];
    if (p.residual) {
#pragma unroll
      for (int it = 0; it < T::OUT_STEPS; ++it) {
        const int r = min(wr + i * 32 + T::out_row(it), p.rows - 1);
        res[it] = *(const dense::u32x4*)((const uint16_t*)p.residual + (int64_t)r * p.cols + min(c, p.cols - 8));
      }
    }
    T::put(acc[i], mine);
#pragma unroll
    for (int it = 0; it < T::OUT_STEPS; ++it) {
      const int r = wr + i * 32 + T::out_row(it);
      float v[8];
      T::get(mine, it, v);
      if (r < p.rows && c < p.cols) finish8(p, ACT, (int64_t)r * p.cols + c, v, bias, (const uint16_t*)&res[it]);
    }
  }
}

// ---- few rows (serving): the time is that of reading w once ---------------------------------------------------------
// A workgroup owns 128 columns and a piece of the reduction; its waves (eight, or four where 64 rows need the registers)
// take the piece's 32-element chunks in turn, w straight from memory into registers (two chunks of 8 KB a wave in flight), turned into MFMA operands by byte
// permutes, 16 rows of x a block.  The waves' sums are added in wave order, the pieces' by finish_kernel in piece order.
// 1 x 4096 x 14336 with w from memory: 24 us in all, 4.9 TB/s (20 in this kernel, 4 in finish_kernel's launch); 61 x 7168
// x 2048 16 us, 12 of them here.
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
template <int J>
__device__ __forceinline__ bf16x8 column(const u32x4 (&in)[8]) {
  constexpr uint32_t sel = (J & 1) ? 0x07060302u : 0x05040100u;
  u32x4 v;
#pragma unroll
  for (int q = 0; q < 4; ++q) v[q] = __builtin_amdgcn_perm(in[2 * q + 1][J / 2], in[2 * q][J / 2], sel);
  return __builtin_bit_cast(bf16x8, v);
}
constexpr int kThinCols = 128, kThinChunk = 32;
// TB: blocks of 16 rows; NW: waves; STREAM: loads of w that leave no copy in the memory-side cache
template <int TB, int NW, bool STREAM>
__global__ __launch_bounds__(NW * 64) void thin_kernel(Args p) {
  constexpr int PADN = kThinCols + 4, kThinWaves = NW;
  __shared__ __attribute__((aligned(16))) float part[kThinWaves][16][PADN];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nn = (p.cols + kThinCols - 1) / kThinCols, nt = blockIdx.x % nn, piece = blockIdx.x / nn;
  const int chunks = (p.red + kThinChunk - 1) / kThinChunk;
  const int c0 = (int)((int64_t)piece * chunks / p.pieces), c1 = (int)((int64_t)(piece + 1) * chunks / p.pieces);
  const int l16 = lane & 15, kq = lane >> 4, nb = (p.rows + 15) >> 4;
  const int col = min(nt * kThinCols + l16 * 8, p.cols - 8);  // past the end: the last columns again, not stored
  const uint16_t* W = (const uint16_t*)p.b + col;
  const uint16_t* x[TB];
#pragma unroll
  for (int b = 0; b < TB; ++b) x[b] = (const uint16_t*)p.a + (int64_t)min(b * 16 + l16, p.rows - 1) * p.red;
  struct Chunk {
    u32x4 w[8];
    u32x4 x[TB];
  };
  auto load = [&](Chunk& c, int ck) {
    const int k = min(ck * kThinChunk + kq * 8, p.red - 8);  // past the end: re-read, zeroed in both operands
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const u32x4* q = (const u32x4*)(W + (int64_t)(k + i) * p.cols);
      c.w[i] = STREAM ? __builtin_nontemporal_load(q) : *q;
    }
#pragma unroll
    for (int b = 0; b < TB; ++b)
      if (b < nb) c.x[b] = *(const u32x4*)(x[b] + k);
  };
  f32x4 acc[8][TB];
#pragma unroll
  for (int f = 0; f < 8; ++f)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[f][b] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto use = [&](Chunk& c, int ck) {
    if (ck * kThinChunk + kThinChunk > p.red) {
      const uint32_t keep = ck * kThinChunk + kq * 8 < p.red ? 0xFFFFFFFFu : 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) c.w[i] &= keep;
#pragma unroll
      for (int b = 0; b < TB; ++b) c.x[b] &= keep;
    }
    const bf16x8 wf[8] = {column<0>(c.w), column<1>(c.w), column<2>(c.w), column<3>(c.w),
                          column<4>(c.w), column<5>(c.w), column<6>(c.w), column<7>(c.w)};
#pragma unroll
    for (int b = 0; b < TB; ++b) {
      if (b >= nb) continue;
      const bf16x8 xf = __builtin_bit_cast(bf16x8, c.x[b]);
#pragma unroll
      for (int f = 0; f < 8; ++f) acc[f][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[f], xf, acc[f][b], 0, 0, 0);
    }
  };
  {
    Chunk a, b;
#pragma unroll
    for (int i = 0; i < TB; ++i) a.x[i] = b.x[i] = u32x4{0u, 0u, 0u, 0u};
    int ck = c0 + wave;
    if (ck < c1) load(a, ck);
    for (; ck + 2 * kThinWaves < c1; ck += 2 * kThinWaves) {
      load(b, ck + kThinWaves);
      use(a, ck);
      load(a, ck + 2 * kThinWaves);
      use(b, ck + kThinWaves);
    }
    if (ck + kThinWaves < c1) {
      load(b, ck + kThinWaves);
      use(a, ck);
      use(b, ck + kThinWaves);
    } else if (ck < c1) {
      use(a, ck);
    }
  }
  // acc[f][b][r] of lane l: row 16 b + l % 16, column 8 (4 (l / 16) + r) + f of the workgroup's
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    if (b >= nb) break;
    if (b > 0) __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float* o = &part[wave][l16][8 * (4 * kq + r)];
      *(f32x4*)o = f32x4{acc[0][b][r], acc[1][b][r], acc[2][b][r], acc[3][b][r]};
      *(f32x4*)(o + 4) = f32x4{acc[4][b][r], acc[5][b][r], acc[6][b][r], acc[7][b][r]};
    }
    __syncthreads();
    for (int i = tid; i < 16 * kThinCols / 8; i += kThinWaves * 64) {
      const int row = i / (kThinCols / 8), c = i % (kThinCols / 8) * 8;
      const int r = b * 16 + row, oc = nt * kThinCols + c;
      if (r >= p.rows || oc >= p.cols) continue;
      float v[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 s = *(const f32x4*)&part[0][row][c + 4 * h];
#pragma unroll
        for (int w = 1; w < kThinWaves; ++w) s += *(const f32x4*)&part[w][row][c + 4 * h];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[4 * h + q] = s[q];
      }
      if (p.pieces > 1) st8(p.part + ((int64_t)piece * p.rows + r) * p.cols + oc, 0, v);
      else finish8(p, r, oc, v);
    }
  }
}

// The pieces' sums in piece order, and the epilogue.  V: columns a thread.  4 to 6 us: a launch and a
// chain of loads.
template <typename T, int V>
__global__ __launch_bounds__(256) void finish_kernel(Args p) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, n = (int64_t)p.rows * p.cols;
  if (i >= n) return;
  float v[V];
  if constexpr (V == 8) {
    ld8(p.part, i, v);
    for (int s = 1; s < p.pieces; ++s) {
      float w[8];
      ld8(p.part + s * n, i, w);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += w[q];
    }
    finish8(p, (int)(i / p.cols), (int)(i % p.cols), v);
  } else {
    float z = p.part[i];
    for (int s = 1; s < p.pieces; ++s) z += p.part[s * n + i];
    const int64_t c = i % p.cols;
    if (p.bias) z += gld<T>((const T*)p.bias, c);
    if (p.pre) gst<T>((T*)p.pre, i, z);
    float y = activate(z, p.act);
    if (p.residual) y += gld<T>((const T*)p.residual, i);
    gst<T>((T*)p.out, i, y);
  }
}

// ---- dz = dy act'(z) and the column sums of dz ---------------------------------------------------------------
// A workgroup takes 32 lanes x V columns of a range of rows, eight rows at a time, and leaves f32 sums of its range; a
// second launch adds the ranges in order, so the sums do not depend on timing.  dz is rounded to the operands' type, in
// which the matrix cores take it (dx and dw end 2.4e-3 off in bf16, the rounding of the result alone is 1.7e-3; a second plane
// for what it loses would double both products), and z was, as it was saved; the column sums take dz before.  One pass over dy and z: 4093 x 7168 in
// bf16, 176 MB, in 36 us with the second launch, 4.9 TB/s (41 with half as many ranges); 8192 x 14336 150 us, 4.7 TB/s.
constexpr int kSlopeRows = 8;
template <typename T, int V>
__global__ __launch_bounds__(256) void slope_kernel(const T* __restrict__ dy, const T* __restrict__ pre, int64_t M,
                                                    int64_t N, int act, T* __restrict__ dz, float* __restrict__ part,
                                                    int64_t range) {
  __shared__ float s[kSlopeRows][32 * V + 1];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + tx) * V;
  const int64_t r0 = (int64_t)blockIdx.y * range, r1 = min(r0 + range, M);
  float sum[V];
#pragma unroll
  for (int q = 0; q < V; ++q) sum[q] = 0.0f;
  if (c < N) {
    for (int64_t r = r0 + ty; r < r1; r += kSlopeRows) {
      float g[V], z[V];
      if constexpr (V == 8) {
        ld8(dy, r * N + c, g);
        if (act != MTX_ACT_NONE) ld8(pre, r * N + c, z);
      } else {
        g[0] = gld<T>(dy, r * N + c);
        if (act != MTX_ACT_NONE) z[0] = gld<T>(pre, r * N + c);
      }
      if (act != MTX_ACT_NONE) {
#pragma unroll
        for (int q = 0; q < V; ++q) g[q] *= activation_slope(z[q], act);
        if constexpr (V == 8) st8(dz, r * N + c, g);
        else gst<T>(dz, r * N + c, g[0]);
      }
#pragma unroll
      for (int q = 0; q < V; ++q) sum[q] += g[q];
    }
  }
  if (!part) return;
#pragma unroll
  for (int q = 0; q < V; ++q) s[ty][tx * V + q] = sum[q];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const int64_t col = (int64_t)blockIdx.x * 32 * V + i;
    if (col >= N) continue;
    float t = 0.0f;
#pragma unroll
    for (int y = 0; y < kSlopeRows; ++y) t += s[y][i];
    part[(int64_t)blockIdx.y * N + col] = t;
  }
}
// 32 columns and eight sums of every eighth range each (73 ranges of 7168 columns: 19 us with a thread a column)
template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const float* __restrict__ part, int n, int64_t N,
                                                         T* __restrict__ out) {
  __shared__ float s[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + tx;
  float t = 0.0f;
  if (c < N) {
#pragma unroll 4
    for (int i = ty; i < n; i += 8) t += part[(int64_t)i * N + c];
  }
  s[ty][tx] = t;
  __syncthreads();
  if (ty > 0 || c >= N) return;
  for (int y = 1; y < 8; ++y) t += s[y][tx];
  gst<T>(out, c, t);
}

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// Row ranges of slope_kernel: up to 4096 workgroups (twice as many, of half the rows at least: 39 instead of 36 us), ranges of
// whole row groups.
static int64_t slope_ranges(int64_t M, int64_t N) {
  const int64_t by_cols = ceil_div(N, 256);
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(M, 4 * kSlopeRows), 4096 / std::max<int64_t>(1, by_cols)));
}

static int check_sizes(int dtype, int64_t M, int64_t K, int64_t N) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return MTX_ERR_ARG;
  const int64_t most = 65535 * 64;  // rows of tiles in a grid; 32-bit offsets inside a tile
  if (M < 0 || K < 0 || N < 0) return MTX_ERR_ARG;
  if (M > most || K > most || N > most) return MTX_ERR_UNSUPPORTED;
  return MTX_OK;
}

// The 16-bit tiles take rows of whole 16-byte chunks: of both operands, and of what is read and written beside them.
static bool takes_tiles(int mode, const Args& p) {
  const int la = mode == DW ? p.rows : p.red, lb = mode == DX ? p.red : p.cols;
  return p.red > 0 && la % 8 == 0 && lb % 8 == 0 && p.cols % 8 == 0 && aligned16(p.a) && aligned16(p.b) &&
         aligned16(p.out) && aligned16(p.bias) && aligned16(p.residual) && aligned16(p.pre);
}

// How a product runs, by its sizes alone, and in how many pieces of its reduction.
enum { PATH_F32, PATH_BIG, PATH_MID, PATH_SMALL, PATH_THIN };
struct Plan {
  int path, pieces;
};
// rows the thin kernel holds in registers, where it is ahead of tiles of 128 rows: 17 x 4096 x 14336 26.0 us against 27.4,
// 64 rows 31.4 against 34.0; 24 x 2048 x 7168 12.2 against 13.9, 64 rows 14.9 against 15.4
constexpr int kThinRows = 64;
static Plan plan(int mode, bool tiles, int64_t rows, int64_t cols, int64_t red) {
  auto count = [&](int64_t b, int64_t n = 0) { return ceil_div(rows, b) * ceil_div(cols, n ? n : b); };
  const int64_t stages = ceil_div(red, 32);
  // pieces that bring `n` workgroups to `want`, of `least` stages or more
  auto split = [&](int64_t n, int64_t want, int64_t least) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want / n, stages / least), 32));
  };
  // 517 x 258 x 706: 14.4 us in pieces of 4 stages or more, 18.0 of 8, 15.5 of 2; 1000 x 2000 x 1000 50.9, 52.9, 49.1
  if (!tiles) return {PATH_F32, split(count(64), 512, 4)};
  // one workgroup a CU: 1 x 4096 x 14336 takes 24.9 us in 2 pieces of 112 workgroups, 30.1 in one, 29.7 in 400 workgroups;
  // 1 x 14336 x 4096 26.9 in 8 pieces, 30.0 in half as many, 30.5 in twice as many
  if (mode == FWD && rows <= kThinRows) return {PATH_THIN, split(ceil_div(cols, kThinCols), 256, 16)};
  // One round of a tile of 256 x 256 a CU takes 1, of 256 x 128 0.8, of 128 x 128 two a CU 1.05, and a second round is
  // paid whole: the middle ones where they fill one round (300 x 4096 x 16384, 256 of them: 62 us against 80 in 128 large
  // and 77 in 384 small ones), the large ones behind that (5000 x 4096 x 2048, 160 of them: 83 us against 115 in 320 middle
  // and 109 in 640 small ones), the small ones below (200 x 4096 x 16384, 256 of them: 56 us against 71 and 81).
  if (count(256, 128) > 256) return {PATH_BIG, 1};
  if (count(256, 128) >= 192) return {PATH_MID, 1};
  // pieces of 16 stages or more (1531 x 1536 x 704: 17 us, 31 in one piece, 20 where pieces may have 8 stages)
  return {PATH_SMALL, split(count(128), 512, 16)};
}
static int64_t part_bytes(int64_t rows, int64_t cols, int64_t red, int mode) {
  int64_t b = 0;
  if (rows > 0 && cols > 0)
    for (const bool tiles : {false, true}) {
      const Plan p = plan(mode, tiles, rows, cols, red);
      if (p.pieces > 1) b = std::max<int64_t>(b, p.pieces * rows * cols * 4);
    }
  return b;
}

template <typename T, int MODE>
static int launch_f32(const Args& p, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.cols, 64), (unsigned)ceil_div(p.rows, 64), (unsigned)p.pieces);
  if (grid.y > 65535) return MTX_ERR_UNSUPPORTED;
  // the operands' row lengths
  const int la = MODE == DW ? p.rows : p.red, lb = MODE == DX ? p.red : p.cols;
  const bool vec = std::is_same<T, float>::value && la % 4 == 0 && lb % 4 == 0 && aligned16(p.a) && aligned16(p.b);
  if constexpr (std::is_same<T, float>::value) {
    if (vec) {
      hipLaunchKernelGGL((f32_kernel<T, MODE, 4>), grid, dim3(f32mm::NT), 0, st, p);
      return check_launch();
    }
  }
  hipLaunchKernelGGL((f32_kernel<T, MODE, 1>), grid, dim3(f32mm::NT), 0, st, p);
  return check_launch();
}

template <int MODE, bool TAIL, int ACT>
static int launch_tiles(const Args& p, int path, hipStream_t st) {
  auto grid = [&](int bm, int bn) {
    return dim3((unsigned)dense::tiles_grid(ceil_div(p.rows, bm) * ceil_div(p.cols, bn) * p.pieces));
  };
  if (path == PATH_BIG) hipLaunchKernelGGL((tile_kernel<Big<MODE, TAIL>, MODE, ACT>), grid(256, 256), dim3(256), 0, st, p);
  else if (path == PATH_MID)
    hipLaunchKernelGGL((tile_kernel<Mid<MODE, TAIL>, MODE, ACT>), grid(256, 128), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((tile_kernel<Small<MODE, TAIL>, MODE, ACT>), grid(128, 128), dim3(256), 0, st, p);
  return check_launch();
}
template <int MODE>
static int launch_mode(const Args& p, int path, int dtype, hipStream_t st) {
  if (path == PATH_F32) return dtype == MTX_F32 ? launch_f32<float, MODE>(p, st) : launch_f32<uint16_t, MODE>(p, st);
  if (path == PATH_THIN) {
    const dim3 grid((unsigned)(ceil_div(p.cols, kThinCols) * p.pieces));
    // half the memory-side cache or more: nothing of w is found there again by the time it is next used (8 x 8192 x 28672:
    // 73 us against 81; w of 29 MB used again and again: 8.5 us streamed, 6.6 kept)
    const bool stream = (int64_t)p.red * p.cols * 2 >= (int64_t)128 << 20;
#define MTX_THIN(TB, NW)                                                                                      \
  do {                                                                                                        \
    if (stream) hipLaunchKernelGGL((thin_kernel<TB, NW, true>), grid, dim3(NW * 64), 0, st, p);               \
    else hipLaunchKernelGGL((thin_kernel<TB, NW, false>), grid, dim3(NW * 64), 0, st, p);                     \
  } while (0)
    if (p.rows <= 16) MTX_THIN(1, 8);
    else if (p.rows <= 32) MTX_THIN(2, 8);
    else MTX_THIN(4, 4);
#undef MTX_THIN
    return check_launch();
  }
#define MTX_TILES(ACT) \
  return p.red % dense::BKS ? launch_tiles<MODE, true, ACT>(p, path, st) : launch_tiles<MODE, false, ACT>(p, path, st)
  if constexpr (MODE == FWD) {
    // the activation is applied where the reduction is whole: by finish_kernel if it is in pieces
    switch (p.pieces > 1 ? MTX_ACT_NONE : p.act) {
      case MTX_ACT_RELU: MTX_TILES(MTX_ACT_RELU);
      case MTX_ACT_SILU: MTX_TILES(MTX_ACT_SILU);
      case MTX_ACT_GELU: MTX_TILES(MTX_ACT_GELU);
      case MTX_ACT_GELU_TANH: MTX_TILES(MTX_ACT_GELU_TANH);
    }
  }
  MTX_TILES(MTX_ACT_NONE);
#undef MTX_TILES
}

static int launch_product(int mode, Args p, int dtype, void* ws, hipStream_t st) {
  if (p.rows == 0 || p.cols == 0) return MTX_OK;
  if (!p.out || (p.red > 0 && (!p.a || !p.b))) return MTX_ERR_ARG;
  const bool tiles = dtype == MTX_BF16 && takes_tiles(mode, p);
  const Plan how = plan(mode, tiles, p.rows, p.cols, p.red);
  p.pieces = how.pieces;
  p.part = (float*)ws;
  if (p.pieces > 1 && (!ws || !aligned16(ws))) return MTX_ERR_WORKSPACE;
  const int rc = mode == FWD ? launch_mode<FWD>(p, how.path, dtype, st)
                 : mode == DX ? launch_mode<DX>(p, how.path, dtype, st) : launch_mode<DW>(p, how.path, dtype, st);
  if (rc != MTX_OK || p.pieces == 1) return rc;
  const int64_t n = (int64_t)p.rows * p.cols;
  if (tiles) hipLaunchKernelGGL((finish_kernel<uint16_t, 8>), dim3((unsigned)ceil_div(n, 2048)), dim3(256), 0, st, p);
  else if (dtype == MTX_F32)
    hipLaunchKernelGGL((finish_kernel<float, 1>), dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((finish_kernel<uint16_t, 1>), dim3((unsigned)ceil_div(n, 256)), dim3(256), 0, st, p);
  return check_launch();
}

}  // namespace lin
}  // namespace mtx

using namespace mtx;

extern "C" int64_t mtx_linear_workspace_size(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K < 0 || N < 0) return -1;
  int64_t b = lin::slope_ranges(M, N) * N * 4;
  b = std::max(b, lin::part_bytes(M, N, K, lin::FWD));
  b = std::max(b, lin::part_bytes(M, K, N, lin::DX));
  return std::max(b, lin::part_bytes(K, N, M, lin::DW));
}

extern "C" int mtx_linear(const void* x, const void* w, const void* bias, const void* residual, int dtype, int64_t M,
                          int64_t K, int64_t N, int act, void* out, void* pre, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  const int rc = lin::check_sizes(dtype, M, K, N);
  if (rc != MTX_OK) return rc;
  if (act < MTX_ACT_NONE || act > MTX_ACT_GELU_TANH) return MTX_ERR_ARG;
  if (workspace_bytes < mtx_linear_workspace_size(M, K, N)) return MTX_ERR_WORKSPACE;
  const lin::Args p{x, w, out, bias, residual, pre, act, (int)M, (int)N, (int)K, 1, nullptr};
  return lin::launch_product(lin::FWD, p, dtype, workspace, (hipStream_t)stream);
}

// dz and the column sums of dz; dz is dy where there is no activation.
static int launch_slope(const void* dy, const void* pre, int dtype, int64_t M, int64_t N, int act, void* dz, void* dbias,
                        void* workspace, hipStream_t st) {
  const int64_t ranges = lin::slope_ranges(M, N);
  const int64_t range = round_up(ceil_div(M, ranges), lin::kSlopeRows);
  float* part = dbias ? (float*)workspace : nullptr;
  const bool vec = N % 8 == 0 && lin::aligned16(dy) && lin::aligned16(pre) && lin::aligned16(dz);
#define MTX_SLOPE(T, V)                                                                                        \
  hipLaunchKernelGGL((lin::slope_kernel<T, V>), dim3((unsigned)ceil_div(N, 32 * V), (unsigned)ranges), dim3(256), 0, \
                     st, (const T*)dy, (const T*)pre, M, N, act, (T*)dz, part, range)
  if (dtype == MTX_F32) {
    if (vec) MTX_SLOPE(float, 8);
    else MTX_SLOPE(float, 1);
  } else {
    if (vec) MTX_SLOPE(uint16_t, 8);
    else MTX_SLOPE(uint16_t, 1);
  }
#undef MTX_SLOPE
  if (dbias) {
    const dim3 grid((unsigned)ceil_div(N, 32));
    if (dtype == MTX_F32)
      hipLaunchKernelGGL(lin::column_sum_kernel<float>, grid, dim3(256), 0, st, part, (int)ranges, N, (float*)dbias);
    else
      hipLaunchKernelGGL(lin::column_sum_kernel<uint16_t>, grid, dim3(256), 0, st, part, (int)ranges, N,
                         (uint16_t*)dbias);
  }
  return check_launch();
}

extern "C" int mtx_linear_bwd(const void* dy, const void* x, const void* w, const void* pre, int dtype, int64_t M,
                              int64_t K, int64_t N, int act, void* dz, void* dx, void* dw, void* dbias, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  int rc = lin::check_sizes(dtype, M, K, N);
  if (rc != MTX_OK) return rc;
  if (act < MTX_ACT_NONE || act > MTX_ACT_GELU_TANH) return MTX_ERR_ARG;
  const bool slope = act != MTX_ACT_NONE && (dx || dw || dbias);
  if (M > 0 && N > 0 && ((!dy && (dx || dw || dbias)) || (slope && (!pre || !dz)))) return MTX_ERR_ARG;
  if (M > 0 && N > 0 && K > 0 && ((dx && !w) || (dw && !x))) return MTX_ERR_ARG;
  if (workspace_bytes < mtx_linear_workspace_size(M, K, N) || (dbias && N > 0 && !workspace)) return MTX_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  if (N > 0 && (slope || dbias)) {
    rc = launch_slope(dy, pre, dtype, M, N, act, dz, dbias, workspace, st);
    if (rc != MTX_OK) return rc;
  }
  const void* g = act == MTX_ACT_NONE ? dy : dz;
  if (dx) {
    const lin::Args p{g, w, dx, nullptr, nullptr, nullptr, MTX_ACT_NONE, (int)M, (int)K, (int)N, 1, nullptr};
    rc = lin::launch_product(lin::DX, p, dtype, workspace, st);
    if (rc != MTX_OK) return rc;
  }
  if (!dw) return MTX_OK;
  const lin::Args p{x, g, dw, nullptr, nullptr, nullptr, MTX_ACT_NONE, (int)K, (int)N, (int)M, 1, nullptr};
  return lin::launch_product(lin::DW, p, dtype, workspace, st);
}

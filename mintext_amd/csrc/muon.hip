// Newton-Schulz orthogonalisation of stacked matrices, and the optimiser step around it (Muon), on gfx950.
//
// X_0 = x / (|x|_F + eps), then for each step X <- a X + (b A + c A^2) X with A = X X^T on the smaller side S of the
// S x L matrix.  With Q = a I + b A + c A^2 this is X <- Q X, and A itself becomes Q A Q, all of them polynomials of
// the first A: symmetric, and they commute.  So g steps need one Gram product, S x S symmetric products and one
// product X <- P X with P = Q_g ... Q_1, in all 3 S^2 L + (4 g - 3) S^3 operations (a symmetric product computes
// half its tiles), where a step by itself needs 3 S^2 L + S^3.  At L = 2.67 S (768 x 2048) five steps need
// 45 S^3 by themselves (63 if all tiles were computed), 35 as 2 + 2 + 1, 30 as 3 + 2; at L = S always 20, fastest by themselves.
// A's small eigenvalues are squares of X's and grow by a^2 a step, so what the rounding of A adds grows as well and is
// not taken back before the next Gram product: a group holds three steps at most.  In simulation with gradients of
// rank 1 to full rank (f16 operands) five steps end 0.07 to 0.19 % off as 2 + 2 + 1, 0.1 to 0.5 % as 3 + 2, up to 14 %
// or beyond f16's range as one group.  The caller chooses: 1 where the result itself is asked for
// ("full": 2), 3 where it is a small change of weights, 1 for matrices that are nearly square.
//
// Numbers: |x|_F bounds every singular value by 1 and the polynomials bound them from there, so every matrix has a
// power-of-two scale, chosen by the caller from those bounds, that puts it into f16's range: 11 bits where
// bf16 has 8, at the same matrix-core rate ("half").  f32 results take two f16 planes, hi + lo, and three products for
// one ("full": 22 bits).  Sums are f32, |x|_F is summed in f64.  ("double", f64 throughout, has kernels of its own.)  Two
// things cost more than all other roundings and are kept apart.  What f16 loses of the diagonals of Q and P, where their
// size is, is an f32 vector beside the matrix and joins each product as a diagonal matrix (rank 8: 0.28 instead of
// 0.85 % off).  And in "half" X has what f16 loses of it as 8-bit floats: in X <- P X the diagonal's share, in f32 on the
// way out, takes it too, as in the directions in which X is small P is a multiple of I (rank 32, 2 + 2 + 1: 0.17 instead
// of 0.63 %).  Momentum is f32.
#include "common.h"
#include "dense_tile.h"
#include "f32_tile.h"
#include "f64_tile.h"
#include <algorithm>
#include <cmath>

namespace mtx {
namespace ns {

using namespace dense;
typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;

// What a stack's matrices share.  Tall (M > N): X is kept as it is, [M][N], and the Gram side is its columns.
struct Shape {
  int M, N, S, L;      // of x; smaller and larger side
  int Mp, Np, Sp;      // padded to 32
  bool tall;
  int64_t xs, ms;      // elements of X and of an S x S matrix, padded
};
static Shape shape_of(int64_t M, int64_t N) {
  Shape s;
  s.M = (int)M;
  s.N = (int)N;
  s.tall = M > N;
  s.S = (int)std::min(M, N);
  s.L = (int)std::max(M, N);
  s.Mp = (int)round_up(M, 32);
  s.Np = (int)round_up(N, 32);
  s.Sp = (int)round_up(s.S, 32);
  s.xs = (int64_t)s.Mp * s.Np;
  s.ms = (int64_t)s.S * s.Sp;
  return s;
}

// A matrix's scales: x 2^e is what X holds of it, `gram` and `x` bring products with it back.
struct Scale {
  float gram, x;
  int e;
  int pad;
};

// ---- |x|_F, with the momentum's update ------------------------------------------------------------------------
struct Source {
  const void* g;      // gradient, or x itself
  int64_t g_batch, g_row;
  float* m;           // momentum or nullptr
  int64_t m_batch, m_row;
  float beta, rest;   // rest: 1 - beta, which beta in f32 would not give to f32 accuracy
  int nesterov;
};
// Eight consecutive elements of what is orthogonalised, from column c (those past N zero).  FIRST: also the momentum's
// update m <- beta m + (1 - beta) g; otherwise m has it already.
template <typename T, bool VEC, bool FIRST>
__device__ __forceinline__ void load_update(const Source& s, int64_t e, int64_t r, int c, int N, float u[8]) {
  const T* g = (const T*)s.g + e * s.g_batch + r * s.g_row;
  float* m = s.m ? s.m + e * s.m_batch + r * s.m_row : nullptr;
  float gv[8], mv[8];
  if constexpr (VEC) {
    ld8(g, c, gv);
    if (m) ld8(m, c, mv);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      gv[q] = c + q < N ? gld<T>(g, c + q) : 0.0f;
      mv[q] = m && c + q < N ? m[c + q] : 0.0f;
    }
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if (!m) {
      u[q] = gv[q];
      continue;
    }
    if (FIRST) mv[q] = s.beta * mv[q] + s.rest * gv[q];
    u[q] = s.nesterov ? s.rest * gv[q] + s.beta * mv[q] : mv[q];
  }
  if (FIRST && m) {
    if constexpr (VEC) {
      st8(m, c, mv);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (c + q < N) m[c + q] = mv[q];
    }
  }
}
// The workgroups of matrix e leave f64 sums of their rows' squares in part[e][blockIdx.x].  A pass over x bound by memory:
// 128 x 768 x 2048 in bf16 90 us, 4.5 TB/s.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void norm_kernel(Source s, int M, int N, int rows, double* __restrict__ part) {
  __shared__ double w[4];
  const int64_t e = blockIdx.y;
  const int nc = (N + 7) / 8, r0 = blockIdx.x * rows, n = max(0, min(rows, M - r0)) * nc;
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) {
    float u[8];
    load_update<T, VEC, true>(s, e, r0 + i / nc, i % nc * 8, N, u);
#pragma unroll
    for (int q = 0; q < 8; ++q) sum += (double)u[q] * (double)u[q];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) part[e * gridDim.x + blockIdx.x] = (w[0] + w[1]) + (w[2] + w[3]);
}
// Eight e5m2 values (an f16 with two bits of mantissa, so of the same range) and back.
__device__ __forceinline__ uint64_t pack8(const float v[8]) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int x = __builtin_amdgcn_cvt_pk_bf8_f32(v[4 * h], v[4 * h + 1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(v[4 * h + 2], v[4 * h + 3], x, true);
  }
  return (uint64_t)w[0] | ((uint64_t)w[1] << 32);
}
__device__ __forceinline__ void unpack8(uint64_t p, float v[8]) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)(p >> (32 * h));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_bf8(w, false), b = __builtin_amdgcn_cvt_pk_f32_bf8(w, true);
    v[4 * h] = a[0];
    v[4 * h + 1] = a[1];
    v[4 * h + 2] = b[0];
    v[4 * h + 3] = b[1];
  }
}
// |x|_F: the workgroup adds the parts of matrix e, in the same order in each.
__device__ __forceinline__ double norm_of(const double* __restrict__ part, int64_t e, int nparts) {
  __shared__ double w[4];
  double sum = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) sum += part[e * nparts + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  return sqrt((w[0] + w[1]) + (w[2] + w[3]));
}
// X = x 2^e in f16; beside it either what that loses as 8-bit floats or the lo plane and what f32 holds beyond it (a bit
// at most: the steps carry it up by a^5 where x is singular); zeros past the last row and column, with e such that |x|_F + eps
// comes to [2^13, 2^14): a bf16 x is held exactly but for elements below 2^-27 of its norm.  Every workgroup adds the
// parts of its matrix in the same order.  Bound by memory: 128 x 768 x 2048 in bf16 148 us, 5.4 TB/s.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void convert_kernel(Source s, int M, int N, int Mp, int Np, int rows,
                                                      const double* __restrict__ part, int nparts, float eps,
                                                      f16* __restrict__ X, f16* __restrict__ Xlo,
                                                      f16* __restrict__ Xrest, uint64_t* __restrict__ Xlo8,
                                                      Scale* scales) {
  const int64_t e = blockIdx.y;
  const double norm = norm_of(part, e, nparts) + (double)eps;
  const bool fine = norm <= 1e300;  // NaN, infinity: the result is NaN
  const int ex = fine ? 13 - ilogb(norm) : 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const float x = fine ? (float)(1.0 / ldexp(norm, ex)) : __builtin_nanf("");
    scales[e] = Scale{x * x, x, ex, 0};
  }
  const int nc = Np / 8, r0 = blockIdx.x * rows, n = max(0, min(rows, Mp - r0)) * nc;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int r = r0 + i / nc, c = i % nc * 8;
    float u[8] = {};
    if (r < M && c < N) load_update<T, VEC, false>(s, e, r, c, N, u);
    f16x8 hi, lo, rest;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float v = ldexpf(u[q], ex);
      hi[q] = (f16)v;
      lo[q] = (f16)(v - (float)hi[q]);
      rest[q] = (f16)(v - (float)hi[q] - (float)lo[q]);
    }
    const int64_t at = e * Mp * (int64_t)Np + (int64_t)r * Np + c;
    *(f16x8*)(X + at) = hi;
    if (Xlo8) {
      float l[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) l[q] = (float)lo[q];
      Xlo8[at / 8] = pack8(l);
    }
    if (Xlo) {
      *(f16x8*)(Xlo + at) = lo;
      *(f16x8*)(Xrest + at) = rest;
    }
  }
}

// ---- symmetric S x S products ----------------------------------------------------------------------------------
// out = s_acc (U V + diagonal terms) + d0 I.  The diagonal terms are diag(row) V + U diag(col), or w V.  With `full`,
// the f32 diagonal goes there, in true units, and what the matrix loses of it to `rest`, in the matrix's.
struct Sym {
  const f16 *u, *v;
  f16* out;
  float *full, *rest;
  const float *row, *col;
  float s_acc, d0, s_out;  // s_acc: everything to out's units; d0 in true units
};
struct SymArgs {
  Sym p[2];             // problems of one launch (the same sizes)
  int np, E, S, Sp, K;  // K: reduction
  float w_hi, w_lo;
  int64_t ld;           // of u and v
  int64_t in_batch, in_plane, out_batch, out_plane;  // elements from matrix to matrix, and from hi to lo plane
  const Scale* scales;  // Gram product of the first X: multiplies s_acc; or nullptr
};

template <class T, bool TWO>
__device__ __forceinline__ void sym_out(const SymArgs& a, const Sym& p, int64_t e, int m0, int n0,
                                        const f32x16 (&acc)[T::TM][T::TN], char* lds) {
  constexpr int TN = T::TN, PL = TWO ? 2 : 1;
  static_assert(T::NW * PL * T::OUT16_BYTES <= T::LDS_BYTES, "staging fits the ring");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, frow = lane & 31, h = lane >> 5;
  char* mine = lds + wave * (PL * T::OUT16_BYTES);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), wc = n0 + (wave % T::WN) * (TN * 32);
  const int S = a.S, Sp = a.Sp;
  const float k = p.s_acc * (a.scales ? a.scales[e].gram : 1.0f);
  f16* out = p.out + e * a.out_batch;
  const bool edge = m0 + T::BM > S || n0 + T::BN > S;
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    const int r = wr + i * 32 + frow;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      float y[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) y[v] = acc[i][j][v] * k;  // column wc + 32 j + 8 (v / 4) + 4 h + v % 4
      if (edge) {
#pragma unroll
        for (int v = 0; v < 16; ++v) y[v] = r < S && wc + j * 32 + 8 * (v / 4) + 4 * h + v % 4 < S ? y[v] : 0.0f;
      }
      static_assert(T::TM == TN, "a wave's part that the diagonal crosses has it in its blocks i = j");
      if (i == j && wr == wc && p.full) {
        // the lane that has the diagonal's element of its row: 8 (v / 4) + 4 h + v % 4 = r % 32
        const int at = ((frow >> 2) & 1) == h ? (frow >> 3) * 4 + (frow & 3) : -1;
        float d = 0.0f;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          if (v == at) d = y[v] += r < S ? p.d0 * p.s_out : 0.0f;
        }
        if (at >= 0 && r < Sp) {
          const f16 hi = (f16)d, lo = (f16)(d - (float)hi);
          p.full[e * Sp + r] = d / p.s_out;
          p.rest[e * Sp + r] = TWO ? d - (float)hi - (float)lo : d - (float)hi;
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f16x4 hi = {(f16)y[4 * g], (f16)y[4 * g + 1], (f16)y[4 * g + 2], (f16)y[4 * g + 3]};
        char* to = mine + T::out16_off(frow, j * 4 + g) + 8 * h;
        *(f16x4*)to = hi;
        if (TWO)
          *(f16x4*)(to + T::OUT16_BYTES) =
              f16x4{(f16)(y[4 * g] - (float)hi[0]), (f16)(y[4 * g + 1] - (float)hi[1]),
                    (f16)(y[4 * g + 2] - (float)hi[2]), (f16)(y[4 * g + 3] - (float)hi[3])};
      }
    }
    __builtin_amdgcn_s_waitcnt(MTX_LGKMCNT0);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int pl = 0; pl < PL; ++pl) {
      const char* from = mine + pl * T::OUT16_BYTES;
      f16* o = out + pl * a.out_plane;
#pragma unroll
      for (int it = 0; it < TN * 2; ++it) {  // whole rows
        const int q = it * 64 + lane, lr = q / (TN * 4), c = wc + q % (TN * 4) * 8, row = wr + i * 32 + lr;
        const u32x4 x = *(const u32x4*)(from + T::out16_off(lr, q % (TN * 4)));
        if (row < S && c < Sp) *(u32x4*)(o + (int64_t)row * Sp + c) = x;
      }
      if (n0 >= m0) continue;
      // the mirrored tile: 16 lanes read 16 columns of eight rows each, turned; 64 contiguous bytes a row of it
#pragma unroll
      for (int it = 0; it < TN * 2; ++it) {
        const int rb = (lane >> 4) * 8, cb = it * 16;
        const int row = wc + cb + (lane & 15), col = wr + i * 32 + rb;
        const int c = cb + 4 * (lane & 3), kr = rb + ((lane & 15) >> 2);
        const s16x4 both[2] = {T::out16_tr(from, kr, c), T::out16_tr(from, kr + 4, c)};
        if (row < S && col < Sp) *(u32x4*)(o + (int64_t)row * Sp + col) = __builtin_bit_cast(u32x4, both);
      }
    }
    __builtin_amdgcn_s_waitcnt(MTX_LGKMCNT0);
    asm volatile("" ::: "memory");
  }
}

// Tile t of the lower triangle, row by row.
__device__ __forceinline__ void lower(int t, int& i, int& j) {
  i = (int)((sqrtf(8.0f * t + 1.0f) - 1.0f) * 0.5f);
  while ((i + 1) * (i + 2) / 2 <= t) ++i;
  while (i * (i + 1) / 2 > t) --i;
  j = t - i * (i + 1) / 2;
}

// One workgroup a tile of the lower triangle, which it also stores mirrored: 128 Gram products of 768 x 2048 take 204 to 214 us,
// 0.96 PFLOP/s of the tiles computed, and 128 products of 768^3 113 to 130 us, 0.64: with 24 ring stages a tile the way out
// (f16 through LDS, once in rows and once turned) is 50 us of it, and the tiles of a CU do not overlap it with products.
// COLS: the reduction runs down u's and v's columns (the Gram product of a tall X); otherwise along their rows.
template <class T, bool COLS, bool TWO, int DIAG>
__global__ __launch_bounds__(T::NT, T::BM == 256 ? 1 : 2) void sym_kernel(SymArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS_BYTES];
  const int nt = (a.S + T::BM - 1) / T::BM, per = nt * (nt + 1) / 2;
  const int t = tile_of(blockIdx.x, a.np * a.E * per);
  if (t < 0) return;
  const int64_t e = t / per % a.E;
  const Sym p = t / per < a.E ? a.p[0] : a.p[1];
  int i, j;
  lower(t % per, i, j);
  const int m0 = i * T::BM, n0 = j * T::BM;
  auto operand = [&](const f16* m, int x0) {
    const f16* at = m + e * a.in_batch + (COLS ? (int64_t)x0 : x0 * a.ld);
    return Operand{{at, at + a.in_plane}, a.ld, (COLS ? a.Sp : a.S) - x0};
  };
  f32x16 acc[T::TM][T::TN];
  const Diagonal dg{p.row ? p.row + e * a.Sp : nullptr, p.col ? p.col + e * a.Sp : nullptr, a.w_hi, a.w_lo, m0, n0, a.S, a.S};
  T::product(operand(p.u, m0), operand(p.v, n0), a.K, lds, acc, &dg);
  __syncthreads();
  sym_out<T, TWO>(a, p, e, m0, n0, acc, lds);
}

// q += b A + a I where c is 0 or too small beside b for the product that squares A to carry b: q holds c A^2, or nothing yet
// (`fresh`).  A thread takes eight columns; a pass over A and Q.
__global__ __launch_bounds__(256) void poly_kernel(const f16* A, f16* q, float* full, float* rest, int S, int Sp, int64_t plane,
                                                   float a, float b, float s_a, float s_q, int fresh, int two) {
  const int64_t e = blockIdx.y, ms = (int64_t)S * Sp;
  const int i = blockIdx.x * 256 + threadIdx.x, r = i / (Sp / 8), c = i % (Sp / 8) * 8;
  if (r >= Sp) return;
  if (r >= S) {
    if (c == 0) full[e * Sp + r] = rest[e * Sp + r] = 0.0f;
    return;
  }
  const int64_t at = e * ms + (int64_t)r * Sp + c;
  const f16x8 h = *(const f16x8*)(A + at), l = two ? *(const f16x8*)(A + plane + at) : f16x8{};
  const f16x8 qh = fresh ? f16x8{} : *(const f16x8*)(q + at), ql = two && !fresh ? *(const f16x8*)(q + plane + at) : f16x8{};
  f16x8 hi, lo;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const bool d = c + k == r;
    float y = (float)qh[k] + (float)ql[k] + (d && !fresh ? rest[e * Sp + r] : 0.0f);
    y += ((float)h[k] + (float)l[k]) * (b * s_q / s_a) + (d ? a * s_q : 0.0f);
    hi[k] = (f16)y;
    lo[k] = (f16)(y - (float)hi[k]);
    if (d) {
      full[e * Sp + r] = y / s_q;
      rest[e * Sp + r] = y - (float)hi[k] - (two ? (float)lo[k] : 0.0f);
    }
  }
  *(f16x8*)(q + at) = hi;
  if (two) *(f16x8*)(q + plane + at) = lo;
}

// Eight f32 values as f16, and what that leaves of them.
__device__ __forceinline__ f16x8 round8(const float y[8]) {
  f16x8 h;
#pragma unroll
  for (int q = 0; q < 8; ++q) h[q] = (f16)y[q];
  return h;
}
__device__ __forceinline__ f16x8 rest8(const float y[8], const f16x8& h) {
  f16x8 l;
#pragma unroll
  for (int q = 0; q < 8; ++q) l[q] = (f16)(y[q] - (float)h[q]);
  return l;
}

// ---- X <- P X (tall: X P) ----------------------------------------------------------------------------------------
enum { OUT_X = 0, OUT_STORE = 1, OUT_STEP = 2 };
struct ApplyArgs {
  const f16* p;
  const float *pd, *pr;  // P's diagonal, and what the matrix has lost of it
  const f16* x;
  const void* xl;    // what x lacks: "half" 8-bit floats, "full" (the first x) f16; or nullptr
  f16* xo;           // OUT_X: hi plane, and in "full" behind it lo
  uint64_t* xol;     // OUT_X in "half": what hi lacks
  void* out;         // OUT_STORE: the result; OUT_STEP: the weights
  int64_t out_batch, out_row;
  int dtype, vec;    // of out; whether its rows are 16-byte aligned
  Shape s;
  int E;
  int64_t p_plane, x_plane;
  float s_p, s_x;    // undo the scales of p and x; x of the first group: from `scales` instead
  const Scale* scales;
  float s_out;       // OUT_X: the new scale
  float lr, decay, factor;
  const float* lr_dev;
};
// One workgroup a tile of X, the diagonal's share, the scale and the optimiser's step on its way out.  Long reductions
// are bound by the matrix cores (2048 x 7168: 1.04 PFLOP/s), 128 x 768 x 2048 by both: 450 to 570 us, 330 of them products,
// the rest 1.2 GB of X and what it lacks, read and written while the CU's matrix cores wait.  What the way out reads is loaded
// a block of 32 rows ahead; with the old weights and X's lost part as the accumulators' start the kernel took 1.4 times as long.
// D: the type of what is stored or stepped.
template <class T, bool TALL, bool TWO, int OUT, typename D>
__global__ __launch_bounds__(T::NT, T::BM == 256 ? 1 : 2) void apply_kernel(ApplyArgs a) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS_BYTES];
  const Shape s = a.s;
  const int nm = (s.Mp + T::BM - 1) / T::BM, nn = (s.Np + T::BN - 1) / T::BN, per = nm * nn;
  const int t = tile_of(blockIdx.x, a.E * per);
  if (t < 0) return;
  const int64_t e = t / per;
  // the S side inside, so that neighbours share the strip of X
  const int m0 = (TALL ? t % per / nn : t % per % nm) * T::BM, n0 = (TALL ? t % per % nn : t % per / nm) * T::BN;
  const f16 *P = a.p + e * s.ms, *X = a.x + e * s.xs;
  const f16 *pa = TALL ? X + (int64_t)m0 * s.Np : P + (int64_t)min(m0, s.S - 1) * s.Sp;
  const f16 *pb = TALL ? P + (int64_t)min(n0, s.S - 1) * s.Sp : X + n0;
  // rows of the padding past S only: one row of P is read again, and zeros are stored
  const Operand oa{{pa, pa + (TALL ? a.x_plane : a.p_plane)}, TALL ? s.Np : s.Sp, TALL ? s.Mp - m0 : max(s.S - m0, 1)};
  const Operand ob{{pb, pb + (TALL ? a.p_plane : a.x_plane)}, TALL ? s.Sp : s.Np, TALL ? max(s.S - n0, 1) : s.Np - n0};
  f32x16 acc[T::TM][T::TN];
  const float* pr = a.pr + e * s.Sp;
  const Diagonal dg{TALL ? nullptr : pr, TALL ? pr : nullptr, 0.0f, 0.0f, m0, n0, TALL ? s.M : s.S, TALL ? s.S : s.N};
  T::product(oa, ob, s.Sp, lds, acc, &dg);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  char* mine = T::out_lds(lds);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), wc = n0 + (wave % T::WN) * (T::TN * 32);
  const float s_x = a.scales ? a.scales[e].x : a.s_x, s_acc = s_x * a.s_p;
  const float* pd = a.pd + e * s.Sp;
  const float lr = OUT == OUT_STEP ? (a.lr_dev ? *a.lr_dev : a.lr) : 0.0f;
  typedef typename std::conditional<TWO, f16x8, uint64_t>::type Lack;  // eight elements of what x lacks
  const Lack* xl = a.xl ? (const Lack*)a.xl + e * (s.xs / 8) : nullptr;
  const int c = wc + T::out_col(0);
  constexpr int DV = sizeof(D) / 2;  // 16-byte pieces of eight D
  constexpr int AHEAD = T::TN == 4 && OUT == OUT_STEP && DV == 2 ? 1 : 2;  // blocks of rows in registers
  Lack lack[AHEAD][T::OUT_STEPS];
  u32x4 old[AHEAD][OUT == OUT_STEP ? T::OUT_STEPS : 1][DV];  // the weights before the step
  D* out = OUT == OUT_X ? nullptr : (D*)a.out + e * a.out_batch;
  const bool vec = a.vec;
  auto ahead = [&](int i) {
    if (OUT == OUT_STEP && vec) {
#pragma unroll
      for (int it = 0; it < T::OUT_STEPS; ++it) {
        const D* w = out + (int64_t)min(wr + i * 32 + T::out_row(it), s.M - 1) * a.out_row + min(c, s.N - 8);
#pragma unroll
        for (int d = 0; d < DV; ++d) old[i % AHEAD][it][d] = ((const u32x4*)w)[d];
      }
    }
    if (xl) {
#pragma unroll
      for (int it = 0; it < T::OUT_STEPS; ++it)
        lack[i % AHEAD][it] = xl[((int64_t)min(wr + i * 32 + T::out_row(it), s.Mp - 1) * s.Np + min(c, s.Np - 8)) / 8];
    }
  };
  float dc[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) dc[q] = 0.0f;
  if (TALL) ld8(pd, min(c, s.Sp - 8), dc);
  ahead(0);
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    if (AHEAD == 2 && i + 1 < T::TM) ahead(i + 1);
    if (AHEAD == 1 && i > 0) ahead(i);
    T::put(acc[i], mine);
#pragma unroll
    for (int it = 0; it < T::OUT_STEPS; ++it) {
      const int r = wr + i * 32 + T::out_row(it);
      float y[8];
      T::get(mine, it, y);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] *= s_acc;
      if (xl) {
        const float dr = TALL ? 0.0f : pd[min(r, s.Sp - 1)];
        float l[8];
        if constexpr (TWO) {
#pragma unroll
          for (int q = 0; q < 8; ++q) l[q] = (float)lack[i % AHEAD][it][q];
        } else {
          unpack8(lack[i % AHEAD][it], l);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) y[q] = __builtin_fmaf(l[q], (TALL ? dc[q] : dr) * s_x, y[q]);
      }
      if (r >= (OUT == OUT_X ? s.Mp : s.M) || c >= (OUT == OUT_X ? s.Np : s.N)) continue;
      if constexpr (OUT == OUT_X) {
        if (r >= s.M || c + 8 > s.N) {
#pragma unroll
          for (int q = 0; q < 8; ++q) y[q] = r < s.M && c + q < s.N ? y[q] : 0.0f;
        }
        const int64_t at = e * s.xs + (int64_t)r * s.Np + c;
#pragma unroll
        for (int q = 0; q < 8; ++q) y[q] *= a.s_out;
        const f16x8 hi = round8(y);
        *(f16x8*)(a.xo + at) = hi;
        if constexpr (TWO) {
          *(f16x8*)(a.xo + a.x_plane + at) = rest8(y, hi);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) y[q] -= (float)hi[q];
          a.xol[at / 8] = pack8(y);
        }
      } else {
        D* o = out + (int64_t)r * a.out_row + c;
        if constexpr (OUT == OUT_STEP) {
          float w[8];
          if (vec) {
            ld8((const D*)old[i % AHEAD][it], 0, w);
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) w[q] = c + q < s.N ? gld<D>(o, q) : 0.0f;
          }
#pragma unroll
          for (int q = 0; q < 8; ++q) y[q] = w[q] * (1.0f - lr * a.decay) - lr * a.factor * y[q];
        }
        if (vec) {
          store8(o, y);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (c + q < s.N) gst<D>(o, q, y[q]);
        }
      }
    }
  }
}

// ---- S <= 128: the Gram product and all S x S products of a group in one workgroup --------------------------------
// Between launches such products wait for memory and for each other, 5 to 9 us apiece for 2 of work.  Here one workgroup
// takes a matrix from X to P, a chain of up to eight products that each wait for the one before: A and P stay in its
// registers in f32, the operands of a product in LDS in two f16 planes, in "half" too, as the products cost little.  Two
// slots of 64 KB: Q, and in turn A, T and P.  8 x 128 x 512 in "full": 6 launches and 107 us, 43 a group of three steps here,
// where products by themselves take 26 launches and 124; 64 x 128 x 1408 210 against 237, 1 x 64 x 256 80 against 88.
// "half" is level (84 and 82, 135 and 134, 69 and 68) with f32 accuracy in between and a quarter of the launches.
constexpr int kChainS = 128;
struct ChainArgs {
  const f16* x;
  SymArgs m;             // of P: out's layout (p[0].out, full, rest), E, S, Sp; and scales
  int K;                 // reduction of the Gram product
  int64_t ld, x_batch, x_plane;
  float x_undo;          // undoes the scale of x (squared); the first x: from m.scales
  int steps;
  float sched[3][9];
};
template <class T, bool TWO>
__global__ __launch_bounds__(256, 1) void chain_kernel(ChainArgs a) {
  constexpr int SLOT = kChainS * kChainS * 4;  // two planes
  __shared__ __attribute__((aligned(1024))) char lds[2 * SLOT];
  static_assert(T::BM == kChainS && T::BN == kChainS && T::LDS_BYTES <= 2 * SLOT, "one tile");
  const int64_t e = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, frow = lane & 31, h = lane >> 5;
  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64, S = a.m.S;
  constexpr bool COLS = T::cols;
  f32x16 A[2][2], P[2][2], acc[2][2];
  {
    const f16* x = a.x + e * a.x_batch;
    const Operand o{{x, x + a.x_plane}, a.ld, COLS ? a.m.Sp : S};
    T::product(o, o, a.K, lds, acc);
    __syncthreads();
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) f(i, j, v, wr + i * 32 + frow, wc + j * 32 + 8 * (v / 4) + 4 * h + v % 4);
  };
  const float gram = a.m.scales ? a.m.scales[e].gram : a.x_undo;
  each([&](int i, int j, int v, int r, int c) { A[i][j][v] = r < S && c < S ? acc[i][j][v] * gram : 0.0f; });
  char* const slot[2] = {lds, lds + SLOT};
  auto at = [&](int r, int c16) { return r * 256 + ((c16 ^ (r & 15)) << 4); };
  auto put = [&](char* to, const f32x16 (&m)[2][2], float scale) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f16x4 hi, lo;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float y = m[i][j][4 * g + q] * scale;
            hi[q] = (f16)y;
            lo[q] = (f16)(y - (float)hi[q]);
          }
          char* p = to + at(wr + i * 32 + frow, (wc + j * 32) / 8 + g) + 8 * h;
          *(f16x4*)p = hi;
          *(f16x4*)(p + SLOT / 2) = lo;
        }
  };
  // acc = u v, symmetric, all workgroup; reads end before the next barrier
  const int steps16 = (S + 15) / 16;
  auto multiply = [&](const char* u, const char* v) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0f;
    if (wr >= S || wc >= S) return;
    // the next 16 elements' operands are read while these are multiplied
    f16x8 fu[2][2][2], fv[2][2][2];
    auto read = [&](int b, int k) {
#pragma unroll
      for (int pl = 0; pl < 2; ++pl)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          fu[b][pl][i] = *(const f16x8*)(u + pl * (SLOT / 2) + at(wr + i * 32 + frow, 2 * k + h));
          fv[b][pl][i] = *(const f16x8*)(v + pl * (SLOT / 2) + at(wc + i * 32 + frow, 2 * k + h));
        }
    };
    auto use = [&](int b) {
#pragma unroll
      for (int t = 0; t < 3; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = F16::mfma(fv[b][t == 1][j], fu[b][t == 2][i], acc[i][j]);
    };
    read(0, 0);
    for (int k = 0; k < steps16; k += 2) {
      read(1, min(k + 1, 7));
      use(0);
      read(0, min(k + 2, 7));
      if (k + 1 < steps16) use(1);
    }
  };
  put(slot[0], A, a.sched[0][3]);
  __syncthreads();
  for (int n = 0; n < a.steps; ++n) {
    const float* c = a.sched[n];
    const float sA = c[3], sQ = c[4], sT = c[5];
    const bool last = n + 1 == a.steps;
    multiply(slot[0], slot[0]);  // A A
    const float k2 = c[2] / (sA * sA);
    each([&](int i, int j, int v, int r, int cc) {
      acc[i][j][v] = k2 * acc[i][j][v] + c[1] * A[i][j][v] + (r == cc && r < S ? c[0] : 0.0f);
    });
    put(slot[1], acc, sQ);
    if (n == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) P[i][j] = acc[i][j];
    }
    __syncthreads();
    if (!last) {
      multiply(slot[1], slot[0]);  // T = Q A
      const float kt = sT / (sQ * sA);
      each([&](int i, int j, int v, int, int) { acc[i][j][v] *= kt; });
      __syncthreads();
      put(slot[0], acc, 1.0f);
      __syncthreads();
      multiply(slot[1], slot[0]);  // the next A = Q T
      const float ka = 1.0f / (sQ * sT);
      each([&](int i, int j, int v, int, int) { A[i][j][v] = acc[i][j][v] * ka; });
      __syncthreads();
    }
    if (n > 0) {
      const float sP = a.sched[n - 1][6];
      put(slot[0], P, sP);
      __syncthreads();
      multiply(slot[1], slot[0]);  // P = Q P
      const float kp = 1.0f / (sQ * sP);
      each([&](int i, int j, int v, int, int) { P[i][j][v] = acc[i][j][v] * kp; });
      __syncthreads();
    }
    if (!last) {
      put(slot[0], A, a.sched[n + 1][3]);
      __syncthreads();
    }
  }
  SymArgs m = a.m;
  m.scales = nullptr;
  sym_out<T, TWO>(m, m.p[0], e, 0, 0, P, lds);
}

// ---- the chain of launches ---------------------------------------------------------------------------------------
template <bool A, bool B, bool TWO, int DIAG> using Big = Tile<F16, 4, 4, 2, 2, 4, A, B, false, TWO, DIAG>;
template <bool A, bool B, bool TWO, int DIAG> using Small = Tile<F16, 2, 2, 2, 2, 4, A, B, false, TWO, DIAG>;
template <bool A, bool B, bool TWO, int DIAG> using Least = Tile<F16, 1, 1, 2, 2, 8, A, B, false, TWO, DIAG>;

// Whether a launch takes its `big` tiles of 256 x 256, one a CU, rather than `small` ones of 128 x 128, two a CU.  A round of
// small ones takes 0.7 of one of big ones, and a last round that is not full costs about half of what it lacks, but
// one is always paid whole.  Symmetric products, big against small: 16 x 1408 (336, 1056 tiles) 97, 80 us; 24 x 1024
// (240, 864) 46, 54; 10 x 1024 (100, 360) 35, 25; 128 x 768 (768, 2688) 122, 142.  X <- P X: 12 x 2048 x 1408 (576, 2112)
// 152, 167; 1 x 2048 x 7168 (224, 896) 70, 82.
static bool takes_big(int64_t S, int64_t big, int64_t small) {
  const double rounds = big / 256.0, cost = std::max(1.0, 0.5 * (rounds + std::ceil(rounds)));
  return S >= 256 && cost <= 0.7 * std::max(1.0, small / 512.0);
}

// Where all tiles of 64 x 64 find a place at once, two a CU, it is one tile's chain of stages and its way out that count, and the
// smallest is the quickest: 1 x 1024 (136 of them, 36 of 128 x 128) 9 us against 13 and its Gram product with 4096 20
// against 35, 8 x 256 in two planes 8 against 13; with more than that 1 x 2048 (528, 136) 28 against 22.  X <- P X likewise: 8 x 128 x
// 512 in two planes, five steps with two of them, 107 us against 113.
constexpr int64_t kLeastTiles = 512;

template <bool COLS, bool TWO, int DIAG>
static int launch_sym(const SymArgs& a, hipStream_t st) {
  auto tiles = [&](int b) { const int64_t n = ceil_div(a.S, b); return a.np * a.E * (n * (n + 1) / 2); };
  if (tiles(64) <= kLeastTiles)
    hipLaunchKernelGGL((sym_kernel<Least<COLS, COLS, TWO, DIAG>, COLS, TWO, DIAG>), dim3((unsigned)tiles_grid(tiles(64))),
                       dim3(256), 0, st, a);
  else if (takes_big(a.S, tiles(256), tiles(128)))
    hipLaunchKernelGGL((sym_kernel<Big<COLS, COLS, TWO, DIAG>, COLS, TWO, DIAG>), dim3((unsigned)tiles_grid(tiles(256))),
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((sym_kernel<Small<COLS, COLS, TWO, DIAG>, COLS, TWO, DIAG>), dim3((unsigned)tiles_grid(tiles(128))),
                       dim3(256), 0, st, a);
  return check_launch();
}
template <bool TALL, bool TWO>
static int launch_chain(const ChainArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((chain_kernel<Small<TALL, TALL, TWO, DIAG_NONE>, TWO>), dim3((unsigned)a.m.E), dim3(256), 0, st, a);
  return check_launch();
}
template <bool TALL, bool TWO, int OUT, typename D>
static int launch_apply_out(const ApplyArgs& a, hipStream_t st) {
  auto tiles = [&](int b) { return a.E * ceil_div(a.s.Mp, b) * ceil_div(a.s.Np, b); };
  if (tiles(64) <= kLeastTiles)
    hipLaunchKernelGGL((apply_kernel<Least<false, !TALL, TWO, DIAG_VECTORS>, TALL, TWO, OUT, D>),
                       dim3((unsigned)tiles_grid(tiles(64))), dim3(256), 0, st, a);
  else if (takes_big(a.s.S, tiles(256), tiles(128)))
    hipLaunchKernelGGL((apply_kernel<Big<false, !TALL, TWO, DIAG_VECTORS>, TALL, TWO, OUT, D>), dim3((unsigned)tiles_grid(tiles(256))),
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((apply_kernel<Small<false, !TALL, TWO, DIAG_VECTORS>, TALL, TWO, OUT, D>), dim3((unsigned)tiles_grid(tiles(128))),
                       dim3(256), 0, st, a);
  return check_launch();
}
template <bool TALL, bool TWO>
static int launch_apply(int out, const ApplyArgs& a, hipStream_t st) {
  if (out == OUT_X) return launch_apply_out<TALL, TWO, OUT_X, uint16_t>(a, st);
  if (a.dtype == MTX_F32)
    return out == OUT_STORE ? launch_apply_out<TALL, TWO, OUT_STORE, float>(a, st)
                            : launch_apply_out<TALL, TWO, OUT_STEP, float>(a, st);
  return out == OUT_STORE ? launch_apply_out<TALL, TWO, OUT_STORE, uint16_t>(a, st)
                          : launch_apply_out<TALL, TWO, OUT_STEP, uint16_t>(a, st);
}

// f64: tiles of 64 x 64 from three a CU on, of 32 x 32 below, which fill the chip more evenly (4 x 768 x 768, 576 of the large
// ones in X <- Q X: 975 us against 1050; with 256 as the bound 4 x 768 x 768 took 1340 where 512 took 1130).
constexpr int64_t kTiles64 = 768;

// Workgroups of a matrix in the norm and conversion launches: 2048 in all (half or twice as many: the same within 2 %).
static int64_t parts_of(int64_t E, const Shape& s) {
  const int64_t by_size = std::max<int64_t>(1, s.xs / 8192);
  return std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(by_size, s.Mp), std::min<int64_t>(512, ceil_div(2048, E))));
}

// The workspace that matrices of one chain share: 64 x 2048 x 7168 takes 26.3 ms with 16 GiB, 26.7 with 4, 30.6 with 1 and 35.8
// with a quarter, as fewer tiles fill a launch's last round.
constexpr int64_t kChunkBytes = (int64_t)4 << 30;
// bytes an element of X takes: the first, with what it lacks, and the second
static int64_t x_bytes(int planes) { return planes == 2 ? 6 + 4 : 3 + 3; }
static int64_t matrix_bytes(const Shape& s, int planes) {
  if (planes == MTX_NS_F64) return 16 * ((int64_t)s.M * s.N + (int64_t)s.S * s.S) + 512 * 8;
  return x_bytes(planes) * s.xs + 10 * s.ms * planes + 7 * round_up((int64_t)s.Sp * 4, 256) + 1024 * 8 + 256;
}
static int64_t chunk_of(int64_t E, const Shape& s, int planes) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(E, kChunkBytes / matrix_bytes(s, planes)));
  return ceil_div(E, ceil_div(E, most));
}
static int64_t workspace_bytes(int64_t E, const Shape& s, int planes) {
  const int64_t n = chunk_of(E, s, planes);
  int64_t b = 0;
  b += round_up(n * 512 * 8, 256);                        // partial sums
  if (planes == MTX_NS_F64)                                // X, twice, A and Q
    return b + 2 * round_up(n * s.M * (int64_t)s.N * 8, 256) + 2 * round_up(n * s.S * (int64_t)s.S * 8, 256);
  b += round_up(n * (int64_t)sizeof(Scale), 256);
  b += 6 * round_up(n * s.Sp * 4, 256);                    // diagonals, and what the matrices lose of them
  for (const int64_t x : {2 * planes, planes == 2 ? 2 : 1, 2 * planes, planes == 2 ? 0 : 1})
    b += round_up(n * s.xs * x, 256);                      // X, twice, and what it lacks
  b += 5 * round_up(n * s.ms * 2 * planes, 256);          // A, T and three of Q and P
  return b;
}

// ---- float64 ------------------------------------------------------------------------------------------------------
// Two f16 planes hold 22 bits and f32 sums add 2^-24 of their terms, which the steps carry up by a^5 where x is singular:
// float32 results in "full" end as far off as f32 products do, 2e-6 at full rank, 3e-5 at rank 32 of 768, 1e-4 at rank 1.
// Here everything is f64, step by step: a Gram product, Q = a I + b A + c A^2, X <- Q X (tall: X Q).  Small stacks are bound by
// their 17 launches of 6 to 13 us (8 x 128 x 512: 145 us; "full" 108), large ones by the f64 matrix cores (12 x 768 x 640:
// 1.7 ms, "full" 0.47).
struct Step64 {
  const double *u, *v;  // X or A; X in the last product of a step: u (tall) or v
  double* out;
  double a, b, c;
  Shape s;
  int E, K;             // K: reduction
  int64_t ld;           // sym: of u and v, where their rows are reduced
};
struct Out64 {  // the last step's: the result or the weights
  void* out;
  int64_t batch, row;
  int dtype, step;
  float lr, decay, factor;
  const float* lr_dev;
};
// X = x / (|x|_F + eps), dense [M][N].
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void convert64_kernel(Source s, int M, int N, int rows, const double* __restrict__ part,
                                                        int nparts, float eps, double* __restrict__ X) {
  const int64_t e = blockIdx.y;
  const double norm = norm_of(part, e, nparts) + (double)eps;
  const bool fine = norm <= 1e300;
  const int nc = (N + 7) / 8, r0 = blockIdx.x * rows, n = max(0, min(rows, M - r0)) * nc;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int r = r0 + i / nc, c = i % nc * 8;
    float u[8];
    load_update<T, VEC, false>(s, e, r, c, N, u);
    double* to = X + (e * M + r) * N + c;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (c + q < N) to[q] = fine ? (double)u[q] / norm : __builtin_nan("");
  }
}
// out = c U V^T + b U + a I, S x S and symmetric: a tile of the lower triangle, stored mirrored too.  COLS: c U^T V.
template <int BT, int KS, bool COLS>
__global__ __launch_bounds__(f64mm::NT) void sym64_kernel(Step64 p) {
  typedef f64mm::Tile<BT, KS> T;
  __shared__ __attribute__((aligned(16))) double lds[T::LDS];
  const int S = p.s.S, nt = (S + BT - 1) / BT, per = nt * (nt + 1) / 2;
  const int t = dense::tile_of(blockIdx.x, p.E * per);
  if (t < 0) return;
  const int64_t e = t / per, ld = COLS ? S : p.ld, size = COLS ? (int64_t)S * p.K : S * p.ld;
  int i, j;
  lower(t % per, i, j);
  const int m0 = i * BT, n0 = j * BT;
  const double *u = p.u + e * size, *v = p.v + e * size;
  f64mm::f64x4 acc[T::TB][T::TB];
  T::template product<!COLS, !COLS>({COLS ? u + m0 : u + m0 * ld, ld, S - m0}, {COLS ? v + n0 : v + n0 * ld, ld, S - n0},
                                    p.K, lds, acc);
  double* out = p.out + e * S * (int64_t)S;
  T::each(acc, [&](int r, int c, double y) {
    const int64_t row = m0 + r, col = n0 + c;
    if (row >= S || col >= S) return;
    y *= p.c;
    if (p.b != 0.0) y += p.b * u[row * ld + col];
    if (row == col) y += p.a;
    out[row * S + col] = y;
    if (n0 < m0) out[col * S + row] = y;
  });
}
// A tile of X <- Q X (tall: X Q); LAST: to the result or the weights.
template <int BT, int KS, bool TALL, bool LAST>
__global__ __launch_bounds__(f64mm::NT) void apply64_kernel(Step64 p, Out64 o) {
  typedef f64mm::Tile<BT, KS> T;
  __shared__ __attribute__((aligned(16))) double lds[T::LDS];
  const int S = p.s.S, M = p.s.M, N = p.s.N, nm = (M + BT - 1) / BT, nn = (N + BT - 1) / BT, per = nm * nn;
  const int t = dense::tile_of(blockIdx.x, p.E * per);
  if (t < 0) return;
  const int64_t e = t / per, xs = (int64_t)M * N, ms = (int64_t)S * S;
  const int m0 = (TALL ? t % per / nn : t % per % nm) * BT, n0 = (TALL ? t % per % nn : t % per / nm) * BT;
  const double *Q = (TALL ? p.v : p.u) + e * ms, *X = (TALL ? p.u : p.v) + e * xs;
  f64mm::f64x4 acc[T::TB][T::TB];
  if constexpr (TALL) T::template product<true, true>({X + (int64_t)m0 * N, N, M - m0}, {Q + (int64_t)n0 * S, S, S - n0}, S, lds, acc);
  else T::template product<true, false>({Q + (int64_t)m0 * S, S, S - m0}, {X + n0, N, N - n0}, S, lds, acc);
  const double lr = LAST && o.step == OUT_STEP ? (double)(o.lr_dev ? *o.lr_dev : o.lr) : 0.0;
  T::each(acc, [&](int r, int c, double y) {
    const int64_t row = m0 + r, col = n0 + c;
    if (row >= M || col >= N) return;
    if constexpr (!LAST) {
      p.out[e * xs + row * N + col] = y;
    } else {
      const int64_t at = e * o.batch + row * o.row + col;
      if (o.dtype == MTX_F32) {
        float* w = (float*)o.out + at;
        *w = (float)(o.step == OUT_STEP ? *w * (1.0 - lr * o.decay) - lr * o.factor * y : y);
      } else {
        uint16_t* w = (uint16_t*)o.out + at;
        gst<uint16_t>(w, 0, (float)(o.step == OUT_STEP ? bf16_to_f32(*w) * (1.0 - lr * o.decay) - lr * o.factor * y : y));
      }
    }
  });
}

struct Job {
  Source src;
  int gdtype, gvec;
  void* out;
  int dtype, vec;
  int64_t out_batch, out_row;
  int step;                     // OUT_STORE or OUT_STEP
  float lr, decay, factor;
  const float* lr_dev;
};

// sched: 9 floats a step: a, b, c, the scales (powers of two) of A, Q, T, P and X, and whether the step ends its group.
template <bool TALL, bool TWO>
static int run_chunk(const Job& j, int64_t E, const Shape& s, const float* sched, int steps, float eps, char* ws,
                     hipStream_t st) {
  constexpr int planes = TWO ? 2 : 1;  // of the S x S matrices
  auto take = [&](int64_t bytes) { char* p = ws; ws += round_up(bytes, 256); return p; };
  double* part = (double*)take(E * 512 * 8);
  Scale* scales = (Scale*)take(E * (int64_t)sizeof(Scale));
  float *full[3], *rest[3];
  for (auto& d : full) d = (float*)take(E * s.Sp * 4);
  for (auto& d : rest) d = (float*)take(E * s.Sp * 4);
  f16* X[2];
  void* lack[2];
  X[0] = (f16*)take(E * s.xs * 2 * planes);
  lack[0] = take(E * s.xs * planes);
  X[1] = (f16*)take(E * s.xs * 2 * planes);
  lack[1] = TWO ? nullptr : take(E * s.xs);
  f16 *A = (f16*)take(E * s.ms * 2 * planes), *Tm = (f16*)take(E * s.ms * 2 * planes), *Q[3];
  for (auto& q : Q) q = (f16*)take(E * s.ms * 2 * planes);
  const int64_t x_plane = E * s.xs, m_plane = E * s.ms;

  const bool first_lacks = TWO || j.src.m || j.gdtype == MTX_F32;  // in "half" f16 holds a bf16 x as it is
  const int parts = (int)parts_of(E, s);
  const int rows = (int)ceil_div(s.M, parts), rows_p = (int)ceil_div(s.Mp, parts);
  const dim3 grid((unsigned)parts, (unsigned)E);
#define MTX_PREP(T, V)                                                                                              \
  do {                                                                                                              \
    hipLaunchKernelGGL((norm_kernel<T, V>), grid, dim3(256), 0, st, j.src, s.M, s.N, rows, part);                   \
    hipLaunchKernelGGL((convert_kernel<T, V>), grid, dim3(256), 0, st, j.src, s.M, s.N, s.Mp, s.Np, rows_p, part, parts, \
                       eps, X[0], TWO ? X[0] + x_plane : nullptr, TWO ? (f16*)lack[0] : nullptr,                    \
                       !TWO && first_lacks ? (uint64_t*)lack[0] : nullptr, scales);                                 \
  } while (0)
  if (j.gdtype == MTX_F32) {
    if (j.gvec) MTX_PREP(float, true);
    else MTX_PREP(float, false);
  } else {
    if (j.gvec) MTX_PREP(uint16_t, true);
    else MTX_PREP(uint16_t, false);
  }
#undef MTX_PREP
  int rc = check_launch();
  if (rc != MTX_OK) return rc;

  SymArgs m{};
  m.E = (int)E;
  m.S = s.S;
  m.Sp = s.Sp;
  m.out_batch = s.ms;
  m.out_plane = m_plane;
  int cur = 0;          // X of the group
  float x_scale = 0.0f;  // of X; 0: the first, by matrix
  int p = -1;           // Q[p], full[p], rest[p] hold P
  // X <- P X behind step i, which ends its group; P in Q[p]
  auto launch_group_apply = [&](int i, int p) {
    const float sP = sched[9 * i + 6], sX = sched[9 * i + 7];
    ApplyArgs a{};
    a.p = Q[p];
    a.pd = full[p];
    a.pr = rest[p];
    a.x = X[cur];
    a.xl = x_scale == 0.0f ? (first_lacks ? lack[0] : nullptr) : (TWO ? nullptr : lack[cur]);
    a.xo = X[cur ^ 1];
    a.xol = TWO ? nullptr : (uint64_t*)lack[cur ^ 1];
    a.out = j.out;
    a.out_batch = j.out_batch;
    a.out_row = j.out_row;
    a.dtype = j.dtype;
    a.vec = j.vec;
    a.s = s;
    a.E = (int)E;
    a.p_plane = m_plane;
    a.x_plane = x_plane;
    a.s_p = 1.0f / sP;
    a.scales = x_scale == 0.0f ? scales : nullptr;
    a.s_x = x_scale == 0.0f ? 0.0f : 1.0f / x_scale;
    a.s_out = sX;
    a.lr = j.lr;
    a.decay = j.decay;
    a.factor = j.factor;
    a.lr_dev = j.lr_dev;
    const int rc = launch_apply<TALL, TWO>(i + 1 == steps ? j.step : OUT_X, a, st);
    x_scale = sX;
    cur ^= 1;
    return rc;
  };
  for (int i = 0; i < steps; ++i) {
    const float* c = sched + 9 * i;
    const float sA = c[3], sQ = c[4], sT = c[5], sP = c[6];
    const bool ends = c[8] != 0.0f || i + 1 == steps;
    if (s.S <= kChainS && p < 0) {
      // the whole group at once, as far as it is three steps long at most
      int n = 1;
      while (sched[9 * (i + n - 1) + 8] == 0.0f && i + n < steps && n < 4) ++n;
      if (n <= 3) {
        ChainArgs a{};
        a.x = X[cur];
        a.m = m;
        a.m.p[0] = Sym{nullptr, nullptr, Q[0], full[0], rest[0], nullptr, nullptr, sched[9 * (i + n - 1) + 6], 0.0f,
                       sched[9 * (i + n - 1) + 6]};
        a.m.scales = x_scale == 0.0f ? scales : nullptr;
        a.K = TALL ? s.Mp : s.Np;
        a.ld = s.Np;
        a.x_batch = s.xs;
        a.x_plane = x_plane;
        a.x_undo = x_scale == 0.0f ? 0.0f : 1.0f / (x_scale * x_scale);
        a.steps = n;
        for (int k = 0; k < n; ++k)
          for (int q = 0; q < 9; ++q) a.sched[k][q] = sched[9 * (i + k) + q];
        rc = launch_chain<TALL, TWO>(a, st);
        if (rc != MTX_OK) return rc;
        i += n - 1;
        p = 0;
        rc = launch_group_apply(i, 0);
        if (rc != MTX_OK) return rc;
        p = -1;
        continue;
      }
    }
    if (p < 0) {
      SymArgs g = m;
      g.np = 1;
      g.K = TALL ? s.Mp : s.Np;
      g.ld = s.Np;
      g.in_batch = s.xs;
      g.in_plane = x_plane;
      g.scales = x_scale == 0.0f ? scales : nullptr;
      g.p[0] = Sym{X[cur], X[cur], A, nullptr, nullptr, nullptr, nullptr,
                   sA * (x_scale == 0.0f ? 1.0f : 1.0f / (x_scale * x_scale)), 0.0f, sA};
      rc = launch_sym<TALL, TWO, DIAG_NONE>(g, st);
      if (rc != MTX_OK) return rc;
    }
    m.K = s.Sp;
    m.ld = s.Sp;
    m.in_batch = s.ms;
    m.in_plane = m_plane;
    const int q = p < 0 ? 0 : (p + 1) % 3, np = p < 0 ? q : (p + 2) % 3;
    // Q = a I + c (A + (b / c) I) A: the product carries b where f16 holds (b / c) sA
    const float w = c[2] != 0.0f ? c[1] / c[2] * sA : 0.0f;
    const bool carried = c[2] != 0.0f && fabsf(w) <= 60000.0f;
    m.np = 1;
    if (c[2] != 0.0f) {
      m.w_hi = carried ? (float)(f16)w : 0.0f;
      m.w_lo = carried ? w - m.w_hi : 0.0f;
      m.p[0] = Sym{A, A, Q[q], full[q], rest[q], nullptr, nullptr, c[2] / (sA * sA) * sQ, carried ? c[0] : 0.0f, sQ};
      rc = launch_sym<false, TWO, DIAG_CONST>(m, st);
      if (rc != MTX_OK) return rc;
    }
    if (!carried) {
      hipLaunchKernelGGL(poly_kernel, dim3((unsigned)ceil_div((int64_t)s.Sp * (s.Sp / 8), 256), (unsigned)E), dim3(256), 0, st,
                         A, Q[q], full[q], rest[q], s.S, s.Sp, m_plane, c[0], c[1], sA, sQ, c[2] == 0.0f, TWO);
      rc = check_launch();
      if (rc != MTX_OK) return rc;
    }
    // P <- Q P and T = Q A in one launch, then A <- Q T
    m.np = 0;
    if (p >= 0) {
      const float sPp = c[6 - 9];
      m.p[m.np++] = Sym{Q[q], Q[p], Q[np], full[np], rest[np], rest[q], rest[p], sP / (sQ * sPp), 0.0f, sP};
    }
    if (!ends) m.p[m.np++] = Sym{Q[q], A, Tm, nullptr, nullptr, rest[q], nullptr, sT / (sQ * sA), 0.0f, sT};
    if (m.np > 0) {
      rc = launch_sym<false, TWO, DIAG_VECTORS>(m, st);
      if (rc != MTX_OK) return rc;
    }
    p = np;
    if (!ends) {
      const float sA2 = c[3 + 9];
      m.np = 1;
      m.p[0] = Sym{Q[q], Tm, A, nullptr, nullptr, rest[q], nullptr, sA2 / (sQ * sT), 0.0f, sA2};
      rc = launch_sym<false, TWO, DIAG_VECTORS>(m, st);
      if (rc != MTX_OK) return rc;
      continue;
    }
    rc = launch_group_apply(i, p);
    if (rc != MTX_OK) return rc;
    p = -1;
  }
  return MTX_OK;
}

template <bool COLS>
static int launch_sym64(const Step64& p, hipStream_t st) {
  auto tiles = [&](int b) { const int64_t n = ceil_div(p.s.S, b); return p.E * (n * (n + 1) / 2); };
  if (tiles(64) < kTiles64)
    hipLaunchKernelGGL((sym64_kernel<32, 32, COLS>), dim3((unsigned)tiles_grid(tiles(32))), dim3(f64mm::NT), 0, st, p);
  else
    hipLaunchKernelGGL((sym64_kernel<64, 16, COLS>), dim3((unsigned)tiles_grid(tiles(64))), dim3(f64mm::NT), 0, st, p);
  return check_launch();
}
template <bool TALL, bool LAST>
static int launch_apply64(const Step64& p, const Out64& o, hipStream_t st) {
  auto tiles = [&](int b) { return p.E * ceil_div(p.s.M, b) * ceil_div(p.s.N, b); };
  if (tiles(64) < kTiles64)
    hipLaunchKernelGGL((apply64_kernel<32, 32, TALL, LAST>), dim3((unsigned)tiles_grid(tiles(32))), dim3(f64mm::NT), 0, st, p, o);
  else
    hipLaunchKernelGGL((apply64_kernel<64, 16, TALL, LAST>), dim3((unsigned)tiles_grid(tiles(64))), dim3(f64mm::NT), 0, st, p, o);
  return check_launch();
}
// sched: 9 floats a step: a, b, c, and what f32 has lost of each of them.
template <bool TALL>
static int run_chunk64(const Job& j, int64_t E, const Shape& s, const float* sched, int steps, float eps, char* ws,
                       hipStream_t st) {
  auto take = [&](int64_t bytes) { char* p = ws; ws += round_up(bytes, 256); return p; };
  const int64_t xs = (int64_t)s.M * s.N, ms = (int64_t)s.S * s.S;
  double* part = (double*)take(E * 512 * 8);
  double* X[2];
  for (auto& x : X) x = (double*)take(E * xs * 8);
  double *A = (double*)take(E * ms * 8), *Q = (double*)take(E * ms * 8);
  const int parts = (int)parts_of(E, s), rows = (int)ceil_div(s.M, parts);
  const dim3 grid((unsigned)parts, (unsigned)E);
#define MTX_PREP(T, V)                                                                                               \
  do {                                                                                                               \
    hipLaunchKernelGGL((norm_kernel<T, V>), grid, dim3(256), 0, st, j.src, s.M, s.N, rows, part);                    \
    hipLaunchKernelGGL((convert64_kernel<T, V>), grid, dim3(256), 0, st, j.src, s.M, s.N, rows, part, parts, eps, X[0]); \
  } while (0)
  if (j.gdtype == MTX_F32) {
    if (j.gvec) MTX_PREP(float, true);
    else MTX_PREP(float, false);
  } else {
    if (j.gvec) MTX_PREP(uint16_t, true);
    else MTX_PREP(uint16_t, false);
  }
#undef MTX_PREP
  int rc = check_launch();
  const Out64 o{j.out, j.out_batch, j.out_row, j.dtype, j.step, j.lr, j.decay, j.factor, j.lr_dev};
  for (int i = 0; i < steps && rc == MTX_OK; ++i) {
    const float* c = sched + 9 * i;
    double *x = X[i & 1], *next = X[(i + 1) & 1];
    rc = launch_sym64<TALL>(Step64{x, x, A, 0.0, 0.0, 1.0, s, (int)E, s.L, s.L}, st);
    if (rc != MTX_OK) return rc;
    const double c2 = (double)c[2] + c[5];
    rc = launch_sym64<false>(Step64{A, A, Q, (double)c[0] + c[3], (double)c[1] + c[4], c2, s, (int)E, c2 != 0.0 ? s.S : 0, s.S}, st);
    if (rc != MTX_OK) return rc;
    const Step64 a{TALL ? x : Q, TALL ? Q : x, next, 0.0, 0.0, 0.0, s, (int)E, s.S, 0};
    rc = i + 1 == steps ? launch_apply64<TALL, true>(a, o, st) : launch_apply64<TALL, false>(a, o, st);
  }
  return rc;
}

static int run(Job j, int64_t E, int64_t M, int64_t N, const float* sched, int steps, float eps, int planes, void* ws,
               int64_t ws_bytes, hipStream_t st) {
  if (E == 0 || M == 0 || N == 0) return MTX_OK;
  const Shape s = shape_of(M, N);
  if (!ws || (uintptr_t)ws % 256 || ws_bytes < workspace_bytes(E, s, planes)) return MTX_ERR_WORKSPACE;
  const int64_t chunk = chunk_of(E, s, planes);
  const int gsize = dtype_size(j.gdtype), osize = dtype_size(j.dtype);
  for (int64_t e = 0; e < E; e += chunk) {
    Job c = j;
    c.src.g = (const char*)j.src.g + e * j.src.g_batch * gsize;
    if (j.src.m) c.src.m = j.src.m + e * j.src.m_batch;
    c.out = (char*)j.out + e * j.out_batch * osize;
    const int64_t n = std::min(chunk, E - e);
    const int rc = planes == MTX_NS_F64 ? (s.tall ? run_chunk64<true>(c, n, s, sched, steps, eps, (char*)ws, st)
                                                  : run_chunk64<false>(c, n, s, sched, steps, eps, (char*)ws, st))
                   : s.tall ? (planes == 2 ? run_chunk<true, true>(c, n, s, sched, steps, eps, (char*)ws, st)
                                         : run_chunk<true, false>(c, n, s, sched, steps, eps, (char*)ws, st))
                          : (planes == 2 ? run_chunk<false, true>(c, n, s, sched, steps, eps, (char*)ws, st)
                                         : run_chunk<false, false>(c, n, s, sched, steps, eps, (char*)ws, st));
    if (rc != MTX_OK) return rc;
  }
  return MTX_OK;
}

static bool sizes_ok(int64_t E, int64_t M, int64_t N) {
  return E >= 0 && M >= 0 && N >= 0 && E <= 65535 && M <= (1 << 20) && N <= (1 << 20) &&
         std::min(M, N) <= (1 << 15);
}
static bool planes_ok(int planes) { return planes == 1 || planes == 2 || planes == MTX_NS_F64; }
static bool sched_ok(const float* sched, int steps, int planes) {
  if (!sched || steps < 1 || steps > 64) return false;
  for (int i = 0; i < 9 * steps; ++i)
    if (!std::isfinite(sched[i])) return false;
  if (planes == MTX_NS_F64) return true;
  for (int i = 0; i < steps; ++i)
    for (int q = 3; q < 8; ++q)
      if (!(sched[9 * i + q] > 0.0f)) return false;
  return true;
}
// whether rows of `dtype` start on 16-byte boundaries and hold whole chunks of eight
static bool rows_aligned(const void* p, int dtype, int64_t batch, int64_t row, int64_t N) {
  const int64_t n = 16 / dtype_size(dtype);
  return (uintptr_t)p % 16 == 0 && batch % n == 0 && row % n == 0 && N % 8 == 0;
}

}  // namespace ns
}  // namespace mtx

using namespace mtx;

extern "C" int64_t mtx_newton_schulz_workspace_size(int64_t E, int64_t M, int64_t N, int planes) {
  if (!ns::sizes_ok(E, M, N) || !ns::planes_ok(planes)) return -1;
  if (E == 0 || M == 0 || N == 0) return 0;
  return ns::workspace_bytes(E, ns::shape_of(M, N), planes);
}

extern "C" int mtx_newton_schulz(const void* x, int dtype, int64_t E, int64_t M, int64_t N, int64_t x_batch, int64_t x_row,
                                 const float* schedule, int steps, float eps, int planes, void* out, int64_t out_batch,
                                 int64_t out_row, void* workspace, int64_t workspace_bytes, void* stream) {
  if ((dtype != MTX_F32 && dtype != MTX_BF16) || !ns::planes_ok(planes) || !(eps > 0.0f)) return MTX_ERR_ARG;
  if (E < 0 || M < 0 || N < 0 || !ns::sched_ok(schedule, steps, planes)) return MTX_ERR_ARG;
  if (!ns::sizes_ok(E, M, N)) return MTX_ERR_UNSUPPORTED;
  if (x_row < N || out_row < N || x_batch < 0 || out_batch < 0) return MTX_ERR_ARG;
  if (E * M * N > 0 && (!x || !out)) return MTX_ERR_ARG;
  ns::Job j{};
  j.src = ns::Source{x, x_batch, x_row, nullptr, 0, 0, 0.0f, 0.0f, 0};
  j.gdtype = j.dtype = dtype;
  j.gvec = ns::rows_aligned(x, dtype, x_batch, x_row, N);
  j.out = out;
  j.vec = ns::rows_aligned(out, dtype, out_batch, out_row, N);
  j.out_batch = out_batch;
  j.out_row = out_row;
  j.step = ns::OUT_STORE;
  return ns::run(j, E, M, N, schedule, steps, eps, planes, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" int mtx_muon_update(void* param, int param_dtype, int64_t p_batch, int64_t p_row, const void* grad,
                               int grad_dtype, int64_t g_batch, int64_t g_row, float* momentum, int64_t m_batch,
                               int64_t m_row, int64_t E, int64_t M, int64_t N, double beta, int nesterov, float lr,
                               const float* lr_dev, float weight_decay, float factor, const float* schedule, int steps,
                               float eps, int planes, void* workspace, int64_t workspace_bytes, void* stream) {
  if ((param_dtype != MTX_F32 && param_dtype != MTX_BF16) || (grad_dtype != MTX_F32 && grad_dtype != MTX_BF16))
    return MTX_ERR_ARG;
  if (!ns::planes_ok(planes) || !(eps > 0.0f) || E < 0 || M < 0 || N < 0 || !ns::sched_ok(schedule, steps, planes))
    return MTX_ERR_ARG;
  if (!ns::sizes_ok(E, M, N)) return MTX_ERR_UNSUPPORTED;
  if (p_row < N || g_row < N || m_row < N || p_batch < 0 || g_batch < 0 || m_batch < 0) return MTX_ERR_ARG;
  if (E * M * N > 0 && (!param || !grad || !momentum)) return MTX_ERR_ARG;
  ns::Job j{};
  j.src = ns::Source{grad, g_batch, g_row, momentum, m_batch, m_row, (float)beta, (float)(1.0 - beta), nesterov};
  j.gdtype = grad_dtype;
  j.dtype = param_dtype;
  j.gvec = ns::rows_aligned(grad, grad_dtype, g_batch, g_row, N) && ns::rows_aligned(momentum, MTX_F32, m_batch, m_row, N);
  j.out = param;
  j.vec = ns::rows_aligned(param, param_dtype, p_batch, p_row, N);
  j.out_batch = p_batch;
  j.out_row = p_row;
  j.step = ns::OUT_STEP;
  j.lr = lr;
  j.decay = weight_decay;
  j.factor = factor;
  j.lr_dev = lr_dev;
  return ns::run(j, E, M, N, schedule, steps, eps, planes, workspace, workspace_bytes, (hipStream_t)stream);
}

// Newton-Schulz orthogonalisation of stacked matrices, and the optimiser step around it (Muon), on gfx950.
//
// X_0 = x / (|x|_F + eps), then for each step X <- a X + (b A + c A^2) X with A = X X^T on the smaller side S of the
// S x L matrix.  With Q = a I + b A + c A^2 this is X <- Q X, and A itself becomes Q A Q, all of them polynomials of
// the first A: symmetric, and they commute.  So g steps need one Gram product, S x S symmetric products and one
// product X <- P X with P = Q_g ... Q_1, in all 3 S^2 L + (4 g - 3) S^3 operations (a symmetric product computes
// half its tiles), where a step by itself needs 3 S^2 L + S^3.  At L = 2.67 S (768 x 2048) five steps need
// 45 S^3 by themselves (63 if all tiles were computed), 35 as 2 + 2 + 1, 30 as 3 + 2; at L = S always 20.
// A's small eigenvalues are squares of X's and grow by a^2 a step, so what the rounding of A adds grows as well and is
// not taken back before the next Gram product: a group holds three steps at most.  In simulation with gradients of
// rank 1 to full rank (f16 operands) five steps end 0.07 to 0.19 % off as 2 + 2 + 1, 0.1 to 0.5 % as 3 + 2, up to 14 %
// or beyond f16's range as one group.  The caller chooses: 2 where the result itself is asked for, 3 where it is
// a small change of weights.
//
// Numbers: |x|_F bounds every singular value by 1 and the polynomials bound them from there, so every matrix has a
// power-of-two scale, chosen by the caller from those bounds, that puts it into f16's range: 11 bits where
// bf16 has 8, at the same matrix-core rate ("half").  f32 results take two f16 planes, hi + lo, and three products for
// one ("full": 22 bits).  Sums are f32, |x|_F is summed in f64.  Two things cost more than all other roundings and are
// kept apart.  The diagonals of Q and P, where their size is, are f32 vectors beside the f16 matrices (rank 8: 0.28
// instead of 0.85 % off).  And X has its lo plane in "half" too: in X <- P X the diagonal's share, in f32 on the way
// out, takes hi + lo, as in the directions in which X is small P is a multiple of I (rank 32, 2 + 2 + 1: 0.17
// instead of 0.63 %).  Momentum is f32.
#include "common.h"
#include "dense_tile.h"
#include "f32_tile.h"
#include <algorithm>
#include <cmath>

namespace mtx {
namespace ns {

using namespace dense;
typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

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
// The workgroups of matrix e leave f64 sums of their rows' squares in part[e][blockIdx.x].
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
// X = x 2^e in f16, hi and lo planes where there are two, and what f32 holds beyond them (a bit at most: the steps carry
// it up by a^5 where x is singular), zeros past the last row and column, with e such that |x|_F + eps
// comes to [2^13, 2^14): a bf16 x is held exactly but for elements below 2^-27 of its norm.  Every workgroup adds the
// parts of its matrix in the same order.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void convert_kernel(Source s, int M, int N, int Mp, int Np, int rows,
                                                      const double* __restrict__ part, int nparts, float eps,
                                                      f16* __restrict__ X, f16* __restrict__ Xlo,
                                                      f16* __restrict__ Xrest, Scale* scales) {
  __shared__ double w[4];
  const int64_t e = blockIdx.y;
  double sum = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) sum += part[e * nparts + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double norm = sqrt((w[0] + w[1]) + (w[2] + w[3])) + (double)eps;
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
    if (Xlo) *(f16x8*)(Xlo + at) = lo;
    if (Xrest) *(f16x8*)(Xrest + at) = rest;
  }
}

// ---- symmetric S x S products ----------------------------------------------------------------------------------
// out = s_acc (U V) + s_v rs V + s_u U cs + d0 I (+ diag(rs cs) where both are given), element (r, c) of V times rs[r]
// (1 without rs) and of U times cs[c].  With `diag` the diagonal goes there and is zero in the matrix.
// Everything in f16 carries its scale; the s_ undo them, `s_out` is out's.
struct Sym {
  const f16 *u, *v;
  f16* out;
  float* diag;
  const float *rs, *cs;
  float s_acc, s_v, s_u, d0, s_out;
};
struct SymArgs {
  Sym p[2];             // problems of one launch (the same sizes)
  int np, E, S, Sp, K;  // K: reduction
  int64_t ld;           // of u and v
  int64_t in_batch, in_plane, out_batch, out_plane;  // elements from matrix to matrix, and from hi to lo plane
  const Scale* scales;  // Gram product of the first X: multiplies s_acc; or nullptr
};

// Eight columns of up to NP f16 planes for each step of a wave's 32 rows, loaded together: the loads of a block of rows
// are in flight while the one before is worked on.
template <class T, int NP>
struct Block {
  f16x8 x[NP][T::OUT_STEPS];
  // `at(it)`: offset of the lane's columns in step `it`, of an element that exists
  template <class At>
  __device__ __forceinline__ void load(int p, const f16* m, At at) {
    if (!m) return;
#pragma unroll
    for (int it = 0; it < T::OUT_STEPS; ++it) x[p][it] = *(const f16x8*)(m + at(it));
  }
};

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
// y += k x, a single instruction an element
__device__ __forceinline__ void add8(float y[8], const f16x8& x, float k) {
#pragma unroll
  for (int q = 0; q < 8; ++q) y[q] = __builtin_fmaf((float)x[q], k, y[q]);
}

// The scales are multiplied together before the elements are seen, and the diagonal is looked for only where a tile has
// it: an epilogue of 56 instructions an element cost more than the products of 768 elements (156 us for 128
// matrices of 768 x 768; 58 us at the matrix cores' peak).
template <class T, bool ADD, bool TWO>
__device__ __forceinline__ void sym_out(const SymArgs& a, const Sym& p, int64_t e, int m0, int n0,
                                        const f32x16 (&acc)[T::TM][T::TN], char* lds) {
  constexpr int TN = T::TN, HROW = TN * 64;  // bytes of a staged f16 row
  constexpr int NP = TWO ? 4 : 2, AHEAD = TWO && TN == 4 ? 1 : 2;  // blocks of addends in registers
  static_assert(T::NW * (T::OUT_BYTES + (TWO ? 2 : 1) * 32 * HROW) <= T::LDS_BYTES, "staging fits the ring");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  char* mine = T::out_lds(lds);
  char* turn = lds + T::NW * T::OUT_BYTES + wave * ((TWO ? 2 : 1) * 32 * HROW);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), c = n0 + (wave % T::WN) * (TN * 32) + T::out_col(0);
  const int S = a.S, Sp = a.Sp;
  const float k_acc = p.s_acc * p.s_out * (a.scales ? a.scales[e].gram : 1.0f), k_v = p.s_v * p.s_out;
  f16* out = p.out + e * a.out_batch;
  const f16 *u = ADD && p.cs ? p.u + e * a.in_batch : nullptr, *v = ADD ? p.v + e * a.in_batch : nullptr;
  const float* rs = ADD && p.rs ? p.rs + e * Sp : nullptr;
  float* diag = p.diag ? p.diag + e * Sp : nullptr;
  float cs[8], k_u[8];
  if (u) {
    ld8(p.cs + e * Sp, min(c, Sp - 8), cs);
#pragma unroll
    for (int q = 0; q < 8; ++q) k_u[q] = cs[q] * (p.s_u * p.s_out);
  }
  Block<T, NP> add[AHEAD];
  auto ahead = [&](int i) {
    auto at = [&](int it) { return (int64_t)min(wr + i * 32 + T::out_row(it), S - 1) * Sp + min(c, Sp - 8); };
    Block<T, NP>& b = add[i % AHEAD];
    b.load(0, v, at);
    b.load(1, u, at);
    if constexpr (TWO) {
      b.load(2, v ? v + a.in_plane : nullptr, at);
      b.load(3, u ? u + a.in_plane : nullptr, at);
    }
  };
  if (ADD) ahead(0);
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    if (ADD && AHEAD == 2 && i + 1 < T::TM) ahead(i + 1);
    if (ADD && AHEAD == 1 && i > 0) ahead(i);
    T::put(acc[i], mine);
    const Block<T, NP>& b = add[i % AHEAD];
#pragma unroll
    for (int it = 0; it < T::OUT_STEPS; ++it) {
      const int lr = T::out_row(it), r = wr + i * 32 + lr;
      const float rr = ADD && rs ? rs[min(r, S - 1)] : 1.0f;
      float y[8];
      T::get(mine, it, y);
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] *= k_acc;
      if (ADD) {
        add8(y, b.x[0][it], rr * k_v);
        if (TWO) add8(y, b.x[TWO ? 2 : 0][it], rr * k_v);
        if (u) {
#pragma unroll
          for (int q = 0; q < 8; ++q) y[q] = __builtin_fmaf((float)b.x[1][it][q], k_u[q], y[q]);
          if (TWO) {
#pragma unroll
            for (int q = 0; q < 8; ++q) y[q] = __builtin_fmaf((float)b.x[TWO ? 3 : 1][it][q], k_u[q], y[q]);
          }
        }
      }
      if (m0 == n0 && ADD) {
        const int dq = r - c;  // the diagonal's place among the lane's columns
        if (dq >= 0 && dq < 8) {
          float d = 0.0f;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            if (q == dq) d = y[q] + (p.d0 + (u && rs ? rr * cs[q] : 0.0f)) * p.s_out;
          }
          if (diag && r < Sp) diag[r] = r < S ? d / p.s_out : 0.0f;
#pragma unroll
          for (int q = 0; q < 8; ++q) y[q] = q == dq ? (diag ? 0.0f : d) : y[q];
        }
      }
      if (c + 8 > S) {
#pragma unroll
        for (int q = 0; q < 8; ++q) y[q] = c + q < S ? y[q] : 0.0f;
      }
      f16x8 hi = round8(y), lo;
      if (TWO) lo = rest8(y, hi);
      if (r < S && c < Sp) {
        *(f16x8*)(out + (int64_t)r * Sp + c) = hi;
        if (TWO) *(f16x8*)(out + a.out_plane + (int64_t)r * Sp + c) = lo;
      }
      if (m0 != n0) {
        const uint32_t keep = r < S ? 0xFFFFFFFFu : 0u;
        char* at = turn + lr * HROW + (((T::out_col(0) >> 3) ^ ((lr & 3) << 1)) << 4);
        *(u32x4*)at = __builtin_bit_cast(u32x4, hi) & keep;
        if (TWO) *(u32x4*)(at + 32 * HROW) = __builtin_bit_cast(u32x4, lo) & keep;
      }
    }
    if (m0 == n0) continue;
    // the mirrored tile: 16 lanes read 16 columns of eight rows each, turned; 64 contiguous bytes a row of it
    __builtin_amdgcn_s_waitcnt(MTX_LGKMCNT0);
    asm volatile("" ::: "memory");
    const int wc = n0 + (wave % T::WN) * (TN * 32);
#pragma unroll
    for (int it = 0; it < TN * 2; ++it) {
      const int rb = (lane >> 4) * 8, cb = it * 16;
      const int row = wc + cb + (lane & 15), col = wr + i * 32 + rb;
      const int n = cb + 4 * (lane & 3), k = rb + ((lane & 15) >> 2);
#pragma unroll
      for (int pl = 0; pl < (TWO ? 2 : 1); ++pl) {
        const char* base = turn + pl * 32 * HROW;
        auto tr = [&](int kk) {
          return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(
              base + kk * HROW + (((n >> 3) ^ ((kk & 3) << 1)) << 4) + (n & 7) * 2));
        };
        const s16x4 both[2] = {tr(k), tr(k + 4)};
        if (row < S && col < Sp)
          *(f16x8*)(out + pl * a.out_plane + (int64_t)row * Sp + col) = __builtin_bit_cast(f16x8, both);
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

// GRAM: X times itself, no addends.  COLS: the reduction runs down u's and v's columns (the Gram product of a tall X);
// otherwise along their rows.
template <class T, bool GRAM, bool COLS, bool TWO>
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
  T::product(operand(p.u, m0), operand(p.v, n0), a.K, lds, acc);
  __syncthreads();
  sym_out<T, !GRAM, TWO>(a, p, e, m0, n0, acc, lds);
}

// ---- X <- P X (tall: X P) ----------------------------------------------------------------------------------------
enum { OUT_X = 0, OUT_STORE = 1, OUT_STEP = 2 };
struct ApplyArgs {
  const f16* p;
  const float* pd;   // P's diagonal
  const f16* x;
  const f16 *xl, *xr;  // x's lo plane and the rest of the first x in "full", or nullptr
  f16 *xo, *xol;     // OUT_X: both planes
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
  T::product(oa, ob, s.Sp, lds, acc);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  char* mine = T::out_lds(lds);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), wc = n0 + (wave % T::WN) * (T::TN * 32);
  const float s_x = a.scales ? a.scales[e].x : a.s_x, s_acc = s_x * a.s_p;
  const float* pd = a.pd + e * s.Sp;
  const float lr = OUT == OUT_STEP ? (a.lr_dev ? *a.lr_dev : a.lr) : 0.0f;
  const f16 *xl = a.xl ? a.xl + e * s.xs : nullptr, *xr = TWO && a.xr ? a.xr + e * s.xs : nullptr;
  const int c = wc + T::out_col(0);
  constexpr int NP = TWO ? 3 : 2, DV = sizeof(D) / 2;  // 16-byte pieces of eight D
  constexpr int AHEAD = T::TN == 4 && (TWO || (OUT == OUT_STEP && DV == 2)) ? 1 : 2;
  Block<T, NP> add[AHEAD];
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
    auto at = [&](int it) { return (int64_t)min(wr + i * 32 + T::out_row(it), s.Mp - 1) * s.Np + min(c, s.Np - 8); };
    Block<T, NP>& b = add[i % AHEAD];
    b.load(0, X, at);
    b.load(1, xl, at);
    if constexpr (TWO) b.load(2, xr, at);
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
    const Block<T, NP>& b = add[i % AHEAD];
#pragma unroll
    for (int it = 0; it < T::OUT_STEPS; ++it) {
      const int r = wr + i * 32 + T::out_row(it);
      float y[8];
      T::get(mine, it, y);
      const float dr = TALL ? 0.0f : pd[min(r, s.Sp - 1)];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float k = (TALL ? dc[q] : dr) * s_x;
        y[q] = __builtin_fmaf((float)b.x[0][it][q], k, y[q] * s_acc);
        if (xl) y[q] = __builtin_fmaf((float)b.x[1][it][q], k, y[q]);
        if (TWO && xr) y[q] = __builtin_fmaf((float)b.x[TWO ? 2 : 1][it][q], k, y[q]);
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
        *(f16x8*)(a.xol + at) = rest8(y, hi);
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

// ---- the chain of launches ---------------------------------------------------------------------------------------
template <bool A, bool B, bool TWO> using Big = Tile<F16, 4, 4, 2, 2, 4, A, B, false, TWO>;
template <bool A, bool B, bool TWO> using Small = Tile<F16, 2, 2, 2, 2, 4, A, B, false, TWO>;

constexpr int kBigTiles = 192;

template <bool GRAM, bool COLS, bool TWO>
static int launch_sym(const SymArgs& a, hipStream_t st) {
  auto tiles = [&](int b) { const int64_t n = ceil_div(a.S, b); return a.np * a.E * (n * (n + 1) / 2); };
  if (tiles(256) >= kBigTiles && a.S >= 256)
    hipLaunchKernelGGL((sym_kernel<Big<COLS, COLS, TWO>, GRAM, COLS, TWO>), dim3((unsigned)tiles_grid(tiles(256))), dim3(256), 0,
                       st, a);
  else
    hipLaunchKernelGGL((sym_kernel<Small<COLS, COLS, TWO>, GRAM, COLS, TWO>), dim3((unsigned)tiles_grid(tiles(128))), dim3(256),
                       0, st, a);
  return check_launch();
}
template <bool TALL, bool TWO, int OUT, typename D>
static int launch_apply_out(const ApplyArgs& a, hipStream_t st) {
  auto tiles = [&](int b) { return a.E * ceil_div(a.s.Mp, b) * ceil_div(a.s.Np, b); };
  if (tiles(256) >= kBigTiles && a.s.S >= 256)
    hipLaunchKernelGGL((apply_kernel<Big<false, !TALL, TWO>, TALL, TWO, OUT, D>), dim3((unsigned)tiles_grid(tiles(256))),
                       dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((apply_kernel<Small<false, !TALL, TWO>, TALL, TWO, OUT, D>), dim3((unsigned)tiles_grid(tiles(128))),
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

// Workgroups of a matrix in the norm and conversion launches.
static int64_t parts_of(int64_t E, const Shape& s) {
  const int64_t by_size = std::max<int64_t>(1, s.xs / 8192);
  return std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(by_size, s.Mp), std::min<int64_t>(512, ceil_div(2048, E))));
}

// Matrices that go through the chain together.
constexpr int64_t kChunkBytes = (int64_t)4 << 30;
static int64_t matrix_bytes(const Shape& s, int planes) {
  return ((4 + planes - 1) * s.xs + 5 * s.ms * planes) * 2 + 4 * round_up((int64_t)s.Sp * 4, 256) + 1024 * 8 + 256;
}
static int64_t chunk_of(int64_t E, const Shape& s, int planes) {
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(E, kChunkBytes / matrix_bytes(s, planes)));
  return ceil_div(E, ceil_div(E, most));
}
static int64_t workspace_bytes(int64_t E, const Shape& s, int planes) {
  const int64_t n = chunk_of(E, s, planes);
  int64_t b = 0;
  b += round_up(n * 512 * 8, 256);                        // partial sums
  b += round_up(n * (int64_t)sizeof(Scale), 256);
  b += 3 * round_up(n * s.Sp * 4, 256);                    // diagonals
  b += 2 * round_up(n * s.xs * 4, 256) + (planes - 1) * round_up(n * s.xs * 2, 256);  // X, twice, in planes
  b += 5 * round_up(n * s.ms * 2 * planes, 256);          // A, T and three of Q and P
  return b;
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
  float* diag[3];
  for (auto& d : diag) d = (float*)take(E * s.Sp * 4);
  f16* X[2];
  for (auto& x : X) x = (f16*)take(E * s.xs * 4);
  f16* rest = TWO ? (f16*)take(E * s.xs * 2) : nullptr;
  f16 *A = (f16*)take(E * s.ms * 2 * planes), *Tm = (f16*)take(E * s.ms * 2 * planes), *Q[3];
  for (auto& q : Q) q = (f16*)take(E * s.ms * 2 * planes);
  const int64_t x_plane = E * s.xs, m_plane = E * s.ms;

  // in "half" f16 holds a bf16 x as it is
  const bool first_lo = TWO || j.src.m || j.gdtype == MTX_F32;
  const int parts = (int)parts_of(E, s);
  const int rows = (int)ceil_div(s.M, parts), rows_p = (int)ceil_div(s.Mp, parts);
  const dim3 grid((unsigned)parts, (unsigned)E);
#define MTX_PREP(T, V)                                                                                              \
  do {                                                                                                              \
    hipLaunchKernelGGL((norm_kernel<T, V>), grid, dim3(256), 0, st, j.src, s.M, s.N, rows, part);                   \
    hipLaunchKernelGGL((convert_kernel<T, V>), grid, dim3(256), 0, st, j.src, s.M, s.N, s.Mp, s.Np, rows_p, part, parts, \
                       eps, X[0], first_lo ? X[0] + x_plane : nullptr, rest, scales);                                      \
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
  int p = -1;           // Q[p], diag[p] hold P
  for (int i = 0; i < steps; ++i) {
    const float* c = sched + 9 * i;
    const float sA = c[3], sQ = c[4], sT = c[5], sP = c[6], sX = c[7];
    const bool ends = c[8] != 0.0f || i + 1 == steps;
    if (p < 0) {
      SymArgs g = m;
      g.np = 1;
      g.K = TALL ? s.Mp : s.Np;
      g.ld = s.Np;
      g.in_batch = s.xs;
      g.in_plane = x_plane;
      g.scales = x_scale == 0.0f ? scales : nullptr;
      g.p[0] = Sym{X[cur], X[cur], A, nullptr, nullptr, nullptr, x_scale == 0.0f ? 1.0f : 1.0f / (x_scale * x_scale),
                   0.0f, 0.0f, 0.0f, sA};
      rc = launch_sym<true, TALL, TWO>(g, st);
      if (rc != MTX_OK) return rc;
    }
    m.K = s.Sp;
    m.ld = s.Sp;
    m.in_batch = s.ms;
    m.in_plane = m_plane;
    const int q = p < 0 ? 0 : (p + 1) % 3, np = p < 0 ? q : (p + 2) % 3;
    m.np = 1;
    m.p[0] = Sym{A, A, Q[q], diag[q], nullptr, nullptr, c[2] / (sA * sA), c[1] / sA, 0.0f, c[0], sQ};
    rc = launch_sym<false, false, TWO>(m, st);
    if (rc != MTX_OK) return rc;
    // P <- Q P and T = Q A in one launch, then A <- Q T
    m.np = 0;
    if (p >= 0) {
      const float sPp = c[6 - 9];
      m.p[m.np++] = Sym{Q[q], Q[p], Q[np], diag[np], diag[q], diag[p], 1.0f / (sQ * sPp), 1.0f / sPp, 1.0f / sQ, 0.0f, sP};
    }
    if (!ends) m.p[m.np++] = Sym{Q[q], A, Tm, nullptr, diag[q], nullptr, 1.0f / (sQ * sA), 1.0f / sA, 0.0f, 0.0f, sT};
    if (m.np > 0) {
      rc = launch_sym<false, false, TWO>(m, st);
      if (rc != MTX_OK) return rc;
    }
    p = np;
    if (!ends) {
      const float sA2 = c[3 + 9];
      m.np = 1;
      m.p[0] = Sym{Q[q], Tm, A, nullptr, diag[q], nullptr, 1.0f / (sQ * sT), 1.0f / sT, 0.0f, 0.0f, sA2};
      rc = launch_sym<false, false, TWO>(m, st);
      if (rc != MTX_OK) return rc;
      continue;
    }
    ApplyArgs a{};
    a.p = Q[p];
    a.pd = diag[p];
    a.x = X[cur];
    a.xl = first_lo || x_scale != 0.0f ? X[cur] + x_plane : nullptr;
    a.xr = x_scale == 0.0f ? rest : nullptr;
    a.xo = X[cur ^ 1];
    a.xol = X[cur ^ 1] + x_plane;
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
    rc = launch_apply<TALL, TWO>(i + 1 == steps ? j.step : OUT_X, a, st);
    if (rc != MTX_OK) return rc;
    x_scale = sX;
    cur ^= 1;
    p = -1;
  }
  return MTX_OK;
}

static int run(Job j, int64_t E, int64_t M, int64_t N, const float* sched, int steps, float eps, int planes, void* ws,
               int64_t ws_bytes, hipStream_t st) {
  if (E == 0 || M == 0 || N == 0) return MTX_OK;
  const Shape s = shape_of(M, N);
  if (!ws || ws_bytes < workspace_bytes(E, s, planes)) return MTX_ERR_WORKSPACE;
  const int64_t chunk = chunk_of(E, s, planes);
  const int gsize = dtype_size(j.gdtype), osize = dtype_size(j.dtype);
  for (int64_t e = 0; e < E; e += chunk) {
    Job c = j;
    c.src.g = (const char*)j.src.g + e * j.src.g_batch * gsize;
    if (j.src.m) c.src.m = j.src.m + e * j.src.m_batch;
    c.out = (char*)j.out + e * j.out_batch * osize;
    const int64_t n = std::min(chunk, E - e);
    const int rc = s.tall ? (planes == 2 ? run_chunk<true, true>(c, n, s, sched, steps, eps, (char*)ws, st)
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
static bool sched_ok(const float* sched, int steps) {
  if (!sched || steps < 1 || steps > 64) return false;
  for (int i = 0; i < 9 * steps; ++i)
    if (!std::isfinite(sched[i])) return false;
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
  if (!ns::sizes_ok(E, M, N) || (planes != 1 && planes != 2)) return -1;
  if (E == 0 || M == 0 || N == 0) return 0;
  return ns::workspace_bytes(E, ns::shape_of(M, N), planes);
}

extern "C" int mtx_newton_schulz(const void* x, int dtype, int64_t E, int64_t M, int64_t N, int64_t x_batch, int64_t x_row,
                                 const float* schedule, int steps, float eps, int planes, void* out, int64_t out_batch,
                                 int64_t out_row, void* workspace, int64_t workspace_bytes, void* stream) {
  if ((dtype != MTX_F32 && dtype != MTX_BF16) || (planes != 1 && planes != 2) || !(eps > 0.0f)) return MTX_ERR_ARG;
  if (E < 0 || M < 0 || N < 0 || !ns::sched_ok(schedule, steps)) return MTX_ERR_ARG;
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
  if ((planes != 1 && planes != 2) || !(eps > 0.0f) || E < 0 || M < 0 || N < 0 || !ns::sched_ok(schedule, steps))
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

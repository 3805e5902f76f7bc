// The products of the head's losses in bf16 on the 16-bit matrix cores (dense_tile.h), and what their tiles do
// with the logits on the way out.
#include "dense_tile.h"
#include "head_loss.h"

namespace mtx {
namespace head {

using dense::Operand;
template <bool VD, bool TAIL> using Big = dense::Tile<dense::Bf16, 4, 4, 2, 2, 4, false, !VD, TAIL>;
template <bool VD, bool TAIL> using Small = dense::Tile<dense::Bf16, 2, 2, 2, 2, 4, false, !VD, TAIL>;
template <bool VD, bool TAIL> using Thin = dense::Tile<dense::Bf16, 1, 2, 2, 2, 6, false, !VD, TAIL, false, dense::DIAG_NONE, 4>;

// Tiles go row by row within groups of kGroup rows of tiles, so that neighbours share both operands' strips in L2.
constexpr int kGroup = 8;
template <class T>
__device__ __forceinline__ void tile_at(int t, int nm, int nn, int& m0, int& n0) {
  const int g = t / (kGroup * nn), gs = min(kGroup, nm - g * kGroup), in = t - g * kGroup * nn;
  m0 = (g * kGroup + in % gs) * T::BM;
  n0 = in / gs * T::BN;
}
// where the way out of a wave (Tile::put) keeps column c of row r
template <class T>
__device__ __forceinline__ float* in_lds(char* mine, int r, int c) {
  return (float*)(mine + r * (T::TN * 128) + (((c >> 2) ^ (r & (T::TN * 8 - 1))) << 4) + (c & 3) * 4);
}

// exp((z - m) / tau).  The difference first: of z scale - m scale, whose second product is rounded, all terms of a row are off by a
// common factor, by 4e-5 where m / tau is 1000, and the largest logit's own term is not 1.
__device__ __forceinline__ float exp_of(float z, float m, float scale) { return __builtin_amdgcn_exp2f((z - m) * scale); }

// The 256 x 256 tiles' way out of the forward pass spills 23 VGPRs, each written once and read once or twice; their product's
// loop has no spill.
// A lane holds, of 32 rows at a time, one row's 16 TN values in columns 32 j + 8 g + 4 (lane / 32) + q (accumulator j, element
// 4 g + q): the row's maximum and sum are taken in the lane and joined with that of lane ^ 32.  Entries are looked up in LDS,
// where the 32 rows are put for that only if one of them has an entry among the wave's columns.
template <class T>
__device__ __forceinline__ void forward_out(const Logits& p, dense::f32x16 (&acc)[T::TM][T::TN], char* mine, int wr, int c0) {
  constexpr int BC = T::TN * 32;  // the wave's columns
  const int lane = threadIdx.x & 63, half = lane >> 5, left = p.cols - c0;
  // the rows' entries among the wave's columns: [lo, hi) of their lists, or column lo
  int lo[T::TM], hi[T::TM];
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    const int row = wr + i * 32 + (lane & 31);
    lo[i] = hi[i] = 0;
    if (row >= p.T) continue;
    if (p.e.targets) {
      const int64_t c = target(p.e, row) - p.v0 - c0;
      if (c >= 0 && c < BC && c < left) {
        lo[i] = (int)c;
        hi[i] = BC;
      }
    } else {
      const uint16_t* b = p.e.bounds + row * p.e.ldb + (p.v0 + c0) / kBlock;
      lo[i] = b[0];
      hi[i] = b[1];
    }
  }
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    const int row = wr + i * 32 + (lane & 31);
    if (left < BC) {
#pragma unroll
      for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (32 * j + 8 * (v >> 2) + 4 * half + (v & 3) >= left) acc[i][j][v] = -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) m = fmaxf(m, acc[i][j][v]);
    m = fmaxf(m, lane_xchg<5>(m));
    const float off = m == -INFINITY ? 0.0f : m;  // nothing but -inf: a sum of 0
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[v & 3] += exp_of(acc[i][j][v], off, p.scale);
    float sum = (s[0] + s[1]) + (s[2] + s[3]);
    sum += lane_xchg<5>(sum);
    if (row < p.T && half == 0) p.part[(int64_t)((p.v0 + c0) / BC) * p.T + row] = make_float2(m, sum);
    if (__ballot(lo[i] < hi[i]) == 0) continue;
    T::put(acc[i], mine);
    if (p.e.targets) {
      if (hi[i] && half == 0) p.chosen[row] = *in_lds<T>(mine, lane & 31, lo[i]);
    } else {
      // eight at a time, so that a row whose entries all lie here (1531 x 1001 x 50257 with 100 of them) waits for few loads
      for (int e = lo[i] + half; e < hi[i]; e += 16) {
        const int64_t at = (int64_t)row * p.e.K;
        int c[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) c[q] = p.e.idx[at + min(e + 2 * q, hi[i] - 1)] - p.v0 - c0;
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (e + 2 * q < hi[i] && (unsigned)c[q] < (unsigned)BC) p.chosen[at + e + 2 * q] = *in_lds<T>(mine, lane & 31, c[q]);
      }
    }
    asm volatile("" ::: "memory");
  }
}

// dz = a softmax, rounded, 32 rows at a time into LDS (16-byte chunk c of a row at chunk c ^ (row % chunks)) and out in whole
// lines; with two planes what the rounding left goes the same way after it.  What a row's entries take from it is
// named_kernel's, which knows their logits.
template <class T, int PLANES>
__device__ __forceinline__ void gradient_out(const Logits& p, dense::f32x16 (&acc)[T::TM][T::TN], char* mine, int wr, int c0) {
  constexpr int BC = T::TN * 32, CH = T::TN * 4, BYTES = 32 * T::TN * 64;  // chunks of a row; bytes of 32 rows
  typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
  const int lane = threadIdx.x & 63, half = lane >> 5, r = lane & 31, left = p.cols - c0;
  float a[T::TM], m[T::TM];
  bool care = left < BC;
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    const int row = min(wr + i * 32 + r, p.T - 1);
    a[i] = p.f.a(row, p.f.b(row), m[i]);
  }
#pragma unroll
  for (int i = 0; i < T::TM; ++i) care |= a[i] == 0.0f;
  care = __ballot(care) != 0;
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float d[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          d[q] = a[i] * exp_of(acc[i][j][4 * g + q], m[i], p.scale);
        if (care) {  // zeros behind the columns, and in rows that are left out, whatever their logits are
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (a[i] == 0.0f || 32 * j + 8 * g + 4 * half + q >= left) d[q] = 0.0f;
        }
        const bf16x4 y{(__bf16)d[0], (__bf16)d[1], (__bf16)d[2], (__bf16)d[3]};
        *(bf16x4*)(mine + i * BYTES + r * (CH * 16) + (((j * 4 + g) ^ (r & (CH - 1))) << 4) + half * 8) = y;
        if constexpr (PLANES == 2)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][4 * g + q] = d[q] - (float)y[q];
      }
  }
  auto leave = [&](uint16_t* dz) {
    __builtin_amdgcn_s_waitcnt(MTX_LGKMCNT0);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int it = 0; it < T::TN * 2; ++it) {
        const int at = it * 64 + lane, o = at / CH, c = at % CH, row = wr + i * 32 + o;
        const v4u32 v = *(const v4u32*)(mine + i * BYTES + o * (CH * 16) + ((c ^ (o & (CH - 1))) << 4));
        if (row < p.T) *(v4u32*)(dz + (int64_t)row * p.ldz + c * 8) = v;
      }
  };
  uint16_t* dz = (uint16_t*)p.dz + c0;
  leave(dz);
  if constexpr (PLANES == 2) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(bf16x4*)(mine + i * BYTES + r * (CH * 16) + (((j * 4 + g) ^ (r & (CH - 1))) << 4) + half * 8) =
              bf16x4{(__bf16)acc[i][j][4 * g], (__bf16)acc[i][j][4 * g + 1], (__bf16)acc[i][j][4 * g + 2],
                     (__bf16)acc[i][j][4 * g + 3]};
    leave(dz + (int64_t)p.T * p.ldz);
  }
}

// PLANES: of dz; 0 for the forward pass
template <class T, int PLANES>
__global__ __launch_bounds__(T::NT, T::LDS_BYTES > 80 * 1024 ? 1 : 2) void logits_kernel(Logits p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS_BYTES];
  constexpr int OUT = PLANES ? T::TM * 32 * T::TN * 64 : T::OUT_BYTES;  // of a wave
  static_assert(T::NW * OUT <= T::LDS_BYTES, "the way out fits the ring");
  const int nm = (p.T + T::BM - 1) / T::BM, nn = (p.cols + T::BN - 1) / T::BN;
  const int t = dense::tile_of(blockIdx.x, nm * nn);
  if (t < 0) return;
  int m0, n0;
  tile_at<T>(t, nm, nn, m0, n0);
  const uint16_t *x = (const uint16_t*)p.x + (int64_t)m0 * p.ldx, *w = (const uint16_t*)p.w;
  w += T::b_cols ? (int64_t)n0 : (int64_t)n0 * p.ldw;
  const Operand ox{{x, x}, p.ldx, p.T - m0}, ow{{w, w}, p.ldw, p.w_left - n0, p.missing};
  dense::f32x16 acc[T::TM][T::TN];
  T::product(ox, ow, p.red, lds, acc);
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), c0 = n0 + (wave % T::WN) * (T::TN * 32);
  if constexpr (PLANES) gradient_out<T, PLANES>(p, acc, lds + wave * OUT, wr, c0);
  else forward_out<T>(p, acc, lds + wave * OUT, wr, c0);
}

// ---- the gradients' products ------------------------------------------------------------------------------------------
template <bool A_COLS, bool B_COLS, bool TAIL> using GradBig = dense::Tile<dense::Bf16, 4, 4, 2, 2, 4, A_COLS, B_COLS, TAIL>;
template <bool A_COLS, bool B_COLS, bool TAIL> using GradSmall = dense::Tile<dense::Bf16, 2, 2, 2, 2, 4, A_COLS, B_COLS, TAIL>;

template <class T>
__global__ __launch_bounds__(T::NT, T::LDS_BYTES > 80 * 1024 ? 1 : 2) void product_kernel(Product p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS_BYTES];
  const int nm = (p.rows + T::BM - 1) / T::BM, nn = (p.cols + T::BN - 1) / T::BN;
  const int id = dense::tile_of(blockIdx.x, nm * nn * p.pieces);
  if (id < 0) return;
  const int t = id / p.pieces, piece = id % p.pieces, stages = (p.red + dense::BKS - 1) / dense::BKS;
  const int k0 = (int)((int64_t)piece * stages / p.pieces) * dense::BKS;
  const int k1 = min((int)((int64_t)(piece + 1) * stages / p.pieces) * dense::BKS, p.red);
  int m0, n0;
  tile_at<T>(t, nm, nn, m0, n0);
  const uint16_t *a = (const uint16_t*)p.a, *b = (const uint16_t*)p.b;
  a += T::cols ? (int64_t)k0 * p.lda + m0 : (int64_t)m0 * p.lda + k0;
  b += T::b_cols ? (int64_t)k0 * p.ldb + n0 : (int64_t)n0 * p.ldb + k0;
  const Operand oa{{a, a}, p.lda, p.a_left - m0}, ob{{b, b}, p.ldb, p.b_left - n0, k1 == p.red ? p.missing : 0};
  dense::f32x16 acc[T::TM][T::TN];
  T::product(oa, ob, k1 - k0, lds, acc);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  char* mine = T::out_lds(lds);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), c0 = n0 + (wave % T::WN) * (T::TN * 32);
  float* sums = p.acc ? p.acc + (int64_t)piece * p.rows * p.ldacc : nullptr;
  const float alpha = p.f.alpha();
  if (sums) {
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
      T::put(acc[i], mine);
#pragma unroll 4
      for (int it = 0; it < T::OUT_STEPS; ++it) {
        const int r = wr + i * 32 + T::out_row(it), c = c0 + T::out_col(it);
        if (r >= p.rows || c >= p.cols) continue;
        float v[8];
        T::get(mine, it, v);
        float* s = sums + (int64_t)r * p.ldacc + c;
        if (p.add) {
          float x[8];
          ld8(s, 0, x);
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] += x[q];
        }
        if (!p.last) {
          st8(s, 0, v);
          continue;
        }
        uint16_t* out = (uint16_t*)p.out + (int64_t)r * p.ldo + c;
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] *= alpha;
        store_part(out, v, p.cols - c);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < T::TM; ++i) {
      T::put(acc[i], mine);
#pragma unroll
      for (int it = 0; it < T::OUT_STEPS; ++it) {
        const int r = wr + i * 32 + T::out_row(it), c = c0 + T::out_col(it);
        if (r >= p.rows || c >= p.cols) continue;
        float v[8];
        T::get(mine, it, v);
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] *= alpha;
        store_part((uint16_t*)p.out + (int64_t)r * p.ldo + c, v, p.cols - c);
      }
    }
  }
}

// PLANES: that a tile writes of dz
template <class T, int PLANES>
static int go_logits(const Logits& p, bool dz, hipStream_t st) {
  if (dz && p.planes != PLANES) return MTX_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)dense::tiles_grid(ceil_div(p.T, T::BM) * ceil_div(p.cols, T::BN)));
  if (dz) hipLaunchKernelGGL((logits_kernel<T, PLANES>), grid, dim3(T::NT), 0, st, p);
  else hipLaunchKernelGGL((logits_kernel<T, 0>), grid, dim3(T::NT), 0, st, p);
  return check_launch();
}
template <bool VD, bool TAIL>
static int go_path(const Logits& p, bool dz, int path, hipStream_t st) {
  if (path == PATH_BIG) return go_logits<Big<VD, TAIL>, 1>(p, dz, st);
  if (path == PATH_SMALL) return go_logits<Small<VD, TAIL>, 1>(p, dz, st);
  return go_logits<Thin<VD, TAIL>, 2>(p, dz, st);
}
int launch_logits(const Logits& p, bool dz, int order, int path, hipStream_t st) {
  const bool tail = p.red % dense::BKS != 0 || p.missing > 0;
  if (order == ORDER_VD) return tail ? go_path<true, true>(p, dz, path, st) : go_path<true, false>(p, dz, path, st);
  return tail ? go_path<false, true>(p, dz, path, st) : go_path<false, false>(p, dz, path, st);
}

template <class T>
static int go_product(const Product& p, hipStream_t st) {
  const dim3 grid((unsigned)dense::tiles_grid(ceil_div(p.rows, T::BM) * ceil_div(p.cols, T::BN) * p.pieces));
  hipLaunchKernelGGL(product_kernel<T>, grid, dim3(T::NT), 0, st, p);
  return check_launch();
}
template <bool A_COLS, bool B_COLS, bool TAIL>
static int go_size(const Product& p, int size, hipStream_t st) {
  return size == SIZE_BIG ? go_product<GradBig<A_COLS, B_COLS, TAIL>>(p, st) : go_product<GradSmall<A_COLS, B_COLS, TAIL>>(p, st);
}
// A dz [T][piece] or x^T, B W^T in either order or dz: (rows, rows), (rows, cols) and (cols, cols)
int launch_product(const Product& p, bool a_cols, bool b_cols, int size, hipStream_t st) {
  const bool tail = p.red % dense::BKS != 0 || p.missing > 0;
  if (a_cols) return tail ? go_size<true, true, true>(p, size, st) : go_size<true, true, false>(p, size, st);
  if (b_cols) return tail ? go_size<false, true, true>(p, size, st) : go_size<false, true, false>(p, size, st);
  return tail ? go_size<false, false, true>(p, size, st) : go_size<false, false, false>(p, size, st);
}

}  // namespace head
}  // namespace mtx

// Dense product with its epilogue, out = act(x w + bias) + residual, and the parts of its gradient.
//
// The bias, the activation, the residual and, for training, the copy of z = x w + bias that the gradient needs
// are applied to the f32 sums on their way out, so that z costs at most one write and the rest no
// pass of their own.  bf16 with rows of whole 16-byte chunks runs on the 16-bit matrix cores (dense_tile.h), 256 x 256
// tiles or, where those are few, 128 x 128; everything else on f32 matrix-core tiles (f32_tile.h).
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
template <typename T, int MODE, int VEC>
__global__ __launch_bounds__(f32mm::NT) void f32_kernel(Args p) {
  using namespace f32mm;
  __shared__ __attribute__((aligned(16))) float as[TILE], bs[TILE];
  const int64_t r0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int64_t rows = p.rows, cols = p.cols, red = p.red;
  const T *A = (const T*)p.a, *B = (const T*)p.b;
  auto at_a = [&](int r, int c, int s) -> const T* {
    if (MODE == DW) {
      const int64_t k = (int64_t)s * KS + r, m = r0 + c;
      return k < red && m < rows ? A + k * rows + m : nullptr;
    }
    const int64_t m = r0 + r, k = (int64_t)s * KS + c;
    return m < rows && k < red ? A + m * red + k : nullptr;
  };
  auto at_b = [&](int r, int c, int s) -> const T* {
    if (MODE == DX) {
      const int64_t n = n0 + r, k = (int64_t)s * KS + c;
      return n < cols && k < red ? B + n * red + k : nullptr;
    }
    const int64_t k = (int64_t)s * KS + r, n = n0 + c;
    return k < red && n < cols ? B + k * cols + n : nullptr;
  };
  f32x16 acc;
  mainloop<T, MODE == DW, MODE != DX, VEC>(acc, p.red, as, bs, at_a, at_b, A, B);
  const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) >> 1, wn = (threadIdx.x >> 6) & 1;
  const int64_t n = n0 + wn * 32 + (lane & 31);
  if (n >= cols) return;
  const float bias = p.bias ? gld<T>((const T*)p.bias, n) : 0.0f;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int64_t r = r0 + wm * 32 + 8 * (v / 4) + 4 * (lane >> 5) + v % 4;
    if (r >= rows) continue;
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
template <int MODE, bool TAIL> using Small = dense::Tile<dense::Bf16, 2, 2, 2, 2, 4, MODE == DW, MODE != DX, TAIL>;

// z = v + bias, out = act(z) + residual for eight columns
__device__ __forceinline__ void finish8(const Args& p, int r, int c, float v[8]) {
  const int64_t at = (int64_t)r * p.cols + c;
  if (p.bias) {
    float b[8];
    ld8((const uint16_t*)p.bias, c, b);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += b[q];
  }
  if (p.pre) dense::store8((uint16_t*)p.pre + at, v);
  if (p.act != MTX_ACT_NONE) {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = activate(v[q], p.act);
  }
  if (p.residual) {
    float b[8];
    ld8((const uint16_t*)p.residual, at, b);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += b[q];
  }
  dense::store8((uint16_t*)p.out + at, v);
}

// Tiles go row by row within groups of kGroup rows of tiles, so that neighbours share both operands' strips in L2.
constexpr int kGroup = 8;
template <class T, int MODE>
__global__ __launch_bounds__(T::NT, T::LDS_BYTES > 80 * 1024 ? 1 : 2) void tile_kernel(Args p) {
  __shared__ __attribute__((aligned(1024))) char lds[T::LDS_BYTES];
  const int nm = (p.rows + T::BM - 1) / T::BM, nn = (p.cols + T::BN - 1) / T::BN;
  const int t = dense::tile_of(blockIdx.x, nm * nn);
  if (t < 0) return;
  const int g = t / (kGroup * nn), gs = min(kGroup, nm - g * kGroup), in = t - g * kGroup * nn;
  const int m0 = (g * kGroup + in % gs) * T::BM, n0 = in / gs * T::BN;
  const uint16_t *a = (const uint16_t*)p.a, *b = (const uint16_t*)p.b;
  const uint16_t* pa = MODE == DW ? a + m0 : a + (int64_t)m0 * p.red;
  const uint16_t* pb = MODE == DX ? b + (int64_t)n0 * p.red : b + n0;
  const Operand oa{{pa, pa}, MODE == DW ? p.rows : p.red, p.rows - m0};
  const Operand ob{{pb, pb}, MODE == DX ? p.red : p.cols, p.cols - n0};
  dense::f32x16 acc[T::TM][T::TN];
  T::product(oa, ob, p.red, lds, acc);
  __syncthreads();
  const int wave = threadIdx.x >> 6;
  char* mine = T::out_lds(lds);
  const int wr = m0 + (wave / T::WN) * (T::TM * 32), c = n0 + (wave % T::WN) * (T::TN * 32) + T::out_col(0);
#pragma unroll
  for (int i = 0; i < T::TM; ++i) {
    T::put(acc[i], mine);
#pragma unroll 2
    for (int it = 0; it < T::OUT_STEPS; ++it) {
      const int r = wr + i * 32 + T::out_row(it);
      float v[8];
      T::get(mine, it, v);
      if (r < p.rows && c < p.cols) finish8(p, r, c, v);
    }
  }
}

// ---- dz = dy act'(z) and the column sums of dz ---------------------------------------------------------------
// A workgroup takes 32 lanes x V columns of a range of rows, eight rows at a time, and leaves f32 sums of its range; a
// second launch adds the ranges in order, so the sums do not depend on timing.  One pass over dy and z.
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
template <typename T>
__global__ __launch_bounds__(256) void column_sum_kernel(const float* __restrict__ part, int n, int64_t N,
                                                         T* __restrict__ out) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float t = 0.0f;
  for (int i = 0; i < n; ++i) t += part[(int64_t)i * N + c];
  gst<T>(out, c, t);
}

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

// Row ranges of slope_kernel: some thousand workgroups, ranges of whole row groups.
static int64_t slope_ranges(int64_t M, int64_t N) {
  const int64_t by_cols = ceil_div(N, 256);
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(M, 4 * kSlopeRows), 2048 / std::max<int64_t>(1, by_cols)));
}

template <typename T, int MODE>
static int launch_f32(const Args& p, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.cols, 64), (unsigned)ceil_div(p.rows, 64));
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

template <int MODE, bool TAIL>
static int launch_tiles(const Args& p, hipStream_t st) {
  auto tiles = [&](int b) { return ceil_div(p.rows, b) * ceil_div(p.cols, b); };
  if (tiles(256) >= 192)
    hipLaunchKernelGGL((tile_kernel<Big<MODE, TAIL>, MODE>), dim3((unsigned)dense::tiles_grid(tiles(256))), dim3(256), 0, st,
                       p);
  else
    hipLaunchKernelGGL((tile_kernel<Small<MODE, TAIL>, MODE>), dim3((unsigned)dense::tiles_grid(tiles(128))), dim3(256), 0,
                       st, p);
  return check_launch();
}
template <int MODE>
static int launch_tiles(const Args& p, hipStream_t st) {
  return p.red % dense::BKS ? launch_tiles<MODE, true>(p, st) : launch_tiles<MODE, false>(p, st);
}

static int launch_product(int mode, const Args& p, int dtype, hipStream_t st) {
  if (p.rows == 0 || p.cols == 0) return MTX_OK;
  if (!p.out || (p.red > 0 && (!p.a || !p.b))) return MTX_ERR_ARG;
  if (dtype == MTX_BF16 && takes_tiles(mode, p))
    return mode == FWD ? launch_tiles<FWD>(p, st) : mode == DX ? launch_tiles<DX>(p, st) : launch_tiles<DW>(p, st);
#define MTX_F32_MODE(T) \
  (mode == FWD ? launch_f32<T, FWD>(p, st) : mode == DX ? launch_f32<T, DX>(p, st) : launch_f32<T, DW>(p, st))
  return dtype == MTX_F32 ? MTX_F32_MODE(float) : MTX_F32_MODE(uint16_t);
#undef MTX_F32_MODE
}

}  // namespace lin
}  // namespace mtx

using namespace mtx;

extern "C" int64_t mtx_linear_workspace_size(int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K < 0 || N < 0) return -1;
  return lin::slope_ranges(M, N) * N * 4;
}

extern "C" int mtx_linear(const void* x, const void* w, const void* bias, const void* residual, int dtype, int64_t M,
                          int64_t K, int64_t N, int act, void* out, void* pre, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  const int rc = lin::check_sizes(dtype, M, K, N);
  if (rc != MTX_OK) return rc;
  if (act < MTX_ACT_NONE || act > MTX_ACT_GELU_TANH) return MTX_ERR_ARG;
  if (workspace_bytes < mtx_linear_workspace_size(M, K, N)) return MTX_ERR_WORKSPACE;
  const lin::Args p{x, w, out, bias, residual, pre, act, (int)M, (int)N, (int)K};
  return lin::launch_product(lin::FWD, p, dtype, (hipStream_t)stream);
}

extern "C" int mtx_linear_dx(const void* dz, const void* w, int dtype, int64_t M, int64_t K, int64_t N, void* dx,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = lin::check_sizes(dtype, M, K, N);
  if (rc != MTX_OK) return rc;
  if (workspace_bytes < mtx_linear_workspace_size(M, K, N)) return MTX_ERR_WORKSPACE;
  const lin::Args p{dz, w, dx, nullptr, nullptr, nullptr, MTX_ACT_NONE, (int)M, (int)K, (int)N};
  return lin::launch_product(lin::DX, p, dtype, (hipStream_t)stream);
}

extern "C" int mtx_linear_dw(const void* x, const void* dz, int dtype, int64_t M, int64_t K, int64_t N, void* dw,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = lin::check_sizes(dtype, M, K, N);
  if (rc != MTX_OK) return rc;
  if (workspace_bytes < mtx_linear_workspace_size(M, K, N)) return MTX_ERR_WORKSPACE;
  const lin::Args p{x, dz, dw, nullptr, nullptr, nullptr, MTX_ACT_NONE, (int)K, (int)N, (int)M};
  return lin::launch_product(lin::DW, p, dtype, (hipStream_t)stream);
}

extern "C" int mtx_linear_act_bwd(const void* dy, const void* pre, int dtype, int64_t M, int64_t N, int act, void* dz,
                                  void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = lin::check_sizes(dtype, M, 0, N);
  if (rc != MTX_OK) return rc;
  if (act < MTX_ACT_NONE || act > MTX_ACT_GELU_TANH) return MTX_ERR_ARG;
  if (workspace_bytes < mtx_linear_workspace_size(M, 0, N) || (dbias && N > 0 && !workspace)) return MTX_ERR_WORKSPACE;
  if (N == 0 || (act == MTX_ACT_NONE && !dbias)) return MTX_OK;
  if (M > 0 && (!dy || (act != MTX_ACT_NONE && (!pre || !dz)))) return MTX_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
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
  const int e = check_launch();
  if (e != MTX_OK || !dbias) return e;
  const dim3 grid((unsigned)ceil_div(N, 256));
  if (dtype == MTX_F32)
    hipLaunchKernelGGL(lin::column_sum_kernel<float>, grid, dim3(256), 0, st, part, (int)ranges, N, (float*)dbias);
  else
    hipLaunchKernelGGL(lin::column_sum_kernel<uint16_t>, grid, dim3(256), 0, st, part, (int)ranges, N, (uint16_t*)dbias);
  return check_launch();
}

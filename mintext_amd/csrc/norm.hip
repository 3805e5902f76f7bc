// Layer norm and RMS norm over rows, with the residual's addition in front and the backward pass.
//
//   h = x + residual, rounded to the tensors' type;  d = h - mean(h) (RMS: d = h);  n = d rstd,
//   rstd = 1 / sqrt(mean(d^2) + eps);  y = n w + b
//   u = dy w;  dx = rstd (u - mean(u) - n mean(u n)) + dh (RMS: without mean(u));  dw = sum n dy;  db = sum dy
//
// A row lies in the registers of WPR waves, 16 values a lane, so that memory is read and written once and the
// variance is taken from the differences to the mean.  Sums are in f32.
#include "common.h"
#include "f32_tile.h"
#include <algorithm>
#include <type_traits>

namespace mtx {
namespace norm {

constexpr int kPer = 16;       // values a lane
constexpr int kMaxD = 16384;   // 16 waves of them

struct Args {
  const void *x, *residual, *weight, *bias;  // residual, bias: or nullptr
  void *y, *h;                               // h: or nullptr (no residual)
  float *mean, *rstd;                        // [T], or nullptr
  int64_t T;
  int D;
  float eps;
  bool w32;                                  // weight and bias in f32, else in the tensors' type
};

// Sums over the WPR waves of a row of N values a lane; `s`: 16 x N floats of the workgroup, one set for each call in turn.
template <int WPR, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] += lane_xchg<0>(v[i]);
    v[i] += lane_xchg<1>(v[i]);
    v[i] += lane_xchg<2>(v[i]);
    v[i] += lane_xchg<3>(v[i]);
    v[i] += lane_xchg<4>(v[i]);
    v[i] += lane_xchg<5>(v[i]);
  }
  if constexpr (WPR > 1) {
    const int wave = threadIdx.x >> 6, first = wave / WPR * WPR;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < WPR; ++w) v[i] += s[first + w][i];
    }
  }
}

// The lane's values of a row: block i of NV at column (i * WPR * 64 + index of the lane in the row) * VEC
template <int VEC, int WPR>
__device__ __forceinline__ int column(int i) {
  return (i * WPR * 64 + (int)(threadIdx.x % (WPR * 64))) * VEC;
}
template <typename T, int VEC, int WPR>
__device__ __forceinline__ void load_row(const T* p, int D, float (&v)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer / VEC; ++i) {
    const int c = column<VEC, WPR>(i);
    if constexpr (VEC == 8) {
      float t[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (c < D) ld8(p, c, t);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[i * 8 + q] = t[q];
    } else {
      v[i] = c < D ? gld<T>(p, c) : 0.0f;
    }
  }
}
// The same in two steps, so that bf16 rows can be on their way while another is worked on, in half the registers.
template <int WPR>
__device__ __forceinline__ void fetch_row(const uint16_t* p, int D, v4u32 (&raw)[kPer / 8]) {
#pragma unroll
  for (int i = 0; i < kPer / 8; ++i) {
    const int c = column<8, WPR>(i);
    raw[i] = c < D ? *(const v4u32*)(p + c) : v4u32{0u, 0u, 0u, 0u};
  }
}
__device__ __forceinline__ void unpack_row(const v4u32 (&raw)[kPer / 8], float (&v)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer / 8; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[i * 8 + 2 * q] = __uint_as_float(raw[i][q] << 16);
      v[i * 8 + 2 * q + 1] = __uint_as_float(raw[i][q] & 0xffff0000u);
    }
}
template <typename T, int VEC, int WPR>
__device__ __forceinline__ void store_row(T* p, int D, const float (&v)[kPer]) {
#pragma unroll
  for (int i = 0; i < kPer / VEC; ++i) {
    const int c = column<VEC, WPR>(i);
    if (c >= D) continue;
    if constexpr (VEC == 8) st8(p, c, &v[i * 8]);
    else gst<T>(p, c, v[i]);
  }
}
// the wave's row among the workgroup's, in a scalar register: rows' addresses are then scalar too
template <int WPR>
__device__ __forceinline__ int row_of_wave() {
  return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) / WPR;
}
// weight or bias, in either type
template <typename T, int VEC, int WPR>
__device__ __forceinline__ void load_param(const void* p, bool w32, int D, float (&v)[kPer]) {
  if (w32) load_row<float, VEC, WPR>((const float*)p, D, v);
  else load_row<T, VEC, WPR>((const T*)p, D, v);
}
template <typename T> __device__ __forceinline__ float rounded(float v);
template <> __device__ __forceinline__ float rounded<float>(float v) { return v; }
template <> __device__ __forceinline__ float rounded<uint16_t>(float v) { return bf16_to_f32(f32_to_bf16(v)); }

template <typename T, bool RMS, int VEC, int WPR>
__global__ __launch_bounds__(WPR > 4 ? WPR * 64 : 256) void forward_kernel(Args p) {
  constexpr int GROUPS = WPR > 4 ? 1 : 4 / WPR;
  __shared__ float s[2][16][1];
  const int64_t row = (int64_t)blockIdx.x * GROUPS + row_of_wave<WPR>();
  const bool live = row < p.T;
  const int64_t at = (live ? row : p.T - 1) * p.D;  // rows past the last work on it again, and store nothing
  float v[kPer], w[kPer], b[kPer];
  load_row<T, VEC, WPR>((const T*)p.x + at, p.D, v);
  load_param<T, VEC, WPR>(p.weight, p.w32, p.D, w);
  if (!RMS && p.bias) load_param<T, VEC, WPR>(p.bias, p.w32, p.D, b);
  if (p.residual) {
    float r[kPer];
    load_row<T, VEC, WPR>((const T*)p.residual + at, p.D, r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = rounded<T>(v[i] + r[i]);
    if (live) store_row<T, VEC, WPR>((T*)p.h + at, p.D, v);
  }
  float mean = 0.0f;
  if constexpr (!RMS) {
    float t[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) t[0] += v[i];
    row_sum<WPR, 1>(t, s[0]);
    mean = t[0] / (float)p.D;
  }
  float t[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (column<VEC, WPR>(i / VEC) >= p.D) continue;
    v[i] -= mean;
    t[0] += v[i] * v[i];
  }
  row_sum<WPR, 1>(t, s[1]);
  const float rstd = 1.0f / sqrtf(t[0] / (float)p.D + p.eps);
  if (!live) return;
  if (p.rstd && threadIdx.x % (WPR * 64) == 0) {
    p.rstd[row] = rstd;
    if (!RMS) p.mean[row] = mean;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    v[i] = v[i] * rstd * w[i];
    if (!RMS && p.bias) v[i] += b[i];
  }
  store_row<T, VEC, WPR>((T*)p.y + at, p.D, v);
}

struct BwdArgs {
  const void *dy, *dh, *h, *weight;  // dh: or nullptr
  const float *mean, *rstd;
  void* dx;                          // or nullptr
  float* part;                       // [workgroups][1 or 2][D]: sums of n dy, of dy; or nullptr
  int64_t T;
  int D;
  bool w32, bias;
};

// A workgroup of one row's waves, eight at least, takes every gridDim.x-th set of rows; a lane's columns are the same in all
// of them, so its share of dw and db stays in registers until the end.  Eight waves leave registers for the next row's
// values on their way.
constexpr int backward_waves(int wpr) { return wpr > 8 ? wpr : 8; }
template <typename T, bool RMS, int VEC, int WPR>
__global__ __launch_bounds__(backward_waves(WPR) * 64) void backward_kernel(BwdArgs p) {
  constexpr int GROUPS = backward_waves(WPR) / WPR;
  __shared__ float s[2][16][2];
  __shared__ float sums[GROUPS > 1 ? WPR * 64 * kPer : 1];
  const int group = row_of_wave<WPR>();
  float w[kPer], dw[kPer], db[kPer];
  load_param<T, VEC, WPR>(p.weight, p.w32, p.D, w);
#pragma unroll
  for (int i = 0; i < kPer; ++i) dw[i] = db[i] = 0.0f;
  // AHEAD: the next row's values are loaded before this one's are worked on
  constexpr bool AHEAD = std::is_same<T, uint16_t>::value && VEC == 8 && WPR <= 8;
  v4u32 next_h[kPer / 8], next_dy[kPer / 8], next_dh[kPer / 8];
  auto fetch = [&](int64_t base) {
    if constexpr (AHEAD) {
      const int64_t at = min(base + group, p.T - 1) * p.D;
      fetch_row<WPR>((const uint16_t*)p.h + at, p.D, next_h);
      fetch_row<WPR>((const uint16_t*)p.dy + at, p.D, next_dy);
      if (p.dh) fetch_row<WPR>((const uint16_t*)p.dh + at, p.D, next_dh);
    }
  };
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  fetch((int64_t)blockIdx.x * GROUPS);
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.T; base += step, turn ^= 1) {
    const int64_t row = base + group;
    const bool live = row < p.T;
    const int64_t r = live ? row : p.T - 1, at = r * p.D;
    float n[kPer], u[kPer];
    v4u32 dh[kPer / 8];
    if constexpr (AHEAD) {
      unpack_row(next_h, n);
      unpack_row(next_dy, u);
#pragma unroll
      for (int i = 0; i < kPer / 8; ++i) dh[i] = next_dh[i];
      if (base + step < p.T) fetch(base + step);
    } else {
      load_row<T, VEC, WPR>((const T*)p.h + at, p.D, n);
      load_row<T, VEC, WPR>((const T*)p.dy + at, p.D, u);
    }
    const float rstd = p.rstd[r], mean = RMS ? 0.0f : p.mean[r];
    float t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      n[i] = (n[i] - mean) * rstd;  // past the row's end u is 0, which keeps it out of the sums
      if (live) {
        dw[i] += n[i] * u[i];
        if (!RMS) db[i] += u[i];
      }
      u[i] *= w[i];
      t[0] += u[i] * n[i];
      t[1] += u[i];
    }
    row_sum<WPR, 2>(t, s[turn]);
    if (!p.dx || !live) continue;
    const float c = t[0] / (float)p.D, m = RMS ? 0.0f : t[1] / (float)p.D;
#pragma unroll
    for (int i = 0; i < kPer; ++i) u[i] = (u[i] - m - n[i] * c) * rstd;
    if (p.dh) {
      if constexpr (AHEAD) unpack_row(dh, n);
      else load_row<T, VEC, WPR>((const T*)p.dh + at, p.D, n);
#pragma unroll
      for (int i = 0; i < kPer; ++i) u[i] += n[i];
    }
    store_row<T, VEC, WPR>((T*)p.dx + at, p.D, u);
  }
  if (!p.part) return;
  const int lanes = WPR * 64, lane = threadIdx.x % lanes;
  const int kinds = p.bias ? 2 : 1;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k >= kinds || (RMS && k > 0)) break;
    float* v = k ? db : dw;
    if constexpr (GROUPS > 1) {  // the groups' sums in order
      for (int g = 0; g < GROUPS; ++g) {
        __syncthreads();
        if (group == g) {
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            float* o = &sums[i * lanes + lane];
            v[i] = g ? *o + v[i] : v[i];
            *o = v[i];
          }
        }
      }
    }
    if (group == GROUPS - 1) {
      float* out = p.part + ((int64_t)blockIdx.x * kinds + k) * p.D;
      store_row<float, VEC, WPR>(out, p.D, *(float(*)[kPer])v);
    }
  }
}

// the workgroups' sums, in order: 32 columns and eight sums of every eighth workgroup each; blockIdx.y: dw, db
template <typename T>
__global__ __launch_bounds__(256) void columns_kernel(const float* __restrict__ part, int n, int kinds, int D, T* dw, T* db) {
  __shared__ float s[8][32];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, k = blockIdx.y;
  const int c = blockIdx.x * 32 + tx;
  float t = 0.0f;
  if (c < D) {
#pragma unroll 8
    for (int i = ty; i < n; i += 8) t += part[((int64_t)i * kinds + k) * D + c];
  }
  s[ty][tx] = t;
  __syncthreads();
  if (ty > 0 || c >= D) return;
  for (int y = 1; y < 8; ++y) t += s[y][tx];
  gst<T>(k ? db : dw, c, t);
}

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
static int waves(int D) {  // of a row
  int w = 1;
  while (w * 64 * kPer < D) w *= 2;
  return w;
}
static int groups(int64_t T, int D) {  // workgroups of the backward pass: one a CU
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(T, backward_waves(waves(D)) / waves(D)), 256));
}
static int check_sizes(int dtype, int weight_dtype, int64_t T, int64_t D) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return MTX_ERR_ARG;
  if (weight_dtype != MTX_F32 && weight_dtype != dtype) return MTX_ERR_ARG;
  if (T < 0 || D <= 0) return MTX_ERR_ARG;
  if (D > kMaxD || T > (int64_t)1 << 30) return MTX_ERR_UNSUPPORTED;
  return MTX_OK;
}

#define MTX_WAVES(KERNEL, T, RMS, VEC, D, GRID, THREADS, ST, P)                                          \
  switch (waves(D)) {                                                                                    \
    case 1: hipLaunchKernelGGL((KERNEL<T, RMS, VEC, 1>), GRID(1), THREADS(1), 0, ST, P); break;          \
    case 2: hipLaunchKernelGGL((KERNEL<T, RMS, VEC, 2>), GRID(2), THREADS(2), 0, ST, P); break;          \
    case 4: hipLaunchKernelGGL((KERNEL<T, RMS, VEC, 4>), GRID(4), THREADS(4), 0, ST, P); break;          \
    case 8: hipLaunchKernelGGL((KERNEL<T, RMS, VEC, 8>), GRID(8), THREADS(8), 0, ST, P); break;          \
    default: hipLaunchKernelGGL((KERNEL<T, RMS, VEC, 16>), GRID(16), THREADS(16), 0, ST, P);             \
  }
#define MTX_KINDS(KERNEL, RMS, DTYPE, VEC8, D, GRID, THREADS, ST, P)                                     \
  if (DTYPE == MTX_F32) {                                                                                \
    if (VEC8) {                                                                                          \
      if (RMS) { MTX_WAVES(KERNEL, float, true, 8, D, GRID, THREADS, ST, P) }                            \
      else { MTX_WAVES(KERNEL, float, false, 8, D, GRID, THREADS, ST, P) }                               \
    } else {                                                                                             \
      if (RMS) { MTX_WAVES(KERNEL, float, true, 1, D, GRID, THREADS, ST, P) }                            \
      else { MTX_WAVES(KERNEL, float, false, 1, D, GRID, THREADS, ST, P) }                               \
    }                                                                                                    \
  } else {                                                                                               \
    if (VEC8) {                                                                                          \
      if (RMS) { MTX_WAVES(KERNEL, uint16_t, true, 8, D, GRID, THREADS, ST, P) }                         \
      else { MTX_WAVES(KERNEL, uint16_t, false, 8, D, GRID, THREADS, ST, P) }                            \
    } else {                                                                                             \
      if (RMS) { MTX_WAVES(KERNEL, uint16_t, true, 1, D, GRID, THREADS, ST, P) }                         \
      else { MTX_WAVES(KERNEL, uint16_t, false, 1, D, GRID, THREADS, ST, P) }                            \
    }                                                                                                    \
  }

}  // namespace norm
}  // namespace mtx

using namespace mtx;

extern "C" int mtx_norm(const void* x, const void* residual, const void* weight, const void* bias, int dtype,
                        int weight_dtype, int rms, int64_t T, int64_t D, float eps, void* y, void* h, float* mean, float* rstd,
                        void* stream) {
  using namespace norm;
  const int rc = check_sizes(dtype, weight_dtype, T, D);
  if (rc != MTX_OK) return rc;
  if ((rms && bias) || !(eps >= 0.0f)) return MTX_ERR_ARG;
  if (T == 0) return MTX_OK;
  if (!x || !weight || !y || (residual && !h) || (rstd && !rms && !mean)) return MTX_ERR_ARG;
  const Args p{x, residual, weight, bias, y, h, mean, rstd, T, (int)D, eps, weight_dtype == MTX_F32};
  const bool vec = D % 8 == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) && aligned16(bias) && aligned16(y) &&
                   aligned16(h);
  hipStream_t st = (hipStream_t)stream;
#define MTX_GRID(W) dim3((unsigned)ceil_div(T, W > 4 ? 1 : 4 / W))
#define MTX_THREADS(W) dim3(W > 4 ? W * 64 : 256)
  MTX_KINDS(forward_kernel, rms, dtype, vec, (int)D, MTX_GRID, MTX_THREADS, st, p)
#undef MTX_GRID
#undef MTX_THREADS
  return check_launch();
}

extern "C" int64_t mtx_norm_bwd_workspace_size(int64_t T, int64_t D) {
  if (T < 0 || D <= 0 || D > norm::kMaxD) return -1;
  return (int64_t)norm::groups(T, (int)D) * 2 * D * 4;
}

extern "C" int mtx_norm_bwd(const void* dy, const void* dh, const void* h, const void* weight, const float* mean,
                            const float* rstd, int dtype, int weight_dtype, int rms, int64_t T, int64_t D, void* dx,
                            void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace norm;
  const int rc = check_sizes(dtype, weight_dtype, T, D);
  if (rc != MTX_OK) return rc;
  if (dbias && (rms || !dweight)) return MTX_ERR_ARG;
  if (!dx && !dweight) return MTX_OK;
  if (T > 0 && (!dy || !h || !weight || !rstd || (!rms && !mean))) return MTX_ERR_ARG;
  const bool sums = dweight != nullptr;
  if (sums && (!workspace || !aligned16(workspace) || workspace_bytes < mtx_norm_bwd_workspace_size(T, D)))
    return MTX_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const int n = T > 0 ? groups(T, (int)D) : 0, kinds = dbias ? 2 : 1;
  if (T > 0) {
    const BwdArgs p{dy, dh, h, weight, mean, rstd, dx, sums ? (float*)workspace : nullptr, T, (int)D, weight_dtype == MTX_F32,
                    dbias != nullptr};
    const bool vec = D % 8 == 0 && aligned16(dy) && aligned16(dh) && aligned16(h) && aligned16(weight) && aligned16(dx);
#define MTX_GRID(W) dim3((unsigned)n)
#define MTX_THREADS(W) dim3(backward_waves(W) * 64)
    MTX_KINDS(backward_kernel, rms, dtype, vec, (int)D, MTX_GRID, MTX_THREADS, st, p)
#undef MTX_GRID
#undef MTX_THREADS
  }
  if (!sums) return check_launch();
  const dim3 grid((unsigned)ceil_div(D, 32), (unsigned)kinds);
  if (weight_dtype == MTX_F32)
    hipLaunchKernelGGL(columns_kernel<float>, grid, dim3(256), 0, st, (const float*)workspace, n, kinds, (int)D, (float*)dweight,
                       (float*)dbias);
  else
    hipLaunchKernelGGL(columns_kernel<uint16_t>, grid, dim3(256), 0, st, (const float*)workspace, n, kinds, (int)D,
                       (uint16_t*)dweight, (uint16_t*)dbias);
  return check_launch();
}

// Layer norm and RMS norm over rows, with the residual's addition in front and the backward pass.
//
//   h = x + residual, rounded to the tensors' type;  d = h - mean(h) (RMS: d = h);  n = d rstd,
//   rstd = 1 / sqrt(mean(d^2) + eps);  y = n w + b
//   u = dy w;  dx = rstd (u - mean(u) - n mean(u n)) + dh (RMS: without mean(u));  dw = sum n dy;  db = sum dy
//
// Bound by memory.  A row lies in the registers of 8 to 1024 lanes, in chunks of eight consecutive values, 8 or 16 values a
// lane, so that memory is read and written once and the variance is taken from the differences to the mean.  Sums are in f32.
// Rows of any length and alignment are read and written in the same 16-byte accesses, which need no alignment beyond an
// element's (single elements: bf16 rows of 2047 took 135 us forward and 500 backward).
// Layer norm of 134 MB in bf16 (forward moves 268 MB, backward 402), us:
//   D          64    200   512   1024  2048  4096  8192  16384  2047  4100
//   forward    57    72    59    40    40    40    41    43     42    64     6.7 TB/s at 4096
//   backward   95    108   84    90    84    77    85    107    95    143    5.2 TB/s at 4096
// RMS norm: 39 to 50 and 75 to 124.
#include "common.h"
#include "f32_tile.h"
#include <algorithm>
#include <type_traits>

namespace mtx {
namespace norm {

constexpr int kMaxD = 16384;  // 1024 lanes of 16

struct Args {
  const void *x, *residual, *weight, *bias;  // residual, bias: or nullptr
  void *y, *h;                               // h: or nullptr (no residual)
  float *mean, *rstd;                        // [T], or nullptr
  int64_t T;
  int D;
  float eps;
};

// Sums of N values over the LANES lanes of a row; `s`: a set of the workgroup's for each call in turn (more than one wave).
template <int LANES, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] += lane_xchg<0>(v[i]);
    v[i] += lane_xchg<1>(v[i]);
    v[i] += lane_xchg<2>(v[i]);
    if constexpr (LANES >= 16) v[i] += lane_xchg<3>(v[i]);
    if constexpr (LANES >= 32) v[i] += lane_xchg<4>(v[i]);
    if constexpr (LANES >= 64) v[i] += lane_xchg<5>(v[i]);
  }
  if constexpr (LANES > 64) {
    constexpr int W = LANES / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[wave][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[i] += s[first + w][i];
    }
  }
}

// the lane's row among the workgroup's; where a wave has one row, in a scalar register, and so are the row's addresses
template <int LANES>
__device__ __forceinline__ int row_of_lane() {
  if constexpr (LANES >= 64) return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) / (LANES / 64);
  else return threadIdx.x / LANES;
}
// first column of the lane's chunk i
template <int LANES>
__device__ __forceinline__ int column(int i) {
  return (i * LANES + (int)(threadIdx.x % LANES)) * 8;
}
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Chunk {  // eight values as they lie in memory
  uint32_t v[2 * sizeof(T)];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(v[i]);
    else return __uint_as_float(i % 2 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
  }
};
template <typename T>
__device__ __forceinline__ Chunk<T> packed(const float* v) {
  Chunk<T> c;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int q = 0; q < 8; ++q) c.v[q] = __float_as_uint(v[q]);
  } else {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
#pragma unroll
    for (int q = 0; q < 4; ++q) c.v[q] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * q], (__bf16)v[2 * q + 1]});
  }
  return c;
}
// A row is loaded in two steps.  load_chunk() is one access whatever the row's length, so that nothing waits for it where rows
// are ahead: a chunk that ends behind the row is the row's last eight values instead.  tidy_chunk(), before the values are
// used, moves them to their places, with zeros behind the end.  (Loads under a condition and zeros beside them, which wait for
// the load into the same registers: 16381 x 7168 backward 214 us.)  Rows of fewer than eight go element by element.
template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p, int at, int D) {
  if (D >= 8) return *(const Chunk<T>*)(p + min(at, D - 8));
  Chunk<T> c;
#pragma unroll
  for (int q = 0; q < (int)(2 * sizeof(T)); ++q) c.v[q] = 0u;
#pragma unroll
  for (int q = 0; q < 7; ++q) {
    if (at + q >= D) continue;
    if constexpr (sizeof(T) == 4) c.v[q] = __float_as_uint(p[at + q]);
    else c.v[q / 2] |= (uint32_t)p[at + q] << (16 * (q & 1));
  }
  return c;
}
template <typename T>
__device__ __forceinline__ void tidy_chunk(Chunk<T>& c, int at, int D) {
  constexpr int W = 2 * sizeof(T), EACH = 4 / sizeof(T);  // words; values in one
  const int by = at + 8 - D;  // values to move down
  if (by <= 0 || D < 8) return;
  if (by & 1) {
#pragma unroll
    for (int q = 0; q < W; ++q) {
      const uint32_t up = q + 1 < W ? c.v[q + 1 < W ? q + 1 : q] : 0u;
      c.v[q] = EACH == 1 ? up : __builtin_amdgcn_alignbit(up, c.v[q], 16);
    }
  }
#pragma unroll
  for (int step = 2; step < 8; step *= 2) {
    if (!(by & step)) continue;
#pragma unroll
    for (int q = 0; q < W; ++q) c.v[q] = q + step / EACH < W ? c.v[q + step / EACH < W ? q + step / EACH : q] : 0u;
  }
  if (by >= 8) {
#pragma unroll
    for (int q = 0; q < W; ++q) c.v[q] = 0u;
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, int at, int D, const Chunk<T>& c) {
  if (at + 8 <= D) {
    *(Chunk<T>*)(p + at) = c;
    return;
  }
#pragma unroll
  for (int q = 0; q < 7; ++q) {
    if (at + q >= D) continue;
    if constexpr (sizeof(T) == 4) p[at + q] = c[q];
    else p[at + q] = (uint16_t)(c.v[q / 2] >> (16 * (q & 1)));
  }
}
// A lane's N values of a row.
template <typename T, int LANES, int N>
struct Row {
  Chunk<T> c[N / 8];
  __device__ __forceinline__ void load(const T* p, int D) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) c[i] = load_chunk<T>(p, column<LANES>(i), D);
  }
  __device__ __forceinline__ void tidy(int D) {
    if (D == LANES * N) return;  // every lane has whole chunks
#pragma unroll
    for (int i = 0; i < N / 8; ++i) tidy_chunk<T>(c[i], column<LANES>(i), D);
  }
  __device__ __forceinline__ float operator[](int i) const { return c[i / 8][i % 8]; }
};

// T: of the rows, W: of weight and bias
template <typename T, typename W, bool RMS, int LANES, int N>
__global__ __launch_bounds__(LANES > 256 ? LANES : 256) void forward_kernel(Args p) {
  constexpr int ROWS = LANES > 256 ? 1 : 256 / LANES;
  __shared__ float s[2][16][1];
  const int64_t row = (int64_t)blockIdx.x * ROWS + row_of_lane<LANES>();
  const bool live = row < p.T;
  const int64_t at = (live ? row : p.T - 1) * p.D;  // rows past the last work on it again, and store nothing
  const int D = p.D;
  float v[N];
  Row<W, LANES, N> w, b;
  {
    Row<T, LANES, N> x, r;
    x.load((const T*)p.x + at, D);
    if (p.residual) r.load((const T*)p.residual + at, D);
    w.load((const W*)p.weight, D);
    if (!RMS && p.bias) b.load((const W*)p.bias, D);
    x.tidy(D);
    if (p.residual) {
      r.tidy(D);
#pragma unroll
      for (int c = 0; c < N / 8; ++c) {
        if (column<LANES>(c) >= D) continue;
        float sum[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) sum[q] = x.c[c][q] + r.c[c][q];
        x.c[c] = packed<T>(sum);
        if (live) store_chunk<T>((T*)p.h + at, column<LANES>(c), D, x.c[c]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x[i];
  }
  float mean = 0.0f;
  if constexpr (!RMS) {
    float t[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) t[0] += v[i];
    row_sum<LANES, 1>(t, s[0]);
    mean = t[0] / (float)D;
  }
  float t[1] = {0.0f};
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    const int left = D - column<LANES>(c);
    if (left <= 0) continue;
#pragma unroll
    for (int q = 0; q < 8; ++q) v[c * 8 + q] -= mean;
    if (!RMS && left < 8) {  // nothing behind the row's end
#pragma unroll
      for (int q = 1; q < 8; ++q) v[c * 8 + q] = q < left ? v[c * 8 + q] : 0.0f;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) t[0] += v[c * 8 + q] * v[c * 8 + q];
  }
  row_sum<LANES, 1>(t, s[1]);
  const float rstd = 1.0f / sqrtf(t[0] / (float)D + p.eps);
  w.tidy(D);
  if (!RMS && p.bias) b.tidy(D);
  if (!live) return;
  if (p.rstd && threadIdx.x % LANES == 0) {
    p.rstd[row] = rstd;
    if (!RMS) p.mean[row] = mean;
  }
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    if (column<LANES>(c) >= D) continue;
    float y[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      y[q] = v[c * 8 + q] * rstd * w.c[c][q];
      if (!RMS && p.bias) y[q] += b.c[c][q];
    }
    store_chunk<T>((T*)p.y + at, column<LANES>(c), D, packed<T>(y));
  }
}

struct BwdArgs {
  const void *dy, *dh, *h, *weight;  // dh: or nullptr
  const float *mean, *rstd;
  void* dx;                          // or nullptr
  float* part;                       // [workgroups][1 or 2][D]: sums of n dy, of dy; or nullptr
  int64_t T;
  int D;
  bool bias;
};

// A workgroup of 512 lanes, or one row's, takes every gridDim.x-th set of rows; a lane's columns are the same in all of them, so
// its share of dw and db stays in registers until the end.  The next row's values are on their way while one is worked on (two
// rows ahead were no faster, or slower: 8192 x 4096 39 us, one ahead 35).
constexpr int backward_lanes(int lanes) { return lanes > 512 ? lanes : 512; }
template <typename T, typename W, bool RMS, int LANES, int N>
__global__ __launch_bounds__(backward_lanes(LANES)) void backward_kernel(BwdArgs p) {
  constexpr int ROWS = backward_lanes(LANES) / LANES;
  // The registers of a workgroup of 1024 lanes (128 each) hold one row's values; the layer norm's spills 7 (bf16), 9 (with f32
  // weights) or 13 (f32) of them, part of its 107 us for D of 16384.
  constexpr bool AHEAD = LANES <= 512;
  __shared__ float s[2][16][2];
  __shared__ float sums[ROWS > 1 ? LANES * N : 1];
  const int mine = row_of_lane<LANES>(), D = p.D;
  Row<W, LANES, N> w;
  w.load((const W*)p.weight, D);
  w.tidy(D);
  float dw[N], db[N];
#pragma unroll
  for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.0f;
  struct Values {
    Row<T, LANES, N> h, dy, dh;
    float mean, rstd;
  };
  auto fetch = [&](Values& v, int64_t base) {
    const int64_t r = min(base + mine, p.T - 1), at = r * D;
    v.h.load((const T*)p.h + at, D);
    v.dy.load((const T*)p.dy + at, D);
    if (AHEAD && p.dh) v.dh.load((const T*)p.dh + at, D);
    v.rstd = p.rstd[r];
    v.mean = RMS ? 0.0f : p.mean[r];
  };
  auto work = [&](Values& v, int64_t base, int turn) {
    v.h.tidy(D);
    v.dy.tidy(D);
    const int64_t row = base + mine;
    const bool live = row < p.T;
    float t[2] = {0.0f, 0.0f}, n[N], u[N];
    // behind the row's end dy and w are 0, which keeps it out of the sums
#pragma unroll
    for (int c = 0; c < N / 8; ++c) {
      if (column<LANES>(c) >= D) continue;
#pragma unroll
      for (int i = c * 8; i < c * 8 + 8; ++i) {
        const float g = v.dy[i];
        n[i] = (v.h[i] - v.mean) * v.rstd;
        u[i] = g * w[i];
        if (live) {
          dw[i] += n[i] * g;
          if (!RMS) db[i] += g;
        }
        t[0] += u[i] * n[i];
        if (!RMS) t[1] += u[i];
      }
    }
    if constexpr (RMS) row_sum<LANES, 1>((float(&)[1])t, (float(*)[1])s[turn]);
    else row_sum<LANES, 2>(t, s[turn]);
    if (!p.dx || !live) return;
    const float k = t[0] / (float)D, m = RMS ? 0.0f : t[1] / (float)D;
#pragma unroll
    for (int c = 0; c < N / 8; ++c) {
      const int at = column<LANES>(c);
      if (at >= D) continue;
      float d[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) d[q] = (u[c * 8 + q] - m - n[c * 8 + q] * k) * v.rstd;
      if (p.dh) {  // where no row is ahead its registers are needed until here
        Chunk<T> dh = !AHEAD ? load_chunk<T>((const T*)p.dh + row * D, at, D) : v.dh.c[c];
        tidy_chunk<T>(dh, at, D);
#pragma unroll
        for (int q = 0; q < 8; ++q) d[q] += dh[q];
      }
      store_chunk<T>((T*)p.dx + row * D, at, D, packed<T>(d));
    }
  };
  const int64_t step = (int64_t)gridDim.x * ROWS;
  int64_t base = (int64_t)blockIdx.x * ROWS;
  if constexpr (!AHEAD) {
    for (int turn = 0; base < p.T; base += step, turn ^= 1) {
      Values v;
      fetch(v, base);
      work(v, base, turn);
    }
  } else {
    Values v, next;
    if (base < p.T) fetch(next, base);
    for (int turn = 0; base < p.T; base += step, turn ^= 1) {
      v = next;
      if (base + step < p.T) fetch(next, base + step);
      work(v, base, turn);
    }
  }
  if (!p.part) return;
  const int lane = threadIdx.x % LANES, kinds = p.bias ? 2 : 1;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k >= kinds || (RMS && k > 0)) break;
    float(&v)[N] = k ? db : dw;
    if constexpr (ROWS > 1) {  // the rows' sums in order
      for (int g = 0; g < ROWS; ++g) {
        __syncthreads();
        if (mine == g) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            float* o = &sums[i * LANES + lane];
            v[i] = g ? *o + v[i] : v[i];
            *o = v[i];
          }
        }
      }
    }
    if (mine == ROWS - 1) {
      float* out = p.part + ((int64_t)blockIdx.x * kinds + k) * D;
#pragma unroll
      for (int c = 0; c < N / 8; ++c) {
        const Chunk<float> x = packed<float>(&v[c * 8]);
        if (column<LANES>(c) < D) store_chunk<float>(out, column<LANES>(c), D, x);
      }
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
static int lanes(int D) {  // of a row: of 8 values up to 512 columns, of 16 behind that
  int n = 8;
  while (n * (D <= 512 ? 8 : 16) < D) n *= 2;
  return n;
}
// Workgroups of the backward pass: one a CU, two where 8 values a lane leave registers for both.
static int groups(int64_t T, int D) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(T, backward_lanes(lanes(D)) / lanes(D)), D <= 512 ? 512 : 256));
}
static int check_sizes(int dtype, int weight_dtype, int64_t T, int64_t D) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return MTX_ERR_ARG;
  if (weight_dtype != MTX_F32 && weight_dtype != dtype) return MTX_ERR_ARG;
  if (T < 0 || D <= 0) return MTX_ERR_ARG;
  if (D > kMaxD || T > (int64_t)1 << 30) return MTX_ERR_UNSUPPORTED;
  return MTX_OK;
}

template <typename T, typename W, bool RMS, int LANES, int N>
static void go_forward(const Args& p, hipStream_t st) {
  hipLaunchKernelGGL((forward_kernel<T, W, RMS, LANES, N>), dim3((unsigned)ceil_div(p.T, LANES > 256 ? 1 : 256 / LANES)),
                     dim3(LANES > 256 ? LANES : 256), 0, st, p);
}
template <typename T, typename W, bool RMS, int LANES, int N>
static void go_backward(const BwdArgs& p, hipStream_t st) {
  hipLaunchKernelGGL((backward_kernel<T, W, RMS, LANES, N>), dim3((unsigned)groups(p.T, p.D)), dim3(backward_lanes(LANES)), 0, st, p);
}
#define MTX_LANES(GO, T, W, RMS, P, ST)                       \
  switch (lanes((P).D)) {                                     \
    case 8: GO<T, W, RMS, 8, 8>(P, ST); break;                \
    case 16: GO<T, W, RMS, 16, 8>(P, ST); break;              \
    case 32: GO<T, W, RMS, 32, 8>(P, ST); break;              \
    case 64:                                                  \
      if ((P).D <= 512) GO<T, W, RMS, 64, 8>(P, ST);          \
      else GO<T, W, RMS, 64, 16>(P, ST);                      \
      break;                                                  \
    case 128: GO<T, W, RMS, 128, 16>(P, ST); break;           \
    case 256: GO<T, W, RMS, 256, 16>(P, ST); break;           \
    case 512: GO<T, W, RMS, 512, 16>(P, ST); break;           \
    default: GO<T, W, RMS, 1024, 16>(P, ST);                  \
  }
#define MTX_TYPES(GO, RMS, DTYPE, WTYPE, P, ST)               \
  if (DTYPE == MTX_F32) {                                     \
    MTX_LANES(GO, float, float, RMS, P, ST)                   \
  } else if (WTYPE == MTX_F32) {                              \
    MTX_LANES(GO, uint16_t, float, RMS, P, ST)                \
  } else {                                                    \
    MTX_LANES(GO, uint16_t, uint16_t, RMS, P, ST)             \
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
  const int64_t most = ((int64_t)1 << 31) / lanes((int)D), bytes = D * (dtype == MTX_F32 ? 4 : 2);  // a grid's threads: 32 bits
  for (int64_t t = 0; t < T; t += most) {
    auto from = [&](auto* v, int64_t each) { return v ? (decltype(v))((char*)v + t * each) : nullptr; };
    const Args p{from(x, bytes), from(residual, bytes), weight, bias, from(y, bytes), from(h, bytes), from(mean, 4), from(rstd, 4),
                 std::min(most, T - t), (int)D, eps};
    if (rms) { MTX_TYPES(go_forward, true, dtype, weight_dtype, p, (hipStream_t)stream) }
    else { MTX_TYPES(go_forward, false, dtype, weight_dtype, p, (hipStream_t)stream) }
  }
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
    const BwdArgs p{dy, dh, h, weight, mean, rstd, dx, sums ? (float*)workspace : nullptr, T, (int)D, dbias != nullptr};
    if (rms) { MTX_TYPES(go_backward, true, dtype, weight_dtype, p, st) }
    else { MTX_TYPES(go_backward, false, dtype, weight_dtype, p, st) }
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

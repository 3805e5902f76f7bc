// The products of the head's losses in f32 on the f32 matrix cores (f32_tile.h): 64 x 64 tiles of any size and alignment.  Bound by
// the tile loop, one accumulator of 32 x 32 a wave and two barriers a stage: both directions of 2048 x 2048 x 32000 take 9500 us
// (8 T D V at 113 TFLOP/s, of the 153 that a library's product of 8192 cubed reaches), of 4096 x 4096 x 32000 41400 (104).
#include "f32_tile.h"
#include "head_loss.h"
#include <type_traits>

namespace mtx {
namespace head {

using f32mm::KS;
using f32mm::NT;
constexpr int kRow = 68;  // floats of a row of the tile in LDS

// the tile to LDS, row by row; thread t then holds columns 16 (t % 4) .. of row t / 4
__device__ __forceinline__ void to_rows(const f32mm::f32x16& acc, float* lds, float v[16]) {
  const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) >> 1, wn = (threadIdx.x >> 6) & 1;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    lds[(wm * 32 + 8 * (e / 4) + 4 * (lane >> 5) + e % 4) * kRow + wn * 32 + (lane & 31)] = acc[e];
  __syncthreads();
  const float* row = lds + (threadIdx.x >> 2) * kRow + (threadIdx.x & 3) * 16;
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = row[e];
}

// PART > 0: every PART stages of the reduction make a sum of their own.
template <bool VD, bool DZ, int VEC, int PART>
__global__ __launch_bounds__(NT) void logits_f32_kernel(Logits p) {
  __shared__ __attribute__((aligned(16))) float lds[2 * f32mm::TILE];
  static_assert(64 * kRow <= 2 * f32mm::TILE, "the tile fits its operands' place");
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const float *X = (const float*)p.x, *W = (const float*)p.w;
  auto at_x = [&](int r, int c, int s) -> const float* {
    const int m = m0 + r, k = s * KS + c;
    return m < p.T && k < p.red ? X + (int64_t)m * p.ldx + k : nullptr;
  };
  auto at_w = [&](int r, int c, int s) -> const float* {
    const int n = VD ? n0 + r : n0 + c, k = VD ? s * KS + c : s * KS + r;
    return n < p.cols && k < p.red ? W + (VD ? (int64_t)n * p.ldw + k : (int64_t)k * p.ldw + n) : nullptr;
  };
  f32mm::f32x16 acc;
  if constexpr (PART == 0) {
    f32mm::mainloop<float, false, !VD, VEC>(acc, p.red, lds, lds + f32mm::TILE, at_x, at_w, X, W);
  } else {
    f32mm::f32x16 sum;
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[e] = 0.0f;
    for (int s0 = 0; s0 * KS < p.red; s0 += PART) {
      f32mm::mainloop<float, false, !VD, VEC>(
          acc, min(PART * KS, p.red - s0 * KS), lds, lds + f32mm::TILE, [&](int r, int c, int s) { return at_x(r, c, s0 + s); },
          [&](int r, int c, int s) { return at_w(r, c, s0 + s); }, X, W);
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[e] += acc[e];
    }
    acc = sum;
  }
  float v[16];
  to_rows(acc, lds, v);
  const int row = m0 + (threadIdx.x >> 2), quarter = threadIdx.x & 3, c0 = n0 + quarter * 16, left = p.cols - c0;
  const bool live = row < p.T;
  const int r = live ? row : p.T - 1;
  float* mine = lds + (threadIdx.x >> 2) * kRow;
  if constexpr (!DZ) {
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, e < left ? v[e] : -INFINITY);
    m = fmaxf(m, lane_xchg<0>(m));
    m = fmaxf(m, lane_xchg<1>(m));
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float d = m == -INFINITY ? v[e] : v[e] - m;
      s += e < left ? exp2f(d * p.scale) : 0.0f;
    }
    s += lane_xchg<0>(s);
    s += lane_xchg<1>(s);
    if (live && quarter == 0) p.part[(int64_t)((p.v0 + n0) / 64) * p.T + row] = make_float2(m, s);
    if (!live) return;
    if (p.e.targets) {
      const int64_t c = target(p.e, r) - p.v0 - n0;
      if (quarter == 0 && c >= 0 && c < 64 && c < p.cols - n0) p.chosen[row] = mine[c];
    } else {
      const uint16_t* b = p.e.bounds + r * p.e.ldb + (p.v0 + n0) / kBlock;
      for (int e = b[0] + quarter; e < b[1]; e += 4) {
        const int c = p.e.idx[(int64_t)r * p.e.K + e] - p.v0 - n0;
        if ((unsigned)c < 64u) p.chosen[(int64_t)r * p.e.K + e] = mine[c];
      }
    }
  } else {
    if (!live) return;
    float m;
    const float a = p.f.a(r, p.f.b(r), m);
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = a == 0.0f || e >= left ? 0.0f : a * exp2f((v[e] - m) * p.scale);
    float* dz = (float*)p.dz + (int64_t)row * p.ldz + c0;
    st8(dz, 0, v);
    st8(dz, 8, v + 8);
  }
}

template <bool A_COLS, bool B_COLS, int VEC>
__global__ __launch_bounds__(NT) void product_f32_kernel(Product p) {
  __shared__ __attribute__((aligned(16))) float as[f32mm::TILE], bs[f32mm::TILE];
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const float *A = (const float*)p.a, *B = (const float*)p.b;
  const int stages = (p.red + KS - 1) / KS, piece = blockIdx.z;
  const int64_t kb = (int64_t)piece * stages / p.pieces * KS, ke = min((int64_t)(piece + 1) * stages / p.pieces * KS, (int64_t)p.red);
  auto at_a = [&](int r, int c, int s) -> const float* {
    const int64_t m = m0 + (A_COLS ? c : r), k = kb + s * KS + (A_COLS ? r : c);
    return m < p.rows && k < ke ? A + (A_COLS ? k * p.lda + m : m * p.lda + k) : nullptr;
  };
  auto at_b = [&](int r, int c, int s) -> const float* {
    const int64_t n = n0 + (B_COLS ? c : r), k = kb + s * KS + (B_COLS ? r : c);
    return n < p.cols && k < ke ? B + (B_COLS ? k * p.ldb + n : n * p.ldb + k) : nullptr;
  };
  f32mm::f32x16 acc;
  f32mm::mainloop<float, A_COLS, B_COLS, VEC>(acc, (int)(ke - kb), as, bs, at_a, at_b, A, B);
  const int lane = threadIdx.x & 63, wm = (threadIdx.x >> 6) >> 1, wn = (threadIdx.x >> 6) & 1;
  const int64_t n = n0 + wn * 32 + (lane & 31);
  if (n >= p.cols) return;
  const float alpha = p.f.alpha();
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int64_t r = m0 + wm * 32 + 8 * (v / 4) + 4 * (lane >> 5) + v % 4;
    if (r >= p.rows) continue;
    float y = acc[v];
    if (p.acc) {
      float* s = p.acc + ((int64_t)piece * p.rows + r) * p.ldacc + n;
      if (p.add) y += *s;
      if (!p.last) {
        *s = y;
        continue;
      }
    }
    ((float*)p.out)[r * p.ldo + n] = y * alpha;
  }
}

static bool quads(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 4 == 0; }

template <bool VD, bool DZ>
static int go_logits(const Logits& p, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.cols, 64), (unsigned)ceil_div(p.T, 64));
  // a whole row of four is inside or outside: of the reduction in x (and W [V][D]), of the columns in W [D][V]
  const bool vec = quads(p.x, p.ldx) && quads(p.w, p.ldw) && p.red % 4 == 0 && (VD || p.cols % 4 == 0);
  // Few rows' gradients are as far off as their few large logits, 7e-6 for 4 x 1324 x 10624 in one run of sums and 0.7e-6 this
  // way.  Over many rows it evens out: 100 x 1000 x 3000 1.3e-6 and 0.5e-6.  64 x 2048 x 32000 takes 385 us in both directions
  // in one run of sums, 401 this way.
  const bool parts = p.T <= kTwoRows;
  if (vec && parts) hipLaunchKernelGGL((logits_f32_kernel<VD, DZ, 4, 4>), grid, dim3(NT), 0, st, p);
  else if (vec) hipLaunchKernelGGL((logits_f32_kernel<VD, DZ, 4, 0>), grid, dim3(NT), 0, st, p);
  else if (parts) hipLaunchKernelGGL((logits_f32_kernel<VD, DZ, 1, 4>), grid, dim3(NT), 0, st, p);
  else hipLaunchKernelGGL((logits_f32_kernel<VD, DZ, 1, 0>), grid, dim3(NT), 0, st, p);
  return check_launch();
}
int launch_logits_f32(const Logits& p, bool dz, int order, hipStream_t st) {
  if (order == ORDER_VD) return dz ? go_logits<true, true>(p, st) : go_logits<true, false>(p, st);
  return dz ? go_logits<false, true>(p, st) : go_logits<false, false>(p, st);
}

template <bool A_COLS, bool B_COLS>
static int go_product(const Product& p, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.cols, 64), (unsigned)ceil_div(p.rows, 64), (unsigned)p.pieces);
  // a quad that begins inside may end behind the rows, columns or reduction elements where there is something to read: dz has
  // zeros there, and what other operands give is multiplied by them or not stored
  const bool vec = quads(p.a, p.lda) && quads(p.b, p.ldb) && (A_COLS ? p.a_left >= round_up(p.rows, 4) : p.lda >= round_up(p.red, 4)) &&
                   (B_COLS ? p.b_left >= round_up(p.cols, 4) : p.red % 4 == 0);
  if (vec) hipLaunchKernelGGL((product_f32_kernel<A_COLS, B_COLS, 4>), grid, dim3(NT), 0, st, p);
  else hipLaunchKernelGGL((product_f32_kernel<A_COLS, B_COLS, 1>), grid, dim3(NT), 0, st, p);
  return check_launch();
}
int launch_product_f32(const Product& p, bool a_cols, bool b_cols, hipStream_t st) {
  if (a_cols) return go_product<true, true>(p, st);
  return b_cols ? go_product<false, true>(p, st) : go_product<false, false>(p, st);
}

}  // namespace head
}  // namespace mtx

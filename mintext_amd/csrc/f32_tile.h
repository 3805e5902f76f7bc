// Matrix products on the f32 matrix cores: the tile loop of the f32 kernels, and of the bf16 ones at widths and
// alignments that the bf16 matrix-core kernels do not take.
#pragma once
#include "common.h"
#include <type_traits>

namespace mtx {

// ---- element access of the kernels that take either type --------------------------------------
template <typename T> __device__ __forceinline__ float gld(const T* p, int64_t i);
template <> __device__ __forceinline__ float gld<float>(const float* p, int64_t i) { return p[i]; }
template <> __device__ __forceinline__ float gld<uint16_t>(const uint16_t* p, int64_t i) { return bf16_to_f32(p[i]); }
template <typename T> __device__ __forceinline__ void gst(T* p, int64_t i, float v);
template <> __device__ __forceinline__ void gst<float>(float* p, int64_t i, float v) { p[i] = v; }
template <> __device__ __forceinline__ void gst<uint16_t>(uint16_t* p, int64_t i, float v) { p[i] = f32_to_bf16(v); }

// ---- f32 path on the f32 matrix cores -------------------------------------------------------------
// 64x64 output tiles, 4 waves of 32x32, 32-deep reduction stages through LDS with the next stage's
// operands loaded into registers meanwhile.  v_mfma_f32_32x32x2_f32 multiplies and accumulates in f32
// at twice the rate of the unpacked FMAs, and needs two LDS values per lane for 64 cycles of work
// where the FMA tile needed 8 per 64.  Measured, FMA kernel -> this: 16384 rows in 16 groups x 1024 x
// 1024 forward 710 -> 329 us (104 TFLOP/s), dlhs 850 -> 332, tgmm 774 -> 333; 4000 rows in 16 skewed
// groups, 512 x 768: 95 -> 45, 150 -> 50, 320 -> 54; 512 rows in 8 groups, 256 x 128: 30 -> 13.  Any
// size and alignment: VEC = 4 moves 16 bytes at a time (every row 16-byte aligned), VEC = 1 single
// values.  Values past the end are zeros in both operands.  T: float, or bf16 where the rows have no
// alignment that the bf16 matrix-core kernels take (VEC = 1).
namespace f32mm {
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
constexpr int BM = 64, BN = 64, KS = 32, NT = 256;
constexpr int RS = KS + 4;  // LDS row of a k-contiguous operand: [64][RS]
constexpr int CS = 64 + 8;  // LDS row of an operand stored [k][64]: the half-waves' rows 4 k apart differ by 32 banks
constexpr int TILE = 64 * RS > KS * CS ? 64 * RS : KS * CS;

// One operand tile of 64 rows x KS reduction elements (COLS = false: the reduction contiguous in
// memory) or KS reduction elements x 64 columns (COLS = true).  at(r, c) is where row r, column c is,
// or nullptr.
template <typename T, bool COLS, int VEC>
struct Stage {
  static_assert(VEC == 1 || std::is_same<T, float>::value, "16-byte loads are of f32");
  static constexpr int W = COLS ? 64 : KS, H = COLS ? KS : 64, N = W * H / NT / VEC;
  // bf16: values as loaded and a bit for each that exists; the others load `any`, a valid address.  A load
  // with its conversion inside the condition was waited for before the next one was issued (tgmm of 4096
  // rows in 4 groups, 500 x 250: 167 us, 81 this way; f32 needs no conversion and is faster with the
  // condition).  Reduction elements past `left` (a multiple of 8) are skipped.
  static constexpr bool BF16 = std::is_same<T, uint16_t>::value;
  T v[N][VEC];
  uint32_t have;
  static_assert(!BF16 || N <= 32, "a bit a value");
  template <typename At>
  __device__ __forceinline__ void load(At at, const T* any, int left, int tid) {
    have = 0;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int q = tid + u * NT, r = q / (W / VEC), c = q % (W / VEC) * VEC;
      if (BF16 && COLS && r >= left) continue;
      const T* src = at(r, c);
      if constexpr (BF16) {
        v[u][0] = *(src ? src : any);
        have |= src ? 1u << u : 0u;
      } else if constexpr (VEC == 4) {
        const f32x4 x = src ? *(const f32x4*)src : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][i] = x[i];
      } else {
        v[u][0] = src ? *src : 0.0f;
      }
    }
  }
  __device__ __forceinline__ void store(float* lds, int left, int tid) const {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int q = tid + u * NT, r = q / (W / VEC), c = q % (W / VEC) * VEC;
      if (BF16 && COLS && r >= left) continue;
      float* dst = lds + r * (COLS ? CS : RS) + c;
      if constexpr (VEC == 4) *(f32x4*)dst = f32x4{v[u][0], v[u][1], v[u][2], v[u][3]};
      else if constexpr (BF16) *dst = (have >> u) & 1 ? bf16_to_f32(v[u][0]) : 0.0f;
      else *dst = v[u][0];
    }
  }
};
// The 16 operand values of a lane for a stage: row or column x0 + lane % 32; MFMA m of the stage
// multiplies reduction elements k = 8 (m / 4) + 4 (lane / 32) + m % 4 (the same for both operands).
template <bool COLS>
__device__ __forceinline__ void fragment(const float* lds, int x0, int lane, float f[16]) {
  const int x = x0 + (lane & 31), h = lane >> 5;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (COLS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * q + i] = lds[(8 * q + 4 * h + i) * CS + x];
    } else {
      const f32x4 v = *(const f32x4*)(lds + x * RS + 8 * q + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[4 * q + i] = v[i];
    }
  }
}
// acc of lane l, element v: row 8 (v / 4) + 4 (l / 32) + v % 4, column l % 32 of the wave's 32x32 tile.
// nred: reduction elements; any_a, any_b: valid addresses of the operands (for nred > 0).
template <typename T, bool ACOLS, bool BCOLS, int VEC, typename AtA, typename AtB>
__device__ __forceinline__ void mainloop(f32x16& acc, int nred, float* as, float* bs, AtA at_a, AtB at_b, const T* any_a,
                                         const T* any_b) {
  constexpr bool BF16 = std::is_same<T, uint16_t>::value;
  const int nk = (nred + KS - 1) / KS;
  const int tid = threadIdx.x, lane = tid & 63, wm = (tid >> 6) >> 1, wn = (tid >> 6) & 1;
  Stage<T, ACOLS, VEC> a;
  Stage<T, BCOLS, VEC> b;
#pragma unroll
  for (int v = 0; v < 16; ++v) acc[v] = 0.0f;
  // bf16: a last stage of few elements (tgmm of small groups) does no more than the eights of them
  auto elements = [&](int s) { return BF16 ? min(KS, (nred - s * KS + 7) & ~7) : KS; };
  auto load = [&](int s) {
    a.load([&](int r, int c) { return at_a(r, c, s); }, any_a, elements(s), tid);
    b.load([&](int r, int c) { return at_b(r, c, s); }, any_b, elements(s), tid);
  };
  if (nk > 0) load(0);
  // one LDS buffer: a second one saves a barrier a stage but halves the workgroups per CU (5-9 % slower)
  for (int s = 0; s < nk; ++s) {
    const int left = elements(s);
    a.store(as, left, tid);
    b.store(bs, left, tid);
    __syncthreads();
    if (s + 1 < nk) load(s + 1);
    float fa[16], fb[16];
    fragment<ACOLS>(as, wm * 32, lane, fa);
    fragment<BCOLS>(bs, wn * 32, lane, fb);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (BF16 && 8 * q >= left) continue;
#pragma unroll
      for (int m = 4 * q; m < 4 * q + 4; ++m) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[m], fb[m], acc, 0, 0, 0);
    }
    __syncthreads();
  }
}

}  // namespace f32mm
}  // namespace mtx

// What the kernels of the head's losses share: a row's target entries, and the arguments of the products.
//
// Of T tokens x [T][D] and the head's weight W the logits z = x W [T][V] are made tile by tile and never stored:
//   forward   a tile leaves, for each row and block of columns, the maximum m and sum exp((z - m) / tau), and the logits of the
//             row's entries; merge_kernel joins the blocks.
//   backward  the vocabulary goes through in pieces: z of a piece again, dz = a softmax(z / tau) - b share (one entry for
//             cross entropy, a teacher's top ones for distillation) rounded to the operands' type into a workspace, from which
//             dx += dz W^T (in f32) and dW of the piece = x^T dz.  A factor that all rows share (1 / count, the gradient of
//             the one loss) is left to the products' results: with it in dz, every row's -1 + q is rounded alike where q is
//             small, and the gradients of 4096 x 4096 x 32000 were 2.8e-3 off instead of 2.0e-3.
// So a step computes 8 T D V operations, 2 of them for the logits made again, and holds kPiece bytes of dz at most, or 320 columns
// of it where T is so large that those are more.
#pragma once
#include "common.h"

namespace mtx {
namespace head {

enum { ORDER_DV = 0, ORDER_VD = 1 };  // of the weight in memory
// Rows up to which precision comes first: bf16 dz in two planes, logits in several sums.  A gradient of few rows hangs on
// few values of dz, whose roundings do not even out: 1 x 64 x 32768 bf16 3.4e-3 off with one plane and 1.5e-3, the result's own
// rounding, with two; 300 x 2000 x 3000 2.4e-3 of 1.7e-3 with one.  Both directions of 48 x 2048 x 32000 take 147 us, with one
// plane 132; 128 rows 197 and 159.
constexpr int kTwoRows = 64;
constexpr int kBlock = 128;           // columns an entry of Entries::bounds stands for

// The classes of a row that its loss names.  Cross entropy: targets[row], int32 or int64.  Distillation: idx and share of
// row * K .., ascending, and bounds[row * ldb + b], the first of them at column 128 b or behind.
struct Entries {
  const void* targets;
  int wide;  // targets are int64
  const int32_t* idx;
  const float* share;
  const uint16_t* bounds;
  int64_t ldb;
  int K;
};
__device__ __forceinline__ int64_t target(const Entries& e, int64_t row) {
  return e.wide ? ((const int64_t*)e.targets)[row] : ((const int32_t*)e.targets)[row];
}

// A row's factors in the backward pass, dz = a softmax - b share, and the one of all rows that is left to the products' results.
struct Factors {
  const float *g, *count;    // the gradient of the one loss and what its sum was divided by; or of each row's, and nullptr
  const float *stats, *state;  // [T][2]: the row's largest logit m and sum exp((z - m) / tau); [T]
  float unit, z_loss;
  __device__ __forceinline__ float b(int64_t row) const {
    const float s = state[row];
    return s == 0.0f ? 0.0f : count ? s : s * unit * g[row];
  }
  // a / sum, so that a softmax is that times exp((z - m) / tau).  Not exp(z / tau - lse): where lse is 15, its rounding alone is
  // 4e-7 of every value of the row, and f32 gradients of 4 x 1324 x 10624 were 8e-6 off.
  __device__ __forceinline__ float a(int64_t row, float b, float& m) const {
    const float s = stats[2 * row + 1];
    m = stats[2 * row];
    if (b == 0.0f) return 0.0f;
    return (z_loss == 0.0f ? b : b * (1.0f + 2.0f * z_loss * (m + logf(s)))) / s;  // z_loss: tau is 1
  }
  __device__ __forceinline__ float alpha() const { return count ? unit * (g[0] / *count) : 1.0f; }
};

struct Logits {
  const void *x, *w;  // w: at column v0
  int64_t ldx, ldw;
  int T, red, missing;  // missing: reduction elements that x has (as zeros) and w has not
  int v0, cols;         // columns of this piece
  int w_left;           // columns of w that can be read
  Entries e;
  float scale;          // log2(e) / tau
  // forward
  float2* part;         // [block][T]: maximum of z, sum of exp2((z - maximum) scale)
  float* chosen;        // [T][K]: z of the entries
  // backward
  Factors f;
  void* dz;             // [planes][T][ldz], zeros behind the piece's columns
  int planes;           // 2: what the rounding took, rounded itself, stands behind dz
  int64_t ldz;
};

// C = A B of a gradient, rows x cols, in `pieces` of the reduction
struct Product {
  const void *a, *b;
  int64_t lda, ldb;
  int rows, cols, red, missing;  // missing: of B at the reduction's end
  int a_left, b_left;            // rows or columns of the operands that can be read
  void* out;
  int64_t ldo;
  int pieces;
  float* acc;                    // [pieces][rows][ldacc] f32, or nullptr: straight to out
  int64_t ldacc;
  int add;                       // acc holds sums of earlier calls
  int last;                      // pieces == 1: the result goes to out
  Factors f;                     // of which alpha
};

// Eight values of a row, or the `left` that exist, in accesses that need no alignment beyond an element's.  (Element by
// element the gradient of a weight of 704 x 50257 took 199 us, so 159.)
__device__ __forceinline__ void store_part(uint16_t* o, const float v[8], int left) {
  typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
  struct __attribute__((packed, aligned(2))) Chunk {
    uint32_t v[4];
  };
  const Chunk c = __builtin_bit_cast(Chunk, bf16x8{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3], (__bf16)v[4],
                                                   (__bf16)v[5], (__bf16)v[6], (__bf16)v[7]});
  if (left >= 8) {
    *(Chunk*)o = c;
  } else {
#pragma unroll
    for (int q = 0; q < 7; ++q)
      if (q < left) o[q] = (uint16_t)(c.v[q / 2] >> (16 * (q & 1)));
  }
}
__device__ __forceinline__ void store_part(float* o, const float v[8], int left) {
  struct __attribute__((packed, aligned(4))) Chunk {
    float v[8];
  };
  if (left >= 8) {
    *(Chunk*)o = Chunk{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int q = 0; q < 7; ++q)
      if (q < left) o[q] = v[q];
  }
}

int launch_logits(const Logits& p, bool dz, int order, int path, hipStream_t st);  // bf16
int launch_product(const Product& p, bool a_cols, bool b_cols, int size, hipStream_t st);
int launch_logits_f32(const Logits& p, bool dz, int order, hipStream_t st);
int launch_product_f32(const Product& p, bool a_cols, bool b_cols, hipStream_t st);

enum { SIZE_BIG, SIZE_SMALL };  // tiles of launch_product: 256 x 256, 128 x 128
// tiles of the logits: 256 x 256, 128 x 128, 64 x 128 (up to kTwoRows, the ones that write two planes of dz); f32 64 x 64
enum { PATH_BIG, PATH_SMALL, PATH_THIN, PATH_F32 };
inline int tile_cols(int path) { return path == PATH_BIG ? 256 : path == PATH_F32 ? 64 : 128; }
inline int block_cols(int path) { return path == PATH_BIG ? 128 : 64; }  // of a partial maximum and sum

}  // namespace head
}  // namespace mtx

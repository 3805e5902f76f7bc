// The losses of a vocabulary-sized head without its logits in memory: softmax cross entropy and distillation from a
// teacher's top logits, with their gradients.  What the products' kernels do is in head_loss.h; here are the kernels beside
// them and the order in which they run.
//
//   cross entropy   L_t = lse_t - z[t, y_t] + c lse_t^2,  dz = g_t ((1 + 2 c lse_t) softmax(z_t) - onehot(y_t))
//   distillation    p = softmax(teacher / tau) over the row's entries, q = softmax(z / tau),
//                   L_t = tau^2 sum_k p_k (log p_k - log q[i_k]),  dz = g_t tau (q - sum_k p_k onehot(i_k))
//
// A row's state is 1, 0 (left out: the ignored class, no entry; its loss is 0 and its gradient too) or NaN (a class
// that is none), which its loss and its gradient become.
#include "head_loss.h"
#include <algorithm>

namespace mtx {
namespace head {

constexpr int kMaxEntries = 1024;
constexpr float kLog2e = 1.4426950408889634f;

// ---- a teacher's entries: shares, in the order of their classes ------------------------------------------------
// A wave takes a row and sorts keys of (class, place in the row) in LDS, in a bitonic network.  8192 rows of 64 entries take 20
// us, of 256 50, of 1024 175 (with the rank of each key among all others 90 and 940).
struct Prep {
  const void *idx, *logits;
  int wide, f32;  // int64 indices; f32 logits (else bf16)
  int64_t T, V;
  int K;
  float inv_tau;
  int32_t* sorted;
  float* share;
  uint16_t* bounds;
  int64_t ldb;
  float2* row;  // state, sum p log p
};
__device__ __forceinline__ float wave_sum(float v) {
  v += lane_xchg<0>(v);
  v += lane_xchg<1>(v);
  v += lane_xchg<2>(v);
  v += lane_xchg<3>(v);
  v += lane_xchg<4>(v);
  return v + lane_xchg<5>(v);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, lane_xchg<0>(v));
  v = fmaxf(v, lane_xchg<1>(v));
  v = fmaxf(v, lane_xchg<2>(v));
  v = fmaxf(v, lane_xchg<3>(v));
  v = fmaxf(v, lane_xchg<4>(v));
  return fmaxf(v, lane_xchg<5>(v));
}
constexpr uint32_t kNoClass = (1u << 22) - 1;  // behind every class: check_sizes() allows fewer
static_assert(kMaxEntries <= 1024, "ten bits of a key");
__global__ __launch_bounds__(64) void entries_kernel(Prep p) {
  __shared__ uint32_t key[kMaxEntries];
  __shared__ float val[kMaxEntries];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x, base = row * p.K;
  float m = -INFINITY;
  bool bad = false;
  for (int k = lane; k < p.K; k += 64) {
    const int64_t i = p.wide ? ((const int64_t*)p.idx)[base + k] : ((const int32_t*)p.idx)[base + k];
    const float t = p.f32 ? ((const float*)p.logits)[base + k] : bf16_to_f32(((const uint16_t*)p.logits)[base + k]);
    const bool live = i >= 0 && !(t == -INFINITY);  // NaN and +inf count, and leave the row no shares
    bad |= i >= p.V || (live && !(t < INFINITY));
    key[k] = (live && i < p.V ? (uint32_t)i : kNoClass) << 10 | (uint32_t)k;
    val[k] = t;
    if (live) m = fmaxf(m, t);
  }
  int n = 1;
  while (n < p.K) n *= 2;
  for (int k = p.K + lane; k < n; k += 64) key[k] = UINT32_MAX;  // before none
  m = wave_max(m);
  const bool invalid = __ballot(bad) != 0;
  __syncthreads();
  // (t - m) / tau, which the type's lowest value does not leave as a product with 1 / tau might
  float sum = 0.0f, count = 0.0f;
  for (int k = lane; k < p.K; k += 64) {
    if (key[k] >> 10 == kNoClass) continue;
    sum += expf((val[k] - m) * p.inv_tau);
    count += 1.0f;
  }
  sum = wave_sum(sum);
  count = wave_sum(count);
  const float log_sum = logf(sum);
  float entropy = 0.0f;
  for (int size = 2; size <= n; size *= 2)
    for (int step = size / 2; step > 0; step /= 2) {
      for (int t = lane; t < n / 2; t += 64) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const uint32_t x = key[i], y = key[j];
        const bool turn = (x > y) == ((i & size) == 0);
        key[i] = turn ? y : x;
        key[j] = turn ? x : y;
      }
      __syncthreads();
    }
  for (int k = lane; k < p.K; k += 64) {
    const uint32_t i = key[k] >> 10;
    const float d = (val[key[k] & 1023] - m) * p.inv_tau, share = i == kNoClass ? 0.0f : expf(d) / sum;
    if (share > 0.0f || share != share) entropy += share * (d - log_sum);
    p.sorted[base + k] = (int32_t)i;
    p.share[base + k] = share;
  }
  entropy = wave_sum(entropy);
  if (lane == 0) p.row[row] = make_float2(invalid ? NAN : count > 0.0f ? 1.0f : 0.0f, entropy);
  const int live = (int)count;
  for (int64_t b = lane; b < p.ldb; b += 64) {
    const int64_t first = b * kBlock;
    int lo = 0, hi = live;  // the first entry at `first` or behind
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (key[mid] >> 10 < first) lo = mid + 1;
      else hi = mid;
    }
    p.bounds[row * p.ldb + b] = (uint16_t)lo;
  }
}

// ---- the blocks' maxima and sums, and the row's loss -------------------------------------------------------
struct Merge {
  const float2* part;
  int64_t blocks, T, V;
  Entries e;
  const float2* row;  // distillation: state, sum p log p
  const float* chosen;
  int64_t ignore;
  float scale, inv_tau, unit, z_loss;  // unit: tau^2
  float *loss, *stats, *state;         // loss: [T]
};
struct Sum {  // of exp2((z - m) scale)
  float m, s;
  __device__ __forceinline__ void join(float om, float os, float scale) {  // -inf with -inf: a sum of 0
    const float n = fmaxf(m, om);
    s = s * exp2f(m == n ? 0.0f : (m - n) * scale) + os * exp2f(om == n ? 0.0f : (om - n) * scale);
    m = n;
  }
};
// blocks first, first + step, .. of a row
__device__ __forceinline__ Sum sum_blocks(const Merge& p, int64_t row, int64_t first, int64_t step) {
  Sum a{-INFINITY, 0.0f};
  int64_t b = first;
  for (; b + 3 * step < p.blocks; b += 4 * step) {
    float2 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = p.part[(b + u * step) * p.T + row];
#pragma unroll
    for (int u = 0; u < 4; ++u) a.join(v[u].x, v[u].y, p.scale);
  }
  for (; b < p.blocks; b += step) {
    const float2 v = p.part[b * p.T + row];
    a.join(v.x, v.y, p.scale);
  }
  return a;
}
// share of entries first, first + step, .. in sum p (m - z) / tau, whose terms are small where the share is not
__device__ __forceinline__ float below_max(const Merge& p, int64_t row, float m, int first, int step) {
  float below = 0.0f;
  if (p.e.targets) return below;
  const int64_t at = row * p.e.K;
  const int n = p.e.bounds[row * p.e.ldb + p.e.ldb - 1];
  for (int k = first; k < n; k += step) {
    const float w = p.e.share[at + k];
    if (w != 0.0f) below += w * ((m - p.chosen[at + k]) * p.inv_tau);
  }
  return below;
}
__device__ __forceinline__ void finish_row(const Merge& p, int64_t row, const Sum& a, float below) {
  float state, konst = 0.0f;
  if (p.e.targets) {
    const int64_t y = target(p.e, row);
    state = y == p.ignore ? 0.0f : y < 0 || y >= p.V ? NAN : 1.0f;
    if (state == 1.0f) below = a.m - p.chosen[row];
  } else {
    state = p.row[row].x;
    konst = p.row[row].y;
  }
  const float log_sum = logf(a.s), lse = a.m * p.inv_tau + log_sum;
  float loss = p.unit * (konst + below + log_sum);
  if (p.z_loss != 0.0f) loss += p.z_loss * lse * lse;
  p.loss[row] = state == 0.0f ? 0.0f : state * loss;
  p.stats[2 * row] = a.m;
  p.stats[2 * row + 1] = a.s;
  p.state[row] = state;
}
// 32 rows a workgroup, eight threads a row, joined in order: neighbours read neighbouring rows' blocks.  4096 rows of 250
// blocks 9 us, 4093 of 1024 28 us.
__global__ __launch_bounds__(256) void merge_kernel(Merge p) {
  __shared__ float ms[8][32], ss[8][32];
  const int tx = threadIdx.x % 32, g = threadIdx.x / 32;
  const int64_t row = (int64_t)blockIdx.x * 32 + tx;
  const bool live = row < p.T;
  Sum a{-INFINITY, 0.0f};
  if (live) a = sum_blocks(p, row, g, 8);
  ms[g][tx] = a.m;
  ss[g][tx] = a.s;
  __syncthreads();
  a = Sum{ms[0][tx], ss[0][tx]};
  for (int i = 1; i < 8; ++i) a.join(ms[i][tx], ss[i][tx], p.scale);
  float below = live ? below_max(p, row, a.m, g, 8) : 0.0f;
  __syncthreads();
  ms[g][tx] = below;
  __syncthreads();
  if (g > 0 || !live) return;
  for (int i = 1; i < 8; ++i) below += ms[i][tx];
  finish_row(p, row, a, below);
}
// A wave a row, for fewer rows than would fill the chip the other way.
template <int S>
__device__ __forceinline__ void wave_join(Sum& a, float scale) {
  if constexpr (S < 6) {
    const float m = lane_xchg<S>(a.m), s = lane_xchg<S>(a.s);
    a.join(m, s, scale);
    wave_join<S + 1>(a, scale);
  }
}
__global__ __launch_bounds__(256) void merge_wave_kernel(Merge p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= p.T) return;
  const int lane = threadIdx.x & 63;
  Sum a = sum_blocks(p, row, lane, 64);
  wave_join<0>(a, p.scale);
  const float below = wave_sum(below_max(p, row, a.m, lane, 64));
  if (lane == 0) finish_row(p, row, a, below);
}

// The sum of the rows' losses and what it is divided by, in 64 bits and one workgroup's order.
__global__ __launch_bounds__(1024) void total_kernel(const float* loss, const float* state, int64_t T, int mean, float* out,
                                                     float* count) {
  __shared__ double s[16][2];
  double sum = 0.0, n = 0.0;
  for (int64_t t = threadIdx.x; t < T; t += 1024) {
    sum += loss[t];
    n += state[t] == 0.0f ? 0.0 : 1.0;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    sum += __shfl_xor(sum, d);
    n += __shfl_xor(n, d);
  }
  if ((threadIdx.x & 63) == 0) {
    s[threadIdx.x >> 6][0] = sum;
    s[threadIdx.x >> 6][1] = n;
  }
  __syncthreads();
  if (threadIdx.x > 0) return;
  for (int w = 1; w < 16; ++w) {
    sum += s[w][0];
    n += s[w][1];
  }
  n = mean ? fmax(n, 1.0) : 1.0;
  *out = (float)(sum / n);
  *count = (float)n;
}

// ---- backward -----------------------------------------------------------------------------------------------------
// dz of the entries among columns v0 .. v0 + cols, from their logits: a softmax - b (the shares of one class), in the place
// of what the tile left there.  A thread an entry; the first of several of one class takes them all.
struct Named {
  Entries e;
  Factors f;
  const float* chosen;
  float scale;
  int64_t T;
  int v0, cols;
  void* dz;
  int64_t ldz;
  int f32, planes;
};
__global__ __launch_bounds__(256) void named_kernel(Named p) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= p.T * p.e.K) return;
  const int64_t t = at / p.e.K;
  const float b = p.f.b(t);
  if (b == 0.0f) return;
  int64_t c;
  float share = 1.0f;
  if (p.e.targets) {
    c = target(p.e, t);
  } else {
    c = p.e.idx[at];
    if (at > t * p.e.K && p.e.idx[at - 1] == c) return;
    share = p.e.share[at];
  }
  c -= p.v0;
  if (c < 0 || c >= p.cols) return;
  if (!p.e.targets)
    for (int64_t k = at + 1; k < (t + 1) * p.e.K && p.e.idx[k] == c + p.v0; ++k) share += p.e.share[k];
  float m;
  const float a = p.f.a(t, b, m), v = a * exp2f((p.chosen[at] - m) * p.scale) - b * share;
  if (p.f32) {
    ((float*)p.dz)[t * p.ldz + c] = v;
    return;
  }
  uint16_t* dz = (uint16_t*)p.dz + t * p.ldz + c;
  *dz = f32_to_bf16(v);
  if (p.planes == 2) dz[p.T * p.ldz] = f32_to_bf16(v - bf16_to_f32(*dz));
}

// rows x cols of a bf16 matrix into one with rows of `ld` (a multiple of 8), zeros behind the columns.  `in` lies on a 4-byte
// boundary and has rows of any length: eight elements come as the words that hold them, shifted by one where the first is odd.
// `times` such matrices, one behind the other.
__global__ __launch_bounds__(256) void pad_kernel(const uint16_t* __restrict__ in, int64_t ldi, int64_t rows, int64_t cols,
                                                  uint16_t* __restrict__ out, int64_t ld, int times) {
  struct __attribute__((aligned(4))) Words {
    uint32_t v[4];
  };
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= times * rows * ld) return;
  const int64_t at = i / ld, r = at % rows, c = i - at * ld, e = r * ldi + c, end = (rows - 1) * ldi + cols;
  v4u32 o = {0u, 0u, 0u, 0u};
  if (c < cols) {
    if (e + 9 < end) {  // all the words lie inside
      const uint32_t* p = (const uint32_t*)in + (e >> 1);
      const Words w = *(const Words*)p;
      const uint32_t next = p[4], odd = (e & 1) * 16;
#pragma unroll
      for (int q = 0; q < 4; ++q) o[q] = __builtin_amdgcn_alignbit(q < 3 ? w.v[q < 3 ? q + 1 : 3] : next, w.v[q], odd);
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (e + q < end) o[q / 2] |= (uint32_t)in[e + q] << (16 * (q & 1));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {  // what lies behind the row's end
      const int64_t left = cols - c - 2 * q;
      if (left < 2) o[q] &= left < 1 ? 0u : 0xFFFFu;
    }
  }
  *(v4u32*)(out + i) = o;
}

// out = the pieces' sums, in order.  Eight columns a thread; rows of acc are whole eights.  32 sums of 61 x 1536 take 5.9 us (one
// at a time 11.5, in workgroups of 256 7.2), 14 of 1531 x 704 12.7 (13.5).
template <typename T>
__global__ __launch_bounds__(64) void join_kernel(const float* __restrict__ acc, int pieces, int64_t rows, int64_t cols,
                                                   int64_t ldacc, T* __restrict__ out, int64_t ldo, Factors factors) {
  const float f = factors.alpha();
  const int64_t per = (cols + 7) / 8, i = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t r = i / per, c = i % per * 8, at = r * ldacc + c, n = rows * ldacc;
  float v[8];
  ld8(acc, at, v);
  int s = 1;
  for (; s + 4 <= pieces; s += 4) {  // four on their way at a time
    float o[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u) ld8(acc + (s + u) * n, at, o[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += o[u][q];
  }
  for (; s < pieces; ++s) {
    float o[8];
    ld8(acc + s * n, at, o);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] += o[q];
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] *= f;
  store_part(out + r * ldo + c, v, (int)min(cols - c, (int64_t)8));
}

// ---- how a call runs, by its sizes alone --------------------------------------------------------------------------
// Bytes of dz held at a time, at most (or those of 256 columns and kTurn), and of a padded copy of the weight's columns (or of 256).
constexpr int64_t kPiece = (int64_t)1 << 30, kCopy = (int64_t)256 << 20;
constexpr int kTurn = 64;  // elements more than a piece in a row of dz, so that rows are no power of two apart in memory
constexpr int kMostPieces = 16;

struct Split {
  int size;  // bf16: of the tiles
  int pieces;
};
// A product's tiles and pieces by an estimate of its time in us: rounds of the chip by what a stage of 32 takes and a tile's way
// in and out, and what the pieces' sums take to write, read and join.  dx by itself, with dz before it (us):
//   61 x 1536 x 32000    128 x 128 in 16 pieces 52, in 8 65, in 4 90; 256 x 256 in 16 67
//   256 x 2048 x 32000   128 x 128 in 8 pieces 100, in 16 111, in 4 129; 256 x 256 in 16 102
//   1531 x 704 x 50256   256 x 256 in 14 pieces 274, in 8 294, in 1 1058; 128 x 128 in 8 380
//   4093 x 2048 x 131072 256 x 256 in 2 pieces 3826, in 4 3958, in 1 5000; 128 x 128 in 1 4783
// and dW of 8000 x 512 x 4000 128 x 128 in 4 pieces 97, in 1 119, in 16 154; 256 x 256 in 8 107, in 1 203.  Where a tile has few
// stages, as dW of few rows, the ways out decide: 128 x 2048 x 32000 in both directions 149 with 128 x 128 tiles of dW, 160 with
// 256 x 256; 128 x 4096 x 131072 1155 and 1198, 128 x 2048 x 65536 354 and 343.
static Split split(bool f32, int64_t rows, int64_t cols, int64_t red) {
  const int64_t stages = ceil_div(red, 32);
  Split best{SIZE_BIG, 1};
  double least = 1e30;
  for (int kind = 0; kind < (f32 ? 1 : 2); ++kind) {
    const int64_t side = f32 ? 64 : kind ? 128 : 256, slots = f32 ? 512 : kind ? 512 : 256;
    const int64_t tiles = ceil_div(rows, side) * ceil_div(cols, side);
    for (int s = 1; s <= kMostPieces && (s == 1 || stages / s >= 8); ++s) {
      const double stage = f32 ? 0.9 : kind == 0 ? 0.7 : tiles * s > 256 ? 0.6 : 0.35;  // two small tiles a CU, or one
      const double out = f32 ? 4.0 : kind ? 4.5 : 12.0;
      const double t = ceil_div(tiles * s, slots) * (ceil_div(stages, s) * stage + out) +
                       (s > 1 ? s * rows * cols * 8 / 4e6 + 6.0 : 0.0);
      if (t < least) {
        least = t;
        best = {kind, s};
      }
    }
  }
  return best;
}

struct Plan {
  bool f32;
  int64_t T, D, V, ldx, red;  // ldx: x's row length in use; red: reduction elements of the logits
  int order;
  bool copy_x, copy_w;
  int planes;                // of dz, and copies of x behind one another
  int64_t piece;             // columns of a piece, a multiple of 256
  int path;
  Split dx, dw;
  int join_dx;               // sums of dx to be joined: the reduction's pieces, of each plane
  int64_t ld_dx, ld_dw, rows_dw;
  // bytes from the workspace's start
  int64_t x, w, part, dz, acc_dx, acc_dw, total;
};
static Plan plan(int dtype, int64_t T, int64_t D, int64_t V, int order, bool backward) {
  Plan p{};
  p.f32 = dtype == MTX_F32;
  p.T = T, p.D = D, p.V = V, p.order = order;
  const int64_t size = p.f32 ? 4 : 2, all = round_up(V, 256);
  p.planes = !p.f32 && backward && T <= kTwoRows ? 2 : 1;
  const bool odd = !p.f32 && D % 8 != 0;
  p.copy_x = odd || p.planes == 2;
  p.copy_w = !p.f32 && (order == ORDER_DV ? V : D) % 8 != 0;
  // Copies have rows of whole 128-byte lines: 4000 x 1001 x 50257 takes 438 us forward and 1230 backward, with rows of 1008
  // elements, which begin inside lines, 485 and 1335.  x's zeros end whole stages where the weight is copied too.
  p.ldx = odd ? round_up(D, 64) : D;
  p.red = odd ? round_up(D, order == ORDER_VD ? 32 : 8) : D;
  int64_t most = std::min(all, std::max<int64_t>(((int64_t)1 << 38) / T / 256 * 256, 256));  // threads of a grid: 2^30
  if (p.copy_w) most = std::min(most, std::max<int64_t>(kCopy / (p.ldx * 2) / 256 * 256, 256));
  if (backward) most = std::min(most, std::max<int64_t>((kPiece / (p.planes * T * size) - kTurn) / 256 * 256, 256));
  p.piece = round_up(ceil_div(V, ceil_div(all, most)), 256);
  const int64_t big = ceil_div(T, 256) * ceil_div(p.piece, 256);
  // Forward in 256 x 256, 128 x 128 and 64 x 128 tiles (us): 48 x 2048 x 32000 54.3, 31.2, 30.2; 65 rows 52.9, 31.2, 37.6; 256 rows
  // 54.1, 47.2, 58.2; 512 x 2048 x 16384 (128 large tiles) 51.5, 44.4, 53.3; 1024 x 2048 x 12288 (192) 57.3, 62.6; 1024 x 2048 x
  // 32000 (500) 120, 147.  Both directions of 128 x 4096 x 131072 take 1242 with large tiles, 1199 with small ones.
  p.path = p.f32 ? PATH_F32 : T <= kTwoRows ? PATH_THIN : big >= 192 && T > 128 ? PATH_BIG : PATH_SMALL;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  p.x = take(p.copy_x ? p.planes * T * p.ldx * 2 : 0);
  p.w = take(p.copy_w ? p.piece * (order == ORDER_DV ? D : p.ldx) * 2 : 0);
  if (!backward) {
    p.part = take(round_up(V, tile_cols(p.path)) / block_cols(p.path) * T * 8);
  } else {
    const int64_t rows = p.planes * T;
    p.dz = take(rows * (p.piece + kTurn) * size);
    p.dx = split(p.f32, rows, D, std::min(p.piece, V));
    p.ld_dx = round_up(D, 8);
    p.join_dx = p.dx.pieces * p.planes;
    p.acc_dx = take(p.join_dx > 1 || p.piece < V ? p.join_dx * T * p.ld_dx * 4 : 0);
    const int64_t n = std::min(p.piece, V);
    p.rows_dw = order == ORDER_DV ? D : n;
    p.ld_dw = round_up(order == ORDER_DV ? n : D, 8);
    p.dw = split(p.f32, p.rows_dw, order == ORDER_DV ? n : D, rows);
    p.acc_dw = take(p.dw.pieces > 1 ? p.dw.pieces * p.rows_dw * p.ld_dw * 4 : 0);
  }
  p.total = std::max<int64_t>(at, 256);
  return p;
}

static int check_sizes(int dtype, int64_t T, int64_t D, int64_t V, int order) {
  if (dtype != MTX_F32 && dtype != MTX_BF16) return MTX_ERR_ARG;
  if (order != ORDER_DV && order != ORDER_VD) return MTX_ERR_ARG;
  if (T < 0 || D <= 0 || V <= 0) return MTX_ERR_ARG;
  const int64_t most = 65535 * 64;  // rows of tiles in a grid; 32-bit offsets inside a tile
  if (T > most || D > most || V > most) return MTX_ERR_UNSUPPORTED;
  return MTX_OK;
}
static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }

static int pad(const void* in, int64_t ldi, int64_t rows, int64_t cols, char* out, int64_t ld, int times, hipStream_t st) {
  hipLaunchKernelGGL(pad_kernel, dim3((unsigned)ceil_div(times * rows * ld, 2048)), dim3(256), 0, st, (const uint16_t*)in, ldi,
                     rows, cols, (uint16_t*)out, ld, times);
  return check_launch();
}
// The operands of the logits of columns v0 ..: x and w where they are, or copies with rows of whole 16-byte chunks
static int operands(const Plan& p, const void* x, const void* w, int64_t v0, char* ws, Logits& a, hipStream_t st) {
  const int64_t size = p.f32 ? 4 : 2, n = std::min(p.piece, p.V - v0);
  int rc = MTX_OK;
  a.x = p.copy_x ? ws + p.x : x;
  if (p.copy_x && v0 == 0) rc = pad(x, p.D, p.T, p.D, ws + p.x, p.ldx, p.planes, st);
  a.ldx = p.ldx;
  a.w = (const char*)w + (p.order == ORDER_DV ? v0 : v0 * p.D) * size;
  a.ldw = p.order == ORDER_DV ? p.V : p.D;
  a.w_left = (int)n;
  if (p.copy_w && rc == MTX_OK) {
    const bool dv = p.order == ORDER_DV;
    rc = pad(a.w, a.ldw, dv ? p.D : n, dv ? n : p.D, ws + p.w, dv ? p.piece : p.ldx, 1, st);
    a.w = ws + p.w;
    a.ldw = dv ? p.piece : p.ldx;
    if (dv) a.w_left = (int)p.piece;
  }
  a.T = (int)p.T;
  a.red = (int)p.red;
  a.missing = p.order == ORDER_DV ? (int)(p.red - p.D) : 0;
  a.v0 = (int)v0;
  a.cols = (int)n;
  return rc;
}
static int logits(const Plan& p, const Logits& a, bool dz, hipStream_t st) {
  return p.f32 ? launch_logits_f32(a, dz, p.order, st) : launch_logits(a, dz, p.order, p.path, st);
}
static int product(const Plan& p, const Product& a, bool a_cols, bool b_cols, const Split& s, hipStream_t st) {
  return p.f32 ? launch_product_f32(a, a_cols, b_cols, st) : launch_product(a, a_cols, b_cols, s.size, st);
}
static int join(bool f32, const float* acc, int pieces, int64_t rows, int64_t cols, int64_t ldacc, void* out, int64_t ldo,
                const Factors& f, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(rows * ceil_div(cols, 8), 64));
  if (f32) hipLaunchKernelGGL(join_kernel<float>, grid, dim3(64), 0, st, acc, pieces, rows, cols, ldacc, (float*)out, ldo, f);
  else hipLaunchKernelGGL(join_kernel<uint16_t>, grid, dim3(64), 0, st, acc, pieces, rows, cols, ldacc, (uint16_t*)out, ldo, f);
  return check_launch();
}

// Both losses: the logits' blocks of every piece, their join, and the sum over the rows if `total` is asked for.
static int forward(const Plan& p, const void* x, const void* w, Merge m, float* chosen, float* total, float* count, int mean,
                   char* ws, hipStream_t st) {
  Logits a{};
  a.e = m.e;
  a.scale = m.scale;
  a.part = (float2*)(ws + p.part);
  a.chosen = chosen;
  for (int64_t v0 = 0; v0 < p.V; v0 += p.piece) {
    int rc = operands(p, x, w, v0, ws, a, st);
    if (rc == MTX_OK) rc = logits(p, a, false, st);
    if (rc != MTX_OK) return rc;
  }
  m.part = a.part;
  m.blocks = ceil_div(p.V, tile_cols(p.path)) * (tile_cols(p.path) / block_cols(p.path));
  m.T = p.T;
  m.V = p.V;
  m.chosen = chosen;
  // forward of 4096 x 64 x 32000: 81 us with neighbouring rows together, 87 with a wave a row; 1024 x 64 x 32000 31.6, 29.9
  if (p.T > 2048) hipLaunchKernelGGL(merge_kernel, dim3((unsigned)ceil_div(p.T, 32)), dim3(256), 0, st, m);
  else hipLaunchKernelGGL(merge_wave_kernel, dim3((unsigned)ceil_div(p.T, 4)), dim3(256), 0, st, m);
  if (total) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, m.loss, m.state, p.T, mean, total, count);
  return check_launch();
}

static int backward(const Plan& p, const Factors& f, const void* x, const void* w, const float* chosen, const Entries& e,
                    float scale, void* dx, void* dw, char* ws, hipStream_t st) {
  const int64_t size = p.f32 ? 4 : 2;
  const bool dv = p.order == ORDER_DV;
  int rc = MTX_OK;
  Logits a{};
  a.f = f;
  a.e = e;
  a.scale = scale;
  a.dz = ws + p.dz;
  a.ldz = p.piece + kTurn;
  a.planes = p.planes;
  const int rows = (int)(p.planes * p.T);
  for (int64_t v0 = 0; v0 < p.V && rc == MTX_OK; v0 += p.piece) {
    rc = operands(p, x, w, v0, ws, a, st);
    if (rc == MTX_OK) rc = logits(p, a, true, st);
    if (rc != MTX_OK) return rc;
    const Named named{e, f, chosen, scale, p.T, a.v0, a.cols, a.dz, a.ldz, p.f32, p.planes};
    hipLaunchKernelGGL(named_kernel, dim3((unsigned)ceil_div(p.T * e.K, 256)), dim3(256), 0, st, named);
    if (dx) {
      const int red = p.f32 ? a.cols : (int)round_up(a.cols, 8);  // dz holds zeros behind its columns
      const bool only = p.piece >= p.V, final = v0 + p.piece >= p.V;
      // the last piece of the vocabulary may be shorter than what the split was made for
      const int pieces = (int)std::min<int64_t>(p.dx.pieces, ceil_div(red, 32));
      Product q{a.dz, a.w, a.ldz, a.ldw, rows, (int)p.D, red, 0, rows, (int)(dv ? p.D : p.ldx), dx, p.D, pieces, nullptr,
                p.ld_dx, v0 > 0, p.join_dx == 1 && final, f};
      if (!dv) q.missing = red - a.cols;
      if (!(only && p.join_dx == 1)) q.acc = (float*)(ws + p.acc_dx);
      rc = product(p, q, false, !dv, p.dx, st);
      if (rc == MTX_OK && final && p.join_dx > 1) rc = join(p.f32, q.acc, p.join_dx, p.T, p.D, p.ld_dx, dx, p.D, f, st);
      if (rc != MTX_OK) return rc;
    }
    if (dw && rc == MTX_OK) {
      void* out = (char*)dw + (dv ? v0 : v0 * p.D) * size;
      const int64_t ldo = dv ? p.V : p.D;
      Product q{};
      if (dv) q = Product{a.x, a.dz, a.ldx, a.ldz, (int)p.D, a.cols, rows, 0, (int)p.ldx, (int)p.piece, out, ldo, p.dw.pieces};
      else q = Product{a.dz, a.x, a.ldz, a.ldx, a.cols, (int)p.D, rows, 0, (int)p.piece, (int)p.ldx, out, ldo, p.dw.pieces};
      q.ldacc = p.ld_dw;
      q.last = p.dw.pieces == 1;
      q.f = f;
      if (p.dw.pieces > 1) q.acc = (float*)(ws + p.acc_dw);
      rc = product(p, q, true, true, p.dw, st);
      if (rc == MTX_OK && p.dw.pieces > 1) rc = join(p.f32, q.acc, p.dw.pieces, q.rows, q.cols, p.ld_dw, out, ldo, f, st);
    }
  }
  return rc;
}

// the teacher's entries as saved from the forward to the backward pass: classes, shares, bounds, rows
struct Saved {
  int64_t share, bounds, row, ldb, total;
};
static Saved saved(int64_t T, int64_t V, int64_t K) {
  Saved s;
  s.ldb = ceil_div(V, kBlock) + 2;  // the blocks' starts and the last one's end, twice: a tile may begin behind the vocabulary
  s.share = round_up(T * K * 4, 256);
  s.bounds = s.share + round_up(T * K * 4, 256);
  s.row = s.bounds + round_up(T * s.ldb * 2, 256);
  s.total = s.row + round_up(T * 8, 256);
  return s;
}
static Entries entries(char* buf, const Saved& s, int64_t K) {
  return Entries{nullptr, 0, (const int32_t*)buf, (const float*)(buf + s.share), (const uint16_t*)(buf + s.bounds), s.ldb, (int)K};
}

}  // namespace head
}  // namespace mtx

using namespace mtx;

extern "C" int64_t mtx_head_loss_workspace_size(int dtype, int64_t T, int64_t D, int64_t V, int order, int backward) {
  if (head::check_sizes(dtype, T, D, V, order) != MTX_OK) return -1;
  return T == 0 ? 256 : head::plan(dtype, T, D, V, order, backward != 0).total;
}
extern "C" int64_t mtx_distillation_entries_size(int64_t T, int64_t V, int64_t K) {
  if (T < 0 || V <= 0 || K <= 0 || K > head::kMaxEntries) return -1;
  return std::max<int64_t>(head::saved(T, V, K).total, 256);
}

extern "C" int mtx_linear_cross_entropy(const void* x, const void* w, const void* targets, int targets_64, int dtype, int64_t T,
                                        int64_t D, int64_t V, int order, int64_t ignore_index, float z_loss, int mean,
                                        float* loss, float* stats, float* state, float* total, float* count, float* chosen,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace head;
  const int rc = check_sizes(dtype, T, D, V, order);
  if (rc != MTX_OK) return rc;
  if (!(z_loss >= 0.0f && z_loss < INFINITY) || (!total != !count)) return MTX_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (T == 0) {
    if (total) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, loss, state, (int64_t)0, mean, total, count);
    return check_launch();
  }
  if (!x || !w || !targets || !loss || !stats || !state || !chosen || !aligned16(x) || !aligned16(w)) return MTX_ERR_ARG;
  const Plan p = plan(dtype, T, D, V, order, false);
  if (!workspace || !aligned16(workspace) || workspace_bytes < p.total) return MTX_ERR_WORKSPACE;
  Merge m{};
  m.e = Entries{targets, targets_64, nullptr, nullptr, nullptr, 0, 1};
  m.ignore = ignore_index;
  m.scale = kLog2e, m.inv_tau = 1.0f, m.unit = 1.0f, m.z_loss = z_loss;
  m.loss = loss, m.stats = stats, m.state = state;
  return forward(p, x, w, m, chosen, total, count, mean, (char*)workspace, st);
}

extern "C" int mtx_linear_cross_entropy_bwd(const float* g, const float* count, const void* x, const void* w, const void* targets,
                                            int targets_64, const float* stats, const float* state, const float* chosen, int dtype,
                                            int64_t T, int64_t D, int64_t V, int order, float z_loss, void* dx, void* dw, void* workspace,
                                            int64_t workspace_bytes, void* stream) {
  using namespace head;
  const int rc = check_sizes(dtype, T, D, V, order);
  if (rc != MTX_OK) return rc;
  if (T == 0 || (!dx && !dw)) return MTX_OK;
  if (!g || !x || !w || !targets || !stats || !state || !chosen || !aligned16(x) || !aligned16(w) || !aligned16(dx) ||
      !aligned16(dw))
    return MTX_ERR_ARG;
  const Plan p = plan(dtype, T, D, V, order, true);
  if (!workspace || !aligned16(workspace) || workspace_bytes < p.total) return MTX_ERR_WORKSPACE;
  const Entries e{targets, targets_64, nullptr, nullptr, nullptr, 0, 1};
  return backward(p, Factors{g, count, stats, state, 1.0f, z_loss}, x, w, chosen, e, kLog2e, dx, dw, (char*)workspace,
                  (hipStream_t)stream);
}

extern "C" int mtx_linear_distillation(const void* x, const void* w, const void* teacher_idx, int idx_64,
                                       const void* teacher_logits, int logits_dtype, int dtype, int64_t T, int64_t D, int64_t V,
                                       int64_t K, int order, float temperature, int mean, float* loss, float* stats, float* state,
                                       float* total, float* count, float* chosen, void* entries_buffer, int64_t entries_bytes,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace head;
  const int rc = check_sizes(dtype, T, D, V, order);
  if (rc != MTX_OK) return rc;
  if (K <= 0 || (logits_dtype != MTX_F32 && logits_dtype != MTX_BF16)) return MTX_ERR_ARG;
  if (K > kMaxEntries) return MTX_ERR_UNSUPPORTED;
  const float inv = 1.0f / temperature;
  if (!(temperature > 0.0f && temperature < INFINITY && inv < INFINITY) || (!total != !count)) return MTX_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (T == 0) {
    if (total) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, loss, state, (int64_t)0, mean, total, count);
    return check_launch();
  }
  if (!x || !w || !teacher_idx || !teacher_logits || !loss || !stats || !state || !chosen || !entries_buffer || !aligned16(x) ||
      !aligned16(w))
    return MTX_ERR_ARG;
  const Plan p = plan(dtype, T, D, V, order, false);
  const Saved s = saved(T, V, K);
  if (!aligned16(entries_buffer) || entries_bytes < s.total) return MTX_ERR_WORKSPACE;
  if (!workspace || !aligned16(workspace) || workspace_bytes < p.total) return MTX_ERR_WORKSPACE;
  char* buf = (char*)entries_buffer;
  const Prep prep{teacher_idx, teacher_logits, idx_64, logits_dtype == MTX_F32, T, V, (int)K, inv, (int32_t*)buf,
                  (float*)(buf + s.share), (uint16_t*)(buf + s.bounds), s.ldb, (float2*)(buf + s.row)};
  hipLaunchKernelGGL(entries_kernel, dim3((unsigned)T), dim3(64), 0, st, prep);
  Merge m{};
  m.e = entries(buf, s, K);
  m.row = prep.row;
  m.scale = kLog2e * inv, m.inv_tau = inv, m.unit = temperature * temperature;
  m.loss = loss, m.stats = stats, m.state = state;
  return forward(p, x, w, m, chosen, total, count, mean, (char*)workspace, st);
}

extern "C" int mtx_linear_distillation_bwd(const float* g, const float* count, const void* x, const void* w,
                                           const void* entries_buffer, int64_t entries_bytes, const float* stats,
                                           const float* state, const float* chosen, int dtype, int64_t T, int64_t D, int64_t V,
                                           int64_t K, int order, float temperature, void* dx, void* dw, void* workspace,
                                           int64_t workspace_bytes, void* stream) {
  using namespace head;
  const int rc = check_sizes(dtype, T, D, V, order);
  if (rc != MTX_OK) return rc;
  if (K <= 0 || !(temperature > 0.0f && temperature < INFINITY)) return MTX_ERR_ARG;
  if (K > kMaxEntries) return MTX_ERR_UNSUPPORTED;
  if (T == 0 || (!dx && !dw)) return MTX_OK;
  if (!g || !x || !w || !entries_buffer || !stats || !state || !chosen || !aligned16(x) || !aligned16(w) || !aligned16(dx) ||
      !aligned16(dw))
    return MTX_ERR_ARG;
  const Plan p = plan(dtype, T, D, V, order, true);
  const Saved s = saved(T, V, K);
  if (!aligned16(entries_buffer) || entries_bytes < s.total) return MTX_ERR_WORKSPACE;
  if (!workspace || !aligned16(workspace) || workspace_bytes < p.total) return MTX_ERR_WORKSPACE;
  return backward(p, Factors{g, count, stats, state, temperature, 0.0f}, x, w, chosen,
                  entries((char*)const_cast<void*>(entries_buffer), s, K), kLog2e / temperature, dx, dw, (char*)workspace,
                  (hipStream_t)stream);
}

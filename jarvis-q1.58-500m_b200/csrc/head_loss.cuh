// What the kernels of the head's losses share (head_loss.cu: logits and statistics, head_grad.cu: the gradient's products).
#pragma once
#include "pair_mma.cuh"

namespace jb {

constexpr int HEAD_TILE = 256, HEAD_BK = 64, HEAD_STAGES = 6;      // rows and columns of a pair's tile, K of a stage, stages
constexpr int HEAD_OPERAND = HEAD_TILE / 2 * HEAD_BK * 2;          // 16 KiB: one CTA's half of an operand's stage
constexpr int HEAD_EPI_WARP0 = 2, HEAD_THREADS = 32 * (HEAD_EPI_WARP0 + 8);
typedef PairRing<HEAD_STAGES> HeadRing;
constexpr size_t HEAD_CTL = (sizeof(HeadRing) + 127) / 128 * 128;
constexpr size_t HEAD_SMEM = 1024 + size_t(HEAD_STAGES) * 2 * HEAD_OPERAND + HEAD_CTL;
static_assert(HEAD_SMEM <= 227 * 1024, "shared memory of one CTA");

// Gradients of the losses and what the forward call left, as the backward kernels read them.
struct HeadGrads {
  const int64_t* targets;                 // null: no cross entropy
  const float* neg_entropy;               // null: no teacher
  const float *lse, *lse_t;               // [2][N]: reference point and sum
  const float *g_ce, *g_kd;               // gradients of the rows' losses (stride 0: the same for all)
  int g_ce_stride, g_kd_stride;
  const float *n_ce, *n_kd;               // divisors (the means' row counts) or null
  float* scale;                           // [1], with gradients row by row: their common factor, made by a launch of its own
  int N, V;
  float tau;
};

#if defined(__CUDACC__)
// The gradients of the logits are kept relative to a factor, which the products apply to their f32 sums.  (With 1 / rows in them a
// target's entry, -1 / rows and half of a row's gradient, had the same rounding in every row.)  It is the largest of the whole call,
// and where rows differ (gradients row by row, or rows with one of two losses) that times the power of two by which the row's own is
// smaller: a light row keeps its bits, dx has its factor back as a row of the product, and for dw, which sums over rows, the copy of its
// hidden row is smaller by that power of two.
__device__ __forceinline__ float common_factor(float ce, float kd) {
  const float s = ce <= 3.4e38f && !(kd <= 3.4e38f && kd > ce) ? ce : kd;
  return s > 0.f && s <= 3.4e38f ? s : 1.f;
}
__device__ __forceinline__ float row_factor(const float* g, int stride, const float* n, int row) {
  const float c = g[size_t(row) * stride];
  return n ? c / *n : c;
}
__device__ __forceinline__ float head_scale(const HeadGrads& p) {
  if (p.scale) return *p.scale;
  return common_factor(p.targets ? fabsf(row_factor(p.g_ce, 0, p.n_ce, 0)) : 0.f, p.neg_entropy ? fabsf(row_factor(p.g_kd, 0, p.n_kd, 0)) * p.tau : 0.f);
}
// Largest finite factors of a row, 0 for a loss that it has no part in.
__device__ __forceinline__ float2 row_factors(const HeadGrads& p, int row) {
  float2 f = make_float2(0.f, 0.f);
  if (p.targets && p.targets[row] != -100) {
    const float c = fabsf(row_factor(p.g_ce, p.g_ce_stride, p.n_ce, row));
    if (c <= 3.4e38f) f.x = c;
  }
  if (p.neg_entropy && p.neg_entropy[row] != INFINITY) {
    const float c = fabsf(row_factor(p.g_kd, p.g_kd_stride, p.n_kd, row)) * p.tau;
    if (c <= 3.4e38f) f.y = c;
  }
  return f;
}
// How many times the call's factor is halved for a row: until its own is more than half of what is left.
__device__ __forceinline__ int row_halvings(const HeadGrads& p, int row, float scale) {
  if (!p.scale && !(p.targets && p.neg_entropy)) return 0;      // one loss's mean: all rows have the same
  const float2 v = row_factors(p, row);
  const float f = fmaxf(v.x, v.y);
  if (!(f > 0.f && f <= scale)) return 0;
  const int k = ilogbf(scale) - ilogbf(f);
  return f > ldexpf(scale, -k) ? k - 1 : k;
}
__device__ __forceinline__ float row_scale(const HeadGrads& p, int row, float scale) {
  const int k = row_halvings(p, row, scale);
  return k ? ldexpf(scale, -k) : scale;
}
#endif

// Operands of the gradient's products are f16, whose rounding is an eighth of bf16's: the logits' gradients times 2^13 (at most 2 of them
// add up to 2^14; they keep all their bits down to 2^-27 and vanish below 2^-38), and copies of weight and rows times the powers of two by
// which the largest finite value of each comes to lie in [2^15, 2^16).  A bf16 value within 2^32 of that is exact there, a smaller one off
// by at most 2^-40 of the largest; the rows' values count as halved with their factors there.  (As bf16 the logits' gradients gave dx
// and dW an error of sqrt(2) times their own rounding.)
constexpr int HEAD_G_EXP = 13, HEAD_RANGE_CTAS = 512;

// How a backward pass is cut: `pieces` pieces of `cols` vocabulary columns (the last one shorter) whose gradients of the logits are
// kept at a time, and `slabs` parts of a piece over which the hidden rows' gradient is summed side by side.
struct HeadPlan {
  int cols, pieces, slabs;
};
HeadPlan head_plan(int N, int V, int C, int pairs);

// The items of a products launch on its pairs: the long ones first, one a pair in turn, then the short ones, of which the pairs that
// got fewer long ones take `more` more each.
struct HeadShares {
  int uneven;                // pairs [0, uneven) have one long item more than the others
  int rounds, more;          // short items of those pairs; the others have rounds + more
  long long span;            // K-blocks of the busiest pair
};
HeadShares head_shares(int n_long, int k_long, int n_short, int k_short, int pairs);

// The i-th item of a pair: a long one below n_long, n_long + a short one from there on, -1 behind the pair's last.
__host__ __device__ __forceinline__ int head_walk(const HeadShares& s, int n_long, int n_short, int pair, int pairs, int i) {
  const bool uneven = pair < s.uneven;
  const int turns = n_long / pairs + (uneven ? 1 : 0), r = i - turns;
  if (r < 0) return pair + i * pairs;
  int t = pair + r * pairs;
  if (r >= s.rounds) {
    if (uneven || r >= s.rounds + s.more) return -1;
    t = s.rounds * pairs + (r - s.rounds) * (pairs - s.uneven) + pair - s.uneven;
  }
  return t < n_short ? n_long + t : -1;
}

// Boxes of 64 columns of a bf16 or f16 matrix whose rows are `pitch` elements apart.
int encode_head_map(CUtensorMap* tm, const void* ptr, long long cols, long long pitch, long long rows, int box_rows, const char* what);
// Pitch of the copies: whole 128-byte lines, where a box's rows are one line each.
__host__ __device__ inline int head_pitch(int C) { return (C + HEAD_BK - 1) / HEAD_BK * HEAD_BK; }

// dx += scale G W and dw = scale G^T xs of one piece (head_grad.cu); a null one is not wanted.
struct HeadProducts {
  int N, V, C;
  int v0, n_cols;            // the piece's vocabulary rows
  int ldg;                   // columns of G
  int slabs;
  int first, last;           // of the pieces
  HeadGrads grads;
  const int* exps;           // [2]: exponents of the factors of the weight's copy and of the rows'
  float* dx_slabs;           // [slabs][N][C] f32: sums so far; may be dx itself
  void* dx;                  // [N][C], written by the last piece
  int dx_bf16;
  void* dw;                  // [V][C]
  int dw_bf16;
  // made by the launch
  int all_slabs;             // of dx_slabs; a short last piece adds to `slabs` of them
  int width;                 // columns of a tile
  int dx_items, dw_items;
  int dw_first;              // dW's items are the long ones
  HeadShares shares;
  unsigned int* status;
};
int head_width(int C);
// g: f16 [N][ldg]; xs, ws: the f16 copies of rows and of the piece's weight, head_pitch(C) apart.
int launch_head_products(HeadProducts p, const void* g, const void* xs, const void* ws, int sms, cudaStream_t stream);

}  // namespace jb

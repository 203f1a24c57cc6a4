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

// How a backward pass is cut: `pieces` pieces of `cols` vocabulary columns (the last one shorter) whose gradients of the logits are
// kept as bf16, and `slabs` parts of a piece over which the hidden rows' gradient is summed side by side.
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

int encode_head_map(CUtensorMap* tm, const void* ptr, long long cols, long long rows, int box_rows, const char* what);

// dx slabs += G W and dW = G^T xs of one piece (head_grad.cu); a null one is not wanted.  g: bf16 [N][cols]; piece columns [0, n_cols) are vocabulary rows
// [v0, v0 + n_cols) of w and dw.
int launch_head_products(const void* g, int cols, int n_cols, const void* xs, const void* w, int N, int V, int C, int v0, int slabs,
                         bool first, const float* scale, float* dx_slabs, void* dw, int dw_dtype, int sms, cudaStream_t stream);

}  // namespace jb

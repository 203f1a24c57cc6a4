// Losses of the language-model head straight from hidden rows and head weight: cross entropy, and distillation from a teacher's top
// logits, with their gradients.  The reference computes logits = lm_head(x) and F.cross_entropy on them
// (jarvis_engine/jarvis_model.py:535-540); here the N x V logits exist only in tensor memory.
//
//   z[n][v] = x[n] . w[v]                                        bf16 operands, f32 accumulation
//   ce[n]   = log sum_v exp(z) - z[target]
//   kd[n]   = tau^2 (sum_k q log q + log sum_v exp(z / tau) - sum_k q[k] z[id_k] / tau),   q = softmax_k(teacher / tau)
//   dz      = g_ce (softmax(z) - 1[target]) + g_kd tau (softmax(z / tau) - sum_k q[k] 1[id_k])
//
// Forward: a product kernel whose epilogue keeps, per row of a 256 x 256 tile, the maximum, the sum of exponentials and the logits that
// the target and the teacher ask for; a second kernel joins the tiles.  Backward: the same product again, whose epilogue writes dz
// of a piece of the vocabulary as f16 (an operand of the products dx += dz W and dW = dz^T x that follow, head_grad.cu), so
// that the workspace stays bounded whatever the vocabulary: 8 N V C operations for a training step, where 6 N V C would need the
// logits kept.
//
// Exponentials are base 2 with a whole number as the reference point: 2^(z k - r), k the f32 value next to log2(e), has one rounding in its
// argument and rescaling by 2^(r - r') has none.  A row's sum travels as the pair (r, sum 2^(z k - r)), and logarithms are divided by
// that very k, so that logits of any size keep their differences.
#include <cuda_fp16.h>
#include <float.h>
#include <limits.h>

#include "head_loss.cuh"
#include "launchers.h"

namespace jb {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int TEACHER_MAX = 256;
// Gradients of the logits kept at a time, at most.  Each piece adds to dx once more: 16384 x 50257 x 1024 in pieces of 64 MiB 5.8 ms, 320 MiB 5.4,
// 640 MiB 5.25, 1280 MiB 5.27.
constexpr size_t PIECE_BYTES = size_t(640) << 20;

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------------------
// The teacher's rows: entries (id, q) by ascending id, [N][K], and where each 256 columns' entries begin, [N][tiles], so that a tile's
// epilogue finds its own with one load.
// ---------------------------------------------------------------------------
constexpr int TEACHER_WARPS = 8;

struct TeacherLayout {
  size_t entries, starts, total;         // neg_entropy, f32 [N], comes first
};
TeacherLayout teacher_layout(int N, int K, int V) {
  TeacherLayout l;
  l.entries = up256(size_t(N) * 4);
  l.starts = l.entries + up256(size_t(N) * K * 8);
  l.total = l.starts + up256(size_t(N) * ((size_t(V) + HEAD_TILE - 1) / HEAD_TILE) * 2);
  return l;
}

__device__ __forceinline__ float teacher_value(const float* p) { return *p; }
__device__ __forceinline__ float teacher_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// A warp a row; an entry's place is the number of entries before it.  neg_entropy: sum q log q; +inf for a row without entries,
// NaN for one with an id beyond the vocabulary.
template <typename T>
__global__ void __launch_bounds__(32 * TEACHER_WARPS)
teacher_rows_kernel(const int64_t* __restrict__ ids, const T* __restrict__ logits, int N, int K, int V, float inv_tau,
                    float* __restrict__ neg_entropy, int2* __restrict__ entries, uint16_t* __restrict__ starts) {
  pdl_wait();
  pdl_trigger();
  constexpr int PER = TEACHER_MAX / 32;
  __shared__ __align__(16) int s_id[TEACHER_WARPS][TEACHER_MAX];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.x * TEACHER_WARPS + warp;
  if (row >= N) return;
  int* mine = s_id[warp];
  const int per = (K + 31) >> 5;         // entries of a lane
  float v[PER];
  int id[PER];
  bool bad = false;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = -INFINITY;
    id[i] = INT_MAX;
    const int k = i * 32 + lane;
    if (k < K) {
      const long long y = ids[size_t(row) * K + k];
      if (y >= 0) {
        v[i] = teacher_value(logits + size_t(row) * K + k);
        if (y >= V) bad = true; else id[i] = int(y);
      }
      top = fmaxf(top, v[i]);
    }
    if (i < per) mine[k] = id[i];        // the places beyond K: behind everything
  }
  bad = __any_sync(0xffffffffu, bad);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // a row whose kept values are all -inf has no probabilities either (a NaN among them: NaN).  The temperature divides the differences: the
  // values themselves may be the type's lowest, which a temperature below 1 would make -inf, or its largest.
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = (v[i] - base) * inv_tau;
    if (id[i] != INT_MAX) sum += expf(v[i]);
  }
  sum = warp_sum(sum);
  const float inv = 1.0f / sum, log_sum = logf(sum);
  const bool none = sum == 0.f && !bad;
  float ent = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float q = expf(v[i]) * inv;
    if (none) id[i] = INT_MAX;
    if (id[i] != INT_MAX && v[i] != -INFINITY) ent += q * (v[i] - log_sum);
    v[i] = q;
  }
  ent = warp_sum(ent);
  if (lane == 0) neg_entropy[row] = bad ? __int_as_float(0x7fc00000) : none ? INFINITY : ent;
  __syncwarp();
  int at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) at[i] = 0;
  for (int j = 0; j < 32 * per; j += 4) {
    const int4 o = *reinterpret_cast<const int4*>(mine + j);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (i >= per) break;
      const int k = i * 32 + lane;       // of equal ids the earlier one comes first
      at[i] += (o.x < id[i] || (o.x == id[i] && j < k)) + (o.y < id[i] || (o.y == id[i] && j + 1 < k)) +
               (o.z < id[i] || (o.z == id[i] && j + 2 < k)) + (o.w < id[i] || (o.w == id[i] && j + 3 < k));
    }
  }
  __syncwarp();
  int2* out = entries + size_t(row) * K;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (i >= per) break;
    if (none) at[i] = i * 32 + lane;     // (its ids in shared memory are not INT_MAX)
    if (at[i] < K) {
      out[at[i]] = make_int2(id[i], __float_as_int(id[i] == INT_MAX ? 0.f : v[i]));
      mine[at[i]] = id[i];
    }
  }
  __syncwarp();
  const int tiles = (V + HEAD_TILE - 1) / HEAD_TILE;
  for (int t = lane; t < tiles; t += 32) {
    int lo = 0, hi = K;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (mine[mid] < t * HEAD_TILE) lo = mid + 1; else hi = mid;
    }
    starts[size_t(row) * tiles + t] = uint16_t(lo);
  }
}

// ---------------------------------------------------------------------------
// Logits of 256 rows x 256 vocabulary columns per CTA pair.
// ---------------------------------------------------------------------------
struct HeadLogits {
  int N, V, C;
  int v0, cols;              // vocabulary columns [v0, v0 + cols) of this launch
  const int64_t* targets;    // CE
  const int2* entries;       // KD: what teacher_rows_kernel leaves
  const uint16_t* starts;
  int K, v_tiles;            // tiles of the whole vocabulary
  float inv_tau;
  float* part;               // statistics: [parts][values][N]
  int carry;                 // a pair's tiles are all of the same rows: it leaves one part a group of epilogue warps, else every tile does
  float* z_target;           // [N]
  unsigned int* ticket;      // set to 0 for the join
  HeadGrads grads;           // gradient
  __half* g;                 // gradient: [N][ldg]
  int ldg;
  const uint4 *x, *w;        // gradient: rows and weight
  uint4 *xs, *ws;            // their copies, the weight's of these columns; null: not wanted
  const unsigned* tops;      // [2][HEAD_RANGE_CTAS], n_tops of each: largest magnitudes of the weight and of the rows, part by part
  int n_tops;
  int* exps;                 // exponents of the copies' factors, weight and rows: made by the first piece, read by the others
  int box_rows;              // rows of x that a CTA asks for at a time
  unsigned int* status;
};

// Tiles of the same columns run side by side, so that a weight tile comes from HBM once; beyond 64 row tiles (32 MB of rows at 1024
// channels) in groups, so that the group's rows stay in L2.
constexpr int HEAD_GROUP = 64;
__device__ __forceinline__ void head_tile(int t, int tm, int tv, int* m, int* v) {
  const int g = t / (HEAD_GROUP * tv), base = g * HEAD_GROUP, size = min(HEAD_GROUP, tm - base);
  const int r = t - base * tv;
  *v = r / size;
  *m = base + r - *v * size;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float pick32(const uint32_t (&v)[32], int j) {
  uint32_t a[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = j & 16 ? v[i + 16] : v[i];
#pragma unroll
  for (int w = 8; w > 0; w >>= 1)
#pragma unroll
    for (int i = 0; i < w; ++i) a[i] = j & w ? a[i + w] : a[i];
  return __uint_as_float(a[0]);
}

// Sum of 2^(z k) relative to 2^ref, ref a whole number.
struct RunningSum {
  float ref = -INFINITY, sum = 0.f;
  __device__ __forceinline__ void add(const uint32_t (&v)[32], float top, float k) {
    const float to = fmaxf(ref, rintf(top * k));
    const float r = to == -INFINITY ? 0.f : to;                // nothing but -inf so far: all terms are 0 (or NaN)
    float s0 = ref == -INFINITY ? sum : sum * ex2(ref - r), s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      s0 += ex2(fmaf(__uint_as_float(v[j]), k, -r));
      s1 += ex2(fmaf(__uint_as_float(v[j + 1]), k, -r));
      s2 += ex2(fmaf(__uint_as_float(v[j + 2]), k, -r));
      s3 += ex2(fmaf(__uint_as_float(v[j + 3]), k, -r));
    }
    sum = (s0 + s1) + (s2 + s3);
    ref = to;
  }
};

// A row's teacher entries from one on; the next is on its way while the current is used.
struct Entries {
  const int2* row;
  int at, K, id = INT_MAX;
  float q = 0.f;
  int2 next = {INT_MAX, 0};
  __device__ __forceinline__ void fetch() {
    next = at < K ? __ldg(row + at) : make_int2(INT_MAX, 0);
    ++at;
  }
  __device__ __forceinline__ void step() {
    id = next.x;
    q = __int_as_float(next.y);
    fetch();
  }
  __device__ __forceinline__ void begin(const int2* entries, int n_entries, int start) {
    row = entries; K = n_entries; at = start;
    fetch();
    step();
  }
};

constexpr int head_values(bool ce, bool kd) { return (ce ? 2 : 0) + (kd ? 3 : 0); }

// A row's part in the gradient: the sums' reference points, the row's factors times 2^13, the factors over the sums.  A row without target
// and teacher takes part in nothing, whatever it holds; one with either has both reference points, with which no exponential is large.
template <bool CE, bool KD>
struct RowGrad {
  float l1 = 0.f, g1 = 0.f, p1 = 0.f, l2 = 0.f, g2 = 0.f, p2 = 0.f;
  bool live = false;
  __device__ __forceinline__ void load(const HeadGrads& p, int row, float scale) {
    const float nan = __int_as_float(0x7fc00000);
    constexpr float unit = float(1 << HEAD_G_EXP);
    if (CE) {
      l1 = p.lse[row];
      const long long y = p.targets[row];
      if (y != -100) {
        live = true;
        g1 = y < 0 || y >= p.V ? nan : row_factor(p.g_ce, p.g_ce_stride, p.n_ce, row) / scale * unit;
        p1 = g1 / p.lse[size_t(p.N) + row];
      }
    }
    if (KD) {
      l2 = p.lse_t[row];
      const float e = p.neg_entropy[row];
      if (e != INFINITY) {
        live = true;
        g2 = e != e ? nan : row_factor(p.g_kd, p.g_kd_stride, p.n_kd, row) * p.tau / scale * unit;
        p2 = g2 / p.lse_t[size_t(p.N) + row];
      }
    }
  }
};
template <bool CE = true, bool KD = true>
__device__ __forceinline__ bool row_is_live(const HeadGrads& p, int row) {
  return (CE && p.targets && p.targets[row] != -100) || (KD && p.neg_entropy && p.neg_entropy[row] != INFINITY);
}

// ---- f16 copies of the products' other operands, by eight warps of every CTA beside the products ----
constexpr int COPY_WARPS = 8;

// Exponent of the factor that brings the largest magnitude (as bf16 bits) to [2^15, 2^16), where f16 ends at 65504 and bf16 has no value
// beyond 65280; nothing but zeros (or subnormal numbers): as far up as there is.
__device__ __forceinline__ int copy_exponent(unsigned top) { return min(126, 127 + 15 - int(top >> 7)); }
// Largest of what head_range_kernel's CTAs found, by a warp.
__device__ __forceinline__ unsigned range_top(const unsigned* tops, int n, int lane) {
  unsigned top = 0;
  for (int i = lane; i < n; i += 32) top = max(top, tops[i]);
  return __reduce_max_sync(0xffffffffu, top);
}

__device__ __forceinline__ uint32_t f16x2_of_bf16x2(uint32_t w, float factor) {
  const __half2 h = __floats2half2_rn(bf16_lo(w) * factor, bf16_hi(w) * factor);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// With few rows of x the weight's copy is what the launch waits for (37 rows of 50257 x 1024: 47 us where the logits alone take 26, and
// HBM 32 for the weight and its copy; four warps: 65; loads ahead of the conversion, or each CTA the rows that its products read:
// no change).  Rows that take no part (a factor of 0) become zeros, so that a NaN or an infinity in one does not reach the others' sums.
template <typename Factor>
__device__ __forceinline__ void copy_f16(const uint4* src, uint4* dst, int n_rows, int C, int warp, int lane, Factor row_factor_of) {
  constexpr int R = 4;
  const int per_row = C / 8, pitch = head_pitch(C) / 8, step = int(gridDim.x) * COPY_WARPS * R;
  for (int r0 = (int(blockIdx.x) * COPY_WARPS + warp) * R; r0 < n_rows; r0 += step) {
    const float mine = lane < R && r0 + lane < n_rows ? row_factor_of(r0 + lane) : 0.f;
    const unsigned rows = __ballot_sync(0xffffffffu, mine != 0.f);
    float factor[R];
#pragma unroll
    for (int i = 0; i < R; ++i) factor[i] = __shfl_sync(0xffffffffu, mine, i);
    for (int c = lane; c < per_row; c += 64) {
      uint4 v[R][2];
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          v[i][u] = (rows >> i & 1u) && c + 32 * u < per_row ? __ldg(src + size_t(r0 + i) * per_row + c + 32 * u) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (r0 + i < n_rows && c + 32 * u < per_row)
            dst[size_t(r0 + i) * pitch + c + 32 * u] = make_uint4(f16x2_of_bf16x2(v[i][u].x, factor[i]), f16x2_of_bf16x2(v[i][u].y, factor[i]),
                                                                 f16x2_of_bf16x2(v[i][u].z, factor[i]), f16x2_of_bf16x2(v[i][u].w, factor[i]));
    }
  }
}

template <bool CE, bool KD>
__device__ __forceinline__ void make_copies(const HeadLogits& p, int warp, int lane) {
  int ew, ex;
  if (p.v0 == 0) {
    ew = copy_exponent(range_top(p.tops, p.n_tops, lane));
    ex = copy_exponent(range_top(p.tops + HEAD_RANGE_CTAS, p.n_tops, lane));
    if (blockIdx.x == 0 && warp == 0 && lane == 0) { p.exps[0] = ew; p.exps[1] = ex; }
  } else {
    ew = p.exps[0];
    ex = p.exps[1];
  }
  if (p.xs) {
    const float scale = head_scale(p.grads);
    copy_f16(p.x, p.xs, p.N, p.C, warp, lane, [&](int row) {
      return row_is_live<CE, KD>(p.grads, row) ? ldexpf(1.f, ex - row_halvings(p.grads, row, scale)) : 0.f;
    });
  }
  if (p.ws) copy_f16(p.w + size_t(p.v0) * (p.C / 8), p.ws, p.cols, p.C, warp, lane, [f = ldexpf(1.f, ew)](int) { return f; });
}

template <bool CE, bool KD>
__device__ __forceinline__ void head_part(const HeadLogits& p, int part, int row, const RunningSum& s1, const RunningSum& s2, float dot) {
  float* o = p.part + size_t(part) * head_values(CE, KD) * p.N + row;
  if (CE) { o[0] = s1.ref; o[p.N] = s1.sum; o += 2 * size_t(p.N); }
  if (KD) { o[0] = s2.ref; o[p.N] = s2.sum; o[2 * size_t(p.N)] = dot; }
}

// A lane of an epilogue warp is a row, its registers are 32 consecutive columns.  Two groups of four epilogue warps drain alternate
// tiles, each the accumulator of its own (eight warps on every tile leave twice the parts to join).  A column of a row that the
// teacher asks for is not known to the compiler: where a warp has one, 16 columns go through shared memory, lanes side by side (32
// compared registers an entry cost 6 to 30 % of a launch at 32 to 64 entries a row).
constexpr int logits_threads(bool grad) { return HEAD_THREADS + (grad ? 32 * COPY_WARPS : 0); }

template <bool CE, bool KD, bool GRAD>
__global__ void __launch_bounds__(logits_threads(GRAD), 1)
head_logits_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                   const __grid_constant__ HeadLogits p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  const uint32_t a_base = base, b_base = base + HEAD_STAGES * HEAD_OPERAND;
  uint8_t* behind = smem_raw + (base - raw_addr) + 2 * HEAD_STAGES * HEAD_OPERAND;
  HeadRing* ctl = reinterpret_cast<HeadRing*>(behind);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = int(cluster_rank());
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_x);
    tma_prefetch_desc(&tmap_w);
  }
  pair_ring_init(ctl, warp, 8);
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  const int pair = int(blockIdx.x >> 1), n_pairs = int(gridDim.x >> 1);
  const int tm = (p.N + HEAD_TILE - 1) / HEAD_TILE, tv = (p.cols + HEAD_TILE - 1) / HEAD_TILE, total = tm * tv;
  const int n_kb = (p.C + HEAD_BK - 1) / HEAD_BK;

  if (!GRAD && blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0u;

  if (warp == 0) {
    // ---------------- TMA: this CTA's rows and its half of the columns ----------------
    // Where 128 rows are more than there are, the rest of the operand's memory holds anything: it makes rows of the accumulator that
    // nobody reads.
    const bool has_rows = rank == 0 || p.N > HEAD_TILE / 2;
    const uint32_t bytes = 2 * HEAD_OPERAND + uint32_t(p.box_rows) * (HEAD_BK * 2) * (p.N > HEAD_TILE / 2 ? 2 : 1);       // of both CTAs
    int s = 0;
    uint32_t ph = 1u;
    bool ok = true;
    for (int t = pair; ok && t < total; t += n_pairs) {
      int m, v;
      head_tile(t, tm, tv, &m, &v);
      const int row = m * HEAD_TILE + rank * (HEAD_TILE / 2), col = p.v0 + v * HEAD_TILE + rank * (HEAD_TILE / 2);
#pragma unroll 1
      for (int kb = 0; kb < n_kb; ++kb) {
        if (!mbar_wait(smem_u32(&ctl->empty[s]), ph, abort_flag, p.status, JB200_STATUS_HEAD_LOAD)) { ok = false; break; }
        const uint32_t full = cluster_map(smem_u32(&ctl->full[s]), 0u);
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&ctl->full[s]), bytes);
          if (has_rows) pair_tma_load_2d(a_base + uint32_t(s) * HEAD_OPERAND, &tmap_x, kb * HEAD_BK, row, full);
          pair_tma_load_2d(b_base + uint32_t(s) * HEAD_OPERAND, &tmap_w, kb * HEAD_BK, col, full);
        }
        __syncwarp();
        if (++s == HEAD_STAGES) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA: the leader's, for both CTAs ----------------
    if (rank == 0) {
      const uint64_t ad0 = umma_desc_k_sw128(a_base), bd0 = umma_desc_k_sw128(b_base);
      constexpr uint32_t idesc = umma_idesc_bf16(HEAD_TILE, HEAD_TILE);
      int s = 0;
      uint32_t ph = 0u, tile = 0u;
      bool ok = true;
      for (int t = pair; ok && t < total; t += n_pairs, ++tile) {
        const uint32_t acc = tile & 1u;
        if (!cluster_mbar_wait(smem_u32(&ctl->acc_empty[acc]), ((tile >> 1) & 1u) ^ 1u, abort_flag, p.status, JB200_STATUS_HEAD_MMA)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + acc * HEAD_TILE;
#pragma unroll 1
        for (int kb = 0; kb < n_kb; ++kb) {
          if (!cluster_mbar_wait(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, JB200_STATUS_HEAD_MMA)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            const uint64_t ad = ad0 + uint64_t(s * (HEAD_OPERAND >> 4)), bd = bd0 + uint64_t(s * (HEAD_OPERAND >> 4));
#pragma unroll
            for (int kk = 0; kk < HEAD_BK / 16; ++kk)
              pair_umma(d, ad + uint64_t(kk * 2), bd + uint64_t(kk * 2), idesc, (kb | kk) != 0 ? 1u : 0u);
            pair_commit(smem_u32(&ctl->empty[s]));
            if (kb + 1 == n_kb) pair_commit(smem_u32(&ctl->acc_full[acc]));
          }
          __syncwarp();
          if (++s == HEAD_STAGES) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else if (GRAD && warp >= HEAD_EPI_WARP0 + 8) {
    make_copies<CE, KD>(p, warp - HEAD_EPI_WARP0 - 8, lane);
  } else {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3;                              // TMEM lanes this warp may read
    const float scale = GRAD ? head_scale(p.grads) : 1.f;
    const uint32_t group = uint32_t(warp - HEAD_EPI_WARP0) >> 2;
    // [16 columns][32 lanes] of this warp
    float* stage = reinterpret_cast<float*>(behind + HEAD_CTL) + (warp - HEAD_EPI_WARP0) * 512 + lane;
    const float k1 = LOG2E, k2 = LOG2E * p.inv_tau;
    RunningSum s1, s2;
    float dot = 0.f;
    uint32_t ph = 0u;
    for (int t = pair + int(group) * n_pairs; t < total; t += 2 * n_pairs, ph ^= 1u) {
      int m, v;
      head_tile(t, tm, tv, &m, &v);
      const int f0 = p.v0 + v * HEAD_TILE;                     // first vocabulary column, and the first beyond the launch's
      const int f_end = min(f0 + HEAD_TILE, p.v0 + p.cols);
      const int row = m * HEAD_TILE + rank * (HEAD_TILE / 2) + quarter * 32 + lane;
      const bool on = row < p.N;
      Entries e;
      if (KD && on) e.begin(p.entries + size_t(row) * p.K, p.K, __ldg(p.starts + size_t(row) * p.v_tiles + f0 / HEAD_TILE));
      int target = -1;
      if (CE && on) {
        const long long y = p.targets[row];
        if (y >= f0 && y < f_end) target = int(y) - f0;
      }
      RowGrad<CE, KD> rg;
      if (GRAD && on) rg.load(p.grads, row, row_scale(p.grads, row, scale));
      if (!mbar_wait(smem_u32(&ctl->acc_full[group]), ph, abort_flag, p.status, JB200_STATUS_HEAD_EPILOGUE)) break;
      tc_fence_after_sync();
      __syncwarp();
      const uint32_t t_lane = tmem + (uint32_t(quarter * 32) << 16) + group * HEAD_TILE;
      // 32 columns a time; the accumulator is free once the last have come.  Statistics: the next are on their way from tensor memory meanwhile
      // (both losses of 4096 rows 285 -> 273 us; gradients have no registers for it, and took as long with them).
      const auto chunk = [&](uint32_t (&z)[32], int c0) {
        const int col = f0 + c0;
        if constexpr (GRAD) {
          float g[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const float x = __uint_as_float(z[j]);
            float y = 0.f;
            if (CE) y = rg.p1 * ex2(fmaf(x, k1, -rg.l1));
            if (KD) y = fmaf(rg.p2, ex2(fmaf(x, k2, -rg.l2)), y);
            g[j] = y;
          }
          if (CE && __any_sync(0xffffffffu, unsigned(target - c0) < 32u)) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (target - c0 == j) g[j] -= rg.g1;
          }
          if (KD) {
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              if (!__any_sync(0xffffffffu, e.id < col + h + 16)) continue;
#pragma unroll
              for (int j = 0; j < 16; ++j) stage[j * 32] = g[h + j];
              while (e.id < col + h + 16) {                    // an id may come twice
                stage[(e.id - col - h) * 32] -= rg.g2 * e.q;
                e.step();
              }
#pragma unroll
              for (int j = 0; j < 16; ++j) g[h + j] = stage[j * 32];
              __syncwarp();
            }
          }
          if (col + 32 > f_end) {                              // columns past the vocabulary: the products read zeros
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col + j >= f_end) g[j] = 0.f;
          }
          if (on) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = rg.live ? pack_f16x2(g[2 * j], g[2 * j + 1]) : 0u;
            __half* d = p.g + size_t(row) * p.ldg + (col - p.v0);
            st_global_256(d, w);
            st_global_256(d + 16, w + 8);
          }
        } else {
          if (CE && __any_sync(0xffffffffu, unsigned(target - c0) < 32u)) {
            const float x = pick32(z, target - c0);
            if (unsigned(target - c0) < 32u) p.z_target[row] = x;
          }
          if (KD) {
#pragma unroll
            for (int h = 0; h < 32; h += 16) {
              if (!__any_sync(0xffffffffu, e.id < col + h + 16)) continue;
#pragma unroll
              for (int j = 0; j < 16; ++j) stage[j * 32] = __uint_as_float(z[h + j]);
              while (e.id < col + h + 16) {
                if (e.q != 0.f) dot = fmaf(e.q, stage[(e.id - col - h) * 32], dot);
                e.step();
              }
              __syncwarp();
            }
          }
          if (col + 32 > f_end) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col + j >= f_end) z[j] = 0xff800000u;        // -inf
          }
          float tops[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            tops[j] = __uint_as_float(z[j]);
#pragma unroll
            for (int i = j + 4; i < 32; i += 4) tops[j] = fmaxf(tops[j], __uint_as_float(z[i]));
          }
          const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          if (CE) s1.add(z, top, k1);
          if (KD) s2.add(z, top, k2);
        }
      };
      const auto drained = [&]() {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) cluster_mbar_arrive(cluster_map(smem_u32(&ctl->acc_empty[group]), 0u));
      };
      uint32_t za[32];
      if constexpr (GRAD) {
#pragma unroll 1
        for (int c0 = 0; c0 < HEAD_TILE; c0 += 32) {
          tmem_ld_32x32(t_lane + c0, za);
          tmem_ld_wait();
          if (c0 + 32 == HEAD_TILE) drained();
          chunk(za, c0);
        }
      } else {
        uint32_t zb[32];
        const int chunks = (f_end - f0 + 31) / 32;
        tmem_ld_32x32(t_lane, za);
#pragma unroll 1
        for (int i = 0; i < chunks; i += 2) {
          tmem_ld_wait();
          if (i + 1 < chunks) tmem_ld_32x32(t_lane + 32 * (i + 1), zb); else drained();
          chunk(za, 32 * i);
          if (i + 1 < chunks) {
            tmem_ld_wait();
            if (i + 2 < chunks) tmem_ld_32x32(t_lane + 32 * (i + 2), za); else drained();
            chunk(zb, 32 * (i + 1));
          }
        }
      }
      if (!GRAD && !p.carry) {
        if (on) head_part<CE, KD>(p, v, row, s1, s2, dot);
        s1 = s2 = RunningSum();
        dot = 0.f;
      }
    }
    if (!GRAD && p.carry) {
      const int row = pair % tm * HEAD_TILE + rank * (HEAD_TILE / 2) + quarter * 32 + lane;
      if (row < p.N) head_part<CE, KD>(p, 2 * (pair / tm) + int(group), row, s1, s2, dot);
    }
  }
  pair_ring_close(tmem, warp);
}

// ---------------------------------------------------------------------------
// Statistics of the tiles -> losses of the rows (and, from a single CTA, their means).
// ---------------------------------------------------------------------------
struct HeadRowsOut {
  const int64_t* targets;
  const float* neg_entropy;
  const float* part;
  const float* z_target;
  float *lse, *ce, *lse_t, *kd;
  float *mean_ce, *mean_kd;  // null: not wanted
  float* counts;             // with means: rows with a target, rows with a teacher
  unsigned int* ticket;
  int N, V, parts;
  float inv_tau, tau;
};

// 2^ref sum += sum over i of 2^r[i] s[i].  Parts without a finite logit have ref = -inf and a sum of 0 or NaN.
template <int N>
__device__ __forceinline__ void join(float& ref, float& sum, const float (&r)[N], const float (&s)[N]) {
  float to = ref;
#pragma unroll
  for (int i = 0; i < N; ++i) to = fmaxf(to, r[i]);
  const float at = to == -INFINITY ? 0.f : to;
  sum *= ex2(ref - at);
#pragma unroll
  for (int i = 0; i < N; ++i) sum = fmaf(s[i], ex2(r[i] - at), sum);
  ref = to;
}
__device__ __forceinline__ void join_lanes(float& ref, float& sum, int o) {
  const float r[1] = {__shfl_xor_sync(0xffffffffu, ref, o)}, s[1] = {__shfl_xor_sync(0xffffffffu, sum, o)};
  join(ref, sum, r, s);
}

// A CTA takes 32 rows: lanes are rows while the parts are read (WARPS of them at a time), then a warp joins the WARPS sums of 32 / WARPS rows.
// The CTA that ends last forms the means over all rows in a fixed order: thread, warp, warps.  Bound by latency; many warps where a
// wave of such CTAs holds all rows, else few, so that it does (16384 rows: 28 us with 32 warps).
template <bool CE, bool KD, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) head_join_kernel(const __grid_constant__ HeadRowsOut p) {
  pdl_wait();
  pdl_trigger();
  constexpr int F = head_values(CE, KD);
  __shared__ float s_v[WARPS][F][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float r1 = -INFINITY, s1 = 0.f, r2 = -INFINITY, s2 = 0.f, dot = 0.f;
  if (const int row = blockIdx.x * 32 + lane; row < p.N) {
    constexpr int U = 8;                 // parts asked for at a time
    for (int i0 = warp; i0 < p.parts; i0 += U * WARPS) {
      float ar[U], as[U], br[U], bs[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * WARPS;
        ar[u] = br[u] = -INFINITY;
        as[u] = bs[u] = 0.f;
        if (i < p.parts) {
          const float* v = p.part + size_t(i) * F * p.N + row;
          if (CE) { ar[u] = __ldcs(v); as[u] = __ldcs(v + p.N); v += 2 * size_t(p.N); }
          if (KD) { br[u] = __ldcs(v); bs[u] = __ldcs(v + p.N); dot += __ldcs(v + 2 * size_t(p.N)); }
        }
      }
      if (CE) join(r1, s1, ar, as);
      if (KD) join(r2, s2, br, bs);
    }
  }
  if (CE) { s_v[warp][0][lane] = r1; s_v[warp][1][lane] = s1; }
  if (KD) { s_v[warp][F - 3][lane] = r2; s_v[warp][F - 2][lane] = s2; s_v[warp][F - 1][lane] = dot; }
  __syncthreads();
  // lanes are now (row of the warp's, part)
  const int mine = warp * (32 / WARPS) + lane / WARPS, from = lane % WARPS;
  if (CE) { r1 = s_v[from][0][mine]; s1 = s_v[from][1][mine]; }
  if (KD) { r2 = s_v[from][F - 3][mine]; s2 = s_v[from][F - 2][mine]; dot = s_v[from][F - 1][mine]; }
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) {
    if (CE) join_lanes(r1, s1, o);
    if (KD) {
      join_lanes(r2, s2, o);
      dot += __shfl_xor_sync(0xffffffffu, dot, o);
    }
  }
  if (const int row = blockIdx.x * 32 + mine; from == 0 && row < p.N) {
    if (CE) {
      const double l = (double(r1) + log2(double(s1))) / double(LOG2E);
      const long long y = p.targets[row];
      p.lse[row] = r1;
      p.lse[size_t(p.N) + row] = s1;
      p.ce[row] = y == -100 ? 0.f : y >= 0 && y < p.V ? float(l - double(p.z_target[row])) : __int_as_float(0x7fc00000);
    }
    if (KD) {
      const double l = (double(r2) + log2(double(s2))) / double(LOG2E * p.inv_tau);      // tau times the logarithm of sum exp(z / tau)
      const float e = p.neg_entropy[row];
      p.lse_t[row] = r2;
      p.lse_t[size_t(p.N) + row] = s2;
      p.kd[row] = e == INFINITY ? 0.f : float(double(p.tau) * (double(p.tau) * double(e) + (l - double(dot))));
    }
  }
  if (!p.counts) return;

  __shared__ bool s_last;
  __shared__ double s_sum[2][WARPS];
  __shared__ int s_cnt[2][WARPS];
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = gridDim.x == 1 || atomicAdd(p.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum[2] = {0.0, 0.0};
  int cnt[2] = {0, 0};
  for (int r = threadIdx.x; r < p.N; r += 32 * WARPS) {
    if (CE) { sum[0] += double(__ldcg(p.ce + r)); cnt[0] += p.targets[r] != -100; }
    if (KD) { sum[1] += double(__ldcg(p.kd + r)); cnt[1] += p.neg_entropy[r] != INFINITY; }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      cnt[i] += __shfl_xor_sync(0xffffffffu, cnt[i], o);
    }
    if (lane == 0) { s_sum[i][warp] = sum[i]; s_cnt[i][warp] = cnt[i]; }
  }
  __syncthreads();
  if (threadIdx.x < 2 && (threadIdx.x == 0 ? CE : KD)) {
    const int i = threadIdx.x;
    double a = 0.0;
    int n = 0;
    for (int w = 0; w < WARPS; ++w) { a += s_sum[i][w]; n += s_cnt[i][w]; }
    float* mean = i == 0 ? p.mean_ce : p.mean_kd;
    if (mean) *mean = float(a / double(n));            // no row that counts: 0 / 0 = NaN, as the mean of the logits' loss has it
    p.counts[i] = float(n);
  }
}

// Ahead of a backward pass: the largest finite magnitudes of the weight and of the rows that take part, which the f16 copies are scaled
// by; a CTA leaves what it found (bf16 bits) of both.  Bound by HBM: 50257 x 1024 take 19 us alone; of a step of 37 rows 11, since it goes backwards
// and what the logits' kernel begins with has come last and is in L2.  With gradients row by row one more CTA finds their common factor, the largest finite one of its kind.
constexpr int RANGE_THREADS = 1024;
struct HeadRange {
  HeadGrads grads;
  const uint4 *w, *x;        // null: not wanted
  int V, N, per_row;         // rows of both, and their length in uint4
  unsigned* tops;            // [2][HEAD_RANGE_CTAS]
  int ctas;
};

// Larger one by 16-bit halves of `top` and v's finite magnitudes.
__device__ __forceinline__ unsigned finite_top(unsigned top, uint4 v) {
  const unsigned a[4] = {v.x & 0x7fff7fffu, v.y & 0x7fff7fffu, v.z & 0x7fff7fffu, v.w & 0x7fff7fffu};
#pragma unroll
  for (int j = 0; j < 4; ++j) top = __vmaxu2(top, a[j] & __vcmpltu2(a[j], 0x7f807f80u));
  return top;
}

__device__ void head_scale_job(const HeadGrads& p) {
  __shared__ float s_top[2][32];
  float ce = 0.f, kd = 0.f;
  for (int r = threadIdx.x; r < p.N; r += RANGE_THREADS) {
    const float2 f = row_factors(p, r);
    ce = fmaxf(ce, f.x);
    kd = fmaxf(kd, f.y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ce = fmaxf(ce, __shfl_xor_sync(0xffffffffu, ce, o));
    kd = fmaxf(kd, __shfl_xor_sync(0xffffffffu, kd, o));
  }
  if ((threadIdx.x & 31) == 0) { s_top[0][threadIdx.x >> 5] = ce; s_top[1][threadIdx.x >> 5] = kd; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < RANGE_THREADS / 32; ++w) { ce = fmaxf(ce, s_top[0][w]); kd = fmaxf(kd, s_top[1][w]); }
    *p.scale = common_factor(ce, kd);
  }
}

__global__ void __launch_bounds__(RANGE_THREADS) head_range_kernel(const __grid_constant__ HeadRange p) {
  pdl_wait();
  pdl_trigger();
  if (int(blockIdx.x) == p.ctas) {
    head_scale_job(p.grads);
    return;
  }
  __shared__ unsigned s_top[2][RANGE_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned tw = 0, tx = 0;
  if (p.x) {
    for (int row = int(blockIdx.x) * (RANGE_THREADS / 32) + warp; row < p.N; row += p.ctas * (RANGE_THREADS / 32)) {
      if (!row_is_live(p.grads, row)) continue;
#pragma unroll 4
      for (int c = lane; c < p.per_row; c += 32) tx = finite_top(tx, __ldg(p.x + size_t(row) * p.per_row + c));
    }
  }
  if (p.w) {
    constexpr int U = 8;
    const long long step = (long long)(p.ctas) * RANGE_THREADS;
    long long i = (long long)(p.V) * p.per_row - 1 - ((long long)(blockIdx.x) * RANGE_THREADS + threadIdx.x);
    for (; i >= (U - 1) * step; i -= U * step) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = __ldg(p.w + (i - u * step));
#pragma unroll
      for (int u = 0; u < U; ++u) tw = finite_top(tw, v[u]);
    }
    for (; i >= 0; i -= step) tw = finite_top(tw, __ldg(p.w + i));
  }
  tw = __reduce_max_sync(0xffffffffu, max(tw & 0xffffu, tw >> 16));
  tx = __reduce_max_sync(0xffffffffu, max(tx & 0xffffu, tx >> 16));
  if (lane == 0) { s_top[0][warp] = tw; s_top[1][warp] = tx; }
  __syncthreads();
  if (warp < 2) {
    const unsigned top = __reduce_max_sync(0xffffffffu, s_top[warp][lane]);
    if (lane == 0) p.tops[warp * HEAD_RANGE_CTAS + blockIdx.x] = top;
  }
}

// Pairs of a launch.  Where as many waves do with a multiple of the row tiles, that: a pair then keeps to its rows.
int head_pairs(int N, int cols, int sms) {
  const long long tm = (N + HEAD_TILE - 1) / HEAD_TILE, tiles = tm * ((cols + HEAD_TILE - 1) / HEAD_TILE);
  const long long pairs = tiles < sms / 2 ? tiles : sms / 2;
  if (tm > pairs) return int(pairs);
  const long long even = pairs / tm * tm;
  return int((tiles + even - 1) / even == (tiles + pairs - 1) / pairs ? even : pairs);
}
template <bool CE, bool KD, bool GRAD>
int launch_logits(const CUtensorMap& tx, const CUtensorMap& tw, const HeadLogits& p, int sms, cudaStream_t stream) {
  auto kernel = head_logits_kernel<CE, KD, GRAD>;
  constexpr size_t smem = HEAD_SMEM + (KD ? 8 * 512 * 4 : 0);
  static_assert(smem <= 227 * 1024, "shared memory of one CTA");
  JB_MAX_SMEM(kernel, smem);
  launch_dep_cluster(kernel, dim3(2 * unsigned(head_pairs(p.N, p.cols, sms))), dim3(logits_threads(GRAD)), smem, 2, stream, tx, tw, p);
  JB_LAUNCH_CHECK("head_logits_kernel");
  return JB200_OK;
}
template <bool GRAD>
int launch_logits(bool ce, bool kd, const CUtensorMap& tx, const CUtensorMap& tw, const HeadLogits& p, int sms, cudaStream_t stream) {
  if (ce && kd) return launch_logits<true, true, GRAD>(tx, tw, p, sms, stream);
  return ce ? launch_logits<true, false, GRAD>(tx, tw, p, sms, stream) : launch_logits<false, true, GRAD>(tx, tw, p, sms, stream);
}

template <bool CE, bool KD>
int launch_join(const HeadRowsOut& o, cudaStream_t stream) {
  const int ctas = o.N > 0 ? (o.N + 31) / 32 : 1;
  const bool many = ctas <= sm_count();
  launch_dep(many ? head_join_kernel<CE, KD, 32> : head_join_kernel<CE, KD, 8>, ctas, many ? 1024 : 256, 0, stream, o);
  JB_LAUNCH_CHECK("head_join_kernel");
  return JB200_OK;
}

// Everything about the arguments that both directions share.
int check_head(const jb200_head* h, const char* what) {
  JB_REQUIRE(h, "%s: null pointer", what);
  JB_REQUIRE(h->N >= 0 && h->V >= 1 && h->C >= 64 && h->C % 8 == 0,
             "%s: bad shape (%d rows, vocabulary %d, %d channels; channels must be a multiple of 8 and at least 64)", what, h->N, h->V, h->C);
  const long long tiles = (long long)((h->N + HEAD_TILE - 1) / HEAD_TILE) * ((h->V + HEAD_TILE - 1) / HEAD_TILE);
  JB_REQUIRE(tiles < INT_MAX / 4 && h->V <= INT_MAX - HEAD_TILE && h->N <= INT_MAX - HEAD_TILE, "%s: too many logits (%d x %d)", what, h->N, h->V);
  JB_REQUIRE(h->N == 0 || (h->x && h->w), "%s: null pointer", what);
  JB_REQUIRE(aligned16(h->x) && aligned16(h->w), "%s: rows and weight must be 16-byte aligned", what);
  JB_REQUIRE(h->N == 0 || h->targets || h->teacher, "%s: neither targets nor a teacher", what);
  JB_REQUIRE(h->N == 0 || !h->targets || h->lse, "%s: lse is needed with targets", what);
  if (h->teacher) {
    JB_REQUIRE(h->K >= 1 && h->K <= TEACHER_MAX, "%s: a teacher has 1 to %d entries a row, got %d", what, TEACHER_MAX, h->K);
    JB_REQUIRE(h->lse_t, "%s: null pointer (teacher)", what);
    JB_REQUIRE((reinterpret_cast<uintptr_t>(h->teacher) & 15u) == 0, "%s: teacher rows must be 16-byte aligned", what);
    JB_REQUIRE(h->temperature > 0.f && h->temperature <= FLT_MAX && 1.5f / h->temperature <= FLT_MAX, "%s: temperature must be positive and finite", what);
  }
  return JB200_OK;
}

}  // namespace

int encode_head_map(CUtensorMap* tm, const void* ptr, long long cols, long long pitch, long long rows, int box_rows, const char* what) {
  const cuuint64_t dim[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t stride[1] = {cuuint64_t(pitch) * 2};
  const cuuint32_t box[2] = {HEAD_BK, cuuint32_t(box_rows)};
  return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, what);
}

HeadShares head_shares(int n_long, int k_long, int n_short, int k_short, int pairs) {
  HeadShares best{};
  best.span = LLONG_MAX;
  const int turns = n_long / pairs, uneven = n_long % pairs, rest = pairs - uneven;
  for (int up = 0; up < 2; ++up) {
    const int more = uneven == 0 ? 0 : k_long / k_short + up;
    const long long left = n_short - (long long)rest * more;
    const int rounds = left > 0 ? int((left + pairs - 1) / pairs) : 0;
    const long long a = uneven ? (long long)(turns + 1) * k_long + (long long)rounds * k_short : 0;
    // (where the others alone have more than there are, they share those)
    const long long take = left > 0 ? rounds + more : (n_short + rest - 1) / rest;
    const long long b = (long long)turns * k_long + take * k_short;
    const long long span = a > b ? a : b;
    if (span < best.span) best = {uneven, rounds, more, span};
  }
  return best;
}

namespace {
// K-blocks' time of an item of k of them: its epilogue hides behind the next item's products, but not below some eight.
int item_time(int k) { return k > 8 ? k : 8; }

// Time of a piece of n tiles in K-blocks of a pair (512 cycles), and of what follows from its slabs.
long long piece_time(long long n, int N, int C, int slabs, int pairs) {
  const int width = head_width(C), tm = (N + HEAD_TILE - 1) / HEAD_TILE, tc = (C + width - 1) / width, kc = (C + HEAD_BK - 1) / HEAD_BK;
  const int k_dw = item_time((N + HEAD_BK - 1) / HEAD_BK), k_dx = item_time(int((n * (HEAD_TILE / HEAD_BK) + slabs - 1) / slabs));
  const int n_dw = int(n) * tc, n_dx = slabs * tm * tc;
  const HeadShares s = k_dw > k_dx ? head_shares(n_dw, k_dw, n_dx, k_dx, pairs) : head_shares(n_dx, k_dx, n_dw, k_dw, pairs);
  return (tm * n + pairs - 1) / pairs * item_time(kc) + s.span * width / HEAD_TILE + 24;      // 24: two launches
}
}  // namespace

// The fastest of some cuts by that count.  Candidates: the fewest pieces that the workspace allows and a few more, even ones, and those
// whose tiles fill the pairs without a rest.  (16384 x 50257 x 1024, backward products: seven even pieces of 29 tiles, the busiest pair
// with 976 K-blocks where the mean is 802, 2390 us; pieces of 37, 1030 for 1024, 2151 us.)
HeadPlan head_plan(int N, int V, int C, int pairs) {
  struct Kept { int N, V, C, pairs; HeadPlan plan; };
  thread_local Kept kept{};
  if (kept.N == N && kept.V == V && kept.C == C && kept.pairs == pairs) return kept.plan;
  const long long tv = (V + HEAD_TILE - 1) / HEAD_TILE, tm = (N + HEAD_TILE - 1) / HEAD_TILE;
  long long most = (long long)(PIECE_BYTES / (size_t(N > 0 ? N : 1) * HEAD_TILE * 2));
  most = most < 1 ? 1 : most > tv ? tv : most;
  long long cand[12];
  int n_cand = 0;
  const long long fewest = (tv + most - 1) / most;
  for (int i = 0; i < 6 && fewest + i <= tv; ++i) cand[n_cand++] = (tv + fewest + i - 1) / (fewest + i);
  long long step = pairs;                                      // smallest number of tiles whose row tiles fill the pairs
  for (long long a = pairs, b = tm; b; ) { const long long r = a % b; a = b; b = r; step = pairs / a; }
  for (int i = 0; i < 4; ++i) {
    const long long n = (most / step - i) * step;
    if (n > 0) cand[n_cand++] = n;
  }
  HeadPlan best{};
  long long best_time = LLONG_MAX;
  for (int i = 0; i < n_cand; ++i) {
    const long long per = cand[i], pieces = (tv + per - 1) / per, last = tv - (pieces - 1) * per;
    for (int slabs = 1; slabs <= 64; slabs += slabs < 4 ? 1 : slabs / 4) {
      if (slabs > 1 && per * (HEAD_TILE / HEAD_BK) / slabs < 8) break;      // at least eight K-blocks each
      const long long reduce = slabs == 1 ? 0 : 12 + (long long)slabs * N * C / 400000;      // a launch; 4 bytes read at 6 TB/s
      const long long time = (pieces - 1) * piece_time(per, N, C, slabs, pairs) + piece_time(last, N, C, slabs, pairs) + reduce;
      if (time < best_time) {
        best_time = time;
        best = {int(per) * HEAD_TILE, int(pieces), slabs};
      }
    }
  }
  kept = {N, V, C, pairs, best};
  return best;
}

size_t teacher_rows_bytes(int N, int K, int V) { return N < 1 || K < 1 || V < 1 ? 0 : teacher_layout(N, K, V).total; }

int launch_teacher_rows(const int64_t* ids, const void* logits, int logits_dtype, int N, int K, int V, float temperature, void* rows,
                        cudaStream_t stream) {
  JB_REQUIRE(N >= 0 && V >= 1, "teacher_rows: bad shape");
  JB_REQUIRE(K >= 1 && K <= TEACHER_MAX, "teacher_rows: a teacher has 1 to %d entries a row, got %d", TEACHER_MAX, K);
  JB_REQUIRE(logits_dtype == 0 || logits_dtype == 1, "teacher_rows: dtype must be 0 (f32) or 1 (bf16)");
  JB_REQUIRE(temperature > 0.f && temperature <= FLT_MAX && 1.5f / temperature <= FLT_MAX, "teacher_rows: temperature must be positive and finite");
  if (N == 0) return JB200_OK;
  JB_REQUIRE(ids && logits && rows, "teacher_rows: null pointer");
  JB_REQUIRE(aligned16(rows), "teacher_rows: rows must be 16-byte aligned");
  const TeacherLayout at = teacher_layout(N, K, V);
  uint8_t* base = static_cast<uint8_t*>(rows);
  float* neg_entropy = static_cast<float*>(rows);
  int2* entries = reinterpret_cast<int2*>(base + at.entries);
  uint16_t* starts = reinterpret_cast<uint16_t*>(base + at.starts);
  const dim3 grid((N + TEACHER_WARPS - 1) / TEACHER_WARPS), block(32 * TEACHER_WARPS);
  if (logits_dtype == 0) {
    launch_dep(teacher_rows_kernel<float>, grid, block, 0, stream, ids, static_cast<const float*>(logits), N, K, V, 1.0f / temperature,
               neg_entropy, entries, starts);
  } else {
    launch_dep(teacher_rows_kernel<__nv_bfloat16>, grid, block, 0, stream, ids, static_cast<const __nv_bfloat16*>(logits), N, K, V,
               1.0f / temperature, neg_entropy, entries, starts);
  }
  JB_LAUNCH_CHECK("teacher_rows_kernel");
  return JB200_OK;
}

namespace {
// (one row: 35 us against 26 us with boxes of 128, nearly all of them beyond the matrix)
int box_rows(int N) { return N >= HEAD_TILE / 2 ? HEAD_TILE / 2 : (N + 7) / 8 * 8; }

void set_teacher(HeadLogits& p, const jb200_head* h) {
  if (!h->teacher) return;
  const TeacherLayout at = teacher_layout(h->N, h->K, h->V);
  const uint8_t* base = static_cast<const uint8_t*>(h->teacher);
  p.entries = reinterpret_cast<const int2*>(base + at.entries);
  p.starts = reinterpret_cast<const uint16_t*>(base + at.starts);
  p.K = h->K;
  p.v_tiles = (h->V + HEAD_TILE - 1) / HEAD_TILE;
}
}  // namespace

// What launch_head_loss lays out in it: the parts, z_target and the rows' losses that the caller does not ask for, the ticket.
size_t head_loss_scratch_bytes(int N, int V, int has_targets, int has_teacher) {
  const size_t parts = (size_t(V) + HEAD_TILE - 1) / HEAD_TILE;
  return (parts * head_values(has_targets != 0, has_teacher != 0) + 3) * size_t(N) * 4 + 4;
}

int launch_head_loss(const jb200_head* h, float* ce, float* kd, float* mean_ce, float* mean_kd, float* counts, void* scratch, cudaStream_t stream) {
  int rc = check_head(h, "head_loss");
  if (rc != JB200_OK) return rc;
  JB_REQUIRE(h->N == 0 || scratch, "head_loss: null pointer (scratch)");
  JB_REQUIRE(counts || (!mean_ce && !mean_kd), "head_loss: null pointer (counts)");
  const bool has_ce = h->targets != nullptr, has_kd = h->teacher != nullptr;
  if (h->N == 0 && !counts) return JB200_OK;
  HeadRowsOut o{};
  o.targets = h->targets; o.neg_entropy = static_cast<const float*>(h->teacher);
  o.lse = h->lse; o.lse_t = h->lse_t;
  o.mean_ce = mean_ce; o.mean_kd = mean_kd; o.counts = counts;
  o.N = h->N; o.V = h->V;
  o.tau = has_kd ? h->temperature : 1.f;
  o.inv_tau = 1.0f / o.tau;
  o.parts = (h->V + HEAD_TILE - 1) / HEAD_TILE;
  if (h->N > 0) {
    const int sms = sm_count();
    if (sms < 2) return JB200_ERR_CUDA;
    HeadLogits p{};
    p.N = h->N; p.V = h->V; p.C = h->C; p.v0 = 0; p.cols = h->V;
    p.targets = h->targets; p.inv_tau = o.inv_tau;
    set_teacher(p, h);
    const int tm = (h->N + HEAD_TILE - 1) / HEAD_TILE, pairs = head_pairs(h->N, h->V, sms);
    p.carry = pairs % tm == 0 && tm <= HEAD_GROUP && 2 * (pairs / tm) <= o.parts;
    if (p.carry) o.parts = 2 * (pairs / tm);
    p.part = static_cast<float*>(scratch);
    p.z_target = p.part + size_t(o.parts) * head_values(has_ce, has_kd) * h->N;
    // rows' losses that the caller does not ask for live here
    o.ce = ce ? ce : p.z_target + size_t(h->N);
    o.kd = kd ? kd : p.z_target + 2 * size_t(h->N);
    p.ticket = o.ticket = reinterpret_cast<unsigned int*>(p.z_target + 3 * size_t(h->N));
    p.status = device_status_ptr();
    if (!p.status) return JB200_ERR_CUDA;
    o.part = p.part; o.z_target = p.z_target;
    CUtensorMap tx, tw;
    p.box_rows = box_rows(h->N);
    if ((rc = encode_head_map(&tx, h->x, h->C, h->C, h->N, p.box_rows, "head_loss (rows)")) != JB200_OK) return rc;
    if ((rc = encode_head_map(&tw, h->w, h->C, h->C, h->V, HEAD_TILE / 2, "head_loss (weight)")) != JB200_OK) return rc;
    if ((rc = launch_logits<false>(has_ce, has_kd, tx, tw, p, sms, stream)) != JB200_OK) return rc;
  }
  // (without rows both means are written: nothing says which was asked for)
  const int rc2 = (has_ce && has_kd) || h->N == 0 ? launch_join<true, true>(o, stream) : has_ce ? launch_join<true, false>(o, stream)
                                                                                                : launch_join<false, true>(o, stream);
  if (rc2 != JB200_OK) return rc2;
  return JB200_OK;
}

namespace {
struct BackwardScratch {
  size_t xs, ws, scale, exps, tops, g, slabs, total;
};
BackwardScratch backward_scratch(int N, int C, const HeadPlan& pl) {
  BackwardScratch s;
  s.xs = 0;
  s.ws = up256(size_t(N) * head_pitch(C) * 2);
  s.scale = s.ws + up256(size_t(pl.cols) * head_pitch(C) * 2);
  s.exps = s.scale + 16;
  s.tops = s.scale + 256;
  s.g = s.tops + up256(2 * HEAD_RANGE_CTAS * 4);
  s.slabs = s.g + up256(size_t(N) * pl.cols * 2);
  s.total = s.slabs + up256(size_t(pl.slabs) * N * C * 4);
  return s;
}
}  // namespace

size_t head_loss_backward_scratch_bytes(int N, int V, int C) {
  const int sms = sm_count();
  if (N < 1 || V < 1 || C < 1 || sms < 2) return 0;
  return backward_scratch(N, C, head_plan(N, V, C, sms / 2)).total;
}

int launch_head_loss_backward(const jb200_head* h, const float* g_ce, int g_ce_stride, const float* n_ce, const float* g_kd, int g_kd_stride,
                              const float* n_kd, void* dx, int dx_dtype, void* dw, int dw_dtype, void* scratch, cudaStream_t stream) {
  int rc = check_head(h, "head_loss_backward");
  if (rc != JB200_OK) return rc;
  JB_REQUIRE((dx_dtype == 0 || dx_dtype == 1) && (dw_dtype == 0 || dw_dtype == 1), "head_loss_backward: dtype must be 0 (f32) or 1 (bf16)");
  JB_REQUIRE(((reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(dx)) & 31u) == 0, "head_loss_backward: dx and dw must be 32-byte aligned");
  if (!dx && !dw) return JB200_OK;
  if (h->N == 0) {
    if (dw) JB_CUDA(cudaMemsetAsync(dw, 0, size_t(h->V) * h->C * (dw_dtype ? 2 : 4), stream));
    return JB200_OK;
  }
  JB_REQUIRE(scratch && (reinterpret_cast<uintptr_t>(scratch) & 255u) == 0, "head_loss_backward: scratch must be 256-byte aligned");
  JB_REQUIRE((!h->targets || g_ce) && (!h->teacher || g_kd), "head_loss_backward: null pointer (gradients of the losses)");
  JB_REQUIRE((g_ce_stride == 0 || g_ce_stride == 1) && (g_kd_stride == 0 || g_kd_stride == 1), "head_loss_backward: strides must be 0 or 1");
  const int sms = sm_count();
  if (sms < 2) return JB200_ERR_CUDA;
  const HeadPlan pl = head_plan(h->N, h->V, h->C, sms / 2);
  const BackwardScratch at = backward_scratch(h->N, h->C, pl);
  uint8_t* base = static_cast<uint8_t*>(scratch);

  HeadGrads r{};
  r.targets = h->targets; r.neg_entropy = static_cast<const float*>(h->teacher);
  r.lse = h->lse; r.lse_t = h->lse_t;
  r.g_ce = g_ce; r.g_kd = g_kd; r.g_ce_stride = g_ce_stride; r.g_kd_stride = g_kd_stride; r.n_ce = n_ce; r.n_kd = n_kd;
  r.N = h->N; r.V = h->V;
  r.tau = h->teacher ? h->temperature : 1.f;
  const bool by_row = (h->targets && g_ce_stride) || (h->teacher && g_kd_stride);
  if (by_row) r.scale = reinterpret_cast<float*>(base + at.scale);

  HeadLogits p{};
  p.N = h->N; p.V = h->V; p.C = h->C;
  p.targets = h->targets; p.inv_tau = 1.0f / r.tau;
  set_teacher(p, h);
  p.grads = r;
  p.g = reinterpret_cast<__half*>(base + at.g);
  p.ldg = pl.cols;
  p.x = static_cast<const uint4*>(h->x);
  p.w = static_cast<const uint4*>(h->w);
  if (dw) p.xs = reinterpret_cast<uint4*>(base + at.xs);
  if (dx) p.ws = reinterpret_cast<uint4*>(base + at.ws);
  p.exps = reinterpret_cast<int*>(base + at.exps);
  HeadRange o{};
  o.grads = r;
  o.w = dx ? p.w : nullptr;
  o.x = dw ? p.x : nullptr;
  o.V = h->V; o.N = h->N; o.per_row = h->C / 8;
  o.tops = reinterpret_cast<unsigned*>(base + at.tops);
  o.ctas = 2 * sms < HEAD_RANGE_CTAS ? 2 * sms : HEAD_RANGE_CTAS;
  p.tops = o.tops;
  p.n_tops = o.ctas;
  launch_dep(head_range_kernel, o.ctas + (by_row ? 1 : 0), RANGE_THREADS, 0, stream, o);
  JB_LAUNCH_CHECK("head_range_kernel");
  HeadProducts q{};
  p.status = device_status_ptr();
  if (!p.status) return JB200_ERR_CUDA;
  p.box_rows = box_rows(h->N);
  CUtensorMap tx, tw;
  if ((rc = encode_head_map(&tx, h->x, h->C, h->C, h->N, p.box_rows, "head_loss_backward (rows)")) != JB200_OK) return rc;
  if ((rc = encode_head_map(&tw, h->w, h->C, h->C, h->V, HEAD_TILE / 2, "head_loss_backward (weight)")) != JB200_OK) return rc;
  q.N = h->N; q.V = h->V; q.C = h->C;
  q.ldg = pl.cols;
  q.grads = r;
  q.exps = p.exps;
  q.dx = dx; q.dx_bf16 = dx_dtype;
  // one slab in f32 is the result itself
  q.dx_slabs = !dx ? nullptr : dx_dtype == 0 && pl.slabs == 1 ? static_cast<float*>(dx) : reinterpret_cast<float*>(base + at.slabs);
  q.dw = dw; q.dw_bf16 = dw_dtype;
  q.status = p.status;
  for (int i = 0; i < pl.pieces; ++i) {
    p.v0 = q.v0 = i * pl.cols;
    p.cols = q.n_cols = h->V - p.v0 < pl.cols ? h->V - p.v0 : pl.cols;
    q.slabs = pl.slabs;
    q.first = i == 0;
    q.last = i + 1 == pl.pieces;
    if ((rc = launch_logits<true>(h->targets != nullptr, h->teacher != nullptr, tx, tw, p, sms, stream)) != JB200_OK) return rc;
    if ((rc = launch_head_products(q, p.g, base + at.xs, base + at.ws, sms, stream)) != JB200_OK) return rc;
    p.xs = nullptr;
  }
  return JB200_OK;
}

int head_plan_host(int N, int V, int C, int sms, int32_t* out3) {
  if (N < 1 || V < 1 || C < 1 || sms < 2 || !out3) return JB200_ERR_ARG;
  const HeadPlan pl = head_plan(N, V, C, sms / 2);
  out3[0] = pl.cols; out3[1] = pl.pieces; out3[2] = pl.slabs;
  return JB200_OK;
}

int head_walk_host(int n_long, int k_long, int n_short, int k_short, int pairs, int pair, int i) {
  if (n_long < 0 || n_short < 0 || k_long < 1 || k_short < 1 || pairs < 1 || pair < 0 || pair >= pairs || i < 0) return JB200_ERR_ARG;
  return head_walk(head_shares(n_long, k_long, n_short, k_short, pairs), n_long, n_short, pair, pairs, i);
}

}  // namespace jb

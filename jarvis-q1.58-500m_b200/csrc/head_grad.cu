// The products of the head's gradient, one launch per piece of the vocabulary:  dx += s G W  and  dW = s G^T xs,  where G (f16, rows x piece)
// is the gradient of the logits, relative to the factor s, that head_loss.cu's epilogue left, beside f16 copies of W and of the rows.
//
// CTA pairs as in the logits' kernel: 256 x 256 tiles, K-blocks of 64.  No operand is transposed in memory: G is the M operand K-major
// for dx (rows x vocabulary) and MN-major for dW (read as vocabulary x rows), the copies are the N operands MN-major, all from the
// same kind of [64 rows][64 columns] boxes.  Both products are items of one list, the longer kind first, so that their last waves
// fill each other's gaps.  Where there are few rows dx is summed over parts of the piece side by side, in slabs of their own, which a
// launch of its own adds up in their order (done by the warps that store a tile last it took 30 us of 37 rows instead of 5).
#include "head_loss.cuh"
#include "launchers.h"

namespace jb {

namespace {

struct Item {
  bool is_dw;
  int m0, n0;                // first row (token, or vocabulary row of the piece) and column (channel)
  int kb0, kb1;              // K-blocks
  int slab;
};

// The i-th item of a pair; false behind its last.
__device__ __forceinline__ bool head_item(const HeadProducts& p, int pair, int n_pairs, int i, Item* it) {
  const int n_long = p.dw_first ? p.dw_items : p.dx_items, n_short = p.dw_first ? p.dx_items : p.dw_items;
  int t = head_walk(p.shares, n_long, n_short, pair, n_pairs, i);
  if (t < 0) return false;
  it->is_dw = (t < n_long) == (p.dw_first != 0);
  if (t >= n_long) t -= n_long;
  const int tc = (p.C + p.width - 1) / p.width, n = t % tc;
  t /= tc;
  it->n0 = n * p.width;
  if (it->is_dw) {
    it->m0 = t * HEAD_TILE;
    it->kb0 = 0;
    it->kb1 = (p.N + HEAD_BK - 1) / HEAD_BK;
    it->slab = 0;
  } else {
    const int tm = (p.N + HEAD_TILE - 1) / HEAD_TILE, kb = (p.n_cols + HEAD_BK - 1) / HEAD_BK;
    it->slab = t / tm;
    it->m0 = (t - it->slab * tm) * HEAD_TILE;
    it->kb0 = int((long long)(kb) * it->slab / p.slabs);
    it->kb1 = int((long long)(kb) * (it->slab + 1) / p.slabs);
  }
  return true;
}

// 32 (or, at the edge, a multiple of 8) consecutive channels of a row.
__device__ __forceinline__ void store_f32(float* d, const uint32_t (&v)[32], int n, bool add) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (8 * j < n) {
      if (add) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                       ::"l"(d + 8 * j + 4 * i), "f"(__uint_as_float(v[8 * j + 4 * i])), "f"(__uint_as_float(v[8 * j + 4 * i + 1])),
                         "f"(__uint_as_float(v[8 * j + 4 * i + 2])), "f"(__uint_as_float(v[8 * j + 4 * i + 3])) : "memory");
      } else {
        st_global_256(d + 8 * j, v + 8 * j);
      }
    }
  }
}
__device__ __forceinline__ void add_f32(uint32_t (&v)[32], const float* d, int n) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (4 * j < n) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(d) + j);
      v[4 * j] = __float_as_uint(x.x + __uint_as_float(v[4 * j]));
      v[4 * j + 1] = __float_as_uint(x.y + __uint_as_float(v[4 * j + 1]));
      v[4 * j + 2] = __float_as_uint(x.z + __uint_as_float(v[4 * j + 2]));
      v[4 * j + 3] = __float_as_uint(x.w + __uint_as_float(v[4 * j + 3]));
    }
}
__device__ __forceinline__ void store_bf16(__nv_bfloat16* d, const uint32_t (&v)[32], int n, bool wide) {
  uint32_t w[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) w[j] = pack_bf16x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
  if (wide && n >= 32) {
    st_global_256(d, w);
    st_global_256(d + 16, w + 8);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (8 * j < n) *reinterpret_cast<uint4*>(d + 8 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}

__global__ void __launch_bounds__(HEAD_THREADS, 1)
head_products_kernel(const __grid_constant__ CUtensorMap tmap_g, const __grid_constant__ CUtensorMap tmap_w,
                     const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ HeadProducts p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t base = (raw_addr + 1023u) & ~1023u;
  const uint32_t a_base = base, b_base = base + HEAD_STAGES * HEAD_OPERAND;
  HeadRing* ctl = reinterpret_cast<HeadRing*>(smem_raw + (base - raw_addr) + 2 * HEAD_STAGES * HEAD_OPERAND);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = int(cluster_rank());
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_g);
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  pair_ring_init(ctl, warp, 16);
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  const int pair = int(blockIdx.x >> 1), n_pairs = int(gridDim.x >> 1);
  Item it;
  constexpr uint32_t BOX = HEAD_BK * HEAD_BK * 2;              // 8 KiB: [64 rows][64 columns]
  const int half_width = p.width / 2, boxes = (half_width + HEAD_BK - 1) / HEAD_BK;      // columns of the pair's tile from this CTA

  if (warp == 0) {
    // ---------------- TMA ----------------
    int s = 0;
    uint32_t ph = 1u;
    bool ok = true;
    for (int i = 0; ok && head_item(p, pair, n_pairs, i, &it); ++i) {
      const int row = it.m0 + rank * (HEAD_TILE / 2), col = it.n0 + rank * half_width;
      const uint32_t bytes = 2u * (uint32_t(HEAD_OPERAND) + uint32_t(boxes) * BOX);     // of both CTAs
#pragma unroll 1
      for (int kb = it.kb0; kb < it.kb1; ++kb) {
        if (!mbar_wait(smem_u32(&ctl->empty[s]), ph, abort_flag, p.status, JB200_STATUS_HEAD_LOAD)) { ok = false; break; }
        const uint32_t full = cluster_map(smem_u32(&ctl->full[s]), 0u);
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&ctl->full[s]), bytes);
          const uint32_t a = a_base + uint32_t(s) * HEAD_OPERAND, b = b_base + uint32_t(s) * HEAD_OPERAND;
          const int k = kb * HEAD_BK;
          if (it.is_dw) {
            pair_tma_load_2d(a, &tmap_g, row, k, full);
            pair_tma_load_2d(a + BOX, &tmap_g, row + HEAD_BK, k, full);
            for (int c = 0; c < boxes; ++c) pair_tma_load_2d(b + uint32_t(c) * BOX, &tmap_x, col + c * HEAD_BK, k, full);
          } else {
            pair_tma_load_2d(a, &tmap_g, k, row, full);
            pair_tma_load_2d(a + BOX, &tmap_g, k, row + HEAD_BK, full);
            for (int c = 0; c < boxes; ++c) pair_tma_load_2d(b + uint32_t(c) * BOX, &tmap_w, col + c * HEAD_BK, k, full);
          }
        }
        __syncwarp();
        if (++s == HEAD_STAGES) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA: the leader's, for both CTAs ----------------
    if (rank == 0) {
      // a K-step of 16: 32 bytes inside K-major rows, two groups of eight 128-byte rows of an MN-major block
      const uint64_t a_k = umma_desc_k_sw128(a_base), a_mn = umma_desc_mn_sw128(a_base, BOX), b_mn = umma_desc_mn_sw128(b_base, BOX);
      const uint32_t idesc = umma_idesc_bf16(HEAD_TILE, p.width) + IDESC_F16 + IDESC_B_MN;
      int s = 0;
      uint32_t ph = 0u, tile = 0u;
      bool ok = true;
      for (; ok && head_item(p, pair, n_pairs, int(tile), &it); ++tile) {
        const uint64_t ad0 = it.is_dw ? a_mn : a_k;
        const uint32_t a_step = it.is_dw ? 128u : 2u, id = it.is_dw ? idesc + IDESC_A_MN : idesc;
        const uint32_t acc = tile & 1u;
        if (!cluster_mbar_wait(smem_u32(&ctl->acc_empty[acc]), ((tile >> 1) & 1u) ^ 1u, abort_flag, p.status, JB200_STATUS_HEAD_MMA)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + acc * HEAD_TILE;
#pragma unroll 1
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!cluster_mbar_wait(smem_u32(&ctl->full[s]), ph, abort_flag, p.status, JB200_STATUS_HEAD_MMA)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            const uint64_t ad = ad0 + uint64_t(s * (HEAD_OPERAND >> 4)), bd = b_mn + uint64_t(s * (HEAD_OPERAND >> 4));
#pragma unroll
            for (int kk = 0; kk < HEAD_BK / 16; ++kk)
              pair_umma(d, ad + uint64_t(kk * a_step), bd + uint64_t(kk * 128), id, (kb > it.kb0 || kk != 0) ? 1u : 0u);
            pair_commit(smem_u32(&ctl->empty[s]));
            if (kb + 1 == it.kb1) pair_commit(smem_u32(&ctl->acc_full[acc]));
          }
          __syncwarp();
          if (++s == HEAD_STAGES) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else {
    // ---------------- epilogue: a lane is a row, its registers are channels ----------------
    const int quarter = warp & 3, half = (warp - HEAD_EPI_WARP0) >> 2;
    const float common = head_scale(p.grads);
    // two factors: their product may be below f32's range where the result is not
    const float dx_unit = ldexpf(1.f, -HEAD_G_EXP - p.exps[0]), dw_unit = ldexpf(1.f, -HEAD_G_EXP - p.exps[1]);
    uint32_t tile = 0u;
    for (; head_item(p, pair, n_pairs, int(tile), &it); ++tile) {
      const uint32_t acc = tile & 1u;
      const int row = it.m0 + rank * (HEAD_TILE / 2) + quarter * 32 + lane;
      const bool on = row < (it.is_dw ? p.n_cols : p.N);
      const float by = !it.is_dw && on ? row_scale(p.grads, row, common) : common;
      if (!mbar_wait(smem_u32(&ctl->acc_full[acc]), (tile >> 1) & 1u, abort_flag, p.status, JB200_STATUS_HEAD_EPILOGUE)) break;
      tc_fence_after_sync();
      __syncwarp();
      const uint32_t t_lane = tmem + (uint32_t(quarter * 32) << 16) + acc * HEAD_TILE;
      for (int c0 = half * 32; c0 < p.width; c0 += 64) {
        const int col = it.n0 + c0;
        if (col >= p.C) break;
        uint32_t v[32];
        tmem_ld_32x32(t_lane + c0, v);
        tmem_ld_wait();
        if (on) {
          const float unit = it.is_dw ? dw_unit : dx_unit;
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(by * (unit * __uint_as_float(v[j])));
          const int n = min(32, p.C - col);
          if (!it.is_dw) {
            const size_t o = size_t(row) * p.C + col;
            if (p.last && p.all_slabs == 1 && p.dx_bf16) {
              // the only slab: its sum so far and this piece's, rounded from here
              if (!p.first) add_f32(v, p.dx_slabs + o, n);
              store_bf16(static_cast<__nv_bfloat16*>(p.dx) + o, v, n, p.C % 16 == 0);
            } else {
              store_f32(p.dx_slabs + size_t(it.slab) * p.N * p.C + o, v, n, p.first == 0);
            }
          } else if (p.dw_bf16) {
            store_bf16(static_cast<__nv_bfloat16*>(p.dw) + (size_t(p.v0) + row) * p.C + col, v, n, p.C % 16 == 0);
          } else {
            store_f32(static_cast<float*>(p.dw) + (size_t(p.v0) + row) * p.C + col, v, n, false);
          }
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) cluster_mbar_arrive(cluster_map(smem_u32(&ctl->acc_empty[acc]), 0u));
    }
  }
  pair_ring_close(tmem, warp);
}

}  // namespace

namespace {
// Sum of the slabs in their order -> dx.
template <bool BF16_OUT>
__global__ void __launch_bounds__(256) head_dx_kernel(const float* __restrict__ slabs, int n_slabs, size_t n, void* __restrict__ dx) {
  pdl_wait();
  pdl_trigger();
  const size_t i = (size_t(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 8
  for (int s = 0; s < n_slabs; ++s) {
    const float4* v = reinterpret_cast<const float4*>(slabs + size_t(s) * n + i);
    const float4 x = __ldcs(v), y = __ldcs(v + 1);
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    b.x += y.x; b.y += y.y; b.z += y.z; b.w += y.w;
  }
  if constexpr (BF16_OUT) {
    reinterpret_cast<uint4*>(dx)[i / 8] = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
  } else {
    reinterpret_cast<float4*>(dx)[i / 4] = a;
    reinterpret_cast<float4*>(dx)[i / 4 + 1] = b;
  }
}
}  // namespace

// Channels of a tile: as few tiles of at most 256 as there can be, of the same width (a multiple of 32, what an MMA of 256 rows takes).
int head_width(int C) {
  const int tc = (C + HEAD_TILE - 1) / HEAD_TILE;
  return ((C + tc - 1) / tc + 31) / 32 * 32;
}

int launch_head_products(HeadProducts p, const void* g, const void* xs, const void* ws, int sms, cudaStream_t stream) {
  p.width = head_width(p.C);
  const int kb = (p.n_cols + HEAD_BK - 1) / HEAD_BK, kn = (p.N + HEAD_BK - 1) / HEAD_BK;
  p.all_slabs = p.slabs;
  p.slabs = p.slabs < kb ? p.slabs : kb;      // a last piece may be shorter than the slabs are many
  const int tc = (p.C + p.width - 1) / p.width, tm = (p.N + HEAD_TILE - 1) / HEAD_TILE;
  p.dx_items = p.dx ? p.slabs * tm * tc : 0;
  p.dw_items = p.dw ? (p.n_cols + HEAD_TILE - 1) / HEAD_TILE * tc : 0;
  const int k_dx = (kb + p.slabs - 1) / p.slabs;
  p.dw_first = kn > k_dx ? 1 : 0;
  const int items = p.dx_items + p.dw_items, pairs = items < sms / 2 ? items : sms / 2;
  p.shares = p.dw_first ? head_shares(p.dw_items, kn, p.dx_items, k_dx, pairs) : head_shares(p.dx_items, k_dx, p.dw_items, kn, pairs);
  CUtensorMap tg, tw, tx;
  int rc;
  if ((rc = encode_head_map(&tg, g, p.ldg, p.ldg, p.N, HEAD_BK, "head_loss_backward (gradient of the logits)")) != JB200_OK) return rc;
  if ((rc = encode_head_map(&tw, ws, p.C, head_pitch(p.C), p.n_cols, HEAD_BK, "head_loss_backward (weight)")) != JB200_OK) return rc;
  if ((rc = encode_head_map(&tx, xs, p.C, head_pitch(p.C), p.N, HEAD_BK, "head_loss_backward (rows)")) != JB200_OK) return rc;
  JB_MAX_SMEM(head_products_kernel, HEAD_SMEM);
  launch_dep_cluster(head_products_kernel, dim3(2 * unsigned(pairs)), dim3(HEAD_THREADS), HEAD_SMEM, 2, stream, tg, tw, tx, p);
  JB_LAUNCH_CHECK("head_products_kernel");
  if (p.dx && p.last && p.all_slabs > 1) {
    const size_t n = size_t(p.N) * p.C;
    launch_dep(p.dx_bf16 ? head_dx_kernel<true> : head_dx_kernel<false>, unsigned((n / 8 + 255) / 256), 256, 0, stream, p.dx_slabs, p.all_slabs, n,
               p.dx);
    JB_LAUNCH_CHECK("head_dx_kernel");
  }
  return JB200_OK;
}

}  // namespace jb

// Norms around a block, fused with the block's gate and with the residual stream:
//   gated_norm:     n = y / rms(y) * w [* silu(gate)]                           the rms over groups of columns (a head) or the whole row
//   residual_norm:  x' = x + scale * (y / rms(y) * w_after [* silu(gate)]),  xn = x' / rms(x') * w_before
// after jarvis_engine/jarvis_model.py:25-26 (RMSNorm) and :428-436 (the residual sums around it).  One pass over memory: rows stay in
// registers between the sums and the products; sums are f32, each result is rounded once.
//
// Bound by memory: 16384 rows of 1024 of residual_norm move 201 MB in 37 us, 5.4 TB/s.  The head norm of as many rows with a gate moves 100 MB in
// 18.5 us, next to its instructions (with exponentials and quotients that mind subnormals, and a division for every vector's row, 21.3); a second
// vector a thread, or one read ahead, took longer.  Few rows take the launch and one chain of two reads, two sums and a write.
#include "common.cuh"
#include "launchers.h"

namespace jb {

namespace {

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
  v[4] = bf16_lo(a.z); v[5] = bf16_hi(a.z); v[6] = bf16_lo(a.w); v[7] = bf16_hi(a.w);
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ float sumsq8(const float (&v)[8]) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
  return s;
}
// x / (1 + e^-x); e^-x beyond the range gives 0 as it should, and subnormal ones are 0 beside 1.  The flushing forms, since the others spend more on
// subnormals than on the rest, and instructions bound the head norm.
__device__ __forceinline__ float silu(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return x * r;
}

// Groups of 8 to 256 columns, a power of two: group / 8 neighbouring lanes hold one, wherever rows end.
template <typename TY, typename TO>
__global__ void __launch_bounds__(256) group_norm_kernel(const TY* __restrict__ y, size_t ldy, const float* __restrict__ w, const TY* __restrict__ gate,
                                                         size_t ldg, TO* __restrict__ out, int vectors_a_row, long long vectors, int group, float eps) {
  pdl_wait();
  pdl_trigger();
  const int lanes = group >> 3;
  const float share = 1.f / float(group);                               // exact
  const bool dense = ldy == size_t(vectors_a_row) * 8 && (gate == nullptr || ldg == ldy);   // then nothing asks for the row
  const long long padded = (vectors + 31) / 32 * 32;                    // whole warps: the sums go over lanes
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < padded; i += gridDim.x * 256ll) {
    const bool on = i < vectors;
    size_t at_y = size_t(i) * 8, at_g = at_y;
    const int col = int(at_y) & (group - 1);                            // rows are whole groups
    if (!dense) {
      const long long row = vectors <= 0xffffffffll ? uint32_t(i) / uint32_t(vectors_a_row) : i / vectors_a_row;
      const size_t in_row = at_y - size_t(row) * vectors_a_row * 8;
      at_y = row * ldy + in_row;
      at_g = row * ldg + in_row;
    }
    float v[8] = {}, g[8], ww[8];
    if (on) load8(y + at_y, v);
    if (on && gate != nullptr) load8(gate + at_g, g);
    float s = sumsq8(v);
    for (int o = 1; o < lanes; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (!on) continue;
    const float r = rsqrtf(fmaf(s, share, eps));
    load8(w + col, ww);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] * r * ww[j];
    if (gate != nullptr)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= silu(g[j]);
    store8(out + i * 8, v);
  }
}

struct RowNorm {
  const float* x;          // residual_norm; null: gated_norm of whole rows
  const void* y;
  size_t ldy;
  const float* w_after;
  const void* gate;
  size_t ldg;
  const float* scale;      // [C] or null (1)
  float* x_out;
  const float* w_before;
  void* out;               // xn, or n
  int n_rows, C;
  float eps;
};

// A CTA a row, V vectors of eight columns a thread.  128 threads up to 1024 columns: a warp a row, eight rows a CTA, reads four times as much at once
// but took 16384 rows of 1024 a third longer and 2048 half again as long.  Above 1024 columns most of a thread's four vectors are idle up to 2048
// (16384 rows of 1032, bf16, without a gate: 68 us, where 8192 of 2048 take 36 and 2048 of 8192 take 19).
template <typename TY, typename TO, int THREADS, int V>
__global__ void __launch_bounds__(THREADS) row_norm_kernel(RowNorm p) {
  __shared__ float part[2][THREADS / 32];
  const int t = threadIdx.x;
  const long long row = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  auto row_sum = [&](float s, float* slots) {
    s = warp_sum(s);
    if ((t & 31) == 0) slots[t >> 5] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) s += slots[i];
    return s;
  };
  const TY* y = static_cast<const TY*>(p.y) + row * p.ldy;
  const TY* gate = p.gate == nullptr ? nullptr : static_cast<const TY*>(p.gate) + row * p.ldg;
  TO* out = static_cast<TO*>(p.out) + row * p.C;
  float v[V][8], x[V][8];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * THREADS + t) * 8;
    if (c < p.C) {
      load8(y + c, v[i]);
      if (p.x != nullptr) load8(p.x + row * p.C + c, x[i]);
      s += sumsq8(v[i]);
    }
  }
  const float r = rsqrtf(row_sum(s, part[0]) / float(p.C) + p.eps);
  float s2 = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * THREADS + t) * 8;
    if (c < p.C) {
      float w[8];
      load8(p.w_after + c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = v[i][j] * r * w[j];
      if (gate != nullptr) {
        load8(gate + c, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] *= silu(w[j]);
      }
      if (p.x == nullptr) {
        store8(out + c, v[i]);
      } else {
        if (p.scale != nullptr) {
          load8(p.scale + c, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[i][j] = fmaf(w[j], v[i][j], x[i][j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[i][j] += v[i][j];
        }
        store8(p.x_out + row * p.C + c, x[i]);
        s2 += sumsq8(x[i]);
      }
    }
  }
  if (p.x == nullptr) return;
  const float r2 = rsqrtf(row_sum(s2, part[1]) / float(p.C) + p.eps);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = (i * THREADS + t) * 8;
    if (c < p.C) {
      float w[8];
      load8(p.w_before + c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = x[i][j] * r2 * w[j];
      store8(out + c, x[i]);
    }
  }
}

constexpr int MAX_C = 8192;

template <typename TY, typename TO>
void launch_rows(const RowNorm& p, cudaStream_t stream) {
  if (p.C > 1024) launch_dep(row_norm_kernel<TY, TO, 256, 4>, p.n_rows, 256, 0, stream, p);
  else launch_dep(row_norm_kernel<TY, TO, 128, 1>, p.n_rows, 128, 0, stream, p);
}

int check_norm(const char* what, const void* y, int y_dtype, long long ldy, const float* w, const void* gate, long long ldg, const void* out,
               int out_dtype, int n_rows, int C) {
  JB_REQUIRE(n_rows >= 0 && C >= 8 && C % 8 == 0 && C <= MAX_C, "%s: bad shape (rows=%d, C=%d): C must be a multiple of 8, at most %d", what, n_rows, C, MAX_C);
  JB_REQUIRE((y_dtype | 1) == 1 && (out_dtype | 1) == 1, "%s: dtypes must be 0 (f32) or 1 (bf16)", what);
  if (n_rows == 0) return JB200_OK;
  JB_REQUIRE(y && w && out, "%s: null pointer", what);
  JB_REQUIRE(ldy >= C && ldy % 8 == 0 && (gate == nullptr || (ldg >= C && ldg % 8 == 0)), "%s: row strides must be multiples of 8, at least C", what);
  JB_REQUIRE(aligned16(y) && aligned16(w) && aligned16(gate) && aligned16(out), "%s: tensors must be 16-byte aligned", what);
  return JB200_OK;
}

template <typename F>
void by_types(int y_dtype, int out_dtype, F&& f) {
  if (y_dtype == 0) {
    if (out_dtype == 0) f(float{}, float{});
    else f(float{}, __nv_bfloat16{});
  } else {
    if (out_dtype == 0) f(__nv_bfloat16{}, float{});
    else f(__nv_bfloat16{}, __nv_bfloat16{});
  }
}

}  // namespace

int launch_gated_norm(const void* y, int y_dtype, long long ldy, const float* w, const void* gate, long long ldg, int group, float eps, void* out,
                      int out_dtype, int n_rows, int C, cudaStream_t stream) {
  const int rc = check_norm("gated_norm", y, y_dtype, ldy, w, gate, ldg, out, out_dtype, n_rows, C);
  if (rc != JB200_OK) return rc;
  JB_REQUIRE(group == C || (group >= 8 && group <= 256 && (group & (group - 1)) == 0 && C % group == 0),
             "gated_norm: a group (%d) is the whole row (%d), or a power of two from 8 to 256 that divides it", group, C);
  if (n_rows == 0) return JB200_OK;
  if (group <= 256 && (group & (group - 1)) == 0) {
    const long long vectors = (long long)n_rows * (C / 8), blocks = (vectors + 255) / 256;
    by_types(y_dtype, out_dtype, [&](auto ty, auto to) {
      using TY = decltype(ty);
      using TO = decltype(to);
      launch_dep(group_norm_kernel<TY, TO>, unsigned(blocks < 8ll * sm_count() ? blocks : 8ll * sm_count()), 256, 0, stream, static_cast<const TY*>(y),
                 size_t(ldy), w, static_cast<const TY*>(gate), size_t(ldg), static_cast<TO*>(out), C / 8, vectors, group, eps);
    });
    JB_LAUNCH_CHECK("group_norm_kernel");
    return JB200_OK;
  }
  const RowNorm p = {nullptr, y, size_t(ldy), w, gate, size_t(ldg), nullptr, nullptr, nullptr, out, n_rows, C, eps};
  by_types(y_dtype, out_dtype, [&](auto ty, auto to) { launch_rows<decltype(ty), decltype(to)>(p, stream); });
  JB_LAUNCH_CHECK("row_norm_kernel");
  return JB200_OK;
}

int launch_residual_norm(const float* x, const void* y, int y_dtype, long long ldy, const float* w_after, const void* gate, long long ldg,
                         const float* scale, const float* w_before, float eps, float* x_out, void* xn, int xn_dtype, int n_rows, int C,
                         cudaStream_t stream) {
  const int rc = check_norm("residual_norm", y, y_dtype, ldy, w_after, gate, ldg, xn, xn_dtype, n_rows, C);
  if (rc != JB200_OK || n_rows == 0) return rc;
  JB_REQUIRE(x && x_out && w_before, "residual_norm: null pointer");
  JB_REQUIRE(aligned16(x) && aligned16(x_out) && aligned16(w_before) && aligned16(scale), "residual_norm: tensors must be 16-byte aligned");
  const RowNorm p = {x, y, size_t(ldy), w_after, gate, size_t(ldg), scale, x_out, w_before, xn, n_rows, C, eps};
  by_types(y_dtype, xn_dtype, [&](auto ty, auto to) { launch_rows<decltype(ty), decltype(to)>(p, stream); });
  JB_LAUNCH_CHECK("row_norm_kernel");
  return JB200_OK;
}

}  // namespace jb

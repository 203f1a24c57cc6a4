// Gradient of the RMS norm (jarvis_engine/jarvis_model.py:25-26), y = x r w with r = rsqrt(mean(x^2) + eps):
//
//   dx = r (w dy) - x (r^3 / C) sum(w dy x),      dw = sum over rows of dy x r
//
// Nothing of the forward is needed but x: both sums of a row come from the values that its dx needs anyway.  Bound by HBM: x and dy
// are read once, dx written once.  A row belongs to as many warps as it has thousands of channels; a lane keeps its channels' sums
// of dw in registers over all rows it sees, the CTAs' sums are added in a fixed order: by a second launch, or, of few rows, by a
// cluster that has them all.  16384 x 1024 f32 rows: 168 MB in 37 us (0.70 of the copy bandwidth), and 9 us for the second launch.  What
// it lacks: a warp asks for a row only after it has reduced and stored the one before.
#include "common.cuh"
#include "launchers.h"

namespace jb {

namespace {

constexpr int NG_WARPS = 8, NG_VEC = 4;               // warps of a CTA; groups of 8 channels a lane keeps
constexpr int NG_SPAN = 32 * 8 * NG_VEC;              // channels of a warp: 1024

__device__ __forceinline__ void ng_load8(const float* p, float (&v)[8]) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void ng_load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
  v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
  v[4] = bf16_lo(a.z); v[5] = bf16_hi(a.z); v[6] = bf16_lo(a.w); v[7] = bf16_hi(a.w);
}
__device__ __forceinline__ void ng_store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void ng_store8(__nv_bfloat16* p, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

__device__ __forceinline__ float cluster_ld(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// WPR: warps of a row (1, 2 or 4).  ONE: the grid is one cluster and leaves dw itself in dw_part.  dx: null where not wanted.
template <typename TX, typename TY, int WPR, bool ONE>
__global__ void __launch_bounds__(32 * NG_WARPS, 2)
rmsnorm_backward_kernel(const TX* __restrict__ x, const float* __restrict__ w, float eps, const TY* __restrict__ dy, int n_rows, int C,
                        TX* __restrict__ dx, float* __restrict__ dw_part) {
  pdl_wait();
  pdl_trigger();
  constexpr int ROWS = NG_WARPS / WPR;                // rows of a CTA at a time
  __shared__ float s_dw[NG_WARPS][NG_SPAN];
  __shared__ float2 s_row[2][NG_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WPR, c0 = part * NG_SPAN + lane * 8;
  float acc[NG_VEC][8];
#pragma unroll
  for (int i = 0; i < NG_VEC; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
  const float inv_c = 1.0f / float(C);
  int turn = 0;
  for (int first = blockIdx.x * ROWS; first < n_rows; first += gridDim.x * ROWS, turn ^= 1) {
    const int row = first + warp / WPR;
    const bool on = row < n_rows;
    float xv[NG_VEC][8], g[NG_VEC][8];
    float ss = 0.f, along = 0.f;
    if (on) {
      const TX* xr = x + size_t(row) * C;
      const TY* gr = dy + size_t(row) * C;
#pragma unroll
      for (int i = 0; i < NG_VEC; ++i)
        if (c0 + i * 256 < C) {
          ng_load8(xr + c0 + i * 256, xv[i]);
          ng_load8(gr + c0 + i * 256, g[i]);
        }
#pragma unroll
      for (int i = 0; i < NG_VEC; ++i)
        if (c0 + i * 256 < C) {
          const float4 wa = __ldg(reinterpret_cast<const float4*>(w + c0 + i * 256)), wb = __ldg(reinterpret_cast<const float4*>(w + c0 + i * 256) + 1);
          const float wv[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ss = fmaf(xv[i][j], xv[i][j], ss);
            along = fmaf(wv[j] * g[i][j], xv[i][j], along);
          }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      along += __shfl_xor_sync(0xffffffffu, along, o);
    }
    if constexpr (WPR > 1) {                          // two buffers: a warp may be a turn ahead of the readers, never two
      if (lane == 0) s_row[turn][warp] = make_float2(ss, along);
      __syncthreads();
      ss = along = 0.f;
#pragma unroll
      for (int i = 0; i < WPR; ++i) {
        const float2 s = s_row[turn][warp - part + i];
        ss += s.x;
        along += s.y;
      }
    }
    if (on) {
      const float r = rsqrtf(ss * inv_c + eps), k = along * inv_c * r * r;      // dx = r (w dy - x k)
      TX* dr = dx ? dx + size_t(row) * C : nullptr;
#pragma unroll
      for (int i = 0; i < NG_VEC; ++i)
        if (c0 + i * 256 < C) {
          const float4 wa = __ldg(reinterpret_cast<const float4*>(w + c0 + i * 256)), wb = __ldg(reinterpret_cast<const float4*>(w + c0 + i * 256) + 1);
          const float wv[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
          float o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[i][j] = fmaf(g[i][j], xv[i][j] * r, acc[i][j]);
            o[j] = r * fmaf(-xv[i][j], k, wv[j] * g[i][j]);
          }
          if (dr) ng_store8(dr + c0 + i * 256, o);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < NG_VEC; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) s_dw[warp][i * 256 + j * 32 + lane] = acc[i][j];
  __syncthreads();
  // channel c of the row is kept by its part's warps at (c / 256, c % 8, c / 8 % 32)
  for (int c = threadIdx.x; c < C; c += 32 * NG_WARPS) {
    const int pt = c / NG_SPAN, in = c % NG_SPAN, at = (in & ~255) + (in & 7) * 32 + (in >> 3 & 31);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) sum += s_dw[i * WPR + pt][at];
    if constexpr (ONE) s_dw[pt][at] = sum;
    else dw_part[size_t(blockIdx.x) * C + c] = sum;
  }
  if constexpr (ONE) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    for (int c = int(blockIdx.x) * 32 * NG_WARPS + threadIdx.x; c < C; c += int(gridDim.x) * 32 * NG_WARPS) {
      const int pt = c / NG_SPAN, in = c % NG_SPAN, at = (in & ~255) + (in & 7) * 32 + (in >> 3 & 31);
      const uint32_t addr = smem_u32(&s_dw[pt][at]);
      float sum = 0.f;
      for (int r = 0; r < int(gridDim.x); ++r) sum += cluster_ld(cluster_map(addr, uint32_t(r)));
      dw_part[c] = sum;
    }
    __syncwarp();
    cluster_arrive();               // none leaves while another reads its sums
    cluster_wait();
  }
}

// dw[c] = sum of the CTAs' parts in a fixed order: a warp every 32nd of them, then the warps.
__global__ void __launch_bounds__(1024) rmsnorm_dw_kernel(const float* __restrict__ part, int n_parts, int C, float* __restrict__ dw) {
  pdl_wait();
  pdl_trigger();
  __shared__ float s[32][33];
  const int g = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < C) {
#pragma unroll 10
    for (int i = g; i < n_parts; i += 32) sum += part[size_t(i) * C + c];
  }
  s[g][lane] = sum;
  __syncthreads();
  sum = warp_sum(s[lane][g]);
  if (lane == 0 && blockIdx.x * 32 + g < C) dw[blockIdx.x * 32 + g] = sum;
}

int norm_warps(int C) { return C <= NG_SPAN ? 1 : C <= 2 * NG_SPAN ? 2 : 4; }
int norm_ctas(int n_rows, int C, int sms) {
  const long long rows = NG_WARPS / norm_warps(C), n = (n_rows + rows - 1) / rows;
  return int(n < 2 * sms ? n : 2 * sms);
}
// CTAs of the one cluster that takes all rows, 0 where there are too many.  A turn of its warps takes 3 us: 128 rows of 1024 channels 11.7 us,
// 256 rows 15 us, where two launches take 11 us of the device but 5 us more of the host, which few rows wait for.
constexpr int NG_ONE_TURNS = 4;                       // rows that a warp of it takes one after the other
int norm_cluster(int n_rows, int C) {
  const int rows = NG_WARPS / norm_warps(C);
  if (n_rows > 8 * rows * NG_ONE_TURNS) return 0;
  int n = 1;
  while (n < 8 && n * rows < n_rows) n *= 2;
  return n;
}

template <typename TX, typename TY, bool ONE>
auto norm_kernel(int wpr) {
  return wpr == 1 ? rmsnorm_backward_kernel<TX, TY, 1, ONE> : wpr == 2 ? rmsnorm_backward_kernel<TX, TY, 2, ONE> : rmsnorm_backward_kernel<TX, TY, 4, ONE>;
}
template <typename TX, typename TY>
int launch_rmsnorm_backward_t(const void* x, const float* w, float eps, const void* dy, int n_rows, int C, void* dx, float* dw, float* part, int sms,
                              cudaStream_t stream) {
  const int wpr = norm_warps(C), cluster = norm_cluster(n_rows, C);
  if (cluster) {
    launch_dep_cluster(norm_kernel<TX, TY, true>(wpr), cluster, 32 * NG_WARPS, 0, cluster, stream, static_cast<const TX*>(x), w, eps,
                       static_cast<const TY*>(dy), n_rows, C, static_cast<TX*>(dx), dw);
    JB_LAUNCH_CHECK("rmsnorm_backward_kernel");
    return JB200_OK;
  }
  const int ctas = norm_ctas(n_rows, C, sms);
  launch_dep(norm_kernel<TX, TY, false>(wpr), ctas, 32 * NG_WARPS, 0, stream, static_cast<const TX*>(x), w, eps, static_cast<const TY*>(dy), n_rows, C,
             static_cast<TX*>(dx), part);
  JB_LAUNCH_CHECK("rmsnorm_backward_kernel");
  launch_dep(rmsnorm_dw_kernel, (C + 31) / 32, 1024, 0, stream, part, ctas, C, dw);
  JB_LAUNCH_CHECK("rmsnorm_dw_kernel");
  return JB200_OK;
}

}  // namespace

size_t rmsnorm_backward_scratch_bytes(int n_rows, int C) {
  const int sms = sm_count();
  if (n_rows < 1 || C < 1 || C > 4 * NG_SPAN || sms < 1 || norm_cluster(n_rows, C)) return 0;
  return size_t(norm_ctas(n_rows, C, sms)) * C * 4;
}

int launch_rmsnorm_backward(const void* x, int x_dtype, const float* w, float eps, const void* dy, int dy_dtype, int n_rows, int C, void* dx,
                            float* dw, void* scratch, cudaStream_t stream) {
  JB_REQUIRE(n_rows >= 0 && C > 0, "rmsnorm_backward: bad shape (%d, %d)", n_rows, C);
  JB_REQUIRE(C % 8 == 0 && C <= 4 * NG_SPAN, "rmsnorm_backward: row length (%d) must be a multiple of 8 and at most %d", C, 4 * NG_SPAN);
  JB_REQUIRE((x_dtype == 0 || x_dtype == 1) && (dy_dtype == 0 || dy_dtype == 1), "rmsnorm_backward: dtype must be 0 (f32) or 1 (bf16)");
  JB_REQUIRE(dw, "rmsnorm_backward: null pointer");
  if (n_rows == 0) {
    JB_CUDA(cudaMemsetAsync(dw, 0, size_t(C) * 4, stream));
    return JB200_OK;
  }
  JB_REQUIRE(x && w && dy && (scratch || norm_cluster(n_rows, C)), "rmsnorm_backward: null pointer");
  JB_REQUIRE(aligned16(x) && aligned16(w) && aligned16(dy) && aligned16(dx), "rmsnorm_backward: pointers must be 16-byte aligned");
  const int sms = sm_count();
  if (sms < 1) return JB200_ERR_CUDA;
  float* part = static_cast<float*>(scratch);
  typedef __nv_bfloat16 b16;
  if (x_dtype == 0 && dy_dtype == 0) return launch_rmsnorm_backward_t<float, float>(x, w, eps, dy, n_rows, C, dx, dw, part, sms, stream);
  if (x_dtype == 0) return launch_rmsnorm_backward_t<float, b16>(x, w, eps, dy, n_rows, C, dx, dw, part, sms, stream);
  if (dy_dtype == 0) return launch_rmsnorm_backward_t<b16, float>(x, w, eps, dy, n_rows, C, dx, dw, part, sms, stream);
  return launch_rmsnorm_backward_t<b16, b16>(x, w, eps, dy, n_rows, C, dx, dw, part, sms, stream);
}

}  // namespace jb

// The gated delta rule, the decayed associative scan (attn_scan.cu) with a write that first takes out what the key holds:
//   S_t = a_t S_{t-1} (I - b_t k_t k_t^T) + b_t v_t k_t^T        o_t = scale S_t q_t
// with the layout of the other scan: q, k, v as rows of a fused projection, S f32 [B][H][64 values][64 keys].  a_t = exp(log_decay), k and q
// divided by sqrt(|.|^2 + 1e-6) when asked (JB200_DELTA_NORMALIZE).  Rows of S are independent of one another: value row i sees v_t[i] alone.
#include "common.cuh"
#include "launchers.h"

namespace jb {

namespace {

constexpr int D = 64;
constexpr float NORM_EPS = 1e-6f;

struct DeltaParams {
  const __nv_bfloat16 *q, *k, *v;
  size_t ldq, ldk, ldv, ldo, ldg;           // elements
  const float *log_decay, *beta;            // [B T][ldg]
  const int32_t* lengths;                   // [B] or null
  const float* s_in;                        // [B][H][64][64] or null
  float* s_out;                             // or null
  __nv_bfloat16* o;
  int B, T, H, per_key;                     // per_key: value heads that share a key head
  float scale;
  int normalize;
};

__device__ __forceinline__ int sequence_length(const DeltaParams& p, int b) {
  return p.lengths == nullptr ? p.T : min(max(__ldg(p.lengths + b), 0), p.T);
}

// ---------------------------------------------------------------------------------------------------------------------
// Token by token.  Eight lanes hold a row of S (lane l: keys 4l..4l+3 and 32 + 4l..), ROWS rows a lane, so that a CTA of 128 threads has
// 16 ROWS rows and a head 4 / ROWS CTAs.  Both products of a token are taken of the state before it,
//   S_t q = a (S q) + u (k.q)   with   u = b (v - a S k),
// so that their sums over the eight lanes run together.  Bound by the state's traffic: 32 KB a head, read and written once.
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float sum8(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  v += __shfl_xor_sync(0xffffffffu, v, 2);
  return v + __shfl_xor_sync(0xffffffffu, v, 4);
}

struct Token {
  uint2 k0, k1, q0, q1;
  float g, beta;
};

__device__ __forceinline__ void unpack8(uint2 a, uint2 b, float (&x)[8]) {
  x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x); x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
  x[4] = bf16_lo(b.x); x[5] = bf16_hi(b.x); x[6] = bf16_lo(b.y); x[7] = bf16_hi(b.y);
}

template <int ROWS>
__global__ void __launch_bounds__(128) delta_step_kernel(DeltaParams p) {
  constexpr int SPLIT = 4 / ROWS;
  const int bh = blockIdx.x / SPLIT, part = blockIdx.x % SPLIT;
  const int b = bh / p.H, h = bh % p.H, l = threadIdx.x & 7, row0 = part * 16 * ROWS + (threadIdx.x >> 3);
  pdl_wait();
  pdl_trigger();
  const int len = sequence_length(p, b);
  float s[ROWS][8];
  const size_t at = size_t(bh) * D * D + size_t(row0) * D + 4 * l;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    if (p.s_in != nullptr) {
      x = __ldcs(reinterpret_cast<const float4*>(p.s_in + at + size_t(r) * 16 * D));
      y = __ldcs(reinterpret_cast<const float4*>(p.s_in + at + size_t(r) * 16 * D + 32));
    }
    s[r][0] = x.x; s[r][1] = x.y; s[r][2] = x.z; s[r][3] = x.w;
    s[r][4] = y.x; s[r][5] = y.y; s[r][6] = y.z; s[r][7] = y.w;
  }
  const size_t first = size_t(b) * p.T;
  const __nv_bfloat16* kp = p.k + first * p.ldk + size_t(h / p.per_key) * D + 4 * l;
  const __nv_bfloat16* qp = p.q + first * p.ldq + size_t(h / p.per_key) * D + 4 * l;
  const __nv_bfloat16* vp = p.v + first * p.ldv + size_t(h) * D + row0;
  const float* gp = p.log_decay + first * p.ldg + h;
  const float* bp = p.beta + first * p.ldg + h;
  Token next;
  float v_next[ROWS];
  auto fetch = [&](int t) {
    next.k0 = *reinterpret_cast<const uint2*>(kp + size_t(t) * p.ldk);
    next.k1 = *reinterpret_cast<const uint2*>(kp + size_t(t) * p.ldk + 32);
    next.q0 = *reinterpret_cast<const uint2*>(qp + size_t(t) * p.ldq);
    next.q1 = *reinterpret_cast<const uint2*>(qp + size_t(t) * p.ldq + 32);
    next.g = gp[size_t(t) * p.ldg];
    next.beta = bp[size_t(t) * p.ldg];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) v_next[r] = __bfloat162float(vp[size_t(t) * p.ldv + 16 * r]);
  };
  if (len > 0) fetch(0);
  for (int t = 0; t < len; ++t) {
    const Token now = next;
    float v[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) v[r] = v_next[r];
    if (t + 1 < len) fetch(t + 1);
    float k[8], q[8];
    unpack8(now.k0, now.k1, k);
    unpack8(now.q0, now.q1, q);
    float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) { kk = fmaf(k[j], k[j], kk); qq = fmaf(q[j], q[j], qq); kq = fmaf(k[j], q[j], kq); }
    kk = sum8(kk);
    qq = sum8(qq);
    kq = sum8(kq);
    const float rk = p.normalize ? rsqrtf(kk + NORM_EPS) : 1.f, rq = (p.normalize ? rsqrtf(qq + NORM_EPS) : 1.f) * p.scale;
    const float a = expf(now.g);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float sk = 0.f, sq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) { sk = fmaf(s[r][j], k[j], sk); sq = fmaf(s[r][j], q[j], sq); }
      sk = sum8(sk);
      sq = sum8(sq);
      const float u = now.beta * fmaf(-a * rk, sk, v[r]) * rk;          // what is written along the unscaled key
#pragma unroll
      for (int j = 0; j < 8; ++j) s[r][j] = fmaf(u, k[j], a * s[r][j]);
      if (l == 0 && p.o != nullptr)
        p.o[(first + t) * p.ldo + size_t(h) * D + row0 + 16 * r] = __float2bfloat16(rq * fmaf(u, kq, a * sq));
    }
  }
  if (p.o != nullptr && l == 0)
    for (int t = len; t < p.T; ++t)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) p.o[(first + t) * p.ldo + size_t(h) * D + row0 + 16 * r] = __float2bfloat16(0.f);
  if (p.s_out != nullptr) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      __stcs(reinterpret_cast<float4*>(p.s_out + at + size_t(r) * 16 * D), make_float4(s[r][0], s[r][1], s[r][2], s[r][3]));
      __stcs(reinterpret_cast<float4*>(p.s_out + at + size_t(r) * 16 * D + 32), make_float4(s[r][4], s[r][5], s[r][6], s[r][7]));
    }
  }
}

}  // namespace

size_t gated_delta_scratch_bytes(int B, int T, int H) { return 0; }

int launch_gated_delta(const jb200_delta* d, void* scratch, cudaStream_t stream) {
  JB_REQUIRE(d != nullptr, "gated_delta: null pointer");
  const int B = d->B, T = d->T, H = d->H, KH = d->key_heads;
  JB_REQUIRE(B >= 0 && T >= 0 && H >= 1 && KH >= 1 && H % KH == 0, "gated_delta: bad shape (B=%d, T=%d, H=%d, key heads=%d)", B, T, H, KH);
  JB_REQUIRE(d->head_dim == D, "gated_delta: head_dim must be 64 (got %d)", d->head_dim);
  JB_REQUIRE((long long)B * H <= 0x1fffffff && (long long)B * T <= 0x7fffffff, "gated_delta: too many heads or tokens");
  if (B == 0) return JB200_OK;
  JB_REQUIRE(d->o != nullptr || d->s_out != nullptr, "gated_delta: neither an output nor a final state is asked for");
  JB_REQUIRE(T == 0 || (d->q && d->k && d->v && d->log_decay && d->beta), "gated_delta: null pointer");
  JB_REQUIRE(d->ldq >= KH * D && d->ldk >= KH * D && d->ldv >= H * D && d->ldg >= H && (d->o == nullptr || d->ldo >= H * D),
             "gated_delta: row strides are smaller than the rows");
  JB_REQUIRE(aligned16(d->q) && aligned16(d->k) && aligned16(d->v) && aligned16(d->o) && aligned16(d->s_in) && aligned16(d->s_out) &&
                 d->ldq % 8 == 0 && d->ldk % 8 == 0 && d->ldv % 8 == 0 && (d->o == nullptr || d->ldo % 8 == 0),
             "gated_delta: q, k, v, o and the states must be 16-byte aligned, their row strides multiples of 8");
  DeltaParams p;
  p.q = static_cast<const __nv_bfloat16*>(d->q);
  p.k = static_cast<const __nv_bfloat16*>(d->k);
  p.v = static_cast<const __nv_bfloat16*>(d->v);
  p.ldq = d->ldq; p.ldk = d->ldk; p.ldv = d->ldv; p.ldo = d->ldo; p.ldg = d->ldg;
  p.log_decay = d->log_decay; p.beta = d->beta; p.lengths = d->lengths; p.s_in = d->s_in; p.s_out = d->s_out;
  p.o = static_cast<__nv_bfloat16*>(d->o);
  p.B = B; p.T = T; p.H = H; p.per_key = H / KH;
  p.scale = d->scale; p.normalize = d->flags & JB200_DELTA_NORMALIZE;
  if (B * H < 2 * sm_count())
    launch_dep(delta_step_kernel<1>, B * H * 4, 128, 0, stream, p);
  else
    launch_dep(delta_step_kernel<4>, B * H, 128, 0, stream, p);
  JB_LAUNCH_CHECK("delta_step_kernel");
  return JB200_OK;
}

}  // namespace jb

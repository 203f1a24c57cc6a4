// The gated delta rule, the decayed associative scan (attn_scan.cu) with a write that first takes out what the key holds:
//   S_t = a_t S_{t-1} (I - b_t k_t k_t^T) + b_t v_t k_t^T        o_t = scale S_t q_t
// with the layout of the other scan: q, k, v as rows of a fused projection, S f32 [B][H][64 values][64 keys].  a_t = exp(log_decay), k and q
// divided by sqrt(|.|^2 + 1e-6) when asked (JB200_DELTA_NORMALIZE).  Rows of S are independent of one another: value row i sees v_t[i] alone.
#include <cuda_fp16.h>

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

// ---------------------------------------------------------------------------------------------------------------------
// Chunks of 64 tokens on the tensor cores.  With G the running sum of log a from the chunk's first token and S the state before it, the writes
// u of a chunk solve a triangular system, and everything else is products of 64 x 64 matrices:
//   X = b (V - e^G K S^T),   U = T X with T = (I + A)^-1,  A_ij = b_i e^(G_i - G_j) k_i.k_j  (j < i)
//   O = e^G Q S^T + P U with P_ij = e^(G_i - G_j) q_i.k_j  (j <= i),   S' = e^Gc S + (e^(Gc - G) U)^T K
// A CTA follows one head of one sequence.  Four warps prepare a chunk (K, Q, T, P: nothing of the state) while the other four take the chunk
// before it through the state; each of those holds 16 value rows of S in its accumulators and everything transposed (X^T, U^T, O^T: 16 values x
// 64 tokens), so that a product's accumulators are the next one's first operand where they are, and the four never wait for one another.
//
// mma.sync, not tcgen05: a chunk is a chain of five dependent products of 16 x 64 x 64 a warp with a rescaling between them; through tensor
// memory each link would cost a commit, a wait and two copies, several times the product itself.
//
// Precision: the state is f32 and stays it.  What is multiplied is f16 in two terms, x = hi + lo (22 bits), with an exact power of two per row that
// puts the row's largest value near the top of f16's range: 2^-24 of the row's maximum each.  K and Q come as bf16 and fit one term, scaled by
// a power of two per row; their norms are factors on rows and columns.  X T^T takes hi hi + hi lo + lo hi.  What only the output sees
// (Q S^T, P U) is one term, 2^-12 of a value where the output's own rounding is 2^-9.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int CHUNK = 64;
constexpr int TILE = CHUNK * D * 2;        // bytes of 64 rows of 128, the 16-byte units of row r at unit ^ (r & 7)
constexpr float LEAST_LOG2 = -300.f;       // 2^-300 is 0 in f32: a decay of less, -inf among them, is this one

struct alignas(128) Stage {
  uint8_t k[TILE], q[TILE], v[TILE];
  uint8_t t_hi[TILE], t_lo[TILE];          // T^T [j][i] on and above the diagonal's 16 x 16 blocks; -A [i][j] below them while T is formed
  uint8_t p[TILE];                         // P [i][j]; before that, the diagonal blocks of -A in f32
  float of_v[CHUNK], of_y[CHUNK], of_u[CHUNK], grow[CHUNK], of_o[CHUNK];
  float whole;
};
struct alignas(128) ChunkSmem {
  Stage stage[2];
  float g_hi[CHUNK], g_lo[CHUNK], beta[CHUNK], rk[CHUNK], nk[CHUNK], rq[CHUNK];
};
static_assert(sizeof(Stage) % 128 == 0 && TILE % 128 == 0, "tiles are read 16 bytes at a time in both stages");

__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
// barriers of the CTA: 1 the four preparing warps, 2 the two that form T, 3 + s stage s is ready, 5 + s stage s is free
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void stm4t(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// (x, y) as two f16 terms each
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16x2(x, y);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_f16x2(x - f.x, y - f.y);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// A power of two s with s m in [2^TO, 2^(TO + 1)) and its inverse; of m = 0, infinities and what is too small any that are finite
template <int TO>
__device__ __forceinline__ void power_scale(float m, float& s, float& inv) {
  const int e = max(int(__float_as_uint(m) >> 23), TO + 3);
  s = __uint_as_float(uint32_t(254 + TO - e) << 23);
  inv = __uint_as_float(uint32_t(e - TO) << 23);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ uint32_t unit_at(int row, int unit) { return uint32_t(row * 128 + ((unit ^ (row & 7)) << 4)); }

// Lane's address part for four 8 x 8 matrices of a tile.  ACROSS: matrices 0, 1 are neighbouring units (columns), 2, 3 those of the next eight
// rows; DOWN: 0, 1 are rows r, r + 8 of one unit, 2, 3 those of the next unit.
__device__ __forceinline__ uint32_t across(int row, int unit, int lane) { return unit_at(row + ((lane >> 4) << 3) + (lane & 7), unit + ((lane >> 3) & 1)); }
__device__ __forceinline__ uint32_t down(int row, int unit, int lane) { return unit_at(row + (((lane >> 3) & 1) << 3) + (lane & 7), unit + (lane >> 4)); }

// ---- the preparing warps ---------------------------------------------------------------------------------------------
struct Loads {
  uint4 k[4], q[4];
  float g[2], beta[2];
};

template <bool OUT>
struct Prepare {
  const DeltaParams& p;
  ChunkSmem& sm;
  int b, h, w, lane, len;

  __device__ __forceinline__ void fetch(Loads& x, int t0) const {
    const size_t first = size_t(b) * p.T + t0;
    const int sub = lane >> 3, unit = lane & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * w + 4 * i + sub;
      const bool on = t0 + row < len;
      x.k[i] = x.q[i] = make_uint4(0, 0, 0, 0);
      if (on) x.k[i] = __ldg(reinterpret_cast<const uint4*>(p.k + (first + row) * p.ldk + size_t(h / p.per_key) * D) + unit);
      if (OUT && on) x.q[i] = __ldg(reinterpret_cast<const uint4*>(p.q + (first + row) * p.ldq + size_t(h / p.per_key) * D) + unit);
    }
    if (w == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 2 * lane + i;
        const bool on = t0 + row < len;
        x.g[i] = on ? __ldg(p.log_decay + (first + row) * p.ldg + h) : 0.f;
        x.beta[i] = on ? __ldg(p.beta + (first + row) * p.ldg + h) : 0.f;
      }
    }
  }

  // one row of bf16 by eight lanes -> f16 times a power of two (the largest value in [1, 2)), the sum of squares of that, the power
  __device__ __forceinline__ uint4 to_f16(uint4 x, float& ss, float& s) const {
    const uint32_t m4 = 0x7fff7fffu;
    const uint32_t m2 = __vmaxu2(__vmaxu2(x.x & m4, x.y & m4), __vmaxu2(x.z & m4, x.w & m4));
    uint32_t m = max(m2 >> 16, m2 & 0xffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
    s = __uint_as_float(uint32_t(max(254 - int(m >> 7), 1)) << 23);
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
    uint32_t out[4];
    ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = bf16_lo(in[j]) * s, c = bf16_hi(in[j]) * s;
      ss = fmaf(a, a, fmaf(c, c, ss));
      out[j] = pack_f16x2(a, c);
    }
    ss = sum8(ss);
    return make_uint4(out[0], out[1], out[2], out[3]);
  }

  __device__ __forceinline__ void convert(const Loads& x, Stage& st) const {
    const int sub = lane >> 3, unit = lane & 7;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * w + 4 * i + sub;
      float ss, s;
      *reinterpret_cast<uint4*>(st.k + unit_at(row, unit)) = to_f16(x.k[i], ss, s);
      if (unit == 0) {
        // k = n (k16 r) with |k16 r| = 1, or of the normalised key n = 1 and k16 r its value
        const float r = p.normalize ? rsqrtf(fmaf(NORM_EPS * s, s, ss)) : ss > 0.f ? rsqrtf(ss) : 0.f;
        sm.rk[row] = r;
        sm.nk[row] = p.normalize ? 1.f : ss * r / s;
      }
      if (OUT) {
        *reinterpret_cast<uint4*>(st.q + unit_at(row, unit)) = to_f16(x.q[i], ss, s);
        if (unit == 0) sm.rq[row] = p.scale * (p.normalize ? rsqrtf(fmaf(NORM_EPS * s, s, ss)) : 1.f / s);
      }
    }
    if (w == 0) {                              // running sums of log2 a, in f64 for differences of late tokens
      double g0 = double(x.g[0]) * 1.4426950408889634, g1 = double(x.g[1]) * 1.4426950408889634;
      if (g0 < double(LEAST_LOG2)) g0 = double(LEAST_LOG2);
      if (g1 < double(LEAST_LOG2)) g1 = double(LEAST_LOG2);
      double sum = g0 + g1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const double at0 = sum - g1, end = __shfl_sync(0xffffffffu, sum, 31);
      const double at[2] = {at0, sum};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 2 * lane + i;
        const float hi = float(at[i]);
        sm.g_hi[row] = hi;
        sm.g_lo[row] = float(at[i] - double(hi));
        sm.beta[row] = x.beta[i];
        st.grow[row] = exp2f(hi);
        st.of_u[row] = exp2f(float(end - at[i]));
      }
      if (lane == 0) st.whole = exp2f(float(end));
    }
  }

  // 16 rows ib of `a` times 16 rows jb of K, 64 long
  __device__ __forceinline__ void products(float (&c)[2][4], const uint32_t (&a)[4][4], const Stage& st, int jb) const {
    const uint32_t kb = smem_u32(st.k);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[0][i] = c[1][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t f[4];
      ldm4(f, kb + across(16 * jb, 2 * ks, lane));
      mma(c[0], a[ks], f[0], f[1]);
      mma(c[1], a[ks], f[2], f[3]);
    }
  }

  __device__ __forceinline__ void row_of_a(Stage& st) const {
    uint32_t a[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) ldm4(a[ks], smem_u32(st.k) + down(16 * w, 2 * ks, lane));
    const int i0 = 16 * w + (lane >> 2), i1 = i0 + 8;
    const float gh0 = sm.g_hi[i0], gl0 = sm.g_lo[i0], gh1 = sm.g_hi[i1], gl1 = sm.g_lo[i1];
    const float n0 = sm.nk[i0], n1 = sm.nk[i1];
    const float f0 = -sm.beta[i0] * n0 * n0 * sm.rk[i0], f1 = -sm.beta[i1] * n1 * n1 * sm.rk[i1];
    float* dg = reinterpret_cast<float*>(st.p) + w * 16 * 20;
    for (int jb = 0; jb <= w; ++jb) {
      float c[2][4];
      products(c, a, st, jb);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int j = 16 * jb + 8 * n + 2 * (lane & 3);
        const float2 gh = *reinterpret_cast<const float2*>(sm.g_hi + j), gl = *reinterpret_cast<const float2*>(sm.g_lo + j);
        const float2 r = *reinterpret_cast<const float2*>(sm.rk + j);
        const float x0 = f0 * r.x * c[n][0] * exp2_fast((gh0 - gh.x) + (gl0 - gl.x)), x1 = f0 * r.y * c[n][1] * exp2_fast((gh0 - gh.y) + (gl0 - gl.y));
        const float x2 = f1 * r.x * c[n][2] * exp2_fast((gh1 - gh.x) + (gl1 - gl.x)), x3 = f1 * r.y * c[n][3] * exp2_fast((gh1 - gh.y) + (gl1 - gl.y));
        if (jb < w) {
          const uint32_t at0 = unit_at(i0, j >> 3) + (j & 7) * 2, at1 = unit_at(i1, j >> 3) + (j & 7) * 2;
          uint32_t hi, lo;
          split(x0, x1, hi, lo);
          *reinterpret_cast<uint32_t*>(st.t_hi + at0) = hi;
          *reinterpret_cast<uint32_t*>(st.t_lo + at0) = lo;
          split(x2, x3, hi, lo);
          *reinterpret_cast<uint32_t*>(st.t_hi + at1) = hi;
          *reinterpret_cast<uint32_t*>(st.t_lo + at1) = lo;
        } else {
          const int jl = 8 * n + 2 * (lane & 3);
          *reinterpret_cast<float2*>(dg + (lane >> 2) * 20 + jl) = make_float2(x0, x1);
          *reinterpret_cast<float2*>(dg + ((lane >> 2) + 8) * 20 + jl) = make_float2(x2, x3);
        }
      }
    }
    __syncwarp();
    // the diagonal block's inverse, a column of T (a row of T^T) a lane: t_i = -sum_(j < i) A_ij t_j below t_c = 1
    float t[16];
    const int c = lane & 15;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float row[16];
#pragma unroll
      for (int q4 = 0; q4 < (i + 3) / 4; ++q4) {
        const float4 x = *reinterpret_cast<const float4*>(dg + i * 20 + 4 * q4);
        row[4 * q4] = x.x; row[4 * q4 + 1] = x.y; row[4 * q4 + 2] = x.z; row[4 * q4 + 3] = x.w;
      }
      float sum = i == c ? 1.f : 0.f, other = 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) {
        if (j & 1) other = fmaf(row[j], t[j], other);
        else sum = fmaf(row[j], t[j], sum);
      }
      t[i] = i < c ? 0.f : sum + other;
    }
    if (lane < 16) {
      uint32_t hi[8], lo[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) split(t[2 * i], t[2 * i + 1], hi[i], lo[i]);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t at = unit_at(16 * w + c, 2 * w + u);
        *reinterpret_cast<uint4*>(st.t_hi + at) = make_uint4(hi[4 * u], hi[4 * u + 1], hi[4 * u + 2], hi[4 * u + 3]);
        *reinterpret_cast<uint4*>(st.t_lo + at) = make_uint4(lo[4 * u], lo[4 * u + 1], lo[4 * u + 2], lo[4 * u + 3]);
      }
    }
  }

  struct Pair { uint32_t hi[4], lo[4]; };     // a 16 x 16 block as first operand, in two terms
  __device__ __forceinline__ Pair first_operand(const Stage& st, int rb, int cb) const {
    Pair x;
    ldm4(x.hi, smem_u32(st.t_hi) + down(16 * rb, 2 * cb, lane));
    ldm4(x.lo, smem_u32(st.t_lo) + down(16 * rb, 2 * cb, lane));
    return x;
  }
  __device__ __forceinline__ static Pair as_operand(const float (&c)[2][4]) {
    Pair x;
    split(c[0][0], c[0][1], x.hi[0], x.lo[0]);
    split(c[0][2], c[0][3], x.hi[1], x.lo[1]);
    split(c[1][0], c[1][1], x.hi[2], x.lo[2]);
    split(c[1][2], c[1][3], x.hi[3], x.lo[3]);
    return x;
  }
  __device__ __forceinline__ static void mma3(float (&c)[2][4], const Pair& a, const uint32_t (&hi)[4], const uint32_t (&lo)[4]) {
    mma(c[0], a.hi, hi[0], hi[1]);
    mma(c[1], a.hi, hi[2], hi[3]);
    mma(c[0], a.hi, lo[0], lo[1]);
    mma(c[1], a.hi, lo[2], lo[3]);
    mma(c[0], a.lo, hi[0], hi[1]);
    mma(c[1], a.lo, hi[2], hi[3]);
  }
  // c += x (-A_il)^T, -A stored by rows i
  __device__ __forceinline__ void times_a(float (&c)[2][4], const Pair& x, const Stage& st, int i, int l) const {
    uint32_t hi[4], lo[4];
    ldm4(hi, smem_u32(st.t_hi) + across(16 * i, 2 * l, lane));
    ldm4(lo, smem_u32(st.t_lo) + across(16 * i, 2 * l, lane));
    mma3(c, x, hi, lo);
  }
  // c += x T_il^T, T^T stored by rows l
  __device__ __forceinline__ void times_t(float (&c)[2][4], const Pair& x, const Stage& st, int i, int l) const {
    uint32_t hi[4], lo[4];
    ldm4t(hi, smem_u32(st.t_hi) + down(16 * l, 2 * i, lane));
    ldm4t(lo, smem_u32(st.t_lo) + down(16 * l, 2 * i, lane));
    mma3(c, x, hi, lo);
  }
  __device__ __forceinline__ void store_t(const float (&c)[2][4], Stage& st, int i, int j) const {
    const Pair x = as_operand(c);
    const int row = 16 * j + (lane >> 2), col = (lane & 3) * 4;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      *reinterpret_cast<uint32_t*>(st.t_hi + unit_at(row, 2 * i + n) + col) = x.hi[2 * n];
      *reinterpret_cast<uint32_t*>(st.t_hi + unit_at(row + 8, 2 * i + n) + col) = x.hi[2 * n + 1];
      *reinterpret_cast<uint32_t*>(st.t_lo + unit_at(row, 2 * i + n) + col) = x.lo[2 * n];
      *reinterpret_cast<uint32_t*>(st.t_lo + unit_at(row + 8, 2 * i + n) + col) = x.lo[2 * n + 1];
    }
  }
  __device__ __forceinline__ static void zero(float (&c)[2][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[0][i] = c[1][i] = 0.f;
  }

  // T's blocks off the diagonal from those on it, by halves: T_10 and T_32 first (warp 0, warp 1), then column 0, column 1 of the lower left quarter:
  //   [T_20 T_21; T_30 T_31] = -[T_22 0; T_32 T_33] [A_20 A_21; A_30 A_31] [T_00 0; T_10 T_11]
  __device__ __forceinline__ void off_diagonal(Stage& st) const {
    float c[2][4], m2[2][4], m3[2][4];
    zero(c);
    times_a(c, first_operand(st, 2 * w, 2 * w), st, 2 * w + 1, 2 * w);
    const Pair x = as_operand(c);
    zero(c);
    times_t(c, x, st, 2 * w + 1, 2 * w + 1);
    store_t(c, st, 2 * w + 1, 2 * w);
    bar_sync(2, 64);
    zero(m2);
    zero(m3);
    for (int l = w; l < 2; ++l) {
      const Pair t = first_operand(st, w, l);
      times_a(m2, t, st, 2, l);
      times_a(m3, t, st, 3, l);
    }
    const Pair a2 = as_operand(m2), a3 = as_operand(m3);
    zero(m2);
    zero(m3);
    times_t(m2, a2, st, 2, 2);
    times_t(m3, a2, st, 3, 2);
    times_t(m3, a3, st, 3, 3);
    store_t(m2, st, 2, w);
    store_t(m3, st, 3, w);
  }

  __device__ __forceinline__ void row_of_p(Stage& st, int ib) const {
    uint32_t a[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) ldm4(a[ks], smem_u32(st.q) + down(16 * ib, 2 * ks, lane));
    const int i0 = 16 * ib + (lane >> 2), i1 = i0 + 8;
    const float gh0 = sm.g_hi[i0], gl0 = sm.g_lo[i0], gh1 = sm.g_hi[i1], gl1 = sm.g_lo[i1];
    for (int jb = 0; jb <= ib; ++jb) {
      float c[2][4];
      products(c, a, st, jb);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int j = 16 * jb + 8 * n + 2 * (lane & 3);
        const float2 gh = *reinterpret_cast<const float2*>(sm.g_hi + j), gl = *reinterpret_cast<const float2*>(sm.g_lo + j);
        const float2 r = *reinterpret_cast<const float2*>(sm.rk + j);
        float x0 = r.x * c[n][0] * exp2_fast((gh0 - gh.x) + (gl0 - gl.x)), x1 = r.y * c[n][1] * exp2_fast((gh0 - gh.y) + (gl0 - gl.y));
        float x2 = r.x * c[n][2] * exp2_fast((gh1 - gh.x) + (gl1 - gl.x)), x3 = r.y * c[n][3] * exp2_fast((gh1 - gh.y) + (gl1 - gl.y));
        if (jb == ib) {                          // above the diagonal nothing
          if (j > i0) x0 = 0.f;
          if (j + 1 > i0) x1 = 0.f;
          if (j > i1) x2 = 0.f;
          if (j + 1 > i1) x3 = 0.f;
        }
        *reinterpret_cast<uint32_t*>(st.p + unit_at(i0, j >> 3) + (j & 7) * 2) = pack_f16x2(x0, x1);
        *reinterpret_cast<uint32_t*>(st.p + unit_at(i1, j >> 3) + (j & 7) * 2) = pack_f16x2(x2, x3);
      }
    }
  }

  __device__ __forceinline__ void run(int t_begin, int chunks) const {
    Loads x;
    fetch(x, t_begin);
    for (int n = 0; n < chunks; ++n) {
      const int s = n & 1, t0 = t_begin + n * CHUNK;
      Stage& st = sm.stage[s];
      if (n >= 2) bar_sync(5 + s, 256);
#pragma unroll
      for (int i = 0; i < 4; ++i) {              // V as it is
        const int row = 16 * w + 4 * i + (lane >> 3), unit = lane & 7;
        uint8_t* to = st.v + unit_at(row, unit);
        if (t0 + row < len) copy_async_16(smem_u32(to), p.v + (size_t(b) * p.T + t0 + row) * p.ldv + size_t(h) * D + unit * 8);
        else *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
      }
      convert(x, st);
      if (n + 1 < chunks) fetch(x, t0 + CHUNK);
      bar_sync(1, 128);
      row_of_a(st);
      if (w == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = lane + 32 * i;
          const float r = sm.rk[row], n1 = sm.nk[row], beta = sm.beta[row];
          st.of_v[row] = beta * n1;
          st.of_y[row] = beta * n1 * n1 * st.grow[row] * r;
          st.of_u[row] *= r;
          if (OUT) st.of_o[row] = sm.rq[row];
        }
      }
      bar_sync(1, 128);
      if (w < 2) {
        off_diagonal(st);
      } else if (OUT) {
        row_of_p(st, w == 2 ? 1 : 3);
        row_of_p(st, w == 2 ? 2 : 0);
      }
      copy_async_wait();
      bar_arrive(3 + s, 256);
      bar_sync(1, 128);                          // rk, g and the others are overwritten next
    }
  }
};

// ---- the warps of the state -------------------------------------------------------------------------------------------
template <bool OUT>
struct Follow {
  const DeltaParams& p;
  ChunkSmem& sm;
  int b, h, w, lane, len;

  __device__ __forceinline__ void chunk(float (&S)[8][4], Stage& st, int t0) const {
    const int c2 = 2 * (lane & 3);
    // S in two terms
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      m0 = fmaxf(m0, fmaxf(fabsf(S[n][0]), fabsf(S[n][1])));
      m1 = fmaxf(m1, fmaxf(fabsf(S[n][2]), fabsf(S[n][3])));
    }
    m0 = quad_max(m0);
    m1 = quad_max(m1);
    float s0, s1, is0, is1;
    power_scale<14>(m0, s0, is0);
    power_scale<14>(m1, s1, is1);
    uint32_t sh[4][4], sl[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      split(S[2 * ks][0] * s0, S[2 * ks][1] * s0, sh[ks][0], sl[ks][0]);
      split(S[2 * ks][2] * s1, S[2 * ks][3] * s1, sh[ks][1], sl[ks][1]);
      split(S[2 * ks + 1][0] * s0, S[2 * ks + 1][1] * s0, sh[ks][2], sl[ks][2]);
      split(S[2 * ks + 1][2] * s1, S[2 * ks + 1][3] * s1, sh[ks][3], sl[ks][3]);
    }
    // Y^T = S K^T
    float y[8][4];
    const uint32_t kb = smem_u32(st.k), lane4 = unit_at(lane & 7, lane >> 3);   // four neighbouring units of eight rows
#pragma unroll
    for (int n = 0; n < 8; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[n][i] = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t f[4];
        ldm4(f, kb + n * 1024 + (lane4 ^ (half << 6)));
        mma(y[n], sh[2 * half], f[0], f[1]);
        mma(y[n], sh[2 * half + 1], f[2], f[3]);
        mma(y[n], sl[2 * half], f[0], f[1]);
        mma(y[n], sl[2 * half + 1], f[2], f[3]);
      }
    }
    // X^T = b (V - e^G Y)
    float x0 = m0 * 8.6736174e-19f, x1 = m1 * 8.6736174e-19f;      // 2^-60: X's power must leave S in range, too
#pragma unroll
    for (int n2 = 0; n2 < 4; ++n2) {
      uint32_t f[4];
      ldm4t(f, smem_u32(st.v) + unit_at(16 * n2 + ((lane >> 4) << 3) + (lane & 7), 2 * w + ((lane >> 3) & 1)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float(&t)[4] = y[2 * n2 + i];
        const int j = 16 * n2 + 8 * i + c2;
        const float2 fv = *reinterpret_cast<const float2*>(st.of_v + j), fy = *reinterpret_cast<const float2*>(st.of_y + j);
        t[0] = fmaf(fv.x, bf16_lo(f[2 * i]), -(fy.x * is0) * t[0]);
        t[1] = fmaf(fv.y, bf16_hi(f[2 * i]), -(fy.y * is0) * t[1]);
        t[2] = fmaf(fv.x, bf16_lo(f[2 * i + 1]), -(fy.x * is1) * t[2]);
        t[3] = fmaf(fv.y, bf16_hi(f[2 * i + 1]), -(fy.y * is1) * t[3]);
        x0 = fmaxf(x0, fmaxf(fabsf(t[0]), fabsf(t[1])));
        x1 = fmaxf(x1, fmaxf(fabsf(t[2]), fabsf(t[3])));
      }
    }
    // |T_ij| <= 2 where b |k|^2 <= 2, so that U <= 128 X stays in range
    float e0, e1, ie0, ie1;
    power_scale<7>(quad_max(x0), e0, ie0);
    power_scale<7>(quad_max(x1), e1, ie1);
    uint32_t xh[4][4], xl[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      split(y[2 * ks][0] * e0, y[2 * ks][1] * e0, xh[ks][0], xl[ks][0]);
      split(y[2 * ks][2] * e1, y[2 * ks][3] * e1, xh[ks][1], xl[ks][1]);
      split(y[2 * ks + 1][0] * e0, y[2 * ks + 1][1] * e0, xh[ks][2], xl[ks][2]);
      split(y[2 * ks + 1][2] * e1, y[2 * ks + 1][3] * e1, xh[ks][3], xl[ks][3]);
    }
    // U^T = X^T T^T, times the row's power
    float u[8][4];
    const uint32_t down0 = down(0, 0, lane);
#pragma unroll
    for (int ib = 0; ib < 4; ++ib) {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[2 * ib][i] = u[2 * ib + 1][i] = 0.f;
#pragma unroll
      for (int jb = 0; jb <= ib; ++jb) {
        uint32_t f[4];
        ldm4t(f, smem_u32(st.t_hi) + jb * 2048 + (down0 ^ (ib << 5)));
        mma(u[2 * ib], xh[jb], f[0], f[1]);
        mma(u[2 * ib + 1], xh[jb], f[2], f[3]);
        mma(u[2 * ib], xl[jb], f[0], f[1]);
        mma(u[2 * ib + 1], xl[jb], f[2], f[3]);
        ldm4t(f, smem_u32(st.t_lo) + jb * 2048 + (down0 ^ (ib << 5)));
        mma(u[2 * ib], xh[jb], f[0], f[1]);
        mma(u[2 * ib + 1], xh[jb], f[2], f[3]);
      }
    }
    if constexpr (OUT) {
      // O^T = e^G S Q^T + U^T P^T
      float o[8][4];
      const uint32_t qb = smem_u32(st.q), across0 = across(0, 0, lane);
      const float q0 = is0 * e0, q1 = is1 * e1;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t f[4];
          ldm4(f, qb + n * 1024 + (lane4 ^ (half << 6)));
          mma(o[n], sh[2 * half], f[0], f[1]);
          mma(o[n], sh[2 * half + 1], f[2], f[3]);
        }
        const float2 grow = *reinterpret_cast<const float2*>(st.grow + 8 * n + c2);
        o[n][0] *= grow.x * q0;
        o[n][1] *= grow.y * q0;
        o[n][2] *= grow.x * q1;
        o[n][3] *= grow.y * q1;
      }
      uint32_t uf[4][4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        uf[ks][0] = pack_f16x2(u[2 * ks][0], u[2 * ks][1]);
        uf[ks][1] = pack_f16x2(u[2 * ks][2], u[2 * ks][3]);
        uf[ks][2] = pack_f16x2(u[2 * ks + 1][0], u[2 * ks + 1][1]);
        uf[ks][3] = pack_f16x2(u[2 * ks + 1][2], u[2 * ks + 1][3]);
      }
#pragma unroll
      for (int ib = 0; ib < 4; ++ib)
#pragma unroll
        for (int jb = 0; jb <= ib; ++jb) {
          uint32_t f[4];
          ldm4(f, smem_u32(st.p) + ib * 2048 + (across0 ^ (jb << 5)));
          mma(o[2 * ib], uf[jb], f[0], f[1]);
          mma(o[2 * ib + 1], uf[jb], f[2], f[3]);
        }
      // into the columns of V that this warp alone has read, then out by rows
#pragma unroll
      for (int n2 = 0; n2 < 4; ++n2) {
        uint32_t f[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 fo = *reinterpret_cast<const float2*>(st.of_o + 16 * n2 + 8 * i + c2);
          const float(&t)[4] = o[2 * n2 + i];
          f[2 * i] = pack_bf16x2(t[0] * (fo.x * ie0), t[1] * (fo.y * ie0));
          f[2 * i + 1] = pack_bf16x2(t[2] * (fo.x * ie1), t[3] * (fo.y * ie1));
        }
        stm4t(smem_u32(st.v) + unit_at(16 * n2 + ((lane >> 4) << 3) + (lane & 7), 2 * w + ((lane >> 3) & 1)), f[0], f[1], f[2], f[3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * i + (lane >> 1), unit = 2 * w + (lane & 1);
        if (t0 + row < len)
          *(reinterpret_cast<uint4*>(p.o + (size_t(b) * p.T + t0 + row) * p.ldo + size_t(h) * D) + unit) = *reinterpret_cast<const uint4*>(st.v + unit_at(row, unit));
      }
    }
    // S' = e^Gc S + (e^(Gc - G) U)^T K, at X's power
    const float whole = st.whole;
    const float k0 = whole * e0, k1 = whole * e1;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      S[n][0] *= k0; S[n][1] *= k0; S[n][2] *= k1; S[n][3] *= k1;
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t uh[4], ul[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 fu = *reinterpret_cast<const float2*>(st.of_u + 16 * ks + 8 * i + c2);
        const float(&t)[4] = u[2 * ks + i];
        split(t[0] * fu.x, t[1] * fu.y, uh[2 * i], ul[2 * i]);
        split(t[2] * fu.x, t[3] * fu.y, uh[2 * i + 1], ul[2 * i + 1]);
      }
#pragma unroll
      for (int n2 = 0; n2 < 4; ++n2) {
        uint32_t f[4];
        ldm4t(f, kb + ks * 2048 + (down0 ^ (n2 << 5)));
        mma(S[2 * n2], uh, f[0], f[1]);
        mma(S[2 * n2 + 1], uh, f[2], f[3]);
        mma(S[2 * n2], ul, f[0], f[1]);
        mma(S[2 * n2 + 1], ul, f[2], f[3]);
      }
    }
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      S[n][0] *= ie0; S[n][1] *= ie0; S[n][2] *= ie1; S[n][3] *= ie1;
    }
  }
};

template <bool OUT>
__global__ void __launch_bounds__(256, 2) delta_chunk_kernel(DeltaParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  ChunkSmem& sm = *reinterpret_cast<ChunkSmem*>(smem_raw);
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.H, h = blockIdx.x % p.H;
  pdl_wait();
  pdl_trigger();
  const int len = sequence_length(p, b), chunks = (len + CHUNK - 1) / CHUNK;
  if (warp >= 4) {
    if (chunks > 0) Prepare<OUT>{p, sm, b, h, warp - 4, lane, len}.run(0, chunks);
    return;
  }
  const Follow<OUT> f{p, sm, b, h, warp, lane, len};
  float S[8][4];
  const size_t at = size_t(blockIdx.x) * D * D + size_t(16 * warp + (lane >> 2)) * D + 2 * (lane & 3);
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    float2 x = make_float2(0.f, 0.f), y = x;
    if (p.s_in != nullptr) {
      x = *reinterpret_cast<const float2*>(p.s_in + at + 8 * n);
      y = *reinterpret_cast<const float2*>(p.s_in + at + 8 * D + 8 * n);
    }
    S[n][0] = x.x; S[n][1] = x.y; S[n][2] = y.x; S[n][3] = y.y;
  }
  for (int n = 0; n < chunks; ++n) {
    const int s = n & 1;
    bar_sync(3 + s, 256);
    f.chunk(S, sm.stage[s], n * CHUNK);
    if (n + 2 < chunks) bar_arrive(5 + s, 256);
  }
  if (p.s_out != nullptr) {
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      *reinterpret_cast<float2*>(p.s_out + at + 8 * n) = make_float2(S[n][0], S[n][1]);
      *reinterpret_cast<float2*>(p.s_out + at + 8 * D + 8 * n) = make_float2(S[n][2], S[n][3]);
    }
  }
  if (OUT)
    for (int t = len + (threadIdx.x >> 3); t < p.T; t += 16)
      *(reinterpret_cast<uint4*>(p.o + (size_t(b) * p.T + t) * p.ldo + size_t(h) * D) + (threadIdx.x & 7)) = make_uint4(0, 0, 0, 0);
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
  if (T >= 24) {
    if (p.o != nullptr) {
      JB_MAX_SMEM(delta_chunk_kernel<true>, sizeof(ChunkSmem));
      launch_dep(delta_chunk_kernel<true>, B * H, 256, sizeof(ChunkSmem), stream, p);
    } else {
      JB_MAX_SMEM(delta_chunk_kernel<false>, sizeof(ChunkSmem));
      launch_dep(delta_chunk_kernel<false>, B * H, 256, sizeof(ChunkSmem), stream, p);
    }
    JB_LAUNCH_CHECK("delta_chunk_kernel");
    return JB200_OK;
  }
  if (B * H < 2 * sm_count())
    launch_dep(delta_step_kernel<1>, B * H * 4, 128, 0, stream, p);
  else
    launch_dep(delta_step_kernel<4>, B * H, 128, 0, stream, p);
  JB_LAUNCH_CHECK("delta_step_kernel");
  return JB200_OK;
}

}  // namespace jb

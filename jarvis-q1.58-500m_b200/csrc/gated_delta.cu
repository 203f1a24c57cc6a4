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
// A CTA follows one head of one sequence, in four groups of four warps.  Two take turns in preparing chunks (K, T: nothing of the state); one
// takes a chunk through the state, each warp 16 value rows of S in its accumulators, everything transposed (X^T, U^T: 16 values x 64 tokens), so that a
// product's accumulators are the next one's first operand where they are, and the four never wait for one another; one forms P and, from
// S and U as the state's warps leave them, the outputs.
//
// mma.sync, not tcgen05: a chunk is a chain of three dependent products of 16 x 64 x 64 a warp with a rescaling between them; through tensor
// memory each link would cost a commit, a wait and two copies, several times the product itself.
//
// Precision: the state is f32 and stays it.  What is multiplied is f16 in two terms, x = hi + lo (22 bits), with an exact power of two per row that
// puts the row's largest value near the top of f16's range: 2^-24 of the row's maximum each.  K and Q come as bf16 and fit one term, scaled by
// a power of two per row; their norms are factors on rows and columns.  X T^T takes hi hi + hi lo + lo hi.  What only the output sees
// (Q S^T, P U) is one term, 2^-12 of a value where the output's own rounding is 2^-9.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int CHUNK = 64;
constexpr int TILE = CHUNK * D * 2;        // bytes of 64 rows of 128, the 16-byte units of row r at unit ^ (r & 7)
constexpr int STAGES = 3;
constexpr int GROUP = 128;                 // threads of a group of warps
constexpr float LEAST_LOG2 = -300.f;       // 2^-300 is 0 in f32: a decay of less, -inf among them, is this one

struct alignas(128) Stage {
  uint8_t k[TILE], v[TILE];
  uint8_t t_hi[TILE], t_lo[TILE];          // T^T [j][i] on and above the diagonal's 16 x 16 blocks; -A [i][j] below them while T is formed
  float diagonal[4][16 * 20];              // the diagonal blocks of -A in f32
  float g_hi[CHUNK], g_lo[CHUNK], rk[CHUNK], nk[CHUNK], beta[CHUNK];
  float of_v[CHUNK], of_y[CHUNK], of_u[CHUNK], grow[CHUNK];
  float whole;
};
struct alignas(128) ChunkSmem {
  Stage stage[STAGES];
  uint8_t q[2][TILE], p[TILE], o[TILE];
  float of_o[2][CHUNK];
  uint4 s16[4][4][32], u16[4][4][32];      // of every warp of the state: S and U as first operands, lane by lane
  float4 scales[4][32];
};
static_assert(sizeof(Stage) % 128 == 0 && TILE % 128 == 0, "tiles are read 16 bytes at a time in every stage");

// The CTA's barriers.  Ready and free of a stage: the preparing group arrives and waits, the others wait and arrive.
enum { BAR_GROUP = 0 /* + group */, BAR_READY = 2 /* + stage: for the state */, BAR_READY_O = 5 /* + stage: for the outputs */, BAR_FREE = 8 /* + stage */,
       BAR_GIVEN = 11, BAR_TAKEN = 12, BAR_OUT = 13 };
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
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

// The tokens that a CTA takes: of sequence b from row `begin` (of the sequence) on, `chunks` chunks, none from `len` on.
struct Part {
  int b, h, begin, len, chunks;
};

// Sixteen rows of a bf16 matrix a warp, eight lanes a row, four rows a lane: from memory ...
__device__ __forceinline__ void fetch_rows(uint4 (&x)[4], const __nv_bfloat16* rows, size_t ld, int row0, int n, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + 4 * i + (lane >> 3);
    x[i] = make_uint4(0, 0, 0, 0);
    if (row < n) x[i] = __ldg(reinterpret_cast<const uint4*>(rows + size_t(row) * ld) + (lane & 7));
  }
}
// ... and to f16 in a tile, times the power of two s that brings their norm into [1, 2); ss: the sum of squares after that.  A sum of squares
// beyond f32's range makes the row NaN, one below it makes it 0.
__device__ __forceinline__ void convert_rows(const uint4 (&x)[4], uint8_t* tile, int row0, int lane, float (&ss)[4], float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float a = 0.f, c = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) { a = fmaf(bf16_lo(in[j]), bf16_lo(in[j]), a); c = fmaf(bf16_hi(in[j]), bf16_hi(in[j]), c); }
    ss[i] = a + c;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int half = (int(__float_as_uint(ss[i]) >> 23) - 127) >> 1;             // ss in [4^half, 4^(half + 1))
    s[i] = __uint_as_float(uint32_t(127 - half) << 23);
    ss[i] = ss[i] * s[i] * s[i];
    const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = pack_f16x2(bf16_lo(in[j]) * s[i], bf16_hi(in[j]) * s[i]);
    *reinterpret_cast<uint4*>(tile + unit_at(row0 + 4 * i + (lane >> 3), lane & 7)) = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// Blocks on and below the diagonal of a 4 x 4 grid, three or two a warp, the diagonal's first
__device__ __forceinline__ int blocks_of(int w) { return w < 2 ? 3 : 2; }
__device__ __forceinline__ int block_row(int w, int i) { return i == 0 ? w : w < 2 ? 1 + i : w == 2 ? 1 : 3; }
__device__ __forceinline__ int block_col(int w, int i) { return i == 0 ? w : w < 2 ? w : w == 2 ? 0 : 2; }

// A block of rows ib of tile `a` times rows jb of tile `b`, 64 long
__device__ __forceinline__ void block_products(float (&c)[2][4], const uint8_t* a, int ib, const uint8_t* b, int jb, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c[0][i] = c[1][i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    uint32_t f[4], r[4];
    ldm4(r, smem_u32(a) + down(16 * ib, 2 * ks, lane));
    ldm4(f, smem_u32(b) + across(16 * jb, 2 * ks, lane));
    mma(c[0], r, f[0], f[1]);
    mma(c[1], r, f[2], f[3]);
  }
}
// ... times f_i r_j e^(G_i - G_j)
__device__ __forceinline__ void decayed(float (&c)[2][4], const Stage& st, int i0, int jb, float f0, float f1, int lane) {
  const float gh0 = st.g_hi[i0], gl0 = st.g_lo[i0], gh1 = st.g_hi[i0 + 8], gl1 = st.g_lo[i0 + 8];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int j = 16 * jb + 8 * n + 2 * (lane & 3);
    const float2 gh = *reinterpret_cast<const float2*>(st.g_hi + j), gl = *reinterpret_cast<const float2*>(st.g_lo + j);
    const float2 r = *reinterpret_cast<const float2*>(st.rk + j);
    c[n][0] *= f0 * r.x * exp2_fast((gh0 - gh.x) + (gl0 - gl.x));
    c[n][1] *= f0 * r.y * exp2_fast((gh0 - gh.y) + (gl0 - gl.y));
    c[n][2] *= f1 * r.x * exp2_fast((gh1 - gh.x) + (gl1 - gl.x));
    c[n][3] *= f1 * r.y * exp2_fast((gh1 - gh.y) + (gl1 - gl.y));
  }
}

// ---- the preparing groups --------------------------------------------------------------------------------------------
struct Prepare {
  const DeltaParams& p;
  ChunkSmem& sm;
  Part part;
  int group, w, lane;
  int takers;                                // threads that wait for a stage and free it

  // running sums of log2 a, in f64 for differences of late tokens
  __device__ __forceinline__ void gates(Stage& st, float ga, float gb, float beta_a, float beta_b) const {
    double g0 = double(ga) * 1.4426950408889634, g1 = double(gb) * 1.4426950408889634;
    if (g0 < double(LEAST_LOG2)) g0 = double(LEAST_LOG2);
    if (g1 < double(LEAST_LOG2)) g1 = double(LEAST_LOG2);
    double sum = g0 + g1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const double end = __shfl_sync(0xffffffffu, sum, 31);
    const double at[2] = {sum - g1, sum};
    float hi[2], lo[2], grow[2], of_u[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      hi[i] = float(at[i]);
      lo[i] = float(at[i] - double(hi[i]));
      grow[i] = exp2f(hi[i]);
      of_u[i] = exp2f(float(end - at[i]));
    }
    *reinterpret_cast<float2*>(st.g_hi + 2 * lane) = make_float2(hi[0], hi[1]);
    *reinterpret_cast<float2*>(st.g_lo + 2 * lane) = make_float2(lo[0], lo[1]);
    *reinterpret_cast<float2*>(st.beta + 2 * lane) = make_float2(beta_a, beta_b);
    *reinterpret_cast<float2*>(st.grow + 2 * lane) = make_float2(grow[0], grow[1]);
    *reinterpret_cast<float2*>(st.of_u + 2 * lane) = make_float2(of_u[0], of_u[1]);
    if (lane == 0) st.whole = exp2f(float(end));
  }

  // the diagonal block's inverse, a column of T (a row of T^T) a lane: t_i = -sum_(j < i) A_ij t_j below t_c = 1
  __device__ __forceinline__ void diagonal(Stage& st) const {
    const float* dg = st.diagonal[w];
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

  // this warp's blocks of -A, the diagonal's inverted
  __device__ __forceinline__ void blocks_of_a(Stage& st) const {
    for (int n = 0; n < blocks_of(w); ++n) {
      const int ib = block_row(w, n), jb = block_col(w, n);
      float c[2][4];
      block_products(c, st.k, ib, st.k, jb, lane);
      const int i0 = 16 * ib + (lane >> 2), i1 = i0 + 8;
      const float n0 = st.nk[i0], n1 = st.nk[i1];
      decayed(c, st, i0, jb, -st.beta[i0] * n0 * n0 * st.rk[i0], -st.beta[i1] * n1 * n1 * st.rk[i1], lane);
      if (n == 0) {
        float* dg = st.diagonal[w] + (lane >> 2) * 20 + 2 * (lane & 3);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          *reinterpret_cast<float2*>(dg + 8 * i) = make_float2(c[i][0], c[i][1]);
          *reinterpret_cast<float2*>(dg + 8 * 20 + 8 * i) = make_float2(c[i][2], c[i][3]);
        }
        __syncwarp();
        diagonal(st);
      } else {
        const Pair x = as_operand(c);
        const int col = (lane & 3) * 4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          *reinterpret_cast<uint32_t*>(st.t_hi + unit_at(i0, 2 * jb + i) + col) = x.hi[2 * i];
          *reinterpret_cast<uint32_t*>(st.t_lo + unit_at(i0, 2 * jb + i) + col) = x.lo[2 * i];
          *reinterpret_cast<uint32_t*>(st.t_hi + unit_at(i1, 2 * jb + i) + col) = x.hi[2 * i + 1];
          *reinterpret_cast<uint32_t*>(st.t_lo + unit_at(i1, 2 * jb + i) + col) = x.lo[2 * i + 1];
        }
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

  // T's blocks off the diagonal from those on it, by halves: T_10 and T_32 first (warps 0, 1), then columns 0 and 1 of the lower left quarter:
  //   [T_20 T_21; T_30 T_31] = -[T_22 0; T_32 T_33] [A_20 A_21; A_30 A_31] [T_00 0; T_10 T_11]
  __device__ __forceinline__ void off_diagonal(Stage& st) const {
    if (w < 2) {
      float c[2][4];
      zero(c);
      times_a(c, first_operand(st, 2 * w, 2 * w), st, 2 * w + 1, 2 * w);
      const Pair x = as_operand(c);
      zero(c);
      times_t(c, x, st, 2 * w + 1, 2 * w + 1);
      store_t(c, st, 2 * w + 1, 2 * w);
    }
    bar_sync(BAR_GROUP + group, GROUP);
    if (w < 2) {
      float m2[2][4], m3[2][4];
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
  }

  __device__ __forceinline__ void run() const {
    const size_t first = size_t(part.b) * p.T;
    const __nv_bfloat16* kp = p.k + first * p.ldk + size_t(part.h / p.per_key) * D;
    const __nv_bfloat16* vp = p.v + first * p.ldv + size_t(part.h) * D;
    uint4 k[4];
    float g0 = 0.f, g1 = 0.f, b0 = 0.f, b1 = 0.f;
    auto fetch = [&](int t0) {
      fetch_rows(k, kp, p.ldk, t0 + 16 * w, part.len, lane);
      if (w == 3) {
        const int t = t0 + 2 * lane;
        g0 = t < part.len ? __ldg(p.log_decay + (first + t) * p.ldg + part.h) : 0.f;
        b0 = t < part.len ? __ldg(p.beta + (first + t) * p.ldg + part.h) : 0.f;
        g1 = t + 1 < part.len ? __ldg(p.log_decay + (first + t + 1) * p.ldg + part.h) : 0.f;
        b1 = t + 1 < part.len ? __ldg(p.beta + (first + t + 1) * p.ldg + part.h) : 0.f;
      }
    };
    if (group < part.chunks) fetch(part.begin + group * CHUNK);
    for (int n = group; n < part.chunks; n += 2) {
      const int s = n % STAGES, t0 = part.begin + n * CHUNK;
      Stage& st = sm.stage[s];
      if (n >= STAGES) bar_sync(BAR_FREE + s, GROUP + takers);
#pragma unroll
      for (int i = 0; i < 4; ++i) {              // V as it is
        const int row = 16 * w + 4 * i + (lane >> 3), unit = lane & 7;
        uint8_t* to = st.v + unit_at(row, unit);
        if (t0 + row < part.len) copy_async_16(smem_u32(to), vp + size_t(t0 + row) * p.ldv + unit * 8);
        else *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
      }
      float ss[4], sc[4];
      convert_rows(k, st.k, 16 * w, lane, ss, sc);
      if ((lane & 7) == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // k = n (k16 r) with |k16 r| = 1, or of the normalised key n = 1 and k16 r its value
          const int row = 16 * w + 4 * i + (lane >> 3);
          const float r = p.normalize ? rsqrtf(fmaf(NORM_EPS * sc[i], sc[i], ss[i])) : ss[i] > 0.f ? rsqrtf(ss[i]) : 0.f;
          st.rk[row] = r;
          st.nk[row] = p.normalize ? 1.f : ss[i] * r / sc[i];
        }
      }
      if (w == 3) gates(st, g0, g1, b0, b1);
      if (n + 2 < part.chunks) fetch(t0 + 2 * CHUNK);
      bar_sync(BAR_GROUP + group, GROUP);
      blocks_of_a(st);
      if (w == 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = lane + 32 * i;
          const float r = st.rk[row], n1 = st.nk[row], beta = st.beta[row];
          st.of_v[row] = beta * n1;
          st.of_y[row] = beta * n1 * n1 * st.grow[row] * r;
          st.of_u[row] *= r;
        }
      }
      bar_sync(BAR_GROUP + group, GROUP);
      off_diagonal(st);
      copy_async_wait();
      bar_arrive(BAR_READY + s, 2 * GROUP);
      if (takers == 2 * GROUP) bar_arrive(BAR_READY_O + s, 2 * GROUP);
    }
  }
};

// ---- the group of the state ------------------------------------------------------------------------------------------
// OUT: gives S and U to the group of the outputs.  VALUES: false where v counts as 0.
template <bool OUT, bool VALUES>
struct Follow {
  ChunkSmem& sm;
  int w, lane;

  // S: accumulators of 16 x 64, times inv0 (rows lane / 4) and inv1 (those and eight) the state
  __device__ __forceinline__ void chunk(float (&S)[8][4], float& inv0, float& inv1, Stage& st, bool wait) const {
    const int c2 = 2 * (lane & 3);
    // S in two terms
    float m0 = 0.f, m1 = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      m0 = fmaxf(m0, fmaxf(fabsf(S[n][0]), fabsf(S[n][1])));
      m1 = fmaxf(m1, fmaxf(fabsf(S[n][2]), fabsf(S[n][3])));
    }
    m0 = quad_max(m0) * inv0;
    m1 = quad_max(m1) * inv1;
    float s0, s1, is0, is1;
    power_scale<14>(m0, s0, is0);
    power_scale<14>(m1, s1, is1);
    s0 *= inv0;
    s1 *= inv1;
    uint32_t sh[4][4], sl[4][4];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      split(S[2 * ks][0] * s0, S[2 * ks][1] * s0, sh[ks][0], sl[ks][0]);
      split(S[2 * ks][2] * s1, S[2 * ks][3] * s1, sh[ks][1], sl[ks][1]);
      split(S[2 * ks + 1][0] * s0, S[2 * ks + 1][1] * s0, sh[ks][2], sl[ks][2]);
      split(S[2 * ks + 1][2] * s1, S[2 * ks + 1][3] * s1, sh[ks][3], sl[ks][3]);
    }
    if (OUT && wait) bar_sync(BAR_TAKEN, 2 * GROUP);
    if constexpr (OUT)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) sm.s16[w][ks][lane] = make_uint4(sh[ks][0], sh[ks][1], sh[ks][2], sh[ks][3]);
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
      uint32_t f[4] = {};
      if constexpr (VALUES) ldm4t(f, smem_u32(st.v) + unit_at(16 * n2 + ((lane >> 4) << 3) + (lane & 7), 2 * w + ((lane >> 3) & 1)));
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
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        sm.u16[w][ks][lane] = make_uint4(pack_f16x2(u[2 * ks][0], u[2 * ks][1]), pack_f16x2(u[2 * ks][2], u[2 * ks][3]),
                                         pack_f16x2(u[2 * ks + 1][0], u[2 * ks + 1][1]), pack_f16x2(u[2 * ks + 1][2], u[2 * ks + 1][3]));
      sm.scales[w][lane] = make_float4(is0 * e0, is1 * e1, ie0, ie1);
      bar_arrive(BAR_GIVEN, 2 * GROUP);
    }
    // S' = e^Gc S + (e^(Gc - G) U)^T K, at X's power
    const float whole = st.whole;
    const float k0 = whole * (e0 * inv0), k1 = whole * (e1 * inv1);
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
    inv0 = ie0;
    inv1 = ie1;
  }

  // from `from` (null: 0; `one`: the identity) through the part's chunks to `to` (or nowhere)
  __device__ __forceinline__ void run(const Part& part, const float* from, bool one, float* to, int ready, int takers) const {
    float S[8][4];
    const int row = 16 * w + (lane >> 2), at = row * D + 2 * (lane & 3);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      float2 x = make_float2(0.f, 0.f), y = x;
      if (from != nullptr) {
        x = *reinterpret_cast<const float2*>(from + at + 8 * n);
        y = *reinterpret_cast<const float2*>(from + at + 8 * D + 8 * n);
      } else if (one) {
        const int d = row - 8 * n - 2 * (lane & 3);
        x = make_float2(d == 0, d == 1);
        y = make_float2(d == -8, d == -7);
      }
      S[n][0] = x.x; S[n][1] = x.y; S[n][2] = y.x; S[n][3] = y.y;
    }
    float inv0 = 1.f, inv1 = 1.f;
    for (int n = 0; n < part.chunks; ++n) {
      const int s = n % STAGES;
      bar_sync(ready + s, 2 * GROUP);
      chunk(S, inv0, inv1, sm.stage[s], n > 0);
      if (n + STAGES < part.chunks) bar_arrive(BAR_FREE + s, GROUP + takers);
    }
    if (to != nullptr) {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        *reinterpret_cast<float2*>(to + at + 8 * n) = make_float2(S[n][0] * inv0, S[n][1] * inv0);
        *reinterpret_cast<float2*>(to + at + 8 * D + 8 * n) = make_float2(S[n][2] * inv1, S[n][3] * inv1);
      }
    }
  }
};

// ---- the group of the outputs ----------------------------------------------------------------------------------------
struct Outputs {
  const DeltaParams& p;
  ChunkSmem& sm;
  Part part;
  int w, lane;

  __device__ __forceinline__ void blocks_of_p(const uint8_t* q, const Stage& st) const {
    for (int n = 0; n < blocks_of(w); ++n) {
      const int ib = block_row(w, n), jb = block_col(w, n), i0 = 16 * ib + (lane >> 2), col = (lane & 3) * 4;
      float c[2][4];
      block_products(c, q, ib, st.k, jb, lane);
      decayed(c, st, i0, jb, 1.f, 1.f, lane);
      if (n == 0) {                            // above the diagonal nothing
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = (lane >> 2) - 8 * i - 2 * (lane & 3);
          if (d < 0) c[i][0] = 0.f;
          if (d < 1) c[i][1] = 0.f;
          if (d < -8) c[i][2] = 0.f;
          if (d < -7) c[i][3] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<uint32_t*>(sm.p + unit_at(i0, 2 * jb + i) + col) = pack_f16x2(c[i][0], c[i][1]);
        *reinterpret_cast<uint32_t*>(sm.p + unit_at(i0 + 8, 2 * jb + i) + col) = pack_f16x2(c[i][2], c[i][3]);
      }
    }
  }

  __device__ __forceinline__ void run() const {
    const size_t first = size_t(part.b) * p.T;
    const __nv_bfloat16* qp = p.q + first * p.ldq + size_t(part.h / p.per_key) * D;
    __nv_bfloat16* op = p.o + first * p.ldo + size_t(part.h) * D;
    const int c2 = 2 * (lane & 3);
    const uint32_t lane4 = unit_at(lane & 7, lane >> 3), across0 = across(0, 0, lane);
    uint4 x[4];
    if (part.chunks > 0) fetch_rows(x, qp, p.ldq, part.begin + 16 * w, part.len, lane);
    for (int n = 0; n < part.chunks; ++n) {
      const int s = n % STAGES, t0 = part.begin + n * CHUNK;
      const Stage& st = sm.stage[s];
      uint8_t* q = sm.q[n & 1];                // the other one may still be read
      float* of_o = sm.of_o[n & 1];
      float ss[4], sc[4];
      convert_rows(x, q, 16 * w, lane, ss, sc);
      if ((lane & 7) == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          of_o[16 * w + 4 * i + (lane >> 3)] = p.scale * (p.normalize ? rsqrtf(fmaf(NORM_EPS * sc[i], sc[i], ss[i])) : 1.f / sc[i]);
      if (n + 1 < part.chunks) fetch_rows(x, qp, p.ldq, t0 + CHUNK + 16 * w, part.len, lane);
      bar_sync(BAR_READY_O + s, 2 * GROUP);
      blocks_of_p(q, st);
      float2 grow[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) grow[i] = *reinterpret_cast<const float2*>(st.grow + 8 * i + c2);
      bar_sync(BAR_OUT, GROUP);
      if (n + STAGES < part.chunks) bar_arrive(BAR_FREE + s, 3 * GROUP);
      bar_sync(BAR_GIVEN, 2 * GROUP);
      uint32_t sh[4][4], uf[4][4];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const uint4 a = sm.s16[w][ks][lane], c = sm.u16[w][ks][lane];
        sh[ks][0] = a.x; sh[ks][1] = a.y; sh[ks][2] = a.z; sh[ks][3] = a.w;
        uf[ks][0] = c.x; uf[ks][1] = c.y; uf[ks][2] = c.z; uf[ks][3] = c.w;
      }
      const float4 scales = sm.scales[w][lane];
      if (n + 1 < part.chunks) bar_arrive(BAR_TAKEN, 2 * GROUP);
      // O^T = e^G S Q^T + U^T P^T
      float o[8][4];
#pragma unroll
      for (int m = 0; m < 8; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[m][i] = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t f[4];
          ldm4(f, smem_u32(q) + m * 1024 + (lane4 ^ (half << 6)));
          mma(o[m], sh[2 * half], f[0], f[1]);
          mma(o[m], sh[2 * half + 1], f[2], f[3]);
        }
        o[m][0] *= grow[m].x * scales.x;
        o[m][1] *= grow[m].y * scales.x;
        o[m][2] *= grow[m].x * scales.y;
        o[m][3] *= grow[m].y * scales.y;
      }
#pragma unroll
      for (int ib = 0; ib < 4; ++ib)
#pragma unroll
        for (int jb = 0; jb <= ib; ++jb) {
          uint32_t f[4];
          ldm4(f, smem_u32(sm.p) + ib * 2048 + (across0 ^ (jb << 5)));
          mma(o[2 * ib], uf[jb], f[0], f[1]);
          mma(o[2 * ib + 1], uf[jb], f[2], f[3]);
        }
      // by way of this warp's columns of a tile, out by rows
#pragma unroll
      for (int n2 = 0; n2 < 4; ++n2) {
        uint32_t f[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 fo = *reinterpret_cast<const float2*>(of_o + 16 * n2 + 8 * i + c2);
          const float(&t)[4] = o[2 * n2 + i];
          f[2 * i] = pack_bf16x2(t[0] * (fo.x * scales.z), t[1] * (fo.y * scales.z));
          f[2 * i + 1] = pack_bf16x2(t[2] * (fo.x * scales.w), t[3] * (fo.y * scales.w));
        }
        stm4t(smem_u32(sm.o) + unit_at(16 * n2 + ((lane >> 4) << 3) + (lane & 7), 2 * w + ((lane >> 3) & 1)), f[0], f[1], f[2], f[3]);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 16 * i + (lane >> 1), unit = 2 * w + (lane & 1);
        if (t0 + row < part.len)
          *(reinterpret_cast<uint4*>(op + size_t(t0 + row) * p.ldo) + unit) = *reinterpret_cast<const uint4*>(sm.o + unit_at(row, unit));
      }
      __syncwarp();
    }
  }
};

template <bool OUT>
__global__ void __launch_bounds__(4 * GROUP, 1) delta_chunk_kernel(DeltaParams p) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  ChunkSmem& sm = *reinterpret_cast<ChunkSmem*>(smem_raw);
  const int warp = warp_index(), lane = threadIdx.x & 31, w = warp & 3;
  Part part;
  part.b = blockIdx.x / p.H;
  part.h = blockIdx.x % p.H;
  part.begin = 0;
  pdl_wait();
  pdl_trigger();
  part.len = sequence_length(p, part.b);
  part.chunks = (part.len + CHUNK - 1) / CHUNK;
  constexpr int TAKERS = OUT ? 2 * GROUP : GROUP;
  const size_t state = size_t(blockIdx.x) * D * D;
  switch (warp >> 2) {
    case 0:
      Follow<OUT, true>{sm, w, lane}.run(part, p.s_in == nullptr ? nullptr : p.s_in + state, false, p.s_out == nullptr ? nullptr : p.s_out + state,
                                         BAR_READY, TAKERS);
      break;
    case 1:
      if (OUT) {
        Outputs{p, sm, part, w, lane}.run();
        for (int t = part.len + (threadIdx.x - GROUP) / 8; t < p.T; t += GROUP / 8)
          *(reinterpret_cast<uint4*>(p.o + (size_t(part.b) * p.T + t) * p.ldo + size_t(part.h) * D) + (threadIdx.x & 7)) = make_uint4(0, 0, 0, 0);
      }
      break;
    default:
      Prepare{p, sm, part, (warp >> 2) - 2, w, lane, TAKERS}.run();
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
  if (T >= 24) {
    if (p.o != nullptr) {
      JB_MAX_SMEM(delta_chunk_kernel<true>, sizeof(ChunkSmem));
      launch_dep(delta_chunk_kernel<true>, B * H, 4 * GROUP, sizeof(ChunkSmem), stream, p);
    } else {
      JB_MAX_SMEM(delta_chunk_kernel<false>, sizeof(ChunkSmem));
      launch_dep(delta_chunk_kernel<false>, B * H, 4 * GROUP, sizeof(ChunkSmem), stream, p);
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

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
constexpr float SMALLER = 6.7762636e-21f, LARGER = 1.2379401e27f;      // 2^-67, 2^90: bring squares that are too large or too small for f32 into it

struct DeltaParams {
  const __nv_bfloat16 *q, *k, *v;
  size_t ldq, ldk, ldv, ldo, ldg, ldb;      // elements
  const float *log_decay, *beta;            // [B T][ldg], [B T][ldb]
  const int32_t* lengths;                   // [B] or null
  const float* s_in;                        // [B][H][64][64] or null
  float* s_out;                             // or null
  __nv_bfloat16* o;
  int B, T, H, per_key;                     // per_key: value heads that share a key head
  float scale;
  int normalize;
  int segments, seg_chunks;                 // pieces of a sequence, 64 tokens times seg_chunks each
  int what;                                 // of this launch: ALL segments (with outputs), the PIECES of all but the last, the LAST segment's state
  float* pieces;                            // [B][H][2 segments - 1][64][64]: what segment s adds (from segment s + 1 on: the state before it), then what
                                            // it multiplies the state by, last the state before segment 0
};
enum { ALL, PIECES, LAST };
__host__ __device__ __forceinline__ size_t piece_at(int segments, int bh, int i) { return (size_t(bh) * (2 * segments - 1) + i) * D * D; }

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
  const float* bp = p.beta + first * p.ldb + h;
  Token next;
  float v_next[ROWS];
  auto fetch = [&](int t) {
    next.k0 = *reinterpret_cast<const uint2*>(kp + size_t(t) * p.ldk);
    next.k1 = *reinterpret_cast<const uint2*>(kp + size_t(t) * p.ldk + 32);
    next.q0 = *reinterpret_cast<const uint2*>(qp + size_t(t) * p.ldq);
    next.q1 = *reinterpret_cast<const uint2*>(qp + size_t(t) * p.ldq + 32);
    next.g = gp[size_t(t) * p.ldg];
    next.beta = bp[size_t(t) * p.ldb];
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
    float kk, qq, kq, eps_k = NORM_EPS, eps_q = NORM_EPS;
    for (bool again = false;; again = true) {
      kk = qq = kq = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) { kk = fmaf(k[j], k[j], kk); qq = fmaf(q[j], q[j], qq); kq = fmaf(k[j], q[j], kq); }
      kk = sum8(kk);
      qq = sum8(qq);
      kq = sum8(kq);
      if (again || !p.normalize || !(fmaxf(kk, qq) == INFINITY)) break;
      // squares that leave f32, the same in all lanes: once more of smaller rows, beside which NORM_EPS is nothing
      const float fk = kk == INFINITY ? SMALLER : 1.f, fq = qq == INFINITY ? SMALLER : 1.f;
      eps_k *= fk;
      eps_q *= fq;
#pragma unroll
      for (int j = 0; j < 8; ++j) { k[j] *= fk; q[j] *= fq; }
    }
    const float rk = p.normalize ? rsqrtf(kk + eps_k) : 1.f, rq = (p.normalize ? rsqrtf(qq + eps_q) : 1.f) * p.scale;
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
// A CTA follows one head of one sequence:
//   warps 0-3          the state: S in registers (f32, a key and 32 values a thread); per chunk three products, K S^T, T X and K^T U, with
//                      X, U and S back in shared memory as their operands between them: the chain that everything waits for
//   warps 4-7, 8-11    by turns prepare a chunk, nothing of the state: K and Q as f16, A and T
//   warps 12, 13       output rows from Q S^T and P U, which the state's warps issue beside their own
//   warps 14, 15       P
// The products are tcgen05.mma, 128 rows at a time: a chunk has 64, so that the operand is there twice (K twice in memory; a second reading
// of T^T and K, MN-major) and all four of a group's warps find 64 rows in their lanes; for P it is [K; Q], of Q and P as operands the
// upper half is what happens to follow, in lanes that nobody reads.  Both terms of S, X and U (below) are one operand of 128 columns: the product
// reads its other operand once for both, and what bounds these small products is reading (6 KB in 48 cycles, 8 KB in 64, for 32 and 64 of
// mathematics).  T's blocks come from mma.sync: products of 16 x 16.
//
// Bound by that chain, some 6200 cycles a chunk on every SM that has a head (8 sequences of 2048 tokens, 16 heads: 114 us, where reading and writing
// takes 21; with one power of two for all value rows, which is wrong beside an outlier, 5900 and 107).  With mma.sync alone a chunk took 10800, with
// these warps' parts but all products unrolled 9600: 77 KB of code, which the SMs fetch again and again.
//
// Precision: the state is f32 and stays it.  What it is multiplied by and into is f16 in two terms, x = hi + lo (22 bits), at a power of two
// that brings a bound of its size to 2^15, so that f16's subnormals lie 2^-39 below.  Value rows of S are independent of one another, and so is each
// one's power: a value row is a column of every product here, so that an infinity, or values far larger than the others, stay in theirs.  With N a
// bound of a value row's norm, a chunk's S, X and U are at most 2 N + 130 max|b v| there and N' = e^Gc N + 64 max|b v|, since a (I - b k k^T)
// with b |k|^2 <= 2 enlarges nothing (a chunk has 64 tokens); every fourth chunk N is at most 8 max|S| as well (a row has 64 entries).  Keys of norm 1
// that bf16 has rounded up to 1 + 2^-8 make that 2.0078, which may enlarge a row by 1.0078^64 = 1.65 in a chunk: N' has that much room.  max|b v|
// comes from the preparing groups, and the next chunk's powers are made while T X is formed.  Typical values lie 2^5 to 2^11 below the bound, and 2^15
// below it two terms still have an f32's 24 bits.  A row's largest |b v| of a chunk counts for the chunk's earlier tokens too: 2^-39 of the bound an
// element of S, X and U, outputs there are off by up to 2^-25 scale |q| of it.  K and Q come as bf16 and fit one term, with a power of two per row;
// their norms are factors of rows and columns.  T X is hi hi + hi lo + lo hi.  What only the output sees (Q S^T, P U) is one term, 2^-12 of a value
// where the output's own rounding is 2^-9.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int CHUNK = 64;
constexpr int TILE = CHUNK * D * 2;        // bytes of 64 rows of 128, the 16-byte units of row r at unit ^ (r & 7): the 128-byte swizzle
constexpr int STAGES = 3;
constexpr int STATE = 128, GROUP = 128;    // threads of the state's group, of a preparing one
constexpr int OUT_THREADS = 64;            // those of the output rows, of P
constexpr float LEAST_LOG2 = -300.f;       // 2^-300 is 0 in f32: a decay of less, -inf among them, is this one

struct alignas(1024) Stage {
  uint8_t k_again[TILE], k[TILE], q[TILE], p[TILE];    // rows of K twice: K; K and K; Q are 128 rows each
  uint8_t t_hi[TILE], t_lo[TILE];                      // T^T [j][i], 0 below the diagonal's 16 x 16 blocks
  float2 column[CHUNK];                                // -G in two terms, the lower one with log2 r: r = k / k16
  float2 g[CHUNK];                                     // G in two terms
  float rk[CHUNK], nk[CHUNK], beta[CHUNK];
  float of_v[CHUNK], of_y[CHUNK], of_u[CHUNK], of_s[CHUNK], of_o[CHUNK];
  alignas(16) uint32_t most_v[D / 2][4];               // the largest |b v| of a value row, two rows' as bf16, of every warp that looked
  float whole;
};
struct Solve {                                         // of a preparing group
  uint8_t a_hi[6][512], a_lo[6][512];                  // -A below the diagonal, blocks (1,0) (2,0) (2,1) (3,0) .. of 16 rows of 32 bytes
  float diagonal[4][16 * 20];                          // its diagonal blocks
};
struct alignas(1024) ChunkSmem {
  Stage stage[STAGES];
  uint8_t s_hi[TILE], s_lo[TILE];                      // S [key][value]
  uint8_t x_hi[TILE], x_lo[TILE];                      // X, then e^(Gc - G) U, [token][value]
  uint8_t u[TILE];                                     // U, one term
  Solve solve[2];
  float power[2][D], inverse[2][D];                    // a value row's power of two, by turns: a chunk's is in use when the next one's is made
  unsigned long long bar_y, bar_u, bar_s, bar_o, bar_a[2], bar_p, bar_k[STAGES];
  uint32_t tmem, abort_flag;
};
static_assert(sizeof(Stage) % 1024 == 0, "tiles lie on 1024-byte boundaries");
constexpr size_t CHUNK_SMEM = sizeof(ChunkSmem) + 1024;

// tensor memory: accumulators of 64 columns; TM_CHAIN, the state's three products one after the other, has two
enum { TM_A = 0 /* + 64 group */, TM_CHAIN = 128, TM_QS = 256, TM_PU = 320, TM_P = 384, TM_COLUMNS = 512 };
// Columns of the thread's lane
#define JB_R8(x, i) "=&r"(x[i]), "=&r"(x[i + 1]), "=&r"(x[i + 2]), "=&r"(x[i + 3]), "=&r"(x[i + 4]), "=&r"(x[i + 5]), "=&r"(x[i + 6]), "=&r"(x[i + 7])
__device__ __forceinline__ void tmem_ld8(uint32_t at, float (&x)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : JB_R8(r, 0)
               : "r"(at)
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r[i]);
}
// 16 from a on and 16 from b on
__device__ __forceinline__ void tmem_ld16x2(uint32_t a, uint32_t b, float2 (&x)[8], float2 (&y)[8]) {
  uint32_t r[16], s[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : JB_R8(r, 0), JB_R8(r, 8), JB_R8(s, 0), JB_R8(s, 8)
      : "r"(a), "r"(b)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    y[i] = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
  }
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const float2 (&x)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "f"(x[0].x), "f"(x[0].y),
               "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y), "f"(x[3].x), "f"(x[3].y), "f"(x[4].x), "f"(x[4].y), "f"(x[5].x), "f"(x[5].y),
               "f"(x[6].x), "f"(x[6].y), "f"(x[7].x), "f"(x[7].y)
               : "memory");
}
// The CTA's barriers.  Ready and free of a stage: the preparing group arrives and waits, the others wait and arrive.
enum {
  BAR_GROUP = 1 /* + group */, BAR_STATE = 3, BAR_READY = 4 /* + stage */, BAR_FREE = 7 /* + stage */, BAR_TAKEN = 10, BAR_GIVEN = 11,
  BAR_PAIR = 12 /* + group */, BAR_SCORES = 14
};
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
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
// Two f32 at a time
__device__ __forceinline__ unsigned long long bits2(float2 x) { return (unsigned long long)(__float_as_uint(x.y)) << 32 | __float_as_uint(x.x); }
__device__ __forceinline__ float2 float2_of(unsigned long long x) { return make_float2(__uint_as_float(uint32_t(x)), __uint_as_float(uint32_t(x >> 32))); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
  return float2_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return float2_of(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits2(a)), "l"(bits2(b)));
  return float2_of(r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// (x, y) as two f16 terms each
__device__ __forceinline__ void split(float2 x, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16x2(x.x, x.y);
  const float2 rest = fma2(__half22float2(*reinterpret_cast<const __half2*>(&hi)), both(-1.f), x);
  lo = pack_f16x2(rest.x, rest.y);
}
__device__ __forceinline__ void split(float x, float y, uint32_t& hi, uint32_t& lo) { split(make_float2(x, y), hi, lo); }
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// A power of two s with s m in [2^14, 2^15) and its inverse; of m = 0, infinities and what is too small any that are finite
__device__ __forceinline__ void power_scale(float m, float& s, float& inv) {
  const int e = max(int(__float_as_uint(m) >> 23), 17);         // 255 at most: m is none below 0
  s = __uint_as_float(uint32_t(254 + 14 - e) << 23);
  inv = __uint_as_float(uint32_t(e - 14) << 23);
}
// Of four pairs of sizes a lane (bf16 or f16: they compare as integers, NaN above all) the largest over the lanes that differ in bits 4 and 3, pair
// (lane >> 3) & 3 for each
__device__ __forceinline__ uint32_t most_of_four(const uint32_t (&m)[4], int lane) {
  const bool up = lane & 16, up8 = lane & 8;
  const uint32_t a = __vmaxu2(up ? m[2] : m[0], __shfl_xor_sync(0xffffffffu, up ? m[0] : m[2], 16));
  const uint32_t b = __vmaxu2(up ? m[3] : m[1], __shfl_xor_sync(0xffffffffu, up ? m[1] : m[3], 16));
  return __vmaxu2(up8 ? b : a, __shfl_xor_sync(0xffffffffu, up8 ? a : b, 8));
}
__device__ __forceinline__ float inverse_power(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }      // of a power of two
__device__ __forceinline__ uint32_t unit_at(int row, int unit) { return uint32_t(row * 128 + ((unit ^ (row & 7)) << 4)); }

// Operands of tcgen05.mma in the 128-byte swizzle.  K-major (rows of the operand are rows of the tile): 16 elements on are +2 in the address field.
// MN-major (its rows are the tile's columns): 16 on are 16 rows, +128, and behind 64 columns those of the tile TWO_TILES away, or the same again.
enum { ONE_TILE = 64, SAME_TWICE = 0, TWO_TILES = TILE >> 4 };
__device__ __forceinline__ uint64_t operand(const uint8_t* tile, int next = ONE_TILE) {
  return uint64_t((smem_u32(tile) & 0x3FFFFu) >> 4) | uint64_t(next) << 16 | uint64_t(64) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
constexpr uint32_t idesc(int n, int a_mn, int b_mn) {  // f16 operands, f32 sums, 128 x n
  return (1u << 4) | uint32_t(a_mn) << 15 | uint32_t(b_mn) << 16 | uint32_t(n >> 3) << 17 | uint32_t(128 >> 4) << 24;
}
// By a whole warp, one lane of it issuing: 64 long
template <int N, int A_MN, int B_MN>
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, bool add) {
  asm volatile(
      "{\n\t"
      ".reg .pred one, more, all;\n\t"
      ".reg .b64 a, b;\n\t"
      "elect.sync _|one, 0xffffffff;\n\t"
      "setp.ne.b32 more, %4, 0;\n\t"
      "setp.eq.b32 all, 0, 0;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, more;\n\t"
      "add.u64 a, %1, %5;\n\t"
      "add.u64 b, %2, %6;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, all;\n\t"
      "add.u64 a, a, %5;\n\t"
      "add.u64 b, b, %6;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, all;\n\t"
      "add.u64 a, a, %5;\n\t"
      "add.u64 b, b, %6;\n\t"
      "@one tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, all;\n\t"
      "}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc(N, A_MN, B_MN)), "r"(add ? 1 : 0), "n"(A_MN ? 128 : 2), "n"(B_MN ? 128 : 2)
      : "memory");
}
__device__ __forceinline__ void commit(unsigned long long& bar) {
  if (elect_one()) umma_commit(smem_u32(&bar));
  __syncwarp();
}

// The tokens that a CTA takes: of sequence b from row `begin` (of the sequence) on, `chunks` chunks, none from `len` on.
struct Part {
  int b, h, begin, len, chunks;
};

// 16 bytes that are asked for here and not where they are used (an ordinary read-only load may be moved there, behind barriers and all), or zeros: in the same
// registers, since a choice behind the load would wait for it here
__device__ __forceinline__ uint4 load_now(const void* p, bool on) {
  uint4 x;
  asm volatile(
      "{\n\t"
      ".reg .pred on;\n\t"
      "setp.ne.b32 on, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\t"
      "mov.b32 %1, 0;\n\t"
      "mov.b32 %2, 0;\n\t"
      "mov.b32 %3, 0;\n\t"
      "@on ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n\t"
      "}"
      : "=&r"(x.x), "=&r"(x.y), "=&r"(x.z), "=&r"(x.w)
      : "l"(p), "r"(int(on))
      : "memory");
  return x;
}
__device__ __forceinline__ float load_now(const float* p) {
  float x;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(x) : "l"(p) : "memory");
  return x;
}

// Half a row of a bf16 matrix a thread: from memory ...
__device__ __forceinline__ void fetch_half(uint4 (&x)[4], const __nv_bfloat16* at, bool on) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = load_now(at + 8 * i, on);
}
// ... and to f16 in a tile (`twice`: and in the next one), times the power of two s that brings the row's norm into [1, 2), or near it where s or its
// inverse would leave f32 (2^126); returns the sum of squares after that.
__device__ __forceinline__ float convert_half(const uint4 (&x)[4], uint8_t* tile, bool twice, int row, int half, float& s) {
  float ss;
  auto squares = [&](float size) {                       // of the row times `size`; the power of two for their root
    float other = 0.f;
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = bf16_lo(in[j]) * size, b = bf16_hi(in[j]) * size;
        ss = fmaf(a, a, ss);
        other = fmaf(b, b, other);
      }
    }
    ss += other;
    ss += __shfl_xor_sync(0xffffffffu, ss, 1);
    const int e = (int(__float_as_uint(ss) >> 23) - 127) >> 1;                   // ss in [4^e, 4^(e + 1))
    return __uint_as_float(uint32_t(127 - e) << 23);
  };
  float t = squares(1.f);
  s = t;
  constexpr float LEAST = 8.2718061e-25f;                // 2^-80: below, squares of its addends may be subnormal
  if (__builtin_expect(__any_sync(0xffffffffu, ss == INFINITY || ss < LEAST), 0)) {
    const float size = ss == INFINITY ? SMALLER : ss < LEAST ? LARGER : 1.f;
    t = fminf(fmaxf(squares(size), 1.17549435e-38f / size), 8.5070592e37f / size);
    s = t * size;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = pack_f16x2(bf16_lo(in[j]) * s, bf16_hi(in[j]) * s);
    uint8_t* to = tile + unit_at(row, 4 * half + i);
    *reinterpret_cast<uint4*>(to) = make_uint4(out[0], out[1], out[2], out[3]);
    if (twice) *reinterpret_cast<uint4*>(to + TILE) = make_uint4(out[0], out[1], out[2], out[3]);
  }
  return ss * t * t;
}

struct Common {
  const DeltaParams& p;
  ChunkSmem& sm;
  Part part;
  int w, lane;
  uint32_t tm;                               // tensor memory, this warp's lanes
  unsigned int* status;

  // The waits are bounded; one that runs out leaves its code in the status word, and everybody carries on with what there is.
  __device__ __forceinline__ void wait(unsigned long long& bar, int n) const {
    if (!mbar_try_wait(smem_u32(&bar), uint32_t(n) & 1u)) wait_on(smem_u32(&bar), uint32_t(n) & 1u, &sm.abort_flag, status);
    tc_fence_after_sync();
  }
  // Eight columns of this thread's row of a product with K^T, c and the row's place in the chunk apart, times f r_j e^(G_i - G_j); g: G_i in two terms
  __device__ __forceinline__ void decayed(uint32_t columns, const Stage& st, int c, float2 g, float f, float (&x)[8]) const {
    tmem_ld8(tm + columns + c, x);
    const float4* col = reinterpret_cast<const float4*>(st.column + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 at = col[e];
      const float2 d = add2(add2(both(g.x), make_float2(at.x, at.z)), add2(both(g.y), make_float2(at.y, at.w)));
      const float2 v = mul2(mul2(make_float2(x[2 * e], x[2 * e + 1]), both(f)), make_float2(exp2_fast(d.x), exp2_fast(d.y)));
      x[2 * e] = v.x;
      x[2 * e + 1] = v.y;
    }
  }
  // 16 factors of value rows, two by two
  __device__ __forceinline__ static void factors(const float* at, float2 (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 x = reinterpret_cast<const float4*>(at)[e];
      f[2 * e] = make_float2(x.x, x.y);
      f[2 * e + 1] = make_float2(x.z, x.w);
    }
  }
  static __device__ __noinline__ void wait_on(uint32_t bar, uint32_t parity, uint32_t* abort_flag, unsigned int* status) {
    (void)mbar_wait(bar, parity, abort_flag, status, JB200_STATUS_ATTN_MMA);
  }
  // before a group's barrier: what was written is there for the tensor cores, what was read of tensor memory may be overwritten
  __device__ __forceinline__ static void settle() {
    fence_proxy_async_smem();
    tc_fence_before_sync();
  }
};

// ---- the preparing groups --------------------------------------------------------------------------------------------
template <bool OUT>
struct Prepare : Common {
  int group;
  bool factor;                               // v counts as 0

  // Running sums of log2 a, in f64 for differences of late tokens: of two tokens a lane
  struct Gates {
    float2 hi, lo, grow, of_u;
    float whole;
  };
  __device__ __forceinline__ Gates gates(float ga, float gb) const {
    double g0 = double(ga) * 1.4426950408889634, g1 = double(gb) * 1.4426950408889634;
    if (g0 < double(LEAST_LOG2)) g0 = double(LEAST_LOG2);
    if (g1 < double(LEAST_LOG2)) g1 = double(LEAST_LOG2);
    double sum = g0 + g1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const double end = __shfl_sync(0xffffffffu, sum, 31), before = sum - g1;
    Gates x;
    x.hi = make_float2(float(before), float(sum));
    x.lo = make_float2(float(before - double(x.hi.x)), float(sum - double(x.hi.y)));
    x.grow = make_float2(exp2f(x.hi.x), exp2f(x.hi.y));
    x.of_u = make_float2(exp2f(float(end - before)), exp2f(float(end - sum)));
    x.whole = exp2f(float(end));
    return x;
  }

  // Rows of -A: K K^T is there for two warps a row, which take half of its columns below the diagonal each
  __device__ __forceinline__ void rows_of_a(const Stage& st, Solve& so) const {
    const int i = 32 * (w & 1) + lane, ib = i >> 4, row = i & 15, units = 2 + 2 * (w & 1);
    const float n = st.nk[i], f = -st.beta[i] * n * n * st.rk[i];
    const float2 g = st.g[i];
#pragma unroll 1
    for (int c = (w >> 1) * units * 8, end = c + units * 8; c < end; c += 8) {
      float x[8];
      decayed(TM_A + 64 * group, st, c, g, f, x);
      const int jb = c >> 4, unit = (c >> 3) & 1;
      if (jb < ib) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split(x[2 * e], x[2 * e + 1], hi[e], lo[e]);
        const int at = (ib * (ib - 1) / 2 + jb) * 512 + row * 32 + ((unit ^ ((row >> 2) & 1)) << 4);
        *reinterpret_cast<uint4*>(so.a_hi[0] + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(so.a_lo[0] + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      } else if (jb == ib) {
        float* to = so.diagonal[ib] + row * 20 + 8 * unit;
        *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
      }
    }
  }

  // A diagonal block's inverse, a column of T (a row of T^T) a lane: t_i = -sum_(j < i) A_ij t_j below t_c = 1
  __device__ __forceinline__ void diagonal(Stage& st, const Solve& so) const {
    const float* dg = so.diagonal[w];
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
      t[i] = sum + other;                        // 0 for i < c: so is every t_j of the sum
    }
    if (lane < 16) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split(t[8 * u + 2 * e], t[8 * u + 2 * e + 1], hi[e], lo[e]);
        const uint32_t at = unit_at(16 * w + c, 2 * w + u);
        *reinterpret_cast<uint4*>(st.t_hi + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(st.t_lo + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
  }

  // Blocks of 16 x 16 by mma.sync.  Everything is transposed, so that a product's accumulators are the next one's first operand.
  struct Pair { uint32_t hi[4], lo[4]; };     // a first operand in two terms
  __device__ __forceinline__ Pair t_block(const Stage& st, int i, int j) const {      // T_ij^T
    Pair x;
    const uint32_t at = unit_at(16 * j + (((lane >> 3) & 1) << 3) + (lane & 7), 2 * i + (lane >> 4));
    ldm4(x.hi, smem_u32(st.t_hi) + at);
    ldm4(x.lo, smem_u32(st.t_lo) + at);
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
  // c += x (-A_il)^T, by rows i
  __device__ __forceinline__ void times_a(float (&c)[2][4], const Pair& x, const Solve& so, int i, int l) const {
    uint32_t hi[4], lo[4];
    const int row = ((lane >> 4) << 3) + (lane & 7), unit = (lane >> 3) & 1, block = i * (i - 1) / 2 + l;
    const uint32_t at = block * 512 + row * 32 + ((unit ^ ((row >> 2) & 1)) << 4);
    ldm4(hi, smem_u32(so.a_hi) + at);
    ldm4(lo, smem_u32(so.a_lo) + at);
    mma3(c, x, hi, lo);
  }
  // c += x T_il^T, T^T by rows l
  __device__ __forceinline__ void times_t(float (&c)[2][4], const Pair& x, const Stage& st, int i, int l) const {
    uint32_t hi[4], lo[4];
    const uint32_t at = unit_at(16 * l + (((lane >> 3) & 1) << 3) + (lane & 7), 2 * i + (lane >> 4));
    ldm4t(hi, smem_u32(st.t_hi) + at);
    ldm4t(lo, smem_u32(st.t_lo) + at);
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
  __device__ __forceinline__ void off_diagonal(Stage& st, const Solve& so) const {
    {
      float c[2][4];
      zero(c);
      times_a(c, t_block(st, 2 * w, 2 * w), so, 2 * w + 1, 2 * w);
      const Pair x = as_operand(c);
      zero(c);
      times_t(c, x, st, 2 * w + 1, 2 * w + 1);
      store_t(c, st, 2 * w + 1, 2 * w);
    }
    bar_sync(BAR_PAIR + group, GROUP / 2);
    {
      float m2[2][4], m3[2][4];
      zero(m2);
      zero(m3);
      for (int l = w; l < 2; ++l) {
        const Pair t = t_block(st, l, w);
        times_a(m2, t, so, 2, l);
        times_a(m3, t, so, 3, l);
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
    const __nv_bfloat16* qp = p.q + first * p.ldq + size_t(part.h / p.per_key) * D;
    Solve& so = sm.solve[group];
    const int tid = 32 * w + lane, row = tid >> 1, half = tid & 1;
    const __nv_bfloat16* vp = p.v + first * p.ldv + size_t(part.h) * D + 8 * (tid & 7);
    uint4 k[4], q[4];
    float g0 = 0.f, g1 = 0.f, b0 = 0.f, b1 = 0.f;
    auto fetch = [&](int t0) {
      const int at = t0 + row;
      fetch_half(k, kp + size_t(at) * p.ldk + 32 * half, at < part.len);
      if (OUT) fetch_half(q, qp + size_t(at) * p.ldq + 32 * half, at < part.len);
      if (w == 3) {
        const int t = t0 + 2 * lane;
        const float *gp = p.log_decay + (first + t) * p.ldg + part.h, *bp = p.beta + (first + t) * p.ldb + part.h;
        g0 = t < part.len ? load_now(gp) : 0.f;
        b0 = t < part.len ? load_now(bp) : 0.f;
        g1 = t + 1 < part.len ? load_now(gp + p.ldg) : 0.f;
        b1 = t + 1 < part.len ? load_now(bp + p.ldb) : 0.f;
      }
    };
    if (group < part.chunks) fetch(part.begin + group * CHUNK);
    for (int n = group; n < part.chunks; n += 2) {
      const int s = n % STAGES, t0 = part.begin + n * CHUNK;
      Stage& st = sm.stage[s];
      Gates x;
      if (w == 3) x = gates(g0, g1);
      uint4 v[4];                                // 16 bytes of four tokens, asked for here, so that they come while the stage gets free
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + 16 * i + (tid >> 3);
        v[i] = load_now(vp + size_t(t) * p.ldv, !factor && t < part.len);
      }
      if (n >= STAGES) bar_sync(BAR_FREE + s, GROUP + STATE + (OUT ? OUT_THREADS : 0));
      if (w == 3) {
        *reinterpret_cast<float2*>(st.beta + 2 * lane) = make_float2(b0, b1);
        *reinterpret_cast<float2*>(st.of_s + 2 * lane) = x.grow;
        *reinterpret_cast<float2*>(st.of_u + 2 * lane) = x.of_u;
        *reinterpret_cast<float4*>(&st.g[2 * lane]) = make_float4(x.hi.x, x.lo.x, x.hi.y, x.lo.y);
        if (lane == 0) st.whole = x.whole;
      }
#pragma unroll 1
      for (int m = 0; m < (OUT ? 2 : 1); ++m) {  // K twice, Q
        float sc;
        const float ss = convert_half(k, m == 0 ? st.k_again : st.q, m == 0, row, half, sc);
        if (half == 0) {
          // k = n (k16 r) with |k16 r| = 1, or of the normalised key n = 1 and k16 r its value
          const float inv = inverse_power(sc);
          const float r = !p.normalize ? ss > 0.f ? rsqrtf(ss) : 0.f : sc > 1e12f ? inv * 1e3f : rsqrtf(fmaf(NORM_EPS * sc, sc, ss));
          if (m == 0) {
            st.rk[row] = r;
            st.nk[row] = p.normalize ? 1.f : ss * r * inv;
          } else {
            st.of_o[row] = p.scale * (p.normalize ? r : inv);
          }
        }
        if (OUT) {
#pragma unroll
          for (int i = 0; i < 4; ++i) k[i] = q[i];
        }
      }
      if (n + 2 < part.chunks) fetch(t0 + 2 * CHUNK);
      settle();
      bar_sync(BAR_GROUP + group, GROUP);
      if (w == 0) {
        tc_fence_after_sync();
        product<64, 0, 0>(sm.tmem + TM_A + 64 * group, operand(st.k_again), operand(st.k), false);
        commit(sm.bar_a[group]);
      } else if (w >= 2) {                       // b v - b e^G r K S^T, its share of K^T U
        const int i = 32 * (w - 2) + lane;
        const float r = st.rk[i], n1 = st.nk[i], beta = st.beta[i];
        const float2 g = st.g[i];
        st.column[i] = make_float2(-g.x, __log2f(r) - g.y);
        st.of_v[i] = beta * n1;
        st.of_y[i] = beta * n1 * n1 * st.of_s[i] * r;
        st.of_u[i] *= r;
      }
      {                                          // rounded twice: less than the 130 for 129 of the bound
        uint32_t m[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = 16 * i + (tid >> 3);
          const __nv_bfloat162 f = __float2bfloat162_rn(st.beta[t] * st.nk[t]);
          const uint32_t in[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&in[j]), f);
            *reinterpret_cast<__nv_bfloat162*>(&m[j]) = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&m[j]), __habs2(y));
          }
        }
        st.most_v[4 * (tid & 7) + ((lane >> 3) & 3)][w] = most_of_four(m, lane);
      }
      bar_sync(BAR_GROUP + group, GROUP);
      if (lane == 0) mbar_arrive(smem_u32(&sm.bar_k[s]));
      wait(sm.bar_a[group], n >> 1);
      rows_of_a(st, so);
      bar_sync(BAR_GROUP + group, GROUP);
      diagonal(st, so);
      bar_sync(BAR_GROUP + group, GROUP);
      if (w < 2) off_diagonal(st, so);
      settle();
      bar_arrive(BAR_READY + s, GROUP + STATE + (OUT ? OUT_THREADS : 0));
    }
  }
};

// ---- P: a row a thread of two warps ----------------------------------------------------------------------------------------
struct Scores : Common {
  __device__ __forceinline__ void run() const {
    const int i = 32 * (w - 2) + lane, reach = 32 * (w - 1);
#pragma unroll 1
    for (int n = 0; n < part.chunks; ++n) {
      const int s = n % STAGES;
      Stage& st = sm.stage[s];
      wait(sm.bar_k[s], n / STAGES);             // the stage is free, K and Q are there
      bar_sync(BAR_SCORES, OUT_THREADS);         // both warps have read the chunk before
      if (w == 2) {
        tc_fence_after_sync();
        product<64, 0, 0>(sm.tmem + TM_P, operand(st.k), operand(st.k), false);
        commit(sm.bar_p);
      }
      st.of_s[i] *= st.of_o[i];
      const float2 g = st.g[i];
      wait(sm.bar_p, n);
#pragma unroll 1
      for (int c = 0; c < 64; c += 8) {
        uint32_t v[4] = {};
        if (c < reach) {
          float x[8];
          decayed(TM_P, st, c, g, 1.f, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = pack_f16x2(c + 2 * e <= i ? x[2 * e] : 0.f, c + 2 * e + 1 <= i ? x[2 * e + 1] : 0.f);
        }
        *reinterpret_cast<uint4*>(st.p + unit_at(i, c >> 3)) = make_uint4(v[0], v[1], v[2], v[3]);
      }
      settle();
      bar_arrive(BAR_READY + s, GROUP + STATE + OUT_THREADS);
    }
  }
};

// ---- the group of the state ------------------------------------------------------------------------------------------
template <bool OUT>
struct Follow : Common {
  // 16 values of a row in two terms, from unit `unit` on
  __device__ __forceinline__ static void put(const float2 (&x)[8], uint8_t* hi_tile, uint8_t* lo_tile, int row, int unit) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) split(x[4 * u + e], hi[e], lo[e]);
      const uint32_t at = unit_at(row, unit + u);
      *reinterpret_cast<uint4*>(hi_tile + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(lo_tile + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
  // The largest |S| of value row 32 (w & 1) + lane, times the row's power, by a warp for 32 of them: of its tile's upper terms
  __device__ __forceinline__ float largest_s() const {
    const int unit = 4 * (w & 1) + (lane & 3), at = (lane >> 3) | (lane & 4);      // the two rows that eight lanes read differ in the swizzle
    uint32_t m[4] = {};
#pragma unroll
    for (int i = 0; i < D; i += 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(sm.s_hi + unit_at(i + at, unit));
      const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) m[j] = __vmaxu2(m[j], in[j] & 0x7fff7fffu);
    }
    uint32_t most = most_of_four(m, lane);
    most = __vmaxu2(most, __shfl_xor_sync(0xffffffffu, most, 4));
    const int pair = lane >> 1;
    most = __shfl_sync(0xffffffffu, most, pair >> 2 | (pair & 3) << 3);
    const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&most));
    return (lane & 1 ? two.y : two.x) + 5.9604645e-8f;           // 2^-24: more than upper terms leave out
  }

  // Loops over a thread's 32 columns stay loops where registers allow: the roles of this kernel share the instruction caches, and with all products unrolled
  // (77 KB in all) every one of them waited for its instructions (a chunk took 9600 cycles on 128 SMs).  The one over X is open, since V, moved down
  // between its turns, would be waited for where it is asked for.
  // from `from` (null: 0) through the part's chunks to `to`; `factor`: from the identity, with v as 0, which gives what the part multiplies a state by
  __device__ __forceinline__ void run(const float* from, float* to, bool factor) const {
    const int row = 32 * (w & 1) + lane, half = w >> 1;          // a key (S) or a token (X, U), and which 32 values of it
    const uint32_t cols = tm + TM_CHAIN + 32 * half;
    const __nv_bfloat16* vp = p.v + size_t(part.b) * p.T * p.ldv + size_t(part.h) * D + 32 * half;
    uint4 v[4];
    float2 S[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int i = 32 * half + 2 * e;
      S[e] = from != nullptr ? make_float2(from[i * D + row], from[(i + 1) * D + row]) : make_float2(factor && i == row, factor && i + 1 == row);
    }
    const float2 none[8] = {};                                   // the product before the first chunk
#pragma unroll
    for (int c = 0; c < 128; c += 64) {
      tmem_st16(cols + c, none);
      tmem_st16(cols + c + 16, none);
    }
    tmem_st_wait();
    auto values = [&](int n) {                                   // of a chunk
      const int t = part.begin + n * CHUNK + row;
      fetch_half(v, vp + size_t(t) * p.ldv, !factor && t < part.len);
    };
    // two of the warps that issue no products have a value row a thread, whose powers they give
    const int v_row = threadIdx.x - 64;
    float bound = 0.f, most_v = 0.f, whole = 1.f;
    if (w >= 2) {
      float m = factor ? 1.f : 0.f;
      if (from != nullptr)
#pragma unroll
        for (int i = 0; i < D / 4; ++i) {
          const float4 x = reinterpret_cast<const float4*>(from + v_row * D)[i];
          m = fmaxf(fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
        }
      bound = 8.f * m;
      sm.power[0][v_row] = sm.inverse[1][v_row] = 1.f;           // where there are no chunks; of that product
    }
    auto powers = [&](int n) {                                   // of a chunk
      wait(sm.bar_k[n % STAGES], n / STAGES);                    // V has been looked at
      const uint4 of = *reinterpret_cast<const uint4*>(sm.stage[n % STAGES].most_v[v_row >> 1]);
      const uint32_t pair = __vmaxu2(__vmaxu2(of.x, of.y), __vmaxu2(of.z, of.w));
      most_v = v_row & 1 ? bf16_hi(pair) : bf16_lo(pair);
      power_scale(fmaf(2.f, bound, 130.f * most_v), sm.power[n & 1][v_row], sm.inverse[n & 1][v_row]);
    };
    if (part.chunks > 0) {
      values(0);
      if (w >= 2) powers(0);
    }
    bar_sync(BAR_STATE, STATE);
    for (int n = 0;; ++n) {
#pragma unroll
      for (int c = 0; c < 16; c += 8) {
        float2 x[8], y[8], f[8];
        factors(sm.inverse[(n + 1) & 1] + 32 * half + 2 * c, f);
        tmem_ld16x2(cols + 2 * c, cols + 64 + 2 * c, x, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) S[c + e] = fma2(add2(x[e], y[e]), f[e], mul2(S[c + e], both(whole)));
        factors(sm.power[n & 1] + 32 * half + 2 * c, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = mul2(S[c + e], f[e]);
        put(x, sm.s_hi, sm.s_lo, row, 4 * half + (c >> 2));
      }
      if (n == part.chunks) break;
      const int s = n % STAGES;
      Stage& st = sm.stage[s];
      bar_sync(BAR_READY + s, GROUP + STATE + (OUT ? OUT_THREADS : 0));
      settle();
      if (OUT && n > 0) bar_sync(BAR_TAKEN, STATE + OUT_THREADS);
      else bar_sync(BAR_STATE, STATE);
      if (w == 0) {
        tc_fence_after_sync();
        product<128, 0, 1>(sm.tmem + TM_CHAIN, operand(st.k_again), operand(sm.s_hi, TWO_TILES), false);
        commit(sm.bar_y);
        if (OUT) product<64, 0, 1>(sm.tmem + TM_QS, operand(st.q), operand(sm.s_hi), false);
        __syncwarp();
      }
      whole = st.whole;
      const float fv = st.of_v[row], fy = st.of_y[row], fu = st.of_u[row];
      wait(sm.bar_y, n);
#pragma unroll
      for (int c = 0; c < 32; c += 16) {
        float2 x[8], y[8], f[8];
        factors(sm.power[n & 1] + 32 * half + c, f);
        tmem_ld16x2(cols + c, cols + 64 + c, x, y);
        const uint4 a = v[c >> 3], b = v[(c >> 3) + 1];
        const uint32_t in[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = fma2(add2(x[e], y[e]), both(-fy), mul2(mul2(make_float2(bf16_lo(in[e]), bf16_hi(in[e])), both(fv)), f[e]));
        put(x, sm.x_hi, sm.x_lo, row, 4 * half + (c >> 3));
      }
      settle();
      bar_sync(BAR_STATE, STATE);
      if (w == 0) {
        tc_fence_after_sync();
        product<128, 1, 1>(sm.tmem + TM_CHAIN, operand(st.t_hi, SAME_TWICE), operand(sm.x_hi, TWO_TILES), false);
        product<64, 1, 1>(sm.tmem + TM_CHAIN, operand(st.t_lo, SAME_TWICE), operand(sm.x_hi), true);
        commit(sm.bar_u);
      }
      if (n + 1 < part.chunks) {
        values(n + 1);
        if (w >= 2) {
          if ((n & 3) == 3) bound = fminf(bound, 8.1f * largest_s() * sm.inverse[n & 1][v_row]);
          bound = fmaf(1.65f * whole, bound, 64.5f * most_v);
          powers(n + 1);
        }
      }
      wait(sm.bar_u, n);
#pragma unroll 1
      for (int c = 0; c < 32; c += 16) {
        float2 x[8], y[8];
        tmem_ld16x2(cols + c, cols + 64 + c, x, y);
        uint32_t one[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = add2(x[e], y[e]);
          one[e] = pack_f16x2(x[e].x, x[e].y);
          x[e] = mul2(x[e], both(fu));
        }
        if (OUT) {
          *reinterpret_cast<uint4*>(sm.u + unit_at(row, 4 * half + (c >> 3))) = make_uint4(one[0], one[1], one[2], one[3]);
          *reinterpret_cast<uint4*>(sm.u + unit_at(row, 4 * half + (c >> 3) + 1)) = make_uint4(one[4], one[5], one[6], one[7]);
        }
        put(x, sm.x_hi, sm.x_lo, row, 4 * half + (c >> 3));
      }
      settle();
      bar_sync(BAR_STATE, STATE);
      if (OUT) bar_arrive(BAR_GIVEN, STATE + OUT_THREADS);
      if (w == 0) {
        tc_fence_after_sync();
        product<128, 1, 1>(sm.tmem + TM_CHAIN, operand(st.k, SAME_TWICE), operand(sm.x_hi, TWO_TILES), false);
        commit(sm.bar_s);
        if (OUT) {
          product<64, 0, 1>(sm.tmem + TM_PU, operand(st.p), operand(sm.u), false);
          commit(sm.bar_o);
        }
      }
      wait(sm.bar_s, n);                         // the outputs' group waits for P U before it frees the stage as well
      if (n + STAGES < part.chunks) bar_arrive(BAR_FREE + s, GROUP + STATE + (OUT ? OUT_THREADS : 0));
    }
    if (to != nullptr) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        to[(32 * half + 2 * e) * D + row] = S[e].x;
        to[(32 * half + 2 * e + 1) * D + row] = S[e].y;
      }
    }
  }
};

// ---- the outputs: a token a thread of two warps --------------------------------------------------------------------------
struct Outputs : Common {
  __device__ __forceinline__ void run() const {
    __nv_bfloat16* op = p.o + size_t(part.b) * p.T * p.ldo + size_t(part.h) * D;
    const int row = 32 * w + lane;
#pragma unroll 1
    for (int n = 0; n < part.chunks; ++n) {
      const int s = n % STAGES, t = part.begin + n * CHUNK + row;
      const Stage& st = sm.stage[s];
      bar_sync(BAR_GIVEN, STATE + OUT_THREADS);
      const float fs = st.of_s[row], fu = st.of_o[row];
      wait(sm.bar_o, n);
      if (n + STAGES < part.chunks) bar_arrive(BAR_FREE + s, GROUP + STATE + OUT_THREADS);
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        float2 a[8], b[8], f[8];
        factors(sm.inverse[n & 1] + c, f);
        tmem_ld16x2(tm + TM_QS + c, tm + TM_PU + c, a, b);
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          a[e] = mul2(fma2(b[e], both(fu), mul2(a[e], both(fs))), f[e]);
          x[e] = pack_bf16x2(a[e].x, a[e].y);
        }
        if (t < part.len) {
          uint4* to = reinterpret_cast<uint4*>(op + size_t(t) * p.ldo + c);
          to[0] = make_uint4(x[0], x[1], x[2], x[3]);
          to[1] = make_uint4(x[4], x[5], x[6], x[7]);
        }
      }
      tc_fence_before_sync();
      if (n + 1 < part.chunks) bar_arrive(BAR_TAKEN, STATE + OUT_THREADS);
    }
    const int last = part.begin + part.chunks * CHUNK, t = last - CHUNK + row, end = min(p.T, part.begin + p.seg_chunks * CHUNK);
    if (part.chunks > 0 && t >= part.len && t < end) zero_row(op, t);
    for (int i = last + row; i < end; i += OUT_THREADS) zero_row(op, i);
  }
  __device__ __forceinline__ void zero_row(__nv_bfloat16* op, int t) const {
#pragma unroll 1
    for (int u = 0; u < 8; ++u) *(reinterpret_cast<uint4*>(op + size_t(t) * p.ldo) + u) = make_uint4(0, 0, 0, 0);
  }
};

template <bool OUT>
__global__ void __launch_bounds__(3 * GROUP + (OUT ? 2 * OUT_THREADS : 0), 1) delta_chunk_kernel(DeltaParams p, unsigned int* status) {
  extern __shared__ uint8_t smem_raw[];
  ChunkSmem& sm = *reinterpret_cast<ChunkSmem*>(smem_raw + (1024u - (smem_u32(smem_raw) & 1023u)) % 1024u);
  const int warp = warp_index(), lane = threadIdx.x & 31, w = warp & 3;
  if (warp == 0) {
    tmem_alloc(smem_u32(&sm.tmem), TM_COLUMNS);
    tmem_relinquish();
    if (lane == 0) {
      mbar_init(smem_u32(&sm.bar_y), 1);
      mbar_init(smem_u32(&sm.bar_u), 1);
      mbar_init(smem_u32(&sm.bar_s), 1);
      mbar_init(smem_u32(&sm.bar_o), 1);
      mbar_init(smem_u32(&sm.bar_a[0]), 1);
      mbar_init(smem_u32(&sm.bar_a[1]), 1);
      mbar_init(smem_u32(&sm.bar_p), 1);
      for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&sm.bar_k[s]), GROUP / 32);
      sm.abort_flag = 0;
      fence_mbar_init();
    }
  }
  for (int s = 0; s < STAGES; ++s)             // T^T: what lies below the blocks of the diagonal stays 0
    for (int i = threadIdx.x; i < 2 * TILE / 16; i += blockDim.x) reinterpret_cast<uint4*>(sm.stage[s].t_hi)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // A CTA a segment; of the pieces one for the first segment, which starts from the state that is given, two for each of the others
  const int ctas = p.what == PIECES ? 2 * p.segments - 3 : p.what == LAST ? 1 : p.segments, bh = blockIdx.x / ctas, j = blockIdx.x % ctas;
  const bool factor = p.what == PIECES && j > 0 && (j & 1) == 0;
  const int segment = p.what == PIECES ? (j + 1) >> 1 : p.what == LAST ? p.segments - 1 : j;
  Part part;
  part.b = bh / p.H;
  part.h = bh % p.H;
  part.begin = segment * p.seg_chunks * CHUNK;
  pdl_wait();
  pdl_trigger();
  part.len = min(sequence_length(p, part.b), part.begin + p.seg_chunks * CHUNK);
  part.chunks = part.len > part.begin ? (part.len - part.begin + CHUNK - 1) / CHUNK : 0;
  const float* from = p.s_in == nullptr ? nullptr : p.s_in + size_t(bh) * D * D;
  float* to = p.s_out == nullptr ? nullptr : p.s_out + size_t(bh) * D * D;
  if (p.what == PIECES) {
    if (segment > 0) from = nullptr;
    to = p.pieces + piece_at(p.segments, bh, (factor ? p.segments - 1 : 0) + segment);
  } else if (p.segments > 1) {
    if (segment > 0) from = p.pieces + piece_at(p.segments, bh, segment - 1);
    else if (p.s_in == p.s_out && p.s_in != nullptr) from = p.pieces + piece_at(p.segments, bh, 2 * p.segments - 2);
    if (segment + 1 < p.segments) to = nullptr;
  }
  const Common common{p, sm, part, w, lane, sm.tmem + (uint32_t(w) << 21), status};
  if (warp < 4) {
    Follow<OUT>{common}.run(from, to, factor);
  } else if (warp < 12) {
    Prepare<OUT>{common, (warp >> 2) - 1, factor}.run();
  } else if (OUT) {
    if (warp < 14) Outputs{common}.run();
    else Scores{common}.run();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(sm.tmem, TM_COLUMNS);
  }
}

// The state before every segment from what the segments add and multiply by: S_(s+1) = S_s M_s + N_s.  Eight value rows a CTA.  A chain of products
// of 8 x 64 x 64, each of them short: the next three M are on their way into shared memory meanwhile (read where they are needed, a segment took 4 us).
constexpr int JOIN_STAGES = 4;
constexpr int JOIN_SMEM = JOIN_STAGES * D * D * 4;
__global__ void __launch_bounds__(128) delta_join_kernel(DeltaParams p) {
  extern __shared__ __align__(16) float join_m[];
  __shared__ __align__(16) float rows[2][8][D];
  const int bh = blockIdx.x >> 3, r = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4, v = (blockIdx.x & 7) * 8 + r;
  pdl_wait();
  pdl_trigger();
  auto fetch = [&](int s) {
    if (s + 1 < p.segments) {
      const float* m = p.pieces + piece_at(p.segments, bh, p.segments - 1 + s);
      const uint32_t to = smem_u32(join_m + (s % JOIN_STAGES) * D * D);
#pragma unroll
      for (int i = 0; i < D * D / 4 / 128; ++i) copy_async_16(to + (i * 128 + threadIdx.x) * 16, m + (i * 128 + threadIdx.x) * 4);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto added = [&](int s) { return reinterpret_cast<float4*>(p.pieces + piece_at(p.segments, bh, s) + v * D + c); };
  for (int s = 1; s < JOIN_STAGES; ++s) fetch(s);
  if (p.s_in == p.s_out && p.s_in != nullptr)        // the last segment may write it before the first one has read it
    *reinterpret_cast<float4*>(p.pieces + piece_at(p.segments, bh, 2 * p.segments - 2) + v * D + c) =
        *reinterpret_cast<const float4*>(p.s_in + size_t(bh) * D * D + v * D + c);
  *reinterpret_cast<float4*>(&rows[0][r][c]) = *added(0);
  float4 next = *added(1);                           // three segments or more
  for (int s = 1; s + 1 < p.segments; ++s) {
    float4 sum = next;
    if (s + 2 < p.segments) next = *added(s + 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(JOIN_STAGES - 2) : "memory");
    __syncthreads();                                 // everybody's part of M_s is there, and nobody reads M_(s-1)
    fetch(s + JOIN_STAGES - 1);
    const float* m = join_m + (s % JOIN_STAGES) * D * D + c;
    const float* row = rows[(s + 1) & 1][r];
#pragma unroll 16
    for (int k = 0; k < D; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(m + k * D);
      const float f = row[k];
      sum.x = fmaf(f, x.x, sum.x);
      sum.y = fmaf(f, x.y, sum.y);
      sum.z = fmaf(f, x.z, sum.z);
      sum.w = fmaf(f, x.w, sum.w);
    }
    *reinterpret_cast<float4*>(&rows[s & 1][r][c]) = sum;
    *added(s) = sum;
  }
}

// In chunks from so many tokens on.  A chunk's pass takes as long for one token as for 64, a token's step the longer the more heads there are.  us
// from cold token by token / in chunks: 16 heads, 8 tokens 12.3 / 12.3, 16 tokens 18.5 / 12.3; 256 heads, 8 tokens 16.4 / 22.5, 16 tokens 24.6 / 22.5;
// 304 heads, 24 tokens 30.7 / 30.8, 32 tokens 38.9 / 31.2; 1024 heads, 24 tokens 63.5 / 69.6, 32 tokens 79.9 / 71.7.
int chunk_tokens(int heads) { return heads < 2 * sm_count() ? 12 : 28; }

// Segments of a sequence where sequences and heads alone leave SMs idle.  In chunks' time, about 3 us: a pass over the tokens costs its chunks, and one
// to fill the pipeline, on as many waves of CTAs as it has (1 CTA an SM); the pieces' pass has 2 n - 3 CTAs a head for the outputs' n; the join takes 1
// and a quarter a segment.  The smaller sum wins, segments only by a tenth.  16 heads, us whole / in segments: 512 tokens 37 / 33 (not taken), 1024
// 63 / 43, 4096 217 / 89, 16384 839 / 269; 2 sequences of 2048 115 / 83; with 4 sequences of 2048 there is nothing to gain.
int segments_of(int B, int T, int H, long long sms) {
  const long long heads = (long long)B * H, chunks = (T + CHUNK - 1) / CHUNK;
  auto waves = [&](long long ctas) { return (ctas + sms - 1) / sms; };
  const double whole = double(waves(heads) * chunks);
  double least = 0.9 * whole;
  int best = 1;
  for (int n = 3; n <= 32 && heads * n <= 2 * sms; ++n) {
    const long long part = (chunks + n - 1) / n;
    if ((chunks + part - 1) / part != n) continue;             // the last ones would be empty
    const double cost = (double(part) + 1.0) * double(waves(heads * (2 * n - 3)) + waves(heads * n)) + 1.0 + 0.25 * n;
    if (cost < least) { least = cost; best = n; }
  }
  return best;
}

}  // namespace

size_t delta_plan_host(int B, int T, int H, int sms, int32_t* out2) {
  const bool any = B >= 1 && H >= 1 && T >= 1;
  const int n = any ? segments_of(B, T, H, sms) : 1, chunks = any ? (T + CHUNK - 1) / CHUNK : 0;
  if (out2 != nullptr) {
    out2[0] = n;
    out2[1] = (chunks + n - 1) / n;
  }
  return n == 1 ? 0 : piece_at(n, B * H, 0) * sizeof(float);
}

size_t gated_delta_scratch_bytes(int B, int T, int H) { return delta_plan_host(B, T, H, sm_count(), nullptr); }

int launch_gated_delta(const jb200_delta* d, void* scratch, cudaStream_t stream) {
  JB_REQUIRE(d != nullptr, "gated_delta: null pointer");
  const int B = d->B, T = d->T, H = d->H, KH = d->key_heads;
  JB_REQUIRE(B >= 0 && T >= 0 && H >= 1 && KH >= 1 && H % KH == 0, "gated_delta: bad shape (B=%d, T=%d, H=%d, key heads=%d)", B, T, H, KH);
  JB_REQUIRE(d->head_dim == D, "gated_delta: head_dim must be 64 (got %d)", d->head_dim);
  JB_REQUIRE((long long)B * H <= 0x1fffffff && (long long)B * T <= 0x7fffffff && T <= 1 << 30,
             "gated_delta: too many heads or tokens");
  if (B == 0) return JB200_OK;
  JB_REQUIRE(d->o != nullptr || d->s_out != nullptr, "gated_delta: neither an output nor a final state is asked for");
  JB_REQUIRE(T == 0 || (d->q && d->k && d->v && d->log_decay && d->beta), "gated_delta: null pointer");
  JB_REQUIRE(d->ldq >= KH * D && d->ldk >= KH * D && d->ldv >= H * D && d->ldg >= H && (d->ldb == 0 || d->ldb >= H) && (d->o == nullptr || d->ldo >= H * D),
             "gated_delta: row strides are smaller than the rows");
  JB_REQUIRE(aligned16(d->q) && aligned16(d->k) && aligned16(d->v) && aligned16(d->o) && aligned16(d->s_in) && aligned16(d->s_out) &&
                 d->ldq % 8 == 0 && d->ldk % 8 == 0 && d->ldv % 8 == 0 && (d->o == nullptr || d->ldo % 8 == 0),
             "gated_delta: q, k, v, o and the states must be 16-byte aligned, their row strides multiples of 8");
  DeltaParams p;
  p.q = static_cast<const __nv_bfloat16*>(d->q);
  p.k = static_cast<const __nv_bfloat16*>(d->k);
  p.v = static_cast<const __nv_bfloat16*>(d->v);
  p.ldq = d->ldq; p.ldk = d->ldk; p.ldv = d->ldv; p.ldo = d->ldo; p.ldg = d->ldg; p.ldb = d->ldb != 0 ? d->ldb : d->ldg;
  p.log_decay = d->log_decay; p.beta = d->beta; p.lengths = d->lengths; p.s_in = d->s_in; p.s_out = d->s_out;
  p.o = static_cast<__nv_bfloat16*>(d->o);
  p.B = B; p.T = T; p.H = H; p.per_key = H / KH;
  p.scale = d->scale; p.normalize = d->flags & JB200_DELTA_NORMALIZE;
  p.segments = 1;
  p.what = ALL;
  p.seg_chunks = (T + CHUNK - 1) / CHUNK;
  p.pieces = static_cast<float*>(scratch);
  if (T >= chunk_tokens(B * H)) {
    JB_MAX_SMEM(delta_chunk_kernel<true>, CHUNK_SMEM);
    JB_MAX_SMEM(delta_chunk_kernel<false>, CHUNK_SMEM);
    if (scratch != nullptr) {
      const int n = segments_of(B, T, H, sm_count());
      JB_REQUIRE(aligned16(scratch), "gated_delta: scratch must be 16-byte aligned");
      if (n > 1) {
        p.segments = n;
        p.seg_chunks = (p.seg_chunks + n - 1) / n;
        p.what = PIECES;
        launch_dep(delta_chunk_kernel<false>, B * H * (2 * n - 3), STATE + 2 * GROUP, CHUNK_SMEM, stream, p, device_status_ptr());
        JB_LAUNCH_CHECK("delta_chunk_kernel");
        JB_MAX_SMEM(delta_join_kernel, JOIN_SMEM);
        launch_dep(delta_join_kernel, B * H * 8, 128, JOIN_SMEM, stream, p);
        JB_LAUNCH_CHECK("delta_join_kernel");
        p.what = p.o != nullptr ? ALL : LAST;
      }
    }
    if (p.o != nullptr)
      launch_dep(delta_chunk_kernel<true>, B * H * p.segments, STATE + 2 * GROUP + 2 * OUT_THREADS, CHUNK_SMEM, stream, p, device_status_ptr());
    else
      launch_dep(delta_chunk_kernel<false>, B * H, STATE + 2 * GROUP, CHUNK_SMEM, stream, p, device_status_ptr());
    JB_LAUNCH_CHECK("delta_chunk_kernel");
    return JB200_OK;
  }
  // rows a lane: one for few heads (16: 6.5 us for a token, with four 8.0; 256: 8.2 and 8.6), four for many (304: 8.3, with one 9.8; 4096: 28 and 42)
  if (B * H < 2 * sm_count())
    launch_dep(delta_step_kernel<1>, B * H * 4, 128, 0, stream, p);
  else
    launch_dep(delta_step_kernel<4>, B * H, 128, 0, stream, p);
  JB_LAUNCH_CHECK("delta_step_kernel");
  return JB200_OK;
}

}  // namespace jb

// Next token of every row with settings of its own, over the whole vocabulary: temperature, then top-k, top-p and min-p, each a cut of the
// descending order of the logits, then one draw from what is left.  Where sampling.cu (sample_next_token,
// jarvis_engine/evaluate_jarvis.py:158-185) sorts up to 2048 survivors of a top-k, nothing is sorted here and there need not be a top-k.
//
//   order:  logits descending, equal ones by the lower id;  w_i = exp((x_i - x_max) / T)
//   top-k:  x_i >= the k-th largest (ties stay)
//   top-p:  the sum of w before i <= top_p times the sum over what top-k left; the first token always stays
//   min-p:  w_i >= min_p
//   draw:   the first i whose running sum over what is left exceeds u times the whole
//
// All of them ask "which token covers position z of the running sum", top-k with every weight 1.  Weights are taken in f64 and held as integers of
// 2^-45 of the largest one's (of 2^-(63 - log2 V) beyond 2^18 tokens), so that sums do not depend on the order of the atomics that form them.  Each is
// off by up to half a step, and what is below that is none: a border of the running sum lies up to V / 2 steps off, 7e-10 of the largest weight for 50257
// tokens, 1.5e-5 for 2^24, and a token that the exact sums choose is missed only where u is that near to one.  A cluster of CTAs has a row, a slice
// each (in shared memory where it fits), with as many CTAs as keep the SMs busy.  A histogram of the sums (for top-k of the counts) over 2048 bins of
// 1/64 of an e-fold finds the bin that covers z.  The tokens of a bin, up to 256, are ranked by comparison with one another; where there are more they are first cut into 512 parts of their order,
// logit then id, until there are not.  What top-k or min-p leaves is listed before it is weighed (and up to 256 ranked at once); where they leave
// everything, the few tokens near the largest are as the sums are taken: most answers are then found without the slices.  Every CTA counts and lists
// its slice in its own memory by atomics.  Behind a meeting each adds up a part of the bins over all CTAs and stores it in the first one's memory
// (plain stores, another meeting follows); the first one searches, the others read what it found.
//
// Bounds: a row alone, the chain of passes, barriers and searches (50257 tokens, nucleus: 18 to 27 us, by where the answer lies); many rows, reading
// them once and again from L2 (256 rows of 50257 f32, min-p: 20 us, the first reading alone 7.8); with a nucleus or the temperature alone over
// everything, the 11 f64 operations and the atomics of every token's weight (256 rows of f32: 103 and 86 us; 64 rows of bf16, every setting of its own:
// 37 to 40).
#include <cooperative_groups.h>

#include "common.cuh"
#include "launchers.h"

namespace jb {

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512;
constexpr int BINS = 2048;              // 1/64 of an e-fold each; the last: all that is some 32 e-folds (2^46) below the largest, whose weight is 0
constexpr float BINS_A_FOLD = 64.f;
constexpr int FINE = 512;
constexpr int LIST = 256;
constexpr int NEAR = 448, NEAR_LIST = 1024;  // bins whose tokens are listed at once (7 e-folds), as long as there are no more than that in a slice
constexpr int TABLE = 64;               // 2^-(j / 64)

struct Sampling {
  const void* logits;
  size_t ld;
  int V, ids, shift, staged;            // bits of an id; weights are multiples of 2^-shift; slices are kept in shared memory
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* token;
  float* prob;
};

struct Item {
  u64 place;                            // what the order goes by, larger first: the logit's key, then the id from the end
  u64 w;
};

// What the first CTA wants of all: the tokens of a bin with places from..to, in parts of 2^cut places (LISTED: the tokens themselves; DONE: nothing more)
struct Command {
  int bin, cut;
  u64 from, to;
};
constexpr int LISTED = -1, DONE = -2;

struct Smem {
  uint32_t count[BINS], lo[BINS], hi[BINS];       // then, as running sums before every bin: count, (lo, hi)
  uint32_t fcount[FINE], flo[FINE], fhi[FINE];
  Item list[LIST];
  u64 near[NEAR_LIST];
  u64 warp_sum[THREADS / 32], warp_ok[THREADS / 32];
  uint32_t warp_count[THREADS / 32];
  uint32_t best, best_id;                         // the largest: key, ~id
  uint32_t n, n_near;
  int listed, kept;                               // tokens of the bins below this are in `near`; how many a filter left
  Command command[2];                             // taken in turn, so that one can be written while the other is read
  int bin;
  u64 place, above, weight;                       // what a search leaves: the token that covers z, the sum before it, its weight
  u64 sum;
  double table[TABLE];
};

// order-preserving map float -> uint32; NaN is treated as -inf, -0 as 0
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

template <typename T>
__device__ __forceinline__ float widen(T x) { return x; }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }

// A CTA's slice of a row: vectors of 16 bytes, every CTAS-th THREADS of them, and the elements before and behind them that are not aligned
template <typename T, int CTAS>
struct Slice {
  static constexpr int PER = 16 / sizeof(T);
  const T* row;
  uint4* stage;                         // null: read again
  int V, rank, head, vectors;

  __device__ __forceinline__ Slice(const T* row, int V, int rank, uint4* stage) : row(row), stage(stage), V(V), rank(rank) {
    head = min(V, int((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / int(sizeof(T)));
    vectors = (V - head) / PER;
  }
  static __device__ __forceinline__ float largest(const uint4& x) {       // NaN only where all are
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&x);
      const __nv_bfloat162 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)), fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
    }
  }
  // the largest of this thread's elements, which go into the stage on the way
  __device__ __forceinline__ float peak() const {
    const int tail = head + vectors * PER;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    float top = -INFINITY;
    uint4* staged = stage + threadIdx.x;
#pragma unroll 4
    for (int i = rank * THREADS + threadIdx.x; i < vectors; i += CTAS * THREADS, staged += THREADS) {
      const uint4 x = __ldg(body + i);
      if (stage != nullptr) *staged = x;
      top = fmaxf(top, largest(x));
    }
    if (rank == 0 && int(threadIdx.x) < head) top = fmaxf(top, widen(row[threadIdx.x]));
    if (rank == CTAS - 1 && tail + int(threadIdx.x) < V) top = fmaxf(top, widen(row[tail + threadIdx.x]));
    return top;
  }
  // f(id, values, n) for four neighbours at a time, so that their chains of arithmetic overlap, without those that are all below `lowest`.  Elements
  // that are not aligned come one by one (n 1), with -infinities behind them.  Not unrolled further: a CTA runs most instructions for the first time,
  // and fetching them is what a row alone waits for (50257 tokens, nucleus: two vectors a turn took 49 us where one took 27).
  template <typename F>
  __device__ __forceinline__ void fours(float lowest, F&& f) const {
    const int tail = head + vectors * PER;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    auto four = [&](int id, int n, float a, float b, float c, float d) {
      if (fmaxf(fmaxf(a, b), fmaxf(c, d)) < lowest) return;
      const float x[4] = {a, b, c, d};
      f(id, x, n);
    };
    const uint4* staged = stage + threadIdx.x;
#pragma unroll 1
    for (int i = rank * THREADS + threadIdx.x; i < vectors; i += CTAS * THREADS, staged += THREADS) {
      const uint4 x = stage == nullptr ? __ldg(body + i) : *staged;
      const int id = head + i * PER;
      if constexpr (sizeof(T) == 2) {
        four(id, 4, bf16_lo(x.x), bf16_hi(x.x), bf16_lo(x.y), bf16_hi(x.y));
        four(id + 4, 4, bf16_lo(x.z), bf16_hi(x.z), bf16_lo(x.w), bf16_hi(x.w));
      } else {
        four(id, 4, __uint_as_float(x.x), __uint_as_float(x.y), __uint_as_float(x.z), __uint_as_float(x.w));
      }
    }
    if (rank == 0 && int(threadIdx.x) < head) four(int(threadIdx.x), 1, widen(row[threadIdx.x]), -INFINITY, -INFINITY, -INFINITY);
    if (rank == CTAS - 1 && tail + int(threadIdx.x) < V) four(tail + int(threadIdx.x), 1, widen(row[tail + threadIdx.x]), -INFINITY, -INFINITY, -INFINITY);
  }
};

// All CTAs of the row, with what they wrote
template <int CTAS>
__device__ __forceinline__ void meet() {
  if constexpr (CTAS == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// This CTA's memory
__device__ __forceinline__ Smem& own_smem() {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  return *reinterpret_cast<Smem*>(smem_raw);
}

// x as f64 (a subnormal x as some other number of 1e-38: no weight shows it); the conversion instruction runs at an eighth of this one's rate
__device__ __forceinline__ double to_f64(float x) {
  const uint32_t b = __float_as_uint(x), m = b & 0x7fffffffu;
  return __hiloint2double(int((b & 0x80000000u) | ((m >> 3) + 0x38000000u)), int(m << 29));
}

// Place in the order of a row: `ids` bits of the id from the end behind the logit's key, of which bf16 has 16 bits
template <typename T>
__device__ __forceinline__ u64 place_of(uint32_t key, int id, int ids) {
  return (u64(sizeof(T) == 2 ? key >> 16 : key) << ids) + ((1u << ids) - 1u - uint32_t(id));
}
template <typename T>
__device__ __forceinline__ int id_at(u64 place, int ids) { return int((1u << ids) - 1u - (uint32_t(place) & ((1u << ids) - 1u))); }
template <typename T>
__device__ __forceinline__ uint32_t key_at(u64 place, int ids) {
  const uint32_t key = uint32_t(place >> ids);
  return sizeof(T) == 4 ? key : key & 0x8000u ? key << 16 : key << 16 | 0xffffu;
}

struct Row {
  float top, fold;                      // the largest logit; bins an e-fold of the row's temperature
  double top64, rate;                   // 64 log2(e) / temperature
  int shift;
  const double* table;

  __device__ __forceinline__ int bin(float x) const {
    const float d = x == top ? 0.f : (top - x) * fold;
    return d < float(BINS - 1) ? int(d) : BINS - 1;            // NaN and infinities are the last bin's
  }
  // a value that none of the bins up to b goes below; an infinite largest has bin 0 for itself, and all others have the last
  __device__ __forceinline__ float below(int b) const {
    if (top == INFINITY && b < BINS - 1) return top;
    const float hi = float(b + 1) / fold;
    return b >= BINS - 1 ? -INFINITY : top - hi - 2e-6f * (fabsf(top) + hi);
  }
  // 2^shift exp((x - top) / temperature) as a double, of an x of any bin but the last: 2^-(n / 64) from the table, the rest from its series (the fifth
  // term is below 2^-44)
  __device__ __forceinline__ double scaled(float x) const {
    if (x == top) return __hiloint2double((1023 + shift) << 20, 0);
    constexpr double C1 = -0.6931471805599453 / 64, C2 = C1 * C1 / 2, C3 = C1 * C1 * C1 / 6, C4 = C1 * C1 * C1 * C1 / 24, MAGIC = 6755399441055744.0;
    const double t = (top64 - to_f64(x)) * rate, m = t + MAGIC, r = t - (m - MAGIC);
    const int n = __double2loint(m);
    const double w = fma(r, fma(r, fma(r, fma(r, C4, C3), C2), C1), 1.0) * table[n & (TABLE - 1)];
    const int hi = __double2hiint(w) + ((shift - (n >> 6)) << 20);
    return __hiloint2double(hi, __double2loint(w));
  }
  __device__ __forceinline__ u64 weight(float x) const {       // to the nearest integer: below 2^52 that is what the sum with 2^52 leaves
    return bin(x) == BINS - 1 ? 0 : __double_as_longlong(scaled(x) + 4503599627370496.0) & 0xfffffffffffffull;
  }
};

__device__ __forceinline__ void add64(uint32_t* lo, uint32_t* hi, u64 w) {
  const uint32_t a = uint32_t(w), before = atomicAdd(lo, a);
  const uint32_t up = uint32_t(w >> 32) + (before + a < before ? 1u : 0u);
  if (up) atomicAdd(hi, up);
}

// Running sums before each bin in place, neighbouring ones with a thread; returns the count of all.
template <int N_BINS>
__device__ __forceinline__ uint32_t running_sums(u64 sum0, uint32_t count0) {
  Smem& sm = own_smem();
  uint32_t* const count = N_BINS == BINS ? sm.count : sm.fcount;
  uint32_t* const lo = N_BINS == BINS ? sm.lo : sm.flo;
  uint32_t* const hi = N_BINS == BINS ? sm.hi : sm.fhi;
  constexpr int PER = N_BINS >= THREADS ? N_BINS / THREADS : 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool on = tid * PER < N_BINS;
  u64 s[PER], mine = 0;
  uint32_t c[PER], cnt = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    s[i] = on ? (u64(hi[tid * PER + i]) << 32) + lo[tid * PER + i] : 0;
    c[i] = on ? count[tid * PER + i] : 0;
    mine += s[i];
    cnt += c[i];
  }
  u64 incl = mine;
  uint32_t cincl = cnt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 a = __shfl_up_sync(0xffffffffu, incl, o);
    const uint32_t b = __shfl_up_sync(0xffffffffu, cincl, o);
    if (lane >= o) { incl += a; cincl += b; }
  }
  if (lane == 31) { sm.warp_sum[warp] = incl; sm.warp_count[warp] = cincl; }
  __syncthreads();
  u64 before = sum0 + incl - mine;
  uint32_t cbefore = count0 + cincl - cnt, all = count0;
  for (int i = 0; i < THREADS / 32; i += 4) {
#pragma unroll
    for (int j = i; j < i + 4; ++j) {
      if (j < warp) { before += sm.warp_sum[j]; cbefore += sm.warp_count[j]; }
      all += sm.warp_count[j];
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (on) {
      lo[tid * PER + i] = uint32_t(before);
      hi[tid * PER + i] = uint32_t(before >> 32);
      count[tid * PER + i] = cbefore;
    }
    before += s[i];
    cbefore += c[i];
  }
  __syncthreads();
  return all;
}

// The bin that covers position z: the last whose sum before it is not beyond z among those that hold anything of it.
template <int N_BINS>
__device__ __forceinline__ int covering(bool by_count, u64 z) {
  Smem& sm = own_smem();
  const uint32_t* const count = N_BINS == BINS ? sm.count : sm.fcount;
  const uint32_t* const lo = N_BINS == BINS ? sm.lo : sm.flo;
  const uint32_t* const hi = N_BINS == BINS ? sm.hi : sm.fhi;
  if (threadIdx.x == 0) sm.bin = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < N_BINS; i += THREADS) {
    const u64 a = by_count ? count[i] : (u64(hi[i]) << 32) + lo[i];
    const u64 b = i + 1 == N_BINS ? ~0ull : by_count ? count[i + 1] : (u64(hi[i + 1]) << 32) + lo[i + 1];
    if (a <= z && z < b) sm.bin = i;
  }
  __syncthreads();
  const int bin = sm.bin;
  __syncthreads();
  return bin;
}

// CTA c's memory, to be read
template <int CTAS>
__device__ __forceinline__ Smem& of_cta(Smem& sm, int c) {
  if constexpr (CTAS == 1) return sm;
  else return *cooperative_groups::this_cluster().map_shared_rank(&sm, c);
}

// The sums over all CTAs, in the first one's memory: a part of the bins to a CTA.  Behind a meeting, and before one.
template <int CTAS>
__device__ __forceinline__ void join_counts(Smem& sm, int rank) {
  if constexpr (CTAS > 1) {
#pragma unroll 1
    for (int i = rank * (BINS / CTAS) + threadIdx.x; i < (rank + 1) * (BINS / CTAS); i += THREADS) {
      uint32_t n = 0;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) n += of_cta<CTAS>(sm, c).count[i];
      of_cta<CTAS>(sm, 0).count[i] = n;
    }
    meet<CTAS>();
  }
}
template <int CTAS>
__device__ __forceinline__ void join_sums(Smem& sm, int rank) {
  if constexpr (CTAS > 1) {
#pragma unroll 1
    for (int i = rank * (BINS / CTAS) + threadIdx.x; i < (rank + 1) * (BINS / CTAS); i += THREADS) {
      u64 sum = 0;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) sum += (u64(of_cta<CTAS>(sm, c).hi[i]) << 32) + of_cta<CTAS>(sm, c).lo[i];
      of_cta<CTAS>(sm, 0).lo[i] = uint32_t(sum);
      of_cta<CTAS>(sm, 0).hi[i] = uint32_t(sum >> 32);
    }
    meet<CTAS>();
  }
}
// The same of the parts of a bin, by the first CTA alone
template <int CTAS>
__device__ __forceinline__ void join_parts(Smem& sm) {
  if constexpr (CTAS > 1) {
#pragma unroll 1
    for (int i = threadIdx.x; i < FINE; i += THREADS) {
      u64 sum = 0;
      uint32_t n = 0;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) {
        Smem& other = of_cta<CTAS>(sm, c);
        sum += (u64(other.fhi[i]) << 32) + other.flo[i];
        n += other.fcount[i];
      }
      sm.flo[i] = uint32_t(sum);
      sm.fhi[i] = uint32_t(sum >> 32);
      sm.fcount[i] = n;
    }
    __syncthreads();
  }
}

// A token of the bin that is searched: few are, but a call (its stack is in cold memory) made a row alone 40 us instead of 27.
template <typename T>
__device__ __forceinline__ void take(const Command now, const Row r, bool by_count, u64 place, float x) {
  Smem& sm = own_smem();
  if (place < now.from || place > now.to) return;
  if (now.cut >= 0) {
    const uint32_t at = uint32_t((now.to - place) >> now.cut);
    atomicAdd(&sm.fcount[at], 1u);
    if (!by_count) add64(&sm.flo[at], &sm.fhi[at], r.weight(x));
  } else {
    const uint32_t slot = atomicAdd(&sm.n, 1u);
    if (slot < LIST) sm.list[slot].place = place;
  }
}

// Of the list's n tokens one for a power of two of neighbouring threads, each with its part of the others: the weights and the number of those before
// it.  True for one thread of each.
__device__ __forceinline__ bool ranked(int n, Item& mine, u64& over, uint32_t& higher) {
  Smem& sm = own_smem();
  const int tid = threadIdx.x;
  int helpers = 1;
  while (helpers < 32 && 2 * helpers * n <= THREADS) helpers *= 2;
  const int me = tid / helpers;
  over = 0;
  higher = 0;
  if (me < n) {
    mine = sm.list[me];
    for (int j = tid & (helpers - 1); j < n; j += helpers) {
      const Item it = sm.list[j];
      if (it.place > mine.place) { over += it.w; ++higher; }
    }
  }
#pragma unroll 1
  for (int o = 1; o < helpers; o *= 2) {
    over += __shfl_xor_sync(0xffffffffu, over, o);
    higher += __shfl_xor_sync(0xffffffffu, higher, o);
  }
  return me < n && (tid & (helpers - 1)) == 0;
}

// The token that covers position z of the running sum (of the running count), in the first CTA's .place, .above and .weight.  z is the first CTA's to
// know.  least: keys below it are not in the sums; near: tokens of the bins below it are in the CTAs' lists; turn: which of the commands is next.
template <typename T, int CTAS>
__device__ __forceinline__ void search(const Slice<T, CTAS> slice, int ids, const Row r, bool by_count, u64 z, uint32_t least, int near, int& turn) {
  Smem& sm = own_smem();
  const int tid = threadIdx.x, rank = slice.rank;
  u64 above = 0;
  uint32_t cabove = 0;
  // how the places from..to of n tokens are searched
  auto next = [&](int bin, u64 from, u64 to, float n) {
    int cut = LISTED;
    if (n > float(LIST)) cut = 64 - __clzll((long long)((to - from) / FINE));
    sm.command[turn].bin = bin;
    sm.command[turn].cut = cut;
    sm.command[turn].from = from;
    sm.command[turn].to = to;
  };
  if (rank == 0) {
    const int bin = covering<BINS>(by_count, z);
    above = (u64(sm.hi[bin]) << 32) + sm.lo[bin];
    cabove = sm.count[bin];
    if (tid == 0) {
      // the bin's logits lie within roundings of its borders; it has at most as many tokens as go into its sum at its lowest weight
      const float lo = float(bin) / r.fold;
      const float x_hi = bin == 0 ? r.top : r.top - lo + 2e-6f * (fabsf(r.top) + lo);
      const float x_lo = r.below(bin);
      float n;
      if (by_count) {
        n = bin == BINS - 1 ? 1e9f : float(sm.count[bin + 1] - cabove);
      } else if (bin == BINS - 1) {                   // nothing lies there
        n = 0.f;
      } else {
        const float sum = float((u64(sm.hi[bin + 1]) << 32) + sm.lo[bin + 1] - above);
        n = sum / fmaxf(__expf(-float(bin + 1) / BINS_A_FOLD) * float(1ull << r.shift) * 0.99f - 1.f, 1.f);
      }
      next(bin, place_of<T>(key_of(x_lo), (1 << ids) - 1, ids), place_of<T>(key_of(x_hi), 0, ids), n);
    }
    __syncthreads();
  }
  bool alone = rank == 0 && sm.command[turn].bin < near;      // what is listed the first CTA reads by itself; the others wait until it is done
  for (;;) {
    if (!alone) meet<CTAS>();
    const Command now = of_cta<CTAS>(sm, 0).command[turn];
    if (now.cut == DONE) break;
    if (!alone) turn ^= 1;
    if (tid == 0) sm.n = 0;
    if (now.cut >= 0)
#pragma unroll 1
      for (int i = tid; i < FINE; i += THREADS) sm.fcount[i] = sm.flo[i] = sm.fhi[i] = 0;
    __syncthreads();
    if (alone) {                                      // a CTA's list to as many threads
      const Smem& other = of_cta<CTAS>(sm, tid / (THREADS / CTAS));
      const int n = int(other.n_near);
      for (int i = tid % (THREADS / CTAS); i < n; i += THREADS / CTAS) {
        const u64 place = other.near[i];
        const float x = value_of(key_at<T>(place, ids));
        if (r.bin(x) == now.bin) take<T>(now, r, by_count, place, x);
      }
      __syncthreads();
    } else {
      const float lowest = value_of(max(least, sizeof(T) == 2 ? uint32_t(now.from >> ids) << 16 : uint32_t(now.from >> ids)));
      const float highest = value_of(key_at<T>(now.to, ids));          // a place of infinity has infinity here, which nothing exceeds
      slice.fours(lowest == lowest ? lowest : -INFINITY, [&](int id, const float (&x)[4], int n) {
        bool some = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) some |= !(x[j] < lowest) && !(x[j] > highest);
        if (!some) return;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t key = key_of(x[j]);
          if (j < n && r.bin(x[j]) == now.bin && key >= least) take<T>(now, r, by_count, place_of<T>(key, id + j, ids), x[j]);
        }
      });
      meet<CTAS>();
    }
    if (rank != 0) continue;
    if (now.cut < 0) {
      uint32_t n = 0;
      if (alone) {
        n = sm.n;
      } else {
#pragma unroll
        for (int c = 0; c < CTAS; ++c) n += of_cta<CTAS>(sm, c).n;
      }
      if (n > LIST) {                                 // more than were to be expected
        if (tid == 0) next(now.bin, now.from, now.to, float(n));
      } else {                                        // the tokens of all slices, ranked by comparison
        Item mine;
        if (tid < int(n)) {
          int c = 0, at = tid;
          if constexpr (CTAS > 1)
            if (!alone)
              for (; at >= int(of_cta<CTAS>(sm, c).n); ++c) at -= int(of_cta<CTAS>(sm, c).n);
          mine.place = of_cta<CTAS>(sm, c).list[at].place;
          mine.w = r.weight(value_of(key_at<T>(mine.place, ids)));
        }
        __syncthreads();
        if (tid < int(n)) sm.list[tid] = mine;
        __syncthreads();
        u64 over;
        uint32_t higher;
        const bool speaks = ranked(int(n), mine, over, higher);
        if (speaks) {
          const u64 start = by_count ? cabove + higher : above + over;
          if (start <= z && z - start < (by_count ? 1 : mine.w)) { sm.place = mine.place; sm.above = above + over; sm.weight = mine.w; }
        }
        if (tid == 0) sm.command[turn].cut = DONE;
        alone = false;                                // to the others
      }
    } else {
      if (!alone) join_parts<CTAS>(sm);
      const uint32_t all = running_sums<FINE>(above, cabove);
      const int at = covering<FINE>(by_count, z);
      above = (u64(sm.fhi[at]) << 32) + sm.flo[at];
      const uint32_t n = (at + 1 == FINE ? all : sm.fcount[at + 1]) - sm.fcount[at];
      cabove = sm.fcount[at];
      if (tid == 0) {
        const u64 top = now.to - (u64(at) << now.cut), size = (u64(1) << now.cut) - 1;
        next(now.bin, top - now.from > size ? top - size : now.from, top, float(n));
      }
    }
    __syncthreads();                                  // the command is there, and what it was found by has been read
  }
  turn ^= 1;
}

__device__ __forceinline__ u64 share(double part, u64 whole) {
  const double z = part * double(whole);
  if (!(z > 0.0)) return 0;
  return min(z < 1.8e19 ? __double2ull_rd(z) : ~0ull, whole - 1);
}

// The draw from `n` listed tokens of all CTAs, at most LIST, by the first one, without any bins (one row of 50257, min-p: 12 us instead of 16).  A call,
// so that rows of which much is left do not carry its registers (inlined, rows with a nucleus took a tenth longer).
template <typename T, int CTAS>
__device__ __noinline__ void draw_of_few(const Sampling p, size_t at, const Row r, int n, int last, int low, int high, uint32_t least, float top_p,
                                         float min_p) {
  Smem& sm = own_smem();
  const int tid = threadIdx.x;
  const double border = double(min_p) * double(1ull << r.shift);
  Item mine;
  u64 in = 0, ok = 0;                                 // what top-k leaves of the whole, and min-p
  if (tid < n) {
    int c = 0, i = tid;
    if constexpr (CTAS > 1)
      for (; i >= of_cta<CTAS>(sm, c).kept; ++c) i -= of_cta<CTAS>(sm, c).kept;
    mine.place = of_cta<CTAS>(sm, c).near[i];
    const float x = value_of(key_at<T>(mine.place, p.ids));
    const int b = r.bin(x);
    if (b <= last && key_of(x) >= least) in = r.weight(x);
    if (b < low || (b <= high && r.scaled(x) >= border)) ok = in;
    mine.w = in;
    sm.list[tid] = mine;
  }
  for (int o = 16; o > 0; o >>= 1) {
    in += __shfl_xor_sync(0xffffffffu, in, o);
    ok += __shfl_xor_sync(0xffffffffu, ok, o);
  }
  if ((tid & 31) == 0) {
    sm.warp_sum[tid >> 5] = in;
    sm.warp_ok[tid >> 5] = ok;
  }
  __syncthreads();
  in = ok = 0;
#pragma unroll 1
  for (int i = 0; i < THREADS / 32; ++i) {
    in += sm.warp_sum[i];
    ok += sm.warp_ok[i];
  }
  u64 over;
  uint32_t higher;
  const bool speaks = ranked(n, mine, over, higher);
  if (top_p > 0.f && top_p < 1.f) {
    const u64 z = share(double(top_p), in);
    if (speaks && over <= z && z - over < mine.w) sm.above = over + mine.w;
    __syncthreads();
    in = sm.above;
  }
  if (min_p > 0.f) in = max(min(in, ok), u64(1) << r.shift);
  const u64 z = share(double(p.u[at]), in);
  if (speaks && over <= z && z - over < mine.w) {
    p.token[at] = id_at<T>(mine.place, p.ids);
    if (p.prob != nullptr) p.prob[at] = float(r.scaled(value_of(key_at<T>(mine.place, p.ids))) / double(in));
  }
}

template <typename T, int CTAS>
__global__ void __launch_bounds__(THREADS, 2) sample_rows_kernel(Sampling p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem& sm = own_smem();
  const int tid = threadIdx.x, V = p.V, rank = CTAS == 1 ? 0 : int(blockIdx.x % CTAS);
  const size_t at = blockIdx.x / CTAS;
  if (tid == 0) { sm.best = 0; sm.best_id = 0; sm.sum = 0; sm.n_near = 0; }
#pragma unroll 1
  for (int i = tid; i < BINS; i += THREADS) sm.count[i] = sm.lo[i] = sm.hi[i] = 0;
  if (tid < TABLE) sm.table[tid] = exp2(-double(tid) / TABLE);
  meet<CTAS>();
  pdl_wait();
  pdl_trigger();
  const T* row = static_cast<const T*>(p.logits) + at * p.ld;
  const float temperature = p.temperature != nullptr ? p.temperature[at] : p.temperature_all;
  const float top_p = p.top_p != nullptr ? p.top_p[at] : p.top_p_all, min_p = p.min_p != nullptr ? p.min_p[at] : p.min_p_all;
  const int top_k = p.top_k != nullptr ? p.top_k[at] : p.top_k_all;

  const Slice<T, CTAS> slice(row, V, rank, p.staged ? reinterpret_cast<uint4*>(smem_raw + (sizeof(Smem) + 15) / 16 * 16) : nullptr);
  uint32_t best = key_of(slice.peak());
  best = __reduce_max_sync(0xffffffffu, best);
  if ((tid & 31) == 0) atomicMax(&sm.best, best);
  meet<CTAS>();
#pragma unroll
  for (int c = 0; c < CTAS; ++c) best = max(best, of_cta<CTAS>(sm, c).best);
  Row r;
  r.top = value_of(best);
  const bool nothing = r.top == -INFINITY;
  if (!(temperature > 0.f) || nothing) {              // the largest, lowest id among equals; no logit above -inf: token 0 with probability 0
    if (!nothing) {
      slice.fours(r.top, [&](int id, const float (&x)[4], int n) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (x[j] == r.top) atomicMax(&sm.best_id, ~uint32_t(id + j));
      });
      meet<CTAS>();
    }
    if (rank == 0 && tid == 0) {
      uint32_t id = nothing ? ~0u : 0u;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) id = max(id, of_cta<CTAS>(sm, c).best_id);
      p.token[at] = int64_t(~id);
      if (p.prob != nullptr) p.prob[at] = nothing ? 0.f : 1.f;
    }
    meet<CTAS>();                                     // as at the end
    return;
  }
  const double rate = 1.0 / fmax(double(temperature), 1e-5);
  r.fold = float(rate) * BINS_A_FOLD;
  r.top64 = to_f64(r.top);
  r.rate = rate * (64 * 1.4426950408889634);
  r.shift = p.shift;
  r.table = sm.table;
  const bool count = top_k > 0 && top_k < V, nucleus = top_p > 0.f && top_p < 1.f;
  // min-p: bins well above the border are in, those well below out; weights decide in the three around it (the bins' borders are rounded)
  int low = 0, high = BINS - 2;
  if (min_p > 0.f) {
    const float d = -logf(min_p) * BINS_A_FOLD;
    const int mid = d < float(BINS - 3) ? max(int(d), 0) : BINS - 3;
    low = max(mid - 1, 0);
    high = mid + 1;
  }
  int last = nucleus ? BINS - 2 : high;               // bins from here on have no say: only a nucleus needs the sum over what min-p cuts
  uint32_t least = 0;
  int turn = 0;
  if (count) {
    // the k-th largest by counts alone, so that nobody takes weights of what lies below it
    slice.fours(-INFINITY, [&](int, const float (&x)[4], int n) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) atomicAdd(&sm.count[r.bin(x[j])], 1u);
    });
    meet<CTAS>();
    join_counts<CTAS>(sm, rank);
    if (rank == 0) running_sums<BINS>(0, 0);
    search<T, CTAS>(slice, p.ids, r, true, u64(top_k - 1), 0, 0, turn);
    least = key_at<T>(of_cta<CTAS>(sm, 0).place, p.ids);
    if (sizeof(T) == 2) least &= 0xffff0000u;
    last = min(last, r.bin(value_of(key_at<T>(of_cta<CTAS>(sm, 0).place, p.ids))));
#pragma unroll 1
    for (int i = tid; i < BINS; i += THREADS) sm.lo[i] = sm.hi[i] = 0;
    __syncthreads();
  }
  const double border = double(min_p) * double(1ull << p.shift);
  const float lowest = fmaxf(r.below(min(last, BINS - 2)), count ? value_of(least) : -INFINITY);
  u64 bordering = 0;
  // a token's weight into its bin (one that has no say: BINS - 1) and, near the border of min-p, into what min-p leaves
  auto weigh = [&](float x, int& b) {
    b = r.bin(x);
    const bool in = b <= last && b < BINS - 1 && key_of(x) >= least;
    const double scaled = r.scaled(x);
    const u64 w = in ? __double_as_longlong(scaled + 4503599627370496.0) & 0xfffffffffffffull : 0;
    if (in && b >= low && b <= high && scaled >= border) bordering += w;
    if (!in) b = BINS - 1;
    return w;
  };
  // Where a filter leaves few, they are listed first, since in a warp some lane nearly always has one: a thread then has one of them.
  bool all = count ? top_k <= NEAR_LIST / 2 * CTAS : min_p > 0.f && !nucleus;
  if (all) {
    slice.fours(lowest, [&](int id, const float (&x)[4], int n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < n && x[j] >= lowest && *static_cast<volatile uint32_t*>(&sm.n_near) <= NEAR_LIST) {
          const uint32_t slot = atomicAdd(&sm.n_near, 1u);
          if (slot < NEAR_LIST) sm.near[slot] = place_of<T>(key_of(x[j]), id + j, p.ids);
        }
      }
    });
    __syncthreads();
    const int n = int(sm.n_near);
    all = n <= NEAR_LIST;
    if (tid == 0) sm.kept = n;
    meet<CTAS>();
    int whole = 0;
#pragma unroll
    for (int c = 0; c < CTAS; ++c) whole += of_cta<CTAS>(sm, c).kept;
    if (whole <= LIST) {                              // so few in all: ranked at once, without any bins
      if (rank == 0) draw_of_few<T, CTAS>(p, at, r, whole, last, low, high, least, top_p, min_p);
      meet<CTAS>();                                   // as at the end
      return;
    }
    if (all) {
      for (int i = tid; i < n; i += THREADS) {
        int b;
        const u64 w = weigh(value_of(key_at<T>(sm.near[i], p.ids)), b);
        if (w) add64(&sm.lo[b], &sm.hi[b], w);
        else sm.near[i] = 0;                          // below every token's place: in no range that is searched
      }
    } else {
      __syncthreads();
      if (tid == 0) sm.n_near = 0;
      __syncthreads();
    }
  }
  if (!all) {
    slice.fours(lowest, [&](int id, const float (&x)[4], int) {
      u64 w[4];
      int b[4];
      uint32_t before[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = weigh(x[j], b[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) before[j] = w[j] ? atomicAdd(&sm.lo[b[j]], uint32_t(w[j])) : 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t up = uint32_t(w[j] >> 32) + (before[j] + uint32_t(w[j]) < before[j] ? 1u : 0u);
        if (up) atomicAdd(&sm.hi[b[j]], up);
        if (b[j] < NEAR && *static_cast<volatile uint32_t*>(&sm.n_near) <= NEAR_LIST) {
          const uint32_t slot = atomicAdd(&sm.n_near, 1u);
          if (slot < NEAR_LIST) sm.near[slot] = place_of<T>(key_of(x[j]), id + j, p.ids);
        }
      }
    });
  }
  if (min_p > 0.f && bordering) atomicAdd(&sm.sum, bordering);
  __syncthreads();
  if (tid == 0) sm.listed = all ? BINS : sm.n_near <= NEAR_LIST ? NEAR : 0;
  meet<CTAS>();
  int near = BINS;
#pragma unroll
  for (int c = 0; c < CTAS; ++c) near = min(near, of_cta<CTAS>(sm, c).listed);
  u64 left = 0;
  join_sums<CTAS>(sm, rank);
  if (rank == 0) {
    // the last bin's weights are 0, so that the sum before it is the whole
    running_sums<BINS>(0, 0);
    left = (u64(sm.hi[BINS - 1]) << 32) + sm.lo[BINS - 1];
  }
  // the nucleus, then the draw: one call, since a second copy of the search would be fetched anew
  for (bool draw = !nucleus;; draw = true) {
    u64 z = share(double(top_p), left);
    if (draw && rank == 0) {
      if (min_p > 0.f) {
        u64 sum = (u64(sm.hi[low]) << 32) + sm.lo[low];
#pragma unroll
        for (int c = 0; c < CTAS; ++c) sum += of_cta<CTAS>(sm, c).sum;
        left = max(min(left, sum), u64(1) << p.shift);         // min_p beyond 1 leaves the largest
      }
      z = share(double(p.u[at]), left);
    }
    search<T, CTAS>(slice, p.ids, r, false, z, least, near, turn);
    if (draw) break;
    left = sm.above + sm.weight;
  }
  if (rank == 0 && tid == 0) {
    p.token[at] = id_at<T>(sm.place, p.ids);
    if (p.prob != nullptr) p.prob[at] = float(r.scaled(value_of(key_at<T>(sm.place, p.ids))) / double(left));
  }
  meet<CTAS>();                                       // a CTA's memory is there until everybody has read it
}

template <typename T, int CTAS>
int launch_rows_by(Sampling p, int n_rows, cudaStream_t stream) {
  // a slice of up to 64 KB is kept, so that two CTAs fit a SM (one row of 16384 tokens 20.6 to 25.6 us, read again from L2 20.5 to 26.3; of 50257 24.3 to
  // 36.6 and 24.6 to 36.9)
  constexpr size_t base = (sizeof(Smem) + 15) / 16 * 16, most = 64 * 1024;
  const size_t slice = size_t((p.V / int(16 / sizeof(T)) + CTAS * THREADS - 1) / (CTAS * THREADS)) * THREADS * 16;
  p.staged = slice <= most;
  JB_MAX_SMEM((sample_rows_kernel<T, CTAS>), base + most);
  if constexpr (CTAS == 1) launch_dep(sample_rows_kernel<T, 1>, n_rows, THREADS, base + (p.staged ? slice : 0), stream, p);
  else launch_dep_cluster(sample_rows_kernel<T, CTAS>, n_rows * CTAS, THREADS, base + (p.staged ? slice : 0), CTAS, stream, p);
  return JB200_OK;
}

// CTAs a row: as many as two a SM leave room for, slices of 4096 tokens or more.  us with the launch from cold, bf16: 64 rows of 50257 with every setting
// of their own 46, with one CTA a SM 54, with four 58 to 64; one row of 50257 (nucleus, by seed) in eight slices 24 to 37, in four 30 to 41, whole 47 to 68;
// of 16384 in four 21 to 26, whole 25 to 31; of 8192 in two 21 to 25, whole 19 to 21; of 4096 in two 21, whole 16.
template <typename T>
int launch_rows(const Sampling& p, int n_rows, cudaStream_t stream) {
  const int most = 2 * sm_count() / n_rows, wide = p.V / 4096, ctas = most < wide ? most : wide;
  return ctas >= 8 ? launch_rows_by<T, 8>(p, n_rows, stream) : ctas >= 4 ? launch_rows_by<T, 4>(p, n_rows, stream)
       : ctas >= 2 ? launch_rows_by<T, 2>(p, n_rows, stream) : launch_rows_by<T, 1>(p, n_rows, stream);
}

}  // namespace

int launch_sample_rows(const jb200_sampling* s, int n_rows, int64_t* token, float* prob, cudaStream_t stream) {
  JB_REQUIRE(s != nullptr, "sample_rows: null pointer");
  JB_REQUIRE(n_rows >= 0 && s->V > 0 && s->ld >= s->V, "sample_rows: bad shape (rows=%d, V=%d, ld=%lld)", n_rows, s->V, s->ld);
  JB_REQUIRE(s->V <= 1 << 24, "sample_rows: at most 2^24 tokens (V=%d)", s->V);
  JB_REQUIRE(s->logits_dtype == 0 || s->logits_dtype == 1, "sample_rows: logits dtype must be 0 (f32) or 1 (bf16)");
  if (n_rows == 0) return JB200_OK;
  JB_REQUIRE(s->logits && s->u && token, "sample_rows: null pointer");
  Sampling p;
  p.logits = s->logits; p.ld = size_t(s->ld); p.V = s->V;
  int bits = 0;
  while ((1 << bits) < s->V) ++bits;
  p.ids = bits > 0 ? bits : 1;
  p.shift = 63 - bits < 45 ? 63 - bits : 45;        // V weights of at most 2^shift fit 63 bits
  p.u = s->u; p.temperature = s->temperature; p.top_k = s->top_k; p.top_p = s->top_p; p.min_p = s->min_p;
  p.temperature_all = s->temperature_all; p.top_k_all = s->top_k_all; p.top_p_all = s->top_p_all; p.min_p_all = s->min_p_all;
  p.token = token; p.prob = prob;
  const int rc = s->logits_dtype == 0 ? launch_rows<float>(p, n_rows, stream) : launch_rows<__nv_bfloat16>(p, n_rows, stream);
  if (rc != JB200_OK) return rc;
  JB_LAUNCH_CHECK("sample_rows_kernel");
  return JB200_OK;
}

}  // namespace jb

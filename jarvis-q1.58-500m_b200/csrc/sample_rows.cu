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
// 2^-45 of the largest one's, so that sums do not depend on the order of the atomics that form them, and a token that the exact sums choose is
// missed only where u lies within some 1e-12 of a border.  A cluster of CTAs has a row, a slice each (in shared memory where it fits), with as many CTAs as
// keep the SMs busy.  A histogram of the sums (for top-k of the counts) over 2048 bins of 1/32 of an e-fold finds the bin that covers z.  The
// tokens of a bin, up to 256, are ranked by comparison with one another; where there are more they are first cut into 512 parts of their order, logit
// then id, until there are not.  The few tokens near the largest, where most answers lie, are listed as the sums are taken.  Every CTA counts and lists its slice in its own memory; the first one reads the others' and searches, the others
// read what it found.
#include <cooperative_groups.h>

#include "common.cuh"
#include "launchers.h"

namespace jb {

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512;
constexpr int BINS = 2048;              // 1/32 of an e-fold each; the last: everything 64 e-folds or more below the largest, whose weight is 0
constexpr float BINS_A_FOLD = 32.f;
constexpr int FINE = 512;
constexpr int LIST = 256;
constexpr int NEAR = 224, NEAR_LIST = 512;   // bins whose tokens are listed at once (7 e-folds), as long as there are no more than that in a slice
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

struct Smem {
  uint32_t count[BINS], lo[BINS], hi[BINS];       // then, as running sums before every bin: count, (lo, hi)
  uint32_t fcount[FINE], flo[FINE], fhi[FINE];
  Item list[LIST];
  u64 near[NEAR_LIST];
  u64 warp_sum[THREADS / 32];
  uint32_t warp_count[THREADS / 32];
  u64 best;                                       // (key, ~id) of the largest
  uint32_t n, n_near;
  int bin, cut;                                   // what is searched next: of this bin the places from..to; cut: in parts of 2^cut of them, < 0: one by one
  u64 from, to;
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

// A CTA's slice of a row: vectors of 16 bytes, every CTAS-th 512 of them, and the elements before and behind them that are not aligned
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
  // f(id, value) for every element; FIRST: from memory and into the stage
  template <bool FIRST = false, typename F>
  __device__ __forceinline__ void every(F&& f) const {
    const int tail = head + vectors * PER;
    const uint4* body = reinterpret_cast<const uint4*>(row + head);
    if (rank == 0 && int(threadIdx.x) < head) f(int(threadIdx.x), widen(row[threadIdx.x]));
    uint4* staged = stage + threadIdx.x;
#pragma unroll 2
    for (int i = rank * THREADS + threadIdx.x; i < vectors; i += CTAS * THREADS, staged += THREADS) {
      uint4 x;
      if (FIRST || stage == nullptr) x = __ldg(body + i);
      else x = *staged;
      if (FIRST && stage != nullptr) *staged = x;
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      const int id = head + i * PER;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) {
          f(id + 2 * j, bf16_lo(w[j]));
          f(id + 2 * j + 1, bf16_hi(w[j]));
        } else {
          f(id + j, __uint_as_float(w[j]));
        }
      }
    }
    if (rank == CTAS - 1 && tail + int(threadIdx.x) < V) f(tail + int(threadIdx.x), widen(row[tail + threadIdx.x]));
  }
};

// All CTAs of the row, with what they wrote
template <int CTAS>
__device__ __forceinline__ void meet() {
  if constexpr (CTAS == 1) __syncthreads();
  else cooperative_groups::this_cluster().sync();
}

// x as f64 (a subnormal x as some other number of 1e-38: no weight shows it); the conversion instruction runs at an eighth of this one's rate
__device__ __forceinline__ double to_f64(float x) {
  const uint32_t b = __float_as_uint(x), m = b & 0x7fffffffu;
  return __hiloint2double(int((b & 0x80000000u) | ((m >> 3) + 0x38000000u)), int(m << 29));
}

// Place in the order of a row: `ids` bits of the id from the end behind the logit's key, of which bf16 has 16 bits
template <typename T>
__device__ __forceinline__ u64 place_of(uint32_t key, int id, int ids) { return (u64(sizeof(T) == 2 ? key >> 16 : key) << ids) + ((1u << ids) - 1u - uint32_t(id)); }
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
__device__ uint32_t running_sums(uint32_t* count, uint32_t* lo, uint32_t* hi, Smem& sm, u64 sum0, uint32_t count0) {
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
  for (int i = 0; i < THREADS / 32; ++i) {
    if (i < warp) { before += sm.warp_sum[i]; cbefore += sm.warp_count[i]; }
    all += sm.warp_count[i];
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
template <int N_BINS, bool BY_COUNT>
__device__ int covering(const uint32_t* count, const uint32_t* lo, const uint32_t* hi, Smem& sm, u64 z) {
  if (threadIdx.x == 0) sm.bin = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < N_BINS; i += THREADS) {
    const u64 a = BY_COUNT ? count[i] : (u64(hi[i]) << 32) + lo[i];
    const u64 b = i + 1 == N_BINS ? ~0ull : BY_COUNT ? count[i + 1] : (u64(hi[i + 1]) << 32) + lo[i + 1];
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

// The first CTA's bins: the sums over all CTAs
template <int CTAS, int N_BINS, typename C, typename L, typename H>
__device__ __forceinline__ void join(Smem& sm, C&& count, L&& lo, H&& hi, bool counts) {
  if constexpr (CTAS > 1) {
    for (int i = threadIdx.x; i < N_BINS; i += THREADS) {
      u64 sum = 0;
      uint32_t n = 0;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) {
        Smem& other = of_cta<CTAS>(sm, c);
        sum += (u64(hi(other)[i]) << 32) + lo(other)[i];
        if (counts) n += count(other)[i];
      }
      lo(sm)[i] = uint32_t(sum);
      hi(sm)[i] = uint32_t(sum >> 32);
      count(sm)[i] = n;
    }
    __syncthreads();
  }
}

// The token that covers position z of the running sum (of the running count), in the first CTA's .place, .above and .weight.  z is the first CTA's to
// know.  least: keys below it are not in the sums; near: bins below it are in the lists of what is near the largest.
template <typename T, int CTAS, bool BY_COUNT>
__device__ void search(const Slice<T, CTAS>& slice, int ids, const Row& r, Smem& sm, u64 z, uint32_t least, int near) {
  const int tid = threadIdx.x, rank = slice.rank;
  const Smem& first = of_cta<CTAS>(sm, 0);
  u64 above = 0;
  uint32_t cabove = 0;
  // how the places from..to of n tokens are searched
  auto next = [&](u64 from, u64 to, float n) {
    int cut = -1;
    if (n > float(LIST)) {
      cut = 0;
      while (((to - from) >> cut) >= FINE) ++cut;
    }
    sm.from = from;
    sm.to = to;
    sm.cut = cut;
  };
  if (rank == 0) {
    const int bin = covering<BINS, BY_COUNT>(sm.count, sm.lo, sm.hi, sm, z);
    above = (u64(sm.hi[bin]) << 32) + sm.lo[bin];
    cabove = sm.count[bin];
    if (tid == 0) {
      // the bin's logits lie within roundings of its borders; it has at most as many tokens as go into its sum at its lowest weight
      const float lo = float(bin) / r.fold, hi = float(bin + 1) / r.fold;
      const float x_hi = bin == 0 ? r.top : r.top - lo + 2e-6f * (fabsf(r.top) + lo);
      const float x_lo = bin == BINS - 1 ? -INFINITY : r.top - hi - 2e-6f * (fabsf(r.top) + hi);
      float n;
      if (BY_COUNT) {
        n = bin == BINS - 1 ? 1e9f : float(sm.count[bin + 1] - cabove);
      } else if (bin == BINS - 1) {                   // nothing lies there
        n = 0.f;
      } else {
        const float sum = float((u64(sm.hi[bin + 1]) << 32) + sm.lo[bin + 1] - above);
        n = sum / fmaxf(__expf(-float(bin + 1) / BINS_A_FOLD) * float(1ull << r.shift) * 0.99f - 1.f, 1.f);
      }
      sm.bin = bin;
      next(place_of<T>(key_of(x_lo), (1 << ids) - 1, ids), place_of<T>(key_of(x_hi), 0, ids), n);
    }
  }
  for (;;) {
    if (tid == 0) sm.n = 0;
    meet<CTAS>();
    const int bin = first.bin, cut = first.cut;
    const u64 from = first.from, to = first.to;
    if (cut >= 0) {
      for (int i = tid; i < FINE; i += THREADS) sm.fcount[i] = sm.flo[i] = sm.fhi[i] = 0;
      __syncthreads();
    }
    auto take = [&](u64 place, float x) {
      if (place < from || place > to) return;
      if (cut >= 0) {
        const uint32_t at = uint32_t((to - place) >> cut);
        atomicAdd(&sm.fcount[at], 1u);
        if (!BY_COUNT) add64(&sm.flo[at], &sm.fhi[at], r.weight(x));
      } else {
        const uint32_t slot = atomicAdd(&sm.n, 1u);
        if (slot < LIST) sm.list[slot].place = place;
      }
    };
    if (bin < near) {
      for (int i = tid; i < int(sm.n_near); i += THREADS) {
        const float x = value_of(key_at<T>(sm.near[i], ids));
        if (r.bin(x) == bin) take(sm.near[i], x);
      }
    } else {
      slice.every([&](int id, float x) {
        if (r.bin(x) != bin) return;
        const uint32_t key = key_of(x);
        if (key >= least) take(place_of<T>(key, id, ids), x);
      });
    }
    meet<CTAS>();
    if (cut < 0) {
      uint32_t n = 0;
#pragma unroll
      for (int c = 0; c < CTAS; ++c) n += of_cta<CTAS>(sm, c).n;
      if (n <= LIST) {
        if (rank == 0) {                              // the tokens of all slices, ranked by comparison
          Item mine;
          if (tid < int(n)) {
            int c = 0, at = tid;
            if constexpr (CTAS > 1)
              for (; at >= int(of_cta<CTAS>(sm, c).n); ++c) at -= int(of_cta<CTAS>(sm, c).n);
            mine.place = of_cta<CTAS>(sm, c).list[at].place;
            mine.w = r.weight(value_of(key_at<T>(mine.place, ids)));
          }
          __syncthreads();
          if (tid < int(n)) sm.list[tid] = mine;
          __syncthreads();
          // a power of two of neighbouring threads an element, each with its part of the others
          int helpers = 1;
          while (helpers < 32 && 2 * helpers * int(n) <= THREADS) helpers *= 2;
          const int me = tid / helpers;
          u64 over = 0;
          uint32_t higher = 0;
          if (me < int(n)) {
            mine = sm.list[me];
            for (int j = tid & (helpers - 1); j < int(n); j += helpers) {
              const Item it = sm.list[j];
              if (it.place > mine.place) { over += it.w; ++higher; }
            }
          }
          for (int o = 1; o < helpers; o *= 2) {
            over += __shfl_xor_sync(0xffffffffu, over, o);
            higher += __shfl_xor_sync(0xffffffffu, higher, o);
          }
          if (me < int(n) && (tid & (helpers - 1)) == 0) {
            const u64 start = BY_COUNT ? cabove + higher : above + over;
            if (start <= z && z - start < (BY_COUNT ? 1 : mine.w)) { sm.place = mine.place; sm.above = above + over; sm.weight = mine.w; }
          }
        }
        break;
      }
      if (rank == 0 && tid == 0) next(from, to, float(n));          // more than were to be expected
      continue;
    }
    if (rank == 0) {
      join<CTAS, FINE>(sm, [](Smem& x) { return x.fcount; }, [](Smem& x) { return x.flo; }, [](Smem& x) { return x.fhi; }, true);
      const uint32_t all = running_sums<FINE>(sm.fcount, sm.flo, sm.fhi, sm, above, cabove);
      const int at = covering<FINE, BY_COUNT>(sm.fcount, sm.flo, sm.fhi, sm, z);
      above = (u64(sm.fhi[at]) << 32) + sm.flo[at];
      const uint32_t n = (at + 1 == FINE ? all : sm.fcount[at + 1]) - sm.fcount[at];
      cabove = sm.fcount[at];
      if (tid == 0) {
        const u64 top = to - (u64(at) << cut), size = (u64(1) << cut) - 1;
        sm.bin = bin;
        next(top - from > size ? top - size : from, top, float(n));
      }
    }
  }
  meet<CTAS>();                                       // everybody has read what this search used
}

__device__ __forceinline__ u64 share(double part, u64 whole) {
  const double z = part * double(whole);
  if (!(z > 0.0)) return 0;
  return min(z < 1.8e19 ? __double2ull_rd(z) : ~0ull, whole - 1);
}

template <typename T, int CTAS>
__global__ void __launch_bounds__(THREADS, 2) sample_rows_kernel(Sampling p) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
  const int tid = threadIdx.x, V = p.V, rank = CTAS == 1 ? 0 : int(blockIdx.x % CTAS);
  const size_t at = blockIdx.x / CTAS;
  if (tid == 0) { sm.best = 0; sm.sum = 0; sm.n_near = 0; }
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
  u64 best = 0;
  slice.template every<true>([&](int id, float x) { best = max(best, (u64(key_of(x)) << 32) | uint32_t(~id)); });
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) atomicMax(&sm.best, best);
  meet<CTAS>();
#pragma unroll
  for (int c = 0; c < CTAS; ++c) best = max(best, of_cta<CTAS>(sm, c).best);
  Row r;
  r.top = value_of(uint32_t(best >> 32));
  const bool nothing = r.top == -INFINITY;
  if (!(temperature > 0.f) || nothing) {              // the largest, lowest id among equals; no logit above -inf: token 0 with probability 0
    if (rank == 0 && tid == 0) {
      p.token[at] = nothing ? 0 : int64_t(~uint32_t(best));
      if (p.prob != nullptr) p.prob[at] = nothing ? 0.f : 1.f;
    }
    meet<CTAS>();                                     // a CTA's memory is there until everybody has read it
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
  if (count) {
    // the k-th largest by counts alone, so that nobody takes weights of what lies below it
    slice.every([&](int id, float x) { atomicAdd(&sm.count[r.bin(x)], 1u); });
    meet<CTAS>();
    if (rank == 0) {
      join<CTAS, BINS>(sm, [](Smem& x) { return x.count; }, [](Smem& x) { return x.lo; }, [](Smem& x) { return x.hi; }, true);
      running_sums<BINS>(sm.count, sm.lo, sm.hi, sm, 0, 0);
    }
    search<T, CTAS, true>(slice, p.ids, r, sm, u64(top_k - 1), 0, 0);
    least = key_at<T>(of_cta<CTAS>(sm, 0).place, p.ids);
    if (sizeof(T) == 2) least &= 0xffff0000u;
    last = min(last, r.bin(value_of(key_at<T>(of_cta<CTAS>(sm, 0).place, p.ids))));
    meet<CTAS>();
    for (int i = tid; i < BINS; i += THREADS) sm.lo[i] = sm.hi[i] = 0;
    __syncthreads();
  }
  const double border = double(min_p) * double(1ull << p.shift);
  u64 bordering = 0;
  slice.every([&](int id, float x) {
    const int b = r.bin(x);
    if (b > last || b == BINS - 1) return;
    const uint32_t key = key_of(x);
    if (key < least) return;
    const double scaled = r.scaled(x);
    const u64 w = __double_as_longlong(scaled + 4503599627370496.0) & 0xfffffffffffffull;
    if (b >= low && b <= high && scaled >= border) bordering += w;
    if (w) add64(&sm.lo[b], &sm.hi[b], w);
    if (b < NEAR && *static_cast<volatile uint32_t*>(&sm.n_near) <= NEAR_LIST) {
      const uint32_t slot = atomicAdd(&sm.n_near, 1u);
      if (slot < NEAR_LIST) sm.near[slot] = place_of<T>(key, id, p.ids);
    }
  });
  if (min_p > 0.f && bordering) atomicAdd(&sm.sum, bordering);
  meet<CTAS>();
  int near = NEAR;
#pragma unroll
  for (int c = 0; c < CTAS; ++c)
    if (of_cta<CTAS>(sm, c).n_near > NEAR_LIST) near = 0;
  u64 left = 0;
  if (rank == 0) {
    join<CTAS, BINS>(sm, [](Smem& x) { return x.count; }, [](Smem& x) { return x.lo; }, [](Smem& x) { return x.hi; }, false);
    // the last bin's weights are 0, so that the sum before it is the whole
    running_sums<BINS>(sm.count, sm.lo, sm.hi, sm, 0, 0);
    left = (u64(sm.hi[BINS - 1]) << 32) + sm.lo[BINS - 1];
  }
  if (nucleus) {
    search<T, CTAS, false>(slice, p.ids, r, sm, share(double(top_p), left), least, near);
    if (rank == 0) left = sm.above + sm.weight;
  }
  if (min_p > 0.f && rank == 0) {
    u64 sum = (u64(sm.hi[low]) << 32) + sm.lo[low];
#pragma unroll
    for (int c = 0; c < CTAS; ++c) sum += of_cta<CTAS>(sm, c).sum;
    left = max(min(left, sum), u64(1) << p.shift);             // min_p beyond 1 leaves the largest
  }
  search<T, CTAS, false>(slice, p.ids, r, sm, rank == 0 ? share(double(p.u[at]), left) : 0, least, near);
  if (rank == 0 && tid == 0) {
    p.token[at] = id_at<T>(sm.place, p.ids);
    if (p.prob != nullptr) p.prob[at] = float(r.scaled(value_of(key_at<T>(sm.place, p.ids))) / double(left));
  }
}

template <typename T, int CTAS>
int launch_rows_by(Sampling p, int n_rows, cudaStream_t stream) {
  // a slice of up to 64 KB is kept: two CTAs a SM
  constexpr size_t base = (sizeof(Smem) + 15) / 16 * 16, most = 64 * 1024;
  const size_t slice = size_t((p.V / int(16 / sizeof(T)) + CTAS * THREADS - 1) / (CTAS * THREADS)) * THREADS * 16;
  p.staged = slice <= most;
  JB_MAX_SMEM((sample_rows_kernel<T, CTAS>), base + most);
  if constexpr (CTAS == 1) launch_dep(sample_rows_kernel<T, 1>, n_rows, THREADS, base + (p.staged ? slice : 0), stream, p);
  else launch_dep_cluster(sample_rows_kernel<T, CTAS>, n_rows * CTAS, THREADS, base + (p.staged ? slice : 0), CTAS, stream, p);
  return JB200_OK;
}

// CTAs a row: as many as two a SM leave room for, slices of 4096 tokens or more
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

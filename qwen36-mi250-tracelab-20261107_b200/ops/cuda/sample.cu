// The next token of every row of logits, by the row's own temperature T, top-k, top-p and min-p and one uniform number u per row.
//
//   w_i = exp((x_i - m) / T), m the row's maximum; tokens stand in descending order of x, the lower id first among equals
//   kept: the first k; of those the ones with (weight before them) <= p * (weight of the k); of those the ones with w_i >= min_p
//   pick: the first kept token with (weight up to it and with it) > u * (weight of the kept)
//
// Each rule keeps a prefix of the order, so a row is three searches for a place in it: by count (k), by weight (p), by weight (u).
// None needs the whole order. Token and logit are one 64-bit number (`comp`: the logit's bits made monotone, then the id reversed),
// all different, so that ties need no rule of their own.
//
// What decides a pick is held in 64 bits: with 248,320 tokens kept, sums that were off by one part in 1e8 would move one draw in
// 400 to a neighbouring token, and a request's tokens would depend on how the sums were cut. The weights of the tokens outside a row's list are added up in
// fp32, with a bound on what that is off by: a row that the bound leaves undecided goes to the wide kernel, which works in 64 bits throughout.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <float.h>

#include "common.cuh"

namespace b200 {
namespace cg = cooperative_groups;

struct SampleArgs {
  const void* logits;
  long long stride;  // elements between rows
  int n, V;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  const int* exclude;  // [n, n_exclude], entries outside [0, V) name no token
  int n_exclude;
  int64_t* out;
};

// What a row's launches tell each other.
struct SamplePlan {
  double tail_by;           // the tail's sum in fp32 times this is its weight beside `ref`
  float slope, zero;        // log2 of a logit's weight: logit * slope - zero
  float reach, least, ref;  // threshold of the list; below `least` a token has no weight; what the tail's weights are relative to
  float low;                // the sample's smallest
  int skip, with_tail;      // the list cannot decide this row; the others' weights are summed up
  uint64_t top;             // of a row that is left with a whole list: its first token
  uint32_t listed, done;    // tokens in the list, CTAs that have finished their part of the row
};
struct SampleWork {
  int* left;         // rows left to the wide kernel, and which
  int* left_rows;
  SamplePlan* plan;  // [n]
  uint64_t* list;    // [n, LIST]
  double* tail;      // [n, tasks]
  double* powers;    // 2^(i / 32)
};

enum LogitType : int { LOGIT_F32 = 0, LOGIT_BF16 = 1, LOGIT_F16 = 2 };
constexpr int SAMPLE_MAX_EXCLUDE = 64;

// A logit as fp32, exact. NaN counts as minus infinity, -0 as 0.
template <typename T>
__device__ __forceinline__ float logit_value(T v);
template <>
__device__ __forceinline__ float logit_value(float v) { return v != v ? -INFINITY : v + 0.f; }
template <>
__device__ __forceinline__ float logit_value(bf16 v) { return logit_value(__bfloat162float(v)); }
template <>
__device__ __forceinline__ float logit_value(__half v) { return logit_value(__half2float(v)); }

// Monotone in x; 0 for minus infinity, which stands for no token.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return x == -INFINITY ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint64_t comp_of(float x, int id) {
  const uint32_t k = order_key(x);
  return k ? static_cast<uint64_t>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(id)) : 0;
}
__device__ __forceinline__ float comp_value(uint64_t c) { return key_value(static_cast<uint32_t>(c >> 32)); }
__device__ __forceinline__ int comp_id(uint64_t c) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(c)); }

// exp((x - m) / T) with 1 / T given; x <= m.
__device__ __forceinline__ double weight_of(float x, float m, double inv_t) {
  if (x == m) return 1.0;
  const double y = (static_cast<double>(x) - static_cast<double>(m)) * inv_t;
  return y <= 0.0 ? exp(y) : 0.0;  // (a NaN: an infinite m and an infinite T)
}

// Descending; n a power of two.
template <int THREADS>
__device__ __forceinline__ void sort_down(uint64_t* a, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += THREADS) {
        const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
        const uint64_t x = a[lo], y = a[hi];
        if ((x < y) == ((lo & k) == 0)) { a[lo] = y; a[hi] = x; }
      }
    }
  __syncthreads();
}

constexpr int LIST = 2048;         // most tokens that are put in order one by one
constexpr int LIST_BINS = 1024;
constexpr uint32_t LIST_COMPARES = 1536;  // comparisons of a thread, up to which the tokens of a bin are compared each with each

struct Order {
  uint64_t item[LIST];
  union {
    uint64_t other[LIST];
    double sum[LIST];  // of the weights of the ordered list, up to and with each
  };
  uint16_t at[LIST];
  uint32_t bins[LIST_BINS], warp_count[32];
};

// Puts s.item[0 .. c) into descending order: bins by value, in a bin each is compared with each. `hi` and `lo`: between which most of the values lie.
// Many equal values are sorted by exchanges instead, which take 66 rounds for a full list (256 open rows of fp32 logits 128 us with 1,000 to 2,560 comparisons
// to a thread before that, 136 with 512; 61 rows of bf16 logits 74 and 84, and 126 with 6,000). All threads of the CTA. A row's list is put in order once, so
// this and what follows is short code and not unrolled: 166 tokens took 11,000 cycles unrolled eight times, nearly all of them for instructions.
template <int THREADS>
__device__ void order_list(Order& s, int c, float hi, float lo) {
  constexpr int BINS = LIST_BINS / THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float scale = hi > lo ? fminf(LIST_BINS / (hi - lo), 1e30f) : 0.f;
  const auto bin_of = [&](uint64_t comp) { return min(LIST_BINS - 1, max(0, static_cast<int>((hi - comp_value(comp)) * scale))); };
  for (int b = tid; b < LIST_BINS; b += THREADS) s.bins[b] = 0;
  __syncthreads();
#pragma unroll 2
  for (int i = tid; i < c; i += THREADS) s.at[i] = static_cast<uint16_t>(atomicAdd(&s.bins[bin_of(s.item[i])], 1u));
  __syncthreads();
  uint32_t own[BINS], most = 0, up = 0;
#pragma unroll
  for (int j = 0; j < BINS; ++j) { own[j] = s.bins[tid * BINS + j]; most = max(most, own[j]); up += own[j]; }
  const uint32_t sum = up;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) s.warp_count[warp] = up;
  if (__syncthreads_or(most * ((c + THREADS - 1) / THREADS) > LIST_COMPARES)) {
    int size = 2;
    while (size < c) size <<= 1;
    for (int i = c + tid; i < size; i += THREADS) s.item[i] = 0;
    sort_down<THREADS>(s.item, size);
    return;
  }
#pragma unroll 1
  for (int w = 0; w < warp; ++w) up += s.warp_count[w];
  up -= sum;
#pragma unroll
  for (int j = 0; j < BINS; ++j) { s.bins[tid * BINS + j] = up; up += own[j]; }  // where a bin starts
  __syncthreads();
#pragma unroll 2
  for (int i = tid; i < c; i += THREADS) s.other[s.bins[bin_of(s.item[i])] + s.at[i]] = s.item[i];
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < c; i += THREADS) {
    const uint64_t mine = s.other[i];
    const int b = bin_of(mine);
    const uint32_t from = s.bins[b], to = b + 1 < LIST_BINS ? s.bins[b + 1] : static_cast<uint32_t>(c);
    uint32_t above = from;
#pragma unroll 4
    for (uint32_t k = from; k < to; ++k) above += s.other[k] > mine;
    s.item[above] = mine;
  }
  __syncthreads();
}

// 2^(s / 32) for s in [-4000, 0] and a little more: the fraction's 32 values are held by a warp's lanes, and what is left of s, at most half either
// way, goes through a polynomial: with f ln 2 / 32 = g, at most 0.011, the powers of g over their factorials up to the fifth (the sixth is one part
// in 2^49). All lanes of the warp take part. Nine 64-bit operations, the multiplication into the caller's sum included.
struct ExpLanes {
  int lo, hi;
  __device__ __forceinline__ explicit ExpLanes(double power_of_lane) {
    lo = __double2loint(power_of_lane);
    hi = __double2hiint(power_of_lane);
  }
  static constexpr double G = 0.69314718055994531 / 32;
  __device__ __forceinline__ double add(double sum, double s) const {
    const double z = s + 0x1.8p52;  // the nearest whole number stands in the low word
    const int n = __double2loint(z);
    const double f = s - (z - 0x1.8p52);
    double q = fma(f, G * G * G * G * G / 120, G * G * G * G / 24);
    q = fma(f, q, G * G * G / 6);
    q = fma(f, q, G * G / 2);
    q = fma(f, q, G);
    const double t = __hiloint2double(__shfl_sync(0xffffffffu, hi, n) + ((n & ~31) << 15), __shfl_sync(0xffffffffu, lo, n));
    return fma(t, fma(f, q, 1.0), sum);
  }
};
constexpr double STEPS = 46.166241308446828;  // 32 / ln 2

constexpr int WIDE_CTAS = 16;       // of a row: one cluster
constexpr int WIDE_THREADS = 1024;
constexpr int WIDE_HELD = 16384;    // logits that a CTA holds; its part of a larger vocabulary is read again in every pass
constexpr int WIDE_BINS = 2048;
constexpr int WIDE_WORDS = 2;
constexpr float WIDE_RANGE = 80.f;  // e^-80 of the largest weight, 2^22 times, is nothing in 64 bits
constexpr int SAMPLE_MAX_VOCAB = 1 << 22;

struct WideTable {  // sums up to and with each bin, of the whole row
  uint32_t count[WIDE_BINS];
  double mass[WIDE_BINS];
};
struct WideShared {
  float held[WIDE_HELD];
  union {
    struct { uint32_t count[WIDE_BINS], mass[WIDE_WORDS][WIDE_BINS]; } bins;  // this CTA's part
    Order list;                                                             // (of the first CTA)
  };
  WideTable first, finer;  // of the first CTA
  uint64_t top[WIDE_CTAS], low[WIDE_CTAS];  // every CTA's
  double part[WIDE_CTAS];
  unsigned long long sums[1 + WIDE_WORDS][WIDE_BINS / WIDE_CTAS];
  double warp_sum[WIDE_THREADS / 32];
  uint64_t warp_top[WIDE_THREADS / 32], warp_low[WIDE_THREADS / 32];
  uint32_t warp_count[WIDE_THREADS / 32];
  int banned[SAMPLE_MAX_EXCLUDE];
  int n_banned;
  uint32_t listed;
  // what the first CTA found, in every CTA
  int bin;
  uint32_t members;
  uint64_t cut;
  // the first CTA's
  int place;
  uint32_t base_count;
  double base_mass, cut_mass;
};

// One row, one cluster: 16 SMs hold the row's logits in shared memory and look for its places with bins of the whole row (2,048 by value), then within the
// place's bin. This is one-off code: what it takes is the latency of its steps and of fetching their instructions, so what is used
// twice is there once. Arguments go by value, into registers. 30 us for up to nine rows of 248,320, 60 for ten to eighteen.
template <typename T>
struct WidePart {  // a CTA's part of the row
  WideShared& s;
  const T* row;
  int begin, end;
  bool held;

  // The logit of token i, minus infinity for one that does not count and behind the end.
  __device__ __forceinline__ float value(int i) const {
    if (i >= end) return -INFINITY;
    if (held) return s.held[i - begin];
    for (int j = 0; j < s.n_banned; ++j)
      if (s.banned[j] == i) return -INFINITY;
    return logit_value(row[i]);
  }
  // f(x, id) for every token, by whole warps
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const int stop = begin + (end - begin + WIDE_THREADS - 1) / WIDE_THREADS * WIDE_THREADS;
    if (held) {
#pragma unroll 4
      for (int i = begin + static_cast<int>(threadIdx.x); i < stop; i += WIDE_THREADS) f(i < end ? s.held[i - begin] : -INFINITY, i);
    } else {
#pragma unroll 1
      for (int i = begin + static_cast<int>(threadIdx.x); i < stop; i += WIDE_THREADS) f(value(i), i);
    }
  }
};
struct WideScale {
  float m, floor, scale;  // maximum; below it no weight; bins per unit of m - x
  float fall;             // powers of two by which weights fall from bin to bin
  double inv_t, step;
  __device__ __forceinline__ int bin(float x) const { return min(WIDE_BINS - 1, static_cast<int>((m - x) * scale)); }
  // A bin's weights are at most 2^-lift, but for a rounding.
  __device__ __forceinline__ int lift(int bin) const { return min(127, static_cast<int>(bin * fall)); }
};

// Largest and smallest over the cluster, in every CTA.
__device__ __noinline__ void wide_extremes(WideShared& s, uint64_t* top_of, uint64_t* low_of) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  uint64_t top = *top_of, low = *low_of;
  for (int o = 16; o; o >>= 1) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if ((tid & 31) == 0) { s.warp_top[tid >> 5] = top; s.warp_low[tid >> 5] = low; }
  __syncthreads();
  if (tid < 32) {
    top = s.warp_top[tid]; low = s.warp_low[tid];
    for (int o = 16; o; o >>= 1) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    if (tid < WIDE_CTAS) {
      *cluster.map_shared_rank(&s.top[cluster_rank()], tid) = top;
      *cluster.map_shared_rank(&s.low[cluster_rank()], tid) = low;
    }
  }
  cluster.sync();
  top = 0; low = ~0ull;
#pragma unroll
  for (int r = 0; r < WIDE_CTAS; ++r) { top = max(top, s.top[r]); low = min(low, s.low[r]); }
  *top_of = top; *low_of = low;
}
// Sum over the cluster in a fixed order, in every CTA.
__device__ double wide_sum(WideShared& s, double v) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((tid & 31) == 0) s.warp_sum[tid >> 5] = v;
  __syncthreads();
  if (tid < 32) {
    v = s.warp_sum[tid];
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (tid < WIDE_CTAS) *cluster.map_shared_rank(&s.part[cluster_rank()], tid) = v;
  }
  cluster.sync();
  v = 0.0;
#pragma unroll
  for (int r = 0; r < WIDE_CTAS; ++r) v += s.part[r];
  cluster.sync();
  return v;
}

// The sums of the threads before this one; all threads of the CTA.
__device__ __forceinline__ double wide_before(WideShared& s, double v, uint32_t c, uint32_t* count) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double up = v;
  uint32_t cup = c;
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, up, o);
    const uint32_t tc = __shfl_up_sync(0xffffffffu, cup, o);
    if (lane >= o) { up += t; cup += tc; }
  }
  __syncthreads();
  if (lane == 31) { s.warp_sum[warp] = up; s.warp_count[warp] = cup; }
  __syncthreads();
  double of = s.warp_sum[lane];
  uint32_t cof = s.warp_count[lane];
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, of, o);
    const uint32_t tc = __shfl_up_sync(0xffffffffu, cof, o);
    if (lane >= o) { of += t; cof += tc; }
  }
  const double before = __shfl_sync(0xffffffffu, of, warp - 1);
  const uint32_t cbefore = __shfl_sync(0xffffffffu, cof, warp - 1);
  const double mine = __shfl_up_sync(0xffffffffu, up, 1);
  const uint32_t cmine = __shfl_up_sync(0xffffffffu, cup, 1);
  *count = (warp ? cbefore : 0u) + (lane ? cmine : 0u);
  return (warp ? before : 0.0) + (lane ? mine : 0.0);
}

// The tokens that `place` gives a bin (none: -1) into this CTA's bins. A weight goes in as a whole number of 64 bits, of which as many are left free as the
// sum of this CTA's tokens needs: whole numbers add up to the same sum in any order. (2^14 tokens in multiples of 2^-49 of a bin's largest weight, 2^18 in
// multiples of 2^-45, so that as many of the largest weight add up to 2^63. `whole`: the bin that all of these are parts of, -1: they are the row's. Multiples of
// the row's largest weight instead of the bin's moved draws that lie among tokens of 1e-11 of it. Two words, the first one's carry goes with the second: three words of 18 bits each took 15.5 thousand tokens 18,000 cycles.)
template <typename T, typename F>
__device__ __forceinline__ void wide_tally(const WidePart<T>& part, const WideScale& c, double power, bool counts, int whole, F place) {
  WideShared& s = part.s;
  for (int b = threadIdx.x; b < WIDE_BINS * (1 + WIDE_WORDS); b += WIDE_THREADS) s.bins.count[b] = 0;  // (and the masses behind the counts)
  __syncthreads();
  const ExpLanes exps(power);
  const double one = part.held ? 0x1p49 : 0x1p45, m = c.m;
  static_assert(WIDE_HELD <= 1 << 14 && SAMPLE_MAX_VOCAB / WIDE_CTAS <= 1 << 18, "no sum runs over: it stays below 2^64");
  part.each([&](float x, int i) {
    double w = exps.add(0.0, (static_cast<double>(x) - m) * c.step);
    if (x < c.floor) w = 0.0;
    if (c.m == INFINITY) w = x == c.m ? 1.0 : 0.0;
    const int b = x == -INFINITY ? -1 : place(x, i);
    if (b < 0) return;
    if (counts) atomicAdd(&s.bins.count[b], 1u);
    const int lift = c.lift(whole < 0 ? b : whole);
    const unsigned long long f = __double2ull_rn(w * one * __hiloint2double((1023 + lift) << 20, 0));
    const uint32_t low = static_cast<uint32_t>(f);
    uint32_t high = static_cast<uint32_t>(f >> 32);
    if (low) high += atomicAdd(&s.bins.mass[0][b], low) > ~low;
    if (high) atomicAdd(&s.bins.mass[1][b], high);
  });
}

// The CTAs' bins to sums up to each bin, in the first CTA.
__device__ __noinline__ void wide_tabulate(WideShared& s, WideScale c, bool finer, int whole, bool held) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  cluster.sync();
  // a thread for each number of the bins that this CTA adds up: a warp's lanes read neighbours from one CTA after the other
  constexpr int OWN = WIDE_BINS / WIDE_CTAS;
  static_assert(OWN * (1 + WIDE_WORDS) <= WIDE_THREADS, "a thread for each number");
  const int b = cluster_rank() * OWN + tid % OWN, l = tid / OWN;
  if (l <= WIDE_WORDS) {
    unsigned long long sum = 0;
#pragma unroll
    for (int r = 0; r < WIDE_CTAS; ++r) sum += *cluster.map_shared_rank(&s.bins.count[l * WIDE_BINS + b], r);
    s.sums[l][tid % OWN] = sum;
  }
  __syncthreads();
  if (tid < OWN) {
    WideTable* table = cluster.map_shared_rank(finer ? &s.finer : &s.first, 0);
    table->count[b] = static_cast<uint32_t>(s.sums[0][tid]);
    const double unit = (held ? 0x1p-49 : 0x1p-45) * __hiloint2double((1023 - c.lift(whole < 0 ? b : whole)) << 20, 0);
    table->mass[b] = (static_cast<double>(s.sums[2][tid]) * 0x1p32 + static_cast<double>(s.sums[1][tid])) * unit;
  }
  cluster.sync();
  if (cluster_rank() != 0) return;
  constexpr int PER = WIDE_BINS / WIDE_THREADS;
  WideTable& t = finer ? s.finer : s.first;
  uint32_t n[PER];
  double v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    n[j] = t.count[tid * PER + j] + (j ? n[j - 1] : 0u);
    v[j] = t.mass[tid * PER + j] + (j ? v[j - 1] : 0.0);
  }
  uint32_t before_c = 0;
  const double before = wide_before(s, v[PER - 1], n[PER - 1], &before_c);
#pragma unroll
  for (int j = 0; j < PER; ++j) { t.count[tid * PER + j] = before_c + n[j]; t.mass[tid * PER + j] = before + v[j]; }
  __syncthreads();
}

// The first CTA looks for the bin with the place: the first one up to which more than `target` of the weight stands, or (by_count)
// at least `rank_target` tokens; the last one with any, if there is none. Behind the barrier all CTAs know the bin.
__device__ __noinline__ void wide_find(WideShared& s, bool finer, bool by_count, uint32_t rank_target, double target, uint32_t base_count,
                                       double base_mass) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x;
  if (cluster_rank() == 0) {
    const WideTable& t = finer ? s.finer : s.first;
    if (tid == 0) s.bin = -1;
    __syncthreads();
    for (int b = tid; b < WIDE_BINS; b += WIDE_THREADS) {
      const bool here = by_count ? base_count + t.count[b] >= rank_target : base_mass + t.mass[b] > target;
      const bool before = b > 0 && (by_count ? base_count + t.count[b - 1] >= rank_target : base_mass + t.mass[b - 1] > target);
      if (here && !before) s.bin = b;
    }
    __syncthreads();
    if (s.bin < 0) {  // all of it stands before the target, by a rounding or by more: the last bin that has any
      __syncthreads();
      for (int b = tid; b < WIDE_BINS; b += WIDE_THREADS) {
        const bool any = by_count ? t.count[b] == t.count[WIDE_BINS - 1] && t.count[b] > (b ? t.count[b - 1] : 0u)
                                  : t.mass[b] == t.mass[WIDE_BINS - 1] && t.mass[b] > (b ? t.mass[b - 1] : 0.0);
        if (any) s.bin = b;
      }
      __syncthreads();
    }
    const int b = max(s.bin, 0);
    if (tid < WIDE_CTAS) {
      *cluster.map_shared_rank(&s.bin, tid) = b;
      *cluster.map_shared_rank(&s.members, tid) = t.count[b] - (b ? t.count[b - 1] : 0u);
    }
    if (tid == 0) {
      s.base_count = base_count + (b ? t.count[b - 1] : 0u);
      s.base_mass = base_mass + (b ? t.mass[b - 1] : 0.0);
    }
  }
  cluster.sync();
}

// The place in the row's order: by count the token of rank `rank_target` (from 1), by weight the first one up to which more than
// `target` stands (target: the first CTA's). Leaves comp in s.cut of every CTA, the weight up to and with it in s.cut_mass of the first.
template <typename T>
__device__ __noinline__ void wide_search(WidePart<T> part, WideScale c, double power, bool by_count, uint32_t rank_target, double target) {
  cg::cluster_group cluster = cg::this_cluster();
  WideShared& s = part.s;
  const int tid = threadIdx.x;
  const bool first = cluster_rank() == 0;
  wide_find(s, false, by_count, rank_target, target, 0, 0.0);
  const int bin = s.bin;
  float hi = c.m - bin / c.scale, lo = c.m - (bin + 1) / c.scale;
  uint64_t range_lo = 0, range_hi = ~0ull;  // of the members
  uint32_t* listed = cluster.map_shared_rank(&s.listed, 0);
  for (;;) {
    if (first && tid == 0) s.listed = 0;
    cluster.sync();  // (also: the bins have been read, the list takes their place)
    uint64_t* item = cluster.map_shared_rank(s.list.item, 0);
    part.each([&](float x, int i) {
      if (x == -INFINITY || c.bin(x) != bin) return;
      const uint64_t comp = comp_of(x, i);
      if (comp < range_lo || comp > range_hi) return;
      const uint32_t to = atomicAdd(listed, 1u);
      if (to < LIST) item[to] = comp;
    });
    cluster.sync();
    uint32_t members = *listed;
    if (members <= LIST) break;
    // bins within the bin, until the place's has few enough
    uint64_t top = 0, low = ~0ull;
    part.each([&](float x, int i) {
      if (x == -INFINITY || c.bin(x) != bin) return;
      top = max(top, comp_of(x, i)); low = min(low, comp_of(x, i));
    });
    wide_extremes(s, &top, &low);
    range_lo = low; range_hi = top;
    while (members > LIST) {
      const int bits = 64 - __clzll(range_hi - range_lo), shift = max(0, bits - 11);
      wide_tally(part, c, power, true, bin, [&](float x, int i) {
        const uint64_t comp = comp_of(x, i);
        return c.bin(x) == bin && comp >= range_lo && comp <= range_hi ? static_cast<int>((range_hi - comp) >> shift) : -1;
      });
      wide_tabulate(s, c, true, bin, part.held);
      wide_find(s, true, by_count, rank_target, target, s.base_count, s.base_mass);
      members = s.members;
      range_hi -= static_cast<uint64_t>(s.bin) << shift;
      const uint64_t wide = (1ull << shift) - 1;
      range_lo = range_hi - range_lo > wide ? range_hi - wide : range_lo;
      cluster.sync();  // s.bin and s.members are read before the next find
    }
    hi = comp_value(range_hi); lo = comp_value(range_lo);
  }
  if (first) {
    const int n = min(static_cast<int>(s.listed), LIST);
    order_list<WIDE_THREADS>(s.list, n, hi, lo);
    constexpr int PER = LIST / WIDE_THREADS, NONE = 1 << 30;
    double v[PER];
    bool adds[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int i = tid * PER + j;
      const double w = i < n ? weight_of(comp_value(s.list.item[i]), c.m, c.inv_t) : 0.0;
      adds[j] = w > 0.0;
      v[j] = w + (j ? v[j - 1] : 0.0);
    }
    uint32_t none;
    const double before = s.base_mass + wide_before(s, v[PER - 1], 0, &none);
    if (tid == 0) { s.place = NONE; s.bin = 0; }
    __syncthreads();
    int last = -1;
#pragma unroll
    for (int j = PER - 1; j >= 0; --j) {
      const int i = tid * PER + j;
      if (by_count ? i + 1 + s.base_count == rank_target : before + v[j] > target && i < n) atomicMin(&s.place, i);
      if (adds[j] && last < 0) last = i;
    }
    if (last >= 0) atomicMax(&s.bin, last);  // where the weight ends, should all of it stand before the target by a rounding
    __syncthreads();
    const int at = s.place < n ? s.place : by_count ? n - 1 : s.bin;
    __syncthreads();
    if (tid < WIDE_CTAS) *cluster.map_shared_rank(&s.cut, tid) = s.list.item[at];
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (tid * PER + j == at) s.cut_mass = before + v[j];
  }
  cluster.sync();
}

template <typename T>
__device__ __forceinline__ void sample_wide_row(const SampleArgs& a, const SampleWork& work, int at, WideShared& s) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, rank = cluster_rank(), per = (a.V + WIDE_CTAS - 1) / WIDE_CTAS;
  const WidePart<T> part{s, static_cast<const T*>(a.logits) + at * a.stride, min(a.V, rank * per), min(a.V, (rank + 1) * per), per <= WIDE_HELD};
  const float temperature = a.temperature[at];
  const int k = a.top_k[at];
  const double p = a.top_p[at], least = a.min_p[at], u = a.u[at], power = work.powers[tid & 31];
  const SamplePlan& plan = work.plan[at];
  if (tid == 0) s.n_banned = 0;
  if (part.held) {
#pragma unroll 8
    for (int i = part.begin + tid; i < part.end; i += WIDE_THREADS) s.held[i - part.begin] = logit_value(part.row[i]);
  }
  __syncthreads();
  for (int j = tid; j < a.n_exclude; j += WIDE_THREADS) {
    const int id = a.exclude[static_cast<long long>(at) * a.n_exclude + j];
    if (id < part.begin || id >= part.end) continue;
    if (part.held) s.held[id - part.begin] = -INFINITY;
    else s.banned[atomicAdd(&s.n_banned, 1)] = id;
  }
  cluster.sync();  // (also: every CTA of the cluster is there, before anything is written into it)
  uint64_t top = plan.top, low = comp_of(plan.low, 0);
  if (top == 0) {
    float hi = -INFINITY, lo = INFINITY;
    int id = 0;
    part.each([&](float x, int i) {
      if (x > hi) { hi = x; id = i; }  // (the first of a thread's)
      if (x != -INFINITY) lo = fminf(lo, x);
    });
    top = comp_of(hi, id);
    low = top ? comp_of(lo, 0) : ~0ull;
    wide_extremes(s, &top, &low);
  }
  const bool first = rank == 0 && tid == 0;
  if (top == 0 || !(temperature > 0.f)) {
    if (first) a.out[at] = top ? comp_id(top) : -1;
    return;  // (nothing reaches into another CTA behind `wide_extremes`)
  }
  const bool cut_k = k > 0 && k < a.V;
  WideScale c;
  c.m = comp_value(top);
  c.inv_t = 1.0 / static_cast<double>(temperature);
  c.step = c.inv_t * STEPS;
  c.floor = fmaxf(c.m - WIDE_RANGE * temperature, -FLT_MAX);
  const float range = fminf(fminf(WIDE_RANGE * temperature, c.m - comp_value(low)), 1e38f);
  c.scale = range > 0.f ? fminf(WIDE_BINS / range, 1e38f) : 0.f;
  c.fall = c.scale > 0.f ? static_cast<float>(c.inv_t / c.scale * 1.4426950408889634) : 0.f;
  wide_tally(part, c, power, cut_k, -1, [&](float x, int) { return c.bin(x); });
  wide_tabulate(s, c, false, -1, part.held);

  uint64_t cut = 0;
  double total = s.first.mass[WIDE_BINS - 1];  // (the first CTA's numbers; nobody else uses them)
  if (cut_k) {
    wide_search(part, c, power, true, static_cast<uint32_t>(k), 0.0);
    cut = s.cut;
    total = s.cut_mass;
  }
  if (p < 1.0) {
    wide_search(part, c, power, false, 0, p * total);
    if (s.cut >= cut) { cut = s.cut; total = s.cut_mass; }
  }
  if (least > 0.0) {  // the weight of what min-p leaves, and its last token
    double mass = 0.0;
    uint64_t last = ~0ull, none = 0;
    part.each([&](float x, int i) {
      const uint64_t comp = comp_of(x, i);
      if (comp == 0 || comp < cut) return;
      const double w = weight_of(x, c.m, c.inv_t);
      if (w >= least || comp == top) { mass += w; last = min(last, comp); }
    });
    total = wide_sum(s, mass);
    wide_extremes(s, &none, &last);
    cut = last;
    cluster.sync();
  }
  wide_search(part, c, power, false, 0, u * total);
  if (first) a.out[at] = comp_id(s.cut > cut ? s.cut : cut);
}

// The rows that the stream left to this kernel: a cluster takes one after the other.
template <typename T>
__global__ void __launch_bounds__(WIDE_THREADS) sample_wide_kernel(SampleArgs a, SampleWork w) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  WideShared& s = *reinterpret_cast<WideShared*>(smem_raw);
  pdl_wait();
  pdl_launch();
  const int rows = *w.left;
  if (static_cast<int>(blockIdx.x / WIDE_CTAS) >= rows) return;
  for (int i = blockIdx.x / WIDE_CTAS; i < rows; i += gridDim.x / WIDE_CTAS) {
    sample_wide_row<T>(a, w, w.left_rows[i], s);
    cg::this_cluster().sync();  // everyone has read what the next row writes over
  }
}

// ------------------------------------------------------------------ the stream
// Most rows are decided by their largest tokens. Three launches:
//  plan    a CTA per row looks at 16,384 of its logits and guesses a threshold that about `want` tokens reach;
//  stream  reads every logit once: tokens that reach the threshold go into the row's list, the weights of the others into the row's tail.
//          The CTA that finishes a row last puts the list in order and searches it; a row whose place lies in the tail (or whose
//          list has run over) is left to
//  wide    the kernel above.
// A guess that is off costs time, never a result: what the list and the tail say is exact.
//
// Rows of 248,320 fp32 logits, device time: one row 15 us (three launches, each a chain of latencies), 16 rows 28, 128 of mixed settings 86, 256 open ones
// 137: plan 10, stream 70 (254 MB: 3.6 TB/s; a number takes about ten instructions, which bound it before the memory does, and a row's end 13 us), wide 30
// to 60.
//
// Sums are added up in an order that goes by V alone: the weights of a lane's tokens of a task, the lanes of a warp, the tasks of a row.
constexpr int PLAN_THREADS = 512, PLAN_PER = 32, PLAN_SAMPLE = PLAN_THREADS * PLAN_PER, PLAN_BLOCK = 256, PLAN_BINS = 1024;
constexpr int STREAM_THREADS = 256, STREAM_WARPS = STREAM_THREADS / 32, STREAM_PER_SM = 4;
constexpr int TASK = 1024;          // tokens that a warp adds up by itself, in two halves
constexpr int LIST_K = 1024;        // top-k up to which a list is expected to hold the k tokens

// What a list is made to hold: all of the k, with room for the guess's error (one part in sqrt(want * 16384 / V): of 248,320 tokens the sample has 11 for a k
// of 20, and less than two of them stand among the k), or as many as leave room above. (2 k + 64: one row of 128 had too few, and took 25 us more.)
__device__ __forceinline__ int list_want(bool greedy, int k) {
  if (greedy) return 48;
  if (k <= 0) return 1400;
  return min(2 * k + 128, 1500);
}

// The settings of a row in a form that all CTAs agree on.
struct RowAsk {
  bool greedy, cut_k;  // cut_k: top-k leaves something out
  int k;
  double p, least, u, inv_t;
  __device__ RowAsk(const SampleArgs& a, int at) {
    const float t = a.temperature[at];
    greedy = !(t > 0.f);
    k = a.top_k[at];
    cut_k = k > 0 && k < a.V;
    p = a.top_p[at];
    least = a.min_p[at];
    u = a.u[at];
    inv_t = greedy ? 1.0 : 1.0 / static_cast<double>(t);
  }
};

// Sums over the threads before this one, in a fixed order; `warp_sum` holds one number per warp. All threads of the CTA.
template <int THREADS>
__device__ __forceinline__ double sum_before(double v, double* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double up = v;
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += t;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = up;
  __syncthreads();
  double before = 0.0;
  for (int w = 0; w < warp; ++w) before += warp_sum[w];
  const double mine = __shfl_up_sync(0xffffffffu, up, 1);
  return before + (lane ? mine : 0.0);
}

struct ListShared {
  Order list;
  double warp_sum[STREAM_WARPS];
  double total;
  int place, last;
};

// By how much a tail's sum in fp32 may be off, as a share of it. A token's weight is 2^y, y = logit * slope - zero: slope and y are rounded (2^-24 of y
// each, times ln 2 in the weight), 2^y is off by 2^-21 of itself, eight additions by 2^-24 each: (1.4 |y| + 8 + 8) 2^-24. Tokens with y below -40 add up to
// less than 2^22 2^-40, so what they are off by is within the 2^-30 that is added; |y| of 40 gives 72 2^-24, 75 is taken for the sums that follow.
constexpr double TAIL_OFF = 75 * 0x1p-24;

// The pick of a row from its `c` largest tokens in s.list (unsorted) and the weight of all others, within `off` of `tail`, relative to `ref`; all: there
// are no others of any weight. -2 where that does not decide it. All threads of a CTA of STREAM_THREADS.
__device__ int pick_from_list(ListShared& s, int c, const RowAsk& r, double tail, double off, float ref, bool all, float hi, float lo) {
  const int tid = threadIdx.x;
  if (c == 0) return ref == -INFINITY && all ? -1 : -2;
  order_list<STREAM_THREADS>(s.list, c, hi, lo);
  if (r.greedy) return comp_id(s.list.item[0]);
  const float m = comp_value(s.list.item[0]);
  // what weighs nothing beside `ref` weighs nothing beside m as well, unless m lies far below (an excluded token is the largest)
  if ((static_cast<double>(ref) - static_cast<double>(m)) * r.inv_t > WIDE_RANGE / 4) return -2;
  if (tail > 0.0 && ref != m) {
    const double by = exp((static_cast<double>(ref) - static_cast<double>(m)) * r.inv_t);
    tail *= by;
    off *= by;
  }
  if (!(tail < 1e300)) return -2;
  if (r.cut_k && c < r.k && !all) return -2;
  const int nk = r.cut_k ? min(r.k, c) : c;
  const bool closed = r.cut_k || all;  // no token outside the list is in play

  int positive = 0, enough = 0;
#pragma unroll 1
  for (int i = tid; i < nk; i += STREAM_THREADS) {
    const double w = weight_of(comp_value(s.list.item[i]), m, r.inv_t);
    positive += w > 0.0;
    enough += w >= r.least;
    s.list.sum[i] = w;
  }
  if (tid == 0) { s.place = s.last = 0; }
  __syncthreads();
  const int per = (nk + STREAM_THREADS - 1) / STREAM_THREADS, from = min(nk, tid * per), to = min(nk, from + per);
  double sum = 0.0;
#pragma unroll 1
  for (int i = from; i < to; ++i) { sum += s.list.sum[i]; s.list.sum[i] = sum; }
  const double before = sum_before<STREAM_THREADS>(sum, s.warp_sum);
#pragma unroll 1
  for (int i = from; i < to; ++i) s.list.sum[i] += before;
  for (int o = 16; o; o >>= 1) { positive += __shfl_xor_sync(0xffffffffu, positive, o); enough += __shfl_xor_sync(0xffffffffu, enough, o); }
  if ((tid & 31) == 0) { atomicAdd(&s.place, positive); atomicAdd(&s.last, enough); }
  __syncthreads();
  positive = s.place; enough = max(1, s.last);  // (neither is written again)
  // the weight that top-p goes by, and then that of the kept, lies between these
  double least_sum = s.list.sum[nk - 1], most_sum = least_sum;
  if (!closed) {
    least_sum += fmax(tail - off, 0.0);
    most_sum += tail + off;
  }
  constexpr int OPEN = 1 << 30;
  int limit = closed ? nk : OPEN;
  // A place with more than `target` up to it and no more before it, OPEN if there is none: each warp looks for it by itself, at 32 places and then between two.
  const int lane = tid & 31, stride = (nk + 31) / 32;
  const auto find = [&](double target) {
    const uint32_t ends = __ballot_sync(0xffffffffu, s.list.sum[min(nk, (lane + 1) * stride) - 1] > target);
    if (ends == 0) return OPEN;
    const int first = (__ffs(ends) - 1) * stride;
    static_assert(LIST <= 32 * 64, "two places for each lane");
    const uint32_t low = __ballot_sync(0xffffffffu, s.list.sum[min(nk - 1, first + lane)] > target);
    const uint32_t high = __ballot_sync(0xffffffffu, s.list.sum[min(nk - 1, first + 32 + lane)] > target);
    return first + (low ? __ffs(low) - 1 : 31 + __ffs(high));
  };
  if (r.p < 1.0) {
    const int at = find(r.p * least_sum);
    if (!closed && at != find(r.p * most_sum)) return -2;
    if (at != OPEN) {
      limit = at + 1;
    } else if (!closed) {  // the nucleus ends in the tail: its weight is p of the sum and up to one token's more
      least_sum *= r.p;
      most_sum = r.p * most_sum + weight_of(comp_value(s.list.item[c - 1]), m, r.inv_t);
    }
  }
  if (r.least > 0.0) {
    if (enough < nk || closed) limit = min(limit, enough);
    else if (limit == OPEN) return -2;
  }
  if (limit != OPEN) least_sum = most_sum = s.list.sum[limit - 1];
  const int at = find(r.u * least_sum);
  if (limit == OPEN) return at != OPEN && at == find(r.u * most_sum * (1.0 + 0x1p-40)) ? comp_id(s.list.item[at]) : -2;
  return comp_id(s.list.item[at < limit ? at : max(0, min(limit, positive) - 1)]);
}

template <typename T>
__global__ void __launch_bounds__(PLAN_THREADS) sample_plan_kernel(SampleArgs a, SampleWork w) {
  __shared__ uint32_t bins[PLAN_BINS];
  __shared__ float warp_top[PLAN_THREADS / 32], warp_low[PLAN_THREADS / 32], warp_over[PLAN_THREADS / 32];
  __shared__ uint32_t warp_count[PLAN_THREADS / 32];
  __shared__ int found;
  pdl_wait();
  pdl_launch();
  const int at = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const T* row = static_cast<const T*>(a.logits) + at * a.stride;
  if (at == 0 && tid == 0) *w.left = 0;
  if (at == 0 && tid < 32) w.powers[tid] = exp2(tid / 32.0);
  for (int b = tid; b < PLAN_BINS; b += PLAN_THREADS) bins[b] = 0;
  if (tid == 0) found = -1;
  float x[PLAN_PER];
  float top = -INFINITY, low = INFINITY;
  const bool whole = V <= PLAN_SAMPLE;
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i) {
    int id = i * PLAN_THREADS + tid;
    if (!whole) {
      const int block = i * (PLAN_THREADS / PLAN_BLOCK) + tid / PLAN_BLOCK;
      id = block * ((V - PLAN_BLOCK) / (PLAN_SAMPLE / PLAN_BLOCK - 1)) + tid % PLAN_BLOCK;
    }
    x[i] = id < V ? logit_value(row[id]) : -INFINITY;
    top = fmaxf(top, x[i]);
    if (x[i] != -INFINITY) low = fminf(low, x[i]);
  }
  const RowAsk ask(a, at);  // (behind the logits' loads: its division waits for the temperature)
  const int want = list_want(ask.greedy, ask.cut_k ? ask.k : 0);
  const uint32_t share = max(1u, static_cast<uint32_t>(static_cast<long long>(want) * min(V, PLAN_SAMPLE) / V));
  // `share` tokens of the sample lie at `over` or above, if as many groups of lanes each have one: of the others none need be counted
  float over = INFINITY;
  int lanes = 32;  // of a group
  while (lanes > 1 && PLAN_THREADS / lanes < static_cast<int>(share)) lanes >>= 1;
  for (int o = 1; o < 32; o <<= 1) {
    if (o == lanes) over = top;
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if (lanes == 32) over = top;
  for (int o = 16; o; o >>= 1) over = fminf(over, __shfl_xor_sync(0xffffffffu, over, o));
  if (lane == 0) { warp_top[warp] = top; warp_low[warp] = low; warp_over[warp] = over; }
  __syncthreads();
  for (int i = 0; i < PLAN_THREADS / 32; ++i) { top = fmaxf(top, warp_top[i]); low = fminf(low, warp_low[i]); over = fminf(over, warp_over[i]); }
  if (PLAN_THREADS / lanes < static_cast<int>(share)) over = low;
  const float t = ask.greedy ? 1.f : a.temperature[at];
  const float least = fmaxf(top - WIDE_RANGE * t, -FLT_MAX);  // below it nothing has any weight
  const float range = fminf(fminf(WIDE_RANGE * t, top - fmaxf(low, over)), 1e38f);
  const float scale = range > 0.f ? fminf(PLAN_BINS / range, 1e38f) : 0.f;
  const float count_from = fmaxf(least, over);
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i)
    if (x[i] >= count_from) atomicAdd(&bins[min(PLAN_BINS - 1, static_cast<int>((top - x[i]) * scale))], 1u);
  __syncthreads();
  // the bin in which the sample has its share of `want`
  static_assert(PLAN_BINS == 2 * PLAN_THREADS, "two bins for each thread");
  const uint32_t c0 = bins[2 * tid], c1 = bins[2 * tid + 1];
  uint32_t up = c0 + c1;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) warp_count[warp] = up;
  __syncthreads();
  for (int i = 0; i < warp; ++i) up += warp_count[i];
  if (up >= share && up - c1 < share) found = 2 * tid + 1;
  if (up - c1 >= share && up - c1 - c0 < share) found = 2 * tid;
  __syncthreads();
  if (tid == 0) {
    float reach = found < 0 || scale == 0.f ? least : fmaxf(top - (found + 1) / scale, least);
    const bool number = reach == reach;  // (infinite logits at an infinite temperature)
    SamplePlan plan;
    plan.reach = number ? reach : -FLT_MAX;
    plan.least = number ? least : -FLT_MAX;
    plan.ref = top;
    plan.low = low;
    plan.top = 0;
    const double slope = ask.inv_t * 1.4426950408889634;  // 1 / ln 2
    plan.slope = static_cast<float>(slope);
    plan.zero = top * plan.slope;
    plan.tail_by = exp2(static_cast<double>(plan.zero) - static_cast<double>(top) * plan.slope);
    plan.with_tail = !ask.greedy && !ask.cut_k && plan.reach > plan.least;
    plan.listed = 0;
    plan.done = 0;
    // (at a huge temperature even a token of `least` weighs something; at |zero| of 2^20 fp32 does not tell weights apart)
    plan.skip = (ask.cut_k && ask.k > LIST_K && reach > least) || t > 1e30f || (plan.with_tail && !(fabsf(plan.zero) < 0x1p20f));
    w.plan[at] = plan;
  }
}

__device__ __forceinline__ float exp2_fast(float y) {  // off by 2^-21 of the result at most
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return r;
}

constexpr int HALF = TASK / 2;
constexpr int SEEN = LIST / STREAM_WARPS;  // entries that a warp has room for

// The logits of a lane in half a task, from `row` on: piece i of 16 bytes holds tokens first + i * 32 * VE ..
template <typename T>
struct HalfLogits {
  static constexpr int VE = 16 / sizeof(T), PIECES = HALF / (32 * VE);
  static __device__ __forceinline__ int id(int first, int e) { return first + e / VE * (32 * VE) + e % VE; }
  uint4 raw[PIECES];
  __device__ __forceinline__ void load(const T* row, int first, int V, bool whole) {  // whole: all of it is there, in pieces of 16 bytes
    if (whole) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(row + first) + i * 32);
      return;
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      T one[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) one[j] = id(first, i * VE + j) < V ? row[id(first, i * VE + j)] : static_cast<T>(-INFINITY);
      memcpy(&raw[i], one, 16);
    }
  }
  __device__ __forceinline__ float value(int e) const {
    T one[VE];
    memcpy(one, &raw[e / VE], 16);
    return static_cast<float>(one[e % VE]);
  }
  // minus infinity in the place of the tokens named
  __device__ __forceinline__ void strike(int first, const int* ids, int n) {
    for (int b = 0; b < n; ++b)
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        T one[VE];
        memcpy(one, &raw[i], 16);
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (id(first, i * VE + j) == ids[b]) one[j] = static_cast<T>(-INFINITY);
        memcpy(&raw[i], one, 16);
      }
  }
};

// CTA x of a row takes `tasks_per_warp` tasks for each warp, from task x * STREAM_WARPS * tasks_per_warp on.
template <typename T>
__global__ void __launch_bounds__(STREAM_THREADS, STREAM_PER_SM) sample_stream_kernel(SampleArgs a, SampleWork w, int tasks, int tasks_per_warp) {
  using Half = HalfLogits<T>;
  __shared__ ListShared s;
  __shared__ int banned[SAMPLE_MAX_EXCLUDE];
  __shared__ int n_banned;
  const int at = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  if (tid == 0) n_banned = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch();
  SamplePlan& plan = w.plan[at];
  const float slope = plan.slope, zero = plan.zero;
  const bool with_tail = plan.with_tail;
  if (plan.skip) {
    if (blockIdx.x == 0 && tid == 0) w.left_rows[atomicAdd(w.left, 1)] = at;
    return;
  }
  const float reach = plan.reach, least = plan.least, ref = plan.ref;
  const T* row = static_cast<const T*>(a.logits) + at * a.stride;
  const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
  const int task0 = blockIdx.x * STREAM_WARPS * tasks_per_warp;
  for (int j = tid; j < a.n_exclude; j += STREAM_THREADS) {
    const int id = a.exclude[static_cast<long long>(at) * a.n_exclude + j];
    if (id >= task0 * TASK && id < min(V, (task0 + STREAM_WARPS * tasks_per_warp) * TASK)) banned[atomicAdd(&n_banned, 1)] = id;
  }
  __syncthreads();
  const int bans = n_banned;
  uint64_t* list = w.list + static_cast<size_t>(at) * LIST;

  // The lanes that have seen tokens for the list, in the order of this warp's halves: first token << 16 | which of the lane's. (One entry for each token, by a
  // counter of the CTA's, took as long as all the rest: 256 open rows 111 -> 76 us.)
  uint64_t* seen = s.list.item + warp * SEEN;
  int n_seen = 0;
  float part[4] = {};
  const auto look = [&](Half& x, int first) {
    if (bans) x.strike(first, banned, bans);
    uint32_t hits = 0;
    if (with_tail) {
#pragma unroll
      for (int e = 0; e < HALF / 32; ++e) {
        const float v = x.value(e), weight = exp2_fast(fmaf(v, slope, -zero));
        if (v < reach) part[e & 3] += weight;
        if (v >= reach) hits |= 1u << e;  // (a NaN is in neither the list nor the tail)
      }
    } else {
#pragma unroll
      for (int e = 0; e < HALF / 32; ++e) hits |= x.value(e) >= reach ? 1u << e : 0u;
    }
    const uint32_t lanes = __ballot_sync(0xffffffffu, hits != 0);
    const int to = n_seen + __popc(lanes & ((1u << lane) - 1));
    if (hits && to < SEEN) seen[to] = static_cast<uint64_t>(first) << 16 | hits;
    n_seen += __popc(lanes);
  };
  // a half is on its way while the other is looked at
  const int stop = min(tasks, task0 + tasks_per_warp * STREAM_WARPS);
  const auto whole = [&](int task) { return aligned && (task + 1) * TASK <= V; };
  Half a0, a1;
  if (task0 + warp < stop) a0.load(row, (task0 + warp) * TASK + lane * Half::VE, V, whole(task0 + warp));
  for (int task = task0 + warp; task < stop; task += STREAM_WARPS) {
    const int first = task * TASK + lane * Half::VE;
    a1.load(row, first + HALF, V, whole(task));
    look(a0, first);
    if (task + STREAM_WARPS < stop) a0.load(row, first + STREAM_WARPS * TASK, V, whole(task + STREAM_WARPS));
    look(a1, first + HALF);
    if (with_tail) {
      double tail = static_cast<double>((part[0] + part[1]) + (part[2] + part[3]));
      part[0] = part[1] = part[2] = part[3] = 0.f;
      for (int o = 16; o; o >>= 1) tail += __shfl_xor_sync(0xffffffffu, tail, o);
      if (lane == 0) w.tail[static_cast<size_t>(at) * tasks + task] = tail;
    }
  }
  // this CTA's tokens into the row's list
  __syncwarp();
  int count = 0;
  for (int e = lane; e < min(n_seen, SEEN); e += 32) count += __popc(static_cast<uint32_t>(seen[e]) & 0xffffu);
  for (int o = 16; o; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
  if (n_seen > SEEN) count = LIST + 1;  // more than there is room for: the row is left to the search over bins
  if (lane == 0) s.list.warp_count[warp] = count;
  __syncthreads();
  if (tid == 0) {
    uint32_t sum = 0;
    for (int i = 0; i < STREAM_WARPS; ++i) sum += s.list.warp_count[i];
    s.place = sum ? atomicAdd(&plan.listed, sum) : 0;
  }
  __syncthreads();
  int at_list = s.place;
  for (int i = 0; i < warp; ++i) at_list += s.list.warp_count[i];
  for (int e0 = 0; e0 < min(n_seen, SEEN); e0 += 32) {
    const uint64_t entry = e0 + lane < min(n_seen, SEEN) ? seen[e0 + lane] : 0;
    uint32_t which = static_cast<uint32_t>(entry) & 0xffffu;
    const int mine = __popc(which);
    int up = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    for (int to = at_list + up - mine; which; which &= which - 1, ++to) {
      const int id = Half::id(static_cast<int>(entry >> 16), __ffs(which) - 1);
      if (to < LIST) list[to] = comp_of(logit_value(row[id]), id);
    }
    at_list += __shfl_sync(0xffffffffu, up, 31);
  }
  __syncthreads();
  if (tid == 0) {  // (one fence for the CTA, behind the barrier: a fence of every warp waited for the others')
    __threadfence();
    s.last = atomicAdd(&plan.done, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!s.last) return;
  // all of it is asked for at a time, the list without knowing how much of it there is
  const uint32_t listed = __ldcg(&plan.listed);
  uint64_t item[LIST / STREAM_THREADS];
#pragma unroll
  for (int j = 0; j < LIST / STREAM_THREADS; ++j) item[j] = __ldcg(list + j * STREAM_THREADS + tid);
  int pick = -2;
  if (listed <= LIST) {
    double tail = 0.0;
    if (with_tail)
      for (int i = tid; i < tasks; i += STREAM_THREADS) tail += __ldcg(w.tail + static_cast<size_t>(at) * tasks + i);
#pragma unroll
    for (int j = 0; j < LIST / STREAM_THREADS; ++j) s.list.item[j * STREAM_THREADS + tid] = item[j];
    if (with_tail) {
      const double before = sum_before<STREAM_THREADS>(tail, s.warp_sum);
      if (tid == STREAM_THREADS - 1) s.total = before + tail;
      __syncthreads();
      tail = s.total * plan.tail_by;
    }
    __syncthreads();
    pick = pick_from_list(s, static_cast<int>(listed), RowAsk(a, at), tail, tail * TAIL_OFF + 0x1p-30, ref, reach <= least, ref, reach);
  }
  if (tid == 0) {
    if (pick == -2) {
      if (listed > 0 && listed <= LIST) plan.top = s.list.item[0];
      w.left_rows[atomicAdd(w.left, 1)] = at;
    } else {
      a.out[at] = pick;
    }
  }
}

// A vocabulary that fits a list: one launch, a CTA per row.
template <typename T>
__global__ void __launch_bounds__(STREAM_THREADS) sample_short_kernel(SampleArgs a) {
  __shared__ ListShared s;
  __shared__ int listed;
  __shared__ uint32_t top, low;  // as order keys
  const int at = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) { listed = 0; top = 0; low = ~0u; }
  pdl_wait();
  pdl_launch();
  __syncthreads();
  const T* row = static_cast<const T*>(a.logits) + at * a.stride;
  for (int i = tid; i < a.V; i += STREAM_THREADS) {
    const uint64_t c = comp_of(logit_value(row[i]), i);
    bool out = c == 0;
    for (int j = 0; j < a.n_exclude; ++j) out |= a.exclude[static_cast<long long>(at) * a.n_exclude + j] == i;
    if (out) continue;
    s.list.item[atomicAdd(&listed, 1)] = c;
    atomicMax(&top, static_cast<uint32_t>(c >> 32));
    atomicMin(&low, static_cast<uint32_t>(c >> 32));
  }
  __syncthreads();
  const int pick = pick_from_list(s, listed, RowAsk(a, at), 0.0, 0.0, -INFINITY, true, key_value(top), key_value(low));
  if (tid == 0) a.out[at] = pick;
}

constexpr int MAX_DEVICES = 64;

static size_t align_up(size_t v) { return (v + 255) / 256 * 256; }
static int task_count(int V) { return (V + TASK - 1) / TASK; }

// Bytes of a call's workspace: [left][left rows][plans][lists][tails]
static size_t sample_work(int n, int V, void* base, SampleWork* w) {
  size_t at = 0;
  uint8_t* p = static_cast<uint8_t*>(base);
  const auto take = [&](size_t bytes) { uint8_t* r = p + at; at += align_up(bytes); return r; };
  w->left = reinterpret_cast<int*>(take(4));
  w->left_rows = reinterpret_cast<int*>(take(static_cast<size_t>(n) * 4));
  w->plan = reinterpret_cast<SamplePlan*>(take(static_cast<size_t>(n) * sizeof(SamplePlan)));
  w->list = reinterpret_cast<uint64_t*>(take(static_cast<size_t>(n) * LIST * 8));
  w->tail = reinterpret_cast<double*>(take(static_cast<size_t>(n) * task_count(V) * 8));
  w->powers = reinterpret_cast<double*>(take(32 * 8));
  return at;
}

template <typename T>
static int launch_sample(const SampleArgs& a, void* work, cudaStream_t st) {
  if (a.V <= LIST)
    return launch_pdl(sample_short_kernel<T>, dim3(a.n), dim3(STREAM_THREADS), 0, st, a) == cudaSuccess ? 0 : -4;
  static int sms[MAX_DEVICES] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= MAX_DEVICES) return -3;
  if (!sms[dev]) {
    if (cudaFuncSetAttribute(sample_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(WideShared)) != cudaSuccess) return -3;
    if (cudaFuncSetAttribute(sample_wide_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return -3;
    if (cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
  }
  SampleWork w;
  sample_work(a.n, a.V, work, &w);
  const int tasks = task_count(a.V);
  // CTAs of a row: those that take the least time in waves of what the SMs hold at once, where a CTA's own start and end count as four tasks
  const int units = (tasks + STREAM_WARPS - 1) / STREAM_WARPS;
  int ctas = 1, per = units;
  long long least = -1;
  for (int c = 1; c <= min(units, 64); ++c) {
    const int p = (units + c - 1) / c;
    const long long cost = (static_cast<long long>(c) * a.n + STREAM_PER_SM * sms[dev] - 1) / (STREAM_PER_SM * sms[dev]) * (p + 4);
    if (least < 0 || cost < least) { least = cost; per = p; ctas = (units + p - 1) / p; }
  }
  const int clusters = a.n < sms[dev] / WIDE_CTAS ? a.n : sms[dev] / WIDE_CTAS;
  if (launch_pdl(sample_plan_kernel<T>, dim3(a.n), dim3(PLAN_THREADS), 0, st, a, w) != cudaSuccess) return -4;
  if (launch_pdl(sample_stream_kernel<T>, dim3(ctas, a.n), dim3(STREAM_THREADS), 0, st, a, w, tasks, per) != cudaSuccess) return -4;
  return launch_clusters(WIDE_CTAS, sample_wide_kernel<T>, dim3(clusters * WIDE_CTAS), dim3(WIDE_THREADS), sizeof(WideShared), st, a, w) == cudaSuccess ? 0 : -4;
}

}  // namespace b200

using namespace b200;

extern "C" long long b200_sample_work_bytes(int n, int V) {
  SampleWork w;
  return V <= LIST ? 0 : static_cast<long long>(sample_work(n, V, nullptr, &w));
}

extern "C" int b200_sample(const void* logits, int type, long long stride, int n, int V, const float* temperature, const int* top_k,
                           const float* top_p, const float* min_p, const float* u, const int* exclude, int n_exclude, int64_t* out,
                           void* work, cudaStream_t st) {
  if (n <= 0) return 0;
  if (V <= 0 || n_exclude < 0 || n_exclude > SAMPLE_MAX_EXCLUDE || V > SAMPLE_MAX_VOCAB || n > 65535) return -7;
  const SampleArgs a{logits, stride, n, V, temperature, top_k, top_p, min_p, u, exclude, n_exclude, out};
  switch (type) {
    case LOGIT_F32: return launch_sample<float>(a, work, st);
    case LOGIT_BF16: return launch_sample<bf16>(a, work, st);
    case LOGIT_F16: return launch_sample<__half>(a, work, st);
  }
  return -7;
}

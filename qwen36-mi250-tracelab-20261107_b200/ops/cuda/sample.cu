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
// Weights and their sums are held in 64 bits: with 248,320 tokens kept, sums that were off by one part in 1e8 would move one draw in
// 400 to a neighbouring token, and a request's tokens would depend on how the sums were cut.
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
  float reach, least, ref;  // threshold of the list; below `least` a token has no weight; what the tail's weights are relative to
  int skip;                 // the list cannot decide this row
  uint32_t listed, done;    // tokens in the list, CTAs that have finished their part of the row
};
struct SampleWork {
  int* left;         // rows left to the wide kernel, and which
  int* left_rows;
  SamplePlan* plan;  // [n]
  uint64_t* list;    // [n, LIST]
  double* tail;      // [n, tasks]
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

constexpr int WIDE_CTAS = 8;       // of a row: one cluster
constexpr int WIDE_THREADS = 1024;
constexpr int WIDE_BATCH = 8;      // logits that a thread asks for at a time
constexpr int WIDE_BINS = 2048;
constexpr int WIDE_LIST = 2048;    // candidates that are put in order one by one
constexpr float WIDE_RANGE = 80.f; // e^-80 of the largest weight, 2^18 times, is nothing in 64 bits

struct WideTable {  // sums up to and with each bin, of the whole row
  uint32_t count[WIDE_BINS];
  double mass[WIDE_BINS];
};
struct WideShared {
  union {
    struct { uint32_t count[WIDE_BINS], m0[WIDE_BINS], m1[WIDE_BINS], m2[WIDE_BINS]; } bins;  // this CTA's part; a mass in 96 bits
    struct { uint64_t item[WIDE_LIST]; double mass[WIDE_LIST]; } list;                       // (of the first CTA)
  };
  WideTable first, finer;  // of the first CTA
  uint64_t top[WIDE_CTAS], low[WIDE_CTAS];  // every CTA's
  double part[WIDE_CTAS];
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
  uint32_t base_count;
  double base_mass, cut_mass;
};

// One row, one cluster. `T` is the type of the logits.
template <typename T>
struct WideRow {
  cg::cluster_group cluster = cg::this_cluster();
  WideShared& s;
  const T* row;
  const int rank, tid, V, begin, end;
  float m, scale;  // maximum; bins per unit of m - x
  double inv_t;
  uint64_t range_lo, range_hi;  // the members of the bin that a search is in

  __device__ WideRow(WideShared& sh, const T* r, int v, int per)
      : s(sh), row(r), rank(cluster_rank()), tid(threadIdx.x), V(v), begin(min(v, rank * per)), end(min(v, rank * per + per)) {}

  __device__ bool banned(int id) const {
    for (int j = 0; j < s.n_banned; ++j)
      if (s.banned[j] == id) return true;
    return false;
  }
  // f(x, comp) for every token of this CTA's part that counts
  template <typename F>
  __device__ void each(F f) const {
    for (int i0 = begin + tid; i0 < end; i0 += WIDE_THREADS * WIDE_BATCH) {
      T raw[WIDE_BATCH];
#pragma unroll
      for (int j = 0; j < WIDE_BATCH; ++j) raw[j] = i0 + j * WIDE_THREADS < end ? row[i0 + j * WIDE_THREADS] : static_cast<T>(-INFINITY);
#pragma unroll
      for (int j = 0; j < WIDE_BATCH; ++j) {
        const int i = i0 + j * WIDE_THREADS;
        const float x = logit_value(raw[j]);
        const uint64_t c = comp_of(x, i);
        if (c != 0 && !(s.n_banned && banned(i))) f(x, c);
      }
    }
  }
  __device__ int bin_of(float x) const { return min(WIDE_BINS - 1, static_cast<int>((m - x) * scale)); }

  // largest and smallest comp over the cluster, in every CTA (0 where there is none)
  __device__ void extremes(uint64_t& top, uint64_t& low) {
    for (int o = 16; o; o >>= 1) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    if ((tid & 31) == 0) { s.warp_top[tid >> 5] = top; s.warp_low[tid >> 5] = low; }
    __syncthreads();
    if (tid < WIDE_CTAS) {
      for (int w = 0; w < WIDE_THREADS / 32; ++w) { top = max(top, s.warp_top[w]); low = min(low, s.warp_low[w]); }
      *cluster.map_shared_rank(&s.top[rank], tid) = top;
      *cluster.map_shared_rank(&s.low[rank], tid) = low;
    }
    cluster.sync();
    top = 0; low = ~0ull;
    for (int r = 0; r < WIDE_CTAS; ++r) { top = max(top, s.top[r]); low = min(low, s.low[r]); }
  }
  // sum over the cluster in a fixed order, in every CTA
  __device__ double sum(double v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((tid & 31) == 0) s.warp_sum[tid >> 5] = v;
    __syncthreads();
    if (tid < WIDE_CTAS) {
      v = 0.0;
      for (int w = 0; w < WIDE_THREADS / 32; ++w) v += s.warp_sum[w];
      *cluster.map_shared_rank(&s.part[rank], tid) = v;
    }
    cluster.sync();
    v = 0.0;
    for (int r = 0; r < WIDE_CTAS; ++r) v += s.part[r];
    cluster.sync();
    return v;
  }

  __device__ void clear() {
    for (int b = tid; b < WIDE_BINS; b += WIDE_THREADS) s.bins.count[b] = s.bins.m0[b] = s.bins.m1[b] = s.bins.m2[b] = 0;
    __syncthreads();
  }
  // a weight as a whole number of 2^-62: integers add up to the same sum in any order
  __device__ void add(int b, double w) {
    atomicAdd(&s.bins.count[b], 1u);
    const unsigned long long f = __double2ull_rn(w * 0x1p62);
    const uint32_t lo = static_cast<uint32_t>(f);
    uint32_t hi = static_cast<uint32_t>(f >> 32);
    if (lo) hi += atomicAdd(&s.bins.m0[b], lo) > 0xffffffffu - lo;
    if (hi && atomicAdd(&s.bins.m1[b], hi) > 0xffffffffu - hi) atomicAdd(&s.bins.m2[b], 1u);
  }
  // the CTAs' bins to sums up to each bin, in the first CTA
  __device__ void tabulate(WideTable WideShared::*which) {
    cluster.sync();
    constexpr int OWN = WIDE_BINS / WIDE_CTAS;
    WideTable* table = cluster.map_shared_rank(&(s.*which), 0);
    if (tid < OWN) {
      const int b = rank * OWN + tid;
      unsigned long long count = 0, m0 = 0, m1 = 0, m2 = 0;
      for (int r = 0; r < WIDE_CTAS; ++r) {
        const auto* from = cluster.map_shared_rank(&s.bins, r);
        count += from->count[b]; m0 += from->m0[b]; m1 += from->m1[b]; m2 += from->m2[b];
      }
      table->count[b] = static_cast<uint32_t>(count);
      table->mass[b] = static_cast<double>(m2) * 4.0 + static_cast<double>(m1) * 0x1p-30 + static_cast<double>(m0) * 0x1p-62;
    }
    cluster.sync();
    if (rank != 0) return;
    constexpr int PER = WIDE_BINS / WIDE_THREADS;
    WideTable& t = s.*which;
    uint32_t c[PER];
    double v[PER];
    for (int j = 0; j < PER; ++j) {
      c[j] = t.count[tid * PER + j] + (j ? c[j - 1] : 0u);
      v[j] = t.mass[tid * PER + j] + (j ? v[j - 1] : 0.0);
    }
    uint32_t before_c = 0;
    const double before = scan_before(v[PER - 1], c[PER - 1], &before_c);
    for (int j = 0; j < PER; ++j) { t.count[tid * PER + j] = before_c + c[j]; t.mass[tid * PER + j] = before + v[j]; }
    __syncthreads();
  }
  // sums of the threads before this one; all threads of the CTA
  __device__ double scan_before(double v, uint32_t c, uint32_t* count) {
    const int lane = tid & 31, warp = tid >> 5;
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
    double before = 0.0;
    uint32_t cbefore = 0;
    for (int w = 0; w < warp; ++w) { before += s.warp_sum[w]; cbefore += s.warp_count[w]; }
    const double mine = __shfl_up_sync(0xffffffffu, up, 1);
    const uint32_t cmine = __shfl_up_sync(0xffffffffu, cup, 1);
    *count = cbefore + (lane ? cmine : 0u);
    return before + (lane ? mine : 0.0);
  }

  // The first CTA looks for the bin with the place: the first one up to which more than `target` of the weight stands, or (by_count)
  // at least `rank_target` tokens; the last one with any, if there is none. Behind the barrier all CTAs know the bin.
  __device__ void find_bin(const WideTable& t, bool by_count, uint32_t rank_target, double target, uint32_t base_count, double base_mass) {
    if (rank == 0) {
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
  __device__ void search(bool by_count, uint32_t rank_target, double target) {
    find_bin(s.first, by_count, rank_target, target, 0, 0.0);
    const int bin = s.bin;
    uint32_t members = s.members;
    range_lo = 0; range_hi = ~0ull;
    const auto member = [&](float x, uint64_t c) { return bin_of(x) == bin && c >= range_lo && c <= range_hi; };
    if (members > WIDE_LIST) {  // bins within the bin, until the place's has few enough
      uint64_t top = 0, low = ~0ull;
      each([&](float x, uint64_t c) { if (bin_of(x) == bin) { top = max(top, c); low = min(low, c); } });
      extremes(top, low);
      range_lo = low; range_hi = top;
      while (members > WIDE_LIST) {
        const int bits = 64 - __clzll(range_hi - range_lo);
        const int shift = max(0, bits - 11);
        clear();
        each([&](float x, uint64_t c) { if (member(x, c)) add(static_cast<int>((range_hi - c) >> shift), weight_of(x, m, inv_t)); });
        tabulate(&WideShared::finer);
        find_bin(s.finer, by_count, rank_target, target, s.base_count, s.base_mass);
        members = s.members;
        range_hi -= static_cast<uint64_t>(s.bin) << shift;
        const uint64_t wide = (1ull << shift) - 1;
        range_lo = range_hi - range_lo > wide ? range_hi - wide : range_lo;
        cluster.sync();  // s.bin and s.members are read before the next find
      }
    }
    if (rank == 0 && tid == 0) s.listed = 0;
    cluster.sync();  // (also: the bins have been read, the list takes their place)
    uint32_t* listed = cluster.map_shared_rank(&s.listed, 0);
    uint64_t* item = cluster.map_shared_rank(s.list.item, 0);
    each([&](float x, uint64_t c) { if (member(x, c)) { const uint32_t at = atomicAdd(listed, 1u); if (at < WIDE_LIST) item[at] = c; } });
    cluster.sync();
    if (rank == 0) {
      const int n = min(static_cast<int>(s.listed), WIDE_LIST);
      int size = 2;
      while (size < n) size <<= 1;
      for (int i = n + tid; i < size; i += WIDE_THREADS) s.list.item[i] = 0;
      sort_down<WIDE_THREADS>(s.list.item, size);
      constexpr int PER = WIDE_LIST / WIDE_THREADS;
      double v[PER];
      for (int j = 0; j < PER; ++j) {
        const int i = tid * PER + j;
        v[j] = (i < n ? weight_of(comp_value(s.list.item[i]), m, inv_t) : 0.0) + (j ? v[j - 1] : 0.0);
      }
      uint32_t none;
      const double before = s.base_mass + scan_before(v[PER - 1], 0, &none);
      for (int j = 0; j < PER; ++j) s.list.mass[tid * PER + j] = before + v[j];
      if (tid == 0) s.bin = -1;
      __syncthreads();
      if (by_count) {
        if (tid == 0) s.bin = min(n - 1, static_cast<int>(rank_target - 1 - s.base_count));
      } else {
        for (int i = tid; i < n; i += WIDE_THREADS)
          if (s.list.mass[i] > target && !(i > 0 && s.list.mass[i - 1] > target)) s.bin = i;
        __syncthreads();
        if (s.bin < 0) {  // as above: the last one that adds anything
          __syncthreads();
          for (int i = tid; i < n; i += WIDE_THREADS)
            if (s.list.mass[i] == s.list.mass[n - 1] && s.list.mass[i] > (i > 0 ? s.list.mass[i - 1] : s.base_mass)) s.bin = i;
        }
      }
      __syncthreads();
      const int at = max(0, s.bin);
      if (tid < WIDE_CTAS) *cluster.map_shared_rank(&s.cut, tid) = s.list.item[at];
      if (tid == 0) s.cut_mass = s.list.mass[at];
    }
    cluster.sync();
  }
};

template <typename T>
__device__ void sample_wide_row(const SampleArgs& a, int at, WideShared& s) {
  const int tid = threadIdx.x;
  const int per = (a.V + WIDE_CTAS * 8 - 1) / (WIDE_CTAS * 8) * 8;
  WideRow<T> r(s, static_cast<const T*>(a.logits) + at * a.stride, a.V, per);
  const float temperature = a.temperature[at];
  const int k = a.top_k[at];
  const double p = a.top_p[at], least = a.min_p[at], u = a.u[at];
  if (tid == 0) {
    int found = 0;
    for (int j = 0; j < a.n_exclude; ++j) {
      const int id = a.exclude[static_cast<long long>(at) * a.n_exclude + j];
      if (id >= r.begin && id < r.end) s.banned[found++] = id;
    }
    s.n_banned = found;
  }
  r.cluster.sync();  // (also: every CTA of the cluster is there, before anything is written into it)
  uint64_t top = 0, low = ~0ull;
  r.each([&](float, uint64_t c) { top = max(top, c); low = min(low, c); });
  r.extremes(top, low);
  const bool first = r.rank == 0 && tid == 0;
  if (top == 0 || !(temperature > 0.f)) {
    if (first) a.out[at] = top ? comp_id(top) : -1;
    return;  // (nothing reaches into another CTA behind `extremes`)
  }
  r.m = comp_value(top);
  r.inv_t = 1.0 / static_cast<double>(temperature);
  const float range = fminf(fminf(WIDE_RANGE * temperature, r.m - comp_value(low)), 1e38f);
  r.scale = range > 0.f ? WIDE_BINS / range : 0.f;
  if (!(r.scale < 1e38f)) r.scale = 1e38f;
  r.clear();
  r.each([&](float x, uint64_t c) { r.add(r.bin_of(x), weight_of(x, r.m, r.inv_t)); });
  r.tabulate(&WideShared::first);

  uint64_t cut = 0;
  double total = s.first.mass[WIDE_BINS - 1];  // (the first CTA's numbers; nobody else uses them)
  if (k > 0 && k < a.V) {
    r.search(true, static_cast<uint32_t>(k), 0.0);
    cut = s.cut;
    total = s.cut_mass;
  }
  if (p < 1.0) {
    r.search(false, 0, p * total);
    if (s.cut >= cut) { cut = s.cut; total = s.cut_mass; }
  }
  if (least > 0.0) {  // the weight of what min-p leaves, and its last token
    double mass = 0.0;
    uint64_t last = ~0ull, none = 0;
    r.each([&](float x, uint64_t c) {
      if (c < cut) return;
      const double w = weight_of(x, r.m, r.inv_t);
      if (w >= least || c == top) { mass += w; last = min(last, c); }
    });
    total = r.sum(mass);
    r.extremes(none, last);
    cut = last;
    r.cluster.sync();
  }
  r.search(false, 0, u * total);
  if (first) a.out[at] = comp_id(s.cut > cut ? s.cut : cut);
}

// The rows that the stream left to this kernel: a cluster takes one after the other.
template <typename T>
__global__ void __cluster_dims__(WIDE_CTAS, 1, 1) __launch_bounds__(WIDE_THREADS)
sample_wide_kernel(SampleArgs a, SampleWork w) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  WideShared& s = *reinterpret_cast<WideShared*>(smem_raw);
  pdl_wait();
  pdl_launch();
  const int rows = *w.left;
  for (int i = blockIdx.x / WIDE_CTAS; i < rows; i += gridDim.x / WIDE_CTAS) {
    sample_wide_row<T>(a, w.left_rows[i], s);
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
// Sums are added up in an order that goes by V alone: the weights of a lane's tokens of a task, the lanes of a warp, the tasks of a row.
constexpr int PLAN_THREADS = 512, PLAN_PER = 32, PLAN_SAMPLE = PLAN_THREADS * PLAN_PER, PLAN_BLOCK = 256, PLAN_BINS = 1024;
constexpr int STREAM_THREADS = 512, STREAM_WARPS = STREAM_THREADS / 32;
constexpr int TASK = 512;           // tokens that a warp takes at a time
constexpr int LIST = 2048;          // most tokens of a list
constexpr int LIST_PER = LIST / STREAM_THREADS;
constexpr int LIST_K = 1024;        // top-k up to which a list is expected to hold the k tokens

// What a list is made to hold: all of the k, with room for the guess's error (one part in sqrt(want * 16384 / V)), or as many as leave room above.
__device__ __forceinline__ int list_want(bool greedy, int k) {
  if (greedy) return 48;
  if (k <= 0) return 1400;
  return k <= 700 ? 2 * k + 64 : 1500;
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

constexpr int LIST_BINS = 1024;
constexpr int LIST_BIN_MOST = 96;  // tokens of a bin that are compared each with each

struct ListShared {
  uint64_t item[LIST], other[LIST];
  uint32_t bins[LIST_BINS];
  uint32_t warp_count[STREAM_WARPS];
  double warp_sum[STREAM_WARPS];
  double total, cut;
  int place, last;
};

// Puts s.item[0 .. c) into descending order: bins by value, in a bin by comparing each with each. `hi` and `lo`: about where the values lie.
// Rows of many equal values are sorted by exchanges instead. (1,400 tokens by exchanges alone: TODO us of a row's 22.)
__device__ void order_list(ListShared& s, int c, float hi, float lo) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  static_assert(LIST_BINS == 2 * STREAM_THREADS, "two bins per thread");
  const float scale = hi > lo ? fminf(LIST_BINS / (hi - lo), 1e30f) : 0.f;
  s.bins[2 * tid] = s.bins[2 * tid + 1] = 0;
  __syncthreads();
  uint64_t mine[LIST_PER];
  uint32_t bin[LIST_PER], at[LIST_PER];
#pragma unroll
  for (int j = 0; j < LIST_PER; ++j) {
    const int i = tid + j * STREAM_THREADS;
    if (i < c) {
      mine[j] = s.item[i];
      bin[j] = min(LIST_BINS - 1, max(0, static_cast<int>((hi - comp_value(mine[j])) * scale)));
      at[j] = atomicAdd(&s.bins[bin[j]], 1u);
    }
  }
  __syncthreads();
  const uint32_t c0 = s.bins[2 * tid], c1 = s.bins[2 * tid + 1];
  uint32_t up = c0 + c1;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += v;
  }
  if (lane == 31) s.warp_count[warp] = up;
  if (__syncthreads_or(max(c0, c1) > LIST_BIN_MOST)) {
    int size = 2;
    while (size < c) size <<= 1;
    for (int i = c + tid; i < size; i += STREAM_THREADS) s.item[i] = 0;
    sort_down<STREAM_THREADS>(s.item, size);
    return;
  }
  for (int w = 0; w < warp; ++w) up += s.warp_count[w];
  s.bins[2 * tid] = up - c1 - c0;  // where a bin starts
  s.bins[2 * tid + 1] = up - c1;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < LIST_PER; ++j)
    if (tid + j * STREAM_THREADS < c) s.other[s.bins[bin[j]] + at[j]] = mine[j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < LIST_PER; ++j)
    if (tid + j * STREAM_THREADS < c) {
      const uint32_t from = s.bins[bin[j]], to = bin[j] + 1 < LIST_BINS ? s.bins[bin[j] + 1] : static_cast<uint32_t>(c);
      uint32_t above = from;
      for (uint32_t i = from; i < to; ++i) above += s.other[i] > mine[j];
      s.item[above] = mine[j];
    }
  __syncthreads();
}

// The pick of a row from its `c` largest tokens in s.item (unsorted) and the weight `tail` of all others, relative to `ref`; all: there
// are no others of any weight. -2 where the tokens do not decide it. All threads of a CTA of STREAM_THREADS.
__device__ int pick_from_list(ListShared& s, int c, const RowAsk& r, double tail, float ref, bool all, float hi, float lo) {
  const int tid = threadIdx.x;
  if (c == 0) return ref == -INFINITY && all ? -1 : -2;
  order_list(s, c, hi, lo);
  if (r.greedy) return comp_id(s.item[0]);
  const float m = comp_value(s.item[0]);
  // what weighs nothing beside `ref` weighs nothing beside m as well, unless m lies far below (an excluded token is the largest)
  if ((static_cast<double>(ref) - static_cast<double>(m)) * r.inv_t > WIDE_RANGE / 4) return -2;
  if (tail > 0.0) tail *= ref == m ? 1.0 : exp((static_cast<double>(ref) - static_cast<double>(m)) * r.inv_t);
  else all = all || !r.cut_k;  // (a row with a top-k has no tail summed up)
  if (!(tail < 1e300)) return -2;
  if (r.cut_k && c < r.k && !all) return -2;
  const int nk = r.cut_k ? min(r.k, c) : c;
  const bool closed = r.cut_k || all;  // no token outside the list is in play

  double cum[LIST_PER];
  int positive = 0, enough = 0;
#pragma unroll
  for (int j = 0; j < LIST_PER; ++j) {
    const int i = tid * LIST_PER + j;
    const double w = i < nk ? weight_of(comp_value(s.item[i]), m, r.inv_t) : 0.0;
    positive += w > 0.0;
    enough += w >= r.least && i < nk;
    cum[j] = w + (j ? cum[j - 1] : 0.0);
  }
  const double before = sum_before<STREAM_THREADS>(cum[LIST_PER - 1], s.warp_sum);
#pragma unroll
  for (int j = 0; j < LIST_PER; ++j) cum[j] += before;
  if (tid == 0) { s.place = s.last = 0; }
  if (tid == STREAM_THREADS - 1) s.total = cum[LIST_PER - 1] + (closed ? 0.0 : tail);
  __syncthreads();
  for (int o = 16; o; o >>= 1) { positive += __shfl_xor_sync(0xffffffffu, positive, o); enough += __shfl_xor_sync(0xffffffffu, enough, o); }
  if ((tid & 31) == 0) { atomicAdd(&s.place, positive); atomicAdd(&s.last, enough); }
  __syncthreads();
  positive = s.place; enough = max(1, s.last);
  const double sum = s.total;
  constexpr int OPEN = 1 << 30;
  int limit = closed ? nk : OPEN;
  // the first place with more than `target` up to it, OPEN if there is none
  const auto find = [&](double target) {
    __syncthreads();
    if (tid == 0) s.place = OPEN;
    __syncthreads();
    int at = OPEN;
#pragma unroll
    for (int j = LIST_PER - 1; j >= 0; --j)
      if (cum[j] > target && tid * LIST_PER + j < nk) at = tid * LIST_PER + j;
    if (at != OPEN) atomicMin(&s.place, at);
    __syncthreads();
    return s.place;
  };
  if (r.p < 1.0) {
    const int at = find(r.p * sum);
    if (at != OPEN) limit = at + 1;
    else if (!closed) return -2;
  }
  if (r.least > 0.0) {
    if (enough < nk || closed) limit = min(limit, enough);
    else if (limit == OPEN) return -2;
  }
  double total = sum;
  if (limit != OPEN) {
    __syncthreads();
    const int j = limit - 1 - tid * LIST_PER;
#pragma unroll
    for (int i = 0; i < LIST_PER; ++i)
      if (i == j) s.cut = cum[i];
    __syncthreads();
    total = s.cut;
  }
  const int at = find(r.u * total);
  if (at < limit && at != OPEN) return comp_id(s.item[at]);
  if (limit == OPEN) return -2;
  return comp_id(s.item[max(0, min(limit, positive) - 1)]);
}

template <typename T>
__global__ void __launch_bounds__(PLAN_THREADS) sample_plan_kernel(SampleArgs a, SampleWork w) {
  __shared__ uint32_t bins[PLAN_BINS];
  __shared__ float warp_top[PLAN_THREADS / 32], warp_low[PLAN_THREADS / 32];
  __shared__ uint32_t warp_count[PLAN_THREADS / 32];
  __shared__ int found;
  pdl_wait();
  pdl_launch();
  const int at = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const T* row = static_cast<const T*>(a.logits) + at * a.stride;
  const RowAsk ask(a, at);
  if (at == 0 && tid == 0) *w.left = 0;
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
  for (int o = 16; o; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  if (lane == 0) { warp_top[warp] = top; warp_low[warp] = low; }
  __syncthreads();
  for (int i = 0; i < PLAN_THREADS / 32; ++i) { top = fmaxf(top, warp_top[i]); low = fminf(low, warp_low[i]); }
  const float t = ask.greedy ? 1.f : a.temperature[at];
  const float least = fmaxf(top - WIDE_RANGE * t, -FLT_MAX);  // below it nothing has any weight
  const float range = fminf(fminf(WIDE_RANGE * t, top - low), 1e38f);
  const float scale = range > 0.f ? fminf(PLAN_BINS / range, 1e38f) : 0.f;
#pragma unroll
  for (int i = 0; i < PLAN_PER; ++i)
    if (x[i] >= least) atomicAdd(&bins[min(PLAN_BINS - 1, static_cast<int>((top - x[i]) * scale))], 1u);
  __syncthreads();
  // the bin in which the sample has its share of `want`
  const int want = list_want(ask.greedy, ask.cut_k ? ask.k : 0);
  const uint32_t share = max(1u, static_cast<uint32_t>(static_cast<long long>(want) * min(V, PLAN_SAMPLE) / V));
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
    plan.listed = 0;
    plan.done = 0;
    plan.skip = (ask.cut_k && ask.k > LIST_K && reach > least) || t > 1e30f;  // (at such a temperature even a token of `least` weighs something)
    w.plan[at] = plan;
  }
}

// 2^(s / 32) for s in [-4000, 0] and a little more: the fraction's 32 values are held by a warp's lanes, and what is left of s, at most half either
// way, goes through a polynomial: with f ln 2 / 32 = g, at most 0.011, the powers of g over their factorials up to the fifth (the sixth is one part
// in 2^49). All lanes of the warp take part. Ten 64-bit operations for each token, the multiplication into the caller's sum included.
struct ExpLanes {
  int lo, hi;
  __device__ __forceinline__ ExpLanes() {
    const double t = exp2((threadIdx.x & 31) / 32.0);
    lo = __double2loint(t);
    hi = __double2hiint(t);
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
// The sixteen logits of a lane in a task, from `row` on: piece i of 16 bytes holds tokens first + i * 32 * VE ..
template <typename T>
struct TaskLogits {
  static constexpr int VE = 16 / sizeof(T), PIECES = TASK / (32 * VE);
  static __device__ __forceinline__ int id(int first, int e) { return first + e / VE * (32 * VE) + e % VE; }
  uint4 raw[PIECES];
  __device__ __forceinline__ void load(const T* row, int first, int V, bool aligned) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = id(first, i * VE);
      if (aligned && at + VE <= V) {
        raw[i] = __ldg(reinterpret_cast<const uint4*>(row + at));
      } else {
        T one[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) one[j] = at + j < V ? row[at + j] : static_cast<T>(-INFINITY);
        memcpy(&raw[i], one, 16);
      }
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
__global__ void __launch_bounds__(STREAM_THREADS, 2) sample_stream_kernel(SampleArgs a, SampleWork w, int tasks, int tasks_per_warp) {
  using Task = TaskLogits<T>;
  __shared__ ListShared s;
  __shared__ int banned[SAMPLE_MAX_EXCLUDE];
  __shared__ int n_banned;
  const int at = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const ExpLanes exps;
  if (tid == 0) n_banned = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch();
  const RowAsk ask(a, at);
  SamplePlan& plan = w.plan[at];
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
  if (a.n_exclude) __syncthreads();
  const int bans = n_banned;
  const bool with_tail = !ask.greedy && !ask.cut_k && reach > least;
  const double step = ask.inv_t * 46.166241308446828, start = -static_cast<double>(ref) * step;  // 32 / ln 2
  uint64_t* list = w.list + static_cast<size_t>(at) * LIST;

  for (int i = 0; i < tasks_per_warp; ++i) {
    const int task = task0 + i * STREAM_WARPS + warp;
    if (task >= tasks) break;
    const int first = task * TASK + lane * Task::VE;
    Task x;
    x.load(row, first, V, aligned);
    if (bans) x.strike(first, banned, bans);
    uint32_t hits = 0;
    if (with_tail) {
      double tail = 0.0;
#pragma unroll
      for (int e = 0; e < TASK / 32; ++e) {
        const float v = x.value(e);
        const bool hit = v >= reach;  // (a NaN is in neither the list nor the tail)
        hits |= hit ? 1u << e : 0u;
        // tokens that are not the tail's add e^-80 each: nothing
        tail = exps.add(tail, fma(static_cast<double>(hit ? least : fmaxf(v, least)), step, start));
      }
      for (int o = 16; o; o >>= 1) tail += __shfl_xor_sync(0xffffffffu, tail, o);
      if (lane == 0) w.tail[static_cast<size_t>(at) * tasks + task] = tail;
    } else {
#pragma unroll
      for (int e = 0; e < TASK / 32; ++e) hits |= x.value(e) >= reach ? 1u << e : 0u;
    }
    if (__any_sync(0xffffffffu, hits)) {
      const uint32_t mine = __popc(hits);
      uint32_t up = mine;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      uint32_t to = lane == 31 ? atomicAdd(&plan.listed, up) : 0;
      to = __shfl_sync(0xffffffffu, to, 31) + up - mine;
      for (; hits; hits &= hits - 1, ++to) {
        const int id = Task::id(first, __ffs(hits) - 1);
        if (to < LIST) list[to] = comp_of(logit_value(row[id]), id);
      }
    }
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) s.last = atomicAdd(&plan.done, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!s.last) return;
  __threadfence();
  const uint32_t listed = __ldcg(&plan.listed);
  int pick = -2;
  if (listed <= LIST) {
    double tail = 0.0;
    if (with_tail) {
      for (int i = tid; i < tasks; i += STREAM_THREADS) tail += __ldcg(w.tail + static_cast<size_t>(at) * tasks + i);
      const double before = sum_before<STREAM_THREADS>(tail, s.warp_sum);
      if (tid == STREAM_THREADS - 1) s.total = before + tail;
      __syncthreads();
      tail = s.total;
    }
    for (int i = tid; i < static_cast<int>(listed); i += STREAM_THREADS) s.item[i] = __ldcg(list + i);
    __syncthreads();
    pick = pick_from_list(s, static_cast<int>(listed), ask, tail, ref, reach <= least, ref, reach);
  }
  if (tid == 0) {
    if (pick == -2) w.left_rows[atomicAdd(w.left, 1)] = at;
    else a.out[at] = pick;
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
    s.item[atomicAdd(&listed, 1)] = c;
    atomicMax(&top, static_cast<uint32_t>(c >> 32));
    atomicMin(&low, static_cast<uint32_t>(c >> 32));
  }
  __syncthreads();
  const int pick = pick_from_list(s, listed, RowAsk(a, at), 0.0, -INFINITY, true, key_value(top), key_value(low));
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
    if (cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
  }
  SampleWork w;
  sample_work(a.n, a.V, work, &w);
  const int tasks = task_count(a.V);
  // tasks for a warp: as many as leave every SM a few CTAs
  const long long all = static_cast<long long>(tasks) * a.n / STREAM_WARPS, most = 16LL * sms[dev];
  const int per = static_cast<int>(all / most < 1 ? 1 : all / most > 16 ? 16 : all / most);
  const int ctas = (tasks + STREAM_WARPS * per - 1) / (STREAM_WARPS * per);
  const int clusters = a.n < sms[dev] / WIDE_CTAS ? a.n : sms[dev] / WIDE_CTAS;
  if (launch_pdl(sample_plan_kernel<T>, dim3(a.n), dim3(PLAN_THREADS), 0, st, a, w) != cudaSuccess) return -4;
  if (launch_pdl(sample_stream_kernel<T>, dim3(ctas, a.n), dim3(STREAM_THREADS), 0, st, a, w, tasks, per) != cudaSuccess) return -4;
  return launch_pdl(sample_wide_kernel<T>, dim3(clusters * WIDE_CTAS), dim3(WIDE_THREADS), sizeof(WideShared), st, a, w) == cudaSuccess ? 0 : -4;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_sample_max_exclude() { return SAMPLE_MAX_EXCLUDE; }
extern "C" int b200_sample_max_rows() { return 65535; }

extern "C" long long b200_sample_work_bytes(int n, int V) {
  SampleWork w;
  return V <= LIST ? 0 : static_cast<long long>(sample_work(n, V, nullptr, &w));
}

extern "C" int b200_sample(const void* logits, int type, long long stride, int n, int V, const float* temperature, const int* top_k,
                           const float* top_p, const float* min_p, const float* u, const int* exclude, int n_exclude, int64_t* out,
                           void* work, cudaStream_t st) {
  if (n <= 0) return 0;
  if (V <= 0 || n_exclude < 0 || n_exclude > SAMPLE_MAX_EXCLUDE || V > (1 << 30) || n > b200_sample_max_rows()) return -7;
  const SampleArgs a{logits, stride, n, V, temperature, top_k, top_p, min_p, u, exclude, n_exclude, out};
  switch (type) {
    case LOGIT_F32: return launch_sample<float>(a, work, st);
    case LOGIT_BF16: return launch_sample<bf16>(a, work, st);
    case LOGIT_F16: return launch_sample<__half>(a, work, st);
  }
  return -7;
}

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

constexpr int WIDE_CTAS = 8;       // of a row: one cluster
constexpr int WIDE_THREADS = 512;
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
    for (int i = begin + tid; i < end; i += WIDE_THREADS) {
      const float x = logit_value(row[i]);
      const uint64_t c = comp_of(x, i);
      if (c != 0 && !(s.n_banned && banned(i))) f(x, c);
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

  // Descending by comp; n a power of two.
  __device__ void sort_list(int n) {
    uint64_t* a = s.list.item;
    for (int k = 2; k <= n; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int i = tid; i < n / 2; i += WIDE_THREADS) {
          const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
          const uint64_t x = a[lo], y = a[hi];
          if ((x < y) == ((lo & k) == 0)) { a[lo] = y; a[hi] = x; }
        }
      }
    __syncthreads();
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
      sort_list(size);
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
__global__ void __cluster_dims__(WIDE_CTAS, 1, 1) __launch_bounds__(WIDE_THREADS)
sample_wide_kernel(SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  WideShared& s = *reinterpret_cast<WideShared*>(smem_raw);
  pdl_wait();
  pdl_launch();
  const int at = blockIdx.x / WIDE_CTAS, tid = threadIdx.x;
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

template <typename T>
static int launch_wide(const SampleArgs& a, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(sample_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(WideShared)) != cudaSuccess) return -3;
    configured[dev] = true;
  }
  return launch_pdl(sample_wide_kernel<T>, dim3(a.n * WIDE_CTAS), dim3(WIDE_THREADS), sizeof(WideShared), st, a) == cudaSuccess ? 0 : -4;
}

}  // namespace b200

using namespace b200;

extern "C" int b200_sample_max_exclude() { return SAMPLE_MAX_EXCLUDE; }

extern "C" int b200_sample(const void* logits, int type, long long stride, int n, int V, const float* temperature, const int* top_k,
                           const float* top_p, const float* min_p, const float* u, const int* exclude, int n_exclude, int64_t* out,
                           cudaStream_t st) {
  if (n <= 0) return 0;
  if (V <= 0 || n_exclude < 0 || n_exclude > SAMPLE_MAX_EXCLUDE || V > (1 << 30) || n > (1 << 27)) return -7;
  const SampleArgs a{logits, stride, n, V, temperature, top_k, top_p, min_p, u, exclude, n_exclude, out};
  switch (type) {
    case LOGIT_F32: return launch_wide<float>(a, st);
    case LOGIT_BF16: return launch_wide<bf16>(a, st);
    case LOGIT_F16: return launch_wide<__half>(a, st);
  }
  return -7;
}

// Causal gated attention of spans of new tokens over the 8-bit paged cache, on tcgen05.
//
//   s_ij = q_i . (k_j 2^a_j) / sqrt D,   o_i = sum_j p_ij (v_j 2^b_j) / sum_j p_ij over the keys j up to i's position,   out = o * sigmoid(gate)
//
// A tile is 128 MMA rows = (128 / group) consecutive positions of a span x the query heads of one KV head, as in flash_prefill.cu; a
// page of 64 keys at a time:
//
//   S[128 x 64]  = Q1 K^T + Q2 K^T     the page's e4m3 bytes as TMA brought them (kind::f8f6f4, twice the rate of bf16). A bf16 query row,
//                                      scaled by a power of two, is Q1 + Q2 in e4m3: exact but for what lies 2^-17 below its largest number.
//                                      The terms lie in TMEM
//   y = s a_j' + b_j                   the key's power of two and, in the exponent, the value's: w = 2^(y - M + LIFT) weighs the stored
//                                      v_j, M the running maximum of y; the softmax's own sum is sum_j w 2^-b_j
//   O[128 x D]  += P[128 x 64] V       P and V as halves: four warps make them of the page's bytes (exact)
//
// Two groups of four warps take alternate pages, a thread a row; the running maximum goes from one to the other, and the output tile in
// TMEM is rescaled where a maximum grew by more than 2^LAZY. Weights as halves reach from 2^15 to 2^-24, 2^-28 of the largest at the least.
// A span of few tiles over a long context is cut into runs of pages for CTAs of their own, by its own length and position alone, whose partial
// sums are added in their order: a row's bits depend on its span, never on the pass. There is a CTA for each (tile, run) that there is, found by a scan of the
// spans, and partials for the rows of cut spans: 16 rows on 32,768 tokens beside three fresh spans of 2,048 take 238 us, where tiles times the most runs of
// any span took 568. A captured pass has as many CTAs as its spans can come to. All waits are bounded. No cluster multicast.
//
// Bound: the tensor pipe would take 1,024 cycles for a page of 256-wide heads, shared memory 1,600 (keys twice and P once as operands, V once, the
// conversion of V, weights and tables); a page takes 1,830 to 1,950. A tile's first scores come about 10,000 cycles after its start (queries to two terms,
// to TMEM), and its end takes 7,000 to 8,000: most of a short context's time.
// Measured, 16 heads of 256 over 2: 4 x 2,048 rows of prompts of about 28,672 tokens 1,565 to 1,645 us (1.55 TFLOP: 0.94 to 0.99 PFLOP/s; the bf16
// cache's kernel 1,940), 8 x 1,024 rows of fresh prompts 150 us (206), 61 rows over 3,584 tokens 23.0 us, seven spans of 1,531 rows of
// heads of 128, 6 over 3, 15.2 us.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace b200 {

constexpr float K8P_LIFT = 4.0f, K8P_LAZY = 11.0f;  // weights stay below 2^15
constexpr int K8P_THREADS = 448;                   // 8 warps softmax, MMA, loads, 4 warps values
constexpr int K8P_CTAS = 128, K8P_MIN_PAGES = 4;   // a span is cut for about so many CTAs, into runs of no fewer pages

struct Kv8PrefillParams {
  const bf16* q;            // [T, n_q, D]
  const bf16* gate;         // [T, n_q * D]
  const int* starts;        // [segs + 1] first row of each span
  const int* pos0;          // [segs] its position
  const int* tables;        // [segs] rows of `width` pages, max_pages apart
  bf16* out;                // [T, n_q * D]
  float* part_acc;          // [part_rows, D]: per span that is cut [rows, n_q, its runs]
  float2* part_ml;          // [part_rows]
  long long part_rows;      // 0: no span is cut
  int T, segs, max_pages, width, num_pages, n_q, n_kv, group, positions;  // positions: of a tile
  int exact;                // the grid has as many pairs as the spans
  int inv_group;            // r * inv_group >> 16 is r / group, for rows below 128 of groups up to 16
  float scale_log2;
  int* err;
};

// A tile of a span, and its run of pages. part: the span's first partial.
struct Kv8Tile { int seg, p0, row0, rows, pos0, run_pages, runs, run; long long part; };
// What a CTA makes of it: rows from `row` on, of n_pos positions from `pos` on, np pages (0: nothing to do) from page `first` of the span's; of a
// cut span (else runs is 1) the partial of its first row's head 0, the heads' `runs` apart.
struct Kv8Work { int seg, row, n_pos, pos, first, np, runs; long long part; };

template <int D>
struct Kv8PrefillCfg {
  static constexpr int ROWB = D < 128 ? D : 128;       // bytes of a row in one swizzled block of stored numbers
  static constexpr int DB = D / ROWB;
  static constexpr int HB = D / 64;                    // 128-byte blocks of a row of halves
  static constexpr int Q_TERM = 128 * D;               // a term of the queries on its way to TMEM: [128 rows][D], chunks of 16 bytes XOR row
  static constexpr int PAGE_BYTES = KV8_PAGE * D;      // [DB][64 rows][ROWB]: keys or values of a page
  static constexpr int V_BYTES = KV8_PAGE * D * 2;     // [HB][64 rows][128]: values as halves
  static constexpr int P_BYTES = 128 * 128;            // [128 rows][64 halves]
  static constexpr int EXPS = 2 * KV8_PAGE;
  static constexpr int SMEM = 7 * PAGE_BYTES + 2 * V_BYTES + 2 * P_BYTES + 4 * EXPS + 4 * 3 * KV8_PAGE * 4 + 512 + 53 * 8 + static_cast<int>(sizeof(Kv8Work));
  static constexpr int TMEM_COLS = 128 + D + D / 2 <= 256 ? 256 : 512;  // two score tiles of 64, the output, two terms of the queries
};

// Runs that a span of n rows whose last key is in page np - 1 is cut into, and their pages: by the span alone.
__host__ __device__ __forceinline__ int k8p_run_pages(int n, int np, int positions, int n_kv) {
  const int ctas = (n + positions - 1) / positions * n_kv;
  const int cuts = K8P_CTAS / (ctas > 0 ? ctas : 1);
  if (cuts <= 1) return np;
  const int pages = (np + cuts - 1) / cuts;
  return pages < K8P_MIN_PAGES ? K8P_MIN_PAGES : pages;
}

// D[tmem] (+)= A[tmem] * B[smem]^T: a lane of A is a row, a column four of its bytes.
__device__ __forceinline__ void k8p_umma_f8(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// K-major operand tile in rows of ROWB bytes (64 or 128) written with the swizzle of that size, groups of eight rows after each other.
template <int ROWB>
__device__ __forceinline__ uint64_t k8p_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | static_cast<uint64_t>(1) << 16 | static_cast<uint64_t>(8 * ROWB >> 4) << 32 |
         static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(ROWB == 128 ? 2 : 4) << 61;
}
// Offset of 16 bytes of such a tile: row r, chunk c.
template <int ROWB>
__device__ __forceinline__ uint32_t k8p_at(int r, int c) {
  const uint32_t byte = r * ROWB;
  return byte + ((c ^ ((byte >> 7) & (ROWB / 16 - 1))) << 4);
}
// Two floats at a time.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
}

// The tile of a CTA, and its run of pages: number `at` of the spans' (run, tile) pairs, found by all lanes of a warp, 32 spans at a time. CUT: number `at`
// of the tiles of spans that are cut. PARTS: spans may be cut. false: there is none. The spans come from device memory that the host may not have seen: one that is not within the T
// rows and its page table, or has no room among the partials, has no tiles, and leaves an error, as do more pairs or tiles than the grid has (all: look for them).
template <bool PARTS, bool CUT>
__device__ __forceinline__ bool k8p_find(const Kv8PrefillParams& p, int at, bool all, Kv8Tile& t) {
  const int lane = threadIdx.x & 31;
  int before = 0, parts_before = 0;
  bool found = false;
  for (int s0 = 0; s0 < p.segs && (all || !found); s0 += 32) {
    const int s = s0 + lane;
    uint32_t word[3] = {0, 0, 0};  // all three under way at once: each of them is a wait for memory
    ask_32(word[0], p.starts + s, s < p.segs);
    ask_32(word[1], p.starts + s + 1, s < p.segs);
    ask_32(word[2], p.pos0 + s, s < p.segs);
    const int a = word[0], b = word[1], pos = word[2];
    int n = (0 <= a) & (a <= b) & (b <= p.T) ? b - a : -1;
    if ((n > 0) & ((pos < 0) | (pos > p.width * KV8_PAGE - n))) n = -1;
    if (n < 0) { atomicCAS(p.err, 0, ERR_BAD_INDEX); n = 0; }
    const int tiles = (n + p.positions - 1) / p.positions;
    int run_pages = p.width, runs = 1;
    if (PARTS && n > 0) {
      const int np = (pos + n - 1) / KV8_PAGE + 1;
      run_pages = k8p_run_pages(n, np, p.positions, p.n_kv);
      runs = (np + run_pages - 1) / run_pages;
    }
    const int work = CUT ? (runs > 1 ? tiles : 0) : tiles * runs, parts = runs > 1 ? n * runs : 0;
    int upto = work;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    upto += before;
    const uint32_t hit = __ballot_sync(0xffffffffu, at < upto);
    if (hit && !found) {
      found = true;
      const int l = __ffs(hit) - 1, n_tiles = __shfl_sync(0xffffffffu, tiles, l);
      t.seg = s0 + l;
      t.row0 = __shfl_sync(0xffffffffu, a, l);
      t.rows = __shfl_sync(0xffffffffu, n, l);
      t.pos0 = __shfl_sync(0xffffffffu, pos, l);
      t.run_pages = __shfl_sync(0xffffffffu, run_pages, l);
      t.runs = __shfl_sync(0xffffffffu, runs, l);
      const int i = at - __shfl_sync(0xffffffffu, upto - work, l);
      t.run = CUT || !PARTS || t.runs == 1 ? 0 : i / n_tiles;
      t.p0 = (i - t.run * n_tiles) * p.positions;
      t.part = 0;
      if (PARTS && t.runs > 1) {
        const int first = parts_before + __reduce_add_sync(0xffffffffu, lane < l ? parts : 0);
        t.part = static_cast<long long>(first) * p.n_q;
        if (t.part + static_cast<long long>(t.rows) * t.runs * p.n_q > p.part_rows) {
          if (lane == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
          return false;
        }
      }
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
    if (PARTS) parts_before += __reduce_add_sync(0xffffffffu, parts);
  }
  if (all && before > static_cast<int>(gridDim.x) && lane == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);  // the host counted other spans
  return found;
}

// PARTS: a pass in which a span is cut. (In one form for all, passes without took 1 % longer.)
template <int D, bool PARTS>
__global__ void __launch_bounds__(K8P_THREADS, 1)
kv8_prefill_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_exps, Kv8PrefillParams p) {
  using C = Kv8PrefillCfg<D>;
  extern __shared__ __align__(1024) uint8_t smem_k8p[];
  if (smem_u32(smem_k8p) & 1023u) {  // the swizzled tiles need this alignment
    if (threadIdx.x == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    return;
  }
  uint8_t* const sQ = smem_k8p;                          // [2 terms]
  // Keys of three pages and values of four, stored: of one and three in the place of the queries, once those are in TMEM. (With two
  // of each, a load had to come and its products to end within two pages.)
  const auto k_slot = [&](int s) { return sQ + (s < 2 ? 4 + s : 0) * C::PAGE_BYTES; };
  const auto v_slot = [&](int s) { return sQ + (s == 0 ? 6 : s) * C::PAGE_BYTES; };
  static_assert(2 * C::Q_TERM == 4 * C::PAGE_BYTES, "slots in the place of the queries");
  uint8_t* const sV = sQ + 7 * C::PAGE_BYTES;            // [2]
  uint8_t* const sP = sV + 2 * C::V_BYTES;               // [2]: page i uses tile i & 1
  uint8_t* const sE = sP + 2 * C::P_BYTES;               // [4][keys' 64, values' 64] exponents
  float* const sT = reinterpret_cast<float*>(sE + 4 * C::EXPS);  // [4][2^a | b | 2^-b][64]
  float* const s_m = sT + 4 * 3 * KV8_PAGE;              // [128] the running maximum of a row, in the hands of the page that is to see its scores next
  uint64_t* const bars = reinterpret_cast<uint64_t*>(s_m + 128);
  uint64_t* const k_full = bars;                         // [3]
  uint64_t* const k_empty = bars + 4;                    // [3]
  uint64_t* const v8_full = bars + 8;                    // [4]
  uint64_t* const v8_empty = bars + 12;                  // [4]
  uint64_t* const e_full = bars + 16;                    // [4]
  uint64_t* const e_empty = bars + 20;                   // [4]
  uint64_t* const v_full = bars + 24;                    // [2]
  uint64_t* const v_empty = bars + 26;                   // [2]
  uint64_t* const s_full = bars + 28;                    // [2]
  uint64_t* const p_full = bars + 30;                    // [2]
  uint64_t* const pv_done = bars + 32;                   // [2]
  uint64_t* const t_full = bars + 44;                    // [4]
  uint64_t* const m_bar = bars + 36;                     // [2]: the row maxima up to an even / odd page
  uint64_t* const acc_done = bars + 38;
  uint64_t* const x_bar = bars + 39;
  uint64_t* const o_full = bars + 34;                    // the outputs are in shared memory
  uint64_t* const q_ready = bars + 40;                   // the queries' terms are in shared memory, in TMEM
  uint64_t* const q_full = bars + 41;
  uint64_t* const s_empty = bars + 42;                   // [2]: the scores are in their threads' registers
  uint64_t* const t_empty = bars + 48;                   // [4]
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(bars + 52);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile Kv8Work* const s_work = reinterpret_cast<volatile Kv8Work*>(bars + 53);  // what is needed at the end alone stays here until then

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  // One warp looks its tile up (all of them would take turns at the same instructions), while others make things ready. The last tiles of the
  // spans see the most keys and go first; where the grid may have more CTAs than pairs, those with one do, of all heads.
  const uint32_t cta = blockIdx.y * gridDim.x + blockIdx.x;
  const int kh = PARTS && !p.exact ? cta % p.n_kv : blockIdx.y;
  if (warp == 0) {
    Kv8Tile t = {};
    const bool found = k8p_find<PARTS, false>(p, static_cast<int>(!PARTS || p.exact ? gridDim.x - 1 - blockIdx.x : cta / p.n_kv), cta == 0, t);
    if (lane == 0) {
      const int n_pos = min(p.positions, t.rows - t.p0), first = t.run * t.run_pages;
      s_work->seg = t.seg;
      s_work->row = t.row0 + t.p0;
      s_work->n_pos = n_pos;
      s_work->pos = t.pos0 + t.p0;
      s_work->first = first;
      s_work->np = found ? min((t.pos0 + t.p0 + n_pos - 1) / KV8_PAGE + 1, first + t.run_pages) - first : 0;  // up to the last that the tile's rows see
      s_work->runs = t.runs;
      s_work->part = t.part + static_cast<long long>(t.p0) * p.n_q * t.runs + t.run;
    }
  }
  if (PARTS && !p.exact) {  // many CTAs have no pair, and leave at once
    __syncthreads();
    if (s_work->np <= 0) return;
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&v_full[s], 128); mbar_init(&v_empty[s], 1); mbar_init(&s_full[s], 1); mbar_init(&p_full[s], 128);
      mbar_init(&pv_done[s], 1); mbar_init(&s_empty[s], 128); mbar_init(&m_bar[s], 128);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); mbar_init(&v8_full[s], 1); mbar_init(&v8_empty[s], 128);
      mbar_init(&e_full[s], 1); mbar_init(&e_empty[s], 128); mbar_init(&t_full[s], 128); mbar_init(&t_empty[s], 128);
    }
    mbar_init(acc_done, 1);
    mbar_init(x_bar, 256);
    mbar_init(o_full, 256);
    mbar_init(q_ready, K8P_THREADS - 64);
    mbar_init(q_full, 256);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm);
    tma_prefetch_desc(&tm_exps);
  }
  if (warp == 8) { tmem_alloc(tmem_slot, C::TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch();  // this CTA holds its TMEM columns
  const int row0 = s_work->row, n_pos = s_work->n_pos, pos0 = s_work->pos, np = s_work->np;
  if (np <= 0) {  // no tile, or nothing of this run for its rows: the sum over the runs passes over it
    if (warp == 8) tmem_dealloc(tmem, C::TMEM_COLS);
    return;
  }
  const uint32_t tmem_S = tmem, tmem_O = tmem + 128, tmem_Q = tmem_O + D;  // score tile of page i at tmem_S + (i & 1) * 64
  float* const s_qs = reinterpret_cast<float*>(sP);      // until the rows' threads have read it
  constexpr int WARPS = K8P_THREADS / 32 - 2;            // of the warps that convert queries and write outputs
  const int w = warp < 8 ? warp : warp - 2;              // its number among them
  if (warp != 8 && warp != 9) {
    // ---- queries: a warp a row at a time, two terms of e4m3; the largest number of a row comes to [128, 256)
    constexpr int PER = (128 + WARPS - 1) / WARPS;
    uint4 raw[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = w + i * WARPS, lp = r * p.inv_group >> 16;
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      ask_128(raw[i], p.q + (static_cast<size_t>(row0 + lp) * p.n_q + kh * p.group + (r - lp * p.group)) * D + lane * 8,
              r < 128 && lp < n_pos && lane * 8 < D);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = w + i * WARPS;
      if (r >= 128) break;
      const uint32_t* word = reinterpret_cast<const uint32_t*>(&raw[i]);
      // magnitudes of bf16 numbers are in the order of their bits
      uint32_t top = __vmaxu2(__vmaxu2(word[0] & 0x7fff7fffu, word[1] & 0x7fff7fffu), __vmaxu2(word[2] & 0x7fff7fffu, word[3] & 0x7fff7fffu));
      top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
      const int e = max(-110, min(110, static_cast<int>(top >> 7) - 127 - 7));
      const float f = kv8_two_to(-e);
      uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // the first four significant bits, and the other four
        const float a = __uint_as_float(word[k] << 16) * f, b = __uint_as_float(word[k] & 0xffff0000u) * f;
        const float ah = __uint_as_float(__float_as_uint(a) & 0xfff00000u), bh = __uint_as_float(__float_as_uint(b) & 0xfff00000u);
        hi[k / 2] |= kv8_pack2(ah, bh) << (16 * (k & 1));
        lo[k / 2] |= kv8_pack2(a - ah, b - bh) << (16 * (k & 1));
      }
      if (lane * 8 < D) {
        uint8_t* const at = sQ + r * D + (((lane >> 1) ^ (r & (D / 16 - 1))) << 4) + (lane & 1) * 8;
        *reinterpret_cast<uint2*>(at) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(at + C::Q_TERM) = make_uint2(lo[0], lo[1]);
      }
      // a NaN or an infinity: all scores of the row are NaN
      if (lane == 0) s_qs[r] = top >= 0x7f80u ? __uint_as_float(0x7fffffffu) : kv8_two_to(e) * p.scale_log2;
    }
    mbar_arrive(q_ready);
  }

  if (warp == 9) {
    // ---------------- loads. The gates are needed at the end, when other loads of this SM's neighbours are under way: they are brought to L2 now.
    for (int i = PARTS && s_work->runs > 1 ? n_pos : lane; i < n_pos; i += 32)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;"
                     ::"l"(p.gate + (static_cast<size_t>(row0 + i) * p.n_q + kh * p.group) * D), "r"(p.group * D * 2) : "memory");
    if (elect_one()) {
      const int* table = p.tables + static_cast<size_t>(s_work->seg) * p.max_pages + s_work->first;
      int next = table[0], i = 0;
      for (; i < np; ++i) {
        const int s = i & 3, ks = i % 3;
        const uint32_t again = ((i >> 2) & 1) ^ 1;
        int page = next;
        if (i + 1 < np) next = table[i + 1];
        if (page < 0 || page >= p.num_pages) { atomicCAS(p.err, 0, ERR_BAD_INDEX); page = 0; }
        const int row = (page * 2 * p.n_kv + kh) * KV8_PAGE;
        if (!mbar_wait(&k_empty[ks], ((i / 3) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag)) break;
        mbar_expect_tx(&k_full[ks], C::PAGE_BYTES);
#pragma unroll
        for (int b = 0; b < C::DB; ++b)
          tma_load_2d(k_slot(ks) + b * KV8_PAGE * C::ROWB, &tm, &k_full[ks], b * C::ROWB, row);
        if (!mbar_wait(&e_empty[s], again, p.err, ERR_WAIT_EMPTY, abort_flag)) break;
        mbar_expect_tx(&e_full[s], C::EXPS);
        tma_load_3d(sE + s * C::EXPS, &tm_exps, &e_full[s], 0, kh, page * 2);
        if (i == 1 && !mbar_wait(q_full, 0, p.err, ERR_WAIT_FULL, abort_flag)) break;  // from here on in the queries' place
        if (!mbar_wait(&v8_empty[s], again, p.err, ERR_WAIT_EMPTY, abort_flag)) break;
        mbar_expect_tx(&v8_full[s], C::PAGE_BYTES);
#pragma unroll
        for (int b = 0; b < C::DB; ++b)
          tma_load_2d(v_slot(s) + b * KV8_PAGE * C::ROWB, &tm, &v8_full[s], b * C::ROWB, row + p.n_kv * KV8_PAGE);
      }
      // after a wait that ran out: loads on their way end before the shared memory goes (a page that was begun may lack some: the limit ends that)
      const auto land = [&](uint64_t* bar, uint32_t parity) {
        const long long t0 = clock64();
        while (!mbar_test(bar, parity) && clock64() - t0 < WAIT_CYCLES / 8) {}
      };
      if (i < np || *abort_flag) {
        for (int k = max(0, i - 3); k <= min(i, np - 1); ++k) {
          land(&k_full[k % 3], (k / 3) & 1);
          land(&e_full[k & 3], (k >> 2) & 1);
          land(&v8_full[k & 3], (k >> 2) & 1);
        }
      }
    }
  } else if (warp == 8) {
    // ---------------- MMAs
    if (elect_one()) {
      constexpr uint32_t idesc_s = (1u << 4) | (64u >> 3) << 17 | (128u >> 4) << 24;                                     // e4m3
      constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | static_cast<uint32_t>(D >> 3) << 17 | (128u >> 4) << 24;     // halves, B MN-major
      // Scores of page q once page q - 2's have been read and the keys are there, products of page v once its weights and values are: whichever
      // comes first: in a fixed order one waited behind the other.
      if (!mbar_wait(q_full, 0, p.err, ERR_WAIT_FULL, abort_flag)) *abort_flag = 1;
      int q = 0, v = 0;
      long long t0 = clock64();
      while (v < np && !*abort_flag) {
        if (v < q && mbar_test(&p_full[v & 1], (v >> 1) & 1) && mbar_test(&v_full[v & 1], (v >> 1) & 1)) {
          tc_fence_after();
          const int s = v & 1;
          const uint32_t pa = smem_u32(sP + s * C::P_BYTES), va = smem_u32(sV + s * C::V_BYTES);
#pragma unroll
          for (int kk = 0; kk < KV8_PAGE / 16; ++kk)
            umma_bf16(tmem_O, umma_smem_desc(pa + kk * 32), umma_smem_desc_mn(va + kk * 2048, KV8_PAGE * 128), idesc_o, (v | kk) != 0);
          umma_commit(&pv_done[s]);
          umma_commit(&v_empty[s]);
          ++v;
          t0 = clock64();
        } else if (q < np && (q < 2 || mbar_test(&s_empty[q & 1], ((q - 2) >> 1) & 1)) && mbar_test(&k_full[q % 3], (q / 3) & 1)) {
          tc_fence_after();
          const int s = q & 1, ks = q % 3;
          const uint32_t ka = smem_u32(k_slot(ks));
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
              constexpr int STEPS = C::ROWB / 32;
              const int blk = kk / STEPS, off = kk % STEPS * 32;
              k8p_umma_f8(tmem_S + s * 64, tmem_Q + term * (D / 4) + kk * 8, k8p_desc<C::ROWB>(ka + blk * KV8_PAGE * C::ROWB + off),
                          idesc_s, (term | kk) != 0);
            }
          umma_commit(&s_full[s]);
          umma_commit(&k_empty[ks]);
          ++q;
          t0 = clock64();
        } else if (clock64() - t0 > WAIT_CYCLES) {
          *abort_flag = 1;
          atomicCAS(p.err, 0, ERR_WAIT_FULL);
        }
      }
      umma_commit(acc_done);
    }
  } else if (warp >= 10) {
    // ---------------- values: bytes to halves; the numbers that go with a page's keys
    const int tid = threadIdx.x - 320;
    // A thread has 16 numbers of every ROWS-th row, neighbours have neighbouring chunks of a row. Its two chunks of halves go out in an
    // order that lets eight neighbours cover all banks. ROWS is a multiple of eight: the swizzle of a thread's rows is the same.
    constexpr int PER_ROW = D / 16, ROWS = 128 / PER_ROW;
    static_assert(ROWS % 8 == 0, "rows of a step");
    const int r = tid / PER_ROW, k = tid % PER_ROW;
    const bool swap = (k >> 2) & 1;
    const uint32_t from = k / (C::ROWB / 16) * KV8_PAGE * C::ROWB + k8p_at<C::ROWB>(r, k % (C::ROWB / 16));
    const uint32_t to0 = k / 4 * KV8_PAGE * 128 + k8p_at<128>(r, (k & 3) * 2 + swap);
    const uint32_t to1 = k / 4 * KV8_PAGE * 128 + k8p_at<128>(r, (k & 3) * 2 + 1 - swap);
    // What goes with a page's keys and values, two pages ahead of the conversion: the scores wait for it
    const auto numbers = [&](int i) {
      const int es = i & 3;
      const bool ok = mbar_wait(&e_full[es], (i >> 2) & 1, p.err, ERR_WAIT_FULL, abort_flag)
                      && mbar_wait(&t_empty[es], ((i >> 2) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
      if (!ok) return false;
      const uint32_t byte = sE[es * C::EXPS + tid];  // threads 0 .. 63: a key's, then a value's
      float* const t = sT + es * 3 * KV8_PAGE;
      if (tid < KV8_PAGE) {
        t[tid] = kv8_factor(byte);
      } else {
        t[tid] = byte == KV8_E_NAN ? __uint_as_float(0x7fffffffu) : static_cast<float>(static_cast<int>(byte) - 127);
        t[KV8_PAGE + tid] = kv8_two_to(max(-126, 127 - static_cast<int>(byte)));
      }
      mbar_arrive(&t_full[es]);
      mbar_arrive(&e_empty[es]);
      return true;
    };
    bool ok = numbers(0) && (np < 2 || numbers(1));
    for (int i = 0; i < np && ok; ++i) {
      const int s = i & 1, vs = i & 3;
      ok = (i + 2 >= np || numbers(i + 2))
           && mbar_wait(&v8_full[vs], (i >> 2) & 1, p.err, ERR_WAIT_FULL, abort_flag)
           && (i < 2 || mbar_wait(&v_empty[s], ((i - 2) >> 1) & 1, p.err, ERR_WAIT_EMPTY, abort_flag));
      if (!ok) break;
      const uint8_t* const src = v_slot(vs) + from;
      uint8_t* const dst = sV + s * C::V_BYTES;
#pragma unroll
      for (int c = 0; c < KV8_PAGE / ROWS; ++c) {
        const uint4 raw = *reinterpret_cast<const uint4*>(src + c * ROWS * C::ROWB);
        uint4 h[2];
        kv8_unpack4(raw.x, h[0].x, h[0].y);
        kv8_unpack4(raw.y, h[0].z, h[0].w);
        kv8_unpack4(raw.z, h[1].x, h[1].y);
        kv8_unpack4(raw.w, h[1].z, h[1].w);
        *reinterpret_cast<uint4*>(dst + to0 + c * ROWS * 128) = swap ? h[1] : h[0];
        *reinterpret_cast<uint4*>(dst + to1 + c * ROWS * 128) = swap ? h[0] : h[1];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&v_full[s]);
      mbar_arrive(&v8_empty[vs]);
    }
  } else {
    // ---------------- softmax + epilogue: thread (r = tid & 127, hf = tid >> 7) owns row r = one (position, head) on the pages
    // i with i & 1 == hf, and the half hf of the output columns at the end.
    const int r = threadIdx.x & 127, hf = threadIdx.x >> 7, rw = warp & 3;
    const uint32_t lane_base = static_cast<uint32_t>(rw * 32) << 16;
    const int lp = r * p.inv_group >> 16, head = r - lp * p.group;
    const int qpos = pos0 + lp;
    const bool row_valid = lp < n_pos;
    const int key0 = s_work->first * KV8_PAGE;
    constexpr int DH = D / 2;
    float m_loc = -INFINITY;  // the maximum and the sum of this thread's own pages, at that maximum
    float2 l2 = make_float2(0.f, 0.f);
    bool ok = mbar_wait(q_ready, 0, p.err, ERR_WAIT_FULL, abort_flag);
    {  // the queries' terms to TMEM, one by either group: as an operand there they take no bandwidth of shared memory, which bounds a page
      const uint8_t* const src = sQ + hf * C::Q_TERM + r * D;
#pragma unroll
      for (int c = 0; c < D / 16; c += 4) {
        uint4 w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(src + (((c + j) ^ (r & (D / 16 - 1))) << 4));
        tmem_st16(tmem_Q + lane_base + hf * (D / 4) + c * 4, reinterpret_cast<const float*>(w));
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      mbar_arrive(q_full);
    }
    const float2 qs2 = make_float2(s_qs[r], s_qs[r]);
    asm volatile("bar.sync 1, 256;" ::: "memory");  // all have read it: the weights' tiles may be written. Nobody has left before
    for (int i = hf; i < np && ok; i += 2) {
      const uint32_t ph = (i >> 1) & 1;
      ok = mbar_wait(&t_full[i & 3], (i >> 2) & 1, p.err, ERR_WAIT_FULL, abort_flag) && mbar_wait(&s_full[hf], ph, p.err, ERR_WAIT_TMEM, abort_flag);
      if (!ok) break;
      tc_fence_after();
      float2 y[32];
      tmem_ld64(tmem_S + hf * 64 + lane_base, reinterpret_cast<float*>(y));
      tc_fence_before();
      mbar_arrive(&s_empty[hf]);
      const float* t = sT + (i & 3) * 3 * KV8_PAGE;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float4 a = *reinterpret_cast<const float4*>(t + 4 * j), b = *reinterpret_cast<const float4*>(t + KV8_PAGE + 4 * j);
        y[2 * j] = fma2(mul2(y[2 * j], qs2), make_float2(a.x, a.y), make_float2(b.x, b.y));
        y[2 * j + 1] = fma2(mul2(y[2 * j + 1], qs2), make_float2(a.z, a.w), make_float2(b.z, b.w));
      }
      const int kbase = key0 + i * KV8_PAGE;
      if (kbase + KV8_PAGE - 1 > pos0) {  // only pages that end behind the tile's first query hide keys
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          y[j].x = kbase + 2 * j <= qpos ? y[j].x : -INFINITY;
          y[j].y = kbase + 2 * j + 1 <= qpos ? y[j].y : -INFINITY;
        }
      }
      float mx4[4] = {y[0].x, y[0].y, y[1].x, y[1].y};
#pragma unroll
      for (int j = 2; j < 32; ++j) { mx4[(2 * j) & 3] = fmaxf(mx4[(2 * j) & 3], y[j].x); mx4[(2 * j + 1) & 3] = fmaxf(mx4[(2 * j + 1) & 3], y[j].y); }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      float m_prev = -INFINITY;
      if (i > 0) {
        ok = mbar_wait(&m_bar[hf ^ 1], ((i - 1) >> 1) & 1, p.err, ERR_WAIT_FULL, abort_flag);
        if (!ok) break;
        m_prev = s_m[r];
      }
      const bool need = mx > m_prev + K8P_LAZY;
      const float m = need ? mx : m_prev;
      s_m[r] = m;
      mbar_arrive(&m_bar[hf]);
      // This page's weights' tile was last read by the products of page i - 2. They are also the ones behind those of page i - 3, without
      // whose end a wait for page i - 1's would take that barrier's phase before for its own and go on at once.
      if (i >= 2) {
        ok = mbar_wait(&pv_done[hf], ph ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
        if (!ok) break;
      }
      // The output tile may only be rescaled once the products of page i - 1 have been added; those of this page and the later ones
      // wait for this page's weights.
      if (__any_sync(0xffffffffu, need) && i > 0) {  // warp-uniform: TMEM loads / stores are warp-collective
        ok = mbar_wait(&pv_done[hf ^ 1], ((i - 1) >> 1) & 1, p.err, ERR_WAIT_EMPTY, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float factor = need ? ex2(m_prev - m) : 1.0f;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float o[16];
          tmem_ld16(tmem_O + lane_base + c, o);
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] *= factor;
          tmem_st16(tmem_O + lane_base + c, o);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      }
      if (m != m_loc) {
        const float f = ex2(m_loc - m);  // 0 on this thread's first page
        l2.x *= f;
        l2.y *= f;
        m_loc = m;
      }
      const float base = m == -INFINITY ? 0.f : K8P_LIFT - m;  // a row that sees no key of the run so far
      const float2 base2 = make_float2(base, base), one2 = make_float2(1.f, 1.f);
      uint8_t* const prow = sP + hf * C::P_BYTES + r * 128;
      t += 2 * KV8_PAGE;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 packed;
        __half2* pe = reinterpret_cast<__half2*>(&packed);
        const float4 i0 = *reinterpret_cast<const float4*>(t + 8 * c), i1 = *reinterpret_cast<const float4*>(t + 8 * c + 4);
        const float2 inv[4] = {make_float2(i0.x, i0.y), make_float2(i0.z, i0.w), make_float2(i1.x, i1.y), make_float2(i1.z, i1.w)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 z = fma2(y[4 * c + j], one2, base2);
          const float2 w = make_float2(ex2(z.x), ex2(z.y));
          l2 = fma2(w, inv[j], l2);
          pe[j] = __floats2half2_rn(w.x, w.y);
        }
        *reinterpret_cast<uint4*>(prow + ((c ^ (r & 7)) * 16)) = packed;  // 128-byte swizzle of the K-major tile
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      mbar_arrive(&p_full[hf]);
      mbar_arrive(&t_empty[i & 3]);
    }
    float l = l2.x + l2.y;
    ok = ok && mbar_wait(acc_done, 0, p.err, ERR_WAIT_TMEM, abort_flag) && !*abort_flag;
    tc_fence_after();
    float m_used = m_loc;
    if (ok) {  // the weights' tiles are free now: even and odd pages put their sums together, even + odd
      float* ex = reinterpret_cast<float*>(sP);
      ex[(hf * 128 + r) * 2] = l;
      ex[(hf * 128 + r) * 2 + 1] = m_loc;
      mbar_arrive(x_bar);
      ok = mbar_wait(x_bar, 0, p.err, ERR_WAIT_FULL, abort_flag);
      const float l0 = ex[r * 2], m0 = ex[r * 2 + 1], l1 = ex[(128 + r) * 2], m1 = ex[(128 + r) * 2 + 1];
      m_used = fmaxf(m0, m1);  // a running maximum never falls: the larger one is the last page's
      l = m_used == -INFINITY ? l0 + l1 : fmaf(l0, ex2(m0 - m_used), l1 * ex2(m1 - m_used));
    }
    // The outputs go through shared memory, 16 bytes of a row in the place of their number XOR the row, so that a warp reads gates and
    // writes outputs of a whole row at a time (with a thread a row from TMEM to the output, the end of a tile took 13 us).
    float* const so = reinterpret_cast<float*>(sQ);        // [128][D], in the place of Q and the pages' bytes
    if (ok) {
      const int runs = PARTS ? s_work->runs : 1;
      const bool cut = runs > 1;
      const float inv = cut ? 1.0f : 1.0f / l;             // (a row sees itself)
#pragma unroll 1
      for (int c = hf * DH; c < hf * DH + DH; c += 16) {
        float o[16];
        tmem_ld16(tmem_O + lane_base + c, o);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float4*>(so + r * D + (((c >> 2) + j) ^ (r & 7)) * 4) =
              make_float4(o[4 * j] * inv, o[4 * j + 1] * inv, o[4 * j + 2] * inv, o[4 * j + 3] * inv);
      }
      if (cut && row_valid && hf == 0)
        p.part_ml[s_work->part + (lp * p.n_q + kh * p.group + head) * runs] = make_float2(m_used, l);
      mbar_arrive(o_full);
    }
  }
  if (warp != 8 && warp != 9) {
    // ---------------- outputs, a warp whole rows at a time, their gates ahead of the last products
    constexpr int LANES = D / 8, ROWS = 32 / LANES, STEPS = (128 + WARPS * ROWS - 1) / (WARPS * ROWS);  // 8 numbers a lane, rows a warp takes at once
    const int sub = lane / LANES, d = lane % LANES * 8, n_rows = n_pos * p.group;
    const size_t head0 = static_cast<size_t>(row0) * p.n_q + kh * p.group;
    const auto head_of = [&](int row) {
      const int pos = row * p.inv_group >> 16;
      return head0 + static_cast<size_t>(pos) * p.n_q + (row - pos * p.group);
    };
    const int runs = PARTS ? s_work->runs : 1;
    const bool cut = runs > 1;
    float* const dst0 = p.part_acc + (cut ? s_work->part + kh * p.group * runs : 0) * D + d;
    uint4 gate[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int row = (i * WARPS + w) * ROWS + sub;
      gate[i] = make_uint4(0u, 0u, 0u, 0u);
      ask_128(gate[i], p.gate + head_of(row) * D + d, !cut && row < n_rows);
    }
    const float* const so = reinterpret_cast<const float*>(sQ);
    if (mbar_wait(o_full, 0, p.err, ERR_WAIT_FULL, abort_flag)) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int row = (i * WARPS + w) * ROWS + sub;
        if (row >= n_rows) break;
        const float* const src = so + row * D;
        const float4 a = *reinterpret_cast<const float4*>(src + ((d >> 2) ^ (row & 7)) * 4), b = *reinterpret_cast<const float4*>(src + (((d >> 2) + 1) ^ (row & 7)) * 4);
        const size_t at = head_of(row);
        if (cut) {
          float* const dst = dst0 + static_cast<int>(at - head0) * runs * D;
          *reinterpret_cast<float4*>(dst) = a;
          *reinterpret_cast<float4*>(dst + 4) = b;
        } else {
          const uint32_t gw[4] = {gate[i].x, gate[i].y, gate[i].z, gate[i].w};
          const float o[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          uint4 out;
          __nv_bfloat162* oe = reinterpret_cast<__nv_bfloat162*>(&out);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 g = kv8_sigmoid2(gw[j]);
            oe[j] = __floats2bfloat162_rn(o[2 * j] * g.x, o[2 * j + 1] * g.y);
          }
          *reinterpret_cast<uint4*>(p.out + at * D + d) = out;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    if (*abort_flag) {  // after a wait that ran out: products on their way end before their TMEM and shared memory go
      const long long t0 = clock64();
      while (!mbar_test(acc_done, 0) && clock64() - t0 < WAIT_CYCLES / 8) {}
    }
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Rows of spans that were cut: their partials in the order of the runs, eight under way. A thread takes four dims of a row's head. What does not
// come from the kernel in front is read ahead of the dependency wait: that kernel has waited for everything before it.
template <int D>
__global__ void __launch_bounds__(128)
kv8_prefill_combine_kernel(Kv8PrefillParams p) {
  constexpr int QUADS = D / 4, AT_ONCE = 8;
  Kv8Tile tile = {};
  const bool found = k8p_find<true, true>(p, blockIdx.x, (blockIdx.x | blockIdx.y | blockIdx.z) == 0, tile);
  const int n_pos = min(p.positions, tile.rows - tile.p0), i = blockIdx.z * (128 / QUADS) + threadIdx.x / QUADS;
  const bool work = found && i < n_pos * p.group;
  const int np_all = (tile.pos0 + tile.p0 + n_pos - 1) / KV8_PAGE + 1, runs = found ? (np_all + tile.run_pages - 1) / tile.run_pages : 0;  // that wrote
  const int pos = i * p.inv_group >> 16, quad = threadIdx.x % QUADS, head = blockIdx.y * p.group + (i - pos * p.group);
  const size_t at = static_cast<size_t>(tile.row0 + tile.p0 + pos) * p.n_q + head;
  // Threads without work leave before the wait, so that the grid does not come in waves behind it; those of the first CTA stay: this kernel must
  // not end before the one in front, for whose end what comes next takes it.
  if (!work && (blockIdx.x | blockIdx.y | blockIdx.z) != 0) return;
  const uint2 gate = work ? *reinterpret_cast<const uint2*>(p.gate + at * D + quad * 4) : make_uint2(0u, 0u);
  pdl_wait();
  pdl_launch();
  if (!work) return;
  const size_t part = tile.part + (static_cast<size_t>(tile.p0 + pos) * p.n_q + head) * tile.runs;
  const float2* ml = p.part_ml + part;
  const float4* pa = reinterpret_cast<const float4*>(p.part_acc + part * D) + quad;
  float2 pm[AT_ONCE];
  float4 v[AT_ONCE];
  const auto ask = [&](int z0) {
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      pm[k] = z0 + k < runs ? ml[z0 + k] : make_float2(-INFINITY, 0.f);
      v[k] = z0 + k < runs ? pa[static_cast<size_t>(z0 + k) * QUADS] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  ask(0);
  float top = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int z = AT_ONCE; z < runs; ++z) top = fmaxf(top, ml[z].x);
#pragma unroll
  for (int k = 0; k < AT_ONCE; ++k) top = fmaxf(top, pm[k].x);
  for (int z0 = 0;;) {
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const float f = pm[k].x == top ? 1.f : ex2(pm[k].x - top);
      l = fmaf(pm[k].y, f, l);
      o.x = fmaf(v[k].x, f, o.x); o.y = fmaf(v[k].y, f, o.y); o.z = fmaf(v[k].z, f, o.z); o.w = fmaf(v[k].w, f, o.w);
    }
    z0 += AT_ONCE;
    if (z0 >= runs) break;
    ask(z0);
  }
  const float inv = 1.0f / l;
  const float2 g0 = kv8_sigmoid2(gate.x), g1 = kv8_sigmoid2(gate.y);
  uint2 raw;
  __nv_bfloat162* e = reinterpret_cast<__nv_bfloat162*>(&raw);
  e[0] = __floats2bfloat162_rn(o.x * inv * g0.x, o.y * inv * g0.y);
  e[1] = __floats2bfloat162_rn(o.z * inv * g1.x, o.w * inv * g1.y);
  *reinterpret_cast<uint2*>(p.out + at * D + quad * 4) = raw;
}

}  // namespace b200

using namespace b200;

namespace {
template <int D>
int k8p_launch(const CUtensorMap& tm, const CUtensorMap& te, const Kv8PrefillParams& p, int pairs, int cut_tiles, cudaStream_t st) {
  auto kern = cut_tiles > 0 ? kv8_prefill_kernel<D, true> : kv8_prefill_kernel<D, false>;
  static bool configured[2][64] = {};  // a function attribute is set per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!configured[cut_tiles > 0][dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8PrefillCfg<D>::SMEM) != cudaSuccess) return -3;
    configured[cut_tiles > 0][dev] = true;
  }
  if (launch_pdl(kern, dim3(pairs, p.n_kv), dim3(K8P_THREADS), Kv8PrefillCfg<D>::SMEM, st, tm, te, p) != cudaSuccess) return -4;
  if (cut_tiles == 0) return 0;
  return launch_pdl(kv8_prefill_combine_kernel<D>, dim3(cut_tiles, p.n_kv, 128 / (128 / (D / 4))), dim3(128), 0, st, p) == cudaSuccess ? 0 : -4;
}
}  // namespace

// Positions of a tile, and what a span is cut by (k8p_run_pages): 0, the CTAs, 1, a run's least pages. The caller sizes grid and partials by them.
extern "C" int b200_kv8_prefill_positions(int group) { return group >= 1 && group <= 16 ? 128 / group : 0; }
extern "C" int b200_kv8_prefill_cut(int which) { return which ? K8P_MIN_PAGES : K8P_CTAS; }

// q: [T, n_q, D] bf16 (normed and rotated), gate, out: [T, n_q * D], in 16-byte rows; data, exps: one layer of the 8-bit cache, which holds the
// spans' own keys; starts [segs + 1], pos0 [segs] of the spans, within T rows, tables [segs] rows of `width` pages. pairs: at least the spans' tiles, each
// times its span's runs (exact: no more than those); cut_tiles: at least those of spans that are cut; part_rows: their rows' heads, times their runs (part_acc [part_rows, D],
// part_ml [part_rows, 2]); of the last two either both or none.
extern "C" int b200_kv8_prefill(const void* q, const void* gate, const void* data, const void* exps, const int* starts, const int* pos0,
                                int T, int segs, int pairs, int exact, int cut_tiles, long long part_rows, const int* tables, int max_pages, int width,
                                int num_pages, int n_q, int n_kv, int D, float* part_acc, float* part_ml, void* out, int* err, cudaStream_t st) {
  if (pairs <= 0 || segs <= 0) return 0;
  const int group = n_kv > 0 ? n_q / n_kv : 0;
  if (group < 1 || group * n_kv != n_q || group > 16 || cut_tiles < 0 || (cut_tiles > 0) != (part_rows > 0) || width < 1 || width > 0x7fffffff / KV8_PAGE) return -7;
  if (D != 256 && D != 128 && D != 64) return -7;
  const long long rows = static_cast<long long>(num_pages) * 2 * n_kv * KV8_PAGE;
  if (rows > 0x7fffffffLL) return -7;  // a TMA coordinate
  for (const void* x : {q, gate, data, exps, static_cast<const void*>(out)})
    if (reinterpret_cast<uintptr_t>(x) % 16) return -7;
  CUtensorMap tm, te;
  const cuuint32_t rowb = D < 128 ? D : 128;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(D)};
  const cuuint32_t box[2] = {rowb, KV8_PAGE};
  if (kv8_encode(&tm, data, 2, dims, strides, box, rowb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B) ||
      kv8_encode_exps(&te, exps, n_kv, num_pages)) return -1;
  const Kv8PrefillParams p{static_cast<const bf16*>(q), static_cast<const bf16*>(gate), starts, pos0, tables, static_cast<bf16*>(out), part_acc,
                           reinterpret_cast<float2*>(part_ml), part_rows, T, segs, max_pages, width, num_pages, n_q, n_kv, group, 128 / group, exact,
                           (65536 + group - 1) / group, 1.4426950408889634f / sqrtf(static_cast<float>(D)), err};
  if (D == 256) return k8p_launch<256>(tm, te, p, pairs, cut_tiles, st);
  if (D == 128) return k8p_launch<128>(tm, te, p, pairs, cut_tiles, st);
  return k8p_launch<64>(tm, te, p, pairs, cut_tiles, st);
}

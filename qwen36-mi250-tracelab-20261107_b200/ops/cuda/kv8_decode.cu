// Attention of a few query rows per sequence (decode steps, verify passes) over the 8-bit paged cache.
//
//   s_j = q . (k_j 2^a_j) / sqrt D,   o = sum_j p_j (v_j 2^b_j) / sum_j p_j,   p_j = exp(s_j),   out = o * sigmoid(gate)
//
// with e4m3 rows k_j, v_j and their powers of two. Neither row is ever scaled: y_j = s_j log2(e) + b_j takes the value's power of
// two into the exponent, w_j = 2^(y_j - M) is the weight of the stored v_j, M the running maximum of y, and the softmax's own sum is
// sum_j w_j 2^-b_j. So what the matrix instructions get are the stored numbers as halves (exact) and weights below 2^15.
//
// Bound: the cache's bytes, 2 (D + 1) per token and KV head. A context is cut into runs of RUN keys at fixed places, so what a row's
// result is put together from depends on its own position only, never on the batch; persistent CTAs, two per SM, take runs in turn. In a
// CTA one warp finds the runs and brings pages of 64 keys by TMA, three pages ahead; four warps take 16 keys each (S = K Q^T, maximum,
// weights); four take D / 4 dims each over all 64 keys (O += V^T P), a page behind. The outputs stay where they are summed: only maxima and
// weights are exchanged, 16 bytes per key. (With all dims of every eighth slab in each of eight warps, the warps' outputs were added up at
// each run's end, which took more instructions than the run: 74 us for 128 sequences of about 1,088 keys, and 35 now.)
// The products are m16n8k16 with keys or dims as the 16 rows and query columns as the 8: one token of one KV head's eight query heads
// fills the columns, where a tcgen05 tile would be 8 rows of 64. (The tcgen05 form, S^T and O^T on tiles of 128 keys with two e4m3 terms of queries and
// weights, took 68 us there: V^T as an operand from rows of values costs 1,300 cycles per 128 keys.) The stored bytes become halves in
// registers, behind ldmatrix. More than 16 columns (verify passes) are units of their own, which find the pages in L2: as 32 columns of
// one CTA of 17 warps they took 65 us, and 50 so, for 40 passes of four rows over about 4,096 keys.
//
// Measured, heads of 256, 16 over 2: 128 sequences of about 1,088 keys 35 us, 142 MB at 4.1 TB/s; four of about 90,000 54 us, 241 MB at 4.4 TB/s;
// 40 passes of four rows over about 4,096 keys 50 us. With one column tile the pages come at the memory's rate once they come; what is left is 5 us
// before the first is asked for, CTAs that wait for the last whole runs, and 4 to 6 us for joining the runs. With two it is a page's chain of steps (2,330
// cycles for a CTA, 1,200 of them the scores' products).
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace b200 {

// Keys of a run: part of the numerics. Of 256: one context of 900 keys 9.6 us and not 12.4, but 128 of about 1,088 in 37.0 and not 35.2, four of about
// 90,000 in 57.7 and not 54.2, 40 passes of four rows over about 4,096 keys in 59.7 and not 51.2: each run's end costs about a page's time.
constexpr int K8D_RUN = 512;
constexpr int K8D_SLAB = 16;                    // keys of a warp's scores
constexpr int K8D_SLABS = KV8_PAGE / K8D_SLAB;  // of a page: a warp each
constexpr int K8D_OUT = 4;                      // warps that take outputs
constexpr int K8D_THREADS = 32 * (K8D_SLABS + K8D_OUT + 1);
constexpr int K8D_CTAS = 2;                     // per SM
constexpr int K8D_SEQS = 256;                   // of one launch
constexpr int K8D_UNITS = 8;                    // descriptions of runs that are kept
constexpr int K8D_PAGES = K8D_RUN / KV8_PAGE;   // of a run
constexpr float K8D_LIFT = 7.0f;                // weights are 2^LIFT at the maximum: halves reach down to 2^-24
constexpr float K8D_LAZY = 8.0f;                // the maximum moves when it grew by more: 2^(LIFT + LAZY) is below the halves' 65504

struct Kv8DecodeParams {
  const bf16* q;             // [rows, n_q, D]
  const bf16* gate;          // [rows, n_q * D]
  const int64_t* positions;  // [rows]
  const int* tables;         // [B] rows of `width` pages, max_pages apart
  bf16* out;                 // [rows, n_q * D]
  float* part_acc;           // [rows, n_q, n_splits, D]: of rows with more than one run
  float2* part_ml;           // [rows, n_q, n_splits]: maximum (log 2) and sum
  int B, G, max_pages, width, num_pages, n_q, n_kv, group, n_splits;
  int rows_per_unit, units_per_seq;  // query rows whose heads fill a unit's columns; units that cover G rows
  int inv_group;             // column * inv_group >> 16 is column / group, for columns up to 16 of groups up to 16
  float scale_log2;
  int* err;
};

template <int D, int NT>
struct Kv8DecodeCfg {
  static constexpr int ROWB = D < 128 ? D : 128;           // bytes of a row in one swizzled block
  static constexpr int TILE = KV8_PAGE * D;                // a page's keys or values: a slot of their ring
  static constexpr int SLOTS = D == 256 ? 3 : D == 128 ? 6 : 8;
  static constexpr int EXPS = 2 * KV8_PAGE;                // exponents of a page's keys and values, with its keys
  static constexpr int SMEM = SLOTS * (2 * TILE + EXPS);
  static constexpr int PER = D / 16 / K8D_OUT;             // output tiles of 16 dims of a warp
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Barriers of the warps that take scores; all of them come to each one, whatever they have to do there.
__device__ __forceinline__ void meet_scores() { asm volatile("bar.sync 1, %0;" ::"n"(32 * K8D_SLABS) : "memory"); }
__device__ __forceinline__ bool meet_scores_or(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(any) : "r"(static_cast<uint32_t>(mine)), "n"(32 * K8D_SLABS) : "memory");
  return any != 0;
}

// A wait for a barrier that was looked at before.
__device__ __forceinline__ bool wait_seen(bool seen, uint64_t* bar, uint32_t parity, int* err, int code, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, seen) || mbar_wait_warp(bar, parity, err, code, abort_flag);
}

// Sequence b whose part [first[b], first[b + 1]) holds x.
template <class T>
__device__ __forceinline__ int kv8_find(const T* first, int B, int x) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// A unit is (sequence, group of its query rows, KV head, run). keys: of the run, up to the last that a row of the unit sees. same: the CTA's
// unit before has the same queries.
struct Kv8Unit {
  int seq, kh, z, row0, rows, keys, same;
};

__device__ __forceinline__ int kv8_length(int64_t position, int most) {
  return static_cast<int>(max(int64_t(-1), min(position, static_cast<int64_t>(most) - 1))) + 1;
}
__device__ __forceinline__ int kv8_length(const int64_t* positions, int row, int most) {
  return kv8_length(positions[row], most);
}

template <int D, int NT>
__global__ void __maxnreg__(96)  // two CTAs of 9 warps: five of a quarter SM at the most
kv8_decode_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ CUtensorMap tm_exps, Kv8DecodeParams p) {
  using C = Kv8DecodeCfg<D, NT>;
  constexpr int SLOTS = C::SLOTS, CHUNKS = D / 16, COLS = 8 * NT, DI = (D + 127) / 128, SLABS = K8D_SLABS;
  extern __shared__ __align__(1024) uint8_t smem_k8[];
  if (smem_u32(smem_k8) & 1023u) {  // the swizzled tiles need this alignment
    if (threadIdx.x == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    return;
  }
  uint8_t* const s_k = smem_k8;                        // [SLOTS] pages' keys
  uint8_t* const s_v = smem_k8 + SLOTS * C::TILE;      // [SLOTS] pages' values
  uint8_t* const s_exps = s_v + SLOTS * C::TILE;       // [SLOTS][keys' 64, values' 64]
  __shared__ __align__(8) uint64_t k_full[SLOTS], k_empty[SLOTS], v_full[SLOTS], v_empty[SLOTS];
  __shared__ __align__(8) uint64_t w_full[2], w_empty[2];   // weights of an even / odd page
  __shared__ __align__(8) uint64_t u_full[K8D_UNITS], u_empty[K8D_UNITS];
  __shared__ __align__(8) uint64_t l_full[2], l_empty[2];   // sums of an even / odd unit
  __shared__ int s_first[K8D_SEQS + 1];                // full runs of the sequences before
  __shared__ uint16_t s_tail[K8D_SEQS + 1];            // last runs that are not full, likewise
  __shared__ Kv8Unit s_unit[K8D_UNITS];
  __shared__ int s_len[K8D_UNITS][COLS];               // keys of the unit's rows
  __shared__ int s_scaled[2];
  __shared__ __align__(16) float s_max[SLABS][COLS], s_factor[2][COLS];   // read two columns at a time
  __shared__ float s_sum[2][SLABS][COLS], s_top[2][COLS], s_scale[COLS];
  __shared__ __align__(8) uint2 s_w[2][SLABS][NT][32]; // weights of a page, as the products' second operand
  __shared__ __align__(8) uint2 s_q[NT][CHUNKS][32];   // queries, likewise
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  volatile int* abort_flag = &s_abort;
  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; ++i) { mbar_init(&k_full[i], 1); mbar_init(&v_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_empty[i], K8D_OUT); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&w_full[i], SLABS); mbar_init(&w_empty[i], K8D_OUT);
      mbar_init(&l_full[i], SLABS); mbar_init(&l_empty[i], K8D_OUT);
    }
    for (int i = 0; i < K8D_UNITS; ++i) { mbar_init(&u_full[i], 1); mbar_init(&u_empty[i], SLABS + K8D_OUT); }
    s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm);
    tma_prefetch_desc(&tm_exps);
  }
  __syncthreads();
  pdl_wait();
  pdl_launch();
  const int most = min(p.width, p.n_splits * (K8D_RUN / KV8_PAGE)) * KV8_PAGE;  // keys that the tables can name

  if (warp == SLABS + K8D_OUT) {
    // ---------------- loads. The units are the runs of all sequences. Those of RUN keys are dealt out first, in one piece to each CTA, so that most follow
    // one of the same queries; what is left of each sequence goes round, beginning with the CTAs that got a unit less. Once the pages are on
    // their way any other load waits behind some 30 MB of them, 4 us: what a unit needs to know is asked for two units ahead, and published one ahead.
    const int per_seq = p.units_per_seq * p.n_kv;
    int full_before = 0, tails_before = 0;
    bool past = false;  // a row that stands behind its page table
    for (int b0 = 0; b0 < p.B; b0 += 128) {
      int len[4] = {0, 0, 0, 0};
#pragma unroll 4
      for (int r = 0; r < p.G; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = b0 + i * 32 + lane;
          if (b < p.B) {
            const int64_t position = p.positions[b * p.G + r];
            len[i] = max(len[i], kv8_length(position, most));
            past |= position >= most;
          }
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = b0 + i * 32 + lane;
        int full = len[i] / K8D_RUN;
        const uint32_t tails = __ballot_sync(0xffffffffu, b < p.B && (len[i] % K8D_RUN || len[i] == 0));  // one without keys has a run, which writes its zeros
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, full, o);
          if (lane >= o) full += u;
        }
        if (b < p.B) { s_first[b + 1] = full_before + full; s_tail[b + 1] = tails_before + __popc(tails & (2u << lane) - 1u); }
        full_before += __shfl_sync(0xffffffffu, full, 31);
        tails_before += __popc(tails);
      }
    }
    if (past) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    if (lane == 0) s_first[0] = s_tail[0] = 0;
    __syncwarp();
    const int grid = gridDim.x, cta = blockIdx.x;
    const int full = full_before * per_seq, tails = tails_before * per_seq, extra = full % grid;
    const int mine = full / grid + (cta < extra), first_full = cta * (full / grid) + min(cta, extra), first_tail = (cta + grid - extra) % grid;
    int seq_before = -1, k_before = 0;
    struct Ahead { Kv8Unit u; int64_t position; uint32_t page; };  // lane i: position of the unit's row i, page i of its run
    const auto ask = [&](int j) {  // unit j; rows of 0: there is none
      Ahead a = {};
      a.position = -1;
      int k;
      if (j < mine) {
        const int id = first_full + j;
        a.u.seq = kv8_find(s_first, p.B, id / per_seq);
        const int runs = s_first[a.u.seq + 1] - s_first[a.u.seq], at = id - s_first[a.u.seq] * per_seq;
        k = at / runs;
        a.u.z = at - k * runs;
      } else {
        const int id = first_tail + (j - mine) * grid, tail = id / per_seq;
        if (id >= tails) return a;
        a.u.seq = kv8_find(s_tail, p.B, tail);
        k = id - tail * per_seq;
        a.u.z = s_first[a.u.seq + 1] - s_first[a.u.seq];
      }
      a.u.same = a.u.seq == seq_before && k == k_before;
      seq_before = a.u.seq;
      k_before = k;
      const int rg = k / p.n_kv;
      a.u.kh = k - rg * p.n_kv;
      a.u.row0 = a.u.seq * p.G + rg * p.rows_per_unit;
      a.u.rows = min(p.rows_per_unit, p.G - rg * p.rows_per_unit);
      ask_64(a.position, p.positions + a.u.row0 + lane, lane < a.u.rows);
      ask_32(a.page, p.tables + static_cast<size_t>(a.u.seq) * p.max_pages + a.u.z * K8D_PAGES + lane,
             lane < K8D_PAGES && a.u.z * K8D_PAGES + lane < p.width);
      return a;
    };
    bool ok = true;
    const auto publish = [&](Ahead& a, int j) {
      const int us = j % K8D_UNITS;
      const int len = kv8_length(a.position, most);
      a.u.keys = max(0, min(K8D_RUN, __reduce_max_sync(0xffffffffu, len) - a.u.z * K8D_RUN));
      ok = ok && mbar_wait_warp(&u_empty[us], ((j / K8D_UNITS) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
      if (ok && lane < COLS) s_len[us][lane] = len;
      __syncwarp();
      if (ok && lane == 0) { s_unit[us] = a.u; mbar_arrive(&u_full[us]); }
    };
    Ahead now = ask(0), next = ask(1);
    publish(now, 0);
    int n = 0;
    for (int j = 0; now.u.rows > 0 && ok; ++j) {
      Ahead later = {};
      int pg = 0;
      const auto load = [&] {
        const int s = n % SLOTS;
        int page = static_cast<int>(__shfl_sync(0xffffffffu, now.page, pg));
        if (page < 0 || page >= p.num_pages) { if (lane == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX); page = 0; }
        const int row = (page * 2 * p.n_kv + now.u.kh) * KV8_PAGE;
        ok = mbar_wait_warp(&k_empty[s], ((n / SLOTS) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
        if (!ok) return;
        if (elect_one()) {
          mbar_expect_tx(&k_full[s], C::TILE + C::EXPS);
          tma_load_3d(s_k + s * C::TILE, &tm, &k_full[s], 0, row, 0);
          tma_load_3d(s_exps + s * C::EXPS, &tm_exps, &k_full[s], 0, now.u.kh, page * 2);
        }
        ok = mbar_wait_warp(&v_empty[s], ((n / SLOTS) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
        if (ok && elect_one()) {
          mbar_expect_tx(&v_full[s], C::TILE);
          tma_load_3d(s_v + s * C::TILE, &tm, &v_full[s], 0, row + p.n_kv * KV8_PAGE, 0);
        }
        ++n;
        ++pg;
      };
      if (now.u.keys > 0) load();
      later = ask(j + 2);
      if (j == 0) publish(next, 1);  // the warps of scores want it before they give a slot back
      while (pg * KV8_PAGE < now.u.keys && ok) load();
      publish(later, j + 2);
      now = next;
      next = later;
    }
    for (int i = max(0, n - SLOTS); !ok && i < n; ++i) {  // a wait that ran out leaves loads on their way: they end before the shared memory goes
      const long long t0 = clock64();
      while (!(mbar_try_wait(&k_full[i % SLOTS], (i / SLOTS) & 1) && mbar_try_wait(&v_full[i % SLOTS], (i / SLOTS) & 1)) && clock64() - t0 < WAIT_CYCLES / 8) {}
    }
    return;
  }
  // shared-memory offset of 16 bytes of a page's swizzled tile: row r, chunk c
  const auto tile_at = [&](uint32_t tile, int r, int c) {
    constexpr int PER = C::ROWB / 16;  // chunks of a block's row
    const int byte = r * C::ROWB;
    return tile + (c / PER) * (KV8_PAGE * C::ROWB) + byte + (((c % PER) ^ ((byte >> 7) & (PER - 1))) << 4);
  };
  const auto column = [&](int col, int& row, int& head) { row = col * p.inv_group >> 16; head = col - row * p.group; };
  const auto sync_arrive = [&](uint64_t* bar) { __syncwarp(); if (lane == 0) mbar_arrive(bar); };
  bool ok = true;
  int n = 0;  // pages so far

  if (warp < SLABS) {
    // ---------------- scores, maxima and weights: slab of keys, tiles of columns
    const int slab = warp;
    constexpr int QC = COLS / SLABS;  // query columns that a warp prepares
    uint2 raw[QC][DI];
    const auto fetch = [&](const Kv8Unit& u) {
#pragma unroll
      for (int i = 0; i < QC; ++i) {
        int row, head;
        column(slab * QC + i, row, head);
        // a column without a row takes the last one's: nothing reads what comes of it. No condition on the load, so that nothing waits for it here.
        const bf16* src = p.q + (static_cast<size_t>(u.row0 + min(row, u.rows - 1)) * p.n_q + u.kh * p.group + head) * D + lane * 4 % D;
#pragma unroll
        for (int k = 0; k < DI; ++k)
          asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(raw[i][k].x), "=r"(raw[i][k].y) : "l"(src + k * 128));
      }
    };
    // A unit's description; its queries are fetched one unit ahead. Either all these warps have it or none goes on: each stays in
    // step with the barriers of the others.
    bool known = false;
    const auto enter = [&](int j) {
      ok = ok && mbar_wait_warp(&u_full[j % K8D_UNITS], (j / K8D_UNITS) & 1, p.err, ERR_WAIT_FULL, abort_flag);
      known = ok = !meet_scores_or(!ok);
      if (!known) return;
      const Kv8Unit u = s_unit[j % K8D_UNITS];
      known = u.rows > 0;
      if (known && !u.same) fetch(u);
    };
    uint2 qf[NT == 1 ? CHUNKS : 1];  // queries of the column tile; those of two are read at each use
    float qscale[NT][2];   // what takes the product to log-2 scores
    enter(0);
    const auto keys_here = [&](int i) { return mbar_test(&k_full[i % SLOTS], (i / SLOTS) & 1); };
    for (int j = 0; known; ++j) {
      const int us = j % K8D_UNITS;
      const Kv8Unit u = s_unit[us];
      int last[NT][2];  // columns 2 t, 2 t + 1: last visible key of the run
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          int row, head;
          column(n8 * 8 + 2 * t + k, row, head);
          last[n8][k] = s_len[us][row] - 1 - u.z * K8D_RUN;
        }
      if (!u.same) {
        // queries as halves with the column's largest number in [2^10, 2^11), in the order of the products' second operand: lane
        // (column % 8, t) holds dims 16 c + 4 t .. + 3 of chunk c
#pragma unroll
        for (int i = 0; i < QC; ++i) {
          const int col = slab * QC + i;
          float x[DI][4];
          float top = 0.f;
          bool bad = false;
#pragma unroll
          for (int k = 0; k < DI; ++k) {
            const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw[i][k]);
            const float2 a = __bfloat1622float2(e[0]), b = __bfloat1622float2(e[1]);
            x[k][0] = a.x; x[k][1] = a.y; x[k][2] = b.x; x[k][3] = b.y;
#pragma unroll
            for (int h = 0; h < 4; ++h) { top = fmaxf(top, fabsf(x[k][h])); bad |= !(fabsf(x[k][h]) <= 3.4e38f); }
          }
          top = warp_max(top);
          const int e = max(-110, min(110, static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10));
          const float f = kv8_two_to(-e);
#pragma unroll
          for (int k = 0; k < DI; ++k) {
            if (lane * 4 + k * 128 < D) {
              const __half2 lo = __floats2half2_rn(x[k][0] * f, x[k][1] * f), hi = __floats2half2_rn(x[k][2] * f, x[k][3] * f);
              s_q[col / 8][k * 8 + lane / 4][col % 8 * 4 + lane % 4] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
          }
          // a NaN or an infinity anywhere in the column: all its scores are NaN
          const bool any = __any_sync(0xffffffffu, bad);
          if (lane == 0) s_scale[col] = any ? __uint_as_float(0x7fffffffu) : kv8_two_to(e) * p.scale_log2;
        }
        meet_scores();
#pragma unroll
        for (int c = 0; c < (NT == 1 ? CHUNKS : 0); ++c) qf[c] = s_q[0][c][lane];
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
          for (int k = 0; k < 2; ++k) qscale[n8][k] = s_scale[n8 * 8 + 2 * t + k];
      }
      enter(j + 1);
      bool k_seen = keys_here(n);  // barriers are looked at ahead of their wait, which takes its time even where there is none
      float m[NT][2], l[NT][2];
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8) {
        m[n8][0] = m[n8][1] = -INFINITY;
        l[n8][0] = l[n8][1] = 0.f;
      }

      for (int key0 = 0; key0 < u.keys; key0 += KV8_PAGE, ++n) {
        const int s = n % SLOTS, half = n & 1;
        const bool mine = key0 + slab * K8D_SLAB < u.keys;
        const bool w_seen = mbar_test(&w_empty[half], ((n >> 1) & 1) ^ 1);
        ok = ok && wait_seen(k_seen, &k_full[s], (n / SLOTS) & 1, p.err, ERR_WAIT_FULL, abort_flag);
        // S[key, column], keys g and g + 8 of this warp's slab
        float y[NT][2][2];  // [key][column 2 t, 2 t + 1]
        float vi[2];
        bool grown = false;
        if (ok && mine) {
          float sc[NT][2][4];  // two chains of products
#pragma unroll
          for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
            for (int k = 0; k < 4; ++k) sc[n8][0][k] = sc[n8][1][k] = 0.f;
          const uint32_t ktile = smem_u32(s_k + s * C::TILE);
#pragma unroll
          for (int c = 0; c < CHUNKS; c += 2) {
            uint32_t r[4];
            ldmatrix4(tile_at(ktile, slab * K8D_SLAB + (lane & 15), c + (lane >> 4)), r);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t a0, a1, a2, a3;
              kv8_unpack4(r[2 * h], a0, a2);
              kv8_unpack4(r[2 * h + 1], a1, a3);
#pragma unroll
              for (int n8 = 0; n8 < NT; ++n8) {
                const uint2 b = NT == 1 ? qf[NT == 1 ? c + h : 0] : s_q[n8][c + h][lane];
                mma_f16(sc[n8][h], a0, a1, a2, a3, b.x, b.y);
              }
            }
          }
          const uint8_t* ex = s_exps + s * C::EXPS + slab * K8D_SLAB + g;
          float kf[2], vb[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t vbyte = ex[KV8_PAGE + 8 * i];
            kf[i] = kv8_factor(ex[8 * i]);
            vb[i] = vbyte == KV8_E_NAN ? __uint_as_float(0x7fffffffu) : static_cast<float>(static_cast<int>(vbyte) - 127);
            vi[i] = kv8_two_to(max(-126, 127 - static_cast<int>(vbyte)));
          }
          const int key = key0 + slab * K8D_SLAB + g;
#pragma unroll
          for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float x = (sc[n8][0][2 * i + k] + sc[n8][1][2 * i + k]) * qscale[n8][k];
                y[n8][i][k] = key + 8 * i <= last[n8][k] ? fmaf(x, kf[i], vb[i]) : -INFINITY;
                grown |= y[n8][i][k] > m[n8][k] + K8D_LAZY;
              }
        }
        // a column whose maximum grew far enough takes the page's, which all warps see alike
        const bool any = meet_scores_or(grown);
        if (slab == 0 && lane == 0) mbar_arrive(&k_empty[s]);  // the group has read the keys
        if (any) {
#pragma unroll
          for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float mx = ok && mine ? fmaxf(y[n8][0][k], y[n8][1][k]) : -INFINITY;
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              if (g == 0) s_max[slab][n8 * 8 + 2 * t + k] = mx;
            }
          meet_scores();
        }
        k_seen = keys_here(n + 1);
        ok = ok && wait_seen(w_seen, &w_empty[half], ((n >> 1) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
        if (any) {
#pragma unroll
          for (int n8 = 0; n8 < NT; ++n8) {
            float2 top = make_float2(-INFINITY, -INFINITY), f = make_float2(1.f, 1.f);
#pragma unroll
            for (int w = 0; w < SLABS; ++w) {
              const float2 v = *reinterpret_cast<const float2*>(&s_max[w][n8 * 8 + 2 * t]);
              top.x = fmaxf(top.x, v.x);
              top.y = fmaxf(top.y, v.y);
            }
            if (top.x > m[n8][0] + K8D_LAZY) { f.x = ex2(m[n8][0] - top.x); m[n8][0] = top.x; l[n8][0] *= f.x; }  // 0 at the first key
            if (top.y > m[n8][1] + K8D_LAZY) { f.y = ex2(m[n8][1] - top.y); m[n8][1] = top.y; l[n8][1] *= f.y; }
            if (slab == 0 && g == 0) *reinterpret_cast<float2*>(&s_factor[half][n8 * 8 + 2 * t]) = f;
          }
        }
        if (slab == 0 && lane == 0) s_scaled[half] = any;
        if (ok && mine) {
#pragma unroll
          for (int n8 = 0; n8 < NT; ++n8) {
            float w[2][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float base = m[n8][k] == -INFINITY ? 0.f : m[n8][k] - K8D_LIFT;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                w[i][k] = ex2(y[n8][i][k] - base);
                l[n8][k] = fmaf(w[i][k], vi[i], l[n8][k]);
              }
            }
            uint32_t pw[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const __half2 two = __floats2half2_rn(w[i][0], w[i][1]);
              pw[i] = movmatrix(*reinterpret_cast<const uint32_t*>(&two));  // [column g][keys 2 t, 2 t + 1]
            }
            s_w[half][slab][n8][lane] = make_uint2(pw[0], pw[1]);
          }
        }
        sync_arrive(&w_full[half]);
      }

      // the unit's sums
      const int half = j & 1;
      ok = ok && mbar_wait_warp(&l_empty[half], ((j >> 1) & 1) ^ 1, p.err, ERR_WAIT_EMPTY, abort_flag);
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float sum = l[n8][k];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          if (g == 0) {
            s_sum[half][slab][n8 * 8 + 2 * t + k] = sum;
            if (slab == 0) s_top[half][n8 * 8 + 2 * t + k] = m[n8][k];
          }
        }
      __syncwarp();
      if (lane == 0) { mbar_arrive(&l_full[half]); mbar_arrive(&u_empty[us]); }
    }
    return;
  }

  // ---------------- outputs: O[dim, column], dims 16 c + 2 g and + 1 of tile c are the rows g and g + 8
  const int tile0 = (warp - SLABS) * C::PER;  // this warp's tiles
  for (int j = 0;; ++j) {
    const int us = j % K8D_UNITS;
    ok = ok && mbar_wait_warp(&u_full[us], (j / K8D_UNITS) & 1, p.err, ERR_WAIT_FULL, abort_flag);
    if (!ok) break;
    const Kv8Unit u = s_unit[us];
    if (u.rows == 0) break;
    float o[NT][C::PER][4];
    uint32_t gates[NT][2][C::PER];  // where a run is all there is, two dims each
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int r, h;
        column(n8 * 8 + 2 * t + k, r, h);
        const bool direct = p.n_splits == 1 && r < u.rows;
        const bf16* src = p.gate + (static_cast<size_t>(u.row0 + r) * p.n_q + u.kh * p.group + h) * D + tile0 * 16 + 2 * g;
#pragma unroll
        for (int i = 0; i < C::PER; ++i) {
          gates[n8][k][i] = 0u;
          ask_32(gates[n8][k][i], src + i * 16, direct);
        }
      }
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
      for (int i = 0; i < C::PER; ++i) o[n8][i][0] = o[n8][i][1] = o[n8][i][2] = o[n8][i][3] = 0.f;

    for (int key0 = 0; key0 < u.keys; key0 += KV8_PAGE, ++n) {
      const int s = n % SLOTS, half = n & 1;
      const int slabs = min(SLABS, (u.keys - key0 + K8D_SLAB - 1) / K8D_SLAB);
      ok = ok && mbar_wait_warp(&v_full[s], (n / SLOTS) & 1, p.err, ERR_WAIT_FULL, abort_flag)
           && mbar_wait_warp(&w_full[half], (n >> 1) & 1, p.err, ERR_WAIT_FULL, abort_flag);
      if (!ok) break;
      if (s_scaled[half]) {
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8) {
          const float2 f = *reinterpret_cast<const float2*>(&s_factor[half][n8 * 8 + 2 * t]);
#pragma unroll
          for (int i = 0; i < C::PER; ++i) { o[n8][i][0] *= f.x; o[n8][i][1] *= f.y; o[n8][i][2] *= f.x; o[n8][i][3] *= f.y; }
        }
      }
      const uint32_t vtile = smem_u32(s_v + s * C::TILE);
      const auto product = [&](float (*c)[4], int stride, const uint32_t* r, int slab) {  // both halves of a column tile's second operand at hand
        uint32_t a0, a1, a2, a3;
        kv8_unpack4(__byte_perm(r[0], 0, 0x3120), a0, a1);
        kv8_unpack4(__byte_perm(r[1], 0, 0x3120), a2, a3);
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8) {
          const uint2 w = s_w[half][slab][n8][lane];
          mma_f16(c[n8 * stride], a0, a1, a2, a3, w.x, w.y);
        }
      };
      if constexpr (C::PER >= 2) {  // two tiles and a slab per load
#pragma unroll
        for (int slab = 0; slab < SLABS; ++slab) {
          if (slab >= slabs) break;
#pragma unroll
          for (int i = 0; i < C::PER; i += 2) {
            uint32_t r[4];
            ldmatrix4_trans(tile_at(vtile, slab * K8D_SLAB + (lane & 15), tile0 + i + (lane >> 4)), r);
            product(&o[0][i], C::PER, r, slab);
            product(&o[0][i + 1], C::PER, r + 2, slab);
          }
        }
      } else {  // a tile and two slabs per load
#pragma unroll
        for (int slab = 0; slab < SLABS; slab += 2) {
          if (slab >= slabs) break;
          uint32_t r[4];
          ldmatrix4_trans(tile_at(vtile, slab * K8D_SLAB + lane, tile0), r);
          product(&o[0][0], 1, r, slab);
          if (slab + 1 < slabs) product(&o[0][0], 1, r + 2, slab + 1);
        }
      }
      __syncwarp();
      if (lane == 0) { mbar_arrive(&v_empty[s]); mbar_arrive(&w_empty[half]); }
    }

    const int half = j & 1;
    ok = ok && mbar_wait_warp(&l_full[half], (j >> 1) & 1, p.err, ERR_WAIT_FULL, abort_flag);
    if (!ok) break;
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int r, h;
        column(n8 * 8 + 2 * t + k, r, h);
        if (r >= u.rows) continue;
        const int len = s_len[us][r];
        const size_t head = static_cast<size_t>(u.row0 + r) * p.n_q + u.kh * p.group + h;
        const auto sum = [&] {
          float x = 0.f;
#pragma unroll
          for (int w = 0; w < SLABS; ++w) x += s_sum[half][w][n8 * 8 + 2 * t + k];
          return x;
        };
        if (p.n_splits > 1) {
          if (u.z * K8D_RUN < len) {
            const size_t slot = head * p.n_splits + u.z;
            if (tile0 == 0 && g == 0) p.part_ml[slot] = make_float2(s_top[half][n8 * 8 + 2 * t + k], sum());
#pragma unroll
            for (int i = 0; i < C::PER; ++i)
              *reinterpret_cast<float2*>(p.part_acc + slot * D + (tile0 + i) * 16 + 2 * g) = make_float2(o[n8][i][k], o[n8][i][2 + k]);
          }
        } else {
          const float inv = len > 0 ? 1.0f / sum() : 0.f;
#pragma unroll
          for (int i = 0; i < C::PER; ++i) {
            const size_t at = head * D + (tile0 + i) * 16 + 2 * g;
            const float2 gate = kv8_sigmoid2(gates[n8][k][i]);
            *reinterpret_cast<__nv_bfloat162*>(p.out + at) =
                __floats2bfloat162_rn(o[n8][i][k] * inv * gate.x, o[n8][i][2 + k] * inv * gate.y);
          }
        }
      }
    __syncwarp();
    if (lane == 0) { mbar_arrive(&l_empty[half]); mbar_arrive(&u_empty[us]); }
  }
}

// What the runs of a row come to. Partial z goes to sum z % 16, at the sum's own maximum, and the sums are added in order: one chain over
// the partials where there are up to 16. What does not come from the kernel in front is read ahead of the dependency wait: that kernel has
// waited for everything before it.
constexpr int K8D_SUMS = 16;
// Sums i0 .. i0 + 3 of four dims, their partials `D` floats apart. (Where a row has up to 16 runs, each is its sum: no step is lost on maxima of one.)
template <int D>
__device__ __forceinline__ void k8d_sums(const float4* pa, const float2* ml, int runs, int i0, float* top, float* l, float4* acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) { top[i] = -INFINITY; l[i] = 0.f; acc[i] = make_float4(0.f, 0.f, 0.f, 0.f); }
#pragma unroll 4
  for (int z0 = i0; z0 < runs; z0 += K8D_SUMS)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (z0 + i < runs) top[i] = fmaxf(top[i], ml[z0 + i].x);
#pragma unroll 2
  for (int z0 = i0; z0 < runs; z0 += K8D_SUMS) {
    float2 pm[4];
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pm[i] = z0 + i < runs ? ml[z0 + i] : make_float2(-INFINITY, 0.f);
      v[i] = z0 + i < runs ? pa[static_cast<size_t>(z0 + i) * (D / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = pm[i].x == top[i] ? 1.f : ex2(pm[i].x - top[i]);
      l[i] = fmaf(pm[i].y, f, l[i]);  // a partial without a maximum holds no key, or scores that are all NaN, in its sum
      acc[i].x = fmaf(v[i].x, f, acc[i].x); acc[i].y = fmaf(v[i].y, f, acc[i].y);
      acc[i].z = fmaf(v[i].z, f, acc[i].z); acc[i].w = fmaf(v[i].w, f, acc[i].w);
    }
  }
}
__device__ __forceinline__ void k8d_add(float best, float top, float l, const float4& acc, float& sum, float4& o) {
  const float f = top == best ? 1.f : ex2(top - best);
  sum = fmaf(l, f, sum);
  o.x = fmaf(acc.x, f, o.x); o.y = fmaf(acc.y, f, o.y); o.z = fmaf(acc.z, f, o.z); o.w = fmaf(acc.w, f, o.w);
}
__device__ __forceinline__ void k8d_store(bf16* out, uint2 gate, const float4& o, float sum, bool any) {
  const float inv = any ? 1.0f / sum : 0.f;  // a row without keys
  const float2 g0 = kv8_sigmoid2(gate.x), g1 = kv8_sigmoid2(gate.y);
  uint2 raw;
  __nv_bfloat162* e = reinterpret_cast<__nv_bfloat162*>(&raw);
  e[0] = __floats2bfloat162_rn(o.x * inv * g0.x, o.y * inv * g0.y);
  e[1] = __floats2bfloat162_rn(o.z * inv * g1.x, o.w * inv * g1.y);
  *reinterpret_cast<uint2*>(out) = raw;
}
// Tables of up to 64 runs (32,768 keys): a thread takes all sums of four dims of a head. Its CTAs are small enough to wait beside the
// kernel in front.
template <int D>
__global__ void __maxnreg__(72)
kv8_combine_few_kernel(const float* part_acc, const float2* part_ml, const bf16* gate, const int64_t* positions, bf16* out, int heads,
                       int n_q, int n_splits, int most) {
  constexpr int QUADS = D / 4;
  const size_t head = static_cast<size_t>(blockIdx.x) * (128 / QUADS) + threadIdx.x / QUADS;
  const int quad = threadIdx.x % QUADS;
  const int runs = head < heads ? (kv8_length(positions, static_cast<int>(head / n_q), most) + K8D_RUN - 1) / K8D_RUN : 0;
  const size_t at = head * D + quad * 4;
  const uint2 g = head < heads ? *reinterpret_cast<const uint2*>(gate + at) : make_uint2(0u, 0u);
  pdl_wait();
  pdl_launch();
  if (head >= heads) return;
  const float2* ml = part_ml + head * n_splits;
  const float4* pa = reinterpret_cast<const float4*>(part_acc + head * n_splits * D) + quad;
  float best = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (runs <= K8D_SUMS) {  // a sum has one partial: it is that one, and all are asked for at once
    constexpr int AT_ONCE = 6;
    float2 pm[AT_ONCE];
    float4 v[AT_ONCE];
    const auto ask = [&](int z0) {
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        pm[i] = z0 + i < runs ? ml[z0 + i] : make_float2(-INFINITY, 0.f);
        v[i] = z0 + i < runs ? pa[static_cast<size_t>(z0 + i) * QUADS] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    };
    ask(0);
    for (int z = AT_ONCE; z < runs; ++z) best = fmaxf(best, ml[z].x);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) best = fmaxf(best, pm[i].x);
    for (int z0 = 0;;) {
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) k8d_add(best, pm[i].x, pm[i].y, v[i], sum, o);
      z0 += AT_ONCE;
      if (z0 >= runs) break;
      ask(z0);
    }
  } else {
#pragma unroll 8
    for (int z = 0; z < runs; ++z) best = fmaxf(best, ml[z].x);
    for (int i = 0; i < K8D_SUMS; i += 4) {
      float top[4], l[4];
      float4 acc[4];
      k8d_sums<D>(pa, ml, runs, i, top, l, acc);
#pragma unroll
      for (int k = 0; k < 4; ++k) k8d_add(best, top[k], l[k], acc[k], sum, o);
    }
  }
  k8d_store(out + at, g, o, sum, runs > 0);
}
// More: a CTA takes 64 dims of a head, a thread one sum of four of them, eight of its partials under way; rows of few runs as above.
template <int D>
__global__ void __launch_bounds__(256)
kv8_combine_kernel(const float* part_acc, const float2* part_ml, const bf16* gate, const int64_t* positions, bf16* out, int n_q,
                   int n_splits, int most) {
  constexpr int DIMS = 64, QUADS = DIMS / 4;
  __shared__ float4 s_acc[K8D_SUMS][QUADS];
  __shared__ float s_top[K8D_SUMS], s_l[K8D_SUMS];
  const size_t head = blockIdx.x;
  const int quad = threadIdx.x % QUADS, i = threadIdx.x / QUADS;
  const int runs = (kv8_length(positions, static_cast<int>(head / n_q), most) + K8D_RUN - 1) / K8D_RUN;
  const size_t at = head * D + blockIdx.y * DIMS + quad * 4;
  const uint2 g = *reinterpret_cast<const uint2*>(gate + at);
  pdl_wait();
  pdl_launch();
  const float2* ml = part_ml + head * n_splits;
  const float4* pa = reinterpret_cast<const float4*>(part_acc + head * n_splits * D + blockIdx.y * DIMS) + quad;
  if (i < K8D_SUMS) {
    float top = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int AT_ONCE = 8;
    for (int z0 = i; z0 < runs; z0 += AT_ONCE * K8D_SUMS) {
      float2 pm[AT_ONCE];
      float4 v[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int z = z0 + k * K8D_SUMS;
        pm[k] = z < runs ? ml[z] : make_float2(-INFINITY, 0.f);
        v[k] = z < runs ? pa[static_cast<size_t>(z) * (D / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float next = top;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) next = fmaxf(next, pm[k].x);
      const float f = next == top ? 1.f : ex2(top - next);
      top = next;
      l *= f; acc.x *= f; acc.y *= f; acc.z *= f; acc.w *= f;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) k8d_add(top, pm[k].x, pm[k].y, v[k], l, acc);
    }
    s_acc[i][quad] = acc;
    if (quad == 0) { s_top[i] = top; s_l[i] = l; }
  }
  __syncthreads();
  if (i > 0) return;
  float best = -INFINITY, sum = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < K8D_SUMS; ++k) best = fmaxf(best, s_top[k]);
  for (int k = 0; k < K8D_SUMS; ++k) k8d_add(best, s_top[k], s_l[k], s_acc[k][quad], sum, o);
  k8d_store(out + at, g, o, sum, runs > 0);
}

}  // namespace b200

using namespace b200;

namespace {
// A page's keys or values of one head, in blocks of at most 128 bytes per row; their exponents, of keys and values together.
int k8d_make_maps(CUtensorMap* tm, CUtensorMap* tm_exps, const void* data, const void* exps, int D, int n_kv, long long pages) {
  const cuuint32_t rowb = D < 128 ? D : 128;
  const cuuint64_t dims[3] = {rowb, static_cast<cuuint64_t>(pages) * 2 * n_kv * KV8_PAGE, D / rowb};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D), rowb};
  const cuuint32_t box[3] = {rowb, KV8_PAGE, D / rowb};
  const int rc = kv8_encode(tm, data, 3, dims, strides, box, rowb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
  return rc ? rc : kv8_encode_exps(tm_exps, exps, n_kv, pages);
}

template <int D, int NT>
int k8d_launch(const CUtensorMap& tm, const CUtensorMap& tm_exps, const Kv8DecodeParams& p, cudaStream_t st) {
  auto kern = kv8_decode_kernel<D, NT>;
  static int sms_of[64] = {};  // per device, with the function attribute set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (sms_of[dev] == 0) {
    int sms = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8DecodeCfg<D, NT>::SMEM) != cudaSuccess) return -3;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
    sms_of[dev] = sms;
  }
  const long long units = static_cast<long long>(p.B) * p.units_per_seq * p.n_kv * p.n_splits;
  const int most_ctas = sms_of[dev] * K8D_CTAS;
  const int grid = static_cast<int>(units < most_ctas ? units : most_ctas);
  if (launch_pdl(kern, dim3(grid), dim3(K8D_THREADS), Kv8DecodeCfg<D, NT>::SMEM, st, tm, tm_exps, p) != cudaSuccess) return -4;
  if (p.n_splits == 1) return 0;
  const int most = (p.width < p.n_splits * (K8D_RUN / KV8_PAGE) ? p.width : p.n_splits * (K8D_RUN / KV8_PAGE)) * KV8_PAGE;
  const int heads = p.B * p.G * p.n_q, per = 128 / (D / 4);
  const cudaError_t rc = p.n_splits <= 64
      ? launch_pdl(kv8_combine_few_kernel<D>, dim3((heads + per - 1) / per), dim3(128), 0, st, p.part_acc, p.part_ml, p.gate,
                   p.positions, p.out, heads, p.n_q, p.n_splits, most)
      : launch_pdl(kv8_combine_kernel<D>, dim3(heads, D / 64), dim3(256), 0, st, p.part_acc, p.part_ml, p.gate,
                   p.positions, p.out, p.n_q, p.n_splits, most);
  return rc == cudaSuccess ? 0 : -4;
}
}  // namespace

// Keys of a run: the caller sizes the partials by it.
extern "C" int b200_kv8_decode_run(void) { return K8D_RUN; }

// q: [B * G, n_q, D] bf16 (normed and rotated), G rows per sequence; gate, out: [B * G, n_q * D]; data, exps: one layer of the 8-bit cache, which
// holds the rows' own keys; positions [B * G] (negative: a row without keys, whose output is 0; behind the page table: an error, and the table's keys); tables [B] rows of `width` pages.
// n_splits runs cover a row of the tables; part_acc [B * G, n_q, n_splits, D] and part_ml [.., 2] where n_splits > 1.
extern "C" int b200_kv8_decode(const void* q, const void* gate, const void* data, const void* exps, const int64_t* positions,
                               const int* tables, int max_pages, int width, int num_pages, int B, int G, int n_q, int n_kv, int D,
                               int n_splits, float* part_acc, float* part_ml, void* out, int* err, cudaStream_t st) {
  if (B <= 0 || G <= 0) return 0;
  const int group = n_kv > 0 ? n_q / n_kv : 0;
  if (group < 1 || group * n_kv != n_q || group > 16 || n_splits < 1) return -7;
  const long long rows = static_cast<long long>(num_pages) * 2 * n_kv * KV8_PAGE;
  if (rows > 0x7fffffffLL) return -7;  // a TMA coordinate
  if (reinterpret_cast<uintptr_t>(data) % 16 || reinterpret_cast<uintptr_t>(exps) % 16 || reinterpret_cast<uintptr_t>(q) % 8) return -7;
  if (D != 256 && D != 128 && D != 64) return -7;
  CUtensorMap tm, tm_exps;
  if (k8d_make_maps(&tm, &tm_exps, data, exps, D, n_kv, num_pages)) return -1;
  const int cols = G * group, nt = cols <= 8 ? 1 : 2, per = 8 * nt / group < G ? 8 * nt / group : G;
  int rc = -7;
  for (int b0 = 0; b0 < B; b0 += K8D_SEQS) {
    const int n = B - b0 < K8D_SEQS ? B - b0 : K8D_SEQS;
    if (static_cast<long long>(n) * G * n_kv * n_splits > 0x3fffffffLL) return -7;  // the units are counted in 32 bits
    const size_t heads = static_cast<size_t>(b0) * G * n_q;
    const Kv8DecodeParams p{static_cast<const bf16*>(q) + heads * D, static_cast<const bf16*>(gate) + heads * D,
                            positions + static_cast<size_t>(b0) * G,
                            tables + static_cast<size_t>(b0) * max_pages, static_cast<bf16*>(out) + heads * D,
                            part_acc + heads * n_splits * D, reinterpret_cast<float2*>(part_ml) + heads * n_splits,
                            n, G, max_pages, width, num_pages, n_q, n_kv, group, n_splits, per, (G + per - 1) / per, (65536 + group - 1) / group,
                            1.4426950408889634f / sqrtf(static_cast<float>(D)), err};
#define K8D(DD) rc = nt == 1 ? k8d_launch<DD, 1>(tm, tm_exps, p, st) : k8d_launch<DD, 2>(tm, tm_exps, p, st)
    if (D == 256) K8D(256);
    else if (D == 128) K8D(128);
    else K8D(64);
#undef K8D
    if (rc) return rc;
  }
  return 0;
}

// Attention of a few query rows per sequence (decode steps, verify passes) over the 8-bit paged cache.
//
//   s_j = q . (k_j 2^a_j) / sqrt D,   o = sum_j p_j (v_j 2^b_j) / sum_j p_j,   p_j = exp(s_j),   out = o * sigmoid(gate)
//
// with e4m3 rows k_j, v_j and their powers of two. Neither row is ever scaled: y_j = s_j log2(e) + b_j takes the value's power of
// two into the exponent, w_j = 2^(y_j - M) is the weight of the stored v_j, M the running maximum of y, and the softmax's own sum is
// sum_j w_j 2^-b_j. So what the matrix instructions get are the stored numbers as halves (exact) and weights below 2^15.
//
// Bound: the cache's bytes, 2 (D + 1) per token and KV head. A context is cut into runs of RUN keys at fixed places, so what a row's
// result is put together from depends on its own position only, never on the batch; a persistent CTA per SM takes runs in turn. Blocks of 128 keys
// come into a ring by TMA, the next runs' blocks ahead of this one's end. On a block the eight warps first take 16 keys each
// (S = K Q^T, maximum, weights), then D / 8 dims each over all keys (O += V^T P): a warp's part of the output is 2 tiles of 16 dims,
// so nothing of the output is ever exchanged, only maxima and weights, 16 bytes per key. (With all dims of every eighth slab in
// each warp, the warps' outputs were added up at each run's end, which took more instructions than the run: 74 us for 128 sequences of about 1,060.)
// The products are m16n8k16 with keys or dims as the 16 rows and query columns as the 8: one token of one KV head's eight query heads
// fills the columns, where a tcgen05 tile would be 8 rows of 64. The stored bytes become halves in registers, behind ldmatrix.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace b200 {

constexpr int K8D_RUN = 512;                    // keys of a run: part of the numerics
constexpr int K8D_WARPS = 8;                    // that compute
constexpr int K8D_SLAB = 16;                    // keys of a warp's scores
constexpr int K8D_BLOCK = K8D_WARPS * K8D_SLAB; // keys of a ring stage: two pages
constexpr int K8D_MAX_SEQS = 1024;              // of one launch
constexpr float K8D_LIFT = 7.0f;                // weights are 2^LIFT at the maximum: halves reach down to 2^-24
constexpr float K8D_LAZY = 8.0f;                // the maximum moves when it grew by more: 2^(LIFT + LAZY) is below the halves' 65504

struct Kv8DecodeParams {
  const bf16* q;             // [rows, n_q, D]
  const bf16* gate;          // [rows, n_q * D]
  const uint8_t* exps;       // [pages, 2, n_kv, 64]
  const int64_t* positions;  // [rows]
  const int* tables;         // [B] rows of `width` pages, max_pages apart
  bf16* out;                 // [rows, n_q * D]
  float* part_acc;           // [rows, n_q, n_splits, D]: of rows with more than one run
  float2* part_ml;           // [rows, n_q, n_splits]: maximum (log 2) and sum
  int B, G, max_pages, width, num_pages, n_q, n_kv, group, n_splits;
  int rows_per_unit, units_per_seq;  // query rows whose heads fill a unit's columns; units that cover G rows
  int inv_group;             // column * inv_group >> 16 is column / group, for columns up to 32 of groups up to 16
  float scale_log2;
  int* err;
};

template <int D, int NT>
struct Kv8DecodeCfg {
  static constexpr int ROWB = D < 128 ? D : 128;           // bytes of a row in one swizzled block
  static constexpr int DB = D / ROWB;
  static constexpr int TILE = KV8_PAGE * D;                // a page's keys or values
  static constexpr int SLOT = 2 * TILE;                    // of the ring: the keys of a block or its values
  static constexpr int CTAS = NT == 1 ? 2 : 1;             // per SM: one column tile's registers leave room for sixteen warps
  static constexpr int SLOTS = (D == 256 ? 3 : D == 128 ? 6 : 8) * (D == 256 && NT > 1 ? 2 : 1);
  static constexpr int EXPS = 4 * KV8_PAGE;                // exponents of a block's keys and values, with its keys
  static constexpr int SMEM = SLOTS * (SLOT + EXPS);
  static constexpr int TILES = D / 16;                     // output tiles of 16 dims
  static constexpr int PER = TILES > K8D_WARPS ? TILES / K8D_WARPS : 1;  // of a warp
  static constexpr int SPLIT = TILES < K8D_WARPS ? K8D_WARPS / TILES : 1;  // warps that share a tile, a part of the keys each
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
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Sequence whose runs [first[b], first[b + 1]) hold run x.
__device__ __forceinline__ int kv8_find(const int* first, int B, int x) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// A unit is (sequence, group of its query rows, KV head, run). keys: of the run, up to the last that a row of the unit sees.
struct Kv8Unit {
  int seq, kh, z, row0, rows, keys;
};

template <int D, int NT>
__global__ void __launch_bounds__(32 * K8D_WARPS, Kv8DecodeCfg<D, NT>::CTAS)
kv8_decode_kernel(const __grid_constant__ CUtensorMap tm, Kv8DecodeParams p) {
  using C = Kv8DecodeCfg<D, NT>;
  constexpr int SLOTS = C::SLOTS, CHUNKS = D / 16, COLS = 8 * NT, SLABS = K8D_WARPS, DI = (D + 127) / 128;
  extern __shared__ __align__(1024) uint8_t smem_k8[];
  if (smem_u32(smem_k8) & 1023u) {  // the swizzled tiles need this alignment
    if (threadIdx.x == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    return;
  }
  uint8_t* s_exps = smem_k8 + SLOTS * C::SLOT;
  __shared__ __align__(8) uint64_t full[SLOTS];
  __shared__ int s_first[K8D_MAX_SEQS + 1];            // runs of the sequences before
  __shared__ Kv8Unit s_unit[64];                       // this CTA's units, a ring in two halves
  __shared__ __align__(16) float s_max[SLABS][COLS], s_sum[SLABS][COLS];  // read two columns at a time
  __shared__ __align__(8) uint2 s_w[SLABS][NT][32];    // weights of a block, as the products' second operand
  __shared__ __align__(8) uint2 s_q[NT][CHUNKS][32];   // queries, likewise
  __shared__ float s_scale[COLS];
  __shared__ __align__(16) float s_o[C::SPLIT > 1 ? K8D_WARPS : 1][C::SPLIT > 1 ? NT * 4 : 1][32];
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1);
    s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm);
  }
  pdl_wait();
  pdl_launch();
  const int most = min(p.width, p.n_splits * (K8D_RUN / KV8_PAGE)) * KV8_PAGE;  // keys that the tables can name
  const auto length = [&](int row) { return max(0, min(static_cast<int>(min(__ldg(p.positions + row), static_cast<int64_t>(most))) + 1, most)); };
  for (int b = threadIdx.x; b < p.B; b += blockDim.x) {
    int len = 0;
    for (int i = 0; i < p.G; ++i) len = max(len, length(b * p.G + i));
    s_first[b + 1] = max(1, (len + K8D_RUN - 1) / K8D_RUN);  // a sequence without keys has a run, which writes its zeros
  }
  __syncthreads();
  if (warp == 0) {  // inclusive sums, a lane a stretch of sequences
    const int per = (p.B + 31) / 32, b0 = min(p.B, lane * per), b1 = min(p.B, b0 + per);
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += s_first[b + 1];
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += u;
    }
    upto -= sum;
    for (int b = b0; b < b1; ++b) { upto += s_first[b + 1]; s_first[b + 1] = upto; }
    if (lane == 0) s_first[0] = 0;
  }
  __syncthreads();
  const int per_run = p.n_kv * p.units_per_seq, total = s_first[p.B] * per_run;
  const int n_units = (total - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);  // of this CTA
  volatile int* abort_flag = &s_abort;
  const auto describe = [&](int j) {  // unit j of this CTA, by one lane
    if (j >= n_units) return;
    Kv8Unit u;
    const int id = blockIdx.x + j * gridDim.x, run = id / per_run, x = id % per_run, rg = x % p.units_per_seq;
    u.kh = x / p.units_per_seq;
    u.seq = kv8_find(s_first, p.B, run);
    u.z = run - s_first[u.seq];
    u.row0 = u.seq * p.G + rg * p.rows_per_unit;
    u.rows = min(p.rows_per_unit, (u.seq + 1) * p.G - u.row0);
    int len = 0;
    for (int r = 0; r < u.rows; ++r) len = max(len, length(u.row0 + r));
    u.keys = max(0, min(K8D_RUN, len - u.z * K8D_RUN));
    s_unit[j % 64] = u;
  };
  if (warp < 2) describe(threadIdx.x);
  __syncthreads();

  // ---------------- loads, by the last warp. The ring takes a block's keys, then its values; by the first meeting on block k all warps have
  // read the keys of block k and the values of block k - 1. The page numbers of a unit are read a unit ahead.
  struct { int j, kh, pages, pg, ids; } cur = {}, nxt = {};
  int issued = 0;  // slots asked for
  const auto look = [&](decltype(cur)& w, int j, int limit) {  // the first unit from j on that has keys, below `limit`
    for (; j < limit && j < n_units; ++j) {
      const Kv8Unit& u = s_unit[j % 64];
      if (u.keys == 0) continue;
      w.kh = u.kh;
      w.pg = 0;
      w.pages = (u.keys + KV8_PAGE - 1) / KV8_PAGE;
      w.ids = 0;
      if (lane < w.pages) w.ids = __ldg(p.tables + static_cast<size_t>(u.seq) * p.max_pages + u.z * (K8D_RUN / KV8_PAGE) + lane);
      break;
    }
    w.j = j;
    return j < limit && j < n_units;
  };
  bool have = false, have_next = false;  // cur, nxt hold a unit
  const auto issue = [&](int upto, int limit) {
    while (issued < upto) {
      if (!have) { have = have_next; cur = nxt; have_next = false; }
      if (!have) { have = look(cur, cur.j, limit); nxt.j = cur.j + have; }
      if (!have_next) have_next = look(nxt, max(nxt.j, cur.j + have), limit);
      if (!have) { cur.j = nxt.j; return; }
      const int s = issued % SLOTS, of = min(2, cur.pages - cur.pg), values = issued & 1;
      int page = __shfl_sync(0xffffffffu, cur.ids, cur.pg + (lane & 1));
      if (lane == 0) mbar_expect_tx(&full[s], of * (C::TILE + (values ? 0 : 2 * KV8_PAGE)));
      __syncwarp();
      if (lane < 4 && (lane & 1) < of) {  // lanes 0, 1: the tiles and their keys' exponents, 2, 3: the values' exponents
        if (page < 0 || page >= p.num_pages) { atomicCAS(p.err, 0, ERR_BAD_INDEX); page = 0; }
        const int row = ((page * 2 + (lane >> 1)) * p.n_kv + cur.kh) * KV8_PAGE;
        if (lane < 2) tma_load_3d(smem_k8 + s * C::SLOT + lane * C::TILE, &tm, &full[s], 0, row + values * p.n_kv * KV8_PAGE, 0);
        if (!values) bulk_load(s_exps + s * C::EXPS + lane * KV8_PAGE, p.exps + row, KV8_PAGE, &full[s]);
      }
      ++issued;
      if (values) {
        cur.pg += 2;
        if (cur.pg >= cur.pages) { have = false; cur.j = nxt.j; }
      }
    }
  };
  if (warp == K8D_WARPS - 1) issue(SLOTS, 64);

  // shared-memory offset of 16 bytes of a page's swizzled tile: row r, chunk c
  const auto tile_at = [&](uint32_t tile, int r, int c) {
    constexpr int PER = C::ROWB / 16;  // chunks of a block's row
    const int byte = r * C::ROWB;
    return tile + (c / PER) * (KV8_PAGE * C::ROWB) + byte + (((c % PER) ^ ((byte >> 7) & (PER - 1))) << 4);
  };
  const int tile0 = warp % C::TILES * C::PER, part = warp / C::TILES;  // this warp's output tiles, and which part of the keys
  bool ok = true;
  int n = 0;  // blocks so far: their keys are in slot 2 n, their values in 2 n + 1

  const auto column = [&](int col, int& row, int& head) { row = col * p.inv_group >> 16; head = col - row * p.group; };
  uint2 qnext[NT][DI];   // the next unit's queries, a warp a column
  const auto fetch = [&](const Kv8Unit& u) {
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8) {
      int row, head;
      column(n8 * 8 + warp, row, head);
      const bf16* src = p.q + (static_cast<size_t>(u.row0 + row) * p.n_q + u.kh * p.group + head) * D + lane * 4;
#pragma unroll
      for (int i = 0; i < DI; ++i)
        qnext[n8][i] = row < u.rows && lane * 4 + i * 128 < D ? *reinterpret_cast<const uint2*>(src + i * 128) : make_uint2(0u, 0u);
    }
  };
  if (n_units > 0) fetch(s_unit[0]);

  for (int j = 0; j < n_units; ++j) {
    const Kv8Unit u = s_unit[j % 64];
    const int n_cols = u.rows * p.group;
    if (warp == K8D_WARPS - 1) issue(2 * n + SLOTS, j / 32 * 32 + 32);
    // ---- queries as halves with the column's largest number in [2^10, 2^11), in the order of the products' second operand: lane
    // (column % 8, t) holds dims 16 c + 4 t .. + 3 of chunk c
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8) {
      float x[DI][4];
      float top = 0.f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < DI; ++i) {
        const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&qnext[n8][i]);
        const float2 a = __bfloat1622float2(e[0]), b = __bfloat1622float2(e[1]);
        x[i][0] = a.x; x[i][1] = a.y; x[i][2] = b.x; x[i][3] = b.y;
#pragma unroll
        for (int k = 0; k < 4; ++k) { top = fmaxf(top, fabsf(x[i][k])); bad |= !(fabsf(x[i][k]) <= 3.4e38f); }
      }
      top = warp_max(top);
      const int e = max(-110, min(110, static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10));
      const float f = kv8_two_to(-e);
#pragma unroll
      for (int i = 0; i < DI; ++i) {
        if (lane * 4 + i * 128 < D) {
          const __half2 lo = __floats2half2_rn(x[i][0] * f, x[i][1] * f), hi = __floats2half2_rn(x[i][2] * f, x[i][3] * f);
          s_q[n8][i * 8 + lane / 4][warp * 4 + lane % 4] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
      }
      // a NaN or an infinity anywhere in the column: all its scores are NaN
      const bool any = __any_sync(0xffffffffu, bad);
      if (lane == 0) s_scale[n8 * 8 + warp] = any ? __uint_as_float(0x7fffffffu) : kv8_two_to(e) * p.scale_log2;
    }
    int len[NT][2];        // columns 2 t, 2 t + 1: keys of their rows (0: no such column)
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        int row, head;
        column(n8 * 8 + 2 * t + k, row, head);
        len[n8][k] = row < u.rows ? length(u.row0 + row) : 0;
      }
    if (j + 1 < n_units) fetch(s_unit[(j + 1) % 64]);
    __syncthreads();
    uint2 qf[NT][CHUNKS];
    float qscale[NT][2];   // what takes the product to log-2 scores
    int last[NT][2];       // last visible key of the run
    float m[NT][2], l[NT][2], o[NT][C::PER][4];
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) qf[n8][c] = s_q[n8][c][lane];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        qscale[n8][k] = s_scale[n8 * 8 + 2 * t + k];
        last[n8][k] = len[n8][k] - 1 - u.z * K8D_RUN;
        m[n8][k] = -INFINITY;
        l[n8][k] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < C::PER; ++i) o[n8][i][0] = o[n8][i][1] = o[n8][i][2] = o[n8][i][3] = 0.f;
    }

    for (int key0 = 0; key0 < u.keys; key0 += K8D_BLOCK, ++n) {
      const int slabs = min(SLABS, (u.keys - key0 + K8D_SLAB - 1) / K8D_SLAB);
      const bool mine = warp < slabs;
      const int ks = 2 * n % SLOTS, vs = (2 * n + 1) % SLOTS;
      ok = ok && mbar_wait_warp(&full[ks], (2 * n / SLOTS) & 1, p.err, ERR_WAIT_FULL, abort_flag);
      // ---- scores of this warp's slab: S[key, column], keys g and g + 8
      float y[NT][2][2];  // [key][column 2 t, 2 t + 1]
      float vi[2];
      bool grown = false;
      if (ok && mine) {
        float sc[NT][2][4];  // two chains of products
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
          for (int k = 0; k < 4; ++k) sc[n8][0][k] = sc[n8][1][k] = 0.f;
        const uint32_t ktile = smem_u32(smem_k8 + ks * C::SLOT) + warp / 4 * C::TILE;
#pragma unroll
        for (int c = 0; c < CHUNKS; c += 2) {
          uint32_t r[4];
          ldmatrix4(tile_at(ktile, warp % 4 * K8D_SLAB + (lane & 15), c + (lane >> 4)), r);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t a0, a1, a2, a3;
            kv8_unpack4(r[2 * h], a0, a2);
            kv8_unpack4(r[2 * h + 1], a1, a3);
#pragma unroll
            for (int n8 = 0; n8 < NT; ++n8) mma_f16(sc[n8][h], a0, a1, a2, a3, qf[n8][c + h].x, qf[n8][c + h].y);
          }
        }
        const uint8_t* ex = s_exps + ks * C::EXPS + warp * K8D_SLAB + g;
        float kf[2], vb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t vbyte = ex[2 * KV8_PAGE + 8 * i];
          kf[i] = kv8_factor(ex[8 * i]);
          vb[i] = vbyte == KV8_E_NAN ? __uint_as_float(0x7fffffffu) : static_cast<float>(static_cast<int>(vbyte) - 127);
          vi[i] = kv8_two_to(max(-126, 127 - static_cast<int>(vbyte)));
        }
        const int key = key0 + warp * K8D_SLAB + g;
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float raw = (sc[n8][0][2 * i + k] + sc[n8][1][2 * i + k]) * qscale[n8][k];
              y[n8][i][k] = key + 8 * i <= last[n8][k] ? fmaf(raw, kf[i], vb[i]) : -INFINITY;
              grown |= y[n8][i][k] > m[n8][k] + K8D_LAZY;
            }
      }
      // ---- a column whose maximum grew far enough takes the block's, which all warps see alike
      const bool any = __syncthreads_or(grown);
      if (warp == K8D_WARPS - 1) issue(2 * n + 1 + SLOTS, j / 32 * 32 + 64);
      if (any) {
        if (ok && mine) {
#pragma unroll
          for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float mx = fmaxf(y[n8][0][k], y[n8][1][k]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              if (g == 0) s_max[warp][n8 * 8 + 2 * t + k] = mx;
            }
        }
        __syncthreads();
#pragma unroll
        for (int n8 = 0; n8 < NT; ++n8) {
          float top[2] = {-INFINITY, -INFINITY};
          for (int w = 0; w < slabs; ++w) {
            const float2 v = *reinterpret_cast<const float2*>(&s_max[w][n8 * 8 + 2 * t]);
            top[0] = fmaxf(top[0], v.x);
            top[1] = fmaxf(top[1], v.y);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (top[k] > m[n8][k] + K8D_LAZY) {
              const float f = ex2(m[n8][k] - top[k]);  // 0 at the first key
              m[n8][k] = top[k];
              l[n8][k] *= f;
#pragma unroll
              for (int i = 0; i < C::PER; ++i) { o[n8][i][k] *= f; o[n8][i][2 + k] *= f; }
            }
          }
        }
      }
      // ---- weights
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
          s_w[warp][n8][lane] = make_uint2(pw[0], pw[1]);
        }
      }
      ok = ok && mbar_wait_warp(&full[vs], ((2 * n + 1) / SLOTS) & 1, p.err, ERR_WAIT_FULL, abort_flag);
      __syncthreads();
      // ---- O[dim, column] += V^T P: dims 16 c + 2 g and + 1 of tile c are the rows g and g + 8
      if (ok) {
        // D = 256: the two tiles of a warp and one slab at a time; below: one tile and two slabs
        const uint32_t vslot = smem_u32(smem_k8 + vs * C::SLOT);
#pragma unroll
        for (int k = 0; k < SLABS / C::SPLIT; k += C::PER == 2 ? 1 : 2) {
          const int slab = part * (SLABS / C::SPLIT) + k;
          if (slab >= slabs) break;
          uint32_t r[4];
          const int row = C::PER == 2 ? lane & 15 : lane;  // lanes 16 .. 31: the second tile, or the second slab
          ldmatrix4_trans(tile_at(vslot + slab / 4 * C::TILE, slab % 4 * K8D_SLAB + row, C::PER == 2 ? tile0 + (lane >> 4) : tile0), r);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (C::PER == 1 && slab + h >= slabs) break;
            uint32_t a0, a1, a2, a3;
            kv8_unpack4(__byte_perm(r[2 * h], 0, 0x3120), a0, a1);
            kv8_unpack4(__byte_perm(r[2 * h + 1], 0, 0x3120), a2, a3);
#pragma unroll
            for (int n8 = 0; n8 < NT; ++n8) {
              const uint2 w = s_w[C::PER == 2 ? slab : slab + h][n8][lane];
              mma_f16(o[n8][C::PER == 2 ? h : 0], a0, a1, a2, a3, w.x, w.y);
            }
          }
        }
      }
    }

    // ---- the sums of all keys, in the warps' order; where warps share a tile, their outputs too
#pragma unroll
    for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float sum = l[n8][k];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) s_sum[warp][n8 * 8 + 2 * t + k] = sum;
      }
    if (C::SPLIT > 1 && part > 0) {
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_o[warp][n8 * 4 + i][lane] = o[n8][0][i];
    }
    __syncthreads();
    if (j % 32 == 31 && warp == 0) describe(j + 33 + lane);  // the half of the list that is done with
    if (part == 0) {
#pragma unroll
      for (int n8 = 0; n8 < NT; ++n8) {
        if (C::SPLIT > 1) {
#pragma unroll
          for (int w = 1; w < C::SPLIT; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n8][0][i] += s_o[w * C::TILES + warp][n8 * 4 + i][lane];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int col = n8 * 8 + 2 * t + k;
          if (col >= n_cols) continue;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < K8D_WARPS; ++w) sum += s_sum[w][col];
          int r, h;
          column(col, r, h);
          const size_t head = static_cast<size_t>(u.row0 + r) * p.n_q + u.kh * p.group + h;
          if (len[n8][k] > K8D_RUN) {
            if (u.z * K8D_RUN < len[n8][k]) {
              const size_t slot = head * p.n_splits + u.z;
              if (tile0 == 0 && g == 0) p.part_ml[slot] = make_float2(m[n8][k], sum);
#pragma unroll
              for (int i = 0; i < C::PER; ++i)
                *reinterpret_cast<float2*>(p.part_acc + slot * D + (tile0 + i) * 16 + 2 * g) = make_float2(o[n8][i][k], o[n8][i][2 + k]);
            }
          } else if (u.z == 0) {  // the row's only run
            const float inv = len[n8][k] > 0 ? 1.0f / sum : 0.f;
#pragma unroll
            for (int i = 0; i < C::PER; ++i) {
              const size_t at = head * D + (tile0 + i) * 16 + 2 * g;
              *reinterpret_cast<__nv_bfloat162*>(p.out + at) =
                  __floats2bfloat162_rn(o[n8][i][k] * inv * sigmoid_f(__bfloat162float(p.gate[at])),
                                        o[n8][i][2 + k] * inv * sigmoid_f(__bfloat162float(p.gate[at + 1])));
            }
          }
        }
      }
    }
  }
  if (warp == K8D_WARPS - 1 && *abort_flag) {  // a wait that ran out leaves loads on their way: they end before the shared memory goes
    for (int i = max(0, issued - SLOTS); i < issued; ++i) {
      const long long t0 = clock64();
      while (!mbar_try_wait(&full[i % SLOTS], (i / SLOTS) & 1) && clock64() - t0 < WAIT_CYCLES) {}
    }
  }
}

// Rows of more than one run: their partials in the order of the runs, four sums of every fourth partial each.
template <int D>
__global__ void __launch_bounds__(D)
kv8_combine_kernel(const float* part_acc, const float2* part_ml, const bf16* gate, const int64_t* positions, bf16* out, int n_q,
                   int n_splits, int most) {
  constexpr int QUADS = D / 4;
  __shared__ __align__(16) float s_acc[4][D];
  __shared__ float s_l[4];
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x;
  const int len = max(0, min(static_cast<int>(min(positions[row], static_cast<int64_t>(most))) + 1, most));
  if (len <= K8D_RUN) return;
  const int runs = (len + K8D_RUN - 1) / K8D_RUN;
  const size_t head = static_cast<size_t>(row) * n_q + blockIdx.y;
  const float2* ml = part_ml + head * n_splits;
  const int quad = threadIdx.x % QUADS, part = threadIdx.x / QUADS;
  float top = -INFINITY;
  for (int z = 0; z < runs; ++z) top = fmaxf(top, ml[z].x);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  const float4* pa = reinterpret_cast<const float4*>(part_acc + head * n_splits * D) + quad;
#pragma unroll 4
  for (int z = part; z < runs; z += 4) {
    const float2 pm = ml[z];
    const float4 v = pa[static_cast<size_t>(z) * QUADS];
    const float f = pm.x == -INFINITY ? 1.f : ex2(pm.x - top);  // without a maximum: scores that are all NaN, in the sum
    l = fmaf(pm.y, f, l);
    acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
  }
  *reinterpret_cast<float4*>(&s_acc[part][quad * 4]) = acc;
  if (quad == 0) s_l[part] = l;
  __syncthreads();
  const int d = threadIdx.x;
  const float sum = (s_l[0] + s_l[1]) + (s_l[2] + s_l[3]);
  const float o = (s_acc[0][d] + s_acc[1][d]) + (s_acc[2][d] + s_acc[3][d]);
  out[head * D + d] = __float2bfloat16(o / sum * sigmoid_f(__bfloat162float(gate[head * D + d])));
}

}  // namespace b200

using namespace b200;

namespace {
typedef CUresult (*K8dEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);
int k8d_make_map(CUtensorMap* m, const void* data, int D, long long rows) {
  static K8dEncodeFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || !ptr) return -1;
    fn = reinterpret_cast<K8dEncodeFn>(ptr);
  }
  const int rowb = D < 128 ? D : 128;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(rowb), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(D / rowb)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rowb)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(rowb), KV8_PAGE, static_cast<cuuint32_t>(D / rowb)}, estr[3] = {1, 1, 1};
  const CUtensorMapSwizzle sw = rowb == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : rowb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -2;
}

template <int D, int NT>
int k8d_launch(const CUtensorMap& tm, const Kv8DecodeParams& p, cudaStream_t st) {
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
  const int most_ctas = sms_of[dev] * Kv8DecodeCfg<D, NT>::CTAS;
  const int grid = static_cast<int>(units < most_ctas ? units : most_ctas);
  if (launch_pdl(kern, dim3(grid), dim3(32 * K8D_WARPS), Kv8DecodeCfg<D, NT>::SMEM, st, tm, p) != cudaSuccess) return -4;
  if (p.n_splits == 1) return 0;
  const int most = (p.width < p.n_splits * (K8D_RUN / KV8_PAGE) ? p.width : p.n_splits * (K8D_RUN / KV8_PAGE)) * KV8_PAGE;
  return launch_pdl(kv8_combine_kernel<D>, dim3(p.B * p.G, p.n_q), dim3(D), 0, st, p.part_acc, p.part_ml, p.gate, p.positions, p.out,
                    p.n_q, p.n_splits, most) == cudaSuccess ? 0 : -4;
}
}  // namespace

// Keys of a run: the caller sizes the partials by it.
extern "C" int b200_kv8_decode_run(void) { return K8D_RUN; }

// q: [B * G, n_q, D] bf16 (normed and rotated), G rows per sequence; gate, out: [B * G, n_q * D]; data, exps: one layer of the 8-bit cache, which
// holds the rows' own keys; positions [B * G] (negative: a row without keys, whose output is 0); tables [B] rows of `width` pages.
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
  CUtensorMap tm;
  if (k8d_make_map(&tm, data, D, rows)) return -1;
  const int cols = G * group, nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4, per = 8 * nt / group < G ? 8 * nt / group : G;
  for (int b0 = 0; b0 < B; b0 += K8D_MAX_SEQS) {
    const int n = B - b0 < K8D_MAX_SEQS ? B - b0 : K8D_MAX_SEQS;
    const size_t heads = static_cast<size_t>(b0) * G * n_q;
    const Kv8DecodeParams p{static_cast<const bf16*>(q) + heads * D, static_cast<const bf16*>(gate) + heads * D,
                            static_cast<const uint8_t*>(exps), positions + static_cast<size_t>(b0) * G,
                            tables + static_cast<size_t>(b0) * max_pages, static_cast<bf16*>(out) + heads * D,
                            part_acc + heads * n_splits * D, reinterpret_cast<float2*>(part_ml) + heads * n_splits,
                            n, G, max_pages, width, num_pages, n_q, n_kv, group, n_splits, per, (G + per - 1) / per, (65536 + group - 1) / group,
                            1.4426950408889634f / sqrtf(static_cast<float>(D)), err};
    int rc = -7;
#define K8D(DD) rc = nt == 1 ? k8d_launch<DD, 1>(tm, p, st) : nt == 2 ? k8d_launch<DD, 2>(tm, p, st) : k8d_launch<DD, 4>(tm, p, st)
    if (D == 256) K8D(256);
    else if (D == 128) K8D(128);
    else if (D == 64) K8D(64);
    else if (D == 32) K8D(32);
#undef K8D
    if (rc) return rc;
  }
  return 0;
}

// Attention of a few query rows per sequence (decode steps, verify passes) over the 8-bit paged cache.
//
//   s_j = q . (k_j 2^a_j) / sqrt D,   o = sum_j p_j (v_j 2^b_j) / sum_j p_j,   p_j = exp(s_j),   out = o * sigmoid(gate)
//
// with e4m3 rows k_j, v_j and their powers of two. Neither row is ever scaled: y_j = s_j log2(e) + b_j takes the value's power of
// two into the exponent, w_j = 2^(y_j - M) is the weight of the stored v_j, M the running maximum of y, and the softmax's own sum is
// sum_j w_j 2^-b_j. So what the matrix instructions get are the stored numbers as halves (exact) and weights below 2^15.
//
// Bound: the cache's bytes, 2 (D + 1) per token and KV head. A context is cut into runs of RUN keys at fixed places, so what a row's
// result is put together from depends on its own position only, never on the batch; a persistent CTA per SM takes runs in turn. In a run each
// of the eight warps takes every eighth slab of 16 keys, brought by TMA into a ring of the warp's own that it refills itself, the
// next runs' slabs included: no barrier stands between a warp and its data, and the finish of a run (the one place where the warps
// meet) has the next runs' loads on their way. The products are m16n8k16 with keys (S = K Q^T) or dims (O = V^T P) as the 16 rows and query
// columns as the 8: one token of one KV head's eight query heads fills the columns, where a tcgen05 tile would be 8 rows of 64.
// The stored bytes become halves in registers, behind ldmatrix.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace b200 {

constexpr int K8D_RUN = 512;                    // keys of a run: part of the numerics
constexpr int K8D_WARPS = 8;
constexpr int K8D_SLAB = 16;                    // keys of a slab
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
  float scale_log2;
  int* err;
};

template <int D>
struct Kv8DecodeCfg {
  static constexpr int ROWB = D < 128 ? D : 128;           // bytes of a row in one swizzled block
  static constexpr int DB = D / ROWB;
  static constexpr int TILE = K8D_SLAB * D;                // one of K or V
  static constexpr int STAGE = 2 * TILE;
  static constexpr int ST = D == 256 ? 3 : D == 128 ? 6 : 8;
  static constexpr int RING = K8D_WARPS * ST * STAGE;
  static constexpr int EXPS = K8D_WARPS * ST * 2 * K8D_SLAB;
  static constexpr int HALF = D < 64 ? D : 64;             // dims that the finish of a run exchanges at a time
  static constexpr int COL = HALF + 4;                     // floats between its columns: the pad spreads them over the banks
  static constexpr int EXCH = K8D_WARPS * 8 * COL * 4;
  static constexpr int BARS = K8D_WARPS * ST * 8;
  static constexpr int TABLE = (2 * K8D_MAX_SEQS + 4) * 4;
  static constexpr int SMEM = RING + EXCH + EXPS + BARS + 256;
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

// A unit is (sequence, group of its query rows, KV head, run). Walked by a warp: the slabs of the CTA's units, one after the other.
struct Kv8Walk {
  int id, b, rg, kh, z;
  int slab, slabs;     // this warp's next slab of the unit, the unit's slabs
  int page;            // lane i: the table's entry i of the run
};

template <int D, int NT>
__global__ void __launch_bounds__(32 * K8D_WARPS, 1)
kv8_decode_kernel(const __grid_constant__ CUtensorMap tm, Kv8DecodeParams p) {
  using C = Kv8DecodeCfg<D>;
  constexpr int ST = C::ST, CHUNKS = D / 16, COLS = 8 * NT;
  extern __shared__ __align__(1024) uint8_t smem_k8[];
  if (smem_u32(smem_k8) & 1023u) {  // the swizzled tiles need this alignment
    if (threadIdx.x == 0) atomicCAS(p.err, 0, ERR_BAD_INDEX);
    return;
  }
  float* exch = reinterpret_cast<float*>(smem_k8 + C::RING);
  uint8_t* s_exps = smem_k8 + C::RING + C::EXCH;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_exps + C::EXPS);
  __shared__ int s_first[K8D_MAX_SEQS + 1];   // runs of the sequences before
  __shared__ float s_m[K8D_WARPS][COLS], s_l[K8D_WARPS][COLS];
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem_k8 + warp * ST * C::STAGE;
  uint8_t* ring_exps = s_exps + warp * ST * 2 * K8D_SLAB;
  uint64_t* full = bars + warp * ST;
  if (threadIdx.x == 0) {
    for (int i = 0; i < K8D_WARPS * ST; ++i) mbar_init(&bars[i], 1);
    s_abort = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tm);
  }
  pdl_wait();
  pdl_launch();
  const int most = min(p.width, p.n_splits * (K8D_RUN / KV8_PAGE)) * KV8_PAGE;  // keys that the tables can name
  const auto length = [&](int row) { return max(0, min(static_cast<int>(min(p.positions[row], static_cast<int64_t>(most))) + 1, most)); };
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
  volatile int* abort_flag = &s_abort;

  const auto enter = [&](Kv8Walk& w) {  // the unit of w.id
    const int run = w.id / per_run, x = w.id % per_run;
    w.rg = x % p.units_per_seq;
    w.kh = x / p.units_per_seq;
    w.b = kv8_find(s_first, p.B, run);
    w.z = run - s_first[w.b];
    int len = 0;
    const int r0 = w.b * p.G + w.rg * p.rows_per_unit, r1 = min(r0 + p.rows_per_unit, (w.b + 1) * p.G);
    for (int r = r0; r < r1; ++r) len = max(len, length(r));
    w.slabs = (max(0, min(K8D_RUN, len - w.z * K8D_RUN)) + K8D_SLAB - 1) / K8D_SLAB;
    w.slab = warp;
  };
  const auto pages = [&](Kv8Walk& w) {
    w.page = 0;
    const int n = (w.slabs + KV8_PAGE / K8D_SLAB - 1) / (KV8_PAGE / K8D_SLAB);
    if (lane < n) w.page = p.tables[static_cast<size_t>(w.b) * p.max_pages + w.z * (K8D_RUN / KV8_PAGE) + lane];
    if (w.page < 0 || w.page >= p.num_pages) { atomicCAS(p.err, 0, ERR_BAD_INDEX); w.page = 0; }
  };
  // The loads run ahead of the work by the ring's stages, into the next units.
  Kv8Walk ahead;
  ahead.id = blockIdx.x;
  const auto seek = [&]() {  // the first unit from ahead.id on that has a slab for this warp
    for (; ahead.id < total; ahead.id += gridDim.x) {
      enter(ahead);
      if (ahead.slab < ahead.slabs) { pages(ahead); return; }
    }
  };
  int issued = 0;
  const auto issue = [&]() {
    if (ahead.id >= total) return;
    const int page = __shfl_sync(0xffffffffu, ahead.page, ahead.slab / (KV8_PAGE / K8D_SLAB));
    if (lane == 0) {
      const int s = issued % ST;
      const int row = (page * 2 * p.n_kv + ahead.kh) * KV8_PAGE + ahead.slab % (KV8_PAGE / K8D_SLAB) * K8D_SLAB;
      const int vrow = row + p.n_kv * KV8_PAGE;
      mbar_expect_tx(&full[s], C::STAGE + 2 * K8D_SLAB);
      uint8_t* at = ring + s * C::STAGE;
      tma_load_3d(at, &tm, &full[s], 0, row, 0);
      tma_load_3d(at + C::TILE, &tm, &full[s], 0, vrow, 0);
      bulk_load(ring_exps + s * 2 * K8D_SLAB, p.exps + row, K8D_SLAB, &full[s]);
      bulk_load(ring_exps + s * 2 * K8D_SLAB + K8D_SLAB, p.exps + vrow, K8D_SLAB, &full[s]);
    }
    ++issued;
    ahead.slab += K8D_WARPS;
    if (ahead.slab >= ahead.slabs) { ahead.id += gridDim.x; seek(); }
  };
  seek();
  for (int i = 0; i < ST; ++i) issue();

  int used = 0;  // slabs consumed
  bool ok = true;
  // shared-memory offset of 16 bytes of a swizzled tile: row r, chunk c
  const auto tile_at = [&](uint32_t tile, int r, int c) {
    constexpr int PER = C::ROWB / 16;  // chunks of a block's row
    const int byte = r * C::ROWB;
    return tile + (c / PER) * (K8D_SLAB * C::ROWB) + byte + (((c % PER) ^ ((byte >> 7) & (PER - 1))) << 4);
  };

  for (int id = blockIdx.x; id < total; id += gridDim.x) {
    Kv8Walk u;
    u.id = id;
    enter(u);
    const int row0 = u.b * p.G + u.rg * p.rows_per_unit;
    const int n_rows = min(p.rows_per_unit, (u.b + 1) * p.G - row0), n_cols = n_rows * p.group;
    // ---- queries: thread (g, t) holds dims 16 c + 4 t .. + 3 of column g, as halves with the column's largest number in [2^10, 2^11)
    uint32_t qf[NT][CHUNKS][2];
    float qscale[NT][2];   // columns 2 t, 2 t + 1: what takes the product to log-2 scores
    int last[NT][2];       // ... position of the last visible key
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int col = n * 8 + g;
      const bool real = col < n_cols;
      const bf16* src = p.q + (static_cast<size_t>(row0 + (real ? col / p.group : 0)) * p.n_q + u.kh * p.group + (real ? col % p.group : 0)) * D + t * 4;
      uint2 raw[CHUNKS];
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) raw[c] = *reinterpret_cast<const uint2*>(src + c * 16);
      float top = 0.f;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw[c]);
        const float2 a = __bfloat1622float2(e[0]), b = __bfloat1622float2(e[1]);
        top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
        bad |= !(fabsf(a.x) <= 3.5e38f && fabsf(a.y) <= 3.5e38f && fabsf(b.x) <= 3.5e38f && fabsf(b.y) <= 3.5e38f);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max(-110, min(110, static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10));
      const float f = kv8_two_to(-e);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&raw[c]);
        const float2 a = __bfloat1622float2(x[0]), b = __bfloat1622float2(x[1]);
        const __half2 lo = __floats2half2_rn(a.x * f, a.y * f), hi = __floats2half2_rn(b.x * f, b.y * f);
        qf[n][c][0] = *reinterpret_cast<const uint32_t*>(&lo);
        qf[n][c][1] = *reinterpret_cast<const uint32_t*>(&hi);
      }
      // a NaN or an infinity anywhere in the column: all its scores are NaN
      const uint32_t bads = __ballot_sync(0xffffffffu, bad);
      const float mine = (bads >> (lane & 28)) & 15u ? __uint_as_float(0x7fffffffu) : kv8_two_to(e) * p.scale_log2;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int c = n * 8 + 2 * t + j;
        qscale[n][j] = __shfl_sync(0xffffffffu, mine, (2 * t + j) * 4);
        last[n][j] = c < n_cols ? length(row0 + c / p.group) - 1 : -1;
      }
    }
    float o[NT][CHUNKS][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

    for (int slab = u.slab; slab < u.slabs; slab += K8D_WARPS, ++used) {
      const int s = used % ST;
      ok = ok && mbar_wait_warp(&full[s], (used / ST) & 1, p.err, ERR_WAIT_FULL, abort_flag);
      if (!ok) break;
      const uint32_t ktile = smem_u32(ring + s * C::STAGE), vtile = ktile + C::TILE;
      // ---- scores: S[key, column], keys g and g + 8 of the slab
      float sc[NT][2][4];  // two chains of products
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[n][0][j] = sc[n][1][j] = 0.f;
#pragma unroll
      for (int c = 0; c < CHUNKS; c += 2) {
        uint32_t r[4];
        ldmatrix4(tile_at(ktile, lane & 15, c + (lane >> 4)), r);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a0, a1, a2, a3;
          kv8_unpack4(r[2 * h], a0, a2);
          kv8_unpack4(r[2 * h + 1], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(sc[n][h], a0, a1, a2, a3, qf[n][c + h][0], qf[n][c + h][1]);
        }
      }
      const uint8_t* ex = ring_exps + s * 2 * K8D_SLAB;
      float kf[2], vb[2], vi[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t vbyte = ex[K8D_SLAB + g + 8 * i];
        kf[i] = kv8_factor(ex[g + 8 * i]);
        vb[i] = vbyte == KV8_E_NAN ? __uint_as_float(0x7fffffffu) : static_cast<float>(static_cast<int>(vbyte) - 127);
        vi[i] = kv8_two_to(max(-126, 127 - static_cast<int>(vbyte)));
      }
      const int key = u.z * K8D_RUN + slab * K8D_SLAB + g;
      uint32_t pw[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float y[2][2];  // [key g, g + 8][column 2 t, 2 t + 1]
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float raw = (sc[n][0][2 * i + j] + sc[n][1][2 * i + j]) * qscale[n][j];
            y[i][j] = key + 8 * i <= last[n][j] ? fmaf(raw, kf[i], vb[i]) : -INFINITY;
          }
        float w[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(y[0][j], y[1][j]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          float f = 1.f;
          if (mx > m[n][j] + K8D_LAZY) {
            f = ex2(m[n][j] - mx);  // 0 at the first key
            m[n][j] = mx;
            l[n][j] *= f;
          }
          const float base = m[n][j] == -INFINITY ? 0.f : m[n][j] - K8D_LIFT;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            w[i][j] = ex2(y[i][j] - base);
            l[n][j] = fmaf(w[i][j], vi[i], l[n][j]);
          }
          if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) { o[n][c][j] *= f; o[n][c][2 + j] *= f; }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const __half2 two = __floats2half2_rn(w[i][0], w[i][1]);
          pw[n][i] = movmatrix(*reinterpret_cast<const uint32_t*>(&two));  // [column g][keys 2 t, 2 t + 1]
        }
      }
      // ---- O[dim, column] += V^T P: dims 16 c + 2 g and + 1 are the rows g and g + 8
#pragma unroll
      for (int c = 0; c < CHUNKS; c += 2) {
        uint32_t r[4];
        ldmatrix4_trans(tile_at(vtile, lane & 15, c + (lane >> 4)), r);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a0, a1, a2, a3;
          kv8_unpack4(__byte_perm(r[2 * h], 0, 0x3120), a0, a1);
          kv8_unpack4(__byte_perm(r[2 * h + 1], 0, 0x3120), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(o[n][c + h], a0, a1, a2, a3, pw[n][0], pw[n][1]);
        }
      }
      __syncwarp();  // every lane has read the stage
      issue();
    }

    // ---- the warps' parts, in the warps' order
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[n][j];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) { s_m[warp][n * 8 + 2 * t + j] = m[n][j]; s_l[warp][n * 8 + 2 * t + j] = sum; }
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < K8D_WARPS; ++w) top = fmaxf(top, s_m[w][n * 8 + 2 * t + j]);
        f[j] = m[n][j] == -INFINITY ? 0.f : ex2(m[n][j] - top);
      }
#pragma unroll
      for (int h = 0; h < D / C::HALF; ++h) {
#pragma unroll
        for (int c = 0; c < C::HALF / 16; ++c)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float* v = o[n][h * (C::HALF / 16) + c];
            *reinterpret_cast<float2*>(exch + (warp * 8 + 2 * t + j) * C::COL + 16 * c + 2 * g) =
                make_float2(v[j] * f[j], v[2 + j] * f[j]);
          }
        __syncthreads();
        constexpr int QUADS = C::HALF / 4;  // threads per column, four numbers each
        for (int i = threadIdx.x; i < 8 * QUADS; i += 32 * K8D_WARPS) {
          const int col8 = i / QUADS, d = i % QUADS * 4, col = n * 8 + col8;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int w = 0; w < K8D_WARPS; ++w) top = fmaxf(top, s_m[w][col]);
#pragma unroll
          for (int w = 0; w < K8D_WARPS; ++w) {
            const float4 v = *reinterpret_cast<const float4*>(exch + (w * 8 + col8) * C::COL + d);
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
            const float mw = s_m[w][col];
            sum += mw == -INFINITY ? s_l[w][col] : s_l[w][col] * ex2(mw - top);  // a NaN among the scores leaves the maximum and marks the sum
          }
          if (col < n_cols) {
            const int row = row0 + col / p.group, len = length(row);
            const size_t head = static_cast<size_t>(row) * p.n_q + u.kh * p.group + col % p.group;
            const int at = h * C::HALF + d;
            if (len <= K8D_RUN) {
              if (u.z == 0) {  // the row's only run
                const float inv = len > 0 ? 1.0f / sum : 0.f;
                const float* e = reinterpret_cast<const float*>(&a);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  p.out[head * D + at + k] = __float2bfloat16(e[k] * inv * sigmoid_f(__bfloat162float(p.gate[head * D + at + k])));
              }
            } else if (u.z * K8D_RUN < len) {
              const size_t slot = head * p.n_splits + u.z;
              *reinterpret_cast<float4*>(p.part_acc + slot * D + at) = a;
              if (at == 0) p.part_ml[slot] = make_float2(top, sum);
            }
          }
        }
        __syncthreads();
      }
    }
  }
  // a wait that ran out leaves loads on their way: they end before the CTA's shared memory goes
  if (!ok) {
    for (; used < issued; ++used) {
      const long long t0 = clock64();
      while (!mbar_try_wait(&full[used % ST], (used / ST) & 1) && clock64() - t0 < WAIT_CYCLES) {}
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
  cuuint32_t box[3] = {static_cast<cuuint32_t>(rowb), K8D_SLAB, static_cast<cuuint32_t>(D / rowb)}, estr[3] = {1, 1, 1};
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
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv8DecodeCfg<D>::SMEM) != cudaSuccess) return -3;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
    sms_of[dev] = sms;
  }
  const long long units = static_cast<long long>(p.B) * p.units_per_seq * p.n_kv * p.n_splits;
  const int grid = static_cast<int>(units < sms_of[dev] ? units : sms_of[dev]);
  if (launch_pdl(kern, dim3(grid), dim3(32 * K8D_WARPS), Kv8DecodeCfg<D>::SMEM, st, tm, p) != cudaSuccess) return -4;
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
  const int nt = G * group <= 8 ? 1 : 2, per = 8 * nt / group < G ? 8 * nt / group : G;
  for (int b0 = 0; b0 < B; b0 += K8D_MAX_SEQS) {
    const int n = B - b0 < K8D_MAX_SEQS ? B - b0 : K8D_MAX_SEQS;
    const size_t heads = static_cast<size_t>(b0) * G * n_q;
    const Kv8DecodeParams p{static_cast<const bf16*>(q) + heads * D, static_cast<const bf16*>(gate) + heads * D,
                            static_cast<const uint8_t*>(exps), positions + static_cast<size_t>(b0) * G,
                            tables + static_cast<size_t>(b0) * max_pages, static_cast<bf16*>(out) + heads * D,
                            part_acc + heads * n_splits * D, reinterpret_cast<float2*>(part_ml) + heads * n_splits,
                            n, G, max_pages, width, num_pages, n_q, n_kv, group, n_splits, per, (G + per - 1) / per,
                            1.4426950408889634f / sqrtf(static_cast<float>(D)), err};
    int rc = -7;
#define K8D(DD) rc = nt == 1 ? k8d_launch<DD, 1>(tm, p, st) : k8d_launch<DD, 2>(tm, p, st)
    if (D == 256) K8D(256);
    else if (D == 128) K8D(128);
    else if (D == 64) K8D(64);
    else if (D == 32) K8D(32);
#undef K8D
    if (rc) return rc;
  }
  return 0;
}

// Low-rank adapters of many requests beside a projection that all rows share:
//
//   y[t, n] = sum_k x[t, k] W[n, k] + sum_r h[t, r] b_a[n, r],   h[t, r] = s_a sum_k x[t, k] a_a[r, k],   a the adapter of row t (below 0: none)
//
// This file makes h; the GEMM goes on over it (lora.cuh).
//
// A CTA takes 16 token rows (64 where the CTAs of 16 would be more than two for each SM) and the adapters among them one after the other, or every
// gridDim.y-th one: in a decode step each row may have its own. Its eight warps share K in pieces of 32, join their sums in a fixed order, and round h to
// bf16, as x itself is rounded: 2^-9 of each h, a part of y's own rounding. Rows of other adapters take part in the product and are not stored. All of
// it goes by the row alone, so its bits do not depend on the batch.
//
// The products are 16 x 8 x 16 instructions fed from global memory, in an order that is the same for one row and for 8,192. In a decode step the latency
// of those reads bounds it, so a warp asks for a whole batch of pieces at a time (64 ranks, K of 4096: 78 us piece by piece, 22 in batches); with 256
// threads and less than 13 KB of shared memory a CTA runs beside the GEMM's, which needs h behind its own k-blocks: the whole call takes 12.7 us for one row
// of 9216 x 2048 where the projection alone takes 11.0, 22.2 and 11.6 for 128 rows of 32 adapters. In a long pass the rate of these instructions bounds
// it (about 144 TFLOP/s for its share of the tiles; 8,192 rows, K of 2048: 28 us at 16 ranks, 35 at 64; of the 28, 23 show beside the GEMM's 197).
#include "lora.cuh"

namespace b200 {

constexpr int SHRINK_WARPS = 8, SHRINK_THREADS = 32 * SHRINK_WARPS;
constexpr int SHRINK_JOIN = 4;  // groups of eight ranks that are joined at a time, through 8 KB

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Sixteen bytes that stay in the order in which they are asked for: left to itself, the compiler puts each load in front of the product that uses it.
__device__ __forceinline__ uint4 ask_16(const bf16* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// NT: groups of eight ranks, of which blockIdx.z says the first; MT: groups of sixteen rows.
template <int NT, int MT>
__global__ void __launch_bounds__(SHRINK_THREADS) lora_shrink_kernel(const bf16* x, int ldx, const bf16* a, const float* scale, const int* rows, int T, int K,
                                                                     int R, int L, LoraTiles tiles, int* err) {
  constexpr int ROWS = 16 * MT;
  constexpr int BATCH = MT == 1 ? 4 : NT == 2 ? 2 : 1;  // pieces of 32 that a warp asks for at a time
  constexpr int JOIN = NT < SHRINK_JOIN ? NT : SHRINK_JOIN;
  __shared__ __align__(16) float red[SHRINK_WARPS / 2 * JOIN * 32 * 4];
  __shared__ uint32_t used[LORA_MAX_ADAPTERS / 32], before[LORA_MAX_ADAPTERS / 32];  // adapters of the token tile; how many below each word
  __shared__ int mine[64];  // adapter of each of the CTA's rows
  __shared__ uint32_t leads[2];  // the rows that are the first with their adapter
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r0 = blockIdx.x * ROWS, tile = r0 / tiles.tile_rows, tile0 = tile * tiles.tile_rows;
  if (tid < LORA_MAX_ADAPTERS / 32) used[tid] = 0;
  if (tid < 64) mine[tid] = -1;
  pdl_wait();
  pdl_launch();
  __syncthreads();
  for (int t = tile0 + tid; t < min(T, tile0 + tiles.tile_rows); t += SHRINK_THREADS) {
    const int id = rows[t];
    if (id >= 0 && id < L) {
      atomicOr(&used[id >> 5], 1u << (id & 31));
      if (t >= r0 && t < r0 + ROWS) mine[t - r0] = id;
    }
    if (id >= L) atomicCAS(err, 0, ERR_BAD_INDEX);
  }
  __syncthreads();
  static_assert(LORA_MAX_ADAPTERS / 32 == 32, "a word for each lane");
  if (warp == 0) {
    const uint32_t word = used[lane];
    int up = __popc(word);
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    before[lane] = up - __popc(word);
    if (blockIdx.y == 0 && blockIdx.z == 0 && r0 == tile0) {
      if (lane == 31) tiles.count[tile] = up;
      int at = tile * tiles.cap + up - __popc(word);
      for (uint32_t w = word; w; w &= w - 1) tiles.list[at++] = lane * 32 + __ffs(w) - 1;
    }
  } else if (warp == 1) {
    const int low = mine[lane], high = mine[32 + lane];
    const uint32_t same = __match_any_sync(0xffffffffu, low), above = __match_any_sync(0xffffffffu, high);
    bool again = false;
    if (MT > 2)
      for (int i = 0; i < 32; ++i) again |= __shfl_sync(0xffffffffu, low, i) == high;
    const uint32_t first = __ballot_sync(0xffffffffu, low >= 0 && __ffs(same) - 1 == lane);
    const uint32_t then = __ballot_sync(0xffffffffu, high >= 0 && !again && __ffs(above) - 1 == lane);
    if (lane == 0) { leads[0] = first; leads[1] = then; }
  }
  __syncthreads();
  const auto index = [&](int id) { return static_cast<int>(before[id >> 5]) + __popc(used[id >> 5] & ((1u << (id & 31)) - 1)); };
  const int count = static_cast<int>(before[31]) + __popc(used[31]);
  // where entry e of the tile has row r0 + i
  const auto place = [&](int e, int i) {
    return tiles.h + ((static_cast<size_t>(tile) * tiles.cap * tiles.chunks + e) * tiles.tile_rows + (r0 - tile0) + i) * tiles.width;
  };
  if (blockIdx.y == 0 && blockIdx.z == 0) {  // zeros in the rows of an entry that have another adapter, or none
    const int pieces = tiles.width / 8, per_row = count * tiles.chunks * pieces;
    for (int row = warp; row < min(ROWS, T - r0); row += SHRINK_WARPS) {
      const int own = mine[row] < 0 ? -1 : index(mine[row]);
      for (int i = lane; i < per_row; i += 32) {
        const int e = i / pieces;
        if (e / tiles.chunks != own) *reinterpret_cast<uint4*>(place(e, row) + i % pieces * 8) = make_uint4(0, 0, 0, 0);
      }
    }
  }

  const int g = lane >> 2, q = lane & 3;
  const bf16* xr[2 * MT];  // (rows behind the last are the last one again, and are not stored)
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) xr[i] = x + static_cast<long long>(min(r0 + g + 8 * i, T - 1)) * ldx + q * 8;
  const int n_first = blockIdx.z * NT;
  int turn = 0;
  for (uint64_t left = leads[0] | static_cast<uint64_t>(leads[1]) << 32; left; left &= left - 1) {  // (the same for all threads)
    const int id = mine[__ffsll(left) - 1];
    if (turn++ % gridDim.y != blockIdx.y) continue;
    float acc[MT][NT][4] = {};
    const bf16* a0 = a + static_cast<size_t>(id) * R * K + q * 8;
    for (int k0 = warp * 32; k0 < K; k0 += BATCH * SHRINK_WARPS * 32) {
      // Lane q of a row holds eight numbers of it: four pairs, of which two instructions take two each. Which k a pair stands for does not matter, as
      // it is the same one in x and in A. All of a batch is asked for before any of it is used; behind the end of K, x counts as 0.
      uint4 u[BATCH][2 * MT], w[BATCH][NT];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int k = k0 + b * SHRINK_WARPS * 32, at = k + q * 8 < K ? k : -q * 8;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) u[b][i] = ask_16(xr[i] + at);
#pragma unroll
        for (int n = 0; n < NT; ++n) w[b][n] = ask_16(a0 + static_cast<size_t>(min((n_first + n) * 8 + g, R - 1)) * K + at);
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const bool in = k0 + b * SHRINK_WARPS * 32 + q * 8 < K;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4 none = make_uint4(0, 0, 0, 0), up = in ? u[b][2 * m] : none, low = in ? u[b][2 * m + 1] : none;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(acc[m][n], up.x, low.x, up.y, low.y, w[b][n].x, w[b][n].y);
            mma_16816(acc[m][n], up.z, low.z, up.w, low.w, w[b][n].z, w[b][n].w);
          }
        }
      }
    }
    const float s = scale[id];
    const int e0 = index(id) * tiles.chunks;
    // the warps' sums: 4 to 7 onto 0 to 3, 2 and 3 onto 0 and 1, 1 onto 0
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n0 = 0; n0 < NT; n0 += JOIN) {
#pragma unroll
        for (int half = SHRINK_WARPS / 2; half; half >>= 1) {
          if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int n = 0; n < JOIN; ++n) {
              const float* v = acc[m][n0 + n];
              *reinterpret_cast<float4*>(red + (((warp - half) * JOIN + n) * 32 + lane) * 4) = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
          __syncthreads();
          if (warp < half) {
#pragma unroll
            for (int n = 0; n < JOIN; ++n) {
              const float4 o = *reinterpret_cast<const float4*>(red + ((warp * JOIN + n) * 32 + lane) * 4);
              float* v = acc[m][n0 + n];
              v[0] += o.x; v[1] += o.y; v[2] += o.z; v[3] += o.w;
            }
          }
          __syncthreads();
        }
        if (warp != 0) continue;
#pragma unroll
        for (int n = n0; n < n0 + JOIN; ++n)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int row = 16 * m + g + 8 * half, col = (n_first + n) * 8 + 2 * q;
            if (mine[row] != id || col >= tiles.width * (tiles.chunks / tiles.parts)) continue;
            // (R is even; columns behind it are 0)
            const float h0 = col < R ? acc[m][n][2 * half] * s : 0.f, h1 = col < R ? acc[m][n][2 * half + 1] * s : 0.f;
            const int e = e0 + col / 64 * tiles.parts;
            const __nv_bfloat162 hi = __floats2bfloat162_rn(h0, h1);
            *reinterpret_cast<__nv_bfloat162*>(place(e, row) + col % 64) = hi;
            if (tiles.parts > 1) {  // (written out: as a loop over the parts it cost bf16 outputs 2 to 5 us)
              const float m0 = h0 - __low2float(hi), m1 = h1 - __high2float(hi);
              const __nv_bfloat162 mid = __floats2bfloat162_rn(m0, m1);
              *reinterpret_cast<__nv_bfloat162*>(place(e + 1, row) + col % 64) = mid;
              *reinterpret_cast<__nv_bfloat162*>(place(e + 2, row) + col % 64) = __floats2bfloat162_rn(m0 - __low2float(mid), m1 - __high2float(mid));
            }
          }
      }
  }
}

template <int NT, int MT>
static int launch_shrink(const void* x, int ldx, const void* a, const float* scale, const int* rows, int T, int K, int R, int L, const LoraTiles& t, int* err,
                         cudaStream_t st) {
  const int blocks = (T + 16 * MT - 1) / (16 * MT), columns = t.width * (t.chunks / t.parts);
  // CTAs for the adapters of 16 rows: as many as there may be while the rows are few, one when they fill the SMs
  const int side = blocks >= 64 ? 1 : min(min(16 * MT, T), L);
  // An SM that runs this kernel gives its memory to shared memory as the GEMM needs it: otherwise no CTA of that one can join before the SM is empty
  // (128 rows of 9216 x 2048, one adapter: 21.0 -> 15.7 us).
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!configured[dev] && cudaFuncSetAttribute(lora_shrink_kernel<NT, MT>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                               cudaSharedmemCarveoutMaxShared) != cudaSuccess) return -3;
  configured[dev] = true;
  return launch_pdl(lora_shrink_kernel<NT, MT>, dim3(blocks, side, (columns + 8 * NT - 1) / (8 * NT)), dim3(SHRINK_THREADS), 0, st,
                    static_cast<const bf16*>(x), ldx, static_cast<const bf16*>(a), scale, rows, T, K, R, L, t, err) == cudaSuccess ? 0 : -4;
}

int lora_shrink(const void* x, int ldx, const void* a, const float* scale, const int* rows, int T, int K, int R, int L, const LoraTiles& t, int* err,
                cudaStream_t st) {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
  const bool many = (T + 15) / 16 * ((R + 15) / 16) > 2 * sms[dev] && t.tile_rows % 64 == 0;
  if (!many) return launch_shrink<2, 1>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
  if (R <= 16) return launch_shrink<2, 4>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
  return launch_shrink<4, 4>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
}

}  // namespace b200

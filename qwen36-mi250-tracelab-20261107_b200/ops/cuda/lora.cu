// Low-rank adapters of many requests beside a projection that all rows share:
//
//   y[t, n] = sum_k x[t, k] W[n, k] + sum_r h[t, r] b_a[n, r],   h[t, r] = s_a sum_k x[t, k] a_a[r, k],   a the adapter of row t (below 0: none)
//
// This file makes h; the GEMM goes on over it (lora.cuh).
//
// A CTA takes 16 token rows and the adapters among them one after the other (or every gridDim.y-th one: in a decode step each row may have its own). Its
// eight warps share K in pieces of 32, join their sums in a fixed order, and round h to bf16. Rows of other adapters take part in the product and
// are not stored. All of it goes by the row alone, so its bits do not depend on the batch.
//
// The products are 16 x 8 x 16 instructions fed from global memory: A and x are read once, at 2 R flops for each number of x, far below what tensor
// memory would be needed for. Bound by those reads (64 KB of A for an adapter of 16 x 2048).
#include "lora.cuh"

namespace b200 {

constexpr int SHRINK_ROWS = 16, SHRINK_WARPS = 8, SHRINK_THREADS = 32 * SHRINK_WARPS;

__device__ __forceinline__ void mma_16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of eight ranks.
template <int NT>
__global__ void __launch_bounds__(SHRINK_THREADS) lora_shrink_kernel(const bf16* x, int ldx, const bf16* a, const float* scale, const int* rows, int T, int K,
                                                                     int R, int L, LoraTiles tiles, int* err) {
  extern __shared__ __align__(16) float red[];  // [4][16][8 NT]
  __shared__ uint32_t used[LORA_MAX_ADAPTERS / 32], before[LORA_MAX_ADAPTERS / 32];  // adapters of the token tile; how many below each word
  __shared__ int mine[SHRINK_ROWS];  // adapter of each of the CTA's rows
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r0 = blockIdx.x * SHRINK_ROWS, tile = r0 / tiles.tile_rows, tile0 = tile * tiles.tile_rows;
  if (tid < LORA_MAX_ADAPTERS / 32) used[tid] = 0;
  pdl_wait();
  pdl_launch();
  __syncthreads();
  for (int t = tile0 + tid; t < min(T, tile0 + tiles.tile_rows); t += SHRINK_THREADS) {
    const int id = rows[t];
    if (id >= 0 && id < L) atomicOr(&used[id >> 5], 1u << (id & 31));
    if (id >= L) atomicCAS(err, 0, ERR_BAD_INDEX);
    if (t >= r0 && t < r0 + SHRINK_ROWS) mine[t - r0] = id < L ? id : -1;
  }
  if (tid < SHRINK_ROWS && r0 + tid >= T) mine[tid] = -1;
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
    if (blockIdx.y == 0 && r0 == tile0) {
      if (lane == 31) tiles.count[tile] = up;
      int at = tile * tiles.cap + up - __popc(word);
      for (uint32_t w = word; w; w &= w - 1) tiles.list[at++] = lane * 32 + __ffs(w) - 1;
    }
  }
  __syncthreads();
  const auto index = [&](int id) { return static_cast<int>(before[id >> 5]) + __popc(used[id >> 5] & ((1u << (id & 31)) - 1)); };
  const int count = static_cast<int>(before[31]) + __popc(used[31]);
  // where entry e of the tile has row r0 + i
  const auto place = [&](int e, int i) {
    return tiles.h + ((static_cast<size_t>(tile) * tiles.cap * tiles.chunks + e) * tiles.tile_rows + (r0 - tile0) + i) * tiles.width;
  };
  if (blockIdx.y == 0) {  // zeros in the rows of an entry that have another adapter, or none
    const int pieces = tiles.width / 8;
    for (int i = tid; i < count * tiles.chunks * SHRINK_ROWS * pieces; i += SHRINK_THREADS) {
      const int piece = i % pieces, row = i / pieces % SHRINK_ROWS, e = i / pieces / SHRINK_ROWS;
      if (r0 + row < T && (mine[row] < 0 || index(mine[row]) != e / tiles.chunks))
        *reinterpret_cast<uint4*>(place(e, row) + piece * 8) = make_uint4(0, 0, 0, 0);
    }
  }

  const int g = lane >> 2, q = lane & 3;
  const bf16* x0 = x + static_cast<long long>(r0 + g) * ldx + q * 8;
  const bf16* x1 = x0 + 8LL * ldx;
  const bool in0 = r0 + g < T, in1 = r0 + g + 8 < T;
  int turn = 0;  // of the distinct adapters among the rows
  for (int lead = 0; lead < SHRINK_ROWS; ++lead) {
    const int id = mine[lead];
    bool again = id < 0;
    for (int i = 0; i < lead; ++i) again |= mine[i] == id;
    if (again || turn++ % gridDim.y != blockIdx.y) continue;  // (the same for all threads)
    float acc[NT][4] = {};
    const bf16* a0 = a + static_cast<size_t>(id) * R * K + q * 8;
    for (int k = warp * 32; k < K; k += SHRINK_WARPS * 32) {
      // lane q of a row holds eight numbers of it: four pairs, of which two instructions take two each. Which k a pair stands for does not matter, as
      // it is the same one in x and in A.
      const bool in = k + q * 8 < K;
      const uint4 none = make_uint4(0, 0, 0, 0);
      const uint4 u = in && in0 ? __ldg(reinterpret_cast<const uint4*>(x0 + k)) : none;
      const uint4 v = in && in1 ? __ldg(reinterpret_cast<const uint4*>(x1 + k)) : none;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = n * 8 + g;
        const uint4 w = in && r < R ? __ldg(reinterpret_cast<const uint4*>(a0 + static_cast<size_t>(r) * K + k)) : none;
        mma_16816(acc[n], u.x, v.x, u.y, v.y, w.x, w.y);
        mma_16816(acc[n], u.z, v.z, u.w, v.w, w.z, w.w);
      }
    }
    // the warps' sums: 4 to 7 onto 0 to 3, 2 and 3 onto 0 and 1, 1 onto 0
#pragma unroll
    for (int half = SHRINK_WARPS / 2; half; half >>= 1) {
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<float4*>(red + (((warp - half) * NT + n) * 32 + lane) * 4) = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 o = *reinterpret_cast<const float4*>(red + ((warp * NT + n) * 32 + lane) * 4);
          acc[n][0] += o.x; acc[n][1] += o.y; acc[n][2] += o.z; acc[n][3] += o.w;
        }
      }
      __syncthreads();
    }
    if (warp == 0) {
      const float s = scale[id];
      const int e0 = index(id) * tiles.chunks;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = g + 8 * half, col = n * 8 + 2 * q;
          if (mine[row] != id) continue;
          const float h0 = acc[n][2 * half] * s, h1 = acc[n][2 * half + 1] * s;
          __nv_bfloat162 hi = __floats2bfloat162_rn(h0, h1);
          const int e = e0 + col / 64 * tiles.parts;
          *reinterpret_cast<__nv_bfloat162*>(place(e, row) + col % 64) = hi;
          if (tiles.parts == 2)
            *reinterpret_cast<__nv_bfloat162*>(place(e + 1, row) + col % 64) =
                __floats2bfloat162_rn(h0 - __low2float(hi), h1 - __high2float(hi));
        }
    }
  }
}

// Every column of an entry is written: NT covers its whole width (A's rows behind R count as zeros).
template <int NT>
static int launch_shrink(const void* x, int ldx, const void* a, const float* scale, const int* rows, int T, int K, int R, int L, const LoraTiles& t, int* err,
                         cudaStream_t st) {
  const int blocks = (T + SHRINK_ROWS - 1) / SHRINK_ROWS;
  // CTAs for the adapters of 16 rows: as many as there may be while the rows are few, one when they fill the SMs
  const int side = blocks >= 64 ? 1 : min(min(SHRINK_ROWS, T), L);
  return launch_pdl(lora_shrink_kernel<NT>, dim3(blocks, side), dim3(SHRINK_THREADS), 4 * 16 * 8 * NT * sizeof(float), st, static_cast<const bf16*>(x), ldx,
                    static_cast<const bf16*>(a), scale, rows, T, K, R, L, t, err) == cudaSuccess ? 0 : -4;
}

int lora_shrink(const void* x, int ldx, const void* a, const float* scale, const int* rows, int T, int K, int R, int L, const LoraTiles& t, int* err,
                cudaStream_t st) {
  if (R <= 16) return launch_shrink<2>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
  if (R <= 32) return launch_shrink<4>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
  if (R <= 64) return launch_shrink<8>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
  return launch_shrink<16>(x, ldx, a, scale, rows, T, K, R, L, t, err, st);
}

}  // namespace b200

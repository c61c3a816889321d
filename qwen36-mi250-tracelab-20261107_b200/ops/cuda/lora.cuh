// What the adapters of a projection's rows bring to its GEMM: more k-blocks.
//
// With h[t] = s_a (x[t] A_a^T) known, y[t] = [x[t] | h[t]] [W | B_a]^T: the product goes on over the rank. A tile of the GEMM has rows of several
// adapters, so it takes a k-block of each of them, with h[t] in the rows that use it and zeros in the others (an exact nothing on their sums, as B is
// finite). The rows' operand is laid out by lora_shrink as the GEMM's tiles read it; B is read as it is. Against a product of its own onto
// y that is one rounding instead of two, one launch, and 4 T N bytes less.
//
// An entry is the part of a tile that one k-block of `width` numbers holds: (adapter, 64 of its ranks, part of h). For fp32 outputs h has three bf16 parts, each
// what the ones before left, rounded: 24 bits. Each meets the same B. (Two parts: outputs off by 1.1e-6 where the projection's own sums are off by 5e-7, at
// K of 520; from K of 2,000 on those are off by more, 2e-6, and 4e-6 at 4,096.)
#pragma once

#ifdef B200_EMU  // host build of the walk over entries for tests/emu
#include "emu_shim.h"
#else
#include "common.cuh"
#endif

namespace b200 {

constexpr int LORA_MAX_RANK = 256;
constexpr int LORA_MAX_ADAPTERS = 1024;

struct NoLora {};
struct LoraExt {
  CUtensorMap b;       // [adapters, N, R], boxes of `width` columns
  CUtensorMap h;       // [tile, entry][tile_rows][width]
  uint64_t desc_base;  // of both operands in shared memory, without the address
  const int* count;    // adapters of each token tile
  const int* list;     // [tile][cap] which
  int cap, chunks, parts, width, tile_rows;  // most adapters of a tile; entries per adapter; parts of h; columns of an entry
  __device__ __forceinline__ uint64_t desc(uint32_t smem_addr) const { return desc_base | ((smem_addr & 0x3FFFF) >> 4); }
};
template <bool LORA>
struct LoraArgOf { typedef NoLora type; };
template <>
struct LoraArgOf<true> { typedef LoraExt type; };
template <bool LORA>
using LoraArg = typename LoraArgOf<LORA>::type;

// The entries of a token tile, as many to a pipeline stage of `k_blocks` k-blocks as fill it.
struct LoraSteps {
  int entries, per_stage;
  __device__ __forceinline__ LoraSteps(const LoraExt& x, int tile, int k_blocks) : entries(x.count[tile] * x.chunks), per_stage(k_blocks * 64 / x.width) {}
  __device__ __forceinline__ int of_stage(int e0) const { return min(per_stage, entries - e0); }
};

// The entries of a token tile one after the other: adapter, first rank, row of h. (Counted on, as each entry of a batch of many adapters would cost the
// producer three divisions and a look-up.)
struct LoraEntry {
  const int* next;
  int adapter, column = 0, row, then, sub = 0, part = 0;
  __device__ __forceinline__ LoraEntry(const LoraExt& x, int tile, int entries)
      : next(x.list + tile * x.cap), row(tile * x.cap * x.chunks * x.tile_rows) {
    adapter = entries > 0 ? *next : 0;
    then = entries > x.chunks ? *++next : 0;
  }
  __device__ __forceinline__ void step(const LoraExt& x, int left) {  // left: entries behind the one that is left
    row += x.tile_rows;
    if (++part == x.parts) { part = 0; column += x.width; }
    if (++sub == x.chunks) {
      sub = column = 0;
      adapter = then;
      if (left > x.chunks) then = *++next;
    }
  }
};

// A call's tables and h in its workspace.
struct LoraTiles {
  int tiles, tile_rows, cap, chunks, parts, width;
  int *count, *list;
  bf16* h;
};
inline size_t lora_tiles(int T, int R, int L, int tile_rows, bool f32, void* base, LoraTiles* t) {
  t->tile_rows = tile_rows;
  t->tiles = (T + tile_rows - 1) / tile_rows;
  t->cap = min(min(tile_rows, T), L);
  t->width = R <= 16 ? 16 : R <= 32 ? 32 : 64;
  t->parts = f32 ? 3 : 1;
  t->chunks = (R + 63) / 64 * t->parts;
  size_t at = 0;
  const auto take = [&](size_t bytes) { void* r = static_cast<uint8_t*>(base) + at; at += (bytes + 255) / 256 * 256; return r; };
  t->count = static_cast<int*>(take(static_cast<size_t>(t->tiles) * 4));
  t->list = static_cast<int*>(take(static_cast<size_t>(t->tiles) * t->cap * 4));
  t->h = static_cast<bf16*>(take(static_cast<size_t>(t->tiles) * t->cap * t->chunks * tile_rows * t->width * 2));
  return at;
}

// h and its tables (lora.cu).
int lora_shrink(const void* x, int ldx, const void* a, const float* scale, const int* rows, int T, int K, int R, int L, const LoraTiles& t, int* err,
                cudaStream_t st);

}  // namespace b200

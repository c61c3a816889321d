// The walk over a token tile's adapter entries (lora.cuh, LoraSteps and LoraEntry) as the GEMM's producer takes it, as host C++: every entry names its
// adapter, first rank and row of h, and of the tile's list nothing behind its last adapter is read.
//   g++ -std=c++20 -O1 -pthread -DB200_EMU -I tests/emu -x c++ tests/emu/lora_entries_emu.cpp -o lora_entries_emu
#include <cstdio>

#include "emu_shim.h"
struct CUtensorMap {};
typedef void* cudaStream_t;
namespace b200 {
using std::min;
}
#include "../../qwen36-mi250-tracelab-20261107_b200/ops/cuda/lora.cuh"

using namespace b200;

int main() {
  int bad = 0, walks = 0;
  for (int R : {8, 16, 24, 32, 64, 72, 128, 256})
    for (int f32 = 0; f32 < 2; ++f32)
      for (int cap : {1, 2, 3, 7, 40})
        for (int k_blocks : {1, 2, 4})
          for (int n = 0; n <= cap; ++n) {
            LoraTiles t;
            lora_tiles(48, R, cap, 16, f32, nullptr, &t);  // three tiles of 16 rows
            const int tile = 2;  // the last one
            t.cap = cap;
            std::vector<int> counts(t.tiles, n), list(static_cast<size_t>(t.tiles) * cap + 1, -7);  // (a word that nobody wrote behind it)
            for (int i = 0; i < n; ++i) list[static_cast<size_t>(tile) * cap + i] = 100 + 3 * i;
            const int* last = list.data() + static_cast<size_t>(tile) * cap + n - 1;
            LoraExt x{};
            x.count = counts.data();
            x.list = list.data();
            x.cap = cap, x.chunks = t.chunks, x.parts = t.parts, x.width = t.width, x.tile_rows = t.tile_rows;
            const LoraSteps steps(x, tile, k_blocks);
            LoraEntry e(x, tile, steps.entries);
            int at = 0;
            for (int e0 = 0; e0 < steps.entries; e0 += steps.per_stage)
              for (int j = 0, m = steps.of_stage(e0); j < m; ++j, e.step(x, steps.entries - e0 - j), ++at) {
                const int adapter = 100 + 3 * (at / t.chunks), column = at % t.chunks / t.parts * t.width, row = (tile * cap * t.chunks + at) * t.tile_rows;
                if (e.adapter != adapter || e.column != column || e.row != row) {
                  std::printf("rank %d, %d of %d adapters, entry %d: adapter %d, rank %d, row %d\n", R, n, cap, at, e.adapter, e.column, e.row);
                  ++bad;
                }
                if (e.next > last) ++bad;
              }
            if (n && e.next > last) {  // (where it has read)
              std::printf("rank %d, %d of %d adapters: read behind the last one\n", R, n, cap);
              ++bad;
            }
            if (at != steps.entries || steps.entries != n * t.chunks) ++bad;
            ++walks;
          }
  if (bad) {
    std::printf("%d faults in %d walks\n", bad, walks);
    return 1;
  }
  std::printf("OK %d walks\n", walks);
  return 0;
}

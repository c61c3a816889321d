// Low-rank adapters of many requests beside a projection that all rows share:
//
//   y[t, n] = sum_k x[t, k] W[n, k] + s_a sum_r b_a[n, r] (sum_k x[t, k] a_a[r, k]),   a the adapter of row t (below 0: none)
#include "common.cuh"

namespace b200 {

// A CTA takes one row and 1,024 of its outputs: h in shared memory, then a dot product over the rank for each output, onto the
// projection's fp32 result; rounded once.
template <typename OUT>
__global__ void __launch_bounds__(256) lora_add_kernel(const bf16* x, long long ldx, const float* base, const bf16* a, const bf16* b, const float* scale,
                                                       const int* rows, OUT* out, int N, int nb, int K, int R, int L, int* err) {
  __shared__ float h[128];
  pdl_wait();
  pdl_launch();
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  int id = rows[t];
  if (id >= L) {
    if (tid == 0 && blockIdx.y == 0) atomicCAS(err, 0, ERR_BAD_INDEX);
    id = -1;
  }
  if (id >= 0) {
    for (int r = tid >> 5; r < R; r += 8) {
      float sum = 0.f;
      for (int k = lane; k < K; k += 32)
        sum += __bfloat162float(x[t * ldx + k]) * __bfloat162float(a[(static_cast<size_t>(id) * R + r) * K + k]);
      sum = warp_sum(sum);
      if (lane == 0) h[r] = sum * scale[id];
    }
  }
  __syncthreads();
  for (int n = blockIdx.y * 1024 + tid; n < min(N, static_cast<int>(blockIdx.y) * 1024 + 1024); n += 256) {
    float v = base[static_cast<size_t>(t) * N + n];
    if (id >= 0 && n < nb)
      for (int r = 0; r < R; ++r) v += h[r] * __bfloat162float(b[(static_cast<size_t>(id) * nb + n) * R + r]);
    if constexpr (sizeof(OUT) == 2) out[static_cast<size_t>(t) * N + n] = __float2bfloat16(v);
    else out[static_cast<size_t>(t) * N + n] = v;
  }
}

}  // namespace b200

using namespace b200;

extern "C" int b200_lora_add(const void* x, long long ldx, const float* base, const void* a, const void* b, const float* scale, const int* rows, void* out,
                             int out_f32, int T, int N, int nb, int K, int R, int L, int* err, cudaStream_t st) {
  if (T <= 0) return 0;
  const dim3 grid(T, (N + 1023) / 1024);
  const auto args = [&](auto kern, auto* o) {
    return launch_pdl(kern, grid, dim3(256), 0, st, static_cast<const bf16*>(x), ldx, base, static_cast<const bf16*>(a), static_cast<const bf16*>(b),
                      scale, rows, o, N, nb, K, R, L, err) == cudaSuccess ? 0 : -4;
  };
  return out_f32 ? args(lora_add_kernel<float>, static_cast<float*>(out)) : args(lora_add_kernel<bf16>, static_cast<bf16*>(out));
}

// Rows of keys and values into the pages of the 8-bit KV cache, and back.
//
//  write:  e = the smallest integer with max |x| <= 448 * 2^e, data = e4m3(x * 2^-e), one rounding.
//  read:   x = data * 2^e as bf16, exact.
//
// Bound: memory, 4 D bytes of bf16 and 2 (D + 1) of the cache per token and KV head. D / 8 (write) or D / 16 (read) neighbouring
// lanes own a row, 16 bytes of input each, and take the key and the value of a (token, head) together: two loads in flight per thread and one
// look-up of the page. The row maximum is a shuffle among its lanes.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace b200 {

// Index of a token's row in the cache (of its key; the value's is n_kv * 64 further), or -1.
__device__ __forceinline__ long long kv8_row(int64_t pos, int seq, int kh, const int* tables, int max_pages, int width, int n_seqs,
                                             int num_pages, int n_kv) {
  if (pos < 0 || pos >= static_cast<int64_t>(width) * KV8_PAGE || seq < 0 || seq >= n_seqs) return -1;
  const int page = tables[static_cast<size_t>(seq) * max_pages + pos / KV8_PAGE];
  if (page < 0 || page >= num_pages) return -1;
  return (static_cast<long long>(page) * 2 * n_kv + kh) * KV8_PAGE + pos % KV8_PAGE;
}

// Eight numbers of a row; ALIGNED: with one 16-byte load.
template <bool ALIGNED>
__device__ __forceinline__ void load8(const bf16* p, float* v) {
  if constexpr (ALIGNED) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = __bfloat1622float2(e[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
  }
}

template <int D, bool ALIGNED>
__global__ void __launch_bounds__(256)
kv8_write_kernel(const bf16* k, long long k_row, long long k_head, const bf16* v, long long v_row, long long v_head,
                 const int64_t* positions, const int* seq_of_row, const int* tables, int max_pages, int width, int n_seqs,
                 uint8_t* data, uint8_t* exps, int T, int n_kv, int num_pages, int* err) {
  constexpr int LANES = D / 8;
  pdl_wait();
  pdl_launch();
  const long long item = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / LANES;  // (token, head)
  const int part = threadIdx.x % LANES;
  const bool real = item < static_cast<long long>(T) * n_kv;
  const int row = real ? static_cast<int>(item / n_kv) : 0, kh = static_cast<int>(item % n_kv);
  float x[2][8];
  load8<ALIGNED>(k + row * k_row + (real ? kh : 0) * k_head + part * 8, x[0]);
  load8<ALIGNED>(v + row * v_row + (real ? kh : 0) * v_head + part * 8, x[1]);
  const long long at = real ? kv8_row(positions[row], seq_of_row[row], kh, tables, max_pages, width, n_seqs, num_pages, n_kv) : -1;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float amax = 0.f, nan = 0.f;  // fmaxf passes over a NaN; a sum of zeros and NaNs keeps it
#pragma unroll
    for (int i = 0; i < 8; ++i) { amax = fmaxf(amax, fabsf(x[which][i])); nan = x[which][i] != x[which][i] ? 1.f : nan; }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      nan = fmaxf(nan, __shfl_xor_sync(0xffffffffu, nan, o));
    }
    const int e = kv8_exponent(amax);
    const float f = kv8_two_to(-e);
    uint2 packed = make_uint2(0u, 0u);
    if (nan == 0.f) {
      packed.x = kv8_pack2(x[which][0] * f, x[which][1] * f) | kv8_pack2(x[which][2] * f, x[which][3] * f) << 16;
      packed.y = kv8_pack2(x[which][4] * f, x[which][5] * f) | kv8_pack2(x[which][6] * f, x[which][7] * f) << 16;
    }
    if (at >= 0) {
      const size_t r = static_cast<size_t>(at) + static_cast<size_t>(which) * n_kv * KV8_PAGE;
      *reinterpret_cast<uint2*>(data + r * D + part * 8) = packed;
      if (part == 0) exps[r] = static_cast<uint8_t>(nan == 0.f ? e + 127 : KV8_E_NAN);
    }
  }
  if (real && at < 0 && part == 0) atomicCAS(err, 0, ERR_BAD_INDEX);
}

template <int D>
__global__ void __launch_bounds__(256)
kv8_read_kernel(const uint8_t* data, const uint8_t* exps, const int64_t* positions, const int* seq_of_row, const int* tables,
                int max_pages, int width, int n_seqs, bf16* k, bf16* v, int T, int n_kv, int num_pages, int* err) {
  constexpr int LANES = D / 16;
  pdl_wait();
  pdl_launch();
  const long long item = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) / LANES;
  const int part = threadIdx.x % LANES;
  if (item >= static_cast<long long>(T) * n_kv) return;
  const int row = static_cast<int>(item / n_kv), kh = static_cast<int>(item % n_kv);
  const long long at = kv8_row(positions[row], seq_of_row[row], kh, tables, max_pages, width, n_seqs, num_pages, n_kv);
  uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  uint32_t byte[2] = {127u, 127u};
  if (at >= 0) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const size_t r = static_cast<size_t>(at) + static_cast<size_t>(which) * n_kv * KV8_PAGE;
      raw[which] = *reinterpret_cast<const uint4*>(data + r * D + part * 16);
      byte[which] = exps[r];
    }
  } else if (part == 0) {
    atomicCAS(err, 0, ERR_BAD_INDEX);
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float f = kv8_factor(byte[which]);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[which]);
    uint4 out[2];
    __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h[2];
      kv8_unpack4(w[i], h[0], h[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        o[2 * i + j] = __floats2bfloat162_rn(x.x * f, x.y * f);
      }
    }
    uint4* dst = reinterpret_cast<uint4*>((which ? v : k) + item * D + part * 16);
    dst[0] = out[0];
    dst[1] = out[1];
  }
}

}  // namespace b200

using namespace b200;

// k, v: [T, n_kv, D] bf16, rows and heads any distance apart (in numbers), a head's numbers next to each other. data, exps: one layer of the cache.
extern "C" int b200_kv8_write(const void* k, long long k_row, long long k_head, const void* v, long long v_row, long long v_head,
                              const int64_t* positions, const int* seq_of_row, const int* tables, int max_pages, int width,
                              int n_seqs, void* data, void* exps, int T, int n_kv, int D, int num_pages, int* err, cudaStream_t st) {
  if (T <= 0) return 0;
  const auto rows_of_16 = [](const void* p, long long row, long long head) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % 8 == 0 && head % 8 == 0;
  };
  const bool aligned = rows_of_16(k, k_row, k_head) && rows_of_16(v, v_row, v_head);
  const long long threads = static_cast<long long>(T) * n_kv * (D / 8);
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
  cudaError_t rc;
#define KV8_WRITE(DD)                                                                                                      \
  rc = launch_pdl(aligned ? kv8_write_kernel<DD, true> : kv8_write_kernel<DD, false>, grid, dim3(256), 0, st,              \
                  static_cast<const bf16*>(k), k_row, k_head, static_cast<const bf16*>(v), v_row, v_head, positions,       \
                  seq_of_row, tables, max_pages, width, n_seqs, static_cast<uint8_t*>(data), static_cast<uint8_t*>(exps),  \
                  T, n_kv, num_pages, err)
  if (D == 256) KV8_WRITE(256);
  else if (D == 128) KV8_WRITE(128);
  else if (D == 64) KV8_WRITE(64);
  else if (D == 32) KV8_WRITE(32);
  else return -7;
#undef KV8_WRITE
  return rc == cudaSuccess ? 0 : -4;
}

// k, v: [T, n_kv, D] bf16, contiguous. Rows without a page are zero and leave an error code.
extern "C" int b200_kv8_read(const void* data, const void* exps, const int64_t* positions, const int* seq_of_row, const int* tables,
                             int max_pages, int width, int n_seqs, void* k, void* v, int T, int n_kv, int D, int num_pages, int* err,
                             cudaStream_t st) {
  if (T <= 0) return 0;
  const long long threads = static_cast<long long>(T) * n_kv * (D / 16);
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
  cudaError_t rc;
#define KV8_READ(DD)                                                                                                        \
  rc = launch_pdl(kv8_read_kernel<DD>, grid, dim3(256), 0, st, static_cast<const uint8_t*>(data),                           \
                  static_cast<const uint8_t*>(exps), positions, seq_of_row, tables, max_pages, width, n_seqs,               \
                  static_cast<bf16*>(k), static_cast<bf16*>(v), T, n_kv, num_pages, err)
  if (D == 256) KV8_READ(256);
  else if (D == 128) KV8_READ(128);
  else if (D == 64) KV8_READ(64);
  else if (D == 32) KV8_READ(32);
  else return -7;
#undef KV8_READ
  return rc == cudaSuccess ? 0 : -4;
}

// Rows of keys and values into the pages of the 8-bit KV cache, and back.
//
//  write:  e = the smallest integer with max |x| <= 448 * 2^e, data = e4m3(x * 2^-e), one rounding.
//  read:   x = data * 2^e as bf16, exact.
//
// Bound: memory, 4 D bytes of bf16 and 2 (D + 1) of the cache per token and KV head. D / 8 (write) or D / 16 (read) neighbouring
// lanes own a row, 16 bytes of input each, and take the key and the value of a (token, head) together: two loads in flight per thread and one
// look-up of the page. The row maximum is one of its lanes' bits. Two rows a thread, all loads under way at once, were no faster (write, 6.9 us and
// 6.8) or slower (read, 58.2 and 55.6; all four before rows were counted in 32 bits).
//
// Measured, 2 heads of 256: 128 rows written in 1.8 us, which is a launch and two look-ups; 8,192 rows in 6.3 us (25 MB at 4.0 TB/s, of which 1.8 us
// as before); 98,304 rows read in 54.3 us (304 MB at 5.6 TB/s: 85 % of the copy rate), 6,001 rows in 5.9 us.
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace b200 {

// Where a token's row is: its page, asked for where the indices name one (nothing waits for it here), and from it the row in the
// cache (of the key; the value's is n_kv * 64 further).
struct Kv8Where {
  uint32_t page;
  int at, kh;
  __device__ __forceinline__ Kv8Where(int64_t pos, int seq, int kh_, const int* tables, int max_pages, int width, int n_seqs, bool real)
      : page(0xffffffffu), at(static_cast<int>(pos & (KV8_PAGE - 1))), kh(kh_) {
    ask_32(page, tables + static_cast<size_t>(seq) * max_pages + pos / KV8_PAGE,
           real && pos >= 0 && pos < static_cast<int64_t>(width) * KV8_PAGE && seq >= 0 && seq < n_seqs);
  }
  __device__ __forceinline__ bool there(int num_pages) const { return static_cast<int>(page) >= 0 && static_cast<int>(page) < num_pages; }
  __device__ __forceinline__ size_t row(int n_kv) const { return (static_cast<size_t>(page) * 2 * n_kv + kh) * KV8_PAGE + at; }
};

// Eight numbers of a row; ALIGNED: with one 16-byte load.
template <bool ALIGNED>
__device__ __forceinline__ uint4 load8(const bf16* p) {
  if constexpr (ALIGNED) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  const auto word = [&](int i) { return static_cast<uint32_t>(h[i]) | static_cast<uint32_t>(h[i + 1]) << 16; };
  return make_uint4(word(0), word(2), word(4), word(6));
}

template <int D, bool ALIGNED>
__global__ void __launch_bounds__(256)
kv8_write_kernel(const bf16* k, long long k_row, long long k_head, const bf16* v, long long v_row, long long v_head,
                 const int64_t* positions, const int* seq_of_row, const int* tables, int max_pages, int width, int n_seqs,
                 uint8_t* data, uint8_t* exps, int T, int n_kv, int num_pages, int* err) {
  constexpr int LANES = D / 8;
  pdl_wait();
  pdl_launch();
  const uint32_t item = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;  // (token, head), in 32 bits: a division of 64 takes as long as the rest
  const int part = threadIdx.x % LANES;
  const bool real = item < static_cast<uint32_t>(T) * n_kv;
  const int row = real ? static_cast<int>(item / static_cast<uint32_t>(n_kv)) : 0, kh = real ? static_cast<int>(item) - row * n_kv : 0;
  const int64_t pos = positions[row];
  const int seq = seq_of_row[row];
  const uint4 raw[2] = {load8<ALIGNED>(k + row * k_row + kh * k_head + part * 8), load8<ALIGNED>(v + row * v_row + kh * v_head + part * 8)};
  const Kv8Where where(pos, seq, kh, tables, max_pages, width, n_seqs, real);
  const bool there = where.there(num_pages);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint32_t w[4] = {raw[which].x, raw[which].y, raw[which].z, raw[which].w};
    // magnitudes of bf16 numbers are in the order of their bits, those of NaNs above all others
    uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    top = max(top & 0xffffu, top >> 16);
    if constexpr (LANES == 32) {
      top = __reduce_max_sync(0xffffffffu, top);
    } else {
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const bool nan = top > 0x7f80u;
    const int e = kv8_exponent(__uint_as_float(top << 16));
    const float f = kv8_two_to(-e);
    uint32_t two[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) two[j] = kv8_pack2(__uint_as_float(w[j] << 16) * f, __uint_as_float(w[j] & 0xffff0000u) * f);
    if (there) {
      const size_t r = where.row(n_kv) + static_cast<size_t>(which) * n_kv * KV8_PAGE;
      *reinterpret_cast<uint2*>(data + r * D + part * 8) = nan ? make_uint2(0u, 0u) : make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
      if (part == 0) exps[r] = static_cast<uint8_t>(nan ? KV8_E_NAN : e + 127);
    }
  }
  if (real && !there && part == 0) atomicCAS(err, 0, ERR_BAD_INDEX);
}

template <int D>
__global__ void __launch_bounds__(256)
kv8_read_kernel(const uint8_t* data, const uint8_t* exps, const int64_t* positions, const int* seq_of_row, const int* tables,
                int max_pages, int width, int n_seqs, bf16* k, bf16* v, int T, int n_kv, int num_pages, int* err) {
  constexpr int LANES = D / 16;
  pdl_wait();
  pdl_launch();
  const uint32_t item = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int part = threadIdx.x % LANES;
  if (item >= static_cast<uint32_t>(T) * n_kv) return;
  const int row = static_cast<int>(item / static_cast<uint32_t>(n_kv)), kh = static_cast<int>(item) - row * n_kv;
  const Kv8Where where(positions[row], seq_of_row[row], kh, tables, max_pages, width, n_seqs, true);
  const bool there = where.there(num_pages);
  uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  uint16_t byte[2] = {127, 127};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const size_t r = where.row(n_kv) + static_cast<size_t>(which) * n_kv * KV8_PAGE;
    ask_128(raw[which], data + r * D + part * 16, there);
    ask_8(byte[which], exps + r, there);
  }
  if (!there && part == 0) atomicCAS(err, 0, ERR_BAD_INDEX);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float f = kv8_factor(byte[which]);
    const uint32_t w[4] = {raw[which].x, raw[which].y, raw[which].z, raw[which].w};
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
    uint4* dst = reinterpret_cast<uint4*>((which ? v : k) + static_cast<size_t>(item) * D + part * 16);
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
  if (static_cast<long long>(T) * n_kv > 0x7fffffffLL) return -7;  // rows are counted in 32 bits
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
  if (static_cast<long long>(T) * n_kv > 0x7fffffffLL) return -7;  // rows are counted in 32 bits
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

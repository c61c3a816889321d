// The 8-bit KV cache's number format: rows of D e4m3 numbers with one power of two each, held as a byte biased by 127. 255 marks
// a row that held a NaN (its data bytes are 0).
#pragma once

#include "common.cuh"

namespace b200 {

constexpr int KV8_PAGE = 64;
constexpr int KV8_E_MAX = 60;
constexpr int KV8_E_NAN = 255;

// The exponent of a row whose largest magnitude is `amax`: the smallest e with amax <= 448 * 2^e, in [-60, 60]. 448 = 1.75 * 2^8.
__device__ __forceinline__ int kv8_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(-KV8_E_MAX, min(KV8_E_MAX, e));  // 0 and subnormal numbers: bits >> 23 is 0, far below
}
__device__ __forceinline__ float kv8_two_to(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The factor that an exponent byte stands for. (A byte of 0 is written by nobody; it reads as 2^-126.)
__device__ __forceinline__ float kv8_factor(uint32_t byte) {
  return byte == KV8_E_NAN ? __uint_as_float(0x7fffffffu) : __uint_as_float(max(byte, 1u) << 23);
}

// Two floats to two e4m3 bytes (the first in the low one), to nearest even, and to +-448 beyond it.
__device__ __forceinline__ uint32_t kv8_pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two e4m3 bytes to two halves, exactly.
__device__ __forceinline__ uint32_t kv8_unpack2(uint16_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The sigmoids of the halves of a word of bf16 gates, for outputs that are rounded to bf16 next: 1 / (1 + 2^-t) with t = x log2(e) on the unit of
// special functions. An exact division is a subroutine: the loop at the end of a prefill tile (128 rows of 256) took 32,500 cycles with it, and 20,000
// so. (Two sigmoids from one reciprocal, 1 / a = b / (a b), need a case of their own where the product overflows or one is NaN: no faster.)
__device__ __forceinline__ float2 kv8_sigmoid2(uint32_t gates) {
  float a[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float x = __uint_as_float(i ? gates & 0xffff0000u : gates << 16);
    a[i] = ex2(x * -1.4426950408889634f) + 1.0f;
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a[i]));
  }
  return make_float2(a[0], a[1]);
}
// The four bytes of a word as two pairs of halves.
__device__ __forceinline__ void kv8_unpack4(uint32_t word, uint32_t& lo, uint32_t& hi) {
  lo = kv8_unpack2(static_cast<uint16_t>(word));
  hi = kv8_unpack2(static_cast<uint16_t>(word >> 16));
}

// Whether a barrier's phase is complete, without a wait.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return done != 0;
}

// Loads under a condition that nothing waits for before their value is used (after one in a branch the compiler waits at the branch's end);
// without it the value stays.
__device__ __forceinline__ void ask_64(int64_t& x, const int64_t* p, bool yes) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.s64 %0, [%1];\n\t}" : "+l"(x) : "l"(p), "r"(static_cast<int>(yes)));
}
__device__ __forceinline__ void ask_32(uint32_t& x, const void* p, bool yes) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.u32 %0, [%1];\n\t}" : "+r"(x) : "l"(p), "r"(static_cast<int>(yes)));
}
__device__ __forceinline__ void ask_8(uint16_t& x, const void* p, bool yes) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q ld.global.u8 %0, [%1];\n\t}" : "+h"(x) : "l"(p), "r"(static_cast<int>(yes)));
}
__device__ __forceinline__ void ask_128(uint4& x, const void* p, bool yes) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t@q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "+r"(x.x), "+r"(x.y), "+r"(x.z), "+r"(x.w) : "l"(p), "r"(static_cast<int>(yes)));
}

// The tensor map of bytes of `rank` dims (2 or 3), the strides of all but the first in bytes. Not 0: it cannot be made.
inline int kv8_encode(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                      CUtensorMapSwizzle sw) {
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static EncodeFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || !ptr) return -1;
    fn = reinterpret_cast<EncodeFn>(ptr);
  }
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : -2;
}
// That of a layer's exponents [pages, 2, n_kv, 64]: a box has those of a page's keys and values of one head.
inline int kv8_encode_exps(CUtensorMap* m, const void* exps, int n_kv, long long pages) {
  const cuuint64_t dims[3] = {KV8_PAGE, static_cast<cuuint64_t>(n_kv), static_cast<cuuint64_t>(pages) * 2};
  const cuuint64_t strides[2] = {KV8_PAGE, static_cast<cuuint64_t>(n_kv) * KV8_PAGE};
  const cuuint32_t box[3] = {KV8_PAGE, 1, 2};
  return kv8_encode(m, exps, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

}  // namespace b200

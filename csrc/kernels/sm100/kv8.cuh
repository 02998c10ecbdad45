// 8-bit key-value pages: the format, and the conversions that the kernels of kv8_store.cu and kv8_attn.cu share.
//
// A pool is [page][kv_head] blocks of 32 * hd + 128 bytes, one block after the other:
//     K codes [16 tokens][hd] | V codes [16][hd] | 16 x (K scale, V scale) fp32
// so that everything attention needs of a page and a KV head is one contiguous piece (4224 bytes at hd 128).
// Every row (one token, one KV head, K or V) has its own scale, max(amax / 127, 2^-64) for int8 codes -127 .. 127 (stored
// with 128 added, so that one byte permute makes the fp16 number 1024 + byte) or max(amax / 448, 2^-64) for e4m3 codes.
// code = round-to-nearest-even(x / scale); the row stands for code * scale.  The lower limit keeps 1 / scale finite and lets
// a row of zeros count as one that adds nothing (the attention weighs rows by their scale's exponent).  A row with an
// infinity or a NaN gets the scale NaN and the codes of zeros: it reads back as NaN instead of as a number that hides the fault.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace b2 {

enum Kv8Format : int { KV8_INT8 = 0, KV8_FP8 = 1 };
constexpr int kKv8Page = 16;
constexpr float kKv8MinScale = 5.421010862427522e-20f;   // 2^-64

__host__ __device__ constexpr int kv8_block_bytes(int hd) { return 2 * kKv8Page * hd + kKv8Page * 8; }

// four e4m3 numbers -> fp16 pairs (0, 1) and (2, 3)
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t& x, uint32_t& y) {
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.rn.f16x2.e4m3x2 %0, lo; cvt.rn.f16x2.e4m3x2 %1, hi; }" : "=r"(x), "=r"(y) : "r"(w));
}

// fp32 values of four stored bytes
template <int FMT>
__device__ __forceinline__ void kv8_values(uint32_t w, float* f) {
  if (FMT == KV8_INT8) {                     // 0x4b0000xx is 2^23 + xx
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + i)) - 8388736.f;
  } else {
    uint32_t lo, hi;
    e4m3_pairs(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  }
}

// stored byte of y = x / scale
template <int FMT>
__device__ __forceinline__ uint32_t kv8_code(float y) {
  if (FMT == KV8_INT8) return (uint32_t)(max(-127, min(127, __float2int_rn(y))) + 128);
  return (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace b2

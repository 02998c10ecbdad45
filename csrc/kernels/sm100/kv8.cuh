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

// fp32 value of a stored byte
template <int FMT>
__device__ __forceinline__ float kv8_value(uint32_t byte) {
  if (FMT == KV8_INT8) return (float)((int)byte - 128);
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

// stored byte of y = x / scale
template <int FMT>
__device__ __forceinline__ uint32_t kv8_code(float y) {
  if (FMT == KV8_INT8) return (uint32_t)(max(-127, min(127, __float2int_rn(y))) + 128);
  return (uint32_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace b2

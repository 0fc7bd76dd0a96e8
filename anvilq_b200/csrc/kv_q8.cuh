// kv_q8.cuh -- the 8-bit paged KV cache: its format, the page table and the
// conversions between codes and values (shared by paged_append.cu, which writes
// the cache, and gqa_decode_q8.cu, which reads it).
//
// Format.  A pool holds num_pages pages of page_tokens tokens (a multiple of
// 16), each head's rows of a page together, and one binary32 scale for every
// block of 16 tokens of a page and kv head:
//   codes   [num_pages][Hkv][page_tokens][D]      int8, or e4m3 (8-bit float)
//   scales  [num_pages][Hkv][page_tokens / 16]    value = code * scale
// A (page, head) is therefore one contiguous run of page_tokens * D bytes, and
// a block of 16 rows one run of 1 or 2 KB: a reader of one head streams whole
// runs, where rows of all heads side by side would give it D bytes at a time.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/anvilq.h"

namespace anvilq {
namespace q8 {

constexpr int kBlock = ANVILQ_KV_Q8_BLOCK;   // tokens that share a scale
constexpr int kInt8 = ANVILQ_KV_Q8_INT8, kE4m3 = ANVILQ_KV_Q8_E4M3;

// Physical page of logical page j of sequence b (bit 31 valid, bits 30:0 the
// page); -1 where the entry of this live page is absent or out of range.
__device__ __forceinline__ int page_of(const uint32_t* table, int max_pages, int num_pages, int b, int j) {
  const uint32_t e = table[(size_t)b * max_pages + j];
  const uint32_t page = e & 0x7FFFFFFFu;
  return (e >> 31) && page < (uint32_t)num_pages ? (int)page : -1;
}

// four codes (ascending bytes) as binary32 values
template <int TYPE>
__device__ __forceinline__ void codes_to_float4(uint32_t w, float* v) {
  if (TYPE == kInt8) {
    // (code + 128) in the last byte of 2^23, made signed by one exact subtraction
    const uint32_t u = w ^ 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)) - 8388736.0f;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2 h(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((w >> (16 * i)) & 0xFFFFu), __NV_E4M3));
      const float2 f = __half22float2(h);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// four binary32 values as codes, each rounded to the nearest (ties to even).  They
// are within the type's range but for their own rounding: |value| <= largest code
// times a few (1 + 2^-24), which rounds to the largest code (int8 uses -127 .. 127).
template <int TYPE>
__device__ __forceinline__ uint32_t float4_to_codes(const float* v) {
  if (TYPE == kInt8) {
    // the sum's last bits are the rounded value's (two's complement)
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(__fadd_rn(v[i], 12582912.0f));   // 1.5 2^23
    return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// The scale of a block whose largest magnitude is `top` (0 for an all-zero one).
// int8: top / 127, the tightest.  e4m3: the smallest power of two with
// top <= 448 * scale -- a floating code keeps its relative precision under a
// power of two, so nothing is gained by a tighter scale, and a block whose scale
// grows later is re-scaled without rounding until its codes run into e4m3's
// subnormals.
template <int TYPE>
__device__ __forceinline__ float scale_for(float top) {
  if (TYPE == kInt8) return __fdiv_rn(top, 127.0f);
  if (top == 0.0f) return 0.0f;
  const uint32_t bits = __float_as_uint(top);           // top = m 2^E, 1 <= m < 2; 448 = 1.75 2^8
  int e = (int)(bits >> 23) - 127;
  e -= (bits & 0x7FFFFFu) <= 0x600000u ? 8 : 7;
  return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

// Whether two runs of bytes share any (an empty one shares none).
inline bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return na && nb && x < y + nb && y < x + na;
}

}  // namespace q8
}  // namespace anvilq

// Register helpers shared by the GEMM epilogues.
#pragma once

#include <cstring>

#include "frx_ptx.cuh"

namespace frx {

// v[idx] for a runtime idx in [0, 32) as a 5-level select tree, so the array stays in
// registers (an indexed read would demote it to local memory).
__device__ __forceinline__ float select32(const float (&v)[32], int idx) {
  float w16[16], w8[8], w4[4], w2[2];
#pragma unroll
  for (int j = 0; j < 16; ++j) w16[j] = (idx & 16) ? v[j + 16] : v[j];
#pragma unroll
  for (int j = 0; j < 8; ++j) w8[j] = (idx & 8) ? w16[j + 8] : w16[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) w4[j] = (idx & 4) ? w8[j + 4] : w8[j];
#pragma unroll
  for (int j = 0; j < 2; ++j) w2[j] = (idx & 2) ? w4[j + 2] : w4[j];
  return (idx & 1) ? w2[1] : w2[0];
}

// The same for idx in [0, 16).
__device__ __forceinline__ float select16(const float (&v)[16], int idx) {
  float w8[8], w4[4], w2[2];
#pragma unroll
  for (int j = 0; j < 8; ++j) w8[j] = (idx & 8) ? v[j + 8] : v[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) w4[j] = (idx & 4) ? w8[j + 4] : w8[j];
#pragma unroll
  for (int j = 0; j < 2; ++j) w2[j] = (idx & 2) ? w4[j + 2] : w4[j];
  return (idx & 1) ? w2[1] : w2[0];
}

// The two 16-bit values packed in `w` (low half first) as floats: bf16 or fp16.
__device__ __forceinline__ float2 unpack2(uint32_t w, bool f16) {
  if (f16) {
    __half2 h;
    memcpy(&h, &w, sizeof(h));
    return __half22float2(h);
  }
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

}  // namespace frx

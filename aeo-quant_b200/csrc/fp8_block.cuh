// Shared by the block-scaled FP8 kernels: e4m3 values with one f32 scale per
// 128 consecutive values of a row (activations) or per 128 x 128 block
// (weights).
//
//   a = max(max|x|, 1e-30)   scale = f32(a / 448)   inv = f32(448 / a)
//   q = e4m3(f32(x * inv))   value = q * scale
//
// 448 is the largest e4m3 value; the floor keeps `inv` finite for blocks of
// zeros. One product with the inverse per value, rounded to nearest even
// twice (to f32, then to e4m3), takes the place of a division. A block that
// holds an infinity or a NaN gets a NaN scale and NaN codes.
#pragma once

#include "common.cuh"

namespace aeoq {

constexpr int kFbBlock = 128;
constexpr float kFbFloor = 1e-30f;

__host__ __device__ __forceinline__ int64_t fb_blocks(int64_t n) { return (n + kFbBlock - 1) / kFbBlock; }

// {inverse, scale} of a block from its largest magnitude (any value from
// infinity on: NaN).
__device__ __forceinline__ float2 fb_scales(float amax) {
  const float a = amax < INFINITY ? fmaxf(amax, kFbFloor) : __int_as_float(0x7FC00000);
  return make_float2(__fdiv_rn(kFp8Max, a), __fdiv_rn(a, kFp8Max));
}

// Four values to e4m3 codes, lowest byte first (round to nearest even; NaN
// stays NaN; |v| <= 448 up to f32 rounding, which the conversion saturates).
__device__ __forceinline__ uint32_t fb_codes4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Eight consecutive input values as floats.
template <int DT>
__device__ __forceinline__ void fb_load8(const typename In<DT>::T* p, float (&v)[8]) {
  if constexpr (DT == AEOQ_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const typename In<DT>::T* e = reinterpret_cast<const typename In<DT>::T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = In<DT>::to_f(e[i]);
  }
}

// Largest magnitude as an ordered bit pattern: NaN above infinity.
__device__ __forceinline__ uint32_t fb_key8(const float (&v)[8]) {
  uint32_t k = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) k = max(k, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return k;
}
__device__ __forceinline__ float fb_key_value(uint32_t k) { return __uint_as_float(k); }

__device__ __forceinline__ uint2 fb_codes8(const float (&v)[8], float inv) {
  return make_uint2(fb_codes4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                    fb_codes4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}

// Rows [0, rows) of x (or x[idx[r]], r < *n_rows) quantized per 128 values; their
// scales (rows, ceil(K / 128)).
int fb_quantize_rows(const void* x, int dtype, int64_t rows, int64_t K, int64_t ld, const int* idx,
                     const int* n_rows, uint8_t* q, int64_t q_ld, float* scale, cudaStream_t st);

}  // namespace aeoq

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

// Eight consecutive input values, as they came (16 bytes, 32 for f32: the
// registers that a value costs while its block's maximum is not known yet).
template <int DT> struct FbEight {
  using T = typename In<DT>::T;
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void load_some(const T* p, int64_t n) {
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = T(0.0f);
      if (i < n) v[i] = p[i];
    }
    u = *reinterpret_cast<const uint4*>(v);
  }
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  // Largest magnitude as an ordered key: two 16-bit patterns side by side, NaN
  // above infinity.
  __device__ __forceinline__ uint32_t key() const {
    constexpr uint32_t m = 0x7FFF7FFFu;
    return __vmaxu2(__vmaxu2(u.x & m, u.y & m), __vmaxu2(u.z & m, u.w & m));
  }
  static __device__ __forceinline__ uint32_t key_max(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
  static __device__ __forceinline__ float key_value(uint32_t k) { return In<DT>::key_to_f(max(k >> 16, k & 0xFFFFu)); }
  __device__ __forceinline__ float at(int i) const { return In<DT>::to_f(reinterpret_cast<const T*>(&u)[i]); }
};
template <> struct FbEight<AEOQ_F32> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldg(reinterpret_cast<const float4*>(p));
    b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void load_some(const float* p, int64_t n) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
    a = make_float4(v[0], v[1], v[2], v[3]);
    b = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float at(int i) const {
    return i < 4 ? (i < 2 ? (i ? a.y : a.x) : (i == 2 ? a.z : a.w)) : (i < 6 ? (i == 4 ? b.x : b.y) : (i == 6 ? b.z : b.w));
  }
  __device__ __forceinline__ uint32_t key() const {
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) k = max(k, __float_as_uint(at(i)) & 0x7FFFFFFFu);
    return k;
  }
  static __device__ __forceinline__ uint32_t key_max(uint32_t x, uint32_t y) { return max(x, y); }
  static __device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k); }
};

template <int DT>
__device__ __forceinline__ uint2 fb_codes8(const FbEight<DT>& v, float inv) {
  return make_uint2(fb_codes4(v.at(0) * inv, v.at(1) * inv, v.at(2) * inv, v.at(3) * inv),
                    fb_codes4(v.at(4) * inv, v.at(5) * inv, v.at(6) * inv, v.at(7) * inv));
}

enum FbActivation : int { kFbGeluTanh = 0, kFbSilu = 1 };

// gelu(x, tanh form) = x * sigmoid(2 z), z = sqrt(2/pi) (x + 0.044715 x^3),
// since 1 + tanh(z) = 2 sigmoid(2 z); silu(x) = x * sigmoid(x). Written so,
// neither cancels for negative x. Both are x / (1 + 2^(-x (c0 + c1 x^2))) with
// constants of their own, log2 e among them. The approximate 2^x and 1/x are
// within 2^-22 each, and an exponent a brings |a| 2^-24; where that is large
// the result is 0 or x to within f32. (The library's __expf and __fdividef
// take care of denormals too: the epilogue of 4096 tokens' gate_up 66 us
// longer.)
__device__ __forceinline__ float2 fb_act_of(int act) {
  return act == kFbSilu ? make_float2(-1.4426950408889634f, 0.0f)
                        : make_float2(-2.302208198f, -0.1029432396f);   // -2 sqrt(2/pi) log2 e, times 0.044715
}
// The exponent of that 2^x: the lower x, the larger.
__device__ __forceinline__ float fb_act_exponent(float2 c, float x) {
  return x * fmaf(c.y, fminf(x * x, 1e30f), c.x);
}

__device__ __forceinline__ float fb_act(float2 c, float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fb_act_exponent(c, x)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return x * r;
}

// Two at once with one reciprocal, 1/a = b/(ab): the two approximations per
// value are what the epilogues wait for (16 per SM and cycle). a = 1 + 2^x is
// held times 2^-63, so that the product of two of up to 2^126 each stays
// finite and its reciprocal normal; from there on 1/a is 0, as the reciprocal
// above makes it. (Gates that far below 0 still count where a whole block of
// 128 values is tiny: their largest sets the scale. With a cut at 2^60
// such a block came out up to 2^66 times too large; that took 206 us for the
// gate_up of 4096 tokens, this 208, and a branch to two reciprocals, which some
// pair of most warps needs, 231.)
__device__ __forceinline__ float2 fb_act2(float2 c, float x, float y) {
  constexpr float kMost = 126.0f, kDown = 0x1p-63f;
  const float u = fb_act_exponent(c, x), v = fb_act_exponent(c, y);
  float a, b, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(fminf(u, kMost)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(fminf(v, kMost)));
  a = fmaf(a, kDown, kDown);
  b = fmaf(b, kDown, kDown);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  const float p = u > kMost ? 0.0f : r * b * kDown, q = v > kMost ? 0.0f : r * a * kDown;
  return make_float2(x * p, y * q);
}

// Few rows of a: the weights are streamed through mma.sync (fp8_block_skinny.cu).
constexpr int kFbSkinnyQuant = 8;        // linear: rows that each CTA quantizes for itself (no workspace)
bool fb_linear_skinny_takes(int64_t M, int64_t N, int64_t K);
int fb_linear_skinny(const void* x, int dtype, int64_t ldx, int64_t M, const uint8_t* w, const float* sw, int64_t N,
                     int64_t K, const void* bias, void* out, int out_dt, int64_t ldc, uint8_t* q, float* qs,
                     cudaStream_t st);
bool fb_experts_skinny_takes(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I);
int64_t fb_experts_skinny_most(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I);
int fb_experts_skinny(const void* hidden, int64_t T, const void* ids, int ids_dt, const float* weights, int64_t k,
                      const uint8_t* gu, const float* gus, const uint8_t* dw, const float* dws, int64_t E, int64_t H,
                      int64_t I, int act, float* h, void* out, cudaStream_t st);

// Rows of x quantized per 128 values; their scales (rows, ceil(K / 128)).
int fb_quantize_rows(const void* x, int dtype, int64_t rows, int64_t K, int64_t ld, uint8_t* q, int64_t q_ld,
                     float* scale, cudaStream_t st);
// The same for contiguous, 16-byte aligned bf16 rows with K % 8 == 0; row r goes
// to the rows to[r * k] .. to[r * k + k - 1] that are not negative.
int fb_quantize_rows_to(const void* x, int64_t rows, int64_t K, const int* to, int k, uint8_t* q, float* scale,
                        cudaStream_t st);

}  // namespace aeoq

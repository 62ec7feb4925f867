// Block-scaled FP8 products of few activation rows: bound by the bytes of the
// weights, so they are streamed from HBM straight into registers, all of a
// warp's loads in flight at once, and multiplied there with mma.sync (a tile
// of tcgen05 would hold 128 rows for them and needs shared memory on the way;
// tensor throughput is no concern here).
//
// One warp holds 16 weight rows and every eighth block of 128 along K. In
// mma.m16n8k32 lane (g, t) = (lane / 4, lane % 4) feeds rows g and g + 8 of the
// weights and column g of the activations, each with two groups of four k
// values. Which k those are is free, as long as both operands agree: lane t
// takes bytes 32 t .. 32 t + 31 of the block, so its weights are two 16-byte
// loads per row, and its 32 activations are quantized where they are loaded,
// with the block's maximum two shuffles away. (The sum over a block is f32;
// e4m3 products are exact in it.)
//
// The eight warps' sums over K meet in shared memory.
#include <algorithm>
#include <cmath>

#include "fp8_block.cuh"

namespace aeoq {

constexpr int kSkWarps = 8, kSkThreads = 32 * kSkWarps;
constexpr int kSkAhead = 3;      // K blocks of a warp in flight

__device__ __forceinline__ void mma_e4m3(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A lane's 64 bytes of one block: 32 of row g and 32 of row g + 8.
struct SkWeights {
  uint4 a[2], b[2];
  // w0, w1: the two rows (null: zeros); k0: first byte of this lane's piece
  __device__ __forceinline__ void load(const uint8_t* w0, const uint8_t* w1, int64_t k0, int64_t K) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t k = k0 + 16 * i;
      a[i] = w0 && k < K ? ldg_stream(w0 + k) : make_uint4(0u, 0u, 0u, 0u);
      b[i] = w1 && k < K ? ldg_stream(w1 + k) : make_uint4(0u, 0u, 0u, 0u);
    }
  }
  // d = the block's 16 x 8 sums with the codes c[8] of this lane's column
  __device__ __forceinline__ void dot(float (&d)[4], const uint32_t (&c)[8]) const {
    d[0] = d[1] = d[2] = d[3] = 0.0f;
    const uint32_t* x = reinterpret_cast<const uint32_t*>(a);
    const uint32_t* y = reinterpret_cast<const uint32_t*>(b);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t f[4] = {x[2 * j], y[2 * j], x[2 * j + 1], y[2 * j + 1]};
      mma_e4m3(d, f, c[2 * j], c[2 * j + 1]);
    }
  }
};

// This lane's 32 values of column g in one block, quantized: codes and the
// block's scale. v: the lane's piece (null: zeros); n: values of it that exist
// (a multiple of 16); VEC: pieces are 16-byte aligned.
template <int DT, bool VEC>
__device__ __forceinline__ void sk_quantize(const typename In<DT>::T* v, int64_t n, uint32_t (&c)[8], float& scale) {
  FbEight<DT> e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (v && 8 * i < n) {
      if constexpr (VEC) e[i].load(v + 8 * i);
      else e[i].load_some(v + 8 * i, 8);
    } else {
      e[i].zero();
    }
  }
  uint32_t key = FbEight<DT>::key_max(FbEight<DT>::key_max(e[0].key(), e[1].key()),
                                      FbEight<DT>::key_max(e[2].key(), e[3].key()));
  key = FbEight<DT>::key_max(key, __shfl_xor_sync(0xFFFFFFFFu, key, 1));
  key = FbEight<DT>::key_max(key, __shfl_xor_sync(0xFFFFFFFFu, key, 2));
  const float2 s = fb_scales(FbEight<DT>::key_value(key));
  scale = s.y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint2 q = fb_codes8(e[i], s.x);
    c[2 * i] = q.x;
    c[2 * i + 1] = q.y;
  }
}

// Adds one block's sums with their scales: column 2 t of d[0], d[2] and 2 t + 1
// of d[1], d[3]; rows g (scale s0) and g + 8 (s1).
__device__ __forceinline__ void sk_add(float (&acc)[4], const float (&d)[4], float scale, float s0, float s1) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  const float x0 = __shfl_sync(0xFFFFFFFFu, scale, 8 * t), x1 = __shfl_sync(0xFFFFFFFFu, scale, 8 * t + 4);
  acc[0] = fmaf(d[0], x0 * s0, acc[0]);
  acc[1] = fmaf(d[1], x1 * s0, acc[1]);
  acc[2] = fmaf(d[2], x0 * s1, acc[2]);
  acc[3] = fmaf(d[3], x1 * s1, acc[3]);
}

// Sum over the warps of element (row, col) of their 16 x 8 sums.
__device__ __forceinline__ float sk_sum(const float (*part)[32][4], int row, int col) {
  const int lane = (row & 7) * 4 + (col >> 1), i = (row >> 3) * 2 + (col & 1);
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < kSkWarps; ++w) s += part[w][lane][i];
  return s;
}

// One warp's codes of a row of one block, four values per lane: written to
// `codes` (128 bytes) in shared memory, the scale returned to every lane.
__device__ __forceinline__ float sk_quantize_warp(const float (&v)[4], uint8_t* codes) {
  const int lane = threadIdx.x & 31;
  uint32_t key = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) key = max(key, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  key = __reduce_max_sync(0xFFFFFFFFu, key);
  const float2 s = fb_scales(__uint_as_float(key));
  reinterpret_cast<uint32_t*>(codes)[lane] = fb_codes4(v[0] * s.x, v[1] * s.x, v[2] * s.x, v[3] * s.x);
  return s.y;
}

// A lane's piece of a row's codes in shared memory, for every column alike.
__device__ __forceinline__ void sk_codes(const uint8_t* codes, uint32_t (&c)[8]) {
  const uint4* q = reinterpret_cast<const uint4*>(codes + 32 * (threadIdx.x & 3));
  const uint4 a = q[0], b = q[1];
  c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
  c[4] = b.x; c[5] = b.y; c[6] = b.z; c[7] = b.w;
}

// ------------------------------------------------------------------ linear
struct SkLinear {
  const void* x; int64_t ldx;          // M rows of the input ...
  const uint8_t* q; const float* qs;   // ... or their codes (M, K) and scales (M, KB)
  int64_t M, N, K;
  int KB;
  const uint8_t* w; const float* sw;
  const __nv_bfloat16* bias;
  void* out; int out_dt; int64_t ldc;
};

// CTA: 16 output columns, all M rows in NB groups of 8. QUANT: quantize x here
// (NB = 1); else read codes.
template <int DT, bool QUANT, bool VEC, int NB>
__global__ void __launch_bounds__(kSkThreads) sk_linear_kernel(const SkLinear p) {
  __shared__ float part[kSkWarps][32][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const uint8_t* w0 = n0 + g < p.N ? p.w + (n0 + g) * p.K : nullptr;
  const uint8_t* w1 = n0 + 8 + g < p.N ? p.w + (n0 + 8 + g) * p.K : nullptr;
  const float* sw = p.sw + (n0 / kFbBlock) * p.KB;     // 16 rows lie in one block row
  float acc[NB][4] = {};
  if (!QUANT && warp >= p.KB) pdl_wait();
  for (int kb0 = warp; kb0 < p.KB; kb0 += kSkWarps * kSkAhead) {
    SkWeights w[kSkAhead];
    float s[kSkAhead];
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const int kb = kb0 + u * kSkWarps;
      w[u].load(w0, w1, (int64_t)kb * kFbBlock + 32 * t, kb < p.KB ? p.K : 0);
      s[u] = kb < p.KB ? __ldg(sw + kb) : 0.0f;
    }
    // the codes come from a kernel that may still be running
    if (!QUANT && kb0 == warp) pdl_wait();
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const int kb = kb0 + u * kSkWarps;
      if (kb >= p.KB) break;
      const int64_t k0 = (int64_t)kb * kFbBlock + 32 * t;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (b && 8 * b >= p.M) break;
        const int64_t m = 8 * b + g;
        uint32_t c[8];
        float xs = 0.0f, d[4];
        if constexpr (QUANT) {
          const auto* x = reinterpret_cast<const typename In<DT>::T*>(p.x);
          sk_quantize<DT, VEC>(m < p.M ? x + m * p.ldx + k0 : nullptr, p.K - k0, c, xs);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool in = m < p.M && k0 + 16 * i < p.K;
            const uint4 v = in ? __ldcg(reinterpret_cast<const uint4*>(p.q + m * p.K + k0 + 16 * i))
                               : make_uint4(0u, 0u, 0u, 0u);
            c[4 * i] = v.x; c[4 * i + 1] = v.y; c[4 * i + 2] = v.z; c[4 * i + 3] = v.w;
          }
          xs = m < p.M ? __ldcg(p.qs + m * p.KB + kb) : 0.0f;
        }
        w[u].dot(d, c);
        sk_add(acc[b], d, xs, s[u], s[u]);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (b && 8 * b >= p.M) break;
    if (b) __syncthreads();
    *reinterpret_cast<float4*>(part[warp][lane]) = make_float4(acc[b][0], acc[b][1], acc[b][2], acc[b][3]);
    __syncthreads();
    const int row = threadIdx.x & 15, col = threadIdx.x >> 4;
    const int64_t n = n0 + row, m = 8 * b + col;
    if (threadIdx.x < 128 && n < p.N && m < p.M) {
      float y = sk_sum(part, row, col);
      if (p.bias) y += __bfloat162float(p.bias[n]);
      if (p.out_dt == AEOQ_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[m * p.ldc + n] = __float2bfloat16_rn(y);
      else reinterpret_cast<float*>(p.out)[m * p.ldc + n] = y;
    }
  }
}

// One row: as above, but a block of x is quantized by the whole warp, four
// values per lane, and every column of the MMA is that row (1 x 8192 x 8192:
// a lane of eight quantizing 32 values for itself took 28.7 us).
template <int DT, bool VEC, int NW>
__global__ void __launch_bounds__(32 * NW, 20 / NW) sk_row_kernel(const SkLinear p) {
  __shared__ float part[NW][16];
  __shared__ __align__(16) uint8_t codes[NW][kSkAhead][128];
  using Tp = typename In<DT>::T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const uint8_t* w0 = n0 + g < p.N ? p.w + (n0 + g) * p.K : nullptr;
  const uint8_t* w1 = n0 + 8 + g < p.N ? p.w + (n0 + 8 + g) * p.K : nullptr;
  const float* sw = p.sw + (n0 / kFbBlock) * p.KB;
  const Tp* x = reinterpret_cast<const Tp*>(p.x) + 4 * lane;
  float acc0 = 0.0f, acc1 = 0.0f;
  for (int kb0 = warp; kb0 < p.KB; kb0 += NW * kSkAhead) {
    SkWeights w[kSkAhead];
    float s[kSkAhead];
    __align__(16) Tp xv[kSkAhead][4];
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const int kb = kb0 + u * NW;
      const bool in = kb < p.KB;
      const Tp* xk = x + (int64_t)kb * kFbBlock;
#pragma unroll
      for (int i = 0; i < 4; ++i) xv[u][i] = Tp(0.0f);
      if (in && (int64_t)kb * kFbBlock + 4 * lane < p.K) {
        if constexpr (!VEC) {
#pragma unroll
          for (int i = 0; i < 4; ++i) xv[u][i] = xk[i];
        } else if constexpr (sizeof(Tp) == 2) {
          *reinterpret_cast<uint2*>(xv[u]) = __ldg(reinterpret_cast<const uint2*>(xk));
        } else {
          *reinterpret_cast<uint4*>(xv[u]) = __ldg(reinterpret_cast<const uint4*>(xk));
        }
      }
      w[u].load(w0, w1, (int64_t)kb * kFbBlock + 32 * t, in ? p.K : 0);
      s[u] = in ? __ldg(sw + kb) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const float v[4] = {In<DT>::to_f(xv[u][0]), In<DT>::to_f(xv[u][1]), In<DT>::to_f(xv[u][2]),
                          In<DT>::to_f(xv[u][3])};
      s[u] *= sk_quantize_warp(v, codes[warp][u]);
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      if (kb0 + u * NW >= p.KB) break;
      uint32_t c[8];
      float d[4];
      sk_codes(codes[warp][u], c);
      w[u].dot(d, c);
      acc0 = fmaf(d[0], s[u], acc0);
      acc1 = fmaf(d[2], s[u], acc1);
    }
    __syncwarp();
  }
  if (t == 0) {
    part[warp][g] = acc0;
    part[warp][g + 8] = acc1;
  }
  __syncthreads();
  const int64_t n = n0 + threadIdx.x;
  if (threadIdx.x < 16 && n < p.N) {
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) y += part[w][threadIdx.x];
    if (p.bias) y += __bfloat162float(p.bias[n]);
    if (p.out_dt == AEOQ_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[n] = __float2bfloat16_rn(y);
    else reinterpret_cast<float*>(p.out)[n] = y;
  }
}

template <int DT>
static int launch_row(const SkLinear& p, cudaStream_t st) {
  const bool vec = (uintptr_t)p.x % (4 * sizeof(typename In<DT>::T)) == 0;
  const unsigned grid = (unsigned)((p.N + 15) / 16);
  // eight warps share a row block's K while there are few of them
  if (grid <= 2u * (unsigned)device_sm_count()) {
    if (vec) sk_row_kernel<DT, true, 8><<<grid, 256, 0, st>>>(p);
    else sk_row_kernel<DT, false, 8><<<grid, 256, 0, st>>>(p);
  } else {
    if (vec) sk_row_kernel<DT, true, 4><<<grid, 128, 0, st>>>(p);
    else sk_row_kernel<DT, false, 4><<<grid, 128, 0, st>>>(p);
  }
  return check_launch("sk_row_kernel");
}

// Cold L2, against the tcgen05 kernel: 16 x 1408 x 2816 12.3 and 20.5 us, 48 x
// 2112 x 2816 18.4 and 20.5, but 32 x 8192 x 8192 67.6 and 36.9 (every CTA
// reads all of the codes), 16 x 8192 x 8192 36.9 and 36.9, 64 x 2816 x 704 18.5
// and 14.3.
bool fb_linear_skinny_takes(int64_t M, int64_t N, int64_t K) {
  return M <= 16 || (M <= 48 && N * K <= (1 << 23));
}

template <int DT>
static int launch_quant(const SkLinear& p, cudaStream_t st) {
  const bool vec = (uintptr_t)p.x % 16 == 0 && (p.ldx * (int64_t)sizeof(typename In<DT>::T)) % 16 == 0;
  const unsigned grid = (unsigned)((p.N + 15) / 16);
  if (vec) sk_linear_kernel<DT, true, true, 1><<<grid, kSkThreads, 0, st>>>(p);
  else sk_linear_kernel<DT, true, false, 1><<<grid, kSkThreads, 0, st>>>(p);
  return check_launch("sk_linear_kernel");
}

int fb_linear_skinny(const void* x, int dtype, int64_t ldx, int64_t M, const uint8_t* w, const float* sw, int64_t N,
                     int64_t K, const void* bias, void* out, int out_dt, int64_t ldc, uint8_t* q, float* qs,
                     cudaStream_t st) {
  SkLinear p{};
  p.x = x;
  p.ldx = ldx;
  p.M = M;
  p.N = N;
  p.K = K;
  p.KB = (int)fb_blocks(K);
  p.w = w;
  p.sw = sw;
  p.bias = reinterpret_cast<const __nv_bfloat16*>(bias);
  p.out = out;
  p.out_dt = out_dt;
  p.ldc = ldc;
  if (x && M == 1) {
    if (dtype == AEOQ_BF16) return launch_row<AEOQ_BF16>(p, st);
    if (dtype == AEOQ_F16) return launch_row<AEOQ_F16>(p, st);
    return launch_row<AEOQ_F32>(p, st);
  }
  if (x && M <= kFbSkinnyQuant) {
    if (dtype == AEOQ_BF16) return launch_quant<AEOQ_BF16>(p, st);
    if (dtype == AEOQ_F16) return launch_quant<AEOQ_F16>(p, st);
    return launch_quant<AEOQ_F32>(p, st);
  }
  if (x) {
    const int rc = fb_quantize_rows(x, dtype, M, K, ldx, q, K, qs, st);
    if (rc) return rc;
  }
  p.q = q;
  p.qs = qs;
  // With the quantizer just before it, the kernel starts while that runs and
  // requests its weights meanwhile.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((N + 15) / 16));
  cfg.blockDim = dim3(kSkThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = x ? 1 : 0;
  if (M <= 8) cudaLaunchKernelEx(&cfg, sk_linear_kernel<AEOQ_BF16, false, true, 1>, p);
  else if (M <= 16) cudaLaunchKernelEx(&cfg, sk_linear_kernel<AEOQ_BF16, false, true, 2>, p);
  else if (M <= 32) cudaLaunchKernelEx(&cfg, sk_linear_kernel<AEOQ_BF16, false, true, 4>, p);
  else cudaLaunchKernelEx(&cfg, sk_linear_kernel<AEOQ_BF16, false, true, 8>, p);
  return check_launch("sk_linear_kernel");
}

// ----------------------------------------------------------------- experts
struct SkExperts {
  const __nv_bfloat16* hidden;
  const void* ids; int ids_dt;
  const float* weights;
  int T, k, E, H, I, KBH, KBI;
  const uint8_t* gu; const float* gus; int64_t NBgu;
  const uint8_t* dw; const float* dws; int64_t NBd;
  int act;
  float* h;                 // (pairs, I)
  __nv_bfloat16* out;       // (T, H)
};

// h = act(gate x) * up x of one pair (token, slot). CTA (x, y): features 8 x ..
// 8 x + 7 (their gate rows are the MMA's rows 0-7, their up rows 8-15) of pair
// y. Four warps and few registers, so that the 88 x 8 CTAs of one token at I =
// 704 are all on the 148 SMs at once: a CTA's time is that of a chain of
// memory latencies, and with two CTAs of eight warps per SM it was paid in
// three waves (17.6 us).
constexpr int kSkGuWarps = 4;
__global__ void __launch_bounds__(32 * kSkGuWarps, 5) sk_gate_up_kernel(const SkExperts p) {
  __shared__ float part[kSkGuWarps][16];
  __shared__ __align__(16) uint8_t codes[kSkGuWarps][kSkAhead][128];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int y = blockIdx.y, f0 = blockIdx.x * 8;
  const int64_t e = load_index(p.ids, p.ids_dt, y);
  const __nv_bfloat16* x = p.hidden + (int64_t)(y / p.k) * p.H + 4 * lane;
  if (e < 0 || e >= p.E) return;
  const uint8_t* w0 = p.gu + (e * 2 * p.I + f0 + g) * p.H;
  const uint8_t* w1 = w0 + (int64_t)p.I * p.H;
  const float* s0 = p.gus + (e * p.NBgu + f0 / kFbBlock) * p.KBH;
  const float* s1 = p.gus + (e * p.NBgu + (p.I + f0) / kFbBlock) * p.KBH;
  float acc0 = 0.0f, acc1 = 0.0f;
  for (int kb0 = warp; kb0 < p.KBH; kb0 += kSkGuWarps * kSkAhead) {
    SkWeights w[kSkAhead];
    float sg[kSkAhead], su[kSkAhead], xs[kSkAhead];
    uint2 xv[kSkAhead];
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const int kb = kb0 + u * kSkGuWarps;
      const bool in = kb < p.KBH;
      xv[u] = in && kb * kFbBlock + 4 * lane < p.H ? __ldg(reinterpret_cast<const uint2*>(x + kb * kFbBlock))
                                                    : make_uint2(0u, 0u);
      w[u].load(w0, w1, kb * kFbBlock + 32 * t, in ? p.H : 0);
      sg[u] = in ? __ldg(s0 + kb) : 0.0f;
      su[u] = in ? __ldg(s1 + kb) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(&xv[u]);
      const float v[4] = {__bfloat162float(b[0]), __bfloat162float(b[1]), __bfloat162float(b[2]),
                          __bfloat162float(b[3])};
      xs[u] = sk_quantize_warp(v, codes[warp][u]);
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      if (kb0 + u * kSkGuWarps >= p.KBH) break;
      uint32_t c[8];
      float d[4];
      sk_codes(codes[warp][u], c);
      w[u].dot(d, c);
      acc0 = fmaf(d[0], xs[u] * sg[u], acc0);
      acc1 = fmaf(d[2], xs[u] * su[u], acc1);
    }
    __syncwarp();
  }
  if (t == 0) {                  // every column is the same
    part[warp][g] = acc0;
    part[warp][g + 8] = acc1;
  }
  __syncthreads();
  if (threadIdx.x < 8) {
    float gate = 0.0f, up = 0.0f;
#pragma unroll
    for (int w = 0; w < kSkGuWarps; ++w) {
      gate += part[w][threadIdx.x];
      up += part[w][threadIdx.x + 8];
    }
    p.h[(int64_t)y * p.I + f0 + threadIdx.x] = fb_act(fb_act_of(p.act), gate) * up;
  }
}

// out[t] = sum over slots of weight * down h. CTA (x, y): output columns 16 x ..
// + 15 of token y; warp w takes the slots w, w + 8, ... The weights of a warp's
// first slot are requested before the kernel that writes h is known to be
// done; h is quantized by each CTA for itself, a block per warp and step.
__global__ void __launch_bounds__(kSkThreads, 2) sk_down_kernel(const SkExperts p) {
  constexpr int U = 6;                   // K blocks in flight: all of them up to I = 768
  __shared__ float part[kSkWarps][16];
  __shared__ __align__(16) uint8_t codes[kSkWarps][U][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, y = blockIdx.y;
  float total0 = 0.0f, total1 = 0.0f;      // rows g and g + 8
  bool waited = false;
  for (int j = warp; j < p.k; j += kSkWarps) {
    const int pair = y * p.k + j;
    const int64_t e = load_index(p.ids, p.ids_dt, pair);
    if (e < 0 || e >= p.E) continue;
    const float weight = __ldg(p.weights + pair);
    const uint8_t* w0 = n0 + g < p.H ? p.dw + (e * p.H + n0 + g) * p.I : nullptr;
    const uint8_t* w1 = n0 + 8 + g < p.H ? p.dw + (e * p.H + n0 + 8 + g) * p.I : nullptr;
    const float* sd = p.dws + (e * p.NBd + n0 / kFbBlock) * p.KBI;
    const float* h = p.h + (int64_t)pair * p.I + 4 * lane;
    float acc0 = 0.0f, acc1 = 0.0f;
    for (int kb0 = 0; kb0 < p.KBI; kb0 += U) {
      SkWeights w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u].load(w0, w1, (kb0 + u) * kFbBlock + 32 * t, kb0 + u < p.KBI ? p.I : 0);
      // lane u keeps the weight scale of block u, then times h's
      float s = lane < U && kb0 + lane < p.KBI ? __ldg(sd + kb0 + lane) : 0.0f;
      if (!waited) {
        pdl_wait();
        waited = true;
      }
#pragma unroll
      for (int u0 = 0; u0 < U; u0 += 3) {
        float4 v[3];
#pragma unroll
        for (int u = 0; u < 3; ++u) {
          const int k = (kb0 + u0 + u) * kFbBlock;
          v[u] = k + 4 * lane < p.I ? __ldcg(reinterpret_cast<const float4*>(h + k)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < 3; ++u) {
          const float f[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
          const float hs = sk_quantize_warp(f, codes[warp][u0 + u]);
          if (lane == u0 + u) s *= hs;
        }
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t c[8];
        float d[4];
        sk_codes(codes[warp][u], c);
        w[u].dot(d, c);
        const float f = __shfl_sync(0xFFFFFFFFu, s, u);
        acc0 = fmaf(d[0], f, acc0);
        acc1 = fmaf(d[2], f, acc1);
      }
      __syncwarp();
    }
    total0 = fmaf(weight, acc0, total0);
    total1 = fmaf(weight, acc1, total1);
  }
  if (!waited) pdl_wait();
  if (t == 0) {
    part[warp][g] = total0;
    part[warp][g + 8] = total1;
  }
  __syncthreads();
  if (threadIdx.x < 16 && n0 + (int)threadIdx.x < p.H) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kSkWarps; ++w) s += part[w][threadIdx.x];
    p.out[(int64_t)y * p.H + n0 + threadIdx.x] = __float2bfloat16_rn(s);
  }
}

// Every pair reads its expert's weights here; the grouped GEMMs read each
// expert's once for 32 rows, but need five launches. So this form takes up to
// 64 pairs while what it reads more than once is under 45 MB, the experts in
// use being as many as with choices that are all equally likely. Measured for
// 1 to 128 experts, top 1 to 8, 1 to 64 pairs, three weights of H x I from 512
// x 128 to 4096 x 14336, cold and warm L2: of 316 such layers this takes the
// slower form by over 10% in five to seven (limits of 30 to 60 MB do worse). In us,
// here and grouped, cold: H = 2816, I = 704: 128 experts, top-8, one token 23
// and 43, 6 tokens 70 and 78, 8 tokens 88 and 95 (12 experts' weights, 74 MB,
// twice); 8 experts, top-2, 4 tokens 27 and 41, 8 tokens 39 and 43, 32 tokens
// 117 and 43; H = 4096, I = 14336, 8 experts, top-2: one token 102 and 131, two
// 188 and 174, 32 tokens 2519 and 250.
constexpr int64_t kSkMaxPairs = 64;
constexpr double kSkMaxReread = 45e6;
bool fb_experts_skinny_takes(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
  if (T > kSkMaxPairs || T * k > kSkMaxPairs) return false;
  const double used = (double)E * (1.0 - std::pow(std::max(0.0, 1.0 - (double)k / (double)E), (double)T));
  return ((double)(T * k) - used) * 3.0 * (double)H * (double)I <= kSkMaxReread;
}

// The most tokens up to T that the rule takes (with T it takes all fewer ones:
// a token adds k pairs and at most k experts in use).
int64_t fb_experts_skinny_most(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
  int64_t lo = 0, hi = std::min(T, kSkMaxPairs) + 1;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    (fb_experts_skinny_takes(mid, k, E, H, I) ? lo : hi) = mid;
  }
  return lo;
}

int fb_experts_skinny(const void* hidden, int64_t T, const void* ids, int ids_dt, const float* weights, int64_t k,
                      const uint8_t* gu, const float* gus, const uint8_t* dw, const float* dws, int64_t E, int64_t H,
                      int64_t I, int act, float* h, void* out, cudaStream_t st) {
  SkExperts p{};
  p.hidden = reinterpret_cast<const __nv_bfloat16*>(hidden);
  p.ids = ids;
  p.ids_dt = ids_dt;
  p.weights = weights;
  p.T = (int)T;
  p.k = (int)k;
  p.E = (int)E;
  p.H = (int)H;
  p.I = (int)I;
  p.KBH = (int)fb_blocks(H);
  p.KBI = (int)fb_blocks(I);
  p.gu = gu;
  p.gus = gus;
  p.NBgu = fb_blocks(2 * I);
  p.dw = dw;
  p.dws = dws;
  p.NBd = fb_blocks(H);
  p.act = act;
  p.h = h;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  sk_gate_up_kernel<<<dim3((unsigned)(I / 8), (unsigned)(T * k)), 32 * kSkGuWarps, 0, st>>>(p);
  int rc = check_launch("sk_gate_up_kernel");
  if (rc) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((H + 15) / 16), (unsigned)T);
  cfg.blockDim = dim3(kSkThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sk_down_kernel, p) != cudaSuccess) return check_launch("sk_down_kernel");
  return check_launch("sk_down_kernel");
}

}  // namespace aeoq

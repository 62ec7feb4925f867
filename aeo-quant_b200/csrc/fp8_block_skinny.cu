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
// (a multiple of 16). CG: the values come from a kernel that may still have
// been running when this one started, and are read past L1.
template <int DT, bool CG>
__device__ __forceinline__ void sk_quantize(const typename In<DT>::T* v, int64_t n, uint32_t (&c)[8], float& scale) {
  FbEight<DT> e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (v && 8 * i < n) {
      if constexpr (CG) {
        static_assert(!CG || DT == AEOQ_F32, "");
        e[i].a = __ldcg(reinterpret_cast<const float4*>(v + 8 * i));
        e[i].b = __ldcg(reinterpret_cast<const float4*>(v + 8 * i) + 1);
      } else {
        e[i].load(v + 8 * i);
      }
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
template <int DT, bool QUANT, int NB>
__global__ void __launch_bounds__(kSkThreads) sk_linear_kernel(const SkLinear p) {
  __shared__ float part[kSkWarps][32][4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const uint8_t* w0 = n0 + g < p.N ? p.w + (n0 + g) * p.K : nullptr;
  const uint8_t* w1 = n0 + 8 + g < p.N ? p.w + (n0 + 8 + g) * p.K : nullptr;
  const float* sw = p.sw + (n0 / kFbBlock) * p.KB;     // 16 rows lie in one block row
  float acc[NB][4] = {};
  for (int kb0 = warp; kb0 < p.KB; kb0 += kSkWarps * kSkAhead) {
    SkWeights w[kSkAhead];
    float s[kSkAhead];
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const int kb = kb0 + u * kSkWarps;
      w[u].load(w0, w1, (int64_t)kb * kFbBlock + 32 * t, kb < p.KB ? p.K : 0);
      s[u] = kb < p.KB ? __ldg(sw + kb) : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < kSkAhead; ++u) {
      const int kb = kb0 + u * kSkWarps;
      if (kb >= p.KB) break;
      const int64_t k0 = (int64_t)kb * kFbBlock + 32 * t;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int64_t m = 8 * b + g;
        uint32_t c[8];
        float xs = 0.0f, d[4];
        if constexpr (QUANT) {
          const auto* x = reinterpret_cast<const typename In<DT>::T*>(p.x);
          sk_quantize<DT, false>(m < p.M ? x + m * p.ldx + k0 : nullptr, p.K - k0, c, xs);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const bool in = m < p.M && k0 + 16 * i < p.K;
            const uint4 v = in ? __ldg(reinterpret_cast<const uint4*>(p.q + m * p.K + k0 + 16 * i))
                               : make_uint4(0u, 0u, 0u, 0u);
            c[4 * i] = v.x; c[4 * i + 1] = v.y; c[4 * i + 2] = v.z; c[4 * i + 3] = v.w;
          }
          xs = m < p.M ? __ldg(p.qs + m * p.KB + kb) : 0.0f;
        }
        w[u].dot(d, c);
        sk_add(acc[b], d, xs, s[u], s[u]);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
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

bool fb_linear_skinny_takes(int64_t M, int64_t N, int64_t K) { return M <= kFbSkinnyRows; }

template <int DT>
static int launch_quant(const SkLinear& p, cudaStream_t st) {
  sk_linear_kernel<DT, true, 1><<<(unsigned)((p.N + 15) / 16), kSkThreads, 0, st>>>(p);
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
  const int es = dtype == AEOQ_F32 ? 4 : 2;
  if (x && M <= 8 && (uintptr_t)x % 16 == 0 && (ldx * es) % 16 == 0) {
    if (dtype == AEOQ_BF16) return launch_quant<AEOQ_BF16>(p, st);
    if (dtype == AEOQ_F16) return launch_quant<AEOQ_F16>(p, st);
    return launch_quant<AEOQ_F32>(p, st);
  }
  if (x) {
    const int rc = fb_quantize_rows(x, dtype, M, K, ldx, nullptr, nullptr, q, K, qs, st);
    if (rc) return rc;
  }
  p.q = q;
  p.qs = qs;
  const unsigned grid = (unsigned)((N + 15) / 16);
  if (M <= 8) sk_linear_kernel<AEOQ_BF16, false, 1><<<grid, kSkThreads, 0, st>>>(p);
  else if (M <= 16) sk_linear_kernel<AEOQ_BF16, false, 2><<<grid, kSkThreads, 0, st>>>(p);
  else if (M <= 32) sk_linear_kernel<AEOQ_BF16, false, 4><<<grid, kSkThreads, 0, st>>>(p);
  else sk_linear_kernel<AEOQ_BF16, false, 8><<<grid, kSkThreads, 0, st>>>(p);
  return check_launch("sk_linear_kernel");
}

// ----------------------------------------------------------------- experts
constexpr int kSkMaxPairs = 512;

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

// h = act(gate x) * up x for the pairs (token, slot) of one expert. CTA (x, y):
// features 8 x .. 8 x + 7 (their gate rows are the MMA's rows 0-7, their up rows
// 8-15) of the expert of pair y, if y is the first pair with it: an expert's
// weights are read once for all its tokens, eight at a time.
__global__ void __launch_bounds__(kSkThreads) sk_gate_up_kernel(const SkExperts p) {
  __shared__ float part[kSkWarps][32][4];
  __shared__ int list[kSkMaxPairs];
  __shared__ int n_list;
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int P = p.T * p.k, y = blockIdx.y;
  const int64_t e = load_index(p.ids, p.ids_dt, y);
  if (threadIdx.x == 0) n_list = 0;
  bool seen = e < 0 || e >= p.E;
  for (int i = threadIdx.x; i < y; i += kSkThreads) seen |= load_index(p.ids, p.ids_dt, i) == e;
  if (__syncthreads_or(seen)) return;
  for (int i = y + threadIdx.x; i < P; i += kSkThreads)
    if (load_index(p.ids, p.ids_dt, i) == e) list[atomicAdd(&n_list, 1)] = i;
  __syncthreads();
  const int n = n_list, f0 = blockIdx.x * 8;
  const int64_t rows = e * 2 * p.I;
  const uint8_t* w0 = p.gu + (rows + f0 + g) * p.H;
  const uint8_t* w1 = w0 + (int64_t)p.I * p.H;
  const float* s0 = p.gus + (e * p.NBgu + f0 / kFbBlock) * p.KBH;
  const float* s1 = p.gus + (e * p.NBgu + (p.I + f0) / kFbBlock) * p.KBH;
  for (int b = 0; b < n; b += 8) {
    const int pair = b + g < n ? list[b + g] : -1;
    const __nv_bfloat16* x = pair >= 0 ? p.hidden + (int64_t)(pair / p.k) * p.H + 32 * t : nullptr;
    float acc[4] = {};
    for (int kb0 = warp; kb0 < p.KBH; kb0 += kSkWarps * kSkAhead) {
      SkWeights w[kSkAhead];
      float sg[kSkAhead], su[kSkAhead];
#pragma unroll
      for (int u = 0; u < kSkAhead; ++u) {
        const int kb = kb0 + u * kSkWarps;
        w[u].load(w0, w1, kb * kFbBlock + 32 * t, kb < p.KBH ? p.H : 0);
        sg[u] = kb < p.KBH ? __ldg(s0 + kb) : 0.0f;
        su[u] = kb < p.KBH ? __ldg(s1 + kb) : 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kSkAhead; ++u) {
        const int kb = kb0 + u * kSkWarps;
        if (kb >= p.KBH) break;
        uint32_t c[8];
        float xs, d[4];
        sk_quantize<AEOQ_BF16, false>(x ? x + kb * kFbBlock : nullptr, p.H - kb * kFbBlock - 32 * t, c, xs);
        w[u].dot(d, c);
        sk_add(acc, d, xs, sg[u], su[u]);
      }
    }
    if (b) __syncthreads();
    *reinterpret_cast<float4*>(part[warp][lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    const int row = threadIdx.x & 7, col = threadIdx.x >> 3;
    if (threadIdx.x < 64 && b + col < n)
      p.h[(int64_t)list[b + col] * p.I + f0 + row] = fb_act(p.act, sk_sum(part, row, col)) * sk_sum(part, row + 8, col);
  }
}

// out[t] = sum over slots of weight * down h. CTA (x, y): output columns 16 x ..
// + 15 of token y; warp w takes the slots w, w + 8, .. (one token: the MMA's
// other seven columns are zeros). The weights of a warp's first slot are
// requested before the kernel that writes h is known to be done.
__global__ void __launch_bounds__(kSkThreads) sk_down_kernel(const SkExperts p) {
  __shared__ float part[kSkWarps][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16, y = blockIdx.y;
  float total0 = 0.0f, total1 = 0.0f;      // rows g and g + 8 (valid in lanes t = 0)
  bool waited = false;
  for (int j = warp; j < p.k; j += kSkWarps) {
    const int pair = y * p.k + j;
    const int64_t e = load_index(p.ids, p.ids_dt, pair);
    if (e < 0 || e >= p.E) continue;
    const float weight = __ldg(p.weights + pair);
    const uint8_t* w0 = n0 + g < p.H ? p.dw + (e * p.H + n0 + g) * p.I : nullptr;
    const uint8_t* w1 = n0 + 8 + g < p.H ? p.dw + (e * p.H + n0 + 8 + g) * p.I : nullptr;
    const float* sd = p.dws + (e * p.NBd + n0 / kFbBlock) * p.KBI;
    const float* h = g == 0 ? p.h + (int64_t)pair * p.I + 32 * t : nullptr;
    float acc[4] = {};
    constexpr int U = 6;                   // K blocks in flight: all of them up to I = 768
    for (int kb0 = 0; kb0 < p.KBI; kb0 += U) {
      SkWeights w[U];
      float s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kb = kb0 + u;
        w[u].load(w0, w1, kb * kFbBlock + 32 * t, kb < p.KBI ? p.I : 0);
        s[u] = kb < p.KBI ? __ldg(sd + kb) : 0.0f;
      }
      if (!waited) {
        pdl_wait();
        waited = true;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int kb = kb0 + u;
        if (kb >= p.KBI) break;
        uint32_t c[8];
        float hs, d[4];
        sk_quantize<AEOQ_F32, true>(h ? h + kb * kFbBlock : nullptr, p.I - kb * kFbBlock - 32 * t, c, hs);
        w[u].dot(d, c);
        sk_add(acc, d, hs, s[u], s[u]);
      }
    }
    total0 = fmaf(weight, acc[0], total0);
    total1 = fmaf(weight, acc[2], total1);
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

bool fb_experts_skinny_takes(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
  return T * k <= kSkMaxPairs && T * k <= 4 * E && T <= 64;
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
  sk_gate_up_kernel<<<dim3((unsigned)(I / 8), (unsigned)(T * k)), kSkThreads, 0, st>>>(p);
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

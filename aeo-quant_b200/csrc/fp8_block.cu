// Block-scaled FP8 quantizers (formulas in fp8_block.cuh).
//
// Rows: a half-warp holds one block of 128 values, 8 per lane, in registers:
// one 16-byte load (two for f32), four shuffles for the maximum, one 8-byte
// store of codes. Weights: one CTA holds a 128 x 128 block in registers.
// Every input value is read once, so both are bound by HBM.
#include <algorithm>

#include "fp8_block.cuh"

namespace aeoq {

constexpr int kFbRowWarps = 8;

// One warp per row and run of `chunk` blocks (an even number, or all). VEC:
// rows, their pieces of 8 and the code rows are aligned for wide accesses and
// K % 8 == 0. `to` (VEC only): instead of to row r the codes and scales of row
// r go to rows to[r * k] .. to[r * k + k - 1], those that are not negative.
//
// U pairs of blocks at a time, a block per half-warp. EDGE: a block may be
// short or past the end. With VEC that is the last pair alone, so that the
// loop over the others has no tests in it (32768 x 2816 of bf16 with tests in
// all of it: 52.9 us, issuing 70% of the time; so: 49.6).
template <int DT, bool VEC, bool SCATTER, int U, bool EDGE>
__device__ __forceinline__ void fb_row_blocks(const typename In<DT>::T* xr, int K, int nb, int b0, int b_end,
                                              uint8_t* q, int64_t q_ld, float* scale, int64_t r, const int* to,
                                              int k) {
  const int lane = threadIdx.x & 31, sub = lane & 15, half = lane >> 4;
  const int first = (b0 + half) * kFbBlock + 8 * sub;      // this lane's piece of pair u: + 256 u
  FbEight<DT> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!EDGE) {
      v[u].load(xr + first + 256 * u);
    } else if (b0 + 2 * u + half < b_end && first + 256 * u < K) {
      if (VEC) v[u].load(xr + first + 256 * u);
      else v[u].load_some(xr + first + 256 * u, K - first - 256 * u);
    } else {
      v[u].zero();
    }
  }
  uint32_t key[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    key[u] = v[u].key();
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) key[u] = FbEight<DT>::key_max(key[u], __shfl_xor_sync(0xFFFFFFFFu, key[u], o));
  }
  // the two divisions of pair u's blocks in lanes u, u + 4, .. of their
  // half-warp alone
  uint32_t mine = key[0];
#pragma unroll
  for (int u = 1; u < U; ++u) mine = (sub & 3) == u ? key[u] : mine;
  const float2 s = fb_scales(FbEight<DT>::key_value(mine));
  const int b = b0 + 2 * sub + half;
  if (sub < U && (!EDGE || b < b_end)) {
    if constexpr (SCATTER) {
      for (int j = 0; j < k; ++j) {
        const int d = __ldg(to + r * k + j);
        if (d >= 0) scale[(int64_t)d * nb + b] = s.y;
      }
    } else {
      scale[r * nb + b] = s.y;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float inv = __shfl_sync(0xFFFFFFFFu, s.x, (lane & 16) | u);
    const int k0 = first + 256 * u;
    if (EDGE && (b0 + 2 * u + half >= b_end || k0 >= K)) continue;
    const uint2 c = fb_codes8(v[u], inv);
    if constexpr (SCATTER) {
      for (int j = 0; j < k; ++j) {
        const int d = __ldg(to + r * k + j);
        if (d >= 0) *reinterpret_cast<uint2*>(q + (int64_t)d * q_ld + k0) = c;
      }
    } else if constexpr (VEC) {
      *reinterpret_cast<uint2*>(q + r * q_ld + k0) = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k0 + i < K) q[r * q_ld + k0 + i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
  }
}

template <int DT, bool VEC, bool SCATTER>
__global__ void __launch_bounds__(32 * kFbRowWarps) fb_rows_kernel(
    const typename In<DT>::T* __restrict__ x, int64_t rows, int K, int64_t ld, int chunk, uint8_t* __restrict__ q,
    int64_t q_ld, float* __restrict__ scale, const int* __restrict__ to, int k) {
  pdl_trigger();      // a dependent that asked for it may start its own loads
  const int64_t r = blockIdx.x * (int64_t)kFbRowWarps + (threadIdx.x >> 5);
  if (r >= rows) return;
  const typename In<DT>::T* xr = x + r * ld;
  const int nb = (K + kFbBlock - 1) / kFbBlock;
  const int b_end = min(nb, ((int)blockIdx.y + 1) * chunk);
  const int whole = VEC ? min(b_end, K / kFbBlock) : 0;      // blocks before the first that needs tests
  int b = (int)blockIdx.y * chunk;
  for (; b + 8 <= whole; b += 8) fb_row_blocks<DT, VEC, SCATTER, 4, false>(xr, K, nb, b, b_end, q, q_ld, scale, r, to, k);
  if (b + 4 <= whole) {
    fb_row_blocks<DT, VEC, SCATTER, 2, false>(xr, K, nb, b, b_end, q, q_ld, scale, r, to, k);
    b += 4;
  }
  constexpr int kEdge = VEC ? 1 : 4;
  for (; b < b_end; b += 2 * kEdge)
    fb_row_blocks<DT, VEC, SCATTER, kEdge, true>(xr, K, nb, b, b_end, q, q_ld, scale, r, to, k);
}

// One 128 x 128 block per CTA: thread t holds columns 8 (t % 16) .. + 7 of
// rows t / 16 + 16 i.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) fb_weights_kernel(const typename In<DT>::T* __restrict__ x, int64_t N,
                                                         int64_t K, uint8_t* __restrict__ q,
                                                         float* __restrict__ scale) {
  __shared__ uint32_t part[8];
  const int64_t e = blockIdx.z, nb = blockIdx.y, kb = blockIdx.x;
  const int64_t k0 = kb * kFbBlock + 8 * (threadIdx.x & 15);
  const int64_t n0 = nb * kFbBlock + (threadIdx.x >> 4);
  const typename In<DT>::T* xe = x + e * N * K;
  FbEight<DT> v[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t n = n0 + 16 * r;
    if (n < N && k0 < K) {
      if (VEC) v[r].load(xe + n * K + k0);
      else v[r].load_some(xe + n * K + k0, K - k0);
    } else {
      v[r].zero();
    }
  }
  uint32_t key = v[0].key();
#pragma unroll
  for (int r = 1; r < 8; ++r) key = FbEight<DT>::key_max(key, v[r].key());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) key = FbEight<DT>::key_max(key, __shfl_xor_sync(0xFFFFFFFFu, key, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = key;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) key = FbEight<DT>::key_max(key, part[i]);
  const float2 s = fb_scales(FbEight<DT>::key_value(key));
  if (threadIdx.x == 0) scale[(e * gridDim.y + nb) * gridDim.x + kb] = s.y;
  uint8_t* qe = q + e * N * K;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int64_t n = n0 + 16 * r;
    if (n >= N || k0 >= K) continue;
    const uint2 c = fb_codes8(v[r], s.x);
    if (VEC) {
      *reinterpret_cast<uint2*>(qe + n * K + k0) = c;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k0 + i < K) qe[n * K + k0 + i] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
  }
}

template <int DT>
static int launch_rows(const void* x, int64_t rows, int64_t K, int64_t ld, uint8_t* q,
                       int64_t q_ld, float* scale, cudaStream_t st) {
  using T = typename In<DT>::T;
  const bool vec = K % 8 == 0 && (uintptr_t)x % 16 == 0 && (ld * (int64_t)sizeof(T)) % 16 == 0 &&
                   (uintptr_t)q % 8 == 0 && q_ld % 8 == 0;
  const int64_t nb = fb_blocks(K);
  // Few rows: split a row over warps until the GPU has some, in runs of
  // whole iterations (8 blocks), then of 2 blocks.
  const int64_t groups = (rows + kFbRowWarps - 1) / kFbRowWarps;
  int64_t chunk = nb + (nb & 1);
  if (groups * 2 <= device_sm_count()) chunk = groups * ((nb + 7) / 8) >= device_sm_count() ? 8 : 2;
  dim3 grid((unsigned)groups, (unsigned)((nb + chunk - 1) / chunk));
  if (vec)
    fb_rows_kernel<DT, true, false><<<grid, 32 * kFbRowWarps, 0, st>>>(reinterpret_cast<const T*>(x), rows, (int)K, ld,
                                                                (int)chunk, q, q_ld, scale, nullptr, 0);
  else
    fb_rows_kernel<DT, false, false><<<grid, 32 * kFbRowWarps, 0, st>>>(reinterpret_cast<const T*>(x), rows, (int)K, ld,
                                                                 (int)chunk, q, q_ld, scale, nullptr, 0);
  return check_launch("fb_rows_kernel");
}

int fb_quantize_rows(const void* x, int dtype, int64_t rows, int64_t K, int64_t ld, uint8_t* q, int64_t q_ld,
                     float* scale, cudaStream_t st) {
  switch (dtype) {
    case AEOQ_BF16: return launch_rows<AEOQ_BF16>(x, rows, K, ld, q, q_ld, scale, st);
    case AEOQ_F16: return launch_rows<AEOQ_F16>(x, rows, K, ld, q, q_ld, scale, st);
    case AEOQ_F32: return launch_rows<AEOQ_F32>(x, rows, K, ld, q, q_ld, scale, st);
  }
  return set_error(AEOQ_ERR_INVALID, "fp8_block_quantize_rows: unsupported dtype %d", dtype);
}

int fb_quantize_rows_to(const void* x, int64_t rows, int64_t K, const int* to, int k, uint8_t* q, float* scale,
                        cudaStream_t st) {
  const int64_t groups = (rows + kFbRowWarps - 1) / kFbRowWarps;
  fb_rows_kernel<AEOQ_BF16, true, true><<<dim3((unsigned)groups, 1), 32 * kFbRowWarps, 0, st>>>(
      reinterpret_cast<const __nv_bfloat16*>(x), rows, (int)K, K, (int)fb_blocks(K), q, K, scale, to, k);
  return check_launch("fb_rows_kernel");
}

template <int DT>
static int launch_weights(const void* x, int64_t E, int64_t N, int64_t K, uint8_t* q, float* scale, cudaStream_t st) {
  using T = typename In<DT>::T;
  const bool vec = K % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)q % 8 == 0;
  dim3 grid((unsigned)fb_blocks(K), (unsigned)fb_blocks(N), (unsigned)E);
  if (vec)
    fb_weights_kernel<DT, true><<<grid, 256, 0, st>>>(reinterpret_cast<const T*>(x), N, K, q, scale);
  else
    fb_weights_kernel<DT, false><<<grid, 256, 0, st>>>(reinterpret_cast<const T*>(x), N, K, q, scale);
  return check_launch("fb_weights_kernel");
}

}  // namespace aeoq

using namespace aeoq;

extern "C" int aeoq_fp8_block_quantize_rows(const void* x, int dtype, int64_t rows, int64_t K, int64_t ld, uint8_t* q,
                                            int64_t q_ld, float* scale, void* stream) {
  AEOQ_REQUIRE(dtype == AEOQ_BF16 || dtype == AEOQ_F16 || dtype == AEOQ_F32, AEOQ_ERR_INVALID,
               "fp8_block_quantize_rows: unsupported dtype %d", dtype);
  AEOQ_REQUIRE(rows >= 0 && K >= 0 && ld >= K && q_ld >= K, AEOQ_ERR_INVALID, "fp8_block_quantize_rows: bad shape");
  AEOQ_REQUIRE(K <= (1LL << 24) && rows <= (1LL << 33), AEOQ_ERR_INVALID,
               "fp8_block_quantize_rows: K at most 2^24, rows at most 2^33");
  if (rows == 0 || K == 0) return AEOQ_OK;
  AEOQ_REQUIRE(x && q && scale, AEOQ_ERR_INVALID, "fp8_block_quantize_rows: null pointer");
  return fb_quantize_rows(x, dtype, rows, K, ld, q, q_ld, scale, (cudaStream_t)stream);
}

extern "C" int aeoq_fp8_block_quantize_weights(const void* x, int dtype, int64_t num_experts, int64_t N, int64_t K,
                                               uint8_t* q, float* scale, void* stream) {
  AEOQ_REQUIRE(num_experts >= 0 && N >= 0 && K >= 0, AEOQ_ERR_INVALID, "fp8_block_quantize_weights: bad shape");
  AEOQ_REQUIRE(num_experts <= 65535 && fb_blocks(N) <= 65535 && K <= (1LL << 31), AEOQ_ERR_INVALID,
               "fp8_block_quantize_weights: at most 65535 matrices of 65535 x 128 rows");
  if (num_experts == 0 || N == 0 || K == 0) return AEOQ_OK;
  AEOQ_REQUIRE(x && q && scale, AEOQ_ERR_INVALID, "fp8_block_quantize_weights: null pointer");
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AEOQ_BF16: return launch_weights<AEOQ_BF16>(x, num_experts, N, K, q, scale, st);
    case AEOQ_F16: return launch_weights<AEOQ_F16>(x, num_experts, N, K, q, scale, st);
    case AEOQ_F32: return launch_weights<AEOQ_F32>(x, num_experts, N, K, q, scale, st);
  }
  return set_error(AEOQ_ERR_INVALID, "fp8_block_quantize_weights: unsupported dtype %d", dtype);
}

// Block-scaled FP8 GEMMs on the 5th-generation tensor cores (tcgen05), and
// the routed experts' forward built on them.
//
//   y[m][n] = sum_b sa[m][b] * sw[n / 128][b] * ( sum_{k in block b} a[m][k] w[n][k] )
//
// a: e4m3 rows (tokens), w: e4m3 rows (output features), one f32 scale per
// 128 values of a row of a and per 128 x 128 block of w.
//
// The tensor core sums one block b (four MMAs of K = 32) into TMEM; the
// epilogue warps read that partial sum, multiply it by its two scales and
// add it to f32 sums in registers. The blocks alternate between two TMEM
// buffers, so the scaling of block b runs under the MMAs of block b + 1.
// Tokens are the MMA's 128 rows: a TMEM lane is a token and a thread owns
// one token, so its scale sa is one value per block and sw is the same for a
// whole run of columns: the scaling is one f32 fma per sum.
//
//   warp 0      TMA: per 128-wide K step one tile of a and one of w
//               (128-byte swizzle)
//   warps 1-2   MMA issuers (warp 1 owns the TMEM)
//   warps 4-11  scaling and epilogue: two warps per TMEM lane quadrant, each
//               with half of the columns (128 f32 sums per thread; setmaxnreg
//               gives them registers of warps 0-3)
//
// One CTA per SM walks the tiles, output features fastest (they share the
// tile of a in L2).
//
// What bounds it (18944 x 2560, bf16 out, ten tiles of 256 columns per CTA):
// about 1050 cycles per K step and 5000 per tile, at 1965 MHz; 32768 x 1408 x
// 2816 takes 150 us. The MMAs of a step are 512 cycles, its operands' 48 KB
// are written to shared memory and read from it once (768 cycles at 128 bytes
// a cycle), and 843 cycles remain when the sums and the TMEM reads are left
// out, so the sums hide under the MMAs but for about 200. A tile's 5000 are
// its conversion and store (2200), and the first scales and the restart of
// the pipeline. Handing each column half over by itself took 154 us, requesting
// the next tile's scales a tile ahead 161 (registers).
//
// Epilogues: store (bf16 or f32, optional bias); GLU: the tile holds 128
// gate columns and the 128 up columns they pair with, h = act(g) * u is
// quantized per 128 in the epilogue and written as the next GEMM's operand.
#include <algorithm>

#include "fp8_block.cuh"
#include "sm100.cuh"

namespace aeoq {

int make_tmap_bytes(CUtensorMap* m, const void* ptr, int64_t rows, int64_t row_bytes, int64_t ld, int box_bytes,
                    int box_rows, bool swizzle128);

constexpr int kFbEpiWarps = 8;
constexpr int kFbThreads = 128 + 32 * kFbEpiWarps;
// Registers per thread after the split: 128 x 56 + 256 x 224 = 64512, what
// the block is launched with (384 x 168).
constexpr int kFbRegsLow = 56, kFbRegsHigh = 224;
constexpr int kFbMaxStages = 8;
constexpr int kFbMaxExperts = 1024;

enum FbEpilogue : int { kFbStore = 0, kFbGlu = 1 };

struct FbParams {
  int64_t M;              // rows of a (dense), or the most there can be (grouped)
  int64_t N;              // rows of w per expert
  int K, KB;              // K and its blocks
  int64_t NB;             // scale rows per expert, ceil(N / 128)
  int E;
  const float* sa;        // (rows of a, KB): a row's scales share lines that stay in L1 for several K
                          // steps (the other order, 8192 x 8192 x 8192: 689 against 521 us)
  const float* sw;        // (E, NB, KB)
  const int* row_src;     // few rows, GLU: sorted row r is row row_src[r] of a (a token's)
  const int* grp_off;     // grouped: rows [grp_off[e], grp_off[e + 1]) are expert e's; null: dense
  const int* tile_off;    // grouped: row tiles before expert e's, E + 1 values
  int64_t tiles_m;        // dense
  int tiles_n;
  void* out; int out_dt; int64_t ldc;   // store: row stride in elements
  const __nv_bfloat16* bias;            // store: N values or null
  bool out_tma;           // whole tiles may leave by TMA
  int64_t I;              // GLU: gate rows are w rows [0, I), up rows [I, 2 I)
  int act;
  uint8_t* hq; int64_t hq_ld;           // GLU: quantized h rows
  float* hs; int64_t hs_ld;             // GLU: their scales, (rows, ceil(I / 128))
  int* err;
};

template <int BN, int EPI>
struct FbLayout {
  static constexpr uint32_t kA = 128 * 128, kB = BN * 128, kStage = kA + kB;
  // the tile on its way out as bf16 (store epilogue)
  static constexpr uint32_t kOut = EPI == kFbStore ? 128 * BN * 2 : 0;
  struct Ctl {
    uint64_t full[kFbMaxStages], empty[kFbMaxStages];
    uint64_t acc_full[2], acc_empty[2];
    uint32_t tmem_base;
    float amax[2][128];                // GLU: the two column halves' maxima per row
    int tile_off[kFbMaxExperts + 1];
  };
  static constexpr int kStages =
      std::min<int>(kFbMaxStages, (227 * 1024 - 1024 - (int)sizeof(Ctl) - (int)kOut) / (int)kStage);
  static_assert(kStages >= 3, "the ring needs three stages");
  static constexpr size_t kBytes = 1024 + (size_t)kStages * kStage + kOut + sizeof(Ctl);
  static constexpr uint32_t kTmemCols = 2 * BN;
};

struct FbTile {
  int64_t expert, row0, n0;   // first row of a, first column (GLU: first gate column)
  int rows;                   // valid rows
};

// Row and column tile of tile number t. Columns go fastest; where the last
// column of tiles is short (`half_last`: no second column half) its tiles,
// which take half as long, come after all others, so that they fill the
// CTAs' uneven ends.
__device__ __forceinline__ int2 fb_place(int t, int tiles_m, int tiles_n, bool half_last) {
  const int wide = tiles_n - (int)half_last, n_wide = tiles_m * wide;
  if (t >= n_wide) return make_int2(t - n_wide, tiles_n - 1);
  const int mt = t / wide;
  return make_int2(mt, t - mt * wide);
}

template <int BN, int EPI>
__device__ __forceinline__ FbTile fb_tile(const FbParams& p, const int* tile_off, int2 at) {
  FbTile r;
  const int mt = at.x;
  r.n0 = (int64_t)at.y * (EPI == kFbGlu ? BN / 2 : BN);
  if (!p.grp_off) {
    r.expert = 0;
    r.row0 = (int64_t)mt * 128;
    r.rows = (int)min((int64_t)128, p.M - r.row0);
    return r;
  }
  int lo = 0, hi = p.E;       // the expert e with tile_off[e] <= mt < tile_off[e + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tile_off[mid] <= mt) lo = mid; else hi = mid;
  }
  r.expert = lo;
  const int g0 = __ldg(p.grp_off + lo), g1 = __ldg(p.grp_off + lo + 1);
  r.row0 = g0 + (mt - tile_off[lo]) * 128;
  r.rows = min(128, g1 - (int)r.row0);
  return r;
}

// ---------------------------------------------------------------- epilogues
// One thread's row of a tile's column half. `row` is the thread's row in its
// 128-row tile; four warps hold one half.

// Store of a whole 128-row tile's kCols bf16 columns from cur.n0 + kCols *
// half on: through shared memory (a thread's row in pieces of 16 bytes, placed
// so that 8 lanes fill 8 different bank groups) and one TMA store per 64
// columns, which stops at row M and column N by itself. Stored directly, the
// 32 rows of a warp's store are 32 half sectors: 53 us of 211 at M = 32768, N
// = 1408, K = 2816. The kernel gives a stage of its ring for the room (with
// half of it, used twice, the second half waits for the first: 161 us
// against 145).
template <int kCols>
__device__ __forceinline__ void fb_store_tile(const FbParams& p, const CUtensorMap& tmO, const FbTile& cur,
                                              uint8_t* box, const float (&acc)[kCols], int row, int half) {
  const int64_t n0 = cur.n0 + half * kCols;
#pragma unroll
  for (int i = 0; i < kCols / 8; ++i) {
    __align__(16) __nv_bfloat162 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __floats2bfloat162_rn(acc[8 * i + 2 * j], acc[8 * i + 2 * j + 1]);
    *reinterpret_cast<uint4*>(box + (i / 8) * 16384 + row * 128 + (((i & 7) ^ (row & 7)) << 4)) =
        *reinterpret_cast<const uint4*>(v);
  }
  sm100::fence_proxy_async_smem();
  asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
  if (row == 0) {
#pragma unroll
    for (int x = 0; x < kCols / 64; ++x)
      if (n0 + 64 * x < p.N)
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                         reinterpret_cast<uint64_t>(&tmO)),
                     "r"((int)((n0 + 64 * x) * 2)), "r"((int)cur.row0), "r"(sm100::smem_u32(box + x * 16384))
                     : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}

// f32 (the experts' outputs among them: behind a short tile lie another
// expert's rows) and rows that are not 16-byte aligned, rows and columns left
// out one by one: each
// warp turns its 32 rows around in 4 KB of shared memory, 128 bytes of a row
// at a time, so that a store instruction writes four whole lines.
template <class T, int kCols>
__device__ __forceinline__ void fb_store_rows(const FbParams& p, const FbTile& cur, uint8_t* box,
                                              const float (&acc)[kCols], int q, int half) {
  constexpr int kPer = 16 / (int)sizeof(T), kRound = 8 * kPer;     // columns per piece, per round
  const int lane = threadIdx.x & 31;
  const int64_t n0 = cur.n0 + half * kCols;
  const bool wide = p.ldc % kPer == 0 && (uintptr_t)p.out % 16 == 0;
  const int sub = lane >> 3, ch = lane & 7;
  T* out = reinterpret_cast<T*>(p.out) + (cur.row0 + 32 * q + sub) * p.ldc + n0 + ch * kPer;
  const int rows = cur.rows - 32 * q - sub;                        // row 4 j exists if 4 j < rows
#pragma unroll
  for (int x = 0; x < kCols / kRound; ++x) {
    const int64_t left = p.N - n0 - x * kRound - ch * kPer;        // columns from this lane's piece on
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* f = acc + x * kRound + i * kPer;
      __align__(16) T v[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if constexpr (sizeof(T) == 2) v[j] = __float2bfloat16_rn(f[j]);
        else v[j] = f[j];
      }
      *reinterpret_cast<uint4*>(box + lane * 128 + ((i ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4*>(v);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (4 * j >= rows || left <= 0) continue;
      const int r = 4 * j + sub;
      const uint4 u = *reinterpret_cast<const uint4*>(box + r * 128 + ((ch ^ (r & 7)) << 4));
      T* d = out + (int64_t)(4 * j) * p.ldc + x * kRound;
      if (wide && left >= kPer) {
        *reinterpret_cast<uint4*>(d) = u;
      } else {
        const T* v = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if (k < left) d[k] = v[k];
      }
    }
    __syncwarp();
  }
}

// h = act(gate) * up of this thread's 64 columns from cur.n0 + 64 * half on:
// acc holds 64 gate, then 64 up sums. Quantized per 128 columns, that is over
// both halves where the second exists (`both`). Columns past I count as
// zeros.
__device__ __forceinline__ void fb_glu_half(const FbParams& p, const FbTile& cur, float (*amax)[128], bool both,
                                            float (&acc)[128], int row, int half) {
  const int64_t n0 = cur.n0 + 64 * half;
  const int n_ok = (int)min((int64_t)64, p.I - n0);
  const float2 ac = fb_act_of(p.act);
  uint32_t key = 0;
#pragma unroll
  for (int i = 0; i < 64; i += 2) {
    const float2 v = fb_act2(ac, acc[i], acc[i + 1]);
    acc[i] = i < n_ok ? v.x * acc[64 + i] : 0.0f;
    acc[i + 1] = i < n_ok ? v.y * acc[65 + i] : 0.0f;      // n_ok is even
    key = max(key, max(__float_as_uint(acc[i]) & 0x7FFFFFFFu, __float_as_uint(acc[i + 1]) & 0x7FFFFFFFu));
  }
  if (both) {
    amax[half][row] = __uint_as_float(key);
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kFbEpiWarps) : "memory");
    key = max(key, __float_as_uint(amax[half ^ 1][row]));
    // the next tile's maxima are written after every read of these
    asm volatile("bar.sync 1, %0;" ::"n"(32 * kFbEpiWarps) : "memory");
  }
  const float2 s = fb_scales(__uint_as_float(key));
  if (row >= cur.rows) return;
  if (half == 0) p.hs[(cur.row0 + row) * p.hs_ld + cur.n0 / kFbBlock] = s.y;
  uint8_t* d = p.hq + (cur.row0 + row) * p.hq_ld + n0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (16 * i >= n_ok) break;
    uint32_t c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* v = acc + 16 * i + 4 * j;
      c[j] = fb_codes4(v[0] * s.x, v[1] * s.x, v[2] * s.x, v[3] * s.x);
    }
    *reinterpret_cast<uint4*>(d + 16 * i) = make_uint4(c[0], c[1], c[2], c[3]);
  }
}

template <int BN, int EPI>
__global__ void __launch_bounds__(kFbThreads, 1) fp8_block_gemm_kernel(const __grid_constant__ CUtensorMap tmA,
                                                                      const __grid_constant__ CUtensorMap tmW,
                                                                      const __grid_constant__ CUtensorMap tmO,
                                                                      const FbParams p) {
  using L = FbLayout<BN, EPI>;
  extern __shared__ __align__(1024) uint8_t dsmem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~uintptr_t(1023));
  auto* sh = reinterpret_cast<typename L::Ctl*>(base + L::kStages * L::kStage + L::kOut);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      sm100::mbar_init(&sh->full[s], 1);
      sm100::mbar_init(&sh->empty[s], 2);      // both issuers
    }
    for (int b = 0; b < 2; ++b) {
      sm100::mbar_init(&sh->acc_full[b], 1);
      sm100::mbar_init(&sh->acc_empty[b], kFbEpiWarps);
    }
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&tmA);
    sm100::prefetch_tmap(&tmW);
    if (EPI == kFbStore && p.out_tma) sm100::prefetch_tmap(&tmO);
  }
  if (p.grp_off)
    for (int e = tid; e <= p.E; e += kFbThreads) sh->tile_off[e] = p.tile_off[e];
  const int* tile_off = sh->tile_off;
  if (warp == 1) sm100::tmem_alloc(&sh->tmem_base, L::kTmemCols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const int tiles_m = p.grp_off ? tile_off[p.E] : (int)p.tiles_m, total = tiles_m * p.tiles_n;
  const int KB = p.KB;
  // Does the second column half of the tile at column n0 exist? Where it does
  // not, its MMAs, sums and stores are left out.
  auto has_two = [&](int64_t n0) { return EPI == kFbGlu ? n0 + BN / 4 < p.I : n0 + BN / 2 < p.N; };
  const bool half_last = !has_two((int64_t)(p.tiles_n - 1) * (EPI == kFbGlu ? BN / 2 : BN));
  auto place = [&](int t) { return fb_place(t, tiles_m, p.tiles_n, half_last); };

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFbRegsLow));
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    const bool leader = sm100::elect_one();
    uint32_t g = 0;      // K steps so far
    bool alive = true;
    for (int t = blockIdx.x; t < total && alive; t += gridDim.x) {
      const FbTile ti = fb_tile<BN, EPI>(p, tile_off, place(t));
      const int64_t w0 = ti.expert * p.N + ti.n0;
      for (int kb = 0; kb < KB; ++kb, ++g) {
        const uint32_t s = g % L::kStages, ph = (g / L::kStages) & 1;
        if (!sm100::mbar_wait(&sh->empty[s], ph ^ 1, p.err, 71)) { alive = false; break; }
        if (leader) {
          uint8_t* st = base + s * L::kStage;
          sm100::mbar_arrive_expect_tx(&sh->full[s], L::kStage);
          sm100::tma_load_2d(st, &tmA, kb * 128, (int32_t)ti.row0, &sh->full[s]);
          if constexpr (EPI == kFbGlu) {
            // per half: its gate rows, then the up rows that go with them
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sm100::tma_load_2d(st + L::kA + i * (L::kB / 4), &tmW, kb * 128,
                                 (int32_t)(w0 + (i >> 1) * (BN / 4) + (i & 1) * p.I), &sh->full[s]);
          } else {
            sm100::tma_load_2d(st + L::kA, &tmW, kb * 128, (int32_t)w0, &sh->full[s]);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp < 3) {
    // ------------------------------------------------------------ MMA issuers
    // Warp 1 takes the even K steps and TMEM buffer 0, warp 2 the odd ones:
    // a wait costs its thread about 100 cycles even when it is already
    // satisfied, and two issuers spend them under one another's MMAs (one, with
    // its two waits a step: 606 cycles per step against the MMAs' 512). A parity
    // wait is only sound where its waiter holds back the barrier's next phase,
    // so both look at every stage and both give it back.
    const bool leader = sm100::elect_one();
    const uint32_t b = warp - 1;
    const int mine = (int)blockIdx.x < total ? (total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;
    const uint32_t steps = (uint32_t)mine * KB;
    int t = blockIdx.x, kb = 0;          // tile and K step of g
    uint32_t idesc = 0;
    for (uint32_t g = 0; g < steps; ++g, ++kb) {
      if (kb == KB) {
        kb = 0;
        t += gridDim.x;
      }
      if (kb == 0)
        idesc = sm100::idesc_f8(half_last && place(t).y == p.tiles_n - 1 ? BN / 2 : BN);
      const uint32_t s = g % L::kStages, ph = (g / L::kStages) & 1, bph = (g >> 1) & 1;
      if ((g & 1) != b) {
        if (!sm100::mbar_wait(&sh->full[s], ph, p.err, 73)) break;
        if (leader) sm100::mbar_arrive(&sh->empty[s]);
        __syncwarp();
        continue;
      }
      // (the accumulator last: it is what comes last)
      if (!sm100::mbar_wait(&sh->full[s], ph, p.err, 73) ||
          !sm100::mbar_wait(&sh->acc_empty[b], bph ^ 1, p.err, 72))
        break;
      sm100::tc_fence_after();
      if (leader) {
        const uint32_t sa = sm100::smem_u32(base + s * L::kStage), sb = sa + L::kA;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sm100::tc_mma_f8(tmem + b * BN, sm100::sdesc_k_sw128(sa + 32 * j), sm100::sdesc_k_sw128(sb + 32 * j), idesc,
                           j ? 1u : 0u);
        sm100::tc_commit(&sh->acc_full[b]);
        sm100::tc_commit(&sh->empty[s]);
      }
      __syncwarp();
    }
  }
  } else {
    // ------------------------------------------------------------ epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFbRegsHigh));
    const int q = warp & 3, half = (warp - 4) >> 2;
    const int row = 32 * q + lane;
    constexpr int kCols = BN / 2;          // columns of this thread
    constexpr int kChunks = kCols / 32;
    uint32_t g = 0;
    // A warp whose wait ran out goes through its remaining tiles without
    // waiting, as the other warps count on it at the barriers below, and
    // stores NaN, so that nobody takes what was there before for the result.
    bool alive = true;
    FbTile ti{};
    const float *sa = p.sa, *sw0 = p.sw, *sw1 = p.sw;
    float a = 0.0f, w0 = 0.0f, w1 = 0.0f;
    // a tile's scales: pointers, and the values of its first K step
    auto open_tile = [&](int t) {
      ti = fb_tile<BN, EPI>(p, tile_off, place(t));
      sa = p.sa + (ti.row0 + (row < ti.rows ? row : 0)) * KB;
      const float* se = p.sw + ti.expert * p.NB * KB;
      // a run of columns that lies past the last row of w reads the last
      // scale; its sums are not used
      const int64_t c0 = min(ti.n0 + half * (EPI == kFbGlu ? BN / 4 : kCols), p.N - 1);
      const int64_t c1 = EPI == kFbGlu ? min(p.I + ti.n0 + half * (BN / 4), p.N - 1) : c0;
      sw0 = se + (c0 / kFbBlock) * KB;
      sw1 = se + (c1 / kFbBlock) * KB;
      a = __ldg(sa);
      w0 = __ldg(sw0);
      w1 = __ldg(sw1);
    };
    if ((int)blockIdx.x < total) open_tile(blockIdx.x);
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const FbTile cur = ti;
      const bool both = has_two(cur.n0);
      if (half && !both) {      // these columns do not exist: only hand the buffers back
        for (int kb = 0; kb < KB; ++kb, ++g) {
          if (alive) alive = sm100::mbar_wait(&sh->acc_full[g & 1], (g >> 1) & 1, p.err, 75);
          if (alive && lane == 0) sm100::mbar_arrive(&sh->acc_empty[g & 1]);
        }
        if (t + (int)gridDim.x < total) open_tile(t + gridDim.x);
        continue;
      }
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
      for (int kb = 0; kb < KB; ++kb, ++g) {
        const uint32_t b = g & 1, bph = (g >> 1) & 1;
        const float c0 = a * w0, c1 = a * w1;
        if (kb + 1 < KB) {
          a = __ldg(sa + kb + 1);
          w0 = __ldg(sw0 + kb + 1);
          w1 = __ldg(sw1 + kb + 1);
        }
        if (!alive || !sm100::mbar_wait(&sh->acc_full[b], bph, p.err, 74)) {
          alive = false;
          break;
        }
        sm100::tc_fence_after();
        const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16) + b * BN + half * kCols;
        // the read of a chunk of 32 columns runs under the sums of the last
        uint32_t r[2][32];
        sm100::tmem_ld32_nowait(tq, r[0]);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          sm100::tmem_ld_wait();
          if (c + 1 < kChunks) {
            sm100::tmem_ld32_nowait(tq + 32 * (c + 1), r[(c + 1) & 1]);
          } else {
            sm100::tc_fence_before();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&sh->acc_empty[b]);
          }
          const float cs = (EPI == kFbGlu && c >= kChunks / 2) ? c1 : c0;
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[32 * c + i] = fmaf(__uint_as_float(r[c & 1][i]), cs, acc[32 * c + i]);
        }
      }
      if (!alive) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[i] = __int_as_float(0x7FC00000);
      }
      if (t + (int)gridDim.x < total) open_tile(t + gridDim.x);   // its loads run under the stores
      if constexpr (EPI == kFbStore) {
        if (p.bias) {
          const int64_t n0 = cur.n0 + half * kCols;
#pragma unroll
          for (int i = 0; i < kCols; ++i) acc[i] += n0 + i < p.N ? __bfloat162float(p.bias[n0 + i]) : 0.0f;
        }
        // the last tile's TMA stores have read this half's room
        uint8_t* box = base + L::kStages * L::kStage + half * (128 * kCols * 2);
        if (row == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
        if (p.out_tma) fb_store_tile(p, tmO, cur, box, acc, row, half);
        else if (p.out_dt == AEOQ_BF16) fb_store_rows<__nv_bfloat16>(p, cur, box + q * 4096, acc, q, half);
        else fb_store_rows<float>(p, cur, box + q * 4096, acc, q, half);
      } else {
        fb_glu_half(p, cur, sh->amax, both, acc, row, half);
      }
    }
  }
  // the stores' reads of shared memory are over before it goes away
  if (EPI == kFbStore && warp >= 4) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, L::kTmemCols);
  }
}

template <int BN, int EPI>
static int launch_gemm(const uint8_t* a, int64_t a_rows, const uint8_t* w, FbParams p, int64_t max_tiles,
                       cudaStream_t st) {
  using L = FbLayout<BN, EPI>;
  CUtensorMap ta, tw, to;
  int rc = make_tmap_bytes(&ta, a, a_rows, p.K, p.K, 128, 128, true);
  if (rc) return rc;
  rc = make_tmap_bytes(&tw, w, p.E * p.N, p.K, p.K, 128, EPI == kFbGlu ? BN / 4 : BN, true);
  if (rc) return rc;
  to = ta;
  // (a column's byte is a 32-bit coordinate of the store, and a row that does
  // not end on 16 bytes was written beyond its last column: N = 127, ldc = 136)
  p.out_tma = EPI == kFbStore && p.out_dt == AEOQ_BF16 && p.ldc % 8 == 0 && (uintptr_t)p.out % 16 == 0 &&
              p.N % 8 == 0 && p.N <= (1 << 30);
  if (p.out_tma) {
    rc = make_tmap_bytes(&to, p.out, p.M, p.N * 2, p.ldc * 2, 128, 128, true);
    if (rc) return rc;
  }
  AEOQ_REQUIRE(max_tiles <= 0x7FFFFFFF, AEOQ_ERR_INVALID, "fp8_block_gemm: too many tiles");
  rc = func_smem_attr((const void*)fp8_block_gemm_kernel<BN, EPI>, L::kBytes, -1, "fp8_block_gemm");
  if (rc) return rc;
  const int ctas = (int)std::min<int64_t>(device_sm_count(), max_tiles);
  fp8_block_gemm_kernel<BN, EPI><<<ctas, kFbThreads, L::kBytes, st>>>(ta, tw, to, p);
  return check_launch("fp8_block_gemm_kernel");
}

// ---------------------------------------------------------------- few rows per expert
// The grouped GEMMs for experts with few tokens: bound by the weights' bytes,
// if nothing else takes longer. With tokens on the MMA's 128 rows the scaling
// of 256 columns does (16 tokens over 128 experts: 78 + 49 us for 505 MB), so
// here the weights are the MMA's rows and up to 32 tokens its columns: a
// thread owns one output feature and 16 tokens, a K step costs it 32 sums.
//
// Tile: 256 rows of w as two MMAs of 128 (GLU: 128 gate rows and the 128 up
// rows that go with them; store: 256 consecutive ones) times 32 tokens.
// GLU gathers its tokens' rows where they are (a gather4 of four rows per
// lane; for tiles of 128 rows that takes too long: 460 against 267 us at 4096
// tokens, so there the quantizer writes a row for each of a token's experts).
//   warp 0 TMA, warp 1 MMA and TMEM, warps 4-11 scaling and epilogue: four
//   warps with tokens 0-15, four with tokens 16-31
struct FbFewLayout {
  static constexpr int kTok = 32;
  static constexpr uint32_t kA = 256 * 128, kB = kTok * 128, kStage = kA + kB;
  struct Ctl {
    uint64_t full[kFbMaxStages], empty[kFbMaxStages];
    uint64_t acc_full[2], acc_empty[2];
    uint32_t tmem_base;
    uint32_t amax[2][4][16];             // GLU: [token half][lane quadrant][token]
    int tile_off[kFbMaxExperts + 1];
  };
  static constexpr int kStages =
      std::min<int>(kFbMaxStages, (227 * 1024 - 1024 - (int)sizeof(Ctl)) / (int)kStage);
  static constexpr size_t kBytes = 1024 + (size_t)kStages * kStage + sizeof(Ctl);
  static constexpr uint32_t kTmemCols = 128;   // 2 buffers x 2 MMAs x 32 tokens
};

// Source rows of the sorted rows r0 .. r0 + 3 of a tile (past its last one:
// the first, whose products are not used).
__device__ __forceinline__ int4 fb_rows4(const FbParams& p, const FbTile& ti, int r0) {
  int v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __ldg(p.row_src + ti.row0 + (r0 + i < ti.rows ? r0 + i : 0));
  return make_int4(v[0], v[1], v[2], v[3]);
}

template <int EPI>
__global__ void __launch_bounds__(kFbThreads, 1) fp8_block_few_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                     const __grid_constant__ CUtensorMap tmB,
                                                                     const FbParams p) {
  using L = FbFewLayout;
  extern __shared__ __align__(1024) uint8_t dsmem[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dsmem) + 1023) & ~uintptr_t(1023));
  auto* sh = reinterpret_cast<L::Ctl*>(base + L::kStages * L::kStage);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      sm100::mbar_init(&sh->full[s], 1);
      sm100::mbar_init(&sh->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      sm100::mbar_init(&sh->acc_full[b], 1);
      sm100::mbar_init(&sh->acc_empty[b], kFbEpiWarps);
    }
    sm100::fence_barrier_init();
    sm100::prefetch_tmap(&tmW);
    sm100::prefetch_tmap(&tmB);
  }
  for (int e = tid; e <= p.E; e += kFbThreads) sh->tile_off[e] = p.tile_off[e];
  if (warp == 1) sm100::tmem_alloc(&sh->tmem_base, L::kTmemCols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  const int total = sh->tile_off[p.E] * p.tiles_n, KB = p.KB;
  constexpr int kWide = EPI == kFbGlu ? 128 : 256;      // output columns of a tile
  auto tile = [&](int t) {
    FbTile r;
    const int ct = t / p.tiles_n;
    r.n0 = (int64_t)(t - ct * p.tiles_n) * kWide;
    int lo = 0, hi = p.E;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sh->tile_off[mid] <= ct) lo = mid; else hi = mid;
    }
    r.expert = lo;
    const int g0 = __ldg(p.grp_off + lo), g1 = __ldg(p.grp_off + lo + 1);
    r.row0 = g0 + (ct - sh->tile_off[lo]) * L::kTok;
    r.rows = min(L::kTok, g1 - (int)r.row0);
    return r;
  };

  if (warp == 0) {
    const bool leader = sm100::elect_one();
    uint32_t g = 0;
    bool alive = true;
    for (int t = blockIdx.x; t < total && alive; t += gridDim.x) {
      const FbTile ti = tile(t);
      const int w0 = (int)(ti.expert * p.N + ti.n0);
      // boxes of 64 rows of w: those that hold an output column
      const int left = (int)((EPI == kFbGlu ? p.I : p.N) - ti.n0), boxes = min(kWide / 64, (left + 63) / 64);
      int4 src = make_int4(0, 0, 0, 0);
      if (EPI == kFbGlu) src = fb_rows4(p, ti, 4 * (lane & 7));
      for (int kb = 0; kb < KB; ++kb, ++g) {
        const uint32_t s = g % L::kStages, ph = (g / L::kStages) & 1;
        if (!sm100::mbar_wait(&sh->empty[s], ph ^ 1, p.err, 81)) { alive = false; break; }
        if (leader) {
          uint8_t* st = base + s * L::kStage;
          sm100::mbar_arrive_expect_tx(&sh->full[s], L::kB + (uint32_t)boxes * (EPI == kFbGlu ? 2 : 1) * 8192);
          for (int i = 0; i < boxes; ++i) {
            sm100::tma_load_2d(st + i * 8192, &tmW, kb * 128, w0 + 64 * i, &sh->full[s]);
            if (EPI == kFbGlu)
              sm100::tma_load_2d(st + 16384 + i * 8192, &tmW, kb * 128, w0 + (int)p.I + 64 * i, &sh->full[s]);
          }
          if (EPI == kFbStore) sm100::tma_load_2d(st + L::kA, &tmB, kb * 128, (int)ti.row0, &sh->full[s]);
        }
        if (EPI == kFbGlu && lane < L::kTok / 4)
          sm100::tma_gather4(base + s * L::kStage + L::kA + lane * 512, &tmB, kb * 128, src, &sh->full[s]);
        __syncwarp();
      }
    }
  } else if (warp == 1) {
    const bool leader = sm100::elect_one();
    constexpr uint32_t idesc = sm100::idesc_f8(L::kTok);
    const int mine = (int)blockIdx.x < total ? (total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x : 0;
    const uint32_t steps = (uint32_t)mine * KB;
    for (uint32_t g = 0; g < steps; ++g) {
      const uint32_t s = g % L::kStages, ph = (g / L::kStages) & 1, b = g & 1, bph = (g >> 1) & 1;
      if (!sm100::mbar_wait(&sh->acc_empty[b], bph ^ 1, p.err, 82) ||
          !sm100::mbar_wait(&sh->full[s], ph, p.err, 83))
        break;
      sm100::tc_fence_after();
      if (leader) {
        const uint32_t sa = sm100::smem_u32(base + s * L::kStage), sb = sa + L::kA;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sm100::tc_mma_f8(tmem + b * 64 + m * 32, sm100::sdesc_k_sw128(sa + m * 16384 + 32 * j),
                             sm100::sdesc_k_sw128(sb + 32 * j), idesc, j ? 1u : 0u);
        sm100::tc_commit(&sh->empty[s]);
        sm100::tc_commit(&sh->acc_full[b]);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    const int q = warp & 3, half = (warp - 4) >> 2, f = 32 * q + lane;      // f: row of w in each MMA
    uint32_t g = 0;
    bool alive = true;      // as in the kernel above
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const FbTile ti = tile(t);
      const int tok0 = 16 * half, n_tok = min(16, ti.rows - tok0);
      if (n_tok <= 0) {
        for (int kb = 0; kb < KB; ++kb, ++g) {
          if (alive) alive = sm100::mbar_wait(&sh->acc_full[g & 1], (g >> 1) & 1, p.err, 84);
          if (alive && lane == 0) sm100::mbar_arrive(&sh->acc_empty[g & 1]);
        }
        continue;
      }
      // lane j's token scale; the two MMAs' weight scales (rows past the last
      // one take its scale, their sums are not used)
      int64_t r = ti.row0 + tok0 + min(lane & 15, n_tok - 1);
      if (EPI == kFbGlu) r = __ldg(p.row_src + r);
      const float* sa = p.sa + r * KB;
      const float* se = p.sw + ti.expert * p.NB * KB;
      const int64_t c0 = min(ti.n0 + f, p.N - 1), c1 = min((EPI == kFbGlu ? p.I : 128) + ti.n0 + f, p.N - 1);
      const float *sw0 = se + (c0 / kFbBlock) * KB, *sw1 = se + (c1 / kFbBlock) * KB;
      float acc[2][16];
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[0][j] = acc[1][j] = 0.0f;
      float a = __ldg(sa), w0 = __ldg(sw0), w1 = __ldg(sw1);
      for (int kb = 0; kb < KB; ++kb, ++g) {
        const uint32_t b = g & 1, bph = (g >> 1) & 1;
        const float a_now = a, w0_now = w0, w1_now = w1;
        if (kb + 1 < KB) {
          a = __ldg(sa + kb + 1);
          w0 = __ldg(sw0 + kb + 1);
          w1 = __ldg(sw1 + kb + 1);
        }
        if (alive) alive = sm100::mbar_wait(&sh->acc_full[b], bph, p.err, 85);
        if (!alive) {
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[0][j] = acc[1][j] = __int_as_float(0x7FC00000);
          continue;
        }
        sm100::tc_fence_after();
        const uint32_t tq = tmem + ((uint32_t)(32 * q) << 16) + b * 64 + tok0;
        float r0[16], r1[16];
        sm100::tmem_ld16(tq, r0);
        sm100::tmem_ld16(tq + 32, r1);
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&sh->acc_empty[b]);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float c = __shfl_sync(0xFFFFFFFFu, a_now, j);
          acc[0][j] = fmaf(r0[j], c * w0_now, acc[0][j]);
          acc[1][j] = fmaf(r1[j], c * w1_now, acc[1][j]);
        }
      }
      if constexpr (EPI == kFbStore) {
        // 32 lanes store 128 consecutive bytes of a token's row
        float* d = reinterpret_cast<float*>(p.out) + (ti.row0 + tok0) * p.ldc + ti.n0 + f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (j >= n_tok) break;
          if (ti.n0 + f < p.N) d[j * p.ldc] = acc[0][j];
          if (ti.n0 + 128 + f < p.N) d[j * p.ldc + 128] = acc[1][j];
        }
      } else {
        // the block of 128 features of a token is this tile's 128 lanes
        const bool in = ti.n0 + f < p.I;
        const float2 ac = fb_act_of(p.act);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          acc[0][j] = in ? fb_act(ac, acc[0][j]) * acc[1][j] : 0.0f;
          const uint32_t k = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(acc[0][j]) & 0x7FFFFFFFu);
          if (lane == j) sh->amax[half][q][j] = k;
        }
        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
        uint32_t k = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) k = max(k, sh->amax[half][i][lane & 15]);
        asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
        const float2 s = fb_scales(__uint_as_float(k));      // of token lane & 15
        if (q == 0 && lane < n_tok) p.hs[(ti.row0 + tok0 + lane) * p.hs_ld + ti.n0 / kFbBlock] = s.y;
        uint8_t* d = p.hq + (ti.row0 + tok0) * p.hq_ld + ti.n0 + f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float inv = __shfl_sync(0xFFFFFFFFu, s.x, j);
          if (j < n_tok && in) d[j * p.hq_ld] = (uint8_t)fb_codes4(acc[0][j] * inv, 0.0f, 0.0f, 0.0f);
        }
      }
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, L::kTmemCols);
  }
}

template <int EPI>
static int launch_few(const uint8_t* a, int64_t a_rows, const uint8_t* w, const FbParams& p, int64_t max_tiles,
                      cudaStream_t st) {
  using L = FbFewLayout;
  CUtensorMap tw, tb;
  int rc = make_tmap_bytes(&tw, w, p.E * p.N, p.K, p.K, 128, 64, true);
  if (rc) return rc;
  rc = make_tmap_bytes(&tb, a, a_rows, p.K, p.K, 128, EPI == kFbGlu ? 1 : L::kTok, true);
  if (rc) return rc;
  AEOQ_REQUIRE(max_tiles <= 0x7FFFFFFF, AEOQ_ERR_INVALID, "fp8_block_few: too many tiles");
  rc = func_smem_attr((const void*)fp8_block_few_kernel<EPI>, L::kBytes, -1, "fp8_block_few");
  if (rc) return rc;
  const int ctas = (int)std::min<int64_t>(device_sm_count(), max_tiles);
  fp8_block_few_kernel<EPI><<<ctas, kFbThreads, L::kBytes, st>>>(tw, tb, p);
  return check_launch("fp8_block_few_kernel");
}

static int gemm_dense(const uint8_t* a, const float* sa, int64_t M, const uint8_t* w, const float* sw, int64_t N,
                      int64_t K, const void* bias, void* out, int out_dt, int64_t ldc, int* err, cudaStream_t st) {
  FbParams p{};
  p.M = M;
  p.N = N;
  p.K = (int)K;
  p.KB = (int)fb_blocks(K);
  p.NB = fb_blocks(N);
  p.E = 1;
  p.sa = sa;
  p.sw = sw;
  p.out = out;
  p.out_dt = out_dt;
  p.ldc = ldc;
  p.bias = reinterpret_cast<const __nv_bfloat16*>(bias);
  p.err = err;
  // A K step of a tile of 128 columns takes not half of but 5/6 of what one of
  // 256 takes (the hand-over of the accumulators, not the MMAs, bounds it), so
  // the narrow tiles pay only where they take fewer rounds of CTAs: 1024 x 1408 x
  // 2816 24.6 against 28.7 us, 2048 x 1408 x 2816 34.8 against 28.7.
  const int64_t sms = device_sm_count();
  p.tiles_m = (M + 127) / 128;
  p.tiles_n = (int)((N + 255) / 256);
  const int64_t wide = p.tiles_m * p.tiles_n, narrow = p.tiles_m * ((N + 127) / 128);
  if (6 * ((wide + sms - 1) / sms) < 5 * ((narrow + sms - 1) / sms))
    return launch_gemm<256, kFbStore>(a, M, w, p, wide, st);
  p.tiles_n = (int)((N + 127) / 128);
  return launch_gemm<128, kFbStore>(a, M, w, p, narrow, st);
}

// ---------------------------------------------------------------- experts
// Pairs (token, slot) sorted by expert: a counting sort by one cluster of
// CTAs, each with its slice of the pairs.
//   grp_off[e]   first row of expert e        (E + 1 values)
//   tile_off[e]  tiles of `tile` rows before expert e (E + 1 values)
//   row_tok[r]   token of sorted row r;  pair_row[i]  row of pair i, or -1
// The order of an expert's rows within one CTA's slice is arbitrary; each row
// is computed by itself and the sum over a token's slots goes by slot.
constexpr int kFbSortCtas = 8;
__global__ void __launch_bounds__(1024) fb_sort_kernel(const void* ids, int ids_dt, int64_t n_pairs, int k, int E,
                                                       int tile, int* grp_off, int* tile_off, int* row_tok,
                                                       int* pair_row) {
  __shared__ int cnt[kFbMaxExperts], fill[kFbMaxExperts];
  __shared__ int s_row[32], s_tile[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, ctas = gridDim.x, rank = blockIdx.x;
  const int64_t slice = (n_pairs + ctas - 1) / ctas, beg = rank * slice, end = min(n_pairs, beg + slice);
  cnt[t] = 0;
  __syncthreads();
  for (int64_t i = beg + t; i < end; i += 1024) {
    const int64_t e = load_index(ids, ids_dt, i);
    if (e >= 0 && e < E) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  int c = cnt[t], before = 0;      // all CTAs' pairs of expert t, those of lower ranks
  if (ctas > 1) {
    sm100::cluster_sync();
    c = 0;
    for (int r = 0; r < ctas; ++r) {
      const int v = __float_as_int(sm100::ld_dsmem_f32(sm100::dsmem_addr(&cnt[t], r)));
      c += v;
      before += r < rank ? v : 0;
    }
  }
  const int d = (c + tile - 1) / tile;      // experts past E count 0
  int r = c, q = d;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int rr = __shfl_up_sync(0xFFFFFFFFu, r, o), qq = __shfl_up_sync(0xFFFFFFFFu, q, o);
    if (lane >= o) { r += rr; q += qq; }
  }
  if (lane == 31) { s_row[warp] = r; s_tile[warp] = q; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { r += s_row[w]; q += s_tile[w]; }
  fill[t] = r - c + before;
  if (t < E && rank == 0) {
    grp_off[t] = r - c;
    tile_off[t] = q - d;
    if (t == E - 1) { grp_off[E] = r; tile_off[E] = q; }
  }
  __syncthreads();
  for (int64_t i = beg + t; i < end; i += 1024) {
    const int64_t e = load_index(ids, ids_dt, i);
    int at = -1;
    if (e >= 0 && e < E) {
      at = atomicAdd(&fill[e], 1);
      row_tok[at] = (int)(i / k);
    }
    pair_row[i] = at;
  }
  if (ctas > 1) sm100::cluster_sync();      // the others have read this CTA's counts
}

static int launch_sort(const void* ids, int ids_dt, int64_t n_pairs, int k, int E, int tile, int* grp_off,
                       int* tile_off, int* row_tok, int* pair_row, cudaStream_t st) {
  // one CTA up to 4096 pairs (4 per thread), else a cluster
  const int ctas = n_pairs > 4096 ? kFbSortCtas : 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ctas;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, fb_sort_kernel, ids, ids_dt, n_pairs, k, E, tile, grp_off, tile_off, row_tok, pair_row);
  return check_launch("fb_sort_kernel");
}

// out[t] = sum over slots j, in order, of weights[t][j] * y[pair_row[t][j]], in
// f32, rounded once; a slot without an expert adds nothing. y is f32 as well:
// held in bf16, each expert's output would be rounded too, 1.41 times the
// error of the one rounding, and where the experts' outputs cancel more (at 4096
// tokens, top-8, H = 2816 that would take 38 us here for 68, and 155 for 192
// in the GEMM that writes it). The loads of kFbCombineSlots slots are in flight
// together (same size: one 69 us, 2 and 4 68 us, which is 6.1 TB/s, 8 102 us).
constexpr int kFbCombineSlots = 4;
__global__ void __launch_bounds__(256) fb_combine_kernel(const float* __restrict__ y,
                                                         const int* __restrict__ pair_row,
                                                         const float* __restrict__ weights, int64_t T, int k,
                                                         int64_t H, __nv_bfloat16* __restrict__ out) {
  const int64_t per = H / 8, n = T * per;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int64_t t = i / per, c = i - t * per;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < k; j0 += kFbCombineSlots) {
      int r[kFbCombineSlots];
      float w[kFbCombineSlots];
      FbEight<AEOQ_F32> v[kFbCombineSlots];
#pragma unroll
      for (int j = 0; j < kFbCombineSlots; ++j) {
        r[j] = j0 + j < k ? __ldg(pair_row + t * k + j0 + j) : -1;
        w[j] = j0 + j < k ? __ldg(weights + t * k + j0 + j) : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kFbCombineSlots; ++j)
        if (r[j] >= 0) v[j].load(y + r[j] * H + 8 * c);
#pragma unroll
      for (int j = 0; j < kFbCombineSlots; ++j)
        if (r[j] >= 0) {
#pragma unroll
          for (int x = 0; x < 8; ++x) s[x] = fmaf(w[j], v[j].at(x), s[x]);
        }
    }
    __align__(16) __nv_bfloat162 o[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) o[x] = __floats2bfloat162_rn(s[2 * x], s[2 * x + 1]);
    *reinterpret_cast<uint4*>(out + t * H + 8 * c) = *reinterpret_cast<const uint4*>(o);
  }
}

// Weights on the MMA's rows up to 40 rows per expert: at 128 experts, top-8, H =
// 2816, I = 704 (cold L2) 64 tokens take 170 us that way and 228 the other,
// 512 tokens (32 rows) 205 and 244, 1024 tokens (64 rows) 328 and 260.
static bool fb_few(int64_t pairs, int64_t experts) { return pairs <= 40 * experts; }

// Workspace: of the grouped forward, or of that for few tokens (h alone).
struct FbExpertsWs {
  size_t grp_off = 0, tile_off = 0, row_tok = 0, pair_row = 0, xq = 0, xs = 0, hq = 0, hs = 0, y = 0, h = 0, bytes = 0;
  FbExpertsWs(int64_t T, int64_t k, int64_t E, int64_t H, int64_t I) {
    size_t o = 0;
    const int64_t P = T * k;
    auto take = [&](int64_t n) {
      const size_t at = o;
      o += (size_t)((n + 255) / 256 * 256);
      return at;
    };
    if (fb_experts_skinny_takes(T, k, E, H, I)) {
      h = take(4 * P * I);
      bytes = o;
      return;
    }
    grp_off = take(4 * (E + 1));
    tile_off = take(4 * (E + 1));
    row_tok = take(4 * P);
    pair_row = take(4 * P);
    const int64_t rows = fb_few(P, E) ? T : P;
    xq = take(rows * H);
    xs = take(4 * rows * fb_blocks(H));
    hq = take(P * I);
    hs = take(4 * P * fb_blocks(I));
    y = take(4 * P * H);
    // never less than for fewer tokens, whose h may take more by itself
    const size_t whole = o;
    o = 0;
    take(4 * fb_experts_skinny_most(T, k, E, H, I) * k * I);
    bytes = std::max(whole, o);
  }
};

}  // namespace aeoq

using namespace aeoq;

static int check_linear(const char* what, int64_t M, int64_t N, int64_t K, int out_dtype, int64_t ldc) {
  AEOQ_REQUIRE(M >= 0 && N >= 0 && K >= 0, AEOQ_ERR_INVALID, "%s: negative shape", what);
  AEOQ_REQUIRE(K > 0 && K % 16 == 0 && K <= (1LL << 24), AEOQ_ERR_INVALID,
               "%s: K (%lld) must be a positive multiple of 16, at most 2^24", what, (long long)K);
  AEOQ_REQUIRE(M <= 0x7FFFFFFF && N <= 0x7FFFFFFF, AEOQ_ERR_INVALID, "%s: M and N must fit 31 bits", what);
  AEOQ_REQUIRE(out_dtype == AEOQ_BF16 || out_dtype == AEOQ_F32, AEOQ_ERR_INVALID, "%s: bad output dtype", what);
  AEOQ_REQUIRE(ldc >= N, AEOQ_ERR_INVALID, "%s: output row stride %lld is below N", what, (long long)ldc);
  return AEOQ_OK;
}

extern "C" int aeoq_fp8_block_gemm(const uint8_t* a, const float* sa, int64_t M, const uint8_t* w, const float* sw,
                                   int64_t N, int64_t K, const void* bias, void* out, int out_dtype, int64_t ldc,
                                   int* err_word, void* stream) {
  int rc = check_linear("fp8_block_gemm", M, N, K, out_dtype, ldc);
  if (rc) return rc;
  if (M == 0 || N == 0) return AEOQ_OK;
  AEOQ_REQUIRE(a && sa && w && sw && out, AEOQ_ERR_INVALID, "fp8_block_gemm: null pointer");
  AEOQ_REQUIRE((uintptr_t)a % 16 == 0 && (uintptr_t)w % 16 == 0, AEOQ_ERR_INVALID,
               "fp8_block_gemm: operands must be 16-byte aligned");
  if (fb_linear_skinny_takes(M, N, K))
    return fb_linear_skinny(nullptr, AEOQ_BF16, K, M, w, sw, N, K, bias, out, out_dtype, ldc, const_cast<uint8_t*>(a),
                            const_cast<float*>(sa), (cudaStream_t)stream);
  return gemm_dense(a, sa, M, w, sw, N, K, bias, out, out_dtype, ldc, err_word, (cudaStream_t)stream);
}

static size_t linear_scales_at(int64_t M, int64_t K) { return (size_t)((M * K + 255) / 256 * 256); }

extern "C" size_t aeoq_fp8_block_linear_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= kFbSkinnyQuant || N <= 0 || K <= 0) return 0;
  return linear_scales_at(M, K) + (size_t)M * fb_blocks(K) * 4;
}

extern "C" int aeoq_fp8_block_linear(const void* x, int dtype, int64_t ldx, int64_t M, const uint8_t* w,
                                     const float* sw, int64_t N, int64_t K, const void* bias, void* out,
                                     int out_dtype, int64_t ldc, void* workspace, size_t workspace_bytes,
                                     int* err_word, void* stream) {
  int rc = check_linear("fp8_block_linear", M, N, K, out_dtype, ldc);
  if (rc) return rc;
  AEOQ_REQUIRE(dtype == AEOQ_BF16 || dtype == AEOQ_F16 || dtype == AEOQ_F32, AEOQ_ERR_INVALID,
               "fp8_block_linear: unsupported input dtype %d", dtype);
  AEOQ_REQUIRE(ldx >= K || M <= 1, AEOQ_ERR_INVALID, "fp8_block_linear: input row stride below K");
  if (M == 0 || N == 0) return AEOQ_OK;
  AEOQ_REQUIRE(x && w && sw && out, AEOQ_ERR_INVALID, "fp8_block_linear: null pointer");
  AEOQ_REQUIRE((uintptr_t)w % 16 == 0, AEOQ_ERR_INVALID, "fp8_block_linear: weights must be 16-byte aligned");
  const size_t need = aeoq_fp8_block_linear_workspace_size(M, N, K);
  AEOQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 256 == 0),
               AEOQ_ERR_WORKSPACE, "fp8_block_linear: a 256-byte aligned workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  uint8_t* q = reinterpret_cast<uint8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + linear_scales_at(M, K));
  if (fb_linear_skinny_takes(M, N, K))
    return fb_linear_skinny(x, dtype, ldx, M, w, sw, N, K, bias, out, out_dtype, ldc, q, s, st);
  rc = fb_quantize_rows(x, dtype, M, K, ldx, q, K, s, st);
  if (rc) return rc;
  return gemm_dense(q, s, M, w, sw, N, K, bias, out, out_dtype, ldc, err_word, st);
}

extern "C" size_t aeoq_moe_fp8_block_workspace_size(int64_t T, int64_t top_k, int64_t num_experts, int64_t hidden,
                                                    int64_t inter) {
  if (T <= 0 || top_k <= 0 || num_experts <= 0 || hidden <= 0 || inter <= 0) return 0;
  return FbExpertsWs(T, top_k, num_experts, hidden, inter).bytes;
}

extern "C" int aeoq_moe_fp8_block_forward(const void* hidden, int64_t T, const void* top_k_index, int idx_dtype,
                                          const float* top_k_weights, int64_t top_k, const uint8_t* gate_up,
                                          const float* gate_up_scale, const uint8_t* down, const float* down_scale,
                                          int64_t num_experts, int64_t hidden_dim, int64_t inter_dim, int activation,
                                          void* out, void* workspace, size_t workspace_bytes, int* err_word,
                                          void* stream) {
  const int64_t H = hidden_dim, I = inter_dim, E = num_experts, k = top_k;
  AEOQ_REQUIRE(E >= 1 && E <= kFbMaxExperts, AEOQ_ERR_INVALID, "moe_fp8_block: 1 <= num_experts <= %d", kFbMaxExperts);
  AEOQ_REQUIRE(k >= 1 && k <= 32, AEOQ_ERR_INVALID, "moe_fp8_block: 1 <= top_k <= 32");
  AEOQ_REQUIRE(H >= 16 && H % 16 == 0 && H <= (1 << 24), AEOQ_ERR_INVALID,
               "moe_fp8_block: hidden size (%lld) must be a multiple of 16", (long long)H);
  AEOQ_REQUIRE(I >= 64 && I % 64 == 0 && I <= (1 << 24), AEOQ_ERR_INVALID,
               "moe_fp8_block: intermediate size (%lld) must be a multiple of 64", (long long)I);
  AEOQ_REQUIRE(E * 2 * I <= 0x7FFFFFFF && E * H <= 0x7FFFFFFF, AEOQ_ERR_INVALID,
               "moe_fp8_block: the experts' weight rows must fit 31 bits");
  AEOQ_REQUIRE(T >= 0 && T <= 0x7FFFFFFF / k, AEOQ_ERR_INVALID, "moe_fp8_block: bad token count");
  AEOQ_REQUIRE(idx_dtype == AEOQ_I32 || idx_dtype == AEOQ_I64, AEOQ_ERR_INVALID, "moe_fp8_block: int32/int64 ids");
  AEOQ_REQUIRE(activation == AEOQ_ACT_GELU_TANH || activation == AEOQ_ACT_SILU, AEOQ_ERR_INVALID,
               "moe_fp8_block: bad activation %d", activation);
  if (T == 0) return AEOQ_OK;
  AEOQ_REQUIRE(hidden && top_k_index && top_k_weights && gate_up && gate_up_scale && down && down_scale && out,
               AEOQ_ERR_INVALID, "moe_fp8_block: null pointer");
  AEOQ_REQUIRE((uintptr_t)hidden % 16 == 0 && (uintptr_t)gate_up % 16 == 0 && (uintptr_t)down % 16 == 0 &&
                   (uintptr_t)out % 16 == 0,
               AEOQ_ERR_INVALID, "moe_fp8_block: hidden, weights and output must be 16-byte aligned");
  const FbExpertsWs l(T, k, E, H, I);
  AEOQ_REQUIRE(workspace && workspace_bytes >= l.bytes && (uintptr_t)workspace % 256 == 0, AEOQ_ERR_WORKSPACE,
               "moe_fp8_block: a 256-byte aligned workspace of %zu bytes needed, %zu given", l.bytes, workspace_bytes);
  cudaStream_t st = (cudaStream_t)stream;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  auto ints = [&](size_t o) { return reinterpret_cast<int*>(ws + o); };
  auto floats = [&](size_t o) { return reinterpret_cast<float*>(ws + o); };
  const int64_t P = T * k;
  if (fb_experts_skinny_takes(T, k, E, H, I))
    return fb_experts_skinny(hidden, T, top_k_index, idx_dtype, top_k_weights, k, gate_up, gate_up_scale, down,
                             down_scale, E, H, I, activation, floats(l.h), out, st);
  const bool few = fb_few(P, E);
  const int tile = few ? FbFewLayout::kTok : 128;
  int rc = launch_sort(top_k_index, idx_dtype, P, (int)k, (int)E, tile, ints(l.grp_off), ints(l.tile_off),
                       ints(l.row_tok), ints(l.pair_row), st);
  if (rc) return rc;
  rc = few ? fb_quantize_rows(hidden, AEOQ_BF16, T, H, H, ws + l.xq, H, floats(l.xs), st)
           : fb_quantize_rows_to(hidden, T, H, ints(l.pair_row), (int)k, ws + l.xq, floats(l.xs), st);
  if (rc) return rc;
  const int64_t max_tiles = std::min<int64_t>(P, (P + tile - 1) / tile + E);
  FbParams p{};
  p.M = P;
  p.N = 2 * I;
  p.K = (int)H;
  p.KB = (int)fb_blocks(H);
  p.NB = fb_blocks(2 * I);
  p.E = (int)E;
  p.sa = floats(l.xs);
  p.sw = gate_up_scale;
  p.row_src = ints(l.row_tok);
  p.grp_off = ints(l.grp_off);
  p.tile_off = ints(l.tile_off);
  p.tiles_n = (int)fb_blocks(I);
  p.I = I;
  p.act = activation;
  p.hq = ws + l.hq;
  p.hq_ld = I;
  p.hs = floats(l.hs);
  p.hs_ld = fb_blocks(I);
  p.err = err_word;
  rc = few ? launch_few<kFbGlu>(ws + l.xq, T, gate_up, p, max_tiles * p.tiles_n, st)
           : launch_gemm<256, kFbGlu>(ws + l.xq, P, gate_up, p, max_tiles * p.tiles_n, st);
  if (rc) return rc;
  FbParams d{};
  d.M = P;
  d.N = H;
  d.K = (int)I;
  d.KB = (int)fb_blocks(I);
  d.NB = fb_blocks(H);
  d.E = (int)E;
  d.sa = floats(l.hs);
  d.sw = down_scale;
  d.grp_off = ints(l.grp_off);
  d.tile_off = ints(l.tile_off);
  d.tiles_n = (int)((H + 255) / 256);
  d.out = ws + l.y;
  d.out_dt = AEOQ_F32;
  d.ldc = H;
  d.err = err_word;
  rc = few ? launch_few<kFbStore>(ws + l.hq, P, down, d, max_tiles * d.tiles_n, st)
           : launch_gemm<256, kFbStore>(ws + l.hq, P, down, d, max_tiles * d.tiles_n, st);
  if (rc) return rc;
  const unsigned blocks = (unsigned)std::min<int64_t>((T * (H / 8) + 255) / 256, (int64_t)device_sm_count() * 16);
  fb_combine_kernel<<<blocks, 256, 0, st>>>(floats(l.y), ints(l.pair_row),
                                            top_k_weights, T, (int)k, H, reinterpret_cast<__nv_bfloat16*>(out));
  return check_launch("fb_combine_kernel");
}

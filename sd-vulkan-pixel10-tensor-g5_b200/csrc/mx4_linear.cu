// mx4_linear.cu — y = act(x w^T + bias + residual) of two MXFP4 operands (format: mx4.cuh).
//
// mx4_rows_kernel: the product on the CUDA cores, one warp per output column (value and gate column for GEGLU)
// and up to MB rows. A lane takes 16 columns at a time (8 bytes of each operand): the codes decode to fp16
// exactly, and the eight products a half of each pair adds up stay exact in fp16 (at most 8 * 36 = 288 in steps of
// 1/4: 1152 steps, fewer than the 2048 an fp16 significand holds). Block scales, and the sums over blocks, are fp32.
#include <algorithm>
#include <atomic>

#include "mx4.cuh"
#include "sdg_kernels.h"
#include "sdg_launch.h"
#include "sdg_ptx.cuh"
#include "sdg_tma.h"

namespace sdg {
namespace {

constexpr int kRowsWarps = 8;

// y * sigmoid(y), a few fp32 ulps
__device__ __forceinline__ float silu_fine(float y) { return __fdividef(y, 1.f + __expf(-y)); }

template <typename T, int MB, bool GEGLU>
__global__ void __launch_bounds__(32 * kRowsWarps) mx4_rows_kernel(Mx4LinearArgs a) {
  const int lane = threadIdx.x & 31;
  const int nout = GEGLU ? a.N / 2 : a.N;
  const int n = blockIdx.x * kRowsWarps + (threadIdx.x >> 5);
  const int m0 = blockIdx.y * MB;
  pdl_wait();
  pdl_trigger();
  if (n >= nout) return;
  constexpr int NW = GEGLU ? 2 : 1;
  const int kp = mx_kp(a.K), kts = mx_ktiles(a.K);
  int wr[NW];  // weight rows: GEGLU interleaves 16 value rows and their 16 gate rows
  wr[0] = GEGLU ? (n >> 4) * 32 + (n & 15) : n;
  if (GEGLU) wr[NW - 1] = wr[0] + 16;
  float acc[NW][MB];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[w][i] = 0.f;
  for (int u = lane; u < kp / 16; u += 32) {
    const int b = u >> 1;
    __half2 wv[NW][8];
    float wsc[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const uint2 q = *(reinterpret_cast<const uint2*>(a.wcodes + (size_t)wr[w] * (kp / 2)) + u);
      wsc[w] = mx_pow2(a.wscales[((size_t)(wr[w] >> 7) * kts + (b >> 2)) * kMxTileBytes + mx_scale_byte(wr[w], b)]);
      __half2 h[4];
      mx_decode8(q.x, h);
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[w][i] = h[i];
      mx_decode8(q.y, h);
#pragma unroll
      for (int i = 0; i < 4; ++i) wv[w][4 + i] = h[i];
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int m = m0 + i;
      if (m >= a.M) break;
      const uint2 q = *(reinterpret_cast<const uint2*>(a.xcodes + (size_t)m * (kp / 2)) + u);
      const float xsc = mx_pow2(a.xscales[((size_t)(m >> 7) * kts + (b >> 2)) * kMxTileBytes + mx_scale_byte(m, b)]);
      __half2 h0[4], h1[4];
      mx_decode8(q.x, h0);
      mx_decode8(q.y, h1);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        __half2 s = __hmul2(h0[0], wv[w][0]);
#pragma unroll
        for (int j = 1; j < 4; ++j) s = __hfma2(h0[j], wv[w][j], s);
#pragma unroll
        for (int j = 0; j < 4; ++j) s = __hfma2(h1[j], wv[w][4 + j], s);
        const float2 f = __half22float2(s);
        acc[w][i] += (f.x + f.y) * xsc * wsc[w];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) {
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int o = 16; o; o >>= 1) acc[w][i] += __shfl_xor_sync(0xffffffffu, acc[w][i], o);
    const int m = m0 + i;
    if (lane == i && m < a.M) {
      float v = acc[0][i] + (a.bias ? a.bias[wr[0]] : 0.f);
      if (GEGLU) {
        v *= gelu_as(acc[NW - 1][i] + (a.bias ? a.bias[wr[NW - 1]] : 0.f));
      } else {
        if (a.residual) v += MxElem<T>::get(static_cast<const T*>(a.residual)[(size_t)m * a.N + n]);
        if (a.act == 1) v = silu_fine(v);
      }
      static_cast<T*>(a.y)[(size_t)m * nout + n] = MxElem<T>::put(v);
    }
  }
}

template <typename T, int MB>
cudaError_t launch_rows(const Mx4LinearArgs& a, cudaStream_t s) {
  const int nout = a.act == 2 ? a.N / 2 : a.N;
  const dim3 grid((nout + kRowsWarps - 1) / kRowsWarps, (a.M + MB - 1) / MB);
  auto k = a.act == 2 ? mx4_rows_kernel<T, MB, true> : mx4_rows_kernel<T, MB, false>;
  return launch_kernel(k, grid, dim3(32 * kRowsWarps), 0, s, 0, a);
}

// ------------------------------------------------------------------ tensor-core product
// mx4_gemm_kernel: persistent, warp-specialised, one CTA per SM, 128 x BN output tiles.
//   warp 0      producer: per stage (256 columns of K) the 128 B-swizzled code tiles of x and w by TMA, and their
//               scale tiles by untiled bulk copies (a tile's 512 bytes are contiguous)
//   warp 1      TMEM allocator and issuer: per stage the scale tiles into TMEM (tcgen05.cp), then up to four
//               tcgen05.mma.kind::mxf4 (K = 64); copies and MMAs of one thread execute in order
//   warps 2..9  epilogue, two per TMEM lane quadrant: 32 rows x 64 accumulator columns at a time through a
//               swizzled shared-memory panel that TMA fills with the residual beforehand and stores from afterwards,
//               so global memory is only touched in full lines and never waited for by the arithmetic
// Accumulators are double-buffered in TMEM. n is the fastest tile index: the tiles in flight share rows of x, and w
// (at most a few MB) stays in L2.
constexpr int kGBM = 128;
constexpr int kGStageCols = 256;  // K columns per stage: one 128-byte swizzled row of codes
constexpr int kGEpiWarps = 8;
constexpr int kGThreads = 64 + 32 * kGEpiWarps;

template <int BN, bool GEGLU>
struct GCfg {
  static constexpr int kBTiles = (BN + kMxTileRows - 1) / kMxTileRows;  // scale tiles of w per 128 columns of K
  static constexpr uint32_t kABytes = kGBM * 128, kBBytes = BN * 128;
  static constexpr uint32_t kSfBytes = 2 * kMxTileBytes * (1 + kBTiles);
  static constexpr uint32_t kStageBytes = kABytes + kBBytes + kSfBytes;
  static constexpr int kPW = GEGLU ? 32 : 64;                 // output columns of a panel (64 accumulator columns)
  static constexpr uint32_t kPanelBytes = 32 * kPW * 2;
  static constexpr int kHalves = BN >= 128 ? 2 : 1;           // BN = 64: the two warps of a quadrant take turns on tiles
  static constexpr uint32_t kTail = kGEpiWarps * 64 * 4 + 512;  // bias, barriers, TMEM slot
  static constexpr int kStages = (232448 - 1024 - kTail - 2 * kGEpiWarps * kPanelBytes) / kStageBytes;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + 2 * kGEpiWarps * kPanelBytes + kTail;
  static constexpr uint32_t kSfCols = 8 + 8 * kBTiles;        // TMEM columns of one stage's scales
  static constexpr uint32_t kTmemCols = 2 * BN + 2 * kSfCols <= 256 ? 256 : 512;
  static_assert(2 * BN + 2 * kSfCols <= 512 && kStages >= 3, "tile does not fit");
};

struct GemmMx4Dev {
  int M, N, K;
  const uint8_t* xs;
  const uint8_t* ws;
  const float* bias;
  int residual;
  int* err;
};

template <int BN, typename T, int ACT>
__global__ void __launch_bounds__(kGThreads, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_r,
                    const GemmMx4Dev p) {
  constexpr bool GEGLU = ACT == 2;
  using C = GCfg<BN, GEGLU>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sPanel = smem + S * (C::kABytes + C::kBBytes);
  uint8_t* sSf = sPanel + 2 * kGEpiWarps * C::kPanelBytes;
  float* sBias = reinterpret_cast<float*>(sSf + S * C::kSfBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sBias + kGEpiWarps * 64);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5 + 2 * kGEpiWarps);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * S + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * S + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * S + 4);
  auto res_bar = [&](int w, int b) { return bar0 + 8u * (2 * S + 5 + 2 * w + b); };

  const int num_m = (p.M + kGBM - 1) / kGBM, num_n = (p.N + BN - 1) / BN;
  const long long num_tiles = (long long)num_m * num_n;
  const int kp = mx_kp(p.K), kts = mx_ktiles(p.K);
  const int nst = (kp + kGStageCols - 1) / kGStageCols;  // stages per tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), C::kHalves * 4);
    }
    mbar_init(drain_bar, 1);
    for (int w = 0; w < kGEpiWarps; ++w)
      for (int b = 0; b < 2; ++b) mbar_init(res_bar(w, b), 1);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_y);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      pdl_wait();
      uint32_t it = 0;
      bool ok = true;
      for (long long tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        const int m0 = (int)(tile / num_n) * kGBM, n0 = (int)(tile % num_n) * BN;
        const uint8_t* xs = p.xs + (size_t)(m0 / kMxTileRows) * kts * kMxTileBytes;
        const uint8_t* ws = p.ws + (size_t)(n0 / kMxTileRows) * kts * kMxTileBytes;
        for (int k = 0; k < nst; ++k, ++it) {
          const int s = it % S;
          if (!mbar_wait(empty_bar(s), ((it / S) & 1u) ^ 1u, p.err, kDevTimeoutEmpty)) { ok = false; break; }
          const uint32_t sfb = (uint32_t)min(2, kts - 2 * k) * kMxTileBytes;  // scale bytes per 128 rows
          int wt = 0;  // scale tiles of w that exist below row N (a tile behind N multiplies columns never stored)
          for (int j = 0; j < C::kBTiles; ++j) wt += n0 + j * kMxTileRows < p.N;
          mbar_arrive_expect_tx(full_bar(s), C::kABytes + C::kBBytes + sfb * (1 + wt));
          const uint32_t dA = smem_u32(smem + s * C::kABytes);
          const uint32_t dB = smem_u32(smem + S * C::kABytes + s * C::kBBytes);
          const uint32_t dS = smem_u32(sSf + s * C::kSfBytes);
          tma_load_2d(dA, &map_x, full_bar(s), k * 128, m0);
          tma_load_2d(dB, &map_w, full_bar(s), k * 128, n0);
          bulk_load(dS, xs + (size_t)k * 2 * kMxTileBytes, sfb, full_bar(s));
          for (int j = 0; j < wt; ++j)
            bulk_load(dS + (1 + j) * 2 * kMxTileBytes, ws + ((size_t)j * kts + k * 2) * kMxTileBytes, sfb, full_bar(s));
        }
      }
      // abort: every copy in flight lands before the shared memory is released
      if (!ok)
        for (uint32_t q = it > (uint32_t)S ? it - S : 0; q < it; ++q)
          mbar_drain(full_bar(q % S), (q / S) & 1u, p.err, kDevTimeoutDrain);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t it = 0, tl = 0;
      bool ok = true;
      for (long long tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++tl) {
        const int n0 = (int)(tile % num_n) * BN;
        const uint32_t acc = tl & 1u;
        if (!mbar_wait(tempty_bar(acc), ((tl >> 1) & 1u) ^ 1u, p.err, kDevTimeoutAcc)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        const uint32_t n_off = (uint32_t)(n0 % kMxTileRows) / 32u;  // BN = 64: the tile's half of its scale tile
        for (int k = 0; k < nst; ++k, ++it) {
          const int s = it % S;
          if (!mbar_wait(full_bar(s), (it / S) & 1u, p.err, kDevTimeoutFull)) { ok = false; break; }
          const uint32_t sf = tmem_base + 2 * BN + (it & 1u) * C::kSfCols;
          const uint32_t dS = smem_u32(sSf + s * C::kSfBytes);
          const int cols = min(kGStageCols, kp - k * kGStageCols);
          const int nkt = (cols + kMxTileCols - 1) / kMxTileCols;
          for (int t = 0; t < nkt; ++t) {  // TMEM: [x: 4 columns per 128 of K] [w: 4 columns per tile, per 128 of K]
            tmem_copy_scales(sf + 4 * t, sdesc_scales(dS + t * kMxTileBytes));
#pragma unroll
            for (int j = 0; j < C::kBTiles; ++j)
              tmem_copy_scales(sf + 8 + 4 * (t * C::kBTiles + j), sdesc_scales(dS + (2 * (1 + j) + t) * kMxTileBytes));
          }
          const uint64_t da = sdesc_sw128(smem_u32(smem + s * C::kABytes), 16, 1024);
          const uint64_t db = sdesc_sw128(smem_u32(smem + S * C::kABytes + s * C::kBBytes), 16, 1024);
          const int nmma = (cols + 63) / 64;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < nmma)
              mma_mxf4_ss(d_tmem, da + 2ull * j, db + 2ull * j, idesc_mxf4(kGBM, BN, (j & 1) * 2), sf + 4 * (j >> 1),
                          sf + 8 + 4 * (j >> 1) * C::kBTiles + n_off, (k | j) != 0);
          mma_commit(empty_bar(s));
        }
        if (!ok) break;
        mma_commit(tfull_bar(acc));
      }
      mma_commit(drain_bar);  // every issued copy and MMA has retired before TMEM is released
      mbar_drain(drain_bar, 0, p.err, kDevTimeoutDrain);
    }
  } else {
    pdl_wait();
    const int w = warp - 2, lg = warp & 3, half = w >> 2;
    const int rl = lg * 32 + lane;
    float* bias_s = sBias + w * 64;
    constexpr int kPanels = BN / 64;                // panels of a tile
    constexpr int kStep = C::kHalves;               // this warp's panels: half, half + kStep, ...
    const int first = kStep == 2 ? half : 0;
    uint8_t* pan0 = sPanel + (w * 2) * C::kPanelBytes;
    // the panel after (tile, pn): the next of this tile, else the first of this warp's next tile
    const long long tstep = kStep == 2 ? gridDim.x : 2ll * gridDim.x;
    const long long tfirst = kStep == 2 ? blockIdx.x : blockIdx.x + (long long)half * gridDim.x;
    uint32_t q = 0, tl = kStep == 2 ? 0 : (uint32_t)half;
    auto load_res = [&](long long tile, int pn, uint32_t b) {  // lane 0
      mbar_arrive_expect_tx(res_bar(w, b), C::kPanelBytes);
      tma_load_2d(smem_u32(pan0 + b * C::kPanelBytes), &map_r, res_bar(w, b), (int)(tile % num_n) * BN + pn * 64,
                  (int)(tile / num_n) * kGBM + lg * 32);
    };
    if (p.residual && lane == 0 && tfirst < num_tiles) load_res(tfirst, first, 0);
    bool ok = true;
    for (long long tile = tfirst; tile < num_tiles; tile += tstep, tl += 3 - kStep) {
      const uint32_t acc = tl & 1u;
      const int m0 = (int)(tile / num_n) * kGBM, n0 = (int)(tile % num_n) * BN;
      ok = mbar_wait(tfull_bar(acc), (tl >> 1) & 1u, p.err, kDevTimeoutAcc);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
#pragma unroll 1
      for (int pn = first; pn < kPanels; pn += kStep, ++q) {
        const uint32_t b = q & 1u;
        uint8_t* pan = pan0 + b * C::kPanelBytes;
        const int n = n0 + pn * 64;
        if (lane == 0) {
          if (p.residual) {
            bulk_wait_read<0>();  // the other buffer's store has read it: it may take the next residual
            const bool more = pn + kStep < kPanels;
            const long long nt = more ? tile : tile + tstep;
            if (nt < num_tiles) load_res(nt, more ? pn + kStep : first, b ^ 1u);
          } else {
            bulk_wait_read<1>();  // this buffer's previous store has read it
          }
        }
        bias_s[lane] = p.bias && n + lane < p.N ? p.bias[n + lane] : 0.f;
        bias_s[32 + lane] = p.bias && n + 32 + lane < p.N ? p.bias[n + 32 + lane] : 0.f;
        __syncwarp();
        if (p.residual) {
          ok = mbar_wait(res_bar(w, b), (q >> 1) & 1u, p.err, kDevTimeoutEmpty);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        }
        const uint32_t t_row = tmem_base + acc * BN + pn * 64 + (static_cast<uint32_t>(lg * 32) << 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tmem_ld32(t_row + 32 * h, r);
          tmem_wait_ld();
          const float4* b4 = reinterpret_cast<const float4*>(bias_s + 32 * h);
          if constexpr (GEGLU) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float4 bv = b4[2 * g + e], bg = b4[4 + 2 * g + e];
                const int i = 8 * g + 4 * e;
                v[4 * e] = (__uint_as_float(r[i]) + bv.x) * gelu_as(__uint_as_float(r[16 + i]) + bg.x);
                v[4 * e + 1] = (__uint_as_float(r[i + 1]) + bv.y) * gelu_as(__uint_as_float(r[17 + i]) + bg.y);
                v[4 * e + 2] = (__uint_as_float(r[i + 2]) + bv.z) * gelu_as(__uint_as_float(r[18 + i]) + bg.z);
                v[4 * e + 3] = (__uint_as_float(r[i + 3]) + bv.w) * gelu_as(__uint_as_float(r[19 + i]) + bg.w);
              }
              // 64-byte rows: 16-byte chunk index XOR address bits 7..8
              mx_store8<T>(reinterpret_cast<T*>(pan + lane * 64 + (((2 * h + g) ^ ((lane >> 1) & 3)) << 4)), v);
            }
          } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              // 128-byte rows: 16-byte chunk index XOR address bits 7..9
              T* at = reinterpret_cast<T*>(pan + lane * 128 + (((4 * h + g) ^ (lane & 7)) << 4));
              const float4 b0 = b4[2 * g], b1 = b4[2 * g + 1];
              float v[8] = {__uint_as_float(r[8 * g]) + b0.x,     __uint_as_float(r[8 * g + 1]) + b0.y,
                            __uint_as_float(r[8 * g + 2]) + b0.z, __uint_as_float(r[8 * g + 3]) + b0.w,
                            __uint_as_float(r[8 * g + 4]) + b1.x, __uint_as_float(r[8 * g + 5]) + b1.y,
                            __uint_as_float(r[8 * g + 6]) + b1.z, __uint_as_float(r[8 * g + 7]) + b1.w};
              if (p.residual) {
                float rv[8];
                mx_unpack8<T>(*reinterpret_cast<const uint4*>(at), rv);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += rv[i];
              }
              if constexpr (ACT == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = silu_fine(v[i]);
              }
              mx_store8<T>(at, v);
            }
          }
        }
        if (pn + kStep >= kPanels) {  // the accumulator's last read of this warp
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(tempty_bar(acc));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&map_y, smem_u32(pan), GEGLU ? n / 2 : n, m0 + lg * 32);
          bulk_commit();
        }
      }
      if (!ok) break;
    }
    if (lane == 0) {
      // abort: the residual loads in flight (panel q's, and q + 1's where it was issued) land first
      if (!ok && p.residual) spin_ns(200000);
      bulk_wait_read<0>();
    }
    (void)rl;
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

template <int BN, typename T, int ACT>
cudaError_t launch_gemm_mx4(const Mx4LinearArgs& a, int* err, cudaStream_t s) {
  using C = GCfg<BN, ACT == 2>;
  auto k = mx4_gemm_kernel<BN, T, ACT>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    if (e != cudaSuccess) return e;
    ready[dev].store(true, std::memory_order_release);
  }
  const int kp = mx_kp(a.K), nout = ACT == 2 ? a.N / 2 : a.N;
  CUtensorMap mx, mw, my, mr;
  auto codes = [&](CUtensorMap* m, const uint8_t* base, int rows, uint32_t box_rows) {
    const uint64_t dims[2] = {(uint64_t)kp / 2, (uint64_t)rows}, str[1] = {(uint64_t)kp / 2};
    const uint32_t box[2] = {128, box_rows};
    return make_tmap(m, base, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT8);
  };
  auto panel = [&](CUtensorMap* m, const void* base) {
    const uint64_t dims[2] = {(uint64_t)nout, (uint64_t)a.M}, str[1] = {(uint64_t)nout * 2};
    const uint32_t box[2] = {(uint32_t)C::kPW, 32};
    return make_tmap(m, base, 2, dims, str, box, C::kPW == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                     CU_TENSOR_MAP_DATA_TYPE_UINT16);
  };
  if (!codes(&mx, a.xcodes, a.M, kGBM) || !codes(&mw, a.wcodes, a.N, BN) || !panel(&my, a.y) ||
      !panel(&mr, a.residual ? a.residual : a.y))
    return cudaErrorInvalidValue;
  GemmMx4Dev p;
  p.M = a.M; p.N = a.N; p.K = a.K;
  p.xs = a.xscales; p.ws = a.wscales; p.bias = a.bias; p.residual = a.residual != nullptr; p.err = err;
  const long long tiles = (long long)((a.M + kGBM - 1) / kGBM) * ((a.N + BN - 1) / BN);
  const int grid = (int)std::min<long long>(tiles, num_sms());
  return launch_kernel(k, dim3(grid), dim3(kGThreads), C::kSmem, s, 0, mx, mw, my, mr, p);
}

template <typename T, int ACT>
cudaError_t gemm_bn(const Mx4LinearArgs& a, int* err, cudaStream_t s) {
  const long long tiles = (long long)((a.M + kGBM - 1) / kGBM) * ((a.N + 127) / 128);
  if (tiles >= num_sms()) return launch_gemm_mx4<128, T, ACT>(a, err, s);
  return launch_gemm_mx4<64, T, ACT>(a, err, s);
}

template <typename T>
cudaError_t linear_t(const Mx4LinearArgs& a, int* err, cudaStream_t s) {
  if (a.M == 1) return launch_rows<T, 1>(a, s);
  if (a.M <= 8) return launch_rows<T, 4>(a, s);
  switch (a.act) {
    case 1: return gemm_bn<T, 1>(a, err, s);
    case 2: return gemm_bn<T, 2>(a, err, s);
    default: return gemm_bn<T, 0>(a, err, s);
  }
}

}  // namespace

cudaError_t launch_mx4_linear(const Mx4LinearArgs& a, int* dev_err, cudaStream_t s) {
  return a.dtype == kBF16 ? linear_t<__nv_bfloat16>(a, dev_err, s) : linear_t<__half>(a, dev_err, s);
}

}  // namespace sdg

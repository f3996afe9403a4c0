// mx4_linear.cu — y = act(x w^T + bias + residual) of two MXFP4 operands (format: mx4.cuh).
//
// mx4_rows_kernel: up to eight rows (time embeddings, single tokens), on the CUDA cores: one warp per output column
// (value and gate column for GEGLU) for all rows. A lane takes 16 columns at a time (8 bytes of each operand): the
// codes decode to fp16 exactly, and the eight products a half of each pair adds up stay exact in fp16 (at most 8 * 36 =
// 288 in steps of 1/4: 1152 steps, fewer than the 2048 an fp16 significand holds). Block scales, and the sums over
// blocks, are fp32. Of two scales the smaller multiplies a sum first: that product (k / 4 2^e with k <= 2304, e >= -127) is
// exact, and where it overflows the true one does too, so a finite term stays finite and a zero one zero. A plain x is quantised by every block itself, so that the whole call is one launch: it is bound by
// launch latency and one pass over the weights.
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
constexpr int kRowsThreads = 32 * kRowsWarps;

// y * sigmoid(y). __expf is off by at most 2 + 1.16 |y| ulps, which counts for y < 0 (the value is about y exp(y) there) and
// stays far below the output's rounding; below y = -87.3, where |value| < 1.1e-36, __fdividef may give 0.
__device__ __forceinline__ float silu_fine(float y) { return __fdividef(y, 1.f + __expf(-y)); }

// x gelu(x) factor: gelu of two values, x Phi(x) with erf from Abramowitz & Stegun 7.1.26 as in gelu_as, written as
// max(x, 0) - |x| q with q = poly(t) exp(-x^2 / 2) / 2 = 1 - Phi(|x|), so that both signs share it without
// cancellation; in f32x2 arithmetic with one reciprocal for both values (three MUFU instructions a pair). |x| is
// capped at 128 where q is long zero, which keeps the product of the denominators and infinite x finite.
__device__ __forceinline__ float2 gelu_pair(float2 x) {
  const float2 a = make_float2(fminf(fabsf(x.x), 128.f), fminf(fabsf(x.y), 128.f));
  const float2 den = fma_f32x2(a, make_float2(0.23164189f, 0.23164189f), make_float2(1.f, 1.f));  // p / sqrt(2)
  const float r = rcp_approx(den.x * den.y);
  const float2 t = mul_f32x2(make_float2(r, r), make_float2(den.y, den.x));
  auto c2 = [](float c) { return make_float2(c, c); };
  float2 q = fma_f32x2(t, c2(0.5f * 1.061405429f), c2(0.5f * -1.453152027f));
  q = fma_f32x2(q, t, c2(0.5f * 1.421413741f));
  q = fma_f32x2(q, t, c2(0.5f * -0.284496736f));
  q = fma_f32x2(q, t, c2(0.5f * 0.254829592f));
  q = mul_f32x2(q, t);
  const float2 e = mul_f32x2(mul_f32x2(x, x), c2(-0.72134752f));  // -x^2 / 2 log2(e)
  q = mul_f32x2(q, make_float2(ex2_approx(e.x), ex2_approx(e.y)));
  return fma_f32x2(make_float2(-a.x, -a.y), q, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
}

// a.x set (QUANT): the block quantises its rows of x itself, once, into shared memory; else it copies the operand there.
template <typename T, int MB, bool GEGLU, bool QUANT>
__global__ void __launch_bounds__(kRowsThreads) mx4_rows_kernel(Mx4LinearArgs a) {
  extern __shared__ __align__(16) uint8_t rows_smem[];
  constexpr int NW = GEGLU ? 2 : 1;
  const int lane = threadIdx.x & 31;
  const int nout = GEGLU ? a.N / 2 : a.N;
  const int n = min((int)(blockIdx.x * kRowsWarps + (threadIdx.x >> 5)), nout - 1);
  const bool live = blockIdx.x * kRowsWarps + (threadIdx.x >> 5) < nout;
  const int kp = mx_kp(a.K), kts = mx_ktiles(a.K), units = kp / 16;
  const int rows = min(MB, a.M);
  uint8_t* xc = rows_smem;                                          // [MB][kp / 2] codes
  float* xs = reinterpret_cast<float*>(rows_smem + MB * (kp / 2));  // [MB][kp / 32] scales
  int wr[NW];  // weight rows: GEGLU interleaves 16 value rows and their 16 gate rows
  wr[0] = GEGLU ? (n >> 4) * 32 + (n & 15) : n;
  if (GEGLU) wr[NW - 1] = wr[0] + 16;
  pdl_wait();
  pdl_trigger();
  // this lane's first weights, in flight while x is quantised
  constexpr int PRE = 4;
  uint2 wq[NW][PRE];
  uint32_t we[NW][PRE];
  auto load_w = [&](int u0) {
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int i = 0; i < PRE; ++i) {
        const int u = u0 + 32 * i, b = u >> 1;
        wq[w][i] = make_uint2(0u, 0u);
        we[w][i] = 0;
        if (u < units) {
          wq[w][i] = *(reinterpret_cast<const uint2*>(a.wcodes + (size_t)wr[w] * (kp / 2)) + u);
          we[w][i] = a.wscales[((size_t)(wr[w] >> 7) * kts + (b >> 2)) * kMxTileBytes + mx_scale_byte(wr[w], b)];
        }
      }
  };
  load_w(lane);
  if constexpr (QUANT) {
    const T* x = static_cast<const T*>(a.x);
    const bool vec = a.K % 8 == 0 && (a.ldx * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
    const int per = kp / 8, total = rows * per;  // units of eight columns; a quad of lanes holds one block
    for (int i0 = 0; i0 < total; i0 += kRowsThreads) {
      const int i = i0 + threadIdx.x, r = min(i / per, rows - 1), c = (i - r * per) * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
      if (i < total) {
        const T* src = x + (size_t)r * a.ldx + c;
        if (vec) {
          if (c < a.K) mx_unpack8<T>(*reinterpret_cast<const uint4*>(src), v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < a.K) v[e] = MxElem<T>::get(src[e]);
        }
      }
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7FFFFFFFu);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const uint32_t e = mx_exponent(m);
      uint32_t q[1];
      mx_codes<8>(v, e, q);
      if (i < total) {
        *reinterpret_cast<uint32_t*>(xc + r * (kp / 2) + c / 2) = q[0];
        if ((i & 3) == 0) xs[r * (kp / 32) + c / 32] = mx_pow2(e);
      }
    }
  } else {
    for (int i = threadIdx.x; i < rows * (kp / 32); i += kRowsThreads) {
      const int r = i / (kp / 32), b = i - r * (kp / 32);
      reinterpret_cast<uint4*>(xc)[i] = reinterpret_cast<const uint4*>(a.xcodes)[i];
      xs[i] = mx_pow2(a.xscales[(size_t)(b >> 2) * kMxTileBytes + mx_scale_byte(r, b)]);
    }
  }
  __syncthreads();
  float acc[NW][MB];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[w][i] = 0.f;
  for (int u0 = lane; u0 < units; u0 += 32 * PRE) {
    if (u0 != lane) load_w(u0);
#pragma unroll
    for (int i = 0; i < PRE; ++i) {
      const int u = u0 + 32 * i;
      if (u >= units) break;
      __half2 wv[NW][8];
      float wsc[NW];
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        wsc[w] = mx_pow2(we[w][i]);
        __half2 h[4];
        mx_decode8(wq[w][i].x, h);
#pragma unroll
        for (int j = 0; j < 4; ++j) wv[w][j] = h[j];
        mx_decode8(wq[w][i].y, h);
#pragma unroll
        for (int j = 0; j < 4; ++j) wv[w][4 + j] = h[j];
      }
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        if (m >= rows) break;
        const uint2 q = *(reinterpret_cast<const uint2*>(xc + m * (kp / 2)) + u);
        const float xsc = xs[m * (kp / 32) + (u >> 1)];
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
          const uint32_t a = __float_as_uint(xsc), b = __float_as_uint(wsc[w]);  // as integers: a NaN is the larger
          acc[w][m] += (f.x + f.y) * __uint_as_float(min(a, b)) * __uint_as_float(max(a, b));
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m) {
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int o = 16; o; o >>= 1) acc[w][m] += __shfl_xor_sync(0xffffffffu, acc[w][m], o);
    if (lane == m && m < rows && live) {
      float v = acc[0][m] + (a.bias ? a.bias[wr[0]] : 0.f);
      if (GEGLU) {
        v *= gelu_as(acc[NW - 1][m] + (a.bias ? a.bias[wr[NW - 1]] : 0.f));
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
  const int nout = a.act == 2 ? a.N / 2 : a.N, kp = mx_kp(a.K);
  const dim3 grid((nout + kRowsWarps - 1) / kRowsWarps);
  const size_t smem = (size_t)MB * (kp / 2 + kp / 8);
  auto k = a.x ? (a.act == 2 ? mx4_rows_kernel<T, MB, true, true> : mx4_rows_kernel<T, MB, false, true>)
               : (a.act == 2 ? mx4_rows_kernel<T, MB, true, false> : mx4_rows_kernel<T, MB, false, false>);
  return launch_kernel(k, grid, dim3(kRowsThreads), smem, s, 0, a);
}

// ------------------------------------------------------------------ tensor-core product
// mx4_gemm_kernel: persistent, warp-specialised, one CTA per SM, 128 x BN output tiles.
// The producer's and the issuer's loops run on all lanes with one elected lane issuing: the operands then stay in uniform
// registers. With the loops on one lane (a divergent branch) every tcgen05 instruction paid for moving its operands
// there: 65536 x 640 x 2560 94 us, 76 us with the issuer converted, 72.6 us with both.
//   warp 0      producer: per stage (256 columns of K) the 128 B-swizzled code tiles of x and w by TMA, and their
//               scale tiles by untiled bulk copies (a tile's 512 bytes are contiguous)
//   warp 1      TMEM allocator and issuer: per stage the scale tiles into TMEM (tcgen05.cp), then up to four
//               tcgen05.mma.kind::mxf4 (K = 64); copies and MMAs of one thread execute in order
//   others      epilogue, two sets of BN / 16 warps that take turns on the tiles (the activations would otherwise be
//               bound by too few warps to hide their latencies: GEGLU 8192 x 2560 x 320 ran 18.5 us with one set). A warp
//               takes 32 rows x 64 accumulator columns through a swizzled shared-memory panel that TMA fills with the
//               residual beforehand and stores from afterwards, so global memory is only touched in full lines
// Accumulators are double-buffered in TMEM, one per set.
// PAIR: two CTAs on two SMs compute 256 x BN with tcgen05.mma.cta_group::2, each with its 128 rows of x and half the rows
// of w: a quarter fewer bytes into and out of shared memory per product, six stages instead of four, but two CTAs
// to synchronise per tile. It pays for long rows only (both sides at kPairStages below).
// FUSE (BN = 64): x is quantised on the way, so the call is one launch without scratch: one more warp brings tiles of
// 128 rows x 128 columns of x into a ring by TMA and sixteen more quantise them into the code stages. (Loading x into
// registers a stage ahead instead ran four times slower: the loads in flight share the scoreboard that the pass in
// hand waits on.) Every n tile quantises its rows of x again: for small products only.
// n is the fastest tile index: the tiles in flight share rows of x, and w (at most a few MB) stays in L2.
constexpr int kGBM = 128;
constexpr int kGStageCols = 256;  // K columns per stage: one 128-byte swizzled row of codes
constexpr int kGQuantWarps = 16;
constexpr int kGRawStages = 3;
constexpr uint32_t kGRawBytes = kGBM * 128 * 2;  // 128 columns of 16 bits, as two 128 B-swizzled boxes of 64

template <int BN, bool GEGLU, bool FUSE, bool PAIR>
struct GCfg {
  static constexpr int kBRows = PAIR ? BN / 2 : BN;  // rows of w in this CTA
  static constexpr uint32_t kABytes = kGBM * 128, kBBytes = kBRows * 128;
  static_assert(BN <= kMxTileRows, "one scale tile of w per 128 columns of K");
  static constexpr uint32_t kSfBytes = 4 * kMxTileBytes;  // two scale tiles of x, two of w
  static constexpr uint32_t kStageBytes = kABytes + kBBytes + kSfBytes;
  static constexpr int kPW = GEGLU ? 32 : 64;                 // output columns of a panel (64 accumulator columns)
  static constexpr uint32_t kPanelBytes = 32 * kPW * 2;
  static_assert(!FUSE || BN == 64, "the fused form has 64-wide tiles");
  static_assert(!PAIR || (BN == 128 && !FUSE), "pairs have 128-wide tiles");
  static constexpr int kSets = FUSE ? 1 : 2;
  static constexpr int kSetWarps = 4 * (BN / 64), kEpiWarps = kSets * kSetWarps;
  static constexpr int kThreads = 64 + 32 * (kEpiWarps + (FUSE ? kGQuantWarps + 1 : 0));
  static constexpr uint32_t kRawRing = FUSE ? kGRawStages * kGRawBytes : 0;
  static constexpr uint32_t kTail = kEpiWarps * 64 * 4 + 512;  // bias, barriers, TMEM slot
  static constexpr int kStages = (232448 - 1024 - kTail - kEpiWarps * kPanelBytes - kRawRing) / kStageBytes;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kEpiWarps * kPanelBytes + kRawRing + kTail;
  static constexpr uint32_t kSfCols = 16;                     // TMEM columns of one stage's scales
  static constexpr uint32_t kTmemCols = 2 * BN + 2 * kSfCols <= 256 ? 256 : 512;
  static_assert(2 * BN + 2 * kSfCols <= 512 && kStages >= 3, "tile does not fit");
  static_assert(!FUSE || kGBM == 2 * 4 * kGQuantWarps, "two passes of four rows a warp");
  static_assert((2 * kStages + 5 + kEpiWarps + 2 * kGRawStages) * 8 + 12 <= 512, "barriers do not fit");
};

// A block's walk over the tiles first, first + step, ... (n fastest), without a division per tile.
struct TileWalk {
  int m, n;  // tile coordinates
  int dm, dn, num_m, num_n;
  __device__ TileWalk(int first, int step, int num_m_, int num_n_) : num_m(num_m_), num_n(num_n_) {
    m = first / num_n;
    n = first - m * num_n;
    dm = step / num_n;
    dn = step - dm * num_n;
  }
  __device__ __forceinline__ bool valid() const { return m < num_m; }
  __device__ __forceinline__ void next() {
    m += dm;
    n += dn;
    if (n >= num_n) {
      n -= num_n;
      ++m;
    }
  }
};

// The bounded waits of a block. A wait that expires records its code in the error word and stops the other waits of its block
// (of both blocks of a pair) through a flag in their shared memory. They do not look at the error word itself: it may be
// shared with other launches, and one that failed must not end the waits of those that follow.
template <bool PAIR>
struct Waits {
  uint32_t stop;  // shared-memory address of the flag
  int* err;
  unsigned long long limit_ns;

  __device__ __forceinline__ bool stopped() const {
    uint32_t v;
    asm volatile("ld.volatile.shared::cta.b32 %0, [%1];" : "=r"(v) : "r"(stop) : "memory");
    return v != 0;
  }
  __device__ __forceinline__ void expire(int code) const {
    atomicCAS(err, 0, code);
    if constexpr (PAIR) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(mapa_shared(stop, r)), "r"(1u) : "memory");
    } else {
      asm volatile("st.volatile.shared::cta.b32 [%0], %1;" ::"r"(stop), "r"(1u) : "memory");
    }
  }
  // CLUSTER: the peer's arrivals count too
  template <bool CLUSTER = false>
  __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int code) const {
    auto done = [&] { return CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity); };
    if (done()) return true;
    const uint64_t t0 = globaltimer();
    for (uint32_t i = 1;; ++i) {
      if (done()) return true;
      if ((i & 255u) == 0u) {
        if (stopped()) return false;
        if (globaltimer() - t0 > limit_ns) {
          expire(code);
          return false;
        }
      }
    }
  }
};

struct GemmMx4Dev {
  int M, N, K;
  const uint8_t* xs;
  const uint8_t* ws;
  const float* bias;
  int residual;
  int* err;
  unsigned long long wait_ns;  // limit of every bounded wait
  int stall_it, stall_who;     // failure-path test: loader stall_who stops before its load number stall_it (-1: never)
};

template <int BN, typename T, int ACT, bool FUSE, bool PAIR>
__global__ void __launch_bounds__(GCfg<BN, ACT == 2, FUSE, PAIR>::kThreads, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                    const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_r,
                    const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_ws,
                    const GemmMx4Dev p) {
  constexpr bool GEGLU = ACT == 2;
  using C = GCfg<BN, GEGLU, FUSE, PAIR>;
  constexpr int TM = PAIR ? 2 * kGBM : kGBM;  // rows of a tile
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sRaw = smem + S * (C::kABytes + C::kBBytes);
  uint8_t* sPanel = sRaw + C::kRawRing;
  uint8_t* sSf = sPanel + C::kEpiWarps * C::kPanelBytes;
  float* sBias = reinterpret_cast<float*>(sSf + S * C::kSfBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sBias + C::kEpiWarps * 64);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 5 + C::kEpiWarps + 2 * kGRawStages);
  uint32_t* issued = tmem_slot + 2;  // stages that this CTA's producer has loaded
  const Waits<PAIR> waits{smem_u32(tmem_slot + 1), p.err, p.wait_ns};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (S + s); };
  auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * S + a); };
  auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * S + 2 + a); };
  const uint32_t drain_bar = bar0 + 8u * (2 * S + 4);
  auto res_bar = [&](int w) { return bar0 + 8u * (2 * S + 5 + w); };
  auto rfull_bar = [&](int s) { return bar0 + 8u * (2 * S + 5 + C::kEpiWarps + s); };
  auto rempty_bar = [&](int s) { return bar0 + 8u * (2 * S + 5 + C::kEpiWarps + kGRawStages + s); };

  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int team = PAIR ? blockIdx.x >> 1 : blockIdx.x, teams = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int num_m = (p.M + TM - 1) / TM, num_n = (p.N + BN - 1) / BN;
  const int kp = mx_kp(p.K), kts = mx_ktiles(p.K);
  const int nst = (kp + kGStageCols - 1) / kGStageCols;  // stages per tile

  if (threadIdx.x == 0) {
    tmem_slot[1] = 0;  // the waits' stop flag
    for (int s = 0; s < S; ++s) {
      mbar_init(full_bar(s), FUSE ? 1 + kGQuantWarps : 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull_bar(a), 1);
      mbar_init(tempty_bar(a), C::kSetWarps * (PAIR ? 2 : 1));  // a pair's warps arrive at the even CTA's
    }
    mbar_init(drain_bar, 1);
    for (int w = 0; w < C::kEpiWarps; ++w) mbar_init(res_bar(w), 1);
    if (FUSE)
      for (int s = 0; s < kGRawStages; ++s) {
        mbar_init(rfull_bar(s), 1);
        mbar_init(rempty_bar(s), kGQuantWarps);
      }
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_y);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc2(smem_u32(tmem_slot), C::kTmemCols);
      tmem_relinquish2();
    } else {
      tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncwarp();
  if constexpr (PAIR)
    cluster_sync_all();  // both CTAs' barriers and TMEM stand before any signal crosses
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // No early trigger: blocks of the next kernel that move in while this one runs hold their SMs' warps and registers
  // unevenly when it ends. Measured on B200, quantise + product in a row: 65536 x 640 x 2560 181 us with a trigger here,
  // 163 us with one after the last MMA, 161 us without; 8192 x 320 x 320 9.3 / 8.3 / 7.8 us.

  uint32_t count = 0;  // stages loaded or filled, raw tiles loaded: what an abort has to wait for
  if (warp == 0) {
    // all lanes walk the loop and wait; one of them issues
    pdl_wait();
    uint32_t it = 0;
    bool ok = true;
    const int stall_it = p.stall_who == rank ? p.stall_it : -1;
    for (TileWalk tw(team, teams, num_m, num_n); tw.valid() && ok; tw.next()) {
      const int m0 = tw.m * TM + rank * kGBM, n0 = tw.n * BN;
      const uint8_t* xs = FUSE ? nullptr : p.xs + (size_t)(m0 / kMxTileRows) * kts * kMxTileBytes;
      const uint8_t* ws = p.ws + (size_t)(n0 / kMxTileRows) * kts * kMxTileBytes;
      // The x tile of this block's next round into L2, by the one block whose next tile is the first of its row, where the
      // rows are long: the ring holds too little to cover HBM's latency (65536 x 640 x 2560 72 -> 66 us; at K <= 1024 the
      // extra requests cost more than they hide)
      TileWalk tn = tw;
      tn.next();
      const bool ahead = !FUSE && nst > 4 && tn.valid() && tn.n == 0;
      const int m1 = tn.m * TM + rank * kGBM;
      for (int k = 0; k < nst; ++k, ++it) {
        const int s = it % S;
        ok = __all_sync(0xffffffffu, waits.wait(empty_bar(s), ((it / S) & 1u) ^ 1u, kDevTimeoutEmpty)) && (int)it != stall_it;
        if (!ok) break;
        const uint32_t sfb = (uint32_t)min(2, kts - 2 * k) * kMxTileBytes;  // scale bytes per 128 rows
        const uint32_t dA = smem_u32(smem + s * C::kABytes);
        const uint32_t dB = smem_u32(smem + S * C::kABytes + s * C::kBBytes);
        const uint32_t dS = smem_u32(sSf + s * C::kSfBytes);
        if (elect_one()) {
          if (ahead) tma_prefetch_2d(&map_x, k * 128, m1);
          if constexpr (PAIR) {
            // both CTAs' bytes count on the even CTA's barrier; scale tiles come through tensor maps (zero behind the last)
            if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * C::kStageBytes);
            const uint32_t fb = mapa_shared(full_bar(s), 0);
            tma_load_2d_pair(dA, &map_x, fb, k * 128, m0);
            tma_load_2d_pair(dS, &map_xs, fb, k * 256, m0 / kMxTileRows);
            tma_load_2d_pair(dB, &map_w, fb, k * 128, n0 + rank * C::kBRows);
            tma_load_2d_pair(dS + 2 * kMxTileBytes, &map_ws, fb, k * 256, n0 / kMxTileRows);
          } else {
            mbar_arrive_expect_tx(full_bar(s), FUSE ? C::kBBytes + sfb : C::kABytes + C::kBBytes + 2 * sfb);
            if constexpr (!FUSE) {
              tma_load_2d(dA, &map_x, full_bar(s), k * 128, m0);
              bulk_load(dS, xs + (size_t)k * 2 * kMxTileBytes, sfb, full_bar(s));
            }
            tma_load_2d(dB, &map_w, full_bar(s), k * 128, n0);
            bulk_load(dS + 2 * kMxTileBytes, ws + (size_t)k * 2 * kMxTileBytes, sfb, full_bar(s));
          }
        }
        __syncwarp();
      }
    }
    count = it;
    if (lane == 0) *issued = it;
  } else if (warp == 1) {
    if (rank == 0) {
      // all lanes walk the loop and wait; one of them issues
      auto copy_scales = [](uint32_t d, uint64_t s) {
        if constexpr (PAIR) tmem_copy_scales2(d, s); else tmem_copy_scales(d, s);
      };
      auto mma = [](uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sa, uint32_t sb, uint32_t accumulate) {
        if constexpr (PAIR) mma_mxf4_ss2(d, a, b, id, sa, sb, accumulate); else mma_mxf4_ss(d, a, b, id, sa, sb, accumulate);
      };
      auto commit = [](uint32_t bar) {  // a pair's signal goes to both CTAs
        if constexpr (PAIR) mma_commit2_mc(bar, 0x3); else mma_commit(bar);
      };
      uint32_t it = 0, tl = 0;
      bool ok = true;
      for (TileWalk tw(team, teams, num_m, num_n); tw.valid() && ok; tw.next(), ++tl) {
        const int n0 = tw.n * BN;
        const uint32_t acc = tl & 1u;
        const uint32_t free_ph = ((tl >> 1) & 1u) ^ 1u;
        ok = __all_sync(0xffffffffu, waits.template wait<PAIR>(tempty_bar(acc), free_ph, kDevTimeoutAcc));
        if (!ok) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        const uint32_t n_off = (uint32_t)(n0 % kMxTileRows) / 32u;  // BN = 64: the tile's half of its scale tile
        for (int k = 0; k < nst; ++k, ++it) {
          const int s = it % S;
          ok = __all_sync(0xffffffffu, waits.wait(full_bar(s), (it / S) & 1u, kDevTimeoutFull));
          if (!ok) break;
          const uint32_t sf = tmem_base + 2 * BN + (it & 1u) * C::kSfCols;
          const uint32_t dS = smem_u32(sSf + s * C::kSfBytes);
          const int cols = min(kGStageCols, kp - k * kGStageCols);
          const int nkt = (cols + kMxTileCols - 1) / kMxTileCols;
          const uint64_t ds = sdesc_scales(dS);
          const uint64_t da = sdesc_sw128(smem_u32(smem + s * C::kABytes), 16, 1024);
          const uint64_t db = sdesc_sw128(smem_u32(smem + S * C::kABytes + s * C::kBBytes), 16, 1024);
          const int nmma = (cols + 63) / 64;
          if (elect_one()) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {  // TMEM: [x: 4 columns per 128 of K] [w: likewise]
              if (t < nkt) {
                copy_scales(sf + 4 * t, ds + (t * kMxTileBytes >> 4));
                copy_scales(sf + 8 + 4 * t, ds + ((2 + t) * kMxTileBytes >> 4));
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < nmma)
                mma(d_tmem, da + 2ull * j, db + 2ull * j, idesc_mxf4(TM, BN, (j & 1) * 2), sf + 4 * (j >> 1),
                    sf + 8 + 4 * (j >> 1) + n_off, (k | j) != 0);
            commit(empty_bar(s));
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elect_one()) commit(tfull_bar(acc));
        __syncwarp();
      }
      if (elect_one()) {
        if constexpr (PAIR) mma_commit2_mc(drain_bar, 0x1); else mma_commit(drain_bar);
      }
      // every issued copy and MMA has retired before TMEM is released
      __syncwarp();
      if (lane == 0) mbar_drain(drain_bar, 0, p.err, kDevTimeoutDrain, p.wait_ns);
    }
  } else if (FUSE && warp == 2 + C::kEpiWarps + kGQuantWarps) {
    // x into the raw ring
    pdl_wait();
    const int nraw = (kp + 127) / 128;
    uint32_t it = 0;
    bool ok = true;
    const int stall_it = p.stall_who == 1 ? p.stall_it : -1;
    for (TileWalk tw(team, teams, num_m, num_n); tw.valid() && ok; tw.next()) {
      const int m0 = tw.m * kGBM;
      for (int k = 0; k < nraw; ++k, ++it) {
        const int s = it % kGRawStages;
        ok = __all_sync(0xffffffffu, waits.wait(rempty_bar(s), ((it / kGRawStages) & 1u) ^ 1u, kDevTimeoutEmpty)) &&
             (int)it != stall_it;
        if (!ok) break;
        const uint32_t d = smem_u32(sRaw + s * kGRawBytes);
        if (elect_one()) {
          mbar_arrive_expect_tx(rfull_bar(s), kGRawBytes);
          tma_load_2d(d, &map_x, rfull_bar(s), k * 128, m0);
          tma_load_2d(d + kGRawBytes / 2, &map_x, rfull_bar(s), k * 128 + 64, m0);
        }
        __syncwarp();
      }
    }
    count = it;
  } else if (FUSE && warp >= 2 + C::kEpiWarps) {
    // quantiser: four rows a pass and warp (64 a pass in all), eight lanes a row, 16 columns a lane
    const int l = lane & 7, r0 = (warp - 2 - C::kEpiWarps) * 4 + (lane >> 3);
    uint32_t it = 0, rit = 0;
    bool ok = true;
    for (TileWalk tw(team, teams, num_m, num_n); tw.valid() && ok; tw.next()) {
      for (int k = 0; k < nst && ok; ++k, ++it) {
        const int s = it % S;
        ok = __all_sync(0xffffffffu, waits.wait(empty_bar(s), ((it / S) & 1u) ^ 1u, kDevTimeoutEmpty));
        if (!ok) break;
        uint8_t* dA = smem + s * C::kABytes;
        uint8_t* dS = sSf + s * C::kSfBytes;
        const int halves = kp - k * kGStageCols > 128 ? 2 : 1;
        for (int h = 0; h < halves; ++h, ++rit) {
          const int rs = rit % kGRawStages;
          ok = __all_sync(0xffffffffu, waits.wait(rfull_bar(rs), (rit / kGRawStages) & 1u, kDevTimeoutFull));
          if (!ok) break;
          // 64-column box l / 4; its 16-byte chunks are XORed with the row as TMA wrote them
          const uint8_t* src = sRaw + rs * kGRawBytes + (l >> 2) * (kGRawBytes / 2);
          // both passes side by side: one alone is a chain of dependent steps (rows behind M are zero)
          MxRaw<T> raw[2];
          uint32_t e[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = r0 + 64 * i;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const uint4 u = *reinterpret_cast<const uint4*>(src + r * 128 + (((2 * (l & 3) + c) ^ (r & 7)) << 4));
              raw[i].w[4 * c] = u.x; raw[i].w[4 * c + 1] = u.y; raw[i].w[4 * c + 2] = u.z; raw[i].w[4 * c + 3] = u.w;
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) e[i] = mx_raw_amax<T>(raw[i]);
#pragma unroll
          for (int i = 0; i < 2; ++i) e[i] = mx_exponent(mx_block_amax<T>(e[i]));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = r0 + 64 * i;
            float v[16];
            mx_unpack<T>(raw[i], v);
            uint32_t q[2];
            mx_codes<16>(v, e[i], q);
            // codes in the 128 B-swizzled layout that TMA would have written; scales in their tile's order
            *reinterpret_cast<uint2*>(dA + r * 128 + (((4 * h + (l >> 1)) ^ (r & 7)) << 4) + (l & 1) * 8) =
                make_uint2(q[0], q[1]);
            if ((l & 1) == 0) dS[h * kMxTileBytes + mx_scale_byte(r, l >> 1)] = (uint8_t)e[i];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(rempty_bar(rs));
        }
        if (!ok) break;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(s));
      }
    }
    count = it;
  } else {
    pdl_wait();
    // set: which tiles (and accumulator); lg: the TMEM lane quadrant a warp may read; pn: its 64 columns
    const int w = warp - 2, set = w / C::kSetWarps, lg = warp & 3, pn = (w % C::kSetWarps) >> 2;
    float* bias_s = sBias + w * 64;
    uint8_t* pan = sPanel + w * C::kPanelBytes;
    auto load_res = [&](int tm, int tn) {  // lane 0
      mbar_arrive_expect_tx(res_bar(w), C::kPanelBytes);
      tma_load_2d(smem_u32(pan), &map_r, res_bar(w), tn * BN + pn * 64, tm * TM + rank * kGBM + lg * 32);
    };
    TileWalk tw(team + set * teams, C::kSets * teams, num_m, num_n);
    bool loading = false;  // a residual copy of this warp is in flight (lane 0)
    if (p.residual && lane == 0 && tw.valid()) {
      load_res(tw.m, tw.n);
      loading = true;
    }
    uint32_t q = 0;
    for (; tw.valid(); ++q) {
      const int m0 = tw.m * TM + rank * kGBM, n = tw.n * BN + pn * 64;
      tw.next();  // from here on the next tile
      bias_s[lane] = p.bias && n + lane < p.N ? p.bias[n + lane] : 0.f;
      bias_s[32 + lane] = p.bias && n + 32 + lane < p.N ? p.bias[n + 32 + lane] : 0.f;
      if (!p.residual && lane == 0) bulk_wait_read<0>();  // the panel's previous store has read it
      __syncwarp();
      const uint32_t tl = q * C::kSets + set, acc = tl & 1u;  // the block's tile number, and its accumulator
      bool ok = waits.wait(tfull_bar(acc), (tl >> 1) & 1u, kDevTimeoutAcc);
      if (ok && p.residual) {
        ok = waits.wait(res_bar(w), q & 1u, kDevTimeoutEmpty);
        if (ok) loading = false;
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + acc * BN + pn * 64 + (static_cast<uint32_t>(lg * 32) << 16);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[32];
        tmem_ld32(t_row + 32 * h, r);
        tmem_wait_ld();
        if (h == 1) {  // the accumulator's last read of this warp
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && rank != 0)
              mbar_arrive_cluster(mapa_shared(tempty_bar(acc), 0));
            else
              mbar_arrive(tempty_bar(acc));
          }
        }
        const float4* b4 = reinterpret_cast<const float4*>(bias_s + 32 * h);
        auto acc2 = [&](int i, float x, float y) {
          return add_f32x2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), make_float2(x, y));
        };
        if constexpr (GEGLU) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float4 bv = b4[2 * g + e], bg = b4[4 + 2 * g + e];
              const int i = 8 * g + 4 * e;
              const float2 lo = mul_f32x2(acc2(i, bv.x, bv.y), gelu_pair(acc2(16 + i, bg.x, bg.y)));
              const float2 hi = mul_f32x2(acc2(i + 2, bv.z, bv.w), gelu_pair(acc2(18 + i, bg.z, bg.w)));
              v[4 * e] = lo.x; v[4 * e + 1] = lo.y; v[4 * e + 2] = hi.x; v[4 * e + 3] = hi.y;
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
            float2 u[4] = {acc2(8 * g, b0.x, b0.y), acc2(8 * g + 2, b0.z, b0.w), acc2(8 * g + 4, b1.x, b1.y),
                           acc2(8 * g + 6, b1.z, b1.w)};
            if (p.residual) {
              float rv[8];
              mx_unpack8<T>(*reinterpret_cast<const uint4*>(at), rv);
#pragma unroll
              for (int i = 0; i < 4; ++i) u[i] = add_f32x2(u[i], make_float2(rv[2 * i], rv[2 * i + 1]));
            }
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[2 * i] = ACT == 1 ? silu_fine(u[i].x) : u[i].x;
              v[2 * i + 1] = ACT == 1 ? silu_fine(u[i].y) : u[i].y;
            }
            mx_store8<T>(at, v);
          }
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d(&map_y, smem_u32(pan), GEGLU ? n / 2 : n, m0 + lg * 32);
        bulk_commit();
        if (p.residual && tw.valid()) {  // the panel takes the next residual once the store has read it
          bulk_wait_read<0>();
          load_res(tw.m, tw.n);
          loading = true;
        }
      }
    }
    if (lane == 0) {
      // abort: a residual copy in flight lands before the shared memory is released
      if (loading) mbar_drain(res_bar(w), q & 1u, p.err, kDevTimeoutDrain, p.wait_ns);
      bulk_wait_read<0>();
    }
  }
  tc_fence_before();
  __syncwarp();
  auto sync_all = [] {
    if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  };
  sync_all();  // neither CTA frees TMEM or shared memory that the pair still uses
  if (waits.stopped()) {
    // A wait expired (all threads, a pair's too, see the same flag: no wait is left). Every copy in flight lands before the
    // shared memory is released: each stage's barrier is brought to the end of its phase and waited for. Producers, quantisers
    // and the two CTAs of a pair are at most S stages apart, so a stage that one side lacks is in its barrier's current phase.
    if (FUSE && warp >= 2 + C::kEpiWarps && warp < 2 + C::kEpiWarps + kGQuantWarps && lane == 0)
      for (uint32_t i = count; i < *issued; ++i) mbar_arrive(full_bar(i % S));  // stages loaded, not filled
    if (FUSE && warp == 2 + C::kEpiWarps + kGQuantWarps && lane == 0)
      for (uint32_t i = count > (uint32_t)kGRawStages ? count - kGRawStages : 0; i < count; ++i)
        mbar_drain(rfull_bar(i % kGRawStages), (i / kGRawStages) & 1u, p.err, kDevTimeoutDrain, p.wait_ns);
    if (warp == 0 && lane == 0 && rank == 0) {
      uint32_t top = count;
      if constexpr (PAIR) {
        const uint32_t odd = ld_cluster(mapa_shared(smem_u32(issued), 1));
        for (uint32_t i = odd; i < count; ++i) mbar_complete_tx(full_bar(i % S), C::kStageBytes);  // never loaded there
        for (uint32_t i = count; i < odd; ++i) mbar_arrive_expect_tx(full_bar(i % S), C::kStageBytes);  // never loaded here
        top = max(count, odd);
      }
      for (uint32_t i = top > (uint32_t)S ? top - S : 0; i < top; ++i)
        mbar_drain(full_bar(i % S), (i / S) & 1u, p.err, kDevTimeoutDrain, p.wait_ns);
    }
    __syncwarp();
    sync_all();
  }
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc2(tmem_base, C::kTmemCols);
    else
      tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

template <int BN, typename T, int ACT, bool FUSE, bool PAIR>
cudaError_t launch_gemm_mx4(const Mx4LinearArgs& a, int* err, cudaStream_t s) {
  using C = GCfg<BN, ACT == 2, FUSE, PAIR>;
  constexpr int TM = PAIR ? 2 * kGBM : kGBM;
  auto k = mx4_gemm_kernel<BN, T, ACT, FUSE, PAIR>;
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
  CUtensorMap mx, mw, my, mr, mxs, mws;
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
  if (!codes(&mw, a.wcodes, a.N, C::kBRows) || !panel(&my, a.y)) return cudaErrorInvalidValue;
  mr = my;
  if (a.residual && !panel(&mr, a.residual)) return cudaErrorInvalidValue;
  if constexpr (FUSE) {
    const uint64_t dims[2] = {(uint64_t)a.K, (uint64_t)a.M}, str[1] = {(uint64_t)a.ldx * 2};
    const uint32_t box[2] = {64, kGBM};
    if (!make_tmap(&mx, a.x, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_UINT16))
      return cudaErrorInvalidValue;
  } else {
    if (!codes(&mx, a.xcodes, a.M, kGBM)) return cudaErrorInvalidValue;
  }
  mxs = mws = mw;
  if constexpr (PAIR) {  // scale tiles as rows of 32-bit words, two of 512 bytes at a time
    auto scales = [&](CUtensorMap* m, const uint8_t* base, int rows) {
      const uint64_t dims[2] = {(uint64_t)mx_ktiles(a.K) * 128, (uint64_t)mx_rtiles(rows)}, str[1] = {dims[0] * 4};
      const uint32_t box[2] = {256, 1};
      return make_tmap(m, base, 2, dims, str, box, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_DATA_TYPE_UINT32);
    };
    if (!scales(&mxs, a.xscales, a.M) || !scales(&mws, a.wscales, a.N)) return cudaErrorInvalidValue;
  }
  GemmMx4Dev p;
  p.M = a.M; p.N = a.N; p.K = a.K;
  p.xs = a.xscales; p.ws = a.wscales; p.bias = a.bias; p.residual = a.residual != nullptr; p.err = err;
  p.wait_ns = a.wait_limit_ns ? a.wait_limit_ns : kWaitTimeoutNs;
  p.stall_it = a.test_stall_iter; p.stall_who = a.test_stall_who;
  const long long tiles = (long long)((a.M + TM - 1) / TM) * ((a.N + BN - 1) / BN);
  if (tiles > (1ll << 30)) return cudaErrorInvalidValue;  // the walk counts tiles in 32 bits
  const int teams = (int)std::min<long long>(tiles, PAIR ? num_sms() / 2 : num_sms());
  return launch_kernel(k, dim3(PAIR ? 2 * teams : teams), dim3(C::kThreads), C::kSmem, s, PAIR ? 2 : 0, mx, mw, my, mr, mxs,
                       mws, p);
}

// Pairs from this many stages (K > 1792) and two rounds of tiles on. Measured on B200, pairs against single CTAs: 65536 x
// 640 x 2560 62.4 / 66.6 us, 20000 x 1280 x 5120 63.3 / 68.8 us, but 8192 x 2560 x 1280 23.5 / 20.4 us and 32768 x 640 x
// 640 23.9 / 17.6 us. (One CTA on 256-wide tiles, as two halves with three accumulators, measured no faster than 128.)
constexpr int kPairStages = 8;

template <typename T, int ACT>
cudaError_t gemm_bn(const Mx4LinearArgs& a, int* err, cudaStream_t s) {
  switch (mx4_linear_form(a)) {
    case kMx4Fused: return launch_gemm_mx4<64, T, ACT, true, false>(a, err, s);
    case kMx4Pair: return launch_gemm_mx4<128, T, ACT, false, true>(a, err, s);
    case kMx4Wide: return launch_gemm_mx4<128, T, ACT, false, false>(a, err, s);
    default: return launch_gemm_mx4<64, T, ACT, false, false>(a, err, s);
  }
}

// The fused form while a block quantises at most this many stages (256 columns of 128 rows, about 1.3 us each). Measured
// on B200, fused against quantise + product: one eager call 12.3 against 16.4 us (the second launch and the scratch's
// allocation cost the host 4 us), the device alone 154 x 2560 x 768 7.9 / 5.2 us, 8192 x 320 x 320 11.0 / 7.2 us; beyond
// six stages the device time passes the host's. A caller whose host time does not count (a captured graph) quantises x
// first and passes the operand.
constexpr long long kFuseStages = 6;

// Few rows run on the CUDA cores, as long as their operand fits 48 KB of shared memory.
bool linear_rows(int M, int K) { return M <= 8 && (size_t)8 * (mx_kp(K) / 2 + mx_kp(K) / 8) <= 48 * 1024; }

template <typename T>
cudaError_t linear_t(const Mx4LinearArgs& a, int* err, cudaStream_t s) {
  if (mx4_linear_form(a) == kMx4Rows) {
    if (a.M == 1) return launch_rows<T, 1>(a, s);
    if (a.M == 2) return launch_rows<T, 2>(a, s);
    return a.M <= 4 ? launch_rows<T, 4>(a, s) : launch_rows<T, 8>(a, s);
  }
  switch (a.act) {
    case 1: return gemm_bn<T, 1>(a, err, s);
    case 2: return gemm_bn<T, 2>(a, err, s);
    default: return gemm_bn<T, 0>(a, err, s);
  }
}

}  // namespace

Mx4Form mx4_linear_form(const Mx4LinearArgs& a) {
  if (linear_rows(a.M, a.K)) return kMx4Rows;
  if (a.x) return kMx4Fused;
  const long long tiles = (long long)((a.M + kGBM - 1) / kGBM) * ((a.N + 127) / 128);
  if (tiles >= 2 * num_sms() && (mx_kp(a.K) + kGStageCols - 1) / kGStageCols >= kPairStages) return kMx4Pair;
  return tiles >= num_sms() ? kMx4Wide : kMx4Narrow;
}

bool mx4_linear_takes_x(const void* x, int M, int K, long long ldx, int N) {
  if (linear_rows(M, K)) return true;
  // the fused form reads x by TMA: aligned rows, a stride that a tensor map can hold
  const bool tma = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % 8 == 0 && ldx >= K;
  if (!tma) return false;
  const long long tiles = (long long)((M + kGBM - 1) / kGBM) * ((N + 63) / 64), rounds = (tiles + num_sms() - 1) / num_sms();
  return rounds * ((mx_kp(K) + kGStageCols - 1) / kGStageCols) <= kFuseStages;
}

cudaError_t launch_mx4_linear(const Mx4LinearArgs& a, int* dev_err, cudaStream_t s) {
  return a.dtype == kBF16 ? linear_t<__nv_bfloat16>(a, dev_err, s) : linear_t<__half>(a, dev_err, s);
}

}  // namespace sdg

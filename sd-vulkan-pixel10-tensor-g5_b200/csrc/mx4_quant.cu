// mx4_quant.cu — MXFP4 quantisation and read-back, and GroupNorm (+ SiLU) written as an MXFP4 operand.
//
// All three walk the operand in its own scale tiles: one block of 256 threads per 128 rows x 128 columns. A lane
// takes 32 bytes of a row (16 columns of a 16-bit type, 8 of fp32), so a 32-column block is a pair (quad) of
// lanes and its maximum one (two) shuffles, and every load of the tile is issued before the first use (32 KB of
// 16-bit input in flight per block). The tiles of a row are neighbours in the grid, so the lines they share at a row
// pitch that is no multiple of 128 bytes are still in L2 for the second of them. A row's codes leave as 64 contiguous bytes; the tile's 512 scale bytes are
// gathered in shared memory and leave as one. Bound by HBM: one read of x and 17/32 of a byte per value written (read
// back: the reverse).
//
// Rows that 32-byte accesses cannot take (odd K, odd strides, unaligned views) go through shared memory: the warp
// moves the row's 128 columns one element a lane, and each lane then handles its own 32 bytes of the tile.
//
// Inputs are read with plain loads, never through the non-coherent path (ld.global.nc, __ldg, const __restrict__): a
// kernel launched early (programmatic launch) may share an SM's L1 with an older kernel that still reads the buffer's
// previous contents, and only plain loads are ordered by griddepcontrol.wait.
#include <algorithm>
#include <type_traits>

#include "mx4.cuh"
#include "sdg_kernels.h"
#include "sdg_launch.h"
#include "sdg_ptx.cuh"

namespace sdg {
namespace {

constexpr int kQThreads = 256;

// How a tile maps to threads for elements of T: kN columns a lane, kLanes lanes a row, kRows rows a pass.
template <typename T>
struct QMap {
  static constexpr int kN = MxRaw<T>::kN;
  static constexpr int kLanes = kMxTileCols / kN;
  static constexpr int kRows = kQThreads / kLanes;
  static constexpr int kPass = kMxTileRows / kRows;
  static constexpr int kPitch = kMxTileCols * (int)sizeof(T) + 16;  // staged row pitch: conflict-free 16-byte reads
};

// Access widths: 32 bytes (K a multiple of the lane's columns, rows 32-byte aligned), 16 bytes, staged.
enum Access { kW32 = 0, kW16 = 1, kStaged = 2 };

// The lane's 32 bytes at src, of which `left` columns are inside the row.
template <typename T, int ACC>
__device__ __forceinline__ void load_raw(const T* src, int left, MxRaw<T>& r) {
  constexpr int H = 16 / (int)sizeof(T);  // columns per 16 bytes
  if constexpr (ACC == kW32) {
    if (left > 0) {
      mx_ld32(src, r.w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.w[i] = 0u;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 u = left > h * H ? reinterpret_cast<const uint4*>(src)[h] : make_uint4(0u, 0u, 0u, 0u);
      r.w[4 * h] = u.x; r.w[4 * h + 1] = u.y; r.w[4 * h + 2] = u.z; r.w[4 * h + 3] = u.w;
    }
  }
}

// The lane's codes and its block's exponent byte into the tile (c: first column of the lane, rl: row of the tile).
template <typename T>
__device__ __forceinline__ void put_codes(const uint32_t (&q)[QMap<T>::kN / 8], uint32_t e, int l, int rl, int c,
                                          uint8_t* row_codes, uint32_t* tile) {
  if constexpr (QMap<T>::kN == 16)
    *reinterpret_cast<uint2*>(row_codes + c / 2) = make_uint2(q[0], q[1]);
  else
    *reinterpret_cast<uint32_t*>(row_codes + c / 2) = q[0];
  constexpr int B = kMxBlock / QMap<T>::kN;  // lanes per block
  if (l % B == 0) reinterpret_cast<uint8_t*>(tile)[mx_scale_byte(rl, l / B)] = (uint8_t)e;
}

template <typename T, int ACC>
__global__ void __launch_bounds__(kQThreads) mx4_quantize_kernel(const T* x, int M, int K, long long ldx,
                                                                 uint8_t* codes,
                                                                 uint8_t* scales) {
  using Q = QMap<T>;
  __shared__ uint32_t tile[kMxTileBytes / 4];
  extern __shared__ uint4 stage[];  // staged access only
  const int kts = mx_ktiles(K), kt = blockIdx.x % kts;
  const int rt = blockIdx.x / kts, row0 = rt * kMxTileRows;
  const int l = threadIdx.x % Q::kLanes, r0 = threadIdx.x / Q::kLanes;
  const int c = kt * kMxTileCols + l * Q::kN;
  const int kp = mx_kp(K);
  if (threadIdx.x < kMxTileBytes / 4) tile[threadIdx.x] = 0u;
  pdl_wait();
  pdl_trigger();
  MxRaw<T> raw[Q::kPass];
  if constexpr (ACC == kStaged) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T* st = reinterpret_cast<T*>(stage);
    const int rows = min(kMxTileRows, M - row0);
#pragma unroll 4
    for (int r = warp; r < rows; r += kQThreads / 32) {
      const T* src = x + (size_t)(row0 + r) * ldx + kt * kMxTileCols;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int cc = lane + 32 * i;
        st[r * (Q::kPitch / (int)sizeof(T)) + cc] = kt * kMxTileCols + cc < K ? src[cc] : MxElem<T>::put(0.f);
      }
    }
  } else {
#pragma unroll
    for (int p = 0; p < Q::kPass; ++p) {
      const int r = row0 + p * Q::kRows + r0;
      load_raw<T, ACC>(x + (size_t)min(r, M - 1) * ldx + c, r < M ? K - c : 0, raw[p]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < Q::kPass; ++p) {
    const int rl = p * Q::kRows + r0, r = row0 + rl;
    if constexpr (ACC == kStaged) {
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(stage) + rl * Q::kPitch + l * 32);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = r < M ? src[h] : make_uint4(0u, 0u, 0u, 0u);
        raw[p].w[4 * h] = u.x; raw[p].w[4 * h + 1] = u.y; raw[p].w[4 * h + 2] = u.z; raw[p].w[4 * h + 3] = u.w;
      }
    }
    const uint32_t e = mx_exponent(mx_block_amax<T>(mx_raw_amax<T>(raw[p])));
    float v[Q::kN];
    mx_unpack<T>(raw[p], v);
    uint32_t q[Q::kN / 8];
    mx_codes<Q::kN>(v, e, q);
    if (r < M && c < kp) put_codes<T>(q, e, l, rl, c, codes + (size_t)r * (kp / 2), tile);
  }
  __syncthreads();
  if (threadIdx.x < kMxTileBytes / 4)
    reinterpret_cast<uint32_t*>(scales + ((size_t)rt * kts + kt) * kMxTileBytes)[threadIdx.x] = tile[threadIdx.x];
}

template <typename T, int ACC>
__global__ void __launch_bounds__(kQThreads) mx4_dequantize_kernel(const uint8_t* codes,
                                                                   const uint8_t* scales, int M, int K,
                                                                   T* y) {
  using Q = QMap<T>;
  __shared__ uint32_t tile[kMxTileBytes / 4];
  extern __shared__ uint4 stage[];  // staged access only
  const int kts = mx_ktiles(K), kt = blockIdx.x % kts;
  const int rt = blockIdx.x / kts, row0 = rt * kMxTileRows;
  const int l = threadIdx.x % Q::kLanes, r0 = threadIdx.x / Q::kLanes;
  const int c = kt * kMxTileCols + l * Q::kN;
  const int kp = mx_kp(K);
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < kMxTileBytes / 4)
    tile[threadIdx.x] =
        reinterpret_cast<const uint32_t*>(scales + ((size_t)rt * kts + kt) * kMxTileBytes)[threadIdx.x];
  uint32_t q[Q::kPass][Q::kN / 8];
#pragma unroll
  for (int p = 0; p < Q::kPass; ++p) {
    const int r = row0 + p * Q::kRows + r0;
    const bool in = r < M && c < kp;
    const uint8_t* src = codes + (size_t)r * (kp / 2) + c / 2;
    if constexpr (Q::kN == 16) {
      const uint2 u = in ? *reinterpret_cast<const uint2*>(src) : make_uint2(0u, 0u);
      q[p][0] = u.x;
      q[p][Q::kN / 8 - 1] = u.y;
    } else {
      q[p][0] = in ? *reinterpret_cast<const uint32_t*>(src) : 0u;
    }
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < Q::kPass; ++p) {
    const int rl = p * Q::kRows + r0, r = row0 + rl;
    const float s = mx_pow2(reinterpret_cast<const uint8_t*>(tile)[mx_scale_byte(rl, l / (kMxBlock / Q::kN))]);
    uint32_t o[8];
#pragma unroll
    for (int w = 0; w < Q::kN / 8; ++w) {
      __half2 h[4];
      mx_decode8(q[p][w], h);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = mul_f32x2(__half22float2(h[i]), make_float2(s, s));
        if constexpr (sizeof(T) == 4) {
          o[2 * i] = __float_as_uint(f.x);
          o[2 * i + 1] = __float_as_uint(f.y);
        } else {
          o[4 * w + i] = MxElem<T>::put2(f.x, f.y);
        }
      }
    }
    if constexpr (ACC == kStaged) {
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(stage) + rl * Q::kPitch + l * 32);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else if (r < M) {
      T* dst = y + (size_t)r * K + c;
      if constexpr (ACC == kW32) {
        if (c < K) mx_st32(dst, o);
      } else {
        if (c < K) reinterpret_cast<uint4*>(dst)[0] = make_uint4(o[0], o[1], o[2], o[3]);
        if (c + Q::kN / 2 < K) reinterpret_cast<uint4*>(dst)[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
  if constexpr (ACC == kStaged) {
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* st = reinterpret_cast<const T*>(stage);
    const int rows = min(kMxTileRows, M - row0), cols = min(kMxTileCols, K - kt * kMxTileCols);
#pragma unroll 4
    for (int r = warp; r < rows; r += kQThreads / 32) {
      T* dst = y + (size_t)(row0 + r) * K + kt * kMxTileCols;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int cc = lane + 32 * i;
        if (cc < cols) dst[cc] = st[r * (Q::kPitch / (int)sizeof(T)) + cc];
      }
    }
  }
}

// ------------------------------------------------------------------ GroupNorm (+ SiLU) -> MXFP4
// Two launches. Statistics: each block reads one chunk of an image's pixels (all channels) once and writes each group's
// (mean, M2 = sum of squared differences from that mean) over the chunk. A chunk has 16 or 32 pixels for each of the threads'
// rows: about 64 KB, 128 KB in larger images, up to 256 KB at 4096 channels; more only where an image would have over 256
// chunks. Apply: each block merges the chunks' pairs of the groups its tiles need, in a fixed order, then normalises,
// activates and quantises one to eight tiles of the same channels. Runs, threads and chunks merge by Chan, Golub and
// LeVeque's update of (n, mean, M2). Chunks depend on (HW, C) alone: an image's result does not depend on the batch, and no
// atomics make the order of a sum vary. The second read of x comes from L2 while an input fits it. Measured on B200 (graph
// replay), 64 x 1024 x 640 bf16 + SiLU: 22 + 33 us, floor 16.2; neither memory (44 and 29 %) nor a pipe is full.
constexpr int kGnThreads = 256;
constexpr int kGnBatch = 8;         // pixels a thread holds at once
constexpr int kGnShift = 4;         // pixels that give the shift
constexpr int kGnPixels = 16;       // least pixels per thread and chunk of an image of several chunks
constexpr int kGnRun = 2 * kGnPixels;  // pixels that a thread sums about one shift
static_assert(kGnRun % kGnBatch == 0, "a run is whole batches");
constexpr int kGnMaxC = 4096;
constexpr int kGnMaxChunks = 256;

// the larger value, NaN if either is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

struct GnPlan {
  int chunk, chunks;  // pixels per chunk, chunks per image
};
__host__ __device__ inline int gn_rows_par(int C) { return C / 8 >= kGnThreads ? 1 : kGnThreads / (C / 8); }
GnPlan gn_plan(int HW, int C) {
  // twice the pixels where that leaves eight chunks: a chunk's fixed work weighs less (both launches, 64 x 1024 x 640 58.7 ->
  // 55.3 us, 2 x 4096 x 320 11.0 -> 11.6 us); smaller images need the blocks (2 x 64 x 1280 7.4 -> 8.7 us)
  const int par = gn_rows_par(C), unit = par * (HW >= 16 * kGnPixels * par ? 2 * kGnPixels : kGnPixels);
  const int units = (HW + unit - 1) / unit;
  const int per = (units + kGnMaxChunks - 1) / kGnMaxChunks;
  GnPlan p;
  p.chunk = per * unit;
  p.chunks = (HW + p.chunk - 1) / p.chunk;
  return p;
}

// A thread takes its pixels of a channel in runs of n <= 32. It sums d and d^2 over a run, d = x - k with k the mean of the
// run's first m = min(n, 4) pixels. (k - mean)^2 <= M2 / m (Cauchy), so sum d^2 <= M2 (1 + n / m) and M2 = sum d^2 -
// (sum d)^2 / n loses at most the factor 1 + n / m <= 9 to cancellation, whatever the data. Runs merge by the update of
// (n, mean, M2) as threads and chunks do; only images of more than kGnMaxChunks units have chunks of several runs.
template <typename T>
__global__ void __launch_bounds__(kGnThreads, 3) mx4_gn_stats_kernel(const T* x, int HW, int C, int groups,
                                                                  int chunk, float2* part) {
  // (mean, M2) per thread row and channel
  __shared__ __align__(16) float2 acc[kGnMaxC];
  const int nv = C / 8, par = gn_rows_par(C), cpg = C / groups;
  const int p0 = blockIdx.x * chunk, p1 = min(HW, p0 + chunk);
  const int r = threadIdx.x / nv;  // thread row (0 where a row of C needs more than all threads)
  pdl_wait();
  pdl_trigger();
  for (int v = threadIdx.x - (par > 1 ? r * nv : 0); v < nv; v += kGnThreads) {
    if (par > 1 && r >= par) break;
    const T* src = x + ((size_t)blockIdx.y * HW + p0) * C + v * 8;
    const int first = par > 1 ? r : 0;
    const int cnt = p1 - p0 > first ? (p1 - p0 - first + par - 1) / par : 0;  // this thread's pixels
    const T* at = src + (size_t)first * C;
    const size_t step = (size_t)par * C;
    float4* dst = reinterpret_cast<float4*>(acc + (par > 1 ? r * C : 0) + v * 8);
#pragma unroll 1
    for (int run = 0; run < cnt; run += kGnRun) {
      const int n = min(kGnRun, cnt - run);
      float2 k[4], s1[4], s2[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = s1[e] = s2[e] = make_float2(0.f, 0.f);
      for (int i0 = 0; i0 < n; i0 += kGnBatch) {
        const int nb = min(kGnBatch, n - i0);
        uint4 raw[kGnBatch];
#pragma unroll
        for (int i = 0; i < kGnBatch; ++i) {
          raw[i] = i < nb ? *reinterpret_cast<const uint4*>(at) : make_uint4(0u, 0u, 0u, 0u);
          at += step;
        }
        if (i0 == 0) {
#pragma unroll
          for (int i = 0; i < kGnShift; ++i) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = add_f32x2(k[e], MxElem<T>::get2(w[e]));
          }
          const float inv = 1.f / (float)min(kGnShift, nb);
#pragma unroll
          for (int e = 0; e < 4; ++e) k[e] = mul_f32x2(k[e], make_float2(inv, inv));
        }
#pragma unroll
        for (int i = 0; i < kGnBatch; ++i) {
          if (i < nb) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 d = sub_f32x2(MxElem<T>::get2(w[e]), k[e]);
              s1[e] = add_f32x2(s1[e], d);
              s2[e] = fma_f32x2(d, d, s2[e]);
            }
          }
        }
      }
      const float inv = 1.f / (float)n;
      const float f = (float)n / (float)(run + n), g = f * (float)run;  // shares of this run in a merge
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mx = s1[e].x * inv, my = s1[e].y * inv;
        float4 st = make_float4(k[e].x + mx, max_nan(fmaf(-mx, s1[e].x, s2[e].x), 0.f), k[e].y + my,
                                max_nan(fmaf(-my, s1[e].y, s2[e].y), 0.f));
        if (run) {  // with the runs before, which this thread left here
          const float4 o = dst[e];
          const float dx = st.x - o.x, dy = st.z - o.z;
          st = make_float4(fmaf(dx, f, o.x), o.y + fmaf(dx * g, dx, st.y), fmaf(dy, f, o.z), o.w + fmaf(dy * g, dy, st.w));
        }
        dst[e] = st;
      }
    }
  }
  __syncthreads();
  // eight lanes per group: its par x cpg pairs, thread row rr holding q or q + 1 pixels
  const int rows = p1 - p0, q = rows / par, rem = rows - q * par, sub = threadIdx.x & 7;
  const float inv_n = 1.f / ((float)rows * cpg);
  for (int g = threadIdx.x >> 3; g < (groups + 3) / 4 * 4; g += kGnThreads / 8) {  // whole warps: the shuffles need them
    const float2* a = acc + min(g, groups - 1) * cpg;
    float s = 0.f;
    for (int rr = 0; rr < par; ++rr) {
      const float n = (float)(q + (rr < rem));
      if (n != 0.f)
        for (int i = sub; i < cpg; i += 8) s = fmaf(n, a[rr * C + i].x, s);
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mu = s * inv_n;
    float m2 = 0.f;
    for (int rr = 0; rr < par; ++rr) {
      const float n = (float)(q + (rr < rem));
      if (n != 0.f)
        for (int i = sub; i < cpg; i += 8) {
          const float2 v = a[rr * C + i];
          const float d = v.x - mu;
          m2 += fmaf(n * d, d, v.y);
        }
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
    if (sub == 0 && g < groups) part[((size_t)blockIdx.y * gridDim.x + blockIdx.x) * groups + g] = make_float2(mu, m2);
  }
}

// (mean, rstd) of group g from the chunks' pairs at part[k * groups + g]; the eight lanes of a group call it together, a
// lane taking every eighth chunk. (Pairs kept in registers between the two sums spill: the tile's loads are in flight.)
__device__ __forceinline__ float2 gn_merge(const float2* part, int g, int groups, int chunks, int chunk, int HW, int cpg,
                                           float eps) {
  const int sub = threadIdx.x & 7;
  auto pixels = [&](int k) { return (float)(min(HW, (k + 1) * chunk) - k * chunk); };
  float s = 0.f;
#pragma unroll 2
  for (int k = sub; k < chunks; k += 8) s = fmaf(pixels(k), part[(size_t)k * groups + g].x, s);
#pragma unroll
  for (int o = 4; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float mu = s / (float)HW;
  float m2 = 0.f;
#pragma unroll 2
  for (int k = sub; k < chunks; k += 8) {
    const float2 v = part[(size_t)k * groups + g];
    const float d = v.x - mu;
    m2 += fmaf(pixels(k) * cpg * d, d, v.y);
  }
#pragma unroll
  for (int o = 4; o; o >>= 1) m2 += __shfl_xor_sync(0xffffffffu, m2, o);
  return make_float2(mu, rsqrtf(m2 / ((float)HW * cpg) + eps));
}

// y * sigmoid(y) of two values as y n / (1 + e), e = exp(-|y|), n = 1 or (y < 0) e: nothing overflows, so a value keeps its
// relative accuracy (|y| 2^-24 and a few ulps) down to y = -87.3, below which e is 0 - a block's exponent follows its
// maximum, however small. One reciprocal, 1 / (a b), serves both: three MUFU instructions instead of four (64 x 1024 x 640,
// both launches, 55.1 against 57.5 us). The rounding to four bits comes after it, so the approximation must not move values
// across the E2M1 midpoints more often than fp32 arithmetic does. A NaN spoils its pair, which shares its block.
__device__ __forceinline__ float2 silu_pair(float2 y) {
  const float2 e = make_float2(ex2_approx(-1.4426950408889634f * fabsf(y.x)), ex2_approx(-1.4426950408889634f * fabsf(y.y)));
  const float2 s = add_f32x2(e, make_float2(1.f, 1.f));
  const float r = rcp_approx(s.x * s.y);
  const float2 n = make_float2(y.x < 0.f ? e.x : 1.f, y.y < 0.f ? e.y : 1.f);
  return mul_f32x2(mul_f32x2(y, n), mul_f32x2(make_float2(r, r), make_float2(s.y, s.x)));
}

// Images that a tile of 128 rows touches at most, unless an image has kGnPixels pixels or fewer (and then one chunk)
constexpr int kImgs = kMxTileRows / (kGnPixels + 1) + 2;

struct GnApply {
  int M, HW, C, groups, chunk, chunks;
  int tiles;  // row tiles per block
  float eps;
  const float* gamma;
  const float* beta;
  const float2* part;
  uint8_t* codes;
  uint8_t* scales;
};

// FEW: images so small that a tile may touch more than kImgs of them; their factors come straight from the
// statistics, in an instantiation of its own (inside the other's unrolled loop the code outgrew the instruction cache).
template <typename T, int ACC, bool SILU, bool FEW>
__global__ void __launch_bounds__(kQThreads, 3) mx4_gn_apply_kernel(const T* x, const GnApply p) {
  using Q = QMap<T>;
  static_assert(Q::kN == 16, "16-bit elements");
  __shared__ uint32_t tile[kMxTileBytes / 4];
  // y = x * a + b per image of the tile and channel; per pair of channels: a, a, b, b. Pair j of
  // lane l is float4 j * 8 + l: the eight lanes of a row read 128 contiguous bytes
  __shared__ __align__(16) float affine[kImgs * 2 * kMxTileCols];
  __shared__ float2 table[kImgs * kMxTileCols];  // (mean, rstd) per image and group, where chunks are merged here
  const int kts = mx_ktiles(p.C), kt = blockIdx.x % kts;
  const int rt0 = blockIdx.x / kts * p.tiles, rt1 = min(rt0 + p.tiles, mx_rtiles(p.M));
  const int l = threadIdx.x % Q::kLanes, r0 = threadIdx.x / Q::kLanes;
  const int c = kt * kMxTileCols + l * Q::kN;
  const int kp = mx_kp(p.C), cpg = p.C / p.groups;
  const int c_end = min(p.C, (kt + 1) * kMxTileCols);
  const int g_lo = kt * kMxTileCols / cpg, ng = (c_end - 1) / cpg - g_lo + 1;
  const float inv_n = 1.f / ((float)p.HW * cpg);
  auto one_chunk = [&](int img, int g) {
    float2 st = p.part[(size_t)img * p.groups + g];
    st.y = rsqrtf(st.y * inv_n + p.eps);
    return st;
  };
  // a channel's factors from its group's statistics
  auto factors = [&](int cc, float2 st) {
    const float a = st.y * p.gamma[cc];
    return make_float2(a, fmaf(-st.x, a, p.beta[cc]));
  };
  int have0 = -1, have1 = -1;  // images that `affine` holds
  pdl_wait();
  pdl_trigger();
#pragma unroll 1
  for (int rt = rt0; rt < rt1; ++rt) {
    const int row0 = rt * kMxTileRows;
    MxRaw<T> raw[Q::kPass];
#pragma unroll
    for (int i = 0; i < Q::kPass; ++i) {
      const int r = row0 + i * Q::kRows + r0;
      load_raw<T, ACC>(x + (size_t)min(r, p.M - 1) * p.C + c, r < p.M ? p.C - c : 0, raw[i]);
    }
    if (threadIdx.x < kMxTileBytes / 4) tile[threadIdx.x] = 0u;
    const int img0 = row0 / p.HW, img1 = (min(p.M, row0 + kMxTileRows) - 1) / p.HW, imgs = img1 - img0 + 1;
    if (!FEW && (img0 != have0 || img1 != have1)) {
      have0 = img0;
      have1 = img1;
      if (p.chunks > 1) {
        for (int i = threadIdx.x >> 3; i < (imgs * ng + 3) / 4 * 4; i += kQThreads / 8) {  // whole warps
          const int q = min(i, imgs * ng - 1), im = q / ng, g = q - im * ng;
          const float2 st = gn_merge(p.part + (size_t)(img0 + im) * p.chunks * p.groups, g_lo + g, p.groups, p.chunks,
                                     p.chunk, p.HW, cpg, p.eps);
          if ((threadIdx.x & 7) == 0) table[im * kMxTileCols + g] = st;
        }
        __syncthreads();
      }
      for (int i = threadIdx.x; i < imgs * kMxTileCols; i += kQThreads) {
        const int im = i / kMxTileCols, cl = i % kMxTileCols, cc = kt * kMxTileCols + cl;
        float2 f = make_float2(0.f, 0.f);
        if (cc < p.C) {
          const int g = cc / cpg;
          f = factors(cc, p.chunks > 1 ? table[im * kMxTileCols + g - g_lo] : one_chunk(img0 + im, g));
        }
        float* dst = affine + im * 2 * kMxTileCols + ((cl / 2 % 8) * 8 + cl / 16) * 4 + (cl & 1);
        dst[0] = f.x;
        dst[2] = f.y;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Q::kPass; i += 2) {  // two rows at a time: they share the factors' loads where they share an image
      float v[2][16], top[2] = {0.f, 0.f};
      int rl[2], img[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        rl[h] = (i + h) * Q::kRows + r0;
        img[h] = imgs == 1 ? img0 : min(row0 + rl[h], p.M - 1) / p.HW;
      }
      const float4* fac0 = reinterpret_cast<const float4*>(affine + (img[0] - img0) * 2 * kMxTileCols + l * 4);
      const float4* fac1 = reinterpret_cast<const float4*>(affine + (img[1] - img0) * 2 * kMxTileCols + l * 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float4 f[2];
        if constexpr (FEW) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int c0 = min(c + 2 * j, p.C - 2);
            const float2 a = factors(c0, one_chunk(img[h], c0 / cpg)), b = factors(c0 + 1, one_chunk(img[h], (c0 + 1) / cpg));
            f[h] = c + 2 * j < p.C ? make_float4(a.x, b.x, a.y, b.y) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        } else {
          f[0] = fac0[8 * j];
          f[1] = imgs == 1 ? f[0] : fac1[8 * j];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float2 y = fma_f32x2(MxElem<T>::get2(raw[i + h].w[j]), make_float2(f[h].x, f[h].y), make_float2(f[h].z, f[h].w));
          if constexpr (SILU) y = silu_pair(y);
          v[h][2 * j] = y.x;
          v[h][2 * j + 1] = y.y;
          top[h] = max_nan(top[h], fabsf(y.x), fabsf(y.y));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = row0 + rl[h];
        uint32_t m = __float_as_uint(top[h]) & 0x7FFFFFFFu;
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t e = mx_exponent(m);
        uint32_t q[2];
        mx_codes<16>(v[h], e, q);
        if (r < p.M && c < kp) put_codes<T>(q, e, l, rl[h], c, p.codes + (size_t)r * (kp / 2), tile);
      }
    }
    __syncthreads();
    if (threadIdx.x < kMxTileBytes / 4)
      reinterpret_cast<uint32_t*>(p.scales + ((size_t)rt * kts + kt) * kMxTileBytes)[threadIdx.x] = tile[threadIdx.x];
  }
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The widest access that a row-major matrix of K columns and row stride ld allows.
template <typename T>
Access access_of(const T* p, int K, long long ld) {
  const long long b = ld * (long long)sizeof(T);
  if (K % (32 / (int)sizeof(T)) == 0 && aligned(p, 32) && b % 32 == 0) return kW32;
  if (K % (16 / (int)sizeof(T)) == 0 && aligned(p, 16) && b % 16 == 0) return kW16;
  return kStaged;
}
template <typename T>
constexpr size_t stage_bytes() { return (size_t)kMxTileRows * QMap<T>::kPitch; }

// Dynamic shared memory above 48 KB (the staged fp32 tile) has to be opted into; done on each such call, for its device.
template <typename K>
cudaError_t allow_smem(K k, size_t bytes) {
  return bytes > 48 * 1024 ? cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) : cudaSuccess;
}

template <typename T>
cudaError_t quantize_t(const T* x, int M, int K, long long ldx, uint8_t* codes, uint8_t* scales, cudaStream_t s) {
  const dim3 grid(mx_rtiles(M) * mx_ktiles(K));
  const Access acc = access_of(x, K, ldx);
  auto k = acc == kW32 ? mx4_quantize_kernel<T, kW32> : acc == kW16 ? mx4_quantize_kernel<T, kW16> : mx4_quantize_kernel<T, kStaged>;
  const size_t sm = acc == kStaged ? stage_bytes<T>() : 0;
  const cudaError_t e = allow_smem(k, sm);
  return e != cudaSuccess ? e : launch_kernel(k, grid, dim3(kQThreads), sm, s, 0, x, M, K, ldx, codes, scales);
}
template <typename T>
cudaError_t dequantize_t(const uint8_t* codes, const uint8_t* scales, int M, int K, T* y, cudaStream_t s) {
  const dim3 grid(mx_rtiles(M) * mx_ktiles(K));
  const Access acc = access_of(y, K, K);
  auto k = acc == kW32   ? mx4_dequantize_kernel<T, kW32>
           : acc == kW16 ? mx4_dequantize_kernel<T, kW16>
                         : mx4_dequantize_kernel<T, kStaged>;
  const size_t sm = acc == kStaged ? stage_bytes<T>() : 0;
  const cudaError_t e = allow_smem(k, sm);
  return e != cudaSuccess ? e : launch_kernel(k, grid, dim3(kQThreads), sm, s, 0, codes, scales, M, K, y);
}
template <typename T>
cudaError_t groupnorm_t(const Mx4GroupNormArgs& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.x);
  float2* part = reinterpret_cast<float2*>(a.stats);
  const GnPlan pl = gn_plan(a.HW, a.C);
  cudaError_t e = launch_kernel(mx4_gn_stats_kernel<T>, dim3(pl.chunks, a.B), dim3(kGnThreads), 0, s, 0, x, a.HW, a.C,
                                a.groups, pl.chunk, part);
  if (e != cudaSuccess) return e;
  GnApply p;
  p.M = a.B * a.HW; p.HW = a.HW; p.C = a.C; p.groups = a.groups; p.chunk = pl.chunk; p.chunks = pl.chunks;
  p.eps = a.eps; p.gamma = a.gamma; p.beta = a.beta; p.part = part; p.codes = a.codes; p.scales = a.scales;
  const bool w32 = access_of(x, a.C, a.C) == kW32;
  auto pick = [&](auto few) {
    constexpr bool F = decltype(few)::value;
    return a.silu ? (w32 ? mx4_gn_apply_kernel<T, kW32, true, F> : mx4_gn_apply_kernel<T, kW16, true, F>)
                  : (w32 ? mx4_gn_apply_kernel<T, kW32, false, F> : mx4_gn_apply_kernel<T, kW16, false, F>);
  };
  auto k = a.HW <= kGnPixels ? pick(std::true_type()) : pick(std::false_type());
  const int rts = mx_rtiles(p.M), kts = mx_ktiles(a.C);
  // tiles per block: fewest rounds of blocks (three per SM) weighted by a block's work, a merge counting half a tile
  double best = 1e30;
  for (int n = 1; n <= 8; ++n) {
    const long long blocks = (long long)((rts + n - 1) / n) * kts, slots = 3ll * num_sms();
    const double cost = (double)((blocks + slots - 1) / slots) * (n + 0.5);
    if (cost < best) { best = cost; p.tiles = n; }
  }
  return launch_kernel(k, dim3((rts + p.tiles - 1) / p.tiles * kts), dim3(kQThreads), 0, s, 0, x, p);
}

}  // namespace

cudaError_t launch_mx4_quantize(const void* x, int dtype, int M, int K, long long ldx, uint8_t* codes, uint8_t* scales,
                                cudaStream_t s) {
  switch (dtype) {
    case kF16: return quantize_t(static_cast<const __half*>(x), M, K, ldx, codes, scales, s);
    case kBF16: return quantize_t(static_cast<const __nv_bfloat16*>(x), M, K, ldx, codes, scales, s);
    case kF32: return quantize_t(static_cast<const float*>(x), M, K, ldx, codes, scales, s);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int M, int K, int dtype, void* y,
                                  cudaStream_t s) {
  switch (dtype) {
    case kF16: return dequantize_t(codes, scales, M, K, static_cast<__half*>(y), s);
    case kBF16: return dequantize_t(codes, scales, M, K, static_cast<__nv_bfloat16*>(y), s);
    case kF32: return dequantize_t(codes, scales, M, K, static_cast<float*>(y), s);
    default: return cudaErrorInvalidValue;
  }
}

size_t mx4_groupnorm_scratch_bytes(int B, int HW, int C, int groups) {
  if (C % 8 || C > kGnMaxC) return 0;
  return (size_t)B * gn_plan(HW, C).chunks * groups * sizeof(float2);
}

cudaError_t launch_mx4_groupnorm(const Mx4GroupNormArgs& a, cudaStream_t s) {
  if (a.C % 8 || a.C > kGnMaxC || a.C % a.groups || !aligned(a.x, 16)) return cudaErrorInvalidValue;
  switch (a.dtype) {
    case kF16: return groupnorm_t<__half>(a, s);
    case kBF16: return groupnorm_t<__nv_bfloat16>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace sdg

// mx4_quant.cu — MXFP4 quantisation and read-back, and GroupNorm (+ SiLU) written as an MXFP4 operand.
//
// All three walk the operand in its own scale tiles: one block of 256 threads per 128 rows x 128 columns,
// a half-warp per row and eight columns a lane (16-byte loads of 16-bit elements), a quad of lanes per
// 32-column block, whose maximum is two shuffles. Every load of the tile is issued before the first use (eight
// per thread), so a block keeps 32 KB of 16-bit input in flight. A row's codes leave as 64 contiguous bytes, the
// tile's 512 scale bytes are gathered in shared memory and leave as one.
#include <algorithm>

#include "mx4.cuh"
#include "sdg_kernels.h"
#include "sdg_launch.h"
#include "sdg_ptx.cuh"

namespace sdg {
namespace {

constexpr int kQThreads = 256;
constexpr int kQRows = kQThreads / 16;             // rows per pass
constexpr int kQPass = kMxTileRows / kQRows;       // passes per tile

template <typename T, bool VEC>
__device__ __forceinline__ void load_raw8(const T* src, int left, MxRaw8<T>& r) {  // left: columns from src to K
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < MxElem<T>::kVec; ++i)
      r.w[i] = left > 0 ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    T* e = reinterpret_cast<T*>(r.w);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < left ? src[i] : MxElem<T>::put(0.f);
  }
}

// Writes the scale tile gathered in shared memory and zeroes it where no row or block is.
__device__ __forceinline__ void put_scale_tile(const uint32_t* tile, uint8_t* dst) {
  if (threadIdx.x < kMxTileBytes / 4) reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = tile[threadIdx.x];
}

// VEC: K a multiple of 8, x and its row stride 16-byte aligned.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kQThreads) mx4_quantize_kernel(const T* __restrict__ x, int M, int K, long long ldx,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales) {
  __shared__ uint32_t tile[kMxTileBytes / 4];
  const int kt = blockIdx.y, kts = gridDim.y;
  const int row0 = blockIdx.x * kMxTileRows;
  const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int c = kt * kMxTileCols + l16 * 8;
  const int kp = mx_kp(K);
  if (threadIdx.x < kMxTileBytes / 4) tile[threadIdx.x] = 0u;
  pdl_wait();
  pdl_trigger();
  MxRaw8<T> raw[kQPass];
#pragma unroll
  for (int p = 0; p < kQPass; ++p) {
    const int r = row0 + p * kQRows + r0;
    load_raw8<T, VEC>(x + (size_t)min(r, M - 1) * ldx + c, r < M ? K - c : 0, raw[p]);
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kQPass; ++p) {
    const int rl = p * kQRows + r0, r = row0 + rl;
    float v[8];
    mx_unpack8<T>(raw[p], v);
    uint32_t e;
    const uint32_t q = mx_quantize_quad(v, e);
    if (r < M && c < kp) {
      *reinterpret_cast<uint32_t*>(codes + (size_t)r * (kp / 2) + c / 2) = q;
      if ((l16 & 3) == 0) reinterpret_cast<uint8_t*>(tile)[mx_scale_byte(rl, l16 >> 2)] = (uint8_t)e;
    }
  }
  __syncthreads();
  put_scale_tile(tile, scales + ((size_t)blockIdx.x * kts + kt) * kMxTileBytes);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQThreads) mx4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, int M, int K,
                                                                   T* __restrict__ y) {
  __shared__ uint32_t tile[kMxTileBytes / 4];
  const int kt = blockIdx.y, kts = gridDim.y;
  const int row0 = blockIdx.x * kMxTileRows;
  const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int c = kt * kMxTileCols + l16 * 8;
  const int kp = mx_kp(K);
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x < kMxTileBytes / 4)
    tile[threadIdx.x] =
        reinterpret_cast<const uint32_t*>(scales + ((size_t)blockIdx.x * kts + kt) * kMxTileBytes)[threadIdx.x];
  uint32_t q[kQPass];
#pragma unroll
  for (int p = 0; p < kQPass; ++p) {
    const int r = row0 + p * kQRows + r0;
    q[p] = (r < M && c < kp) ? *reinterpret_cast<const uint32_t*>(codes + (size_t)r * (kp / 2) + c / 2) : 0u;
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kQPass; ++p) {
    const int rl = p * kQRows + r0, r = row0 + rl;
    if (r >= M || c >= K) continue;
    const float s = mx_pow2(reinterpret_cast<const uint8_t*>(tile)[mx_scale_byte(rl, l16 >> 2)]);
    __half2 h[4];
    mx_decode8(q[p], h);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = f.x * s;
      v[2 * i + 1] = f.y * s;
    }
    T* dst = y + (size_t)r * K + c;
    if constexpr (VEC) {
      mx_store8<T>(dst, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < K) dst[i] = MxElem<T>::put(v[i]);
    }
  }
}

// ------------------------------------------------------------------ GroupNorm (+ SiLU) -> MXFP4
__device__ __forceinline__ float gn_block_sum(float v, float* red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) t += red[w];
  __syncthreads();
  return t;
}

// One block per (group, image): mean, then the centred variance, in a fixed order.
template <typename T>
__global__ void __launch_bounds__(512) mx4_gn_stats_kernel(const T* __restrict__ x, int HW, int C, int groups, float eps,
                                                           float2* __restrict__ stat) {
  __shared__ float red[16];
  pdl_wait();
  pdl_trigger();
  const int g = blockIdx.x, img = blockIdx.y, cpg = C / groups;
  const T* base = x + (size_t)img * HW * C + g * cpg;
  const long long n = (long long)HW * cpg;
  float s = 0.f;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) s += MxElem<T>::get(base[(i / cpg) * C + i % cpg]);
  const float mu = gn_block_sum(s, red) / (float)n;
  float m2 = 0.f;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) {
    const float d = MxElem<T>::get(base[(i / cpg) * C + i % cpg]) - mu;
    m2 += d * d;
  }
  const float var = gn_block_sum(m2, red) / (float)n;
  if (threadIdx.x == 0) stat[img * groups + g] = make_float2(mu, rsqrtf(var + eps));
}

// y * sigmoid(y) to a few fp32 ulps: the rounding to four bits comes after it, so the approximation must not move
// values across the E2M1 midpoints more often than fp32 arithmetic does
__device__ __forceinline__ float silu_exact(float y) { return __fdividef(y, 1.f + __expf(-y)); }

template <typename T>
__global__ void __launch_bounds__(kQThreads) mx4_gn_apply_kernel(const T* __restrict__ x, int M, int HW, int C, int groups,
                                                                 const float* __restrict__ gamma,
                                                                 const float* __restrict__ beta, int silu,
                                                                 const float2* __restrict__ stat,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales) {
  __shared__ uint32_t tile[kMxTileBytes / 4];
  const int kt = blockIdx.y, kts = gridDim.y;
  const int row0 = blockIdx.x * kMxTileRows;
  const int l16 = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int c = kt * kMxTileCols + l16 * 8;
  const int kp = mx_kp(C), cpg = C / groups;
  if (threadIdx.x < kMxTileBytes / 4) tile[threadIdx.x] = 0u;
  float ga[8], be[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ga[i] = c < C ? __ldg(gamma + c + i) : 0.f;
    be[i] = c < C ? __ldg(beta + c + i) : 0.f;
  }
  pdl_wait();
  pdl_trigger();
  MxRaw8<T> raw[kQPass];
#pragma unroll
  for (int p = 0; p < kQPass; ++p) {
    const int r = row0 + p * kQRows + r0;
    load_raw8<T, true>(x + (size_t)min(r, M - 1) * C + c, r < M ? C - c : 0, raw[p]);
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < kQPass; ++p) {
    const int rl = p * kQRows + r0, r = row0 + rl;
    float v[8];
    mx_unpack8<T>(raw[p], v);
    if (r < M && c < C) {
      const float2* st = stat + (size_t)(r / HW) * groups;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 s = st[(c + i) / cpg];
        v[i] = (v[i] - s.x) * s.y * ga[i] + be[i];
        if (silu) v[i] = silu_exact(v[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    uint32_t e;
    const uint32_t q = mx_quantize_quad(v, e);
    if (r < M && c < kp) {
      *reinterpret_cast<uint32_t*>(codes + (size_t)r * (kp / 2) + c / 2) = q;
      if ((l16 & 3) == 0) reinterpret_cast<uint8_t*>(tile)[mx_scale_byte(rl, l16 >> 2)] = (uint8_t)e;
    }
  }
  __syncthreads();
  put_scale_tile(tile, scales + ((size_t)blockIdx.x * kts + kt) * kMxTileBytes);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
cudaError_t quantize_t(const T* x, int M, int K, long long ldx, uint8_t* codes, uint8_t* scales, cudaStream_t s) {
  const dim3 grid(mx_rtiles(M), mx_ktiles(K));
  const bool vec = K % 8 == 0 && aligned16(x) && (ldx * sizeof(T)) % 16 == 0;
  auto k = vec ? mx4_quantize_kernel<T, true> : mx4_quantize_kernel<T, false>;
  return launch_kernel(k, grid, dim3(kQThreads), 0, s, 0, x, M, K, ldx, codes, scales);
}
template <typename T>
cudaError_t dequantize_t(const uint8_t* codes, const uint8_t* scales, int M, int K, T* y, cudaStream_t s) {
  const dim3 grid(mx_rtiles(M), mx_ktiles(K));
  const bool vec = K % 8 == 0 && aligned16(y);
  auto k = vec ? mx4_dequantize_kernel<T, true> : mx4_dequantize_kernel<T, false>;
  return launch_kernel(k, grid, dim3(kQThreads), 0, s, 0, codes, scales, M, K, y);
}
template <typename T>
cudaError_t groupnorm_t(const Mx4GroupNormArgs& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.x);
  float2* stat = reinterpret_cast<float2*>(a.stats);
  cudaError_t e = launch_kernel(mx4_gn_stats_kernel<T>, dim3(a.groups, a.B), dim3(512), 0, s, 0, x, a.HW, a.C, a.groups,
                                a.eps, stat);
  if (e != cudaSuccess) return e;
  const int M = a.B * a.HW;
  return launch_kernel(mx4_gn_apply_kernel<T>, dim3(mx_rtiles(M), mx_ktiles(a.C)), dim3(kQThreads), 0, s, 0, x, M, a.HW,
                       a.C, a.groups, a.gamma, a.beta, a.silu, (const float2*)stat, a.codes, a.scales);
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
  (void)HW;
  (void)C;
  return (size_t)B * groups * sizeof(float2);
}

cudaError_t launch_mx4_groupnorm(const Mx4GroupNormArgs& a, cudaStream_t s) {
  if (a.C % 8 || a.C % a.groups || !aligned16(a.x)) return cudaErrorInvalidValue;
  switch (a.dtype) {
    case kF16: return groupnorm_t<__half>(a, s);
    case kBF16: return groupnorm_t<__nv_bfloat16>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace sdg

// mx4_linear.cu — y = act(x w^T + bias + residual) of two MXFP4 operands (format: mx4.cuh).
//
// mx4_rows_kernel: the product on the CUDA cores, one warp per output column (value and gate column for GEGLU)
// and up to MB rows. A lane takes 16 columns at a time (8 bytes of each operand): the codes decode to fp16
// exactly, and the eight products a half of each pair adds up stay exact in fp16 (at most 8 * 36 = 288 in steps of
// 1/4: 1152 steps, fewer than the 2048 an fp16 significand holds). Block scales, and the sums over blocks, are fp32.
#include <algorithm>

#include "mx4.cuh"
#include "sdg_kernels.h"
#include "sdg_launch.h"
#include "sdg_ptx.cuh"

namespace sdg {
namespace {

constexpr int kRowsWarps = 8;

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
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(a.wcodes + (size_t)wr[w] * (kp / 2)) + u);
      wsc[w] = mx_pow2(__ldg(a.wscales + ((size_t)(wr[w] >> 7) * kts + (b >> 2)) * kMxTileBytes + mx_scale_byte(wr[w], b)));
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
        if (a.act == 1) v = silu_f(v);
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

template <typename T>
cudaError_t linear_t(const Mx4LinearArgs& a, cudaStream_t s) {
  return a.M == 1 ? launch_rows<T, 1>(a, s) : launch_rows<T, 4>(a, s);
}

}  // namespace

cudaError_t launch_mx4_linear(const Mx4LinearArgs& a, int* dev_err, cudaStream_t s) {
  (void)dev_err;
  return a.dtype == kBF16 ? linear_t<__nv_bfloat16>(a, s) : linear_t<__half>(a, s);
}

}  // namespace sdg

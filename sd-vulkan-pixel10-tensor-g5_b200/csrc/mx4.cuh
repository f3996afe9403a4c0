// mx4.cuh — the MXFP4 operand format (OCP Microscaling Formats 1.0: E2M1 values, one E8M0 exponent per
// 32 consecutive columns of a row) and its device helpers.
//
// A matrix [R, K] is two arrays. codes [R][Kp/2] (Kp = K rounded up to 32), two values a byte, the even
// column in the low nibble, zero behind column K: a row's pitch is a multiple of 16 bytes, so TMA reads
// it as a plain byte matrix. scales in tiles of 128 rows x 4 blocks (128 columns), [ceil(R/128)]
// [ceil(Kp/128)][512]: the exponent of row r, block b is byte (r % 32) * 16 + (r / 32 % 4) * 4 + b % 4 of
// its tile, which is the order in which tcgen05.cp.32x128b.warpx4 puts one tile into 32 TMEM lanes x 4
// columns for tcgen05.mma.kind::mxf4 (lane r % 32, column r / 32, byte b), so a tile goes from HBM to TMEM
// without a rearrangement. Bytes that belong to no block are zero (2^-127): with the zero codes that TMA
// fills in they add zero, never a NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "sdg_ptx.cuh"

namespace sdg {

constexpr int kMxBlock = 32;        // columns per exponent
constexpr int kMxTileRows = 128;    // scale tile: rows ...
constexpr int kMxTileCols = 128;    // ... x columns (4 blocks)
constexpr int kMxTileBytes = 512;

__host__ __device__ inline int mx_kp(int K) { return (K + kMxBlock - 1) / kMxBlock * kMxBlock; }
__host__ __device__ inline int mx_ktiles(int K) { return (K + kMxTileCols - 1) / kMxTileCols; }
__host__ __device__ inline int mx_rtiles(int R) { return (R + kMxTileRows - 1) / kMxTileRows; }

// byte of (row r, block b) inside its scale tile
__host__ __device__ inline int mx_scale_byte(int r, int b) { return (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3); }

// 2^(e - 127); e = 0 is the subnormal 2^-127, 255 is NaN
__device__ __forceinline__ float mx_pow2(uint32_t e) {
  return __uint_as_float(e == 0 ? 0x00400000u : (e == 255u ? 0x7FC00000u : e << 23));
}

// Biased block exponent from the bits of max|x|: floor(log2 max) - 2 (2 = E2M1's largest exponent), at least
// -127; 255 (NaN) when the block holds an infinity or a NaN. fp32 subnormals (bits >> 23 == 0) clamp to 0.
__device__ __forceinline__ uint32_t mx_exponent(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 1 / 2^(e - 127) for e <= 252: multiplying by it is exact (a result small enough to round is far below
// E2M1's first midpoint)
__device__ __forceinline__ float mx_inverse(uint32_t e) { return __uint_as_float((254u - e) << 23); }

// eight values already divided by their block's scale -> eight E2M1 codes (value i in nibble i), rounded to
// nearest even, saturated at +-6
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// eight E2M1 codes -> four fp16 pairs (exact)
__device__ __forceinline__ void mx_decode8(uint32_t c, __half2 (&h)[4]) {
  uint32_t r[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(c));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = reinterpret_cast<__half2&>(r[i]);
}

// Codes of N (8 or 16) values under exponent e, N/8 words; a block with an infinity or a NaN (e = 255) gets codes 0.
template <int N>
__device__ __forceinline__ void mx_codes(float (&v)[N], uint32_t e, uint32_t (&q)[N / 8]) {
  const float inv = e == 255u ? 0.f : mx_inverse(e);
  const float2 inv2 = make_float2(inv, inv);
#pragma unroll
  for (int w = 0; w < N / 8; ++w) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = mul_f32x2(make_float2(v[8 * w + 2 * i], v[8 * w + 2 * i + 1]), inv2);
      s[2 * i] = f.x;
      s[2 * i + 1] = f.y;
    }
    const uint32_t c = mx_encode8(s);
    q[w] = e == 255u ? 0u : c;
  }
}

// ------------------------------------------------------------------ 16/32-bit element types
template <typename T> struct MxElem;
template <> struct MxElem<__half> {
  // fp32 bits of a |value| from its 16 bits (ordered alike, infinities and NaNs on top)
  static __device__ __forceinline__ uint32_t abs_bits(uint32_t h) {
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
  }
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t put2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return reinterpret_cast<const uint32_t&>(h);
  }
  static __device__ __forceinline__ float2 get2(uint32_t w) { return __half22float2(reinterpret_cast<__half2&>(w)); }
};
template <> struct MxElem<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t abs_bits(uint32_t h) { return h << 16; }
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t put2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<const uint32_t&>(h);
  }
  static __device__ __forceinline__ float2 get2(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
};
template <> struct MxElem<float> {
  static __device__ __forceinline__ float put(float v) { return v; }
};

// 32 bytes of a row as loaded: 16 values of 16 bits or 8 of 32 bits
template <typename T>
struct MxRaw {
  static constexpr int kN = 32 / sizeof(T);
  uint32_t w[8];
};

template <typename T>
__device__ __forceinline__ void mx_unpack(const MxRaw<T>& r, float (&v)[MxRaw<T>::kN]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(r.w[i]);
    } else {
      const float2 f = MxElem<T>::get2(r.w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// max |value| of the raw 32 bytes: 32-bit values as fp32 bits; 16-bit values two at a time as packed 16-bit
// integers (half the integer instructions of widening first)
template <typename T>
__device__ __forceinline__ uint32_t mx_raw_amax(const MxRaw<T>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = sizeof(T) == 4 ? max(m, r.w[i] & 0x7FFFFFFFu) : __vmaxu2(m, r.w[i] & 0x7FFF7FFFu);
  return m;
}
// ... of the whole block, over the lanes that share it (a pair of lanes of 16 values, a quad of 8), as fp32 bits
template <typename T>
__device__ __forceinline__ uint32_t mx_block_amax(uint32_t m) {
  if constexpr (sizeof(T) == 4) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  } else {
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    return MxElem<T>::abs_bits(max(m & 0xFFFFu, m >> 16));
  }
}

__device__ __forceinline__ void mx_ld32(const void* p, uint32_t (&w)[8]) {  // 32-byte aligned
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void mx_st32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p)
               : "memory");
}

// eight 16-bit values <-> fp32
template <typename T>
__device__ __forceinline__ void mx_unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = MxElem<T>::get2(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void mx_store8(T* dst, const float (&v)[8]) {  // dst 16-byte aligned
  uint4 u;
  u.x = MxElem<T>::put2(v[0], v[1]);
  u.y = MxElem<T>::put2(v[2], v[3]);
  u.z = MxElem<T>::put2(v[4], v[5]);
  u.w = MxElem<T>::put2(v[6], v[7]);
  *reinterpret_cast<uint4*>(dst) = u;
}

}  // namespace sdg

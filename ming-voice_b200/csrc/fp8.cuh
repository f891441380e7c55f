// Shared pieces of the products with 8-bit floating-point weights: conversions, the activations' block scale, arguments.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace mv {
namespace fp8 {

constexpr int kBlock = 128;  // columns (and rows of a weight) that share a scale

struct LinearArgs {
  const void* x;           // activations as they come
  long long x_st;
  int x_dtype;
  const uint8_t* w;        // [N, K] e4m3
  const float* ws;         // [N / 128, K / 128]
  uint8_t* q;              // activations [T, blocks * 128] e4m3
  uint8_t* scale;          // [blocks, T]: the exponents of the powers of two, 127 added (an fp32 number's)
  const void* residual;
  void* out;
  long long w_st, ws_st, q_st, s_st, r_st, o_st;
  int T, N, K, blocks;
  WsHeader* header;
};

// the products (fp8_gemm.cu); w is 16-byte aligned with rows of whole 16 bytes, q and scale are in the scratch
int run_product(const LinearArgs& a, int out_dtype, cudaStream_t st);
// whether it rounds the activations itself (of T, N, K, blocks)
bool one_launch(const LinearArgs& a);

// row stride of the activations' scales: rows begin at whole 16 bytes
inline long long scale_stride(int T) { return (static_cast<long long>(T) + 15) / 16 * 16; }

template <int DT>
__device__ __forceinline__ float load1(const void* p, long long i) {
  if (DT == MV_F32) return static_cast<const float*>(p)[i];
  if (DT == MV_BF16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
  return __half2float(static_cast<const __half*>(p)[i]);
}

template <int DT>
__device__ __forceinline__ void store1(void* p, long long i, float v) {
  if (DT == MV_F32)
    static_cast<float*>(p)[i] = v;
  else if (DT == MV_BF16)
    static_cast<uint16_t*>(p)[i] = f2bf(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

template <int DT>
__device__ __forceinline__ float2 unpack(uint32_t w) {
  if (DT == MV_BF16) return make_float2(bf16lo(w), bf16hi(w));
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return __half22float2(h);
}

template <int DT>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if (DT == MV_BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Values c0 .. c0 + 7 of the row at element offset `row`; zeros from column K on. VEC (of 16-bit types): 8 and 4 load 16 and 8
// bytes at a time, where row and K allow it; f32 with VEC 8 loads 16 bytes twice.
template <int DT, int VEC>
__device__ __forceinline__ void load8(const void* x, long long row, int c0, int K, float (&v)[8]) {
  if (VEC == 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < K ? load1<DT>(x, row + c0 + i) : 0.f;
  } else if (DT == MV_F32) {
    float4 p = make_float4(0.f, 0.f, 0.f, 0.f), r = p;
    if (c0 < K) {
      const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(x) + row + c0);
      p = src[0], r = src[1];
    }
    v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = r.x, v[5] = r.y, v[6] = r.z, v[7] = r.w;
  } else {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    const uint16_t* src = static_cast<const uint16_t*>(x) + row + c0;
    if (VEC == 8) {
      if (c0 < K) {
        const uint4 p = *reinterpret_cast<const uint4*>(src);
        w[0] = p.x, w[1] = p.y, w[2] = p.z, w[3] = p.w;
      }
    } else {
      if (c0 < K) {
        const uint2 p = *reinterpret_cast<const uint2*>(src);
        w[0] = p.x, w[1] = p.y;
      }
      if (c0 + 4 < K) {
        const uint2 p = *reinterpret_cast<const uint2*>(src + 4);
        w[2] = p.x, w[3] = p.y;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack<DT>(w[i]);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

// The scale 2^e of a block whose largest magnitude has these bits, and 2^-e: e is the smallest integer >= -126 with
// max <= 448 * 2^e = 1.75 * 2^(e + 8). Infinities and NaNs: scale NaN, factor 0.
__device__ __forceinline__ void block_scale(uint32_t top, float& up, float& down) {
  if (top >= 0x7f800000u) {
    up = __uint_as_float(0x7fc00000u), down = 0.f;
    return;
  }
  const int e = max(static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
  up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
  down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
}

// two values to e4m3, nearest even: `lo` in bits 0-7, `hi` in bits 8-15
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint2 round8(const float (&v)[8], float down) {
  uint2 o;
  o.x = e4m3x2(v[0] * down, v[1] * down) | e4m3x2(v[2] * down, v[3] * down) << 16;
  o.y = e4m3x2(v[4] * down, v[5] * down) | e4m3x2(v[6] * down, v[7] * down) << 16;
  return o;
}

}  // namespace fp8
}  // namespace mv

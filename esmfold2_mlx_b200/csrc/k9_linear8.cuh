// K9: linear layer with 8-bit (e4m3) operands and a scale for each block of 128 values.
//
//   out[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} x8[m, k] w8[n, k]  (+ bias[n])
//
// x8 [M, K] with one scale a row and block of 128 along K, w8 [N, K] with one scale a 128 x 128
// block.  quantize_kernel makes x8, xs from a 16-bit x: xs = max(amax / 448, 2^-126) (448 is
// e4m3's largest value) and x8 = e4m3(x / xs), both quotients rounded as IEEE fp32 divisions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "k8_qk_rope.cuh"

namespace tmu {
namespace k9 {

constexpr int kQuantThreads = 256;

struct QuantParams {
  const void* x;
  long long ld;
  int M, K, kb;
  uint8_t* x8;  // [M, K]
  float* xs;    // [M, kb]
};

__device__ __forceinline__ float max_nan(float a, float b) {  // keeps a NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two fp32 to two e4m3 (the low one in the low byte), to nearest even, saturating at 448; NaN stays.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Half a warp takes one block of 128 of one row: 8 values (16 bytes) a lane, amax by shuffles.
// Bound: HBM (2 bytes read and 1 written a value).
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(const __grid_constant__ QuantParams p) {
  const int l = threadIdx.x & 15;
  const long long items = static_cast<long long>(p.M) * p.kb;
  const long long step = static_cast<long long>(gridDim.x) * (kQuantThreads / 16);
  const long long first = (static_cast<long long>(blockIdx.x) * kQuantThreads + threadIdx.x) >> 4;
  griddep_wait();
  // the two halves of a warp run the same number of turns, so the shuffles meet
  for (long long base = first - ((threadIdx.x >> 4) & 1); base < items; base += step) {
    const long long it = base + ((threadIdx.x >> 4) & 1);
    const long long m = it / p.kb;
    const int b = static_cast<int>(it - m * p.kb), k = b * 128 + l * 8;
    const bool on = it < items && k < p.K;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (on) raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + m * p.ld + k);
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    float y[8], amax = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = k8::unpack2(u[e], T());
      y[2 * e] = f.x;
      y[2 * e + 1] = f.y;
      amax = max_nan(amax, max_nan(fabsf(f.x), fabsf(f.y)));
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float s = max_nan(__fdiv_rn(amax, 448.f), 0x1p-126f);
    if (on) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = e4m3x2(__fdiv_rn(y[2 * e], s), __fdiv_rn(y[2 * e + 1], s));
      *reinterpret_cast<uint2*>(p.x8 + m * p.K + k) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    }
    if (it < items && l == 0) p.xs[m * p.kb + b] = s;
  }
  griddep_trigger();
}

enum Out : int { kF16 = 0, kBf16 = 1, kF32 = 2 };

struct Params {
  const uint8_t* x8;
  const float* xs;
  const uint8_t* w8;
  const float* ws;
  const float* bias;
  void* out;
  long long ldo;
  int M, N, K, kb, out_type;
};

__device__ __forceinline__ void store_out(void* out, int type, long long at, float v) {
  if (type == kF16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else if (type == kBf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(out)[at] = v;
}

__device__ __forceinline__ float from_e4m3(uint8_t v) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(v, __NV_E4M3);
  return __half2float(__half(h));
}

// One thread an output.
__global__ void __launch_bounds__(256) linear8_simple_kernel(const __grid_constant__ Params p) {
  griddep_wait();
  const int n = blockIdx.x * 16 + (threadIdx.x & 15), m = blockIdx.y * 16 + (threadIdx.x >> 4);
  if (n >= p.N || m >= p.M) return;
  float acc = 0.f;
  for (int b = 0; b < p.kb; ++b) {
    float s = 0.f;
    const int k1 = min(p.K, b * 128 + 128);
    for (int k = b * 128; k < k1; ++k)
      s = fmaf(from_e4m3(p.x8[static_cast<long long>(m) * p.K + k]), from_e4m3(p.w8[static_cast<long long>(n) * p.K + k]), s);
    acc = fmaf(s, p.xs[static_cast<long long>(m) * p.kb + b] * p.ws[static_cast<long long>(n >> 7) * p.kb + b], acc);
  }
  store_out(p.out, p.out_type, m * p.ldo + n, acc + (p.bias ? p.bias[n] : 0.f));
}

}  // namespace k9
}  // namespace tmu

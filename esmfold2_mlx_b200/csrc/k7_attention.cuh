// K7: attention over packed sequences.
//
// Row i of sequence s (tokens cu[s] .. cu[s + 1]) and query head h, key head h / (Hq / Hkv):
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(x_ij - max_j x_ij),   x_ij = scale q_i . k_j + bias_ij
// over the keys j of the same sequence, j <= i if causal.  A row whose keys are all at -inf is zero.
#pragma once

#include <cuda_bf16.h>

#include "k8_qk_rope.cuh"

namespace tmu {
namespace k7 {

struct Params {
  k8::View q, k, v, o;
  const int* cu;
  const void* bias;  // [S or 1, Hq, n, n] or null, the last axis contiguous
  long long bias_ss, bias_sh, bias_sr;
  int bias_n;
  int S, T, hq, hkv, d, causal;
  float scale;
};

constexpr int kSimpleThreads = 128;

// One warp a row and head; lanes take keys for the scores and head values for the output.
template <typename T>
__global__ void __launch_bounds__(kSimpleThreads) attention_rows_kernel(const __grid_constant__ Params p) {
  __shared__ float qs[kSimpleThreads / 32][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long item = static_cast<long long>(blockIdx.x) * (kSimpleThreads / 32) + warp;
  if (item >= static_cast<long long>(p.T) * p.hq) return;
  const int t = static_cast<int>(item / p.hq), h = static_cast<int>(item % p.hq);
  int beg = 0, end = 0, seq = -1;
  for (int s = 0; s < p.S; ++s) {
    const int b = min(max(p.cu[s], 0), p.T), e = min(max(p.cu[s + 1], b), p.T);
    if (t >= b && t < e) {
      beg = b;
      end = e;
      seq = s;
      break;
    }
  }
  if (seq < 0) return;
  const int kv = h / (p.hq / p.hkv), i = t - beg;
  const T* q = static_cast<const T*>(p.q.p) + t * p.q.st + h * p.q.sh;
  for (int d = lane; d < 128; d += 32) qs[warp][d] = d < p.d ? static_cast<float>(q[d]) : 0.f;
  __syncwarp();
  const int last = p.causal ? i + 1 : end - beg;
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < last; j0 += 32) {
    const int j = j0 + lane;
    float x = -INFINITY;
    if (j < last) {
      const T* k = static_cast<const T*>(p.k.p) + static_cast<long long>(beg + j) * p.k.st + kv * p.k.sh;
      float acc = 0.f;
      for (int d = 0; d < p.d; ++d) acc = fmaf(qs[warp][d], static_cast<float>(k[d]), acc);
      x = acc * p.scale;
      if (p.bias != nullptr && i < p.bias_n && j < p.bias_n)
        x += static_cast<float>(static_cast<const T*>(p.bias)[seq * p.bias_ss + h * p.bias_sh + i * p.bias_sr + j]);
    }
    float mx = x;
    for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    const float mn = fmaxf(m, mx);
    if (mn == -INFINITY) continue;
    const float f = expf(m - mn);
    const float pj = expf(x - mn);
    float ps = pj;
    for (int w = 16; w > 0; w >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, w);
    l = l * f + ps;
    m = mn;
    for (int e = 0; e < 4; ++e) o[e] *= f;
    for (int jj = 0; jj < 32 && j0 + jj < last; ++jj) {
      const float w = __shfl_sync(0xffffffffu, pj, jj);
      const T* v = static_cast<const T*>(p.v.p) + static_cast<long long>(beg + j0 + jj) * p.v.st + kv * p.v.sh;
      for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < p.d) o[e] = fmaf(w, static_cast<float>(v[lane + 32 * e]), o[e]);
    }
  }
  T* out = static_cast<T*>(p.o.p) + t * p.o.st + h * p.o.sh;
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < p.d) out[lane + 32 * e] = static_cast<T>(o[e] * inv);
}

}  // namespace k7
}  // namespace tmu

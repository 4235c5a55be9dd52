// K8: norm of every query and key head and the rotation by position, in one pass over q and k.
//
// For head h of token t, x = its D values, in fp32:
//   rms    y = x / sqrt(mean(x^2) + eps) * w            layer  y = (x - mean) / sqrt(var + eps) * w + b
// then the pairs (y1, y2) of the first `rot` values turn by angle pos[t] * f_i,
//   (y1 cos - y2 sin, y2 cos + y1 sin) * gain,
// pair i being (i, i + rot / 2) in the half layout and (2i, 2i + 1) in the interleaved one, and the
// row is rounded once to its 16-bit type.
//
// The angle.  f_i is kept as turns a position in 64-bit fixed point, F_i = round(f_i / 2 pi * 2^64):
// the product pos * F_i wraps modulo 2^64, which is modulo one turn, so its top 32 bits are the
// angle's fraction of a turn to 2^-32 (1.5e-9 rad) for every position, however far, and no table
// of positions has to be kept or bounded.  (An fp32 product pos * f_i is off by up to pos * 2^-24 rad.)
//
// Bound: HBM (each value is read once and written once, 4 bytes moved for about 20 operations).
// Split: 16 bytes a lane and LPH = D / 8 lanes (rounded up to a power of two) a head, so a warp
// reads 32 / LPH heads at a time and the sums over a head are shuffles inside its lanes; a lane's
// eight values belong to the same pairs in every head, so the sines of a token are computed once
// for all the heads that the warp visits.  The partner of a half-layout pair sits rot / 16 lanes
// away: one shuffle a value.  Few tokens: the heads are split over more warps (the host's `slices`).
#pragma once

#include <cuda_bf16.h>

#include "tmu_common.cuh"

namespace tmu {

// The producer and MMA warps of the sequence kernels walk their loops as whole warps and let one
// elected lane issue: the values that TMA and MMA instructions take from uniform registers are then
// computed there instead of being moved there one by one (the 8-bit pair kernel: 585 -> 521 us).

// Where the sequence kernels' status goes in calls without a status block of their own.
__device__ DeviceStatus g_own_status;

// The whole warp waits for a phase of an mbarrier, every lane polling: from a commit to the answering
// arrive of 16 warps it took 475 cycles, against 667 with one lane waiting and telling the others.
// Bounded like mbar_wait; the verdict is the warp's.
__device__ __forceinline__ bool warp_poll(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, unsigned int site) {
  bool ok = false;
  for (int i = 0; i < 64 && !ok; ++i) ok = mbar_test(bar, parity);
  if (!__all_sync(0xffffffffu, ok)) {
    if (!ok) ok = mbar_wait(bar, parity, ctx, site);
    ok = __all_sync(0xffffffffu, ok);
  }
  return ok;
}

__device__ __forceinline__ bool elect_one() {  // one lane of the warp
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(on));
  return on != 0;
}

namespace k8 {

constexpr int kThreads = 128;

enum Norm : int { kNone = 0, kRms = 1, kLayer = 2 };

struct View {  // [T, H, D], the last axis contiguous
  void* p;
  long long st, sh;  // element strides of a token and a head
};

struct Params {
  View q, k, qo, ko;
  const void* pos;
  const unsigned long long* turns;  // [rot / 2]
  const float *qw, *qb, *kw, *kb;   // [D] or null
  float gain, eps, inv_d;
  int pos64, rot, T, hq, heads, d, slices, passes;  // a warp makes `passes` passes of 32 / LPH heads
};

__device__ __forceinline__ float2 unpack2(uint32_t u, __half) { return unpack_half2(u); }
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int LPH>
__device__ __forceinline__ float head_sum(float x) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <typename T, int LPH, int NORM, bool INTER>
__global__ void __launch_bounds__(kThreads) qk_rope_kernel(const __grid_constant__ Params p) {
  constexpr int HPW = 32 / LPH;
  const int lane = threadIdx.x & 31;
  const int c = lane & (LPH - 1);
  const long long item = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const long long t = item / p.slices;
  if (t >= p.T) return;  // a whole warp
  const int slice = static_cast<int>(item - t * p.slices);
  const bool act = c * 8 < p.d;
  const int d0 = act ? c * 8 : 0;
  griddep_wait();

  // cos, sin of this lane's values (cos = 1, sin = 0 past the rotated part)
  constexpr int NA = INTER ? 4 : 8;
  float cs[NA], sn[NA];
  const bool turned = act && c * 8 < p.rot;
#pragma unroll
  for (int e = 0; e < NA; ++e) {
    cs[e] = 1.f;
    sn[e] = 0.f;
  }
  if (turned) {
    const unsigned long long pos = p.pos64 ? static_cast<unsigned long long>(static_cast<const long long*>(p.pos)[t])
                                           : static_cast<unsigned long long>(static_cast<long long>(static_cast<const int*>(p.pos)[t]));
    const int half = p.rot >> 1;
    const int i0 = INTER ? c * 4 : (c * 8 < half ? c * 8 : c * 8 - half);
    const bool second = !INTER && c * 8 >= half;
#pragma unroll
    for (int e = 0; e < NA; ++e) {
      const long long turn = static_cast<long long>(pos * __ldg(p.turns + i0 + e));
      sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 0x1p-31f, &sn[e], &cs[e]);
      cs[e] *= p.gain;
      sn[e] *= second || INTER ? p.gain : -p.gain;  // y1 cos - y2 sin, y2 cos + y1 sin
    }
  }
  const int shift = p.rot >> 4;
  const int src = turned && !INTER ? (c < shift ? lane + shift : lane - shift) : lane;

  const int h_begin = slice * p.passes * HPW + lane / LPH;
#pragma unroll 2
  for (int k = 0; k < p.passes; ++k) {
    const int h = h_begin + k * HPW;
    const bool isq = h < p.hq;
    const bool on = act && h < p.heads;
    const int hh = isq ? h : h - p.hq;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (on) {
      const View& in = isq ? p.q : p.k;
      raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(in.p) + t * in.st + hh * in.sh + d0);
    }
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
    float y[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2(u[e], T());
      y[2 * e] = f.x;
      y[2 * e + 1] = f.y;
    }
    if (NORM != kNone) {
      if (NORM == kLayer) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += y[e];
        const float mean = head_sum<LPH>(s) * p.inv_d;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = act ? y[e] - mean : 0.f;
      }
      float s2 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s2 = fmaf(y[e], y[e], s2);
      const float r = rsqrtf(fmaf(head_sum<LPH>(s2), p.inv_d, p.eps));
      const float* w = isq ? p.qw : p.kw;
      const float* b = isq ? p.qb : p.kb;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const float4 ww = w ? __ldg(reinterpret_cast<const float4*>(w + d0) + v) : make_float4(1.f, 1.f, 1.f, 1.f);
        const float4 bb = b ? __ldg(reinterpret_cast<const float4*>(b + d0) + v) : make_float4(0.f, 0.f, 0.f, 0.f);
        y[4 * v] = fmaf(y[4 * v] * r, ww.x, bb.x);
        y[4 * v + 1] = fmaf(y[4 * v + 1] * r, ww.y, bb.y);
        y[4 * v + 2] = fmaf(y[4 * v + 2] * r, ww.z, bb.z);
        y[4 * v + 3] = fmaf(y[4 * v + 3] * r, ww.w, bb.w);
      }
    }
    float o[8];
    if (INTER) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[2 * e] = turned ? y[2 * e] * cs[e] - y[2 * e + 1] * sn[e] : y[2 * e];
        o[2 * e + 1] = turned ? y[2 * e + 1] * cs[e] + y[2 * e] * sn[e] : y[2 * e + 1];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = __shfl_sync(0xffffffffu, y[e], src);
        o[e] = turned ? fmaf(y[e], cs[e], other * sn[e]) : y[e];
      }
    }
    if (on) {
      const View& out = isq ? p.qo : p.ko;
      *reinterpret_cast<uint4*>(static_cast<T*>(out.p) + t * out.st + hh * out.sh + d0) =
          make_uint4(pack2(o[0], o[1], T()), pack2(o[2], o[3], T()), pack2(o[4], o[5], T()), pack2(o[6], o[7], T()));
    }
  }
  griddep_trigger();
}

}  // namespace k8
}  // namespace tmu

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
// angle's fraction of a turn, and no table of positions has to be kept or bounded.  F_i's rounding puts
// it off by |pos| 2^-65 of a turn (2^-33 at 2^32 positions), its own to fp32 by 2^-26 of a turn (9e-8 rad).
// (An fp32 product pos * f_i is off by up to pos * 2^-24 rad.)
//
// Bound: HBM (each value is read once and written once, 4 bytes moved for about 20 operations).
// Split: D / 8 lanes (rounded up to a power of two, LPH) a head and 8 values a lane, as two runs of
// four: in the half layout the runs of both members of four pairs, so no value leaves its lane for
// its rotation; else eight in a row.  A warp takes 32 / LPH heads at a time and the sums over a
// head are shuffles inside its lanes.  A lane's values belong to the same four pairs in every
// head, so the sines of a token, and a tensor's weights, are made once for all the heads that the
// warp visits.  The loads of kBatch turns are issued before the first is worked on.  Few tokens: the
// heads are split over more warps (the host's `slices`).
// Measured: 16384 tokens, 80 heads of 64, layer norm 62 us, 5.4 TB/s; 40 heads of 64 without a norm 30 us.
#pragma once

#include <cuda_bf16.h>

#include "tmu_common.cuh"

namespace tmu {

// The producer and MMA warps of the sequence kernels walk their loops as whole warps and let one
// elected lane issue: the values that TMA and MMA instructions take from uniform registers are then
// computed there instead of being moved there one by one (the 8-bit pair kernel: 585 -> 521 us).

// Where the sequence kernels' status goes in calls without a status block of their own
// (tmu_sequence_status gives it to the host).
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
  int pos64, rot, T, hq, hk, d;
  int q_turns, all_turns;  // turns of 32 / LPH heads that q, and q and k, take
  int slices, turns_each;  // warps of a token, and the turns that each takes
};

constexpr int kBatch = 4, kJoin = 2;  // turns whose loads are issued together, and whose sums are made together

__device__ __forceinline__ float2 unpack2(uint32_t u, __half) { return unpack_half2(u); }
__device__ __forceinline__ float2 unpack2(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 1 / sqrt(x) for normal x by the hardware's approximation (off by about 2^-22.9); x of 0 gives
// infinity, and with eps = 0 a head of zeros a NaN, as the division does.
__device__ __forceinline__ float rsqrt_near(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums over the LPH lanes of a head, of several values at a time.
template <int LPH, int N>
__device__ __forceinline__ void head_sums(float (&x)[N]) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
}

template <typename T, int LPH, int NORM, bool INTER>
__global__ void __launch_bounds__(kThreads, NORM == kNone ? 0 : 6) qk_rope_kernel(const __grid_constant__ Params p) {
  constexpr int HPW = 32 / LPH;
  // With a layer norm, whose two sums a turn waits for, the loads of a later turn follow each turn's
  // stores (16384 tokens, 80 heads of 64: 69 -> 65 us); with one sum or none that costs more than it brings
  // (5003 tokens, 40 heads of 128: 19.8 -> 20.3 us with the rms norm, 15.3 -> 15.9 without one).  A norm's
  // kernels keep to the registers of six blocks an SM: 65 -> 62 us, and 62.8 -> 58 at 16384 tokens, 20 heads of
  // 256, rms.
  constexpr bool kAhead = NORM == kLayer;
  const int lane = threadIdx.x & 31;
  const int c = lane & (LPH - 1), sub = lane / LPH;
  const long long item = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const long long t = item / p.slices;
  if (t >= p.T) return;  // a whole warp
  const int first = static_cast<int>(item - t * p.slices) * p.turns_each, last = min(first + p.turns_each, p.all_turns);
  const bool act = c * 8 < p.d, turned = c * 8 < p.rot;  // (rot <= d)
  // the lane's two runs of four values
  int d0 = c * 8, d1 = c * 8 + 4;
  if (!INTER && turned) {
    d0 = c * 4;
    d1 = (p.rot >> 1) + c * 4;
  }
  griddep_wait();

  // cos, sin of the lane's four pairs
  float cs[4], sn[4], ns[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    cs[e] = 1.f;
    sn[e] = ns[e] = 0.f;
  }
  if (turned) {
    const long long pos = p.pos64 ? static_cast<const long long*>(p.pos)[t] : static_cast<const int*>(p.pos)[t];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long long turn = static_cast<long long>(static_cast<unsigned long long>(pos) * __ldg(p.turns + c * 4 + e));
      sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 0x1p-31f, &sn[e], &cs[e]);
      cs[e] *= p.gain;
      sn[e] *= p.gain;
      ns[e] = -sn[e];
    }
  }

  // turns [begin, end) of one tensor
  auto run = [&](const View& in, const View& out, int heads, int begin, int end, const float* w, const float* b) {
    if (begin >= end) return;
    float2 ww[4], bb[4];
    if (NORM != kNone) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int at = (v < 2 ? d0 : d1) + (v & 1) * 2;
        ww[v] = w != nullptr && act ? __ldg(reinterpret_cast<const float2*>(w + at)) : make_float2(1.f, 1.f);
        bb[v] = b != nullptr && act ? __ldg(reinterpret_cast<const float2*>(b + at)) : make_float2(0.f, 0.f);
      }
    }
    // the lane's first value of head begin * HPW + sub; a turn further is `ahead` bytes on
    const int d01 = (d1 - d0) * 2;
    const int h0 = begin * HPW + sub;
    const char* src = reinterpret_cast<const char*>(static_cast<const T*>(in.p) + t * in.st + h0 * in.sh + d0);
    char* dst = reinterpret_cast<char*>(static_cast<T*>(out.p) + t * out.st + h0 * out.sh + d0);
    const long long src_ahead = 2ll * HPW * in.sh, dst_ahead = 2ll * HPW * out.sh;
    // turns in which this lane has a head
    const int mine = act ? min(end - begin, (heads - h0 + HPW - 1) / HPW) : 0;
    uint2 raw[kBatch][2];
    auto load = [&](int i, int k) {
      raw[i][0] = raw[i][1] = make_uint2(0u, 0u);
      if (k < mine) {
        raw[i][0] = *reinterpret_cast<const uint2*>(src);
        raw[i][1] = *reinterpret_cast<const uint2*>(src + d01);
      }
      src += src_ahead;
    };
    auto load_batch = [&](int k0) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) load(i, k0 + i);
    };
    if (kAhead) load_batch(0);
    for (int k0 = 0; k0 < end - begin; k0 += kBatch) {
      if (!kAhead) load_batch(k0);
#pragma unroll
      for (int g = 0; g < kBatch; g += kJoin) {
        if (k0 + g >= end - begin) break;
        // the sums of kJoin turns side by side: one after the other, a warp mostly waits for shuffles
        float mean[kJoin], r[kJoin];
        auto values = [&](int i, float2 (&y)[4]) {  // of turn g + i
          const uint2 a = raw[g + i][0], b = raw[g + i][1];
          y[0] = unpack2(a.x, T());
          y[1] = unpack2(a.y, T());
          y[2] = unpack2(b.x, T());
          y[3] = unpack2(b.y, T());
        };
        auto centre = [&](int i, float2 (&y)[4]) {
          if (NORM == kLayer) {
            const float m = act ? mean[i] : 0.f;
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = __fadd2_rn(y[v], make_float2(m, m));
          }
        };
        float2 y[4];
        if (NORM == kLayer) {
#pragma unroll
          for (int i = 0; i < kJoin; ++i) {
            values(i, y);
            const float2 s = __fadd2_rn(__fadd2_rn(y[0], y[1]), __fadd2_rn(y[2], y[3]));
            mean[i] = s.x + s.y;
          }
          head_sums<LPH>(mean);
#pragma unroll
          for (int i = 0; i < kJoin; ++i) mean[i] *= -p.inv_d;
        }
        if (NORM != kNone) {
#pragma unroll
          for (int i = 0; i < kJoin; ++i) {
            values(i, y);
            centre(i, y);
            float2 s2 = __fmul2_rn(y[0], y[0]);
#pragma unroll
            for (int v = 1; v < 4; ++v) s2 = __ffma2_rn(y[v], y[v], s2);
            r[i] = s2.x + s2.y;
          }
          head_sums<LPH>(r);
#pragma unroll
          for (int i = 0; i < kJoin; ++i) r[i] = rsqrt_near(fmaf(r[i], p.inv_d, p.eps));
        }
#pragma unroll
        for (int i = 0; i < kJoin; ++i) {
          values(i, y);
          centre(i, y);
          if (NORM != kNone) {
#pragma unroll
            for (int v = 0; v < 4; ++v) y[v] = __ffma2_rn(__fmul2_rn(y[v], make_float2(r[i], r[i])), ww[v], bb[v]);
          }
          if (turned) {
            if (INTER) {
#pragma unroll
              for (int v = 0; v < 4; ++v)
                y[v] = make_float2(y[v].x * cs[v] - y[v].y * sn[v], y[v].y * cs[v] + y[v].x * sn[v]);
            } else {
#pragma unroll
              for (int v = 0; v < 2; ++v) {
                const float2 cc = make_float2(cs[2 * v], cs[2 * v + 1]), ss = make_float2(sn[2 * v], sn[2 * v + 1]);
                const float2 a = y[v], o = y[v + 2];
                y[v] = __ffma2_rn(a, cc, __fmul2_rn(o, make_float2(ns[2 * v], ns[2 * v + 1])));
                y[v + 2] = __ffma2_rn(o, cc, __fmul2_rn(a, ss));
              }
            }
          }
          if (k0 + g + i < mine) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(y[0].x, y[0].y, T()), pack2(y[1].x, y[1].y, T()));
            *reinterpret_cast<uint2*>(dst + d01) = make_uint2(pack2(y[2].x, y[2].y, T()), pack2(y[3].x, y[3].y, T()));
          }
          dst += dst_ahead;
          if (kAhead) load(g + i, k0 + kBatch + g + i);
        }
      }
    }
  };
  run(p.q, p.qo, p.hq, first, min(last, p.q_turns), p.qw, p.qb);
  run(p.k, p.ko, p.hk, max(first, p.q_turns) - p.q_turns, last - p.q_turns, p.kw, p.kb);
  griddep_trigger();
}

}  // namespace k8
}  // namespace tmu

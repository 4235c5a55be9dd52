// K9: linear layer with 8-bit (e4m3) operands and a scale for each block of 128 values.
//
//   out[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} x8[m, k] w8[n, k]  (+ bias[n])
//
// x8 [M, K] with one scale a row and block of 128 along K, w8 [N, K] with one scale a 128 x 128
// block.  quantize_kernel makes x8, xs from a 16-bit x: xs = max(amax / 448, 2^-126) (448 is
// e4m3's largest value) and x8 = e4m3(x / xs), both quotients rounded as IEEE fp32 divisions.
//
// Few rows (linear8_rows_kernel): bound by reading w8 once.  Many rows (linear8_kernel): tcgen05
// kind::f8f6f4 products of one block of 128 at a time into TMEM, scaled and summed in registers.
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
  int chained;  // the outputs are a workspace that only the next kernel of the same call reads
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

// 8 values a lane, 16 lanes a block of 128 (all of the warp takes part): the block's scale and the lane's e4m3.
template <typename T>
__device__ __forceinline__ void quantize8(const uint32_t (&u)[4], float& s, uint2& o) {
  float y[8], amax = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = k8::unpack2(u[e], T());
    y[2 * e] = f.x;
    y[2 * e + 1] = f.y;
    amax = max_nan(amax, max_nan(fabsf(f.x), fabsf(f.y)));
  }
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  s = max_nan(__fdiv_rn(amax, 448.f), 0x1p-126f);
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = e4m3x2(__fdiv_rn(y[2 * e], s), __fdiv_rn(y[2 * e + 1], s));
  o = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
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
    uint2 o;
    float s;
    quantize8<T>(u, s, o);
    if (on) *reinterpret_cast<uint2*>(p.x8 + m * p.K + k) = o;
    if (it < items && l == 0) p.xs[m * p.kb + b] = s;
  }
  // linear8_rows_kernel reads w8 before its dependency wait, so nothing that could be a weight may
  // be announced before it is visible
  if (p.chained) griddep_trigger();
}

enum Out : int { kF16 = 0, kBf16 = 1, kF32 = 2 };

__device__ __forceinline__ void store_out(void* out, int type, long long at, float v) {
  if (type == kF16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else if (type == kBf16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<float*>(out)[at] = v;
}

// ------------------------------------------------------------------------------------------
// Few rows.  A block takes 16 rows of w8 (the MMA's M) and up to 8 * G rows of x (its N, 8 a
// group): mma.sync m16n8k32 on e4m3, so a weight byte is used as loaded.  The K order inside a
// 64-byte chunk is free as long as both operands share it: lane t of a row's four takes the 16
// bytes at 16 t, which are its fragments of two MMAs.  Warp w takes the blocks of 128 b = w, w + 8,
// ...: it quantises their part of x itself (so a call is one launch and the weights are already
// on their way meanwhile), scales each block's sums, and the eight warps' sums are added in order
// at the end.
// ------------------------------------------------------------------------------------------
struct RowsParams {
  const void* x;      // 16-bit [M, K] (rows ldx apart), or e4m3 [M, K] with xs
  long long ldx;
  const float* xs;
  const uint8_t* w8;
  const float* ws;
  const float* bias;
  void* out;
  long long ldo;
  int M, N, K, kb, out_type;
};

constexpr int kRowsThreads = 256, kRowsN = 16;
constexpr int kRowsMax = 16;  // rows of x
constexpr int kXPitch = 144;  // bytes of a staged x row: rows of a group start 4 banks apart

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_once(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// X: __half or __nv_bfloat16 (quantised here), or uint8_t (e4m3 already).
template <typename X, int G>
__global__ void __launch_bounds__(kRowsThreads) linear8_rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int kWarps = kRowsThreads / 32;
  __shared__ __align__(16) uint8_t xq[kWarps][8 * G][kXPitch];
  __shared__ float xsc[kWarps][8 * G];
  __shared__ float part[kWarps][8 * G][kRowsN + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kRowsN;
  const uint8_t* w[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int n = n0 + g + 8 * r;
    w[r] = n < p.N ? p.w8 + static_cast<long long>(n) * p.K : nullptr;
  }
  auto load_w = [&](int b, uint4 (&v)[2][2]) {  // [row half][64-byte chunk]
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = b * 128 + c * 64 + t * 16;
        v[r][c] = w[r] != nullptr && k < p.K ? load_once(w[r] + k) : make_uint4(0u, 0u, 0u, 0u);
      }
  };
  uint4 cur[2][2];
  load_w(warp, cur);  // no kernel that starts its successor early writes a weight, so this need not wait
  griddep_wait();
  float total[G][4];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) total[i][e] = 0.f;
  for (int b = warp; b < p.kb; b += kWarps) {
    uint4 next[2][2];
    load_w(b + kWarps, next);
    // this block of x, two rows at a time: 16 lanes of 8 values a row
    const int l = lane & 15, k = b * 128 + l * 8;
    __syncwarp();
    for (int m = lane >> 4; m < 8 * G; m += 2) {
      uint2 o = make_uint2(0u, 0u);
      float s = 0.f;
      const bool on = m < p.M && k < p.K;
      if constexpr (sizeof(X) == 1) {
        if (on) o = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.x) + m * p.ldx + k);
        if (m < p.M) s = __ldg(p.xs + static_cast<long long>(m) * p.kb + b);
      } else {
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (on) raw = *reinterpret_cast<const uint4*>(static_cast<const X*>(p.x) + m * p.ldx + k);
        const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
        quantize8<X>(u, s, o);
      }
      *reinterpret_cast<uint2*>(&xq[warp][m][l * 8]) = o;
      if (l == 0) xsc[warp][m] = s;
    }
    __syncwarp();
    const float ws = __ldg(p.ws + static_cast<long long>(n0 >> 7) * p.kb + b);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint4 x = *reinterpret_cast<const uint4*>(&xq[warp][i * 8 + g][c * 64 + t * 16]);
        mma_e4m3(d, cur[0][c].x, cur[1][c].x, cur[0][c].y, cur[1][c].y, x.x, x.y);
        mma_e4m3(d, cur[0][c].z, cur[1][c].z, cur[0][c].w, cur[1][c].w, x.z, x.w);
      }
      const float s0 = ws * xsc[warp][i * 8 + 2 * t], s1 = ws * xsc[warp][i * 8 + 2 * t + 1];
      total[i][0] = fmaf(d[0], s0, total[i][0]);
      total[i][1] = fmaf(d[1], s1, total[i][1]);
      total[i][2] = fmaf(d[2], s0, total[i][2]);
      total[i][3] = fmaf(d[3], s1, total[i][3]);
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) cur[r][c] = next[r][c];
  }
#pragma unroll
  for (int i = 0; i < G; ++i) {
    part[warp][i * 8 + 2 * t][g] = total[i][0];
    part[warp][i * 8 + 2 * t + 1][g] = total[i][1];
    part[warp][i * 8 + 2 * t][g + 8] = total[i][2];
    part[warp][i * 8 + 2 * t + 1][g + 8] = total[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * G * kRowsN; i += kRowsThreads) {
    const int m = i / kRowsN, n = n0 + i % kRowsN;
    if (m >= p.M || n >= p.N) continue;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) s += part[v][m][i % kRowsN];
    store_out(p.out, p.out_type, m * p.ldo + n, s + (p.bias ? __ldg(p.bias + n) : 0.f));
  }
  griddep_trigger();
}

// ------------------------------------------------------------------------------------------
// Many rows.  A block takes 128 rows of x (TMEM lanes) and 128 of w8 (TMEM columns), whose block
// of 128 has one scale: a thread holds one row's sums of 64 columns, and a step adds
// xs[row, b] * ws[b] times the step's products, read from one of four TMEM slots.
//   warp 0      TMA: x8 and w8 through a ring of kStages steps
//   warp 1      TMEM and the MMAs (four of K = 32 a step)
//   warps 2-3   idle
//   warps 4-11  sums: two warps a TMEM lane quadrant, each on half of the columns
// Few tiles: a cluster of blocks shares one tile along K.  Each leaves its sums in shared memory
// and adds its share of the columns over the cluster's blocks, in rank order.
// ------------------------------------------------------------------------------------------
constexpr int kTile = 128;
constexpr int kStages = 5;
constexpr int kSlots = 4;
constexpr int kThreads = 384;
constexpr int kOperand = kTile * 128;
constexpr int OFF_A = 0;
constexpr int OFF_B = kStages * kOperand;
constexpr int OFF_BAR = 2 * kStages * kOperand;
constexpr int SMEM_BYTES = OFF_BAR + 256;
constexpr int kSumPitch = kTile + 4;  // floats of a row of sums in shared memory (over the ring)
static_assert(SMEM_BYTES <= 232448 && kTile * kSumPitch * 4 <= OFF_BAR, "K9 shared memory");

struct Params {
  CUtensorMap tm_x, tm_w;  // [rows, K] bytes: box {128, 128}, 128B swizzle, zero past the ends
  const float* xs;
  const float* ws;
  const float* bias;
  void* out;
  long long ldo;
  int M, N, kb, out_type, vec;  // vec: rows of out take 16-byte stores
  int tiles_m, split;           // blocks of a cluster share a tile along K
  DeviceStatus* status;
  unsigned long long timeout_ns;
};

enum Site : unsigned int { kSiteProd = 0x901, kSiteMma = 0x902, kSiteSlot = 0x903, kSiteSum = 0x904, kSiteLayout = 0x9ff };

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of kind::f8f6f4 with e4m3 operands (format 0), K-major, fp32 sums.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) { return idesc_f16_f32(M, N, false, false); }

// 16 sums of row m from column n on, with the bias, to the output.
__device__ __forceinline__ void store16(const Params& p, int m, int n, const float (&v)[16]) {
  float y[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e] = v[e] + (p.bias != nullptr && n + e < p.N ? __ldg(p.bias + n + e) : 0.f);
  const long long at = static_cast<long long>(m) * p.ldo + n;
  if (p.vec && n + 16 <= p.N) {
    if (p.out_type == kF32) {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[e] = make_float4(y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
    } else {
      uint32_t u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        u[e] = p.out_type == kF16 ? k8::pack2(y[2 * e], y[2 * e + 1], __half()) : k8::pack2(y[2 * e], y[2 * e + 1], __nv_bfloat16());
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at);
      dst[0] = make_uint4(u[0], u[1], u[2], u[3]);
      dst[1] = make_uint4(u[4], u[5], u[6], u[7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (n + e < p.N) store_out(p.out, p.out_type, at + e, y[e]);
  }
}

__global__ void __launch_bounds__(kThreads, 1) linear8_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem[];
  DeviceStatus* const status = p.status != nullptr ? p.status : &g_own_status;
  const bool laid = (smem_u32(smem) & 1023) == 0;  // uniform over the grid
  if (!laid) {
    if (threadIdx.x == 0) record_status(status, kStatusLayout, kSiteLayout);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  uint64_t* full = bars;                      // [kStages]
  uint64_t* empty = bars + kStages;           // [kStages]
  uint64_t* sfull = bars + 2 * kStages;       // [kSlots] a step's products are in the slot
  uint64_t* sempty = sfull + kSlots;          // [kSlots] its eight readers have them
  uint64_t& drain_bar = sempty[kSlots];
  uint32_t& tmem_base_sh = *reinterpret_cast<uint32_t*>(&drain_bar + 1);
  volatile int& abort_sh = *reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(&drain_bar + 1) + 4);
  const WaitCtx ctx{status, &abort_sh, p.timeout_ns};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.split, tile = static_cast<int>(blockIdx.x) / p.split;
  const int m0 = tile % p.tiles_m * kTile, n0 = tile / p.tiles_m * kTile;
  const int b0 = static_cast<int>(static_cast<long long>(p.kb) * rank / p.split);
  const int b1 = static_cast<int>(static_cast<long long>(p.kb) * (rank + 1) / p.split);
  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&sfull[s], 1);
      mbar_init(&sempty[s], 8);
    }
    mbar_init(&drain_bar, 1);
    fence_mbar_init();
    tma_prefetch_desc(&p.tm_x);
    tma_prefetch_desc(&p.tm_w);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  griddep_trigger();
  griddep_wait();

  float sum[64];
  if (warp == 0) {
    if (lane == 0) {
      int i = 0;
      for (int b = b0; b < b1; ++b, ++i) {
        const int s = i % kStages;
        if (!mbar_wait(&empty[s], ((i / kStages) & 1) ^ 1, ctx, kSiteProd)) break;
        mbar_arrive_expect_tx(&full[s], 2 * kOperand);
        tma_load_2d(smem + OFF_A + s * kOperand, &p.tm_x, &full[s], b * 128, m0);
        tma_load_2d(smem + OFF_B + s * kOperand, &p.tm_w, &full[s], b * 128, n0);
      }
      if (abort_sh)
        for (int s = 0; s < kStages; ++s) {
          const int armed = i > s ? (i - s + kStages - 1) / kStages : 0;
          if (armed) mbar_drain(&full[s], (armed - 1) & 1, 200000000ull);
        }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_e4m3_f32(kTile, kTile);
      const uint64_t ad = sdesc_sw128(smem_u32(smem + OFF_A), 16, 1024), bd = sdesc_sw128(smem_u32(smem + OFF_B), 16, 1024);
      for (int i = 0; i < b1 - b0; ++i) {
        const int s = i % kStages, c = i % kSlots;
        if (!mbar_wait(&sempty[c], ((i / kSlots) & 1) ^ 1, ctx, kSiteSlot)) break;
        if (!mbar_wait(&full[s], (i / kStages) & 1, ctx, kSiteMma)) break;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f8(tmem + c * kTile, sdesc_add(ad, s * kOperand + k * 32), sdesc_add(bd, s * kOperand + k * 32), idesc,
                  k > 0 ? 1u : 0u);
        umma_commit(&empty[s]);
        umma_commit(&sfull[c]);
      }
      umma_commit(&drain_bar);
      mbar_drain(&drain_bar, 0, 200000000ull);
    }
  } else if (warp >= 4) {
    const int q = warp & 3, half = (warp - 4) >> 2;
    const int m = m0 + q * 32 + lane;
    const uint32_t tl = tmem + (static_cast<uint32_t>(q * 32) << 16) + half * 64;
    const float* xs = p.xs + static_cast<long long>(min(m, p.M - 1)) * p.kb;
    const float* ws = p.ws + static_cast<long long>(n0 >> 7) * p.kb;
#pragma unroll
    for (int e = 0; e < 64; ++e) sum[e] = 0.f;
    float sc = b0 < b1 ? __ldg(xs + b0) * __ldg(ws + b0) : 0.f;
    for (int b = b0; b < b1; ++b) {
      const int i = b - b0, c = i % kSlots;
      const float next = b + 1 < b1 ? __ldg(xs + b + 1) * __ldg(ws + b + 1) : 0.f;
      if (!warp_wait(&sfull[c], (i / kSlots) & 1, ctx, kSiteSum)) break;
      tc_fence_after();
      uint32_t r[2][32];
      tmem_ld32(tl + c * kTile, r[0]);
      tmem_ld32(tl + c * kTile + 32, r[1]);
      tmem_wait_ld2(r[0], r[1]);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sempty[c]);
      const float2 s2 = make_float2(sc, sc);
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float2 v = make_float2(__uint_as_float(r[e >> 4][(2 * e) & 31]), __uint_as_float(r[e >> 4][(2 * e + 1) & 31]));
        const float2 a = __ffma2_rn(v, s2, make_float2(sum[2 * e], sum[2 * e + 1]));
        sum[2 * e] = a.x;
        sum[2 * e + 1] = a.y;
      }
      sc = next;
    }
    if (p.split == 1 && m < p.M)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v[16];
#pragma unroll
        for (int f = 0; f < 16; ++f) v[f] = sum[e * 16 + f];
        store16(p, m, n0 + half * 64 + e * 16, v);
      }
  }

  if (p.split > 1) {
    // the ring's last reads are done: a block's sums replace its operands
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    if (warp >= 4) {
      const int row = (warp & 3) * 32 + lane, c0 = ((warp - 4) >> 2) * 64;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        *reinterpret_cast<float4*>(sums + row * kSumPitch + c0 + 4 * e) = make_float4(sum[4 * e], sum[4 * e + 1], sum[4 * e + 2], sum[4 * e + 3]);
    }
    cluster_sync_all();
    // share r of the tile: groups of 16 columns of a row, dealt over the cluster's threads
    for (int i = rank * kThreads + threadIdx.x; i < kTile * 8; i += p.split * kThreads) {
      const int row = i >> 3, c = (i & 7) * 16;
      if (m0 + row >= p.M) continue;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
      for (int r = 0; r < p.split; ++r) {
        const uint32_t src = cluster_addr(sums + row * kSumPitch + c, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float4 f;
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                       : "r"(src + e * 16)
                       : "memory");
          v[4 * e] += f.x;
          v[4 * e + 1] += f.y;
          v[4 * e + 2] += f.z;
          v[4 * e + 3] += f.w;
        }
      }
      store16(p, m0 + row, n0 + c, v);
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are being read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace k9
}  // namespace tmu

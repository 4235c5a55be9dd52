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

constexpr int kQuantThreads = 256, kQuantRows = kQuantThreads / 8;

struct QuantParams {
  const void* x;
  long long ld;
  int M, K, kb;
  uint8_t* x8;  // [M, K]
  float* xs;    // scale of row m and block b at m * xs_m + b * xs_b
  long long xs_m, xs_b;
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

__device__ __forceinline__ uint32_t absmax2(uint32_t a, uint32_t b, __half) {  // of two pairs, keeps a NaN
  const __half2 r = __hmax2_nan(__habs2(*reinterpret_cast<__half2*>(&a)), __habs2(*reinterpret_cast<__half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t absmax2(uint32_t a, uint32_t b, __nv_bfloat16) {
  const __nv_bfloat162 r =
      __hmax2_nan(__habs2(*reinterpret_cast<__nv_bfloat162*>(&a)), __habs2(*reinterpret_cast<__nv_bfloat162*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// C runs of 8 values a lane, 16 / C lanes a block of 128 (all of the warp takes part): the block's
// scale and the lane's e4m3.  A quotient a / b is rounded correctly from the correctly rounded r = 1 / b: q = a r, then
// q + (a - q b) r with fused multiply-adds (Markstein 1990; right but for divisors whose significand
// is all ones: 448 = 7 * 2^6 is none, nor is an 8 or 11-bit number over it, whose 24 bits repeat
// with the period 3 of sevenths).  The remainder must not underflow, which the scale's lower limit
// sees to for itself (a quotient below 2^-126 is replaced) and a power of two for the values.
template <typename T, int C>
__device__ __forceinline__ void quantize(const uint4 (&raw)[C], float& s, uint2 (&o)[C]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < C; ++i) m = absmax2(m, absmax2(absmax2(raw[i].x, raw[i].y, T()), absmax2(raw[i].z, raw[i].w, T()), T()), T());
#pragma unroll
  for (int d = 8 / C; d > 0; d >>= 1) m = absmax2(m, __shfl_xor_sync(0xffffffffu, m, d), T());
  const float2 pair = k8::unpack2(m, T());
  const float amax = max_nan(pair.x, pair.y);
  constexpr float r448 = 1.f / 448.f;
  const float q0 = amax * r448;
  s = max_nan(amax < INFINITY ? fmaf(fmaf(-q0, 448.f, amax), r448, q0) : amax, 0x1p-126f);
  const float up = s < 0x1p-60f ? 0x1p66f : 1.f;
  const float t = s * up, r = __frcp_rn(t);
  const float2 r2 = make_float2(r, r), nt2 = make_float2(-t, -t);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 a = k8::unpack2(u[e], T());
      if (up != 1.f) a = make_float2(a.x * up, a.y * up);
      const float2 q = __fmul2_rn(a, r2);
      const float2 v = __ffma2_rn(__ffma2_rn(q, nt2, a), r2, q);
      w[e] = e4m3x2(v.x, v.y);
    }
    o[i] = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
  }
}

// Eight lanes take U blocks of 128 of one row (16 values a lane and block), all loaded before the
// first is worked on, and a block of threads 32 rows, so that the scales of a block of 128, transposed
// for the tensor-core kernels, are written 128 bytes at a time.
// Bound: HBM, 2 bytes read and 1 written a value: 82 us at 16384 x 10240, 6.2 TB/s.  (With 16 lanes a
// block, and so twice the scales' arithmetic, the instructions bound it: 97 us, 84 % of the issue slots.)
template <typename T, int U>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(const __grid_constant__ QuantParams p) {
  const int l = threadIdx.x & 7;
  const int per = (p.kb + U - 1) / U;
  const int rows = blockIdx.x / per;
  const int m = rows * kQuantRows + (threadIdx.x >> 3), b0 = (blockIdx.x - rows * per) * U;
  griddep_wait();
  uint4 raw[U][2];
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int k = (b0 + i) * 128 + c * 64 + l * 8;
      raw[i][c] = make_uint4(0u, 0u, 0u, 0u);
      if (m < p.M && k < p.K) raw[i][c] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + m * p.ld + k);
    }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    uint2 o[2];
    float s;
    quantize<T, 2>(raw[i], s, o);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int k = (b0 + i) * 128 + c * 64 + l * 8;
      if (m < p.M && k < p.K) *reinterpret_cast<uint2*>(p.x8 + static_cast<long long>(m) * p.K + k) = o[c];
    }
    if (m < p.M && b0 + i < p.kb && l == 0) p.xs[m * p.xs_m + (b0 + i) * p.xs_b] = s;
  }
  // (Announced at the start, the products' blocks come while these still run, two on some SMs and none
  // on others: 13.4 -> 16 us at 1283 x 1000 x 1360.)
  griddep_trigger();
}

// Row-major scales [M, kb] to [kb, ld], for the tensor-core kernels.
struct ScaleParams {
  const float* xs;
  float* xst;
  int M, kb, ld;
};
__global__ void __launch_bounds__(256) transpose_scales_kernel(const __grid_constant__ ScaleParams p) {
  griddep_wait();
  const int m = blockIdx.x * 256 + threadIdx.x;
  if (m < p.M)
    for (int b = 0; b < p.kb; ++b) p.xst[static_cast<long long>(b) * p.ld + m] = p.xs[static_cast<long long>(m) * p.kb + b];
  griddep_trigger();
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

// X: __half or __nv_bfloat16 (quantised here), or uint8_t (e4m3 already).  PAIRS: row pairs of x, M <= 2 * PAIRS.
template <typename X, int PAIRS>
__global__ void __launch_bounds__(kRowsThreads, PAIRS == 1 ? 4 : PAIRS == 4 ? 3 : 2) linear8_rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int kWarps = kRowsThreads / 32, G = PAIRS > 4 ? 2 : 1;
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
  // row 2 i + lane / 16 of x, 16 lanes of 8 values a row
  const int l = lane & 15;
  auto load_x = [&](int b, uint4 (&v)[PAIRS], float (&s)[PAIRS]) {
    const int k = b * 128 + l * 8;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const int m = 2 * i + (lane >> 4);
      const bool on = m < p.M && k < p.K;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (sizeof(X) == 1) {
        if (on) {
          const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.x) + m * p.ldx + k);
          v[i].x = u.x;
          v[i].y = u.y;
          s[i] = p.xs[static_cast<long long>(m) * p.kb + b];
        }
      } else {
        if (on) v[i] = *reinterpret_cast<const uint4*>(static_cast<const X*>(p.x) + m * p.ldx + k);
      }
    }
  };
  uint4 cur[2][2], xcur[PAIRS];
  float scur[PAIRS];
  griddep_wait();  // w8 too may be what the kernel in front of this one writes
  load_w(warp, cur);
  load_x(warp, xcur, scur);
  float total[G][4];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) total[i][e] = 0.f;
  for (int b = warp; b < p.kb; b += kWarps) {
    uint4 next[2][2], xnext[PAIRS];
    float snext[PAIRS];
    load_w(b + kWarps, next);
    load_x(b + kWarps, xnext, snext);
    __syncwarp();
    // (rows past M are staged as they come: a column of products depends on its own row only)
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      if (2 * i >= p.M) break;
      uint2 o[1] = {make_uint2(xcur[i].x, xcur[i].y)};
      float s = scur[i];
      if constexpr (sizeof(X) != 1) {
        const uint4 raw[1] = {xcur[i]};
        quantize<X, 1>(raw, s, o);
      }
      *reinterpret_cast<uint2*>(&xq[warp][2 * i + (lane >> 4)][l * 8]) = o[0];
      if (l == 0) xsc[warp][2 * i + (lane >> 4)] = s;
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
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      xcur[i] = xnext[i];
      scur[i] = snext[i];
    }
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
// xs[row, b] * ws[b] times the step's products, read from one of two TMEM slots.
//   warps 0-7   sums: two warps a TMEM lane quadrant, each on half of the columns
//   warp 8      TMA: x8 and w8 through a ring of kStages steps
//   warp 9      TMEM and the MMAs (four of K = 32 a step)
// Two blocks an SM, so one's start and end and its waits fall into the other's work.
// The scales of a step's rows are read transposed, 32 rows in one access of a warp, and by
// cp.async, four steps ahead: a lane later reads the value that it copied itself.  (Read as they lie,
// a sector a row, they cost as much L2 traffic as half the operands; handed on from register to
// register each step, the move waited for the load: 800 of a step's 1550 cycles.)
// Few tiles: a cluster of blocks shares one tile along K.  Each leaves its sums in shared memory
// and adds its share of the columns over the cluster's blocks, in rank order.
// ------------------------------------------------------------------------------------------
constexpr int kTile = 128;
constexpr int kStages = 3;
constexpr int kSlots = 2;
constexpr int kThreads = 320;
constexpr int kOperand = kTile * 128;
constexpr int OFF_A = 0;
constexpr int OFF_B = kStages * kOperand;
constexpr int OFF_XS = 2 * kStages * kOperand;  // the warps' rings of scales
constexpr int OFF_BAR = OFF_XS + 8 * 4 * 128;
constexpr int SMEM_BYTES = OFF_BAR + 256;
constexpr int kOutPitch = 80, kOutBytes = 32 * kOutPitch;  // a warp's staged rows of the output
constexpr int kMaxSplit = 8;        // blocks of a cluster
constexpr int kSumPitch = kTile + 4;  // floats of a row of sums in shared memory (over the ring)
static_assert(2 * (SMEM_BYTES + 1024) <= 233472 && kTile * kSumPitch * 4 <= OFF_BAR && 8 * kOutBytes <= OFF_BAR, "K9 shared memory");

struct Params {
  CUtensorMap tm_x, tm_w;  // [rows, K] bytes: box {128, 128}, 128B swizzle, zero past the ends
  const float* xst;  // [kb, ld_xs]: x's scales, rows of x fastest, ld_xs M rounded up to 256
  const float* ws;
  const float* bias;
  void* out;
  long long ldo;
  int ld_xs;
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

// The scales of a warp's 32 rows on their way to shared memory, kScaleAhead steps ahead.
constexpr int kScaleAhead = 4;

struct ScaleRing {
  const float* xs;  // this lane's row, block 0
  long long ld;
  uint32_t slot;    // this lane's word of the warp's kScaleAhead x 32
  int end;
  __device__ __forceinline__ void fetch(int b, int i) const {  // the scale of block b, for step i
    if (b < end)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot + (i % kScaleAhead) * 128),
                   "l"(xs + static_cast<long long>(b) * ld)
                   : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ float get(int i) const {  // of step i, fetched kScaleAhead steps ago
    asm volatile("cp.async.wait_group %0;" ::"n"(kScaleAhead - 1) : "memory");
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(slot + (i % kScaleAhead) * 128) : "memory");
    return v;
  }
};

// Instruction descriptor of kind::f8f6f4 with e4m3 operands (format 0), K-major, fp32 sums.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) { return idesc_f16_f32(M, N, false, false); }

// A warp's sums to the output: lane = row m0 + lane, 64 columns from n0 on, with the bias.  64 bytes of
// each row at a time go through shared memory (rows 80 bytes apart, so eight lanes' 16-byte accesses
// meet 8 different bank groups), from where four lanes write a row's 16-byte pieces, or, with
// unaligned rows of out, 32 lanes its single values: written straight from the lane of the row, an unaligned
// output took 32 us at 1283 x 1000 x 1360, most of it in its 2-byte stores.
__device__ __forceinline__ void store_rows(const Params& p, uint8_t* buf, int m0, int n0, const float (&sum)[64]) {
  const int lane = threadIdx.x & 31;
  float b0 = 0.f, b1 = 0.f;  // bias of columns n0 + lane, n0 + 32 + lane
  if (p.bias != nullptr) {
    if (n0 + lane < p.N) b0 = __ldg(p.bias + n0 + lane);
    if (n0 + 32 + lane < p.N) b1 = __ldg(p.bias + n0 + 32 + lane);
  }
  const bool wide = p.out_type == kF32;
  const int es = wide ? 4 : 2, cols = 64 / es;  // columns of a pass
#pragma unroll
  for (int g = 0; g < 4; ++g) {  // 16 columns a step
    float y[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = sum[g * 16 + e] + __shfl_sync(0xffffffffu, g < 2 ? b0 : b1, (g & 1) * 16 + e);
    uint4* row = reinterpret_cast<uint4*>(buf + lane * kOutPitch);
    if (wide) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        row[e] = make_uint4(__float_as_uint(y[4 * e]), __float_as_uint(y[4 * e + 1]), __float_as_uint(y[4 * e + 2]),
                            __float_as_uint(y[4 * e + 3]));
    } else {
      uint32_t u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        u[e] = p.out_type == kF16 ? k8::pack2(y[2 * e], y[2 * e + 1], __half()) : k8::pack2(y[2 * e], y[2 * e + 1], __nv_bfloat16());
      row[(g & 1) * 2] = make_uint4(u[0], u[1], u[2], u[3]);
      row[(g & 1) * 2 + 1] = make_uint4(u[4], u[5], u[6], u[7]);
      if (!(g & 1)) continue;
    }
    const int c0 = n0 + (wide ? g * 16 : (g >> 1) * 32);
    __syncwarp();
    if (p.vec && c0 + cols <= p.N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2), c = lane & 3;
        if (m0 + r < p.M)
          *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + ((m0 + r) * p.ldo + c0) * es + c * 16) =
              *reinterpret_cast<const uint4*>(buf + r * kOutPitch + c * 16);
      }
    } else {
      for (int i = lane; i < 32 * cols; i += 32) {
        const int r = i / cols, c = i - r * cols;
        if (m0 + r >= p.M || c0 + c >= p.N) continue;
        const long long at = (m0 + r) * p.ldo + c0 + c;
        if (wide) static_cast<float*>(p.out)[at] = *reinterpret_cast<const float*>(buf + r * kOutPitch + c * 4);
        else static_cast<uint16_t*>(p.out)[at] = *reinterpret_cast<const uint16_t*>(buf + r * kOutPitch + c * 2);
      }
    }
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kThreads, 2) linear8_kernel(const __grid_constant__ Params p) {
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
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
  if (warp == 9) {
    tmem_alloc(&tmem_base_sh, kSlots * kTile);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  griddep_trigger();
  griddep_wait();

  float sum[64];
  if (warp == 8) {
    const bool leader = elect_one();
    int s = 0, ph = 0, i = 0;
    bool ok = true;
    for (int b = b0; b < b1; ++b, ++i) {
      if (!(ok = warp_poll(&empty[s], ph ^ 1, ctx, kSiteProd))) break;
      if (leader) {
        mbar_arrive_expect_tx(&full[s], 2 * kOperand);
        tma_load_2d(smem + OFF_A + s * kOperand, &p.tm_x, &full[s], b * 128, m0);
        tma_load_2d(smem + OFF_B + s * kOperand, &p.tm_w, &full[s], b * 128, n0);
      }
      __syncwarp();
      if (++s == kStages) {
        s = 0;
        ph ^= 1;
      }
    }
    if (!ok && leader)
      for (int r = 0; r < kStages; ++r) {
        const int armed = i > r ? (i - r + kStages - 1) / kStages : 0;
        if (armed) mbar_drain(&full[r], (armed - 1) & 1, 200000000ull);
      }
    __syncwarp();
  } else if (warp == 9) {
    const bool leader = elect_one();
    const uint32_t idesc = idesc_e4m3_f32(kTile, kTile);
    const uint64_t ad = sdesc_sw128(smem_u32(smem + OFF_A), 16, 1024), bd = sdesc_sw128(smem_u32(smem + OFF_B), 16, 1024);
    int s = 0, ph = 0;
    for (int i = 0; i < b1 - b0; ++i) {
      const int c = i % kSlots;
      if (!warp_poll(&full[s], ph, ctx, kSiteMma)) break;
      if (!warp_poll(&sempty[c], ((i / kSlots) & 1) ^ 1, ctx, kSiteSlot)) break;
      tc_fence_after();
      const uint64_t as = sdesc_add(ad, s * kOperand), bs = sdesc_add(bd, s * kOperand);
      const uint32_t d = tmem + c * kTile;
      if (leader) {
        umma_f8(d, as, bs, idesc, 0u);
        umma_f8(d, sdesc_add(as, 32), sdesc_add(bs, 32), idesc, 1u);
        umma_f8(d, sdesc_add(as, 64), sdesc_add(bs, 64), idesc, 1u);
        umma_f8(d, sdesc_add(as, 96), sdesc_add(bs, 96), idesc, 1u);
        umma_commit(&sfull[c]);
        umma_commit(&empty[s]);
      }
      __syncwarp();
      if (++s == kStages) {
        s = 0;
        ph ^= 1;
      }
    }
    if (leader) {
      umma_commit(&drain_bar);
      mbar_drain(&drain_bar, 0, 200000000ull);
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = warp >> 2;
    const uint32_t tl = tmem + (static_cast<uint32_t>(q * 32) << 16) + half * 64;
    const float* ws = p.ws + static_cast<long long>(n0 >> 7) * p.kb;
    const float* xs = p.xst + m0 + q * 32 + lane;
#pragma unroll
    for (int e = 0; e < 64; ++e) sum[e] = 0.f;
    // the weight's scales: lane j holds that of step 32 i + j, and of the next 32 steps
    auto load_ws = [&](int b) { return b + lane < b1 ? __ldg(ws + b + lane) : 0.f; };
    float w0 = load_ws(b0), w1 = load_ws(b0 + 32);
    const ScaleRing ring{xs, p.ld_xs, smem_u32(smem + OFF_XS + warp * (kScaleAhead * 128)) + lane * 4, b1};
    for (int u = 0; u < kScaleAhead; ++u) ring.fetch(b0 + u, u);
    for (int b = b0; b < b1; ++b) {
      const int i = b - b0, c = i % kSlots;
      if (i > 0 && (i & 31) == 0) {
        w0 = w1;
        w1 = load_ws(b + 32);
      }
      const float sc = __shfl_sync(0xffffffffu, w0, i & 31) * ring.get(i);
      ring.fetch(b + kScaleAhead, i);
      if (!warp_poll(&sfull[c], (i / kSlots) & 1, ctx, kSiteSum)) break;
      tc_fence_after();
      const float2 s2 = make_float2(sc, sc);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint32_t r[16];
        tmem_ld16(tl + c * kTile + h * 16, r);
        tmem_wait_ld16(r);
        if (h == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sempty[c]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float2& a = reinterpret_cast<float2*>(sum)[h * 8 + e];
          a = __ffma2_rn(make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), s2, a);
        }
      }
    }
  }

  __syncthreads();  // the ring's last reads are done: sums and staged rows take its place
  if (p.split == 1) {
    if (warp < 8) store_rows(p, smem + warp * kOutBytes, m0 + (warp & 3) * 32, n0 + (warp >> 2) * 64, sum);
  } else {
    float* sums = reinterpret_cast<float*>(smem);
    if (warp < 8) {
      const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * 64;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        *reinterpret_cast<float4*>(sums + row * kSumPitch + c0 + 4 * e) = make_float4(sum[4 * e], sum[4 * e + 1], sum[4 * e + 2], sum[4 * e + 3]);
    }
    cluster_sync_all();
    // rows dealt over the cluster's warps, four columns a lane: a warp reads whole rows of the other
    // blocks' sums (read 16 bytes a row, the exchange alone took 6 us)
    const int n = n0 + lane * 4;
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = p.bias != nullptr && n + e < p.N ? __ldg(p.bias + n + e) : 0.f;
    for (int row = rank * 8 + warp; warp < 8 && row < kTile && m0 + row < p.M; row += p.split * 8) {
      float4 f[kMaxSplit];
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < p.split)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(f[r].x), "=f"(f[r].y), "=f"(f[r].z), "=f"(f[r].w)
                       : "r"(cluster_addr(sums + row * kSumPitch + lane * 4, r)));
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < kMaxSplit; ++r)
        if (r < p.split) {
          v[0] += f[r].x;
          v[1] += f[r].y;
          v[2] += f[r].z;
          v[3] += f[r].w;
        }
      const long long at = (m0 + row) * p.ldo + n;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += bias[e];
      if (p.vec && n + 4 <= p.N) {
        if (p.out_type == kF32) {
          *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
          const uint2 u = p.out_type == kF16 ? make_uint2(k8::pack2(v[0], v[1], __half()), k8::pack2(v[2], v[3], __half()))
                                             : make_uint2(k8::pack2(v[0], v[1], __nv_bfloat16()), k8::pack2(v[2], v[3], __nv_bfloat16()));
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = u;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.N) store_out(p.out, p.out_type, at + e, v[e]);
      }
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are being read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kSlots * kTile);
  }
}


// ------------------------------------------------------------------------------------------
// Many rows and columns: the same sums on CTA pairs, 256 rows of x by 256 of w8 a tile, through
// MMAs that span both SMs (M = 256): each CTA brings half of either operand, so an SM reads half
// the bytes a product of the 128 x 128 tiles' kernel, whose reads the L2 cannot feed at the tensor
// cores' rate.  CTA r holds the sums of rows [128 r, + 128) of the tile.  One pair a two SMs,
// persistent over tiles; tiles go in groups of kGroup row tiles by all column tiles, so the
// operands of the tiles that run together stay in L2.
//
// A step's products are needed apart from the next step's, and TMEM holds two steps (512
// columns), so the rate hangs on how soon a slot is free again.  A step is made as two halves of 128
// columns with slots of their own, so that one is taken out while the other is made.  Eight warps a
// half take the products out, 64 columns each, and touch no mbarrier on the way: an mbarrier
// operation waits behind the MMAs' reads of shared memory (100 to 270 cycles each were seen), so a
// warp of each half polls for the MMAs' commits and hands the slots back, and meets the eight at
// named barriers.
//   warp 0      TMA of this CTA's halves, counted on the even CTA's barrier (.cta_group::2)
//   warp 1      TMEM and, in the even CTA, the MMAs (M = 256, N = 128, four of K = 32 a half)
//   warps 2-3   half 0's and 1's barriers
//   warps 4-19  sums: half h of the columns = warps 4 + 8 h .., two warps a TMEM lane quadrant
// ------------------------------------------------------------------------------------------
namespace pair {

constexpr int kStages = 5;
constexpr int kThreads = 640;
constexpr int kTileMN = 256;
constexpr int kGroup = 8;
constexpr int kSumThreads = 256;           // of a half
constexpr int kBarFull = 1, kBarRead = 5;  // named barriers of the four slots: products there, products read
constexpr int kSumRegs = 104, kOtherRegs = 64;  // 512 * 104 + 128 * 64 = 640 * 96
constexpr int OFF_A = 0;
constexpr int OFF_B = kStages * kOperand;
constexpr int OFF_OUT = 2 * kStages * kOperand;  // staged rows of the output, a warp each
constexpr int OFF_XS = OFF_OUT + 16 * kOutBytes;  // the warps' rings of scales
constexpr int OFF_BAR = OFF_XS + 16 * kScaleAhead * 128;
constexpr int SMEM_BYTES = OFF_BAR + 256;
static_assert(SMEM_BYTES <= 232448, "K9 pair shared memory");

enum Site : unsigned int { kSiteProd = 0x911, kSiteMma = 0x912, kSiteSlot = 0x913, kSiteSum = 0x914, kSiteLayout = 0x91f };

__device__ __forceinline__ void named_bar_arrive(uint32_t id, uint32_t nthreads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// A load into this CTA's shared memory whose bytes count on `bar`, a barrier of either CTA of the
// pair (a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

// warp_poll for a barrier that the other CTA of the pair completes, in the cluster's scope: relaxed
// polls, and once the phase is there an acquire of shared memory alone, the counterpart of
// mbar_arrive_cluster_smem's release.  All the barriers of a pair are waited for so: the other CTA's loads
// and readers and the paired MMAs' commits complete them.  (16384 x 10240 -> 2560: 470 us, with acquires of
// all memory 472; in the CTA's own scope, which orders nothing between two CTAs, 460.)
__device__ __forceinline__ bool mbar_test_pair(uint64_t* bar, uint32_t parity, uint32_t hint_ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(hint_ns)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ bool warp_poll_pair(uint64_t* bar, uint32_t parity, const WaitCtx& ctx, unsigned int site) {
  bool ok = false;
  for (int i = 0; i < 64 && !ok; ++i) ok = mbar_test_pair(bar, parity, 0);
  if (!__all_sync(0xffffffffu, ok)) {
    const uint64_t t0 = globaltimer_ns();
    while (!ok) {
      ok = mbar_test_pair(bar, parity, kSuspendHintNs);
      if (ok || *ctx.abort) break;
      if (globaltimer_ns() - t0 > ctx.timeout_ns) {
        raise_abort(ctx, site);
        break;
      }
    }
    ok = __all_sync(0xffffffffu, ok);
  }
  asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
  return ok;
}

// Tile t: row tiles in groups of kGroup, column tiles inside a group, row tiles fastest.
__device__ __forceinline__ void decode(const Params& p, int t, int& m0, int& n0) {
  const int tiles_n = (p.N + kTileMN - 1) / kTileMN;
  const int per = kGroup * tiles_n, g = t / per, r = t - g * per;
  const int rows = min(kGroup, p.tiles_m - g * kGroup);
  m0 = (g * kGroup + r % rows) * kTileMN;
  n0 = r / rows * kTileMN;
}

__global__ void __launch_bounds__(kThreads, 1) linear8_pair_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t smem[];
  DeviceStatus* const status = p.status != nullptr ? p.status : &g_own_status;
  if (smem_u32(smem) & 1023) {  // a property of the kernel: both CTAs take the same branch
    if (threadIdx.x == 0) record_status(status, kStatusLayout, kSiteLayout);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  uint64_t* full = bars;              // [kStages] even CTA: both CTAs' halves have landed
  uint64_t* empty = bars + kStages;   // [kStages] the paired MMAs have read the stage (both CTAs)
  uint64_t* sfull = bars + 2 * kStages;  // [2 steps][2 halves] the products are in the slot (both CTAs)
  uint64_t* sempty = sfull + 4;          // [2 steps][2 halves] even CTA: both CTAs' readers have them
  uint64_t& drain_bar = sempty[4];
  uint32_t& tmem_base_sh = *reinterpret_cast<uint32_t*>(&drain_bar + 1);
  volatile int& abort_sh = *reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(&drain_bar + 1) + 4);
  const WaitCtx ctx{status, &abort_sh, p.timeout_ns};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int tiles = p.tiles_m * ((p.N + kTileMN - 1) / kTileMN);
  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&sfull[s], 1);
      mbar_init(&sempty[s], 2);
    }
    mbar_init(&drain_bar, 1);
    fence_mbar_init();
    tma_prefetch_desc(&p.tm_x);
    tma_prefetch_desc(&p.tm_w);
  }
  if (warp == 1) {
    tmem_alloc_pair(&tmem_base_sh, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers are initialised before any arrive across
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  griddep_trigger();
  griddep_wait();

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 0) {
      const bool leader = elect_one();
      const uint32_t bar0 = cluster_addr(&full[0], 0);
      uint32_t s = 0, ph = 0, i = 0;
      bool ok = true;
      for (int t = first; ok && t < tiles; t += step) {
        int m0, n0;
        decode(p, t, m0, n0);
        m0 += static_cast<int>(rank) * kTile;
        n0 += static_cast<int>(rank) * (kTile / 2);
        for (int b = 0; b < p.kb; ++b, ++i) {
          if (!(ok = warp_poll_pair(&empty[s], ph ^ 1, ctx, kSiteProd))) break;
          if (leader) {
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 4 * kOperand);
            tma_load_2d_pair(smem + OFF_A + s * kOperand, &p.tm_x, bar0 + s * sizeof(uint64_t), b * 128, m0);
            // of each half's 128 rows of w8 the CTA brings 64
            tma_load_2d_pair(smem + OFF_B + s * kOperand, &p.tm_w, bar0 + s * sizeof(uint64_t), b * 128, n0);
            tma_load_2d_pair(smem + OFF_B + s * kOperand + kOperand / 2, &p.tm_w, bar0 + s * sizeof(uint64_t), b * 128, n0 + kTile);
          }
          __syncwarp();
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok && rank == 0 && leader)
        for (uint32_t r = 0; r < kStages; ++r) {
          const uint32_t armed = i > r ? (i - r + kStages - 1) / kStages : 0;
          if (armed) mbar_drain(&full[r], (armed - 1) & 1, 200000000ull);
        }
      __syncwarp();
    } else if (warp == 1 && rank == 0) {
      // The whole warp walks the steps and one lane issues: what the MMAs take from uniform registers
      // (descriptors, addresses) is then computed there, and not moved there value by value.
      const uint32_t idesc = idesc_e4m3_f32(kTileMN, kTile);
      const uint64_t ad = sdesc_sw128(smem_u32(smem + OFF_A), 16, 1024), bd = sdesc_sw128(smem_u32(smem + OFF_B), 16, 1024);
      const bool leader = elect_one();
      uint32_t s = 0, ph = 0, i = 0;
      // (after an abort every wait fails at once, and the loop runs out on whatever is there)
      for (int t = first; t < tiles; t += step)
        for (int b = 0; b < p.kb; ++b, ++i) {
          const uint32_t c = i & 1;
          warp_poll_pair(&full[s], ph, ctx, kSiteMma);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            warp_poll_pair(&sempty[2 * c + h], ((i >> 1) & 1) ^ 1, ctx, kSiteSlot);
            tc_fence_after();
            const uint64_t as = sdesc_add(ad, s * kOperand), bs = sdesc_add(bd, s * kOperand + h * (kOperand / 2));
            const uint32_t d = tmem + c * 256 + h * kTile;
            if (leader) {
              umma_f8_pair(d, as, bs, idesc, 0u);
              umma_f8_pair(d, sdesc_add(as, 32), sdesc_add(bs, 32), idesc, 1u);
              umma_f8_pair(d, sdesc_add(as, 64), sdesc_add(bs, 64), idesc, 1u);
              umma_f8_pair(d, sdesc_add(as, 96), sdesc_add(bs, 96), idesc, 1u);
              umma_commit_pair(&sfull[2 * c + h], 0x3);
              if (h == 1) umma_commit_pair(&empty[s], 0x3);
            }
            __syncwarp();
          }
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      if (leader) {
        umma_commit_pair(&drain_bar, 0x1);
        mbar_drain(&drain_bar, 0, 200000000ull);
      }
      __syncwarp();
    } else if (warp >= 2) {
      const int h = warp - 2;
      const uint32_t slots = cluster_addr(&sempty[h], 0);
      uint32_t i = 0;
      for (int t = first; t < tiles; t += step)
        for (int b = 0; b < p.kb; ++b, ++i) {
          const uint32_t c = i & 1;
          warp_poll_pair(&sfull[2 * c + h], (i >> 1) & 1, ctx, kSiteSum);
          named_bar_arrive(kBarFull + 2 * c + h, kSumThreads + 32);
          named_bar_sync(kBarRead + 2 * c + h, kSumThreads + 32);
          tc_fence_after();
          tc_fence_before();
          if (lane == 0) {
            if (rank == 0) mbar_arrive(&sempty[2 * c + h]);
            else mbar_arrive_cluster_smem(slots + 2 * c * sizeof(uint64_t));
          }
          __syncwarp();
        }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
    const int q = warp & 3, half = (warp - 4) >> 3, col = half * kTile + ((warp >> 2) & 1 ? 0 : 64);
    const uint32_t tl = tmem + (static_cast<uint32_t>(q * 32) << 16) + col;
    const int nb_last = (p.N + 127) / 128 - 1;
    uint32_t i = 0;
    for (int t = first; t < tiles; t += step) {
      int m0, n0;
      decode(p, t, m0, n0);
      const float* ws = p.ws + static_cast<long long>(min((n0 >> 7) + half, nb_last)) * p.kb;
      float sum[64];
#pragma unroll
      for (int e = 0; e < 64; ++e) sum[e] = 0.f;
      // the weight's scales: lane j holds that of step 32 i + j, and of the next 32 steps
      auto load_ws = [&](int b) { return b + lane < p.kb ? __ldg(ws + b + lane) : 0.f; };
      float w0 = load_ws(0), w1 = load_ws(32);
      const float* xs = p.xst + m0 + static_cast<int>(rank) * kTile + q * 32 + lane;
      const ScaleRing ring{xs, p.ld_xs, smem_u32(smem + OFF_XS + (warp - 4) * (kScaleAhead * 128)) + lane * 4, p.kb};
      for (int u = 0; u < kScaleAhead; ++u) ring.fetch(u, u);
      for (int b = 0; b < p.kb; ++b, ++i) {
        const uint32_t c = i & 1;
        if (b > 0 && (b & 31) == 0) {
          w0 = w1;
          w1 = load_ws(b + 32);
        }
        const float sc = __shfl_sync(0xffffffffu, w0, b & 31) * ring.get(b);
        ring.fetch(b + kScaleAhead, b);
        named_bar_sync(kBarFull + 2 * c + half, kSumThreads + 32);
        tc_fence_after();
        const float2 s2 = make_float2(sc, sc);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[16], r1[16];
          tmem_ld16(tl + c * 256 + h * 32, r);
          tmem_ld16(tl + c * 256 + h * 32 + 16, r1);
          tmem_wait_ld16x2(r, r1);
          if (h == 1) {
            tc_fence_before();
            named_bar_arrive(kBarRead + 2 * c + half, kSumThreads + 32);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float2& a = reinterpret_cast<float2*>(sum)[h * 16 + e];
            a = __ffma2_rn(make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), s2, a);
            float2& a1 = reinterpret_cast<float2*>(sum)[h * 16 + 8 + e];
            a1 = __ffma2_rn(make_float2(__uint_as_float(r1[2 * e]), __uint_as_float(r1[2 * e + 1])), s2, a1);
          }
        }
      }
      store_rows(p, smem + OFF_OUT + (warp - 4) * kOutBytes, m0 + static_cast<int>(rank) * kTile + q * 32, n0 + col, sum);
    }
  }

  tc_fence_before();
  __syncthreads();
  // neither CTA leaves (or frees the pair's TMEM) while the other can still arrive on its barriers
  // or run a paired MMA over its shared memory
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace pair
}  // namespace k9
}  // namespace tmu

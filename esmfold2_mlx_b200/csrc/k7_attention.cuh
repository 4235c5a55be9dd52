// K7: attention over packed sequences.
//
// Row i of sequence s (tokens cu[s] .. cu[s + 1]) and query head h, key head h / (Hq / Hkv):
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(x_ij - max_j x_ij),   x_ij = scale q_i . k_j + bias_ij
// over the keys j of the same sequence, j <= i if causal, that bias_ij = -inf does not hide.  A row
// that sees no key is zero.
//
// One pass over the keys with the running maximum m and sum l of the softmax (Milakov and Gimelshein
// 2018), in base 2 (x times log2 e).  The accumulator O = sum_j 2^(x_ij - m) v_j stays in tensor memory,
// so moving m would mean reading and writing all of it: m only moves when a tile's maximum exceeds it by
// more than 8 (a published refinement of that pass), so weights reach at most 2^8 (exact in fp32 sums, and
// a common factor of the 16-bit weights; fp16: kLift more), and the result, O / l, does not depend on when
// it moved.
//
// A tile is 128 rows of one head; a step takes 128 keys: S = Q K^T (128 x 128, fp32 in TMEM), the
// softmax of S's rows, P in TMEM in the inputs' type, and O += P V with P as the MMA's A operand out of
// TMEM.  A tile's step is a chain, S to P to O to S, so an SM always has two tiles in hand, and the
// tensor cores work for one while the softmax of the other runs:
//   D <= 64  two blocks an SM, of one tile each: with sequences of a few hundred tokens, two tiles of one
//            sequence would often be one, and with equal blocks the last round is half as long
//   D > 64   one block an SM, of two tiles A and B of one sequence that share their keys and values,
//            which two blocks would not find room for
// (A row's softmax spread over two threads was no faster at D = 64 and 8 % slower at 128.)
// Warps of a block: the softmax, a thread a row (warp w: tile w / 4, TMEM lanes 32 (w % 4) ..), then one
// for TMA (Q, then K and V through rings of kStages tiles), one for TMEM and the MMAs, and two idle
// ones that complete the warpgroup which gives its registers to the softmax.
// TMEM columns: D <= 64: O 64, S 128, P 64: S has its own columns, so the next S is made while the
// softmax works on this one.  D > 64: O 2 x 128, S 2 x 128, and P overwrites S; the MMAs of a block
// execute in issue order, so S of step j + 1 follows the P V that reads them.
//
// A product cannot leave out a hidden key: its weight is 0, and 0 times an infinity or a NaN in its v is a
// NaN (as is -inf plus a NaN score).  A row that comes out non-finite, and that a key it does not see may
// have made so (spoiled_rows), is therefore made again key by key (exact_row), by its warp.  (The check
// and the two functions' presence cost 0 to 2 %: causal prompts 630 -> 631 us, 2048 tokens 69.1 -> 69.6,
// 4 x 384 tokens with bias 13.9 -> 14.2.  2048 tokens, 16 heads of 64 with a bias, one call alone: 65 us; a NaN
// that rows see 231, for the search, and 18 ms while every such row was made again; a NaN in hidden v 8 ms.)
//
// Blocks find their sequence without a prefix sum over the lengths: sequence s owns the slots
// from floor(cu[s] / R) + s (R rows a block), at least as many as it has blocks, and the slots it does
// not need return at once.  The heads are the grid's fast axis, and later rows come first when
// causal, so the long blocks start first.
#pragma once

#include <cuda_bf16.h>

#include "k8_qk_rope.cuh"

namespace tmu {
namespace k7 {

constexpr int kTile = 128;     // query rows of a tile, keys of a step
constexpr int kAtom = kTile * 128;  // 64 values of 128 rows
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMoveMax = 8.f;
// fp16 weights are 2^7 times as large, up to 2^15: those that round to 0 in the product (and stay in the
// sum) are below 2^-32 of the row's largest, not 2^-25, under which the keys of a long row can add up to
// a visible share.  bf16 has the range.
template <typename T>
constexpr float kLift = __is_same(T, __half) ? 7.f : 0.f;

struct Params {
  CUtensorMap tm_q, tm_k, tm_v;  // [H, T, D]: box {64, 128, 1}, 128B swizzle, zero past the ends
  k8::View q, k, v, o;  // (q, k and v again, for exact_row)
  const int* cu;
  const void* bias;  // [S or 1, Hq, n, n] or null, the last axis contiguous
  long long bias_ss, bias_sh, bias_sr;
  int bias_n, bias_width;  // elements a copy of the bias may take: 8, 4 or 2, by its alignment
  int S, T, hq, group, d, causal;
  float scale;
  DeviceStatus* status;
  unsigned long long timeout_ns;
};

template <int DP, bool BIAS>
struct Cfg {
  static constexpr int kTiles = DP == 64 ? 1 : 2;       // of a block
  static constexpr int kBlocks = DP == 64 ? 2 : 1;      // an SM
  static constexpr int kRows = kTiles * kTile;
  static constexpr int kSoftmaxWarps = 4 * kTiles;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 4);
  // 128 * 200 + 128 * 56 = 256 * 128, 256 * 208 + 128 * 88 = 384 * 168
  static constexpr int kSoftmaxRegs = DP == 64 ? 200 : 208, kOtherRegs = DP == 64 ? 56 : 88;
  static constexpr int kAtoms = DP / 64;
  static constexpr int kTileBytes = kAtoms * kAtom;
  static constexpr int kStages = DP == 64 && !BIAS ? 3 : 2;
  static constexpr bool kOwnP = DP == 64;  // P beside S instead of over it
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = kTiles * kTileBytes;
  static constexpr int OFF_V = OFF_K + kStages * kTileBytes;
  // A quarter of the exponentials on the FMA units, where two of the special function unit's 16 a
  // cycle and SM are as long as the products (a half as long at D > 64): 108 -> 100 us at 4096 tokens,
  // 18 heads of 64.  At D = 128 it does not pay: the causal prompts took 643 us with it and 629 without.
  static constexpr bool kMixedExp = DP == 64;
  // Bias of a warp's 32 rows: a step's 128 keys, or as many as fit beside the tiles.  The rows' 16-byte
  // accesses of eight rows meet 8 different bank groups by a swizzle (128 keys: no room for more than
  // the word behind each row, kept apart) or by the rows' pitch.
  static constexpr int kBiasCols = DP == 64 ? 128 : 32;
  static constexpr int kBiasPitch = DP == 64 ? 256 : 80;
  static constexpr int OFF_BIAS = OFF_V + kStages * kTileBytes;
  static constexpr int OFF_ROW = OFF_BIAS + (BIAS ? kSoftmaxWarps * 32 * kBiasPitch : 0);  // a word a softmax thread
  static constexpr int OFF_BAR = OFF_ROW + (BIAS && DP == 64 ? kSoftmaxWarps * 128 : 0);
  static constexpr int SMEM_BYTES = OFF_BAR + 256;
  static_assert(kBlocks * (SMEM_BYTES + 1024) <= 233472, "K7 shared memory");
  // TMEM columns of tile x
  static constexpr uint32_t kColumns = kTiles * 256;
  __device__ static constexpr uint32_t o_col(int x) { return x * DP; }
  __device__ static constexpr uint32_t s_col(int x) { return kTiles * DP + x * 128; }
  __device__ static constexpr uint32_t p_col(int x) { return kOwnP ? DP + 128 : s_col(x); }
};

enum Site : unsigned int {
  kSiteProdK = 0x701, kSiteProdV = 0x702, kSiteMmaQ = 0x703, kSiteMmaK = 0x704, kSiteMmaV = 0x705, kSiteMmaS = 0x706,
  kSiteMmaP = 0x707, kSiteFix = 0x708, kSiteSoftS = 0x709, kSiteSoftO = 0x70a, kSiteEpi = 0x70b, kSiteLayout = 0x7ff
};

__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {  // as tmem_st32, 16 columns
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Ties registers of an earlier tcgen05.ld to the wait in front of it.
__device__ __forceinline__ void tie(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// max of three that keeps a NaN
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^t of a pair, t <= kMoveMax + kLift or so, on the fused multiply-add units, by the reduction and
// polynomial of Cody and Waite 1980 (sharing a softmax's exponentials between the two units is published
// too): t = n + f with n the nearest integer (adding 1.5 * 2^23 leaves it in the low bits) and |f| <= 1/2,
// 2^f by a polynomial of degree 4 with constant term 1 (minimax in the relative error, 2^-18.4, against 2^-9
// and 2^-11 of the weights' types), n added to the exponent.  t is held at -127 or above, where the sum of
// exponents is exactly 0: -inf gives +0.  A NaN is lost.
__device__ __forceinline__ float2 exp2_fma(float2 t) {
  t = make_float2(fmaxf(t.x, -127.f), fmaxf(t.y, -127.f));
  const float2 r = __fadd2_rn(t, make_float2(12582912.f, 12582912.f));
  const float2 n = __fadd2_rn(r, make_float2(-12582912.f, -12582912.f));
  const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), t);
  float2 p = make_float2(0.009581047110259533f, 0.009581047110259533f);
  p = __ffma2_rn(p, f, make_float2(0.05590597167611122f, 0.05590597167611122f));
  p = __ffma2_rn(p, f, make_float2(0.24024145305156708f, 0.24024145305156708f));
  p = __ffma2_rn(p, f, make_float2(0.6931243538856506f, 0.6931243538856506f));
  p = __ffma2_rn(p, f, make_float2(1.f, 1.f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23)));
}

template <int N>
struct Int {
  static constexpr int value = N;
};

__device__ __forceinline__ int clamp_token(int t, int T) { return min(max(t, 0), T); }

// The sequence that owns `slot` (a warp searches 32-ary): the last s with floor(cu[s] / R) + s <= slot.
template <int R>
__device__ __forceinline__ int find_sequence(const int* cu, int S, int T, int slot) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const long long s = lo + static_cast<long long>(lane) * step;
    const bool in = s < hi && (lane == 0 || clamp_token(__ldg(cu + s), T) / R + s <= slot);
    const int b = 31 - __clz(__ballot_sync(0xffffffffu, in));
    lo += b * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// Row `row` of a sequence by a warp, over the keys that the row sees and no others: 32 keys at a time, a
// lane a key for the scores and a column (of every 32) for the output.  Weights stay in fp32.  Slow (0.11 ms
// a row of 1200 keys of 64), and reached only as said at the top; it stops where the whole row is NaN.
template <typename T>
__device__ __noinline__ void exact_row(const Params& p, int seq, int head, int beg, int len, int row) {
  const int lane = threadIdx.x & 31, kv = head / p.group, lim = p.causal ? min(len, row + 1) : len;
  const T* q = static_cast<const T*>(p.q.p) + (beg + row) * p.q.st + head * p.q.sh;
  const T* k = static_cast<const T*>(p.k.p) + beg * p.k.st + kv * p.k.sh;
  const T* v = static_cast<const T*>(p.v.p) + beg * p.v.st + kv * p.v.sh;
  const bool biased = row < p.bias_n;
  const T* b = static_cast<const T*>(p.bias) + seq * p.bias_ss + head * p.bias_sh + row * p.bias_sr;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < lim; j0 += 32) {
    const int j = j0 + lane;
    const float bias = biased && j < min(lim, p.bias_n) ? static_cast<float>(b[j]) : 0.f;
    const bool seen = j < lim && bias != -INFINITY;
    float x = -INFINITY;
    if (seen) {
      float s = 0.f;
#pragma unroll 4
      for (int c = 0; c < p.d; c += 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(q + c), e = *reinterpret_cast<const uint4*>(k + j * p.k.st + c);
        const uint32_t au[4] = {a.x, a.y, a.z, a.w}, eu[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = k8::unpack2(au[i], T()), g = k8::unpack2(eu[i], T());
          s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
        }
      }
      x = fmaf(s, p.scale, bias);
    }
    float top = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = fmaxf(m, top);
    const float at = top == -INFINITY ? 0.f : top;
    const float f = ex2_approx((m - at) * kLog2e), w = seen ? ex2_approx((x - at) * kLog2e) : 0.f;
    m = top;
    float sum = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = fmaf(l, f, sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= f;
    // eight keys' loads at a time: one key after the other, a row of 1200 keys took 290 us
    const unsigned in = __ballot_sync(0xffffffffu, seen);
#pragma unroll 1
    for (int s0 = 0; s0 < 32; s0 += 8) {
      float y[8][4];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const T* vs = v + min(j0 + s0 + s, lim - 1) * p.v.st;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[s][i] = static_cast<float>(vs[i * 32 + lane < p.d ? i * 32 + lane : 0]);
      }
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const float ws = __shfl_sync(0xffffffffu, w, s0 + s);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = in >> (s0 + s) & 1u ? fmaf(ws, y[s][i], acc[i]) : acc[i];
      }
    }
    bool lost = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) lost = lost && (i * 32 + lane >= p.d || acc[i] != acc[i]);
    if (__all_sync(0xffffffffu, lost)) break;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(p.o.p) + (beg + row) * p.o.st + head * p.o.sh;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i * 32 + lane < p.d) out[i * 32 + lane] = static_cast<T>(acc[i] * inv);
  __syncwarp();
}

// Which rows of `left` (bit r: row row0 + r) a key that they do not see may have made non-finite; for a
// warp.  Such a key, in [from, to), has a v that is not finite, or, where its score met a -inf bias, a k
// that is not or that is past 2^60; a row whose q is past 2^60 counts too (below both, 128 products stay
// finite in fp32).  A lane a key, then the rows against the keys that were found.
template <typename T, bool BIAS>
__device__ __noinline__ unsigned spoiled_rows(const Params& p, int seq, int head, int beg, int from, int to, int row0,
                                              unsigned left) {
  const int lane = threadIdx.x & 31, kv = head / p.group;
  const T* q = static_cast<const T*>(p.q.p) + (beg + row0 + lane) * p.q.st + head * p.q.sh;
  const T* k = static_cast<const T*>(p.k.p) + beg * p.k.st + kv * p.k.sh;
  const T* v = static_cast<const T*>(p.v.p) + beg * p.v.st + kv * p.v.sh;
  const T* b = static_cast<const T*>(p.bias) + seq * p.bias_ss + head * p.bias_sh;
  auto beyond = [&](const T* x, float limit) {  // is a value of the row not below `limit` (a NaN is not)
    bool any = false;
#pragma unroll 4
    for (int c = 0; c < p.d; c += 8) {
      const uint4 a = *reinterpret_cast<const uint4*>(x + c);
      const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = k8::unpack2(u[i], T());
        any |= !(fabsf(f.x) < limit) | !(fabsf(f.y) < limit);
      }
    }
    return any;
  };
  unsigned found = BIAS ? __ballot_sync(0xffffffffu, (left >> lane & 1u) && beyond(q, 0x1p60f)) : 0u;
  for (int j0 = from; j0 < to && found != left; j0 += 32) {
    const int j = j0 + lane;
    const bool bad = j < to && (beyond(v + j * p.v.st, INFINITY) || (BIAS && beyond(k + j * p.k.st, 0x1p60f)));
    if (!__any_sync(0xffffffffu, bad)) continue;
    for (unsigned rest = left & ~found; rest != 0u; rest &= rest - 1) {
      const int r = __ffs(rest) - 1, row = row0 + r;
      const bool hidden = (p.causal && j > row) || (BIAS && bad && row < p.bias_n && j < p.bias_n &&
                                                    static_cast<float>(b[row * p.bias_sr + j]) == -INFINITY);
      if (__any_sync(0xffffffffu, bad && hidden)) found |= 1u << r;
    }
  }
  return found;
}

template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(Cfg<DP, BIAS>::kThreads, Cfg<DP, BIAS>::kBlocks) attention_kernel(const __grid_constant__ Params p) {
  using C = Cfg<DP, BIAS>;
  constexpr int NS = C::kStages, kSoftmaxWarps = C::kSoftmaxWarps, kRows = C::kRows;
  extern __shared__ uint8_t smem[];
  DeviceStatus* const status = p.status != nullptr ? p.status : &g_own_status;
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) record_status(status, kStatusLayout, kSiteLayout);
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  griddep_wait();

  const int slot = blockIdx.x / p.hq, head = blockIdx.x - slot * p.hq;
  const int seq = find_sequence<kRows>(p.cu, p.S, p.T, slot);
  const int beg = clamp_token(__ldg(p.cu + seq), p.T);
  const int len = max(clamp_token(__ldg(p.cu + seq + 1), p.T) - beg, 0);
  const int blocks = (len + kRows - 1) / kRows;
  const int blk = slot - (beg / kRows + seq);
  if (blk < 0 || blk >= blocks) return;
  const int q0 = (p.causal ? blocks - 1 - blk : blk) * kRows;
  // steps of tiles A and B (B may have no rows)
  auto steps = [&](int x) {
    const int first = q0 + x * kTile;
    if (first >= len) return 0;
    const int keys = p.causal ? min(len, first + kTile) : len;
    return (keys + kTile - 1) / kTile;
  };
  const int n0 = steps(0), n1 = C::kTiles == 2 ? steps(1) : 0, n = max(n0, n1);

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* kfull = bars;
  uint64_t* kempty = bars + 4;
  uint64_t* vfull = bars + 8;
  uint64_t* vempty = bars + 12;
  uint64_t* qfull = bars + 16;   // [2]
  uint64_t* sfull = bars + 18;   // [2] S of a step is in TMEM
  uint64_t* sfree = bars + 20;   // [2] the softmax has read S (own P columns only)
  uint64_t* pfull = bars + 22;   // [2] P of a step is in TMEM
  uint64_t* ofull = bars + 24;   // [2] P V of a step is done
  uint64_t& vfixed = bars[26];   // the last V tile's foreign rows are cleared
  uint64_t& drain_bar = bars[27];
  uint32_t& tmem_base_sh = *reinterpret_cast<uint32_t*>(bars + 28);
  volatile int& abort_sh = *reinterpret_cast<volatile int*>(reinterpret_cast<uint8_t*>(bars + 28) + 4);
  const WaitCtx ctx{status, &abort_sh, p.timeout_ns};
  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < NS; ++s) {
      mbar_init(&kfull[s], 1);
      mbar_init(&kempty[s], 1);
      mbar_init(&vfull[s], 1);
      mbar_init(&vempty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&qfull[x], 1);
      mbar_init(&sfull[x], 1);
      mbar_init(&sfree[x], 4);  // the tile's warps
      mbar_init(&pfull[x], 4);
      mbar_init(&ofull[x], 1);
    }
    mbar_init(&vfixed, 1);
    mbar_init(&drain_bar, 1);
    fence_mbar_init();
  }
  if (warp == kSoftmaxWarps + 1) {
    tmem_alloc(&tmem_base_sh, C::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  griddep_trigger();
  const bool fix = n * kTile > len;  // the last step's keys end inside the tile

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    if (warp == kSoftmaxWarps) {
      // ------------------------------ loads ------------------------------
      const bool leader = elect_one();
      const int kv = head / p.group;
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int h) {
        if (leader) {
          mbar_arrive_expect_tx(bar, C::kTileBytes);
#pragma unroll
          for (int a = 0; a < C::kAtoms; ++a) tma_load_3d(dst + a * kAtom, map, bar, a * 64, row, h);
        }
        __syncwarp();
      };
      int j = 0;
      bool ok = true;
      load(smem + C::OFF_Q, &p.tm_q, &qfull[0], beg + q0, head);
      for (; j < n; ++j) {
        const int s = j % NS, ph = (j / NS) & 1;
        if (!(ok = warp_poll(&kempty[s], ph ^ 1, ctx, kSiteProdK))) break;
        load(smem + C::OFF_K + s * C::kTileBytes, &p.tm_k, &kfull[s], beg + j * kTile, kv);
        if (j == 0 && n1 > 0) load(smem + C::OFF_Q + C::kTileBytes, &p.tm_q, &qfull[1], beg + q0 + kTile, head);
        if (!(ok = warp_poll(&vempty[s], ph ^ 1, ctx, kSiteProdV))) {
          if (leader) mbar_drain(&kfull[s], ph, 200000000ull);
          break;
        }
        load(smem + C::OFF_V + s * C::kTileBytes, &p.tm_v, &vfull[s], beg + j * kTile, kv);
      }
      if (!ok && leader) {
        mbar_drain(&qfull[0], 0, 200000000ull);
        if (n1 > 0 && j > 0) mbar_drain(&qfull[1], 0, 200000000ull);
        for (int s = 0; s < NS; ++s) {
          const int armed = j > s ? (j - s + NS - 1) / NS : 0;
          if (armed) {
            mbar_drain(&kfull[s], (armed - 1) & 1, 200000000ull);
            mbar_drain(&vfull[s], (armed - 1) & 1, 200000000ull);
          }
        }
      }
      __syncwarp();
      // Clear the last V tile's rows that belong to no key of the sequence: their weights are 0, but
      // 0 times another sequence's NaN would be a NaN.  This warp made the load, so the phase it
      // waits for is the barrier's current one.
      const int s = (n - 1) % NS, keep = len - (n - 1) * kTile;
      if (fix && warp_poll(&vfull[s], ((n - 1) / NS) & 1, ctx, kSiteFix)) {
        for (int c = keep * 8 + lane; c < kTile * 8; c += 32)
          for (int a = 0; a < C::kAtoms; ++a)
            *reinterpret_cast<uint4*>(smem + C::OFF_V + s * C::kTileBytes + a * kAtom + c * 16) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&vfixed);
      }
    } else if (warp == kSoftmaxWarps + 1) {
      // ------------------------------ MMAs ------------------------------
      constexpr bool kBf16 = !__is_same(T, __half);
      const bool leader = elect_one();
      const int ksteps = (p.d + 15) / 16;
      const uint32_t id_s = kBf16 ? idesc_bf16_f32(128, 128, false, false) : idesc_f16_f32(128, 128, false, false);
      const uint32_t id_o = kBf16 ? idesc_bf16_f32(128, ksteps * 16, false, true) : idesc_f16_f32(128, ksteps * 16, false, true);
      const uint64_t qd = sdesc_sw128(smem_u32(smem + C::OFF_Q), 16, 1024);
      const uint64_t kd = sdesc_sw128(smem_u32(smem + C::OFF_K), 16, 1024);
      const uint64_t vd = sdesc_sw128(smem_u32(smem + C::OFF_V), kAtom, 1024);
      auto issue_s = [&](int x, int j) {  // S_x(j) = Q_x K_j^T
        const int s = j % NS;
        if (j == 0 && !warp_poll(&qfull[x], 0, ctx, kSiteMmaQ)) return false;
        if (!warp_poll(&kfull[s], (j / NS) & 1, ctx, kSiteMmaK)) return false;
        tc_fence_after();
        const uint64_t qs = sdesc_add(qd, x * C::kTileBytes), ks = sdesc_add(kd, s * C::kTileBytes);
        const uint32_t d = tmem + C::s_col(x);
        if (leader) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
            if (k < ksteps)
              umma_f16(d, sdesc_add(qs, (k >> 2) * kAtom + (k & 3) * 32), sdesc_add(ks, (k >> 2) * kAtom + (k & 3) * 32), id_s,
                       k > 0 ? 1u : 0u);
          umma_commit(&sfull[x]);
          if (x == 1 || j >= n1) umma_commit(&kempty[s]);  // the last use of K_j
        }
        __syncwarp();
        return true;
      };
      // tile x's part of step j: S of the next step, and O += P V
      auto tile_step = [&](int x, int j, int nx) {
        const int s = j % NS;
        if (C::kOwnP && j + 1 < nx)
          if (!warp_poll(&sfree[x], j & 1, ctx, kSiteMmaS) || !issue_s(x, j + 1)) return false;
        if (!warp_poll(&pfull[x], j & 1, ctx, kSiteMmaP)) return false;
        tc_fence_after();
        const uint64_t vs = sdesc_add(vd, s * C::kTileBytes);
        const uint32_t d = tmem + C::o_col(x), a = tmem + C::p_col(x);
        if (leader) {
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k) umma_ts(d, a + k * 8, sdesc_add(vs, k * 2048), id_o, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit(&ofull[x]);
        }
        __syncwarp();
        return C::kOwnP || j + 1 >= nx || issue_s(x, j + 1);
      };
      bool ok = issue_s(0, 0) && (n1 == 0 || issue_s(1, 0));
      for (int j = 0; ok && j < n; ++j) {
        const int s = j % NS;
        if (!(ok = warp_poll(&vfull[s], (j / NS) & 1, ctx, kSiteMmaV))) break;
        if (fix && j == n - 1 && !(ok = warp_poll(&vfixed, 0, ctx, kSiteMmaV))) break;
        if (j < n0 && !(ok = tile_step(0, j, n0))) break;
        if (j < n1 && !(ok = tile_step(1, j, n1))) break;
        if (leader) umma_commit(&vempty[s]);
        __syncwarp();
      }
      if (leader) {
        umma_commit(&drain_bar);
        mbar_drain(&drain_bar, 0, 200000000ull);
      }
      __syncwarp();
    }
  } else {
    // ------------------------------ softmax ------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
    const int x = warp >> 2;
    const int nx = x == 0 ? n0 : n1;
    const int tile0 = q0 + x * kTile;
    const int row = tile0 + (warp & 3) * 32 + lane;  // within the sequence
    const uint32_t tl = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const bool flip = p.scale < 0.f;
    // a scale of 0 would turn a hidden key's -inf into a NaN
    const float c = fmaxf(fabsf(p.scale) * (BIAS ? 1.f : kLog2e), 1e-30f);
    // The bias of the warp's rows comes through shared memory, copied asynchronously a step ahead in
    // whole rows: read by the row's thread from where it lies, 32 rows at a time, it cost
    // 64 us at 4 x 384 tokens.  Copies take 16, 8 or 4 bytes, whatever the rows' alignment
    // allows; a row that starts in the middle of a 4-byte word is shifted when it is read.  (An
    // aligned word that holds a value of the bias lies inside its allocation.)
    const int bn = min(p.bias_n, len);  // rows and keys that have a bias
    uint8_t* bbuf = smem + C::OFF_BIAS + warp * (32 * C::kBiasPitch);
    const T* bbase = static_cast<const T*>(p.bias) + seq * p.bias_ss + head * p.bias_sh;
    auto bias_at = [&](int r, int byte) {  // address of a staged byte of row r
      if (C::kBiasCols == 128) {
        if (byte == 256) return smem_u32(smem + C::OFF_ROW) + (warp * 32 + r) * 4u;
        return smem_u32(bbuf) + r * 256u + ((((byte >> 4) ^ (r & 7)) << 4) | (byte & 15));
      }
      return smem_u32(bbuf) + r * static_cast<uint32_t>(C::kBiasPitch) + byte;
    };
    // copies of W values, kBiasCols / W lanes a row (W = 2: 32 lanes, and one value more in shifted rows)
    auto copy_rows = [&](int k0, auto width) {
      constexpr int W = decltype(width)::value, kLanes = C::kBiasCols / W < 32 ? C::kBiasCols / W : 32;
      const int first = tile0 + (warp & 3) * 32, r0 = lane / kLanes, c = lane % kLanes * W;
      const T* src = bbase + (first + r0) * p.bias_sr + k0 + c;
      const int rows = bn - first, left = bn - k0 - c;  // values of this lane's columns that are there
#pragma unroll 4
      for (int r = r0; r < 32; r += 32 / kLanes) {
        if (r >= rows) break;
        if (W == 8) {
          if (left > 0) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(bias_at(r, c * 2)), "l"(src) : "memory");
        } else if (W == 4) {
          if (left > 0) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(bias_at(r, c * 2)), "l"(src) : "memory");
        } else {
          const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(src) >> 1) & 1;
#pragma unroll
          for (int e = 0; e <= C::kBiasCols; e += kLanes * 2)
            if (c + e < C::kBiasCols + shift && left + shift > e)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(bias_at(r, (c + e) * 2)), "l"(src + e - shift)
                           : "memory");
        }
        src += (32 / kLanes) * p.bias_sr;
      }
    };
    auto fetch_bias = [&](int k0) {
      if (p.bias_width == 8) copy_rows(k0, Int<8>());
      else if (p.bias_width == 4) copy_rows(k0, Int<4>());
      else copy_rows(k0, Int<2>());
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const uint32_t bshift =
        BIAS && p.bias_width == 2 ? (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(bbase + row * p.bias_sr) >> 1) & 1u) * 16u : 0u;
    const bool shifted = BIAS && __any_sync(0xffffffffu, bshift != 0u);
    const float2 c2 = make_float2(flip ? -c : c, flip ? -c : c);
    // bf16's lowest value times log2 e is past fp32's range: with a bf16 bias the maximum is kept in x's
    // own units and subtracted before the factor, so a row that is masked by nothing but lowest values
    // still sees its keys evenly.  (4 x 384 tokens, 16 heads of 48: 13.6 -> 14.2 us.  fp16 values
    // are far from it, and take the factor in one operation.)
    constexpr bool kUnits = BIAS && !__is_same(T, __half);
    constexpr float kMove = kUnits ? kMoveMax / kLog2e : kMoveMax;
    if (BIAS && nx > 0) fetch_bias(0);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nx; ++j) {
      if (!(ok = warp_poll(&sfull[x], j & 1, ctx, kSiteSoftS))) break;
      tc_fence_after();
      uint32_t r[kTile / 32][32];
#pragma unroll
      for (int b = 0; b < kTile / 32; ++b) tmem_ld32(tl + C::s_col(x) + b * 32, r[b]);
      tmem_wait_ld(r[0]);
#pragma unroll
      for (int b = 1; b < kTile / 32; ++b) tie(r[b]);
      if (C::kOwnP) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfree[x]);
      }
      float* v = reinterpret_cast<float*>(&r[0][0]);
      const int k0 = j * kTile;
      float mul = c;
      if (BIAS) {
        // x = s scale + bias, the exponential's factor is log2 e (without a bias the scale is folded into it)
        mul = kLog2e;
        const int have = row < bn ? bn - k0 : 0;
        const bool whole = __all_sync(0xffffffffu, have >= kTile);
#pragma unroll
        for (int b0 = 0; b0 < kTile; b0 += C::kBiasCols) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
          auto staged = [&](int g) {  // 16 bytes of the row, or the word behind it
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (C::kBiasCols == 128 && g == 16)
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(u.x) : "r"(bias_at(lane, 256)) : "memory");
            else
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                           : "r"(bias_at(lane, g * 16))
                           : "memory");
            return u;
          };
          auto add = [&](auto check) {
            constexpr bool kCheck = decltype(check)::value != 0;  // rows that start in a word, or end in the tile
            uint4 q = staged(0);
#pragma unroll
            for (int g = 0; g < C::kBiasCols / 8; ++g) {
              const uint4 next = kCheck || g + 1 < C::kBiasCols / 8 ? staged(g + 1) : q;
              const uint32_t u[5] = {q.x, q.y, q.z, q.w, next.x};
              q = next;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = b0 + g * 8 + 2 * e;
                float2 f = k8::unpack2(kCheck ? __funnelshift_r(u[e], u[e + 1], bshift) : u[e], T());
                if (kCheck) f = make_float2(i < have ? f.x : 0.f, i + 1 < have ? f.y : 0.f);
                const float2 x = __ffma2_rn(make_float2(v[i], v[i + 1]), c2, f);
                v[i] = x.x;
                v[i + 1] = x.y;
              }
            }
          };
          if (whole && !shifted) add(Int<0>());
          else add(Int<1>());
          __syncwarp();
          if (b0 + C::kBiasCols < kTile || j + 1 < nx) fetch_bias(k0 + b0 + C::kBiasCols);
        }
      } else if (flip) {
#pragma unroll
        for (int e = 0; e < kTile; ++e) v[e] = -v[e];
      }
      if (k0 + kTile > len || (p.causal && k0 + kTile - 1 > tile0)) {
        const int lim = (p.causal ? min(len, row + 1) : len) - k0;
#pragma unroll
        for (int e = 0; e < kTile; ++e) v[e] = e < lim ? v[e] : -INFINITY;
      }
      float mx[4] = {v[0], v[1], v[2], v[3]};
      float part;
      if (C::kMixedExp) {
#pragma unroll
        for (int e = 4; e < kTile - 4; e += 8)
#pragma unroll
          for (int f = 0; f < 4; ++f) mx[f] = max3_nan(mx[f], v[e + f], v[e + 4 + f]);
        mx[0] = max3_nan(mx[0], v[kTile - 4], v[kTile - 3]);
        mx[1] = max3_nan(mx[1], v[kTile - 2], v[kTile - 1]);
        part = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]);
      } else {
#pragma unroll
        for (int e = 4; e < kTile; ++e) mx[e & 3] = fmaxf(mx[e & 3], v[e]);
        part = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      }
      const float top = kUnits ? part : part * mul;
      if (j > 0 && C::kOwnP) {  // P's columns and O belong to P V of the last step (else S's being there says so)
        if (!(ok = warp_poll(&ofull[x], (j - 1) & 1, ctx, kSiteSoftO))) break;
        tc_fence_after();
      }
      const bool move = top > m + kMove || (m == -INFINITY && top > m);
      if (j == 0) {
        m = fmaxf(m, top);
      } else if (__any_sync(0xffffffffu, move)) {
        const float f = move ? ex2_approx(kUnits ? (m - top) * kLog2e : m - top) : 1.f;
        if (move) m = top;
        l *= f;
#pragma unroll 1
        for (int b = 0; b < DP / 16; ++b) {
          uint32_t o[16];
          const uint32_t at = tl + C::o_col(x) + b * 16;
          tmem_ld16(at, o);
          tmem_wait_ld16(o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st16(at, o);
        }
      }
      const float neg = m == -INFINITY ? 0.f : kLift<T> - m;
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int b = 0; b < kTile / 32; ++b) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x2 = make_float2(v[b * 32 + 2 * e], v[b * 32 + 2 * e + 1]), n2 = make_float2(neg, neg);
          const float2 t = kUnits ? __fmul2_rn(__fadd2_rn(x2, n2), make_float2(mul, mul)) : __ffma2_rn(x2, make_float2(mul, mul), n2);
          const float2 q = C::kMixedExp && (e & 3) == 3 ? exp2_fma(t) : make_float2(ex2_approx(t.x), ex2_approx(t.y));
          sum = __fadd2_rn(sum, q);
          w[e] = k8::pack2(q.x, q.y, T());
        }
        tmem_st16(tl + C::p_col(x) + b * 16, w);
      }
      l += sum.x + sum.y;
      // a NaN or an infinite score: its row is NaN, whichever way its exponential went
      if (C::kMixedExp && !(top < INFINITY)) l = NAN;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pfull[x]);
    }
    if (ok && nx > 0 && warp_poll(&ofull[x], (nx - 1) & 1, ctx, kSiteEpi)) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* out = static_cast<T*>(p.o.p) + static_cast<long long>(beg + row) * p.o.st + head * p.o.sh;
      float zero = l * 0.f;  // or a NaN, if anything of the row is not finite
#pragma unroll
      for (int b = 0; b < DP / 32; ++b) {
        const int c0 = b * 32;
        uint32_t o[32];
        tmem_ld32(tl + C::o_col(x) + c0, o);
        tmem_wait_ld(o);
        if (row >= len) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (c0 + g * 8 >= p.d) break;
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 y = make_float2(__uint_as_float(o[g * 8 + 2 * e]), __uint_as_float(o[g * 8 + 2 * e + 1]));
            zero = fmaf(y.x, 0.f, fmaf(y.y, 0.f, zero));
            u[e] = k8::pack2(y.x * inv, y.y * inv, T());
          }
          *reinterpret_cast<uint4*>(out + c0 + g * 8) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
      __syncwarp();  // (exact_row's stores follow the lanes' own)
      if (BIAS || p.causal) {
        unsigned left = __ballot_sync(0xffffffffu, row < len && zero != 0.f);
        // without a bias, only the last step has keys that some of its rows do not see
        if (left != 0u)
          left = spoiled_rows<T, BIAS>(p, seq, head, beg, BIAS ? 0 : tile0, min(len, nx * kTile), row - lane, left);
        for (; left != 0u; left &= left - 1) exact_row<T>(p, seq, head, beg, len, row - lane + __ffs(left) - 1);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kSoftmaxWarps + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kColumns);
  }
}

}  // namespace k7
}  // namespace tmu

// Host side of the sequence operators (tmu_attention, tmu_qk_norm_rope, tmu_quantize_rows,
// tmu_linear_fp8): argument checks and launches.  Included by tmu_capi.cu, whose helpers it uses.
#pragma once

namespace {

// The sequence kernels' shared-memory opt-in, once a device and kernel (bits of their own).
unsigned long long g_seq_attr_done[kMaxDevices] = {0};

int seq_device(Dev& d, int bit, const void* kernel, int smem) {
  int st = current_device(d, 0, nullptr, 0);
  if (st) return st;
  if (g_seq_attr_done[d.id] >> bit & 1) return TMU_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  // all of the SM's memory for blocks: some kernels run two an SM
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
  g_seq_attr_done[d.id] |= 1ull << bit;
  return TMU_OK;
}

// A [T, H, D] view of 16-bit values that 16-byte accesses can read: aligned base and strides.
int check_heads(const void* p, long long st, long long sh, const char* what) {
  if (p == nullptr) return fail(TMU_ERR_INVALID_ARGUMENT, what);
  if (!aligned16(p) || st % 8 || sh % 8) return fail(TMU_ERR_MISALIGNED, what);
  if (st < 0 || sh < 0) return fail(TMU_ERR_INVALID_ARGUMENT, what);
  return TMU_OK;
}

bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_packed(int T, int hq, int hkv, int D) {
  if (T < 0 || hq < 1 || hkv < 1 || D < 1) return fail(TMU_ERR_INVALID_ARGUMENT, "T, heads and D must be positive");
  if (T > 1 << 30) return fail(TMU_ERR_UNSUPPORTED, "T > 2^30");
  return TMU_OK;
}

template <typename T, int LPH, int NORM>
void (*k8_kernel(bool inter))(k8::Params) {
  return inter ? k8::qk_rope_kernel<T, LPH, NORM, true> : k8::qk_rope_kernel<T, LPH, NORM, false>;
}

template <typename T, int LPH>
void (*k8_kernel(int norm, bool inter))(k8::Params) {
  if (norm == TMU_NORM_NONE) return k8_kernel<T, LPH, k8::kNone>(inter);
  return norm == TMU_NORM_RMS ? k8_kernel<T, LPH, k8::kRms>(inter) : k8_kernel<T, LPH, k8::kLayer>(inter);
}

template <typename T>
void (*k8_kernel(int lph, int norm, bool inter))(k8::Params) {
  switch (lph) {
    case 2: return k8_kernel<T, 2>(norm, inter);
    case 4: return k8_kernel<T, 4>(norm, inter);
    case 8: return k8_kernel<T, 8>(norm, inter);
    case 16: return k8_kernel<T, 16>(norm, inter);
    default: return k8_kernel<T, 32>(norm, inter);
  }
}

template <int DP>
int launch_k7(const k7::Params& p, bool bf16, bool biased, int blocks, cudaStream_t stream) {
  void (*kern)(k7::Params) =
      bf16 ? (biased ? k7::attention_kernel<__nv_bfloat16, DP, true> : k7::attention_kernel<__nv_bfloat16, DP, false>)
           : (biased ? k7::attention_kernel<__half, DP, true> : k7::attention_kernel<__half, DP, false>);
  const int smem = biased ? k7::Cfg<DP, true>::SMEM_BYTES : k7::Cfg<DP, false>::SMEM_BYTES;
  Dev dev;
  const int bit = (DP == 128 ? 4 : 0) + (bf16 ? 2 : 0) + (biased ? 1 : 0);
  int st = seq_device(dev, bit, reinterpret_cast<const void*>(kern), smem);
  if (st) return st;
  cudaError_t e = launch_pdl(kern, blocks, k7::Cfg<DP, true>::kThreads, smem, stream, p);
  return e == cudaSuccess ? TMU_OK : cuda_fail(e, "launch attention_kernel");
}

template <typename X>
void (*k9_rows_kernel(int M))(k9::RowsParams) {
  return M <= 2 ? k9::linear8_rows_kernel<X, 1> : M <= 8 ? k9::linear8_rows_kernel<X, 4> : k9::linear8_rows_kernel<X, 8>;
}

int launch_k9_rows(const void* x, int x_dtype, long long ldx, const float* xs, const void* w8, const float* ws,
                   const float* bias, void* out, int out_dtype, long long ldo, int M, int N, int K, cudaStream_t stream) {
  k9::RowsParams p;
  memset(&p, 0, sizeof(p));
  p.x = x;
  p.ldx = ldx;
  p.xs = xs;
  p.w8 = static_cast<const uint8_t*>(w8);
  p.ws = ws;
  p.bias = bias;
  p.out = out;
  p.ldo = ldo;
  p.M = M;
  p.N = N;
  p.K = K;
  p.kb = (K + 127) / 128;
  p.out_type = out_dtype;
  void (*kern)(k9::RowsParams) = x_dtype == TMU_F16    ? k9_rows_kernel<__half>(M)
                                 : x_dtype == TMU_BF16 ? k9_rows_kernel<__nv_bfloat16>(M) : k9_rows_kernel<uint8_t>(M);
  cudaError_t e = launch_pdl(kern, (N + k9::kRowsN - 1) / k9::kRowsN, k9::kRowsThreads, 0, stream, p);
  return e == cudaSuccess ? TMU_OK : cuda_fail(e, "launch linear8_rows_kernel");
}

// A [rows, K] e4m3 matrix, read as bytes in boxes of box_rows rows of 128 bytes.
int encode_bytes(CUtensorMap* m, const void* base, uint64_t rows, uint64_t K, uint32_t box_rows) {
  int st = get_encoder();
  if (st) return st;
  const cuuint64_t dims[2] = {K, rows}, strides[1] = {K};
  const cuuint32_t box[2] = {128, box_rows}, es[2] = {1, 1};
  CUresult r = g_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TMU_OK : fail(TMU_ERR_DRIVER, "cuTensorMapEncodeTiled failed for an 8-bit operand");
}

// The workspace: x's scales [kb, M rounded up to 256], then x8 [M, K] where x is not e4m3 already.
size_t k9_scale_bytes(int M, int K) {
  return static_cast<size_t>((M + 255) / 256) * 256 * ((K + 127) / 128) * 4;
}

int launch_k9(const void* x8, const float* xst, int ld_xs, const void* w8, const float* ws, const float* bias, void* out,
              int out_dtype, long long ldo, int M, int N, int K, DeviceStatus* status, cudaStream_t stream) {
  Dev dev;
  int st = seq_device(dev, 8, reinterpret_cast<const void*>(&k9::linear8_kernel), k9::SMEM_BYTES);
  if (!st) st = seq_device(dev, 9, reinterpret_cast<const void*>(&k9::pair::linear8_pair_kernel), k9::pair::SMEM_BYTES);
  if (st) return st;
  k9::Params p;
  memset(&p, 0, sizeof(p));
  const long long pair_m = (M + 255) / 256, pair_tiles = pair_m * ((N + 255) / 256);
  const bool pairs_of_ctas = pair_tiles >= dev.sms && pair_tiles <= 0x7fffffffll;
  if ((st = encode_bytes(&p.tm_x, x8, M, K, k9::kTile)) ||
      (st = encode_bytes(&p.tm_w, w8, N, K, pairs_of_ctas ? k9::kTile / 2 : k9::kTile)))
    return st;
  p.xst = xst;
  p.ld_xs = ld_xs;
  p.ws = ws;
  p.bias = bias;
  p.out = out;
  p.ldo = ldo;
  p.M = M;
  p.N = N;
  p.kb = (K + 127) / 128;
  p.out_type = out_dtype;
  const int es = out_dtype == TMU_F32 ? 4 : 2;
  p.vec = aligned16(out) && ldo * es % 16 == 0;
  p.status = status;
  p.timeout_ns = g_timeout_ns;
  if (pairs_of_ctas) {
    static int max_pairs[kMaxDevices] = {0};
    if (max_pairs[dev.id] == 0) {
      const int r = max_resident_pairs(&k9::pair::linear8_pair_kernel, k9::pair::kThreads, k9::pair::SMEM_BYTES);
      max_pairs[dev.id] = r > 0 ? r : std::max(1, dev.sms / 2);
    }
    p.tiles_m = static_cast<int>(pair_m);
    const int pairs = static_cast<int>(std::min<long long>(pair_tiles, max_pairs[dev.id]));
    cudaError_t e = launch_pdl_pair(&k9::pair::linear8_pair_kernel, 2 * pairs, k9::pair::kThreads, k9::pair::SMEM_BYTES,
                                    stream, p);
    return e == cudaSuccess ? TMU_OK : cuda_fail(e, "launch linear8_pair_kernel");
  }
  p.tiles_m = (M + k9::kTile - 1) / k9::kTile;
  const long long tiles = static_cast<long long>(p.tiles_m) * ((N + k9::kTile - 1) / k9::kTile);
  // blocks of a cluster share a tile along K while the card has room for more blocks
  p.split = 1;
  while (p.split < 8 && tiles * p.split * 2 <= dev.sms && p.kb >= p.split * 4) p.split *= 2;
  if (tiles * p.split > 0x7fffffffll) return fail(TMU_ERR_UNSUPPORTED, "M and N are too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * p.split));
  cfg.blockDim = dim3(k9::kThreads);
  cfg.dynamicSmemBytes = k9::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, &k9::linear8_kernel, p);
  return e == cudaSuccess ? TMU_OK : cuda_fail(e, "launch linear8_kernel");
}

int quantize_rows(const void* x, int dtype, long long ld, int M, int K, void* x8, float* scales, long long xs_m,
                  long long xs_b, cudaStream_t stream) {
  if (M < 0 || K < 1) return fail(TMU_ERR_INVALID_ARGUMENT, "M must not be negative, K positive");
  if (M > 1 << 30 || K > 1 << 30) return fail(TMU_ERR_UNSUPPORTED, "M or K > 2^30");
  if (K % 16) return fail(TMU_ERR_UNSUPPORTED, "K must be a multiple of 16");
  if (dtype != TMU_F16 && dtype != TMU_BF16) return fail(TMU_ERR_UNSUPPORTED, "dtype must be fp16 or bf16");
  if (M == 0) return TMU_OK;
  if (!x || !x8 || !scales) return fail(TMU_ERR_INVALID_ARGUMENT, "NULL tensor");
  if (ld < K && M > 1) return fail(TMU_ERR_INVALID_ARGUMENT, "rows overlap: ld < K");
  if (!aligned16(x) || !aligned16(x8) || ld % 8) return fail(TMU_ERR_MISALIGNED, "x, x8 must be 16-byte aligned, ld a multiple of 8");
  if (!aligned_to(scales, 4)) return fail(TMU_ERR_MISALIGNED, "scales not aligned to their type");
  Dev dev;
  int st = current_device(dev, 0, nullptr, 0);
  if (st) return st;
  k9::QuantParams p;
  memset(&p, 0, sizeof(p));
  p.x = x;
  p.ld = ld;
  p.M = M;
  p.K = K;
  p.kb = (K + 127) / 128;
  p.x8 = static_cast<uint8_t*>(x8);
  p.xs = scales;
  p.xs_m = xs_m;
  p.xs_b = xs_b;
  // two blocks of 128 at a time once that still gives every SM eight blocks of threads
  const long long groups = (M + k9::kQuantRows - 1) / k9::kQuantRows;
  const bool two = groups * ((p.kb + 1) / 2) >= 8ll * dev.sms;
  const long long grid = groups * (two ? (p.kb + 1) / 2 : p.kb);
  if (grid > 0x7fffffffll) return fail(TMU_ERR_UNSUPPORTED, "M and K are too large");
  void (*kern)(k9::QuantParams) =
      dtype == TMU_F16 ? (two ? k9::quantize_kernel<__half, 2> : k9::quantize_kernel<__half, 1>)
                       : (two ? k9::quantize_kernel<__nv_bfloat16, 2> : k9::quantize_kernel<__nv_bfloat16, 1>);
  cudaError_t e = launch_pdl(kern, static_cast<int>(grid), k9::kQuantThreads, 0, stream, p);
  return e == cudaSuccess ? TMU_OK : cuda_fail(e, "launch quantize_kernel");
}

}  // namespace

extern "C" {

int tmu_sequence_status(void** status) {
  if (!status) return fail(TMU_ERR_INVALID_ARGUMENT, "NULL argument");
  cudaError_t e = cudaGetSymbolAddress(status, g_own_status);
  return e == cudaSuccess ? TMU_OK : cuda_fail(e, "cudaGetSymbolAddress");
}

int tmu_qk_norm_rope(const tmu_qk_norm_rope_args* args, void* stream) {
  if (!args) return fail(TMU_ERR_INVALID_ARGUMENT, "NULL argument");
  const tmu_heads *q = &args->q, *k = &args->k, *q_out = &args->q_out, *k_out = &args->k_out;
  const tmu_qk_norm* norm = &args->norm;
  const tmu_rotary* rot = &args->rotary;
  const int T = args->T, Hq = args->Hq, Hkv = args->Hkv, D = args->D, dtype = args->dtype;
  int st = check_packed(T, Hq, Hkv, D);
  if (st) return st;
  if (D % 16 || D > 256) return fail(TMU_ERR_UNSUPPORTED, "D must be a multiple of 16, at most 256");
  if (dtype != TMU_F16 && dtype != TMU_BF16) return fail(TMU_ERR_UNSUPPORTED, "dtype must be fp16 or bf16");
  if (norm->kind < TMU_NORM_NONE || norm->kind > TMU_NORM_LAYER) return fail(TMU_ERR_INVALID_ARGUMENT, "norm kind");
  if (norm->kind != TMU_NORM_NONE && !(norm->eps >= 0.0f && std::isfinite(norm->eps)))
    return fail(TMU_ERR_INVALID_ARGUMENT, "eps must not be negative, and finite");
  if (rot->rot < 0 || rot->rot > D || rot->rot % 16)
    return fail(TMU_ERR_UNSUPPORTED, "the rotated part must be a multiple of 16, at most D");
  if (rot->rot > 0 && (!rot->positions || !rot->turns)) return fail(TMU_ERR_INVALID_ARGUMENT, "positions or turns is NULL");
  if (rot->position_bytes != 4 && rot->position_bytes != 8) return fail(TMU_ERR_INVALID_ARGUMENT, "position_bytes must be 4 or 8");
  if (T == 0) return TMU_OK;
  const tmu_heads* views[4] = {q, k, q_out, k_out};
  static const char* const names[4] = {"q", "k", "q_out", "k_out"};
  for (int i = 0; i < 4; ++i)
    if ((st = check_heads(views[i]->data, views[i]->stride_token, views[i]->stride_head, names[i]))) return st;
  const float* par[4] = {norm->q_weight, norm->q_bias, norm->k_weight, norm->k_bias};
  for (const float* x : par)
    if (x != nullptr && !aligned16(x)) return fail(TMU_ERR_MISALIGNED, "norm parameter not 16-byte aligned");
  if (rot->rot > 0 && (!aligned_to(rot->positions, rot->position_bytes) || !aligned_to(rot->turns, 8)))
    return fail(TMU_ERR_MISALIGNED, "positions or turns not aligned to their type");
  Dev dev;
  if ((st = current_device(dev, 0, nullptr, 0))) return st;
  int lph = 2;
  while (lph * 8 < D) lph *= 2;
  k8::Params p;
  memset(&p, 0, sizeof(p));
  k8::View* dst[4] = {&p.q, &p.k, &p.qo, &p.ko};
  for (int i = 0; i < 4; ++i) *dst[i] = k8::View{views[i]->data, views[i]->stride_token, views[i]->stride_head};
  p.pos = rot->positions;
  p.pos64 = rot->position_bytes == 8;
  p.turns = rot->turns;
  p.gain = rot->gain;
  p.rot = rot->rot;
  p.qw = norm->q_weight;
  p.qb = norm->q_bias;
  p.kw = norm->k_weight;
  p.kb = norm->k_bias;
  p.eps = norm->eps;
  p.inv_d = 1.0f / static_cast<float>(D);
  p.T = T;
  p.hq = Hq;
  p.hk = Hkv;
  p.d = D;
  // turns of 32 / lph heads; split over more warps until the card has 16 warps an SM
  const int hpw = 32 / lph;
  p.q_turns = (Hq + hpw - 1) / hpw;
  p.all_turns = p.q_turns + (Hkv + hpw - 1) / hpw;
  const long long want = 16ll * dev.sms;
  const long long slices = std::min<long long>(p.all_turns, std::max<long long>(1, (want + T - 1) / T));
  p.turns_each = static_cast<int>((p.all_turns + slices - 1) / slices);
  p.slices = (p.all_turns + p.turns_each - 1) / p.turns_each;
  const long long blocks = (static_cast<long long>(T) * p.slices + k8::kThreads / 32 - 1) / (k8::kThreads / 32);
  if (blocks > 0x7fffffffll) return fail(TMU_ERR_UNSUPPORTED, "too many tokens");
  const bool inter = rot->interleaved != 0;
  void (*kern)(k8::Params) = dtype == TMU_F16 ? k8_kernel<__half>(lph, norm->kind, inter)
                                              : k8_kernel<__nv_bfloat16>(lph, norm->kind, inter);
  cudaError_t e = launch_pdl(kern, static_cast<int>(blocks), k8::kThreads, 0, static_cast<cudaStream_t>(stream), p);
  return e == cudaSuccess ? TMU_OK : cuda_fail(e, "launch qk_rope_kernel");
}

int tmu_attention(const tmu_attention_args* args, void* stream) {
  if (!args) return fail(TMU_ERR_INVALID_ARGUMENT, "NULL argument");
  const tmu_heads *q = &args->q, *k = &args->k, *v = &args->v, *out = &args->out;
  const int* cu_seqlens = args->cu_seqlens;
  const tmu_attn_bias* bias = &args->bias;
  const int S = args->S, T = args->T, Hq = args->Hq, Hkv = args->Hkv, D = args->D, dtype = args->dtype;
  const int causal = args->causal;
  const float scale = args->scale;
  void* status = args->status;
  int st = check_packed(T, Hq, Hkv, D);
  if (st) return st;
  if (S < 0) return fail(TMU_ERR_INVALID_ARGUMENT, "S must not be negative");
  if (!std::isfinite(scale)) return fail(TMU_ERR_INVALID_ARGUMENT, "scale must be finite");
  if (Hq % Hkv) return fail(TMU_ERR_INVALID_ARGUMENT, "Hq must be a multiple of Hkv");
  if (D % 8 || D > 128) return fail(TMU_ERR_UNSUPPORTED, "D must be a multiple of 8, at most 128");
  if (dtype != TMU_F16 && dtype != TMU_BF16) return fail(TMU_ERR_UNSUPPORTED, "dtype must be fp16 or bf16");
  if (T == 0 || S == 0) return TMU_OK;
  if (!cu_seqlens) return fail(TMU_ERR_INVALID_ARGUMENT, "cu_seqlens is NULL");
  const tmu_heads* views[4] = {q, k, v, out};
  static const char* const names[4] = {"q", "k", "v", "out"};
  for (int i = 0; i < 4; ++i)
    if ((st = check_heads(views[i]->data, views[i]->stride_token, views[i]->stride_head, names[i]))) return st;
  if (bias->n < 0 || (bias->n > 0 && !bias->data)) return fail(TMU_ERR_INVALID_ARGUMENT, "bias");
  if (!aligned16(status)) return fail(TMU_ERR_MISALIGNED, "status not 16-byte aligned");
  if (!aligned_to(cu_seqlens, 4) || (bias->n > 0 && !aligned_to(bias->data, 2)))
    return fail(TMU_ERR_MISALIGNED, "cu_seqlens or bias not aligned to its type");
  // a tensor map cannot step by 0
  const int heads[3] = {Hq, Hkv, Hkv};
  for (int i = 0; i < 3; ++i)
    if ((T > 1 && views[i]->stride_token == 0) || (heads[i] > 1 && views[i]->stride_head == 0))
      return fail(TMU_ERR_UNSUPPORTED, "q, k and v must not be broadcast views");
  const bool bf16 = dtype == TMU_BF16, biased = bias->n > 0;
  k7::Params p;
  memset(&p, 0, sizeof(p));
  CUtensorMap* maps[3] = {&p.tm_q, &p.tm_k, &p.tm_v};
  for (int i = 0; i < 3; ++i) {
    const uint64_t row = ((uint64_t)D * 2 + 15) / 16 * 16;
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)T, (uint64_t)heads[i]};
    const uint64_t str[2] = {T > 1 ? 2ull * views[i]->stride_token : row, heads[i] > 1 ? 2ull * views[i]->stride_head : row};
    const uint32_t box[3] = {64, (uint32_t)k7::kTile, 1};
    if ((st = encode_map(maps[i], views[i]->data, 3, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B))) return st;
  }
  k8::View* dst[4] = {&p.q, &p.k, &p.v, &p.o};
  for (int i = 0; i < 4; ++i) *dst[i] = k8::View{views[i]->data, views[i]->stride_token, views[i]->stride_head};
  p.cu = cu_seqlens;
  if (biased) {
    p.bias = bias->data;
    p.bias_ss = bias->stride_seq;
    p.bias_sh = bias->stride_head;
    p.bias_sr = bias->stride_row;
    p.bias_n = bias->n;
    // the widest copy that every row allows: 16, 8 or (with a shift of odd rows) 4 bytes
    const unsigned long long a = static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(bias->data)) |
                                 2ull * bias->stride_seq | 2ull * bias->stride_head | 2ull * bias->stride_row;
    p.bias_width = a % 16 == 0 ? 8 : a % 8 == 0 ? 4 : 2;
  }
  p.S = S;
  p.T = T;
  p.hq = Hq;
  p.group = Hq / Hkv;
  p.d = D;
  p.causal = causal != 0;
  p.scale = scale;
  p.status = static_cast<DeviceStatus*>(status);
  p.timeout_ns = g_timeout_ns;
  const int rows = D <= 64 ? k7::Cfg<64, false>::kRows : k7::Cfg<128, false>::kRows;
  const long long blocks = (static_cast<long long>(T) / rows + S) * Hq;
  if (blocks > 0x7fffffffll) return fail(TMU_ERR_UNSUPPORTED, "too many sequences and heads");
  return D <= 64 ? launch_k7<64>(p, bf16, biased, static_cast<int>(blocks), static_cast<cudaStream_t>(stream))
                 : launch_k7<128>(p, bf16, biased, static_cast<int>(blocks), static_cast<cudaStream_t>(stream));
}

int tmu_quantize_rows(const void* x, int dtype, long long ld, int M, int K, void* x8, float* scales, void* stream) {
  return quantize_rows(x, dtype, ld, M, K, x8, scales, (K + 127) / 128, 1, static_cast<cudaStream_t>(stream));
}

size_t tmu_linear_fp8_scaled_workspace_bytes(int M, int N, int K) {
  if (M <= k9::kRowsMax || M > 1 << 30 || N < 1 || K < 1 || K > 1 << 30) return 0;
  return k9_scale_bytes(M, K);
}

size_t tmu_linear_fp8_workspace_bytes(int M, int N, int K) {
  const size_t scales = tmu_linear_fp8_scaled_workspace_bytes(M, N, K);
  return scales == 0 ? 0 : scales + static_cast<size_t>(M) * K;
}

int tmu_linear_fp8(const void* x, int x_dtype, long long ldx, const float* x_scales, const void* w8, const float* w_scales,
                   const float* bias, void* out, int out_dtype, long long ldo, int M, int N, int K, void* workspace,
                   size_t workspace_bytes, void* status, void* stream) {
  if (M < 0 || N < 1 || K < 1) return fail(TMU_ERR_INVALID_ARGUMENT, "M must not be negative, N and K positive");
  if (M > 1 << 30 || N > 1 << 30 || K > 1 << 30) return fail(TMU_ERR_UNSUPPORTED, "M, N or K > 2^30");
  if (K % 16) return fail(TMU_ERR_UNSUPPORTED, "K must be a multiple of 16");
  if (x_dtype != TMU_F16 && x_dtype != TMU_BF16 && x_dtype != TMU_E4M3) return fail(TMU_ERR_UNSUPPORTED, "x must be fp16, bf16 or e4m3");
  if (out_dtype != TMU_F16 && out_dtype != TMU_BF16 && out_dtype != TMU_F32) return fail(TMU_ERR_UNSUPPORTED, "out must be fp16, bf16 or fp32");
  if (M == 0) return TMU_OK;
  if (!x || !w8 || !w_scales || !out || (x_dtype == TMU_E4M3 && !x_scales)) return fail(TMU_ERR_INVALID_ARGUMENT, "NULL tensor");
  if (ldo < N && M > 1) return fail(TMU_ERR_INVALID_ARGUMENT, "rows of out overlap: ldo < N");
  if (!aligned16(x) || !aligned16(w8)) return fail(TMU_ERR_MISALIGNED, "x, w8 must be 16-byte aligned");
  if (!aligned16(status)) return fail(TMU_ERR_MISALIGNED, "status not 16-byte aligned");
  if (!aligned_to(out, out_dtype == TMU_F32 ? 4 : 2) || !aligned_to(w_scales, 4) || !aligned_to(bias, 4) ||
      !aligned_to(x_scales, 4))
    return fail(TMU_ERR_MISALIGNED, "out, a scale or bias not aligned to its type");
  if (x_dtype == TMU_E4M3 && ldx != K) return fail(TMU_ERR_UNSUPPORTED, "e4m3 x must be contiguous");
  if (ldx % 8) return fail(TMU_ERR_MISALIGNED, "ldx must be a multiple of 8");
  if (ldx < K && M > 1) return fail(TMU_ERR_INVALID_ARGUMENT, "rows of x overlap: ldx < K");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M <= k9::kRowsMax) return launch_k9_rows(x, x_dtype, ldx, x_scales, w8, w_scales, bias, out, out_dtype, ldo, M, N, K, s);
  if (!workspace || workspace_bytes < (x_dtype == TMU_E4M3 ? tmu_linear_fp8_scaled_workspace_bytes(M, N, K)
                                                           : tmu_linear_fp8_workspace_bytes(M, N, K)))
    return fail(TMU_ERR_WORKSPACE_TOO_SMALL, "workspace too small");
  if (!aligned16(workspace)) return fail(TMU_ERR_MISALIGNED, "workspace not 16-byte aligned");
  float* xst = static_cast<float*>(workspace);
  const int ld_xs = (M + 255) / 256 * 256;
  const uint8_t* x8 = static_cast<const uint8_t*>(x);
  if (x_dtype != TMU_E4M3) {
    uint8_t* ws = static_cast<uint8_t*>(workspace) + k9_scale_bytes(M, K);
    int st = quantize_rows(x, x_dtype, ldx, M, K, ws, xst, 1, ld_xs, s);
    if (st) return st;
    x8 = ws;
  } else {
    k9::ScaleParams sp{x_scales, xst, M, (K + 127) / 128, ld_xs};
    cudaError_t e = launch_pdl(&k9::transpose_scales_kernel, (M + 255) / 256, 256, 0, s, sp);
    if (e != cudaSuccess) return cuda_fail(e, "launch transpose_scales_kernel");
  }
  return launch_k9(x8, xst, ld_xs, w8, w_scales, bias, out, out_dtype, ldo, M, N, K, static_cast<DeviceStatus*>(status), s);
}

}  // extern "C"

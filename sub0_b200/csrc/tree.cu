// Attention of drafted tokens over the compressed paged cache (tree_attention), and the weight its queries give to every
// cached key (attention_mass).
//
// With k_n, v_n the decoded rows fp16(level * norm) of key n in the rotated frame, q_r the rotated query of row r = (token t,
// query head h) and ctx = seq_len - q_len:
//   x_rn  = scale * q_r.k_n,   capped: softcap * tanh(x_rn / softcap),   plus slope_h * (pos_n - pos_t)
//   sees  = n < ctx or bit (n - ctx) of tree_mask[t] (chain: n <= ctx + t), and pos_t - pos_n < window
//   lse_r = log sum_n exp(x_rn)      out_r = H (sum_n exp(x_rn - lse_r) v_n)      mass_n += sum_r weight_t exp(x_rn - lse_r)
// pos of a context key is its place, pos of a new token ctx + depth.  A row that sees no key gives zeros and lse -inf.
#include "attend.cuh"

namespace cda {
__device__ int g_tree_status = 0;
}

#include "mass_umma.cuh"
#include "tree_umma.cuh"

#include <cmath>

namespace cda {

// ---- host side ----------------------------------------------------------------------------------------------------------
static unsigned long long g_wait_limit_ns = umma::kWaitLimitNs;   // diagnostic knobs (cda_b200_kv_debug)
static int g_withhold_first_k = 0;

static int fill_params(AttendParams& p, const char* what, const void* Q, const void* kv_cache, const int32_t* block_table,
                       const int32_t* cu_q, const int32_t* seq_lens, const float* cb_K, const int64_t* tree_mask,
                       const float* slopes, int64_t T, int B, int H_q, int H_kv, int block_size, int bt_stride, int max_q,
                       int max_n, int64_t num_slots, int slot_bytes, int k_bits, int v_bits, float scale, float softcap, int window) {
  if (T < 0 || B < 0 || H_q <= 0 || H_kv <= 0 || max_q < 0 || max_n < 0 || num_slots < 0 || window < 0)
    return fail(CDA_ERR_BAD_ARG, "%s: negative size", what);
  if (!(softcap >= 0.f) || std::isinf(softcap) || !std::isfinite(scale)) return fail(CDA_ERR_BAD_ARG, "%s: scale and softcap must be finite, softcap not negative", what);
  if (!bits_ok(k_bits) || !bits_ok(v_bits)) return fail(CDA_ERR_UNSUPPORTED, "%s: bits must be 2 or 4", what);
  if (H_q % H_kv) return fail(CDA_ERR_BAD_SHAPE, "%s: H_q=%d is not a multiple of H_kv=%d", what, H_q, H_kv);
  if (H_q / H_kv > 64) return fail(CDA_ERR_UNSUPPORTED, "%s: GQA group %d > 64", what, H_q / H_kv);
  if (slot_bytes != slot_bytes_for(k_bits, v_bits)) return fail(CDA_ERR_BAD_SHAPE, "%s: slot width %d does not fit k%dv%d", what, slot_bytes, k_bits, v_bits);
  if (block_size <= 0 || block_size % 16) return fail(CDA_ERR_BAD_SHAPE, "%s: block_size=%d is not a multiple of 16", what, block_size);
  if (static_cast<int64_t>(bt_stride) * block_size < max_n) return fail(CDA_ERR_BAD_SHAPE, "%s: block table row shorter than max_seq_len", what);
  if (tree_mask && max_q > 64) return fail(CDA_ERR_UNSUPPORTED, "%s: a tree has at most 64 tokens, max_query_len is %d", what, max_q);
  if (max_n > 0x7fff0000) return fail(CDA_ERR_N_TOO_LARGE, "%s: max_seq_len %d is too large", what, max_n);
  if (num_slots > 0x7fffffffll) return fail(CDA_ERR_N_TOO_LARGE, "%s: too many slots", what);
  // (a row's token is found by a product with 2^32 / group, exact below 2^26 rows)
  if (static_cast<int64_t>(max_q) * (H_q / H_kv) > 1ll << 26) return fail(CDA_ERR_N_TOO_LARGE, "%s: %d new tokens of %d query heads a KV head are too many", what, max_q, H_q / H_kv);
  if (B == 0 || T == 0 || max_q == 0 || max_n == 0) return 1;
  if (num_slots < block_size) return fail(CDA_ERR_BAD_SHAPE, "%s: the cache holds no block", what);
  if (!Q || !kv_cache || !block_table || !cu_q || !seq_lens || !cb_K) return fail(CDA_ERR_BAD_ARG, "%s: null pointer", what);
  if (!aligned16(Q) || !aligned16(kv_cache)) return fail(CDA_ERR_BAD_ALIGN, "%s: Q and cache must be 16-byte aligned", what);
  p.q = static_cast<const __half*>(Q);
  p.cache = static_cast<const uint8_t*>(kv_cache);
  p.block_table = block_table; p.cu_q = cu_q; p.seq_lens = seq_lens; p.cb_k = cb_K; p.tree_mask = tree_mask; p.slopes = slopes;
  p.T = T; p.B = B; p.H_q = H_q; p.H_kv = H_kv; p.group = H_q / H_kv; p.block_size = block_size; p.bt_stride = bt_stride;
  p.bs_shift = -1;
  for (int sft = 4; sft < 31; ++sft) if ((1 << sft) == block_size) p.bs_shift = sft;
  p.num_blocks = static_cast<int>(num_slots / block_size);
  p.max_q = max_q; p.max_n = max_n; p.k_bits = k_bits; p.v_bits = v_bits; p.slot_bytes = slot_bytes;
  p.scale = scale; p.softcap = softcap; p.window = window;
  p.wait_limit_ns = g_wait_limit_ns; p.withhold = g_withhold_first_k;
  return CDA_OK;
}

}  // namespace cda

using namespace cda;

namespace cda {
// Rows of a block: the smallest of 16, 32, 64, 128 that holds all rows of the longest chunk, else 128.  A block expands every tile
// of keys once, so fewer, larger blocks win as soon as their columns are filled (512 rows a sequence: 705 us in blocks of 128,
// 966 us in blocks of 64).
static int rows_per_block(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

static size_t tree_workspace(int NR, int ctas) {
  return static_cast<size_t>(ctas) * sizeof(tru::Record) + static_cast<size_t>(2) * ctas * NR * (kHeadDim + 2) * sizeof(float);
}

template <int NR>
static int launch_tree(AttendParams& p, void* ws, int ctas, const CUtensorMap& map, cudaStream_t st) {
  static bool configured[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(tru::tree_attention_kernel<NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, tru::Cfg<NR>::kSmemBytes) != cudaSuccess)
      return check_launch("tree_attention: shared memory opt-in");
    cudaFuncAttributes attr;                                    // the warps share out the launch's registers; more would be waited for in vain
    if (cudaFuncGetAttributes(&attr, tru::tree_attention_kernel<NR>) != cudaSuccess) return check_launch("tree_attention: attributes");
    if (attr.numRegs * tru::Cfg<NR>::kThreads < tru::Cfg<NR>::kRegsAll) return fail(CDA_ERR_UNSUPPORTED, "tree_attention: built with %d registers a thread, too few", attr.numRegs);
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  tru::tree_attention_kernel<NR><<<ctas, tru::Cfg<NR>::kThreads, tru::Cfg<NR>::kSmemBytes, st>>>(p, ws, map);
  const int rc = check_launch("tree_attention");
  if (rc != CDA_OK) return rc;
  // the merge starts before the first kernel ends (its blocks wait there): its launch costs no time of its own
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, NR / 8);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, tru::tree_merge_kernel<NR>, const_cast<const AttendParams&>(p), ws, ctas) != cudaSuccess) return check_launch("tree_attention: merge");
  return CDA_OK;
}

template <int NR>
static int launch_mass(const AttendParams& p, const CUtensorMap& map, cudaStream_t st) {
  using C = msu::MassCfg<NR>;
  static bool configured[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(msu::attention_mass_kernel<NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes) != cudaSuccess)
      return check_launch("attention_mass: shared memory opt-in");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  msu::attention_mass_kernel<NR><<<device_sm_count(-1), C::kThreads, C::kSmemBytes, st>>>(p, map);
  return check_launch("attention_mass");
}
}  // namespace cda

extern "C" size_t cda_b200_tree_attention_workspace_bytes(int H_q, int H_kv, int max_query_len, int device) {
  if (H_q <= 0 || H_kv <= 0 || max_query_len < 0) return 0;
  return tree_workspace(rows_per_block(static_cast<int64_t>(max_query_len) * (H_q / H_kv)), device_sm_count(device));
}

extern "C" int cda_b200_tree_attention(const void* Q, const void* kv_cache, const int32_t* block_table, const int32_t* cu_seqlens_q,
                                       const int32_t* seq_lens, const float* cb_K, const float* cb_V, const int64_t* tree_mask,
                                       const float* alibi_slopes, void* out, float* lse, void* workspace, size_t workspace_bytes,
                                       int64_t T, int B, int H_q, int H_kv, int block_size, int block_table_stride, int max_query_len,
                                       int max_seq_len, int64_t num_slots, int slot_bytes, int k_bits, int v_bits, float scale,
                                       float softcap, int window, void* stream) {
  AttendParams p{};
  const int rc = fill_params(p, "tree_attention", Q, kv_cache, block_table, cu_seqlens_q, seq_lens, cb_K, tree_mask, alibi_slopes, T, B,
                             H_q, H_kv, block_size, block_table_stride, max_query_len, max_seq_len, num_slots, slot_bytes, k_bits,
                             v_bits, scale, softcap, window);
  if (rc == 1) return CDA_OK;
  if (rc != CDA_OK) return rc;
  if (!cb_V || !out) return fail(CDA_ERR_BAD_ARG, "tree_attention: null pointer");
  if (!aligned16(out)) return fail(CDA_ERR_BAD_ALIGN, "tree_attention: out must be 16-byte aligned");
  if (workspace_bytes < cda_b200_tree_attention_workspace_bytes(H_q, H_kv, max_query_len, -1) || !workspace)
    return fail(CDA_ERR_WORKSPACE, "tree_attention: workspace of %zu bytes, need %zu", workspace_bytes,
                cda_b200_tree_attention_workspace_bytes(H_q, H_kv, max_query_len, -1));
  if (!aligned16(workspace)) return fail(CDA_ERR_BAD_ALIGN, "tree_attention: workspace must be 16-byte aligned");
  p.cb_v = cb_V; p.out = static_cast<__half*>(out); p.lse_out = lse;
  const int ctas = device_sm_count(-1);
  const int64_t rows = static_cast<int64_t>(max_query_len) * p.group;
  const int NR = rows_per_block(rows);
  const int64_t blocks = (rows + NR - 1) / NR;
  if (blocks * B * H_kv * ((max_seq_len + 127) / 128) > 0x7fffffffll)
    return fail(CDA_ERR_N_TOO_LARGE, "tree_attention: %d sequences of %d new and %d old tokens are too many tiles for one call", B, max_query_len, max_seq_len);
  p.row_blocks = static_cast<int>(blocks);
  p.group_magic = static_cast<uint32_t>(((1ull << 32) + p.group - 1) / p.group);
  CUtensorMap map;
  if (const int map_rc = make_cache_map("tree_attention", kv_cache, H_kv, slot_bytes, static_cast<int64_t>(p.num_blocks) * block_size, slot_bytes, &map)) return map_rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (NR) {
    case 16: return launch_tree<16>(p, workspace, ctas, map, st);
    case 32: return launch_tree<32>(p, workspace, ctas, map, st);
    case 64: return launch_tree<64>(p, workspace, ctas, map, st);
    default: return launch_tree<128>(p, workspace, ctas, map, st);
  }
}

extern "C" int cda_b200_attention_mass(const void* Q, const void* kv_cache, const int32_t* block_table, const int32_t* cu_seqlens_q,
                                       const int32_t* seq_lens, const float* cb_K, const int64_t* tree_mask, const float* alibi_slopes,
                                       const float* lse, const float* weights, float* mass, int64_t mass_stride, int64_t T, int B, int H_q,
                                       int H_kv, int block_size, int block_table_stride, int max_query_len, int max_seq_len,
                                       int64_t num_slots, int slot_bytes, int k_bits, int v_bits, float scale, float softcap, int window,
                                       void* stream) {
  AttendParams p{};
  const int rc = fill_params(p, "attention_mass", Q, kv_cache, block_table, cu_seqlens_q, seq_lens, cb_K, tree_mask, alibi_slopes, T, B,
                             H_q, H_kv, block_size, block_table_stride, max_query_len, max_seq_len, num_slots, slot_bytes, k_bits,
                             v_bits, scale, softcap, window);
  if (rc == 1) return CDA_OK;
  if (rc != CDA_OK) return rc;
  if (!lse || !mass) return fail(CDA_ERR_BAD_ARG, "attention_mass: null pointer");
  if (mass_stride < max_seq_len) return fail(CDA_ERR_BAD_SHAPE, "attention_mass: rows of %lld weights, max_seq_len is %d", static_cast<long long>(mass_stride), max_seq_len);
  p.lse = lse; p.weights = weights; p.mass = mass; p.mass_stride = mass_stride;
  for (p.side = H_kv < 8 ? H_kv : 8; H_kv % p.side; ) --p.side;
  const int64_t rows = static_cast<int64_t>(max_query_len) * p.group;
  if ((rows + 15) / 16 * B * H_kv * ((max_seq_len + 127) / 128) > 0x7fffffffll)
    return fail(CDA_ERR_N_TOO_LARGE, "attention_mass: %d sequences of %d new and %d old tokens are too many tiles for one call", B, max_query_len, max_seq_len);
  CUtensorMap map;
  if (const int map_rc = make_cache_map("attention_mass", kv_cache, H_kv, slot_bytes, static_cast<int64_t>(p.num_blocks) * block_size, slot_bytes, &map)) return map_rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // the fewest columns that hold a chunk's rows: a block of more costs the tensor cores and the exponentials as many columns,
  // a block of fewer another pass of the K producers over all tiles
  return rows <= 16 ? launch_mass<16>(p, map, st) : rows <= 64 ? launch_mass<64>(p, map, st) : launch_mass<128>(p, map, st);
}

extern "C" int cda_b200_kv_debug(int wait_limit_us, int withhold_first_k_arrive) {
  g_wait_limit_ns = wait_limit_us > 0 ? static_cast<unsigned long long>(wait_limit_us) * 1000ull : umma::kWaitLimitNs;
  g_withhold_first_k = withhold_first_k_arrive ? 1 : 0;
  return CDA_OK;
}

namespace cda {
int tree_status(bool clear, int* value) {
  const int zero = 0;
  const cudaError_t e = clear ? cudaMemcpyToSymbol(g_tree_status, &zero, sizeof(int)) : cudaMemcpyFromSymbol(value, g_tree_status, sizeof(int));
  return e == cudaSuccess ? CDA_OK : check_launch("kv_status");
}
}  // namespace cda

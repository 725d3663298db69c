// What the attention kernels over short query chunks (tree_attention, attention_mass) share: their arguments, the checks of
// a sequence's lengths, and the rule that says which key a query row sees and with which bias.
#pragma once
#include "common.cuh"

namespace cda {

// Status bits (cda_b200_kv_status): a block-table entry outside the cache, a bounded wait that gave up, lengths that do not
// fit (more new tokens than tokens, more than the call's maximum, beyond the block table), a refused entry of a keep list.
constexpr int kStatusBadBlock = 1, kStatusWait = 4, kStatusLengths = 8, kStatusKeep = 16;

struct AttendParams {
  const __half* q;
  const uint8_t* cache;
  const int32_t* block_table;
  const int32_t* cu_q;
  const int32_t* seq_lens;
  const float* cb_k;
  const float* cb_v;
  const int64_t* tree_mask;      // (T) ancestor bits, or null: a causal chain
  const float* slopes;           // (H_q) or null
  __half* out;                   // tree_attention
  float* lse_out;                // tree_attention: optional (T, H_q)
  const float* lse;              // attention_mass: (T, H_q)
  const float* weights;          // attention_mass: optional (T)
  float* mass;                   // attention_mass: (B, H_kv, mass_stride), added to
  int64_t mass_stride;
  int64_t T;
  int B, H_q, H_kv, group, block_size, bs_shift, bt_stride, num_blocks, max_q, max_n, k_bits, v_bits, slot_bytes;
  int side;                      // attention_mass: KV heads that neighbouring CTAs walk together
  int row_blocks;                // row blocks per sequence
  uint32_t group_magic;          // ceil(2^32 / group): row / group = umulhi(row, magic) for rows below 2^26
  float scale, softcap;          // softcap 0: none
  int window;                    // 0: none
  int withhold;                  // diagnostic: CTA 0 waits for a signal too many of its first K tile
  unsigned long long wait_limit_ns;
};

__device__ __forceinline__ int withheld(const AttendParams& p, int k_buffer) { return p.withhold && k_buffer == 0 && blockIdx.x == 0; }

// The lengths of sequence b; q_len = 0 when there is nothing to do or the lengths do not fit the call (`bad`).
struct SequenceView { int q_begin, q_len, seq_len; bool bad; };
__device__ __forceinline__ SequenceView sequence_view(const AttendParams& p, int b) {
  const int lo = p.cu_q[b], hi = p.cu_q[b + 1], n = p.seq_lens[b];
  SequenceView s{lo, hi - lo, n, false};
  if (lo < 0 || hi < lo || hi > p.T || hi - lo > p.max_q || n < hi - lo || n > p.max_n) {
    s.q_len = 0;
    s.bad = true;
  }
  return s;
}

// Position of new token t: the context before the chunk plus its depth -- its place in a chain, the number of its
// ancestors in a tree.
__device__ __forceinline__ int depth_of(const AttendParams& p, int q_begin, int t) {
  return p.tree_mask ? max(__popcll(static_cast<unsigned long long>(p.tree_mask[q_begin + t])) - 1, 0) : t;
}

// How many positions, from the context's end on, new tokens may stand at: a mask's bits at and above q_len name no token, but
// they count for the depth (63 at most).
__device__ __forceinline__ int positions_of(const AttendParams& p, int q_len) { return p.tree_mask ? 64 : q_len; }

// tanh for capped scores.  tanh.approx is off by up to 2^-11, which on a score near a cap of 50 is 0.02 and on its
// probability 2 %, so: below 0.55 the odd Taylor series to x^15 (truncation below 5e-8 of the value), above it 1 - 2 / (e^2x +
// 1), where the two approximate instructions leave less than 2^-22.
__device__ __forceinline__ float soft_tanh(float x) {
  const float ax = fabsf(x), x2 = x * x;
  float t = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -929569.0f / 638512875.0f, 21844.0f / 6081075.0f), -1382.0f / 155925.0f), 62.0f / 2835.0f), -17.0f / 315.0f), 2.0f / 15.0f);
  t = x * fmaf(x2, fmaf(x2, t, -1.0f / 3.0f), 1.0f);
  if (ax >= 0.55f) {
    const float e = fast_exp2(2.0f * kLog2e * fminf(ax, 20.0f));
    t = copysignf(1.0f - __fdividef(2.0f, e + 1.0f), x);
  }
  return t;
}

}  // namespace cda

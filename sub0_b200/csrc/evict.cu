// Eviction from the compressed paged cache: which keys of every (sequence, KV head) to keep by their accumulated attention
// weight (select_keys), and the move of the kept slots to the front of the sequence's pages (compact_cache).
#include "attend.cuh"

namespace cda {

__device__ int g_evict_status = 0;
int tree_status(bool clear, int* value);   // tree.cu

// ---- select -----------------------------------------------------------------------------------------------------------
// Kept of a row of n weights, when n > budget: the first `sink`, the last `recent`, and of the others the budget - sink -
// recent largest, ties to the lower index.  The threshold is found by radix selection over the ordered bit patterns.
constexpr int kSelectThreads = 512, kDigitBits = 11, kBins = 1 << kDigitBits;

// Larger weights have larger keys; -0 counts as 0 and NaN as minus infinity, like any value below every other.
__device__ __forceinline__ uint32_t weight_key(float x) {
  x = isnan(x) ? -INFINITY : x + 0.0f;
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix sum of one value per thread over the CTA; returns the total through `total`.
__device__ __forceinline__ int block_exclusive_scan(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
  }
  __syncthreads();
  return before + x - v;
}

__global__ void __launch_bounds__(kSelectThreads) select_keys_kernel(const float* __restrict__ mass, const int32_t* __restrict__ seq_lens,
                                                                     int32_t* __restrict__ keep, int32_t* __restrict__ new_lens, int H,
                                                                     int64_t stride, int budget, int sink, int recent) {
  __shared__ int s_hist[kBins], s_warp[kSelectThreads / 32], s_digit, s_left;
  const int tid = threadIdx.x, b = blockIdx.x / H;
  const int64_t row = blockIdx.x;
  int n = seq_lens[b];
  if (n > stride) {
    if (tid == 0) atomicOr(&g_evict_status, kStatusLengths);
    n = static_cast<int>(stride);
  }
  n = max(n, 0);
  int32_t* out = keep + row * budget;
  if (tid == 0 && blockIdx.x % H == 0) new_lens[b] = min(n, budget);
  if (n <= budget) {
    for (int i = tid; i < budget; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const float* w = mass + row * stride;
  const int lo = sink, hi = n - recent;
  int left = budget - sink - recent;             // how many of [lo, hi) are kept
  uint32_t prefix = 0, prefix_mask = 0;
  if (left > 0) {
    for (int shift = 32 - kDigitBits, bits = kDigitBits;; ) {
      for (int i = tid; i < kBins; i += kSelectThreads) s_hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelectThreads) {
        const uint32_t k = weight_key(w[i]);
        if ((k & prefix_mask) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1 << bits) - 1)], 1);
      }
      __syncthreads();
      // bins from the top: thread t owns bins kBins - 1 - 4t .. kBins - 4 - 4t
      constexpr int kOwn = kBins / kSelectThreads;
      int c[kOwn], sum = 0, total;
#pragma unroll
      for (int j = 0; j < kOwn; ++j) sum += c[j] = s_hist[kBins - 1 - kOwn * tid - j];
      int above = block_exclusive_scan(sum, s_warp, total);
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        if (above < left && left <= above + c[j]) { s_digit = kBins - 1 - kOwn * tid - j; s_left = left - above; }
        above += c[j];
      }
      __syncthreads();
      left = s_left;
      prefix |= static_cast<uint32_t>(s_digit) << shift;
      prefix_mask |= ((1u << bits) - 1u) << shift;
      __syncthreads();
      if (shift == 0) break;
      bits = shift < kDigitBits ? shift : kDigitBits;
      shift -= bits;
    }
  }
  // `prefix` is the key of the smallest kept weight, `left` how many weights equal to it are kept, lowest index first
  for (int i = tid; i < sink; i += kSelectThreads) out[i] = i;
  for (int i = tid; i < recent; i += kSelectThreads) out[budget - recent + i] = hi + i;
  const bool any = budget - sink - recent > 0;
  int at = sink, equal = 0;
  for (int i0 = lo; any && i0 < hi; i0 += kSelectThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < hi ? weight_key(w[i]) : 0u;
    const bool eq = i < hi && k == prefix;
    int eq_total, total;
    const int rank = equal + block_exclusive_scan(eq ? 1 : 0, s_warp, eq_total);
    const bool take = i < hi && (k > prefix || (eq && rank < left));
    const int pos = at + block_exclusive_scan(take ? 1 : 0, s_warp, total);
    if (take) out[pos] = i;
    at += total;
    equal += eq_total;
  }
}

// ---- compact ----------------------------------------------------------------------------------------------------------
// Entry i of a list moves the slot of token keep[i] to token start + i.  Every entry must point at or behind its
// destination, so that slots may be moved in place a step at a time: what a step reads lies at or behind the first place
// it writes, i.e. behind everything that earlier steps wrote.
constexpr int kCompactThreads = 256;

struct CompactParams {
  uint8_t* cache;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const int32_t* keep;
  const int32_t* start;     // (B) or null: 0
  float* mass;              // (B, H, mass_stride) or null
  int64_t mass_stride;
  int B, H, K, block_size, bt_stride, num_blocks, slot_bytes;
  int keep_shared;          // one list for all KV heads
};

__global__ void __launch_bounds__(kCompactThreads) compact_cache_kernel(const CompactParams p) {
  const int tid = threadIdx.x, b = blockIdx.y, h = blockIdx.x;
  const int n = min(static_cast<int64_t>(p.seq_lens[b]), static_cast<int64_t>(p.bt_stride) * p.block_size);
  const int start = p.start ? p.start[b] : 0;
  const int32_t* list = p.keep + (p.keep_shared ? static_cast<int64_t>(b) : static_cast<int64_t>(b) * p.H + h) * p.K;
  float* mass = p.mass ? p.mass + (static_cast<int64_t>(b) * p.H + h) * p.mass_stride : nullptr;
  if (start < 0) {
    if (tid == 0) atomicOr(&g_evict_status, kStatusKeep);
    return;
  }
  auto slot = [&](int t) -> uint8_t* {
    const int blk = p.block_table[static_cast<int64_t>(b) * p.bt_stride + t / p.block_size];
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(p.num_blocks)) { atomicOr(&g_evict_status, kStatusBadBlock); return nullptr; }
    return p.cache + ((static_cast<int64_t>(blk) * p.block_size + t % p.block_size) * p.H + h) * p.slot_bytes;
  };
  for (int i0 = 0; i0 < p.K; i0 += kCompactThreads) {
    const int i = i0 + tid;
    uint4 row[9];
    float m = 0.f;
    uint8_t* to = nullptr;
    if (i < p.K) {
      const int src = list[i];
      const int64_t dst = static_cast<int64_t>(start) + i;
      if (src >= 0 && (src < dst || src >= n)) atomicOr(&g_evict_status, kStatusKeep);
      else if (src >= 0) {
        const uint8_t* from = slot(src);
        if (from && src != dst) {
          to = slot(static_cast<int>(dst));
          if (to)
            for (int c = 0; c < 9; ++c)
              if (16 * c < p.slot_bytes) row[c] = *reinterpret_cast<const uint4*>(from + 16 * c);
        }
        if (mass && src < p.mass_stride) m = mass[src];
      }
    }
    __syncthreads();
    if (to)
      for (int c = 0; c < 9; ++c)
        if (16 * c < p.slot_bytes) *reinterpret_cast<uint4*>(to + 16 * c) = row[c];
    if (mass && i < p.K && static_cast<int64_t>(start) + i < p.mass_stride) mass[start + i] = m;
    __syncthreads();
  }
  if (mass)
    for (int64_t t = static_cast<int64_t>(start) + p.K + tid; t < n && t < p.mass_stride; t += kCompactThreads) mass[t] = 0.f;
}

}  // namespace cda

using namespace cda;

extern "C" int cda_b200_select_keys(const float* mass, const int32_t* seq_lens, int32_t* keep, int32_t* new_lens, int B, int H_kv,
                                    int64_t mass_stride, int budget, int sink, int recent, void* stream) {
  if (B < 0 || H_kv <= 0 || mass_stride < 0 || budget <= 0 || sink < 0 || recent < 0) return fail(CDA_ERR_BAD_ARG, "select_keys: negative size or no budget");
  if (static_cast<int64_t>(sink) + recent > budget) return fail(CDA_ERR_BAD_SHAPE, "select_keys: sink %d + recent %d exceed the budget %d", sink, recent, budget);
  if (mass_stride > 0x7fffffffll || static_cast<int64_t>(B) * H_kv > 0x7fffffffll / 8) return fail(CDA_ERR_N_TOO_LARGE, "select_keys: too many weights or rows");
  if (B == 0) return CDA_OK;
  if (!mass || !seq_lens || !keep || !new_lens) return fail(CDA_ERR_BAD_ARG, "select_keys: null pointer");
  select_keys_kernel<<<B * H_kv, kSelectThreads, 0, static_cast<cudaStream_t>(stream)>>>(mass, seq_lens, keep, new_lens, H_kv, mass_stride, budget, sink, recent);
  return check_launch("select_keys");
}

extern "C" int cda_b200_compact_cache(void* kv_cache, const int32_t* block_table, const int32_t* seq_lens, const int32_t* keep,
                                      const int32_t* start, float* mass, int64_t mass_stride, int B, int H_kv, int K, int keep_heads,
                                      int block_size, int block_table_stride, int64_t num_slots, int slot_bytes, void* stream) {
  if (B < 0 || H_kv <= 0 || K < 0 || num_slots < 0 || block_table_stride < 0 || (mass && mass_stride < 0)) return fail(CDA_ERR_BAD_ARG, "compact_cache: negative size");
  if (slot_bytes != 144 && slot_bytes != 112 && slot_bytes != 80) return fail(CDA_ERR_BAD_SHAPE, "compact_cache: slot width %d is none of 144, 112, 80", slot_bytes);
  if (block_size <= 0 || block_size % 16) return fail(CDA_ERR_BAD_SHAPE, "compact_cache: block_size=%d is not a multiple of 16", block_size);
  if (keep_heads != 1 && keep_heads != H_kv) return fail(CDA_ERR_BAD_SHAPE, "compact_cache: keep has %d heads, the cache %d", keep_heads, H_kv);
  if (num_slots / block_size > 0x7fffffffll || B > 65535) return fail(CDA_ERR_N_TOO_LARGE, "compact_cache: too many slots or sequences");
  if (B == 0 || (K == 0 && !mass)) return CDA_OK;
  if (!kv_cache || !block_table || !seq_lens || (K > 0 && !keep)) return fail(CDA_ERR_BAD_ARG, "compact_cache: null pointer");
  if (!aligned16(kv_cache)) return fail(CDA_ERR_BAD_ALIGN, "compact_cache: cache must be 16-byte aligned");
  const CompactParams p{static_cast<uint8_t*>(kv_cache), block_table, seq_lens, keep, start, mass, mass_stride, B, H_kv, K, block_size,
                        block_table_stride, static_cast<int>(num_slots / block_size), slot_bytes, keep_heads == 1 ? 1 : 0};
  compact_cache_kernel<<<dim3(H_kv, B), kCompactThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("compact_cache");
}

extern "C" int cda_b200_kv_status(void) {
  int v = 0, t = 0;
  if (cudaMemcpyFromSymbol(&v, g_evict_status, sizeof(int)) != cudaSuccess) return check_launch("kv_status");
  const int rc = tree_status(false, &t);
  return rc != CDA_OK ? rc : (v | t) & 0x7fffffff;
}

extern "C" int cda_b200_kv_clear_status(void) {
  const int zero = 0;
  if (cudaMemcpyToSymbol(g_evict_status, &zero, sizeof(int)) != cudaSuccess) return check_launch("kv_clear_status");
  return tree_status(true, nullptr);
}

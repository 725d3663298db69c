// Eviction from the compressed paged cache: which keys of every (sequence, KV head) to keep by their accumulated attention
// weight (select_keys), and the move of the kept slots to the front of the sequence's pages (compact_cache).
#include "attend.cuh"

namespace cda {

__device__ int g_evict_status = 0;
int tree_status(bool clear, int* value);   // tree.cu

// ---- thread-block clusters ------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ int4 remote_int4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ int2 remote_int2(uint32_t addr) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// ---- select -----------------------------------------------------------------------------------------------------------
// Kept of a row of n weights, when n > budget: the first `sink`, the last `recent`, and of the others the budget - sink -
// recent largest, ties to the lower index.  A cluster of CTAs serves one row, a contiguous slice of it each: the slice is read
// once and kept in shared memory as ordered keys (slices too long for it are read again in every pass); the threshold is found
// by radix selection, 11 + 11 + 10 bits, with the CTAs' histograms added up over distributed shared memory; then every warp
// counts and writes what it keeps of its part in ascending order.  Reading the row once is the floor (256 rows of 65536: 67 MB,
// 10 us; measured 101 us: two CTAs of 16384 keys fit an SM, a CTA takes 26 us -- 3.4 for the first pass over its keys, 2.5 for each
// of the other two, 1.7 to count, 4.1 to write, the rest in barriers, remote bins and scans -- and there are 3.5 rounds of them;
// with 1024 threads a CTA 129 us).
constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32, kBins = 1 << 11;
constexpr int kSliceMax = 32768;                  // keys in shared memory (128 KB)

// Larger weights have larger keys; -0 counts as 0 and NaN as minus infinity, like any value below every other.
__device__ __forceinline__ uint32_t weight_key(float x) {
  x = isnan(x) ? -INFINITY : x + 0.0f;
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Exclusive prefix sum of one value per thread over the CTA.
__device__ __forceinline__ int block_exclusive_scan(int v, int* s_warp) {
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
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) before += w < warp ? s_warp[w] : 0;
  return before + x - v;
}

__global__ void __launch_bounds__(kSelectThreads) select_keys_kernel(const float* __restrict__ mass, const int32_t* __restrict__ seq_lens,
                                                                     int32_t* __restrict__ keep, int32_t* __restrict__ new_lens, int H,
                                                                     int64_t stride, int budget, int sink, int recent, int cached) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ __align__(16) int s_hist[3][kBins];
  __shared__ int s_warp[3][kSelectWarps], s_digit, s_left;
  __shared__ __align__(8) int2 s_count, s_part[kSelectWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int64_t row = blockIdx.x / ranks;
  const int b = static_cast<int>(row / H);
  int n = seq_lens[b];
  if (n > stride) {
    if (tid == 0 && rank == 0) atomicOr(&g_evict_status, kStatusLengths);
    n = static_cast<int>(stride);
  }
  n = max(n, 0);
  int32_t* out = keep + row * budget;
  if (tid == 0 && rank == 0 && row % H == 0) new_lens[b] = min(n, budget);
  const int first = rank * kSelectThreads + tid, hop = ranks * kSelectThreads;      // this thread's share of plain writes
  if (n <= budget) {                              // (the same for all CTAs of the cluster)
    for (int i = first; i < budget; i += hop) out[i] = i < n ? i : -1;
    return;
  }
  const float* w = mass + row * stride;
  const int lo = sink, hi = n - recent, wanted = budget - sink - recent;
  for (int i = first; i < sink; i += hop) out[i] = i;
  for (int i = first; i < recent; i += hop) out[budget - recent + i] = hi + i;
  if (wanted == 0) return;
  // slices of whole warps' worth, so that the order of ranks and warps is the order of the keys
  const int slice = ((hi - lo + static_cast<int>(ranks) - 1) / static_cast<int>(ranks) + 511) / 512 * 512;
  const int s0 = min(lo + static_cast<int>(rank) * slice, hi), s1 = min(s0 + slice, hi);
  const bool in_shared = cached >= slice;
  for (int i = tid; i < 3 * kBins; i += kSelectThreads) s_hist[0][i] = 0;
  __syncthreads();
  auto key_at = [&](int i) { return in_shared ? s_keys[i - s0] : weight_key(w[i]); };
  uint32_t prefix = 0, prefix_mask = 0;
  int left = wanted;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    constexpr int kBatch = 16;                    // keys of a thread in flight
    for (int i0 = s0 + tid; i0 < s1; i0 += kBatch * kSelectThreads) {
      uint32_t k[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kSelectThreads;
        if (i < s1) k[u] = pass == 0 ? __float_as_uint(w[i]) : key_at(i);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = i0 + u * kSelectThreads;
        if (i >= s1) break;
        if (pass == 0) {
          k[u] = weight_key(__uint_as_float(k[u]));
          if (in_shared) s_keys[i - s0] = k[u];
        }
        if ((k[u] & prefix_mask) == prefix) atomicAdd(&s_hist[pass][(k[u] >> shift) & ((1 << bits) - 1)], 1);
      }
    }
    if (ranks > 1) cluster_sync();
    else __syncthreads();
    // bins from the top: thread t owns bins kBins - 4 - 4 t .. kBins - 1 - 4 t
    static_assert(kBins == 4 * kSelectThreads, "four bins a thread");
    const int bin0 = kBins - 4 - 4 * tid;
    int4 c = *reinterpret_cast<const int4*>(&s_hist[pass][bin0]);
    if (ranks > 1) {
      int4 v[7];                                  // the other CTAs' bins, all in flight together
#pragma unroll
      for (uint32_t r = 1; r < 8; ++r)
        if (r < ranks) v[r - 1] = remote_int4(remote(smem_addr(&s_hist[pass][bin0]), (rank + r) & (ranks - 1)));
#pragma unroll
      for (uint32_t r = 1; r < 8; ++r)
        if (r < ranks) { c.x += v[r - 1].x; c.y += v[r - 1].y; c.z += v[r - 1].z; c.w += v[r - 1].w; }
    }
    int above = block_exclusive_scan(c.x + c.y + c.z + c.w, s_warp[pass]);
    const int counts[4] = {c.w, c.z, c.y, c.x};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (above < left && left <= above + counts[j]) { s_digit = bin0 + 3 - j; s_left = left - above; }
      above += counts[j];
    }
    __syncthreads();
    left = s_left;
    prefix |= static_cast<uint32_t>(s_digit) << shift;
    prefix_mask |= ((1u << bits) - 1u) << shift;
    __syncthreads();
  }
  // `prefix` is the key of the smallest kept weight, `left` how many weights equal to it are kept, lowest index first.  A warp
  // has a contiguous part of the slice.
  const int part = slice / kSelectWarps, p0 = min(s0 + warp * part, s1), p1 = min(p0 + part, s1);
  int above = 0, equal = 0;
  for (int i0 = p0 + lane; i0 < p1; i0 += 256) {
    uint32_t k[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) k[u] = i0 + 32 * u < p1 ? key_at(i0 + 32 * u) : 0u;
#pragma unroll
    for (int u = 0; u < 8; ++u) {                 // (the key 0 is no weight's)
      above += k[u] > prefix;
      equal += k[u] == prefix;
    }
  }
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) s_part[warp] = make_int2(above, equal);
  __syncthreads();
  int2 before = make_int2(0, 0), all = make_int2(0, 0);
#pragma unroll
  for (int u = 0; u < kSelectWarps; ++u) {
    const int2 v = s_part[u];
    if (u < warp) { before.x += v.x; before.y += v.y; }
    all.x += v.x;
    all.y += v.y;
  }
  if (ranks > 1) {
    if (tid == 0) s_count = all;
    cluster_sync();
    for (uint32_t r = 0; r < rank; ++r) {
      const int2 v = remote_int2(remote(smem_addr(&s_count), r));
      before.x += v.x;
      before.y += v.y;
    }
  }
  int at = sink + before.x + min(before.y, left), eq_seen = before.y;      // kept and equal ones in front of this warp's part
  const uint32_t lower = (1u << lane) - 1u;
  for (int i0 = p0; i0 < p1; i0 += 128) {         // 128 keys at a time, loads first
    uint32_t k[4], eq[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) k[u] = i0 + 32 * u + lane < p1 ? key_at(i0 + 32 * u + lane) : 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u) eq[u] = __ballot_sync(0xffffffffu, k[u] == prefix);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      bool take = k[u] > prefix;
      if (eq[u]) {                                // some at the threshold: the first `left` of the row
        take = take || (k[u] == prefix && eq_seen + __popc(eq[u] & lower) < left);
        eq_seen += __popc(eq[u]);
      }
      const uint32_t taken = __ballot_sync(0xffffffffu, take);
      if (take) out[at + __popc(taken & lower)] = i0 + 32 * u + lane;
      at += __popc(taken);
    }
  }
  if (ranks > 1) cluster_sync();                  // nobody leaves while its shared memory may be read
}

// ---- compact ----------------------------------------------------------------------------------------------------------
// Entry i of a list moves the slot of token keep[i] to token start + i.  Every entry must point at or behind its
// destination, so that slots may be moved in place a step at a time: what a step reads lies at or behind the first place
// it writes, i.e. behind everything that earlier steps wrote.  A cluster of CTAs shares a step: all read, all wait for one
// another, all write.  A slot is 5 to 9 pieces of 16 bytes, read and written by neighbouring threads.
// Floor: every moved slot read and written once (128 lists of 4096 of 16k slots: 23 us at copy bandwidth; measured 45 us;
// single cold launches: 52 us with four CTAs an SM, 58 with the two that 122 registers a thread allow, 63 when a step's entries
// are looked up while the slots of the one before are read).
constexpr int kCompactThreads = 256, kCompactStep = 256;      // entries of one CTA in a step

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

template <int PIECES>
__global__ void __launch_bounds__(kCompactThreads, 4) compact_cache_kernel(const CompactParams p) {
  __shared__ int64_t s_from[kCompactStep], s_to[kCompactStep];  // byte offsets of the slots, -1: nothing to move
  const int tid = threadIdx.x;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int row = blockIdx.x / ranks, b = row / p.H, h = row % p.H;
  const int64_t room = static_cast<int64_t>(p.bt_stride) * p.block_size;
  const int n = p.seq_lens[b] < room ? p.seq_lens[b] : static_cast<int>(room);
  const int start = p.start ? p.start[b] : 0;
  const int32_t* list = p.keep + (p.keep_shared ? static_cast<int64_t>(b) : static_cast<int64_t>(b) * p.H + h) * p.K;
  float* mass = p.mass ? p.mass + (static_cast<int64_t>(b) * p.H + h) * p.mass_stride : nullptr;
  if (start < 0) {                                // (the same for all CTAs of the cluster)
    if (tid == 0 && rank == 0) atomicOr(&g_evict_status, kStatusKeep);
    return;
  }
  auto slot = [&](int t) -> int64_t {
    const int blk = p.block_table[static_cast<int64_t>(b) * p.bt_stride + t / p.block_size];
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(p.num_blocks)) { atomicOr(&g_evict_status, kStatusBadBlock); return -1; }
    return ((static_cast<int64_t>(blk) * p.block_size + t % p.block_size) * p.H + h) * p.slot_bytes;
  };
  for (int i0 = 0; i0 < p.K; i0 += kCompactStep * static_cast<int>(ranks)) {
    const int first = i0 + static_cast<int>(rank) * kCompactStep, i = first + tid;
    const int count = min(kCompactStep, p.K - first);            // entries of this CTA (may be negative)
    float m = 0.f;
    int64_t from = -1, to = -1;
    if (i < p.K) {
      const int src = list[i];
      const int64_t dst = static_cast<int64_t>(start) + i;
      if (src >= 0 && (src < dst || src >= n)) {
        atomicOr(&g_evict_status, kStatusKeep);
      } else if (src >= 0) {
        from = slot(src);
        to = from < 0 ? -1 : src != dst ? slot(static_cast<int>(dst)) : from;
        if (mass && to >= 0 && src < p.mass_stride) m = mass[src];      // a weight goes where its slot goes
        if (src == dst) to = -1;                  // (it stays)
      }
    }
    s_from[tid] = to >= 0 ? from : -1;
    s_to[tid] = to;
    __syncthreads();
    uint4 piece[PIECES];
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const int q = tid + c * kCompactThreads, e = q / PIECES;
      if (e < count && s_from[e] >= 0) piece[c] = *reinterpret_cast<const uint4*>(p.cache + s_from[e] + 16 * (q - e * PIECES));
    }
    if (ranks > 1) cluster_sync();
    else __syncthreads();
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      const int q = tid + c * kCompactThreads, e = q / PIECES;
      if (e < count && s_from[e] >= 0) *reinterpret_cast<uint4*>(p.cache + s_to[e] + 16 * (q - e * PIECES)) = piece[c];
    }
    if (mass && i < p.K && static_cast<int64_t>(start) + i < p.mass_stride) mass[start + i] = m;
    __syncthreads();                              // the offsets may be overwritten
  }
  // all moved weights were read in front of the last step's barrier
  if (mass)
    for (int64_t t = static_cast<int64_t>(start) + p.K + rank * kCompactThreads + tid; t < n && t < p.mass_stride; t += ranks * kCompactThreads) mass[t] = 0.f;
}

// A launch in clusters of `ranks` CTAs along x.
template <class... Params, class... Args>
static int launch_clusters(const char* what, void (*kernel)(Params...), int rows, int ranks, int threads, size_t smem, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * ranks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) return check_launch(what);
  return check_launch(what);
}

}  // namespace cda

using namespace cda;

extern "C" int cda_b200_select_keys(const float* mass, const int32_t* seq_lens, int32_t* keep, int32_t* new_lens, int B, int H_kv,
                                    int64_t mass_stride, int budget, int sink, int recent, void* stream) {
  if (B < 0 || H_kv <= 0 || mass_stride < 0 || budget <= 0 || sink < 0 || recent < 0) return fail(CDA_ERR_BAD_ARG, "select_keys: negative size or no budget");
  if (static_cast<int64_t>(sink) + recent > budget) return fail(CDA_ERR_BAD_SHAPE, "select_keys: sink %d + recent %d exceed the budget %d", sink, recent, budget);
  // (places are 32-bit integers that loops step past the end of a list)
  if (mass_stride > 0x7fff0000ll || budget > 0x7fff0000 || static_cast<int64_t>(B) * H_kv > 0x7fffffffll / 8) return fail(CDA_ERR_N_TOO_LARGE, "select_keys: too many weights, rows or kept keys");
  if (B == 0) return CDA_OK;
  if (!mass || !seq_lens || !keep || !new_lens) return fail(CDA_ERR_BAD_ARG, "select_keys: null pointer");
  // CTAs of a row: as few as hold a slice of 16384 keys each, since adding up the histograms costs a CTA as much as some 10000
  // keys (256 rows of 65536: 101 us with 4 CTAs a row; before the last steps 113 us with 4, 215 with 8, 127 with 2); more where rows are few and the GPU idle
  const int rows = B * H_kv, sms = device_sm_count(-1);
  int ranks = 1;
  while (ranks < 8 && (mass_stride > 16384ll * ranks || (mass_stride > 2048ll * ranks && rows * ranks <= sms / 2))) ranks *= 2;
  const int64_t slice = ((mass_stride + ranks - 1) / ranks + 511) / 512 * 512;
  const int cached = slice <= kSliceMax ? static_cast<int>(slice) : 0;
  static bool configured[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    if (cudaFuncSetAttribute(select_keys_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceMax * 4) != cudaSuccess)
      return check_launch("select_keys: shared memory opt-in");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return launch_clusters("select_keys", select_keys_kernel, rows, ranks, kSelectThreads, static_cast<size_t>(cached) * 4, static_cast<cudaStream_t>(stream),
                         mass, seq_lens, keep, new_lens, H_kv, mass_stride, budget, sink, recent, cached);
}

extern "C" int cda_b200_compact_cache(void* kv_cache, const int32_t* block_table, const int32_t* seq_lens, const int32_t* keep,
                                      const int32_t* start, float* mass, int64_t mass_stride, int B, int H_kv, int K, int keep_heads,
                                      int block_size, int block_table_stride, int64_t num_slots, int slot_bytes, void* stream) {
  if (B < 0 || H_kv <= 0 || K < 0 || num_slots < 0 || block_table_stride < 0 || (mass && mass_stride < 0)) return fail(CDA_ERR_BAD_ARG, "compact_cache: negative size");
  if (slot_bytes != 144 && slot_bytes != 112 && slot_bytes != 80) return fail(CDA_ERR_BAD_SHAPE, "compact_cache: slot width %d is none of 144, 112, 80", slot_bytes);
  if (block_size <= 0 || block_size % 16) return fail(CDA_ERR_BAD_SHAPE, "compact_cache: block_size=%d is not a multiple of 16", block_size);
  if (keep_heads != 1 && keep_heads != H_kv) return fail(CDA_ERR_BAD_SHAPE, "compact_cache: keep has %d heads, the cache %d", keep_heads, H_kv);
  if (num_slots / block_size > 0x7fffffffll || K > 0x7fff0000 || static_cast<int64_t>(B) * H_kv > 0x7fffffffll / 8) return fail(CDA_ERR_N_TOO_LARGE, "compact_cache: too many slots, entries or sequences");
  if (B == 0 || (K == 0 && !mass)) return CDA_OK;
  if (!kv_cache || !block_table || !seq_lens || (K > 0 && !keep)) return fail(CDA_ERR_BAD_ARG, "compact_cache: null pointer");
  if (!aligned16(kv_cache)) return fail(CDA_ERR_BAD_ALIGN, "compact_cache: cache must be 16-byte aligned");
  const CompactParams p{static_cast<uint8_t*>(kv_cache), block_table, seq_lens, keep, start, mass, mass_stride, B, H_kv, K, block_size,
                        block_table_stride, static_cast<int>(num_slots / block_size), slot_bytes, keep_heads == 1 ? 1 : 0};
  // CTAs of a list: until each has one step, or all SMs have two (128 lists of 4096, two CTAs an SM: 57 us with 4 CTAs each, 63 with 8)
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rows = B * H_kv, sms = device_sm_count(-1);
  int ranks = 1;
  while (ranks < 8 && K > kCompactStep * ranks && rows * ranks < 2 * sms) ranks *= 2;
  return slot_bytes == 144 ? launch_clusters("compact_cache", compact_cache_kernel<9>, rows, ranks, kCompactThreads, 0, st, p)
       : slot_bytes == 112 ? launch_clusters("compact_cache", compact_cache_kernel<7>, rows, ranks, kCompactThreads, 0, st, p)
                           : launch_clusters("compact_cache", compact_cache_kernel<5>, rows, ranks, kCompactThreads, 0, st, p);
}

// The copies below run on the legacy default stream, which non-blocking streams neither wait for nor are waited for by: the
// device is synchronised first, so that every call made before has reported.
extern "C" int cda_b200_kv_status(void) {
  int v = 0, t = 0;
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&v, g_evict_status, sizeof(int)) != cudaSuccess) return check_launch("kv_status");
  const int rc = tree_status(false, &t);
  return rc != CDA_OK ? rc : (v | t) & 0x7fffffff;
}

extern "C" int cda_b200_kv_clear_status(void) {
  const int zero = 0;
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyToSymbol(g_evict_status, &zero, sizeof(int)) != cudaSuccess) return check_launch("kv_clear_status");
  return tree_status(true, nullptr);
}

// Attention of short query chunks over the paged compressed cache on the tcgen05 tensor cores: keys on the M axis.
//
// A row block is NR (16, 32, 64 or 128) of the rows (token, query head of one KV head) of one sequence.  Keys are processed
// 128 at a time, one key per tensor-memory lane:
//   S^T (128 keys x NR)  = K (tensor memory) . Q^T (shared memory; the fp32 query as two fp16 terms, hi and lo, so a score
//                          carries no rounding of the query)
//   P^T                  = exp2(S^T - reference of the row), rounded to fp16 -- the one rounding made before the product
//   O^T (128 x NR)      += V^T (shared memory) . P^T (shared memory)
// With the keys on M a block of few rows costs few columns, where rows on M would fill a 128-row operand with padding; and
// since a lane is a key, the K producers hand their expanded rows to the tensor core through tensor memory, lane by lane,
// without a pass through shared memory.
//
// Warps: softmax (2 or 4 groups of four warps; a thread is a key, a group has NR / groups of the rows), K producers and V
// producers (four each; a thread is a key), one MMA warp, one feeder that brings the slots into a ring in shared memory with
// tensor-map copies of 16 slots of one head.
// A CTA walks an equal share of all (sequence, row block, KV head) segments' tiles; a segment that starts and ends in one CTA
// is finished there, the pieces of the others are merged by tree_merge_kernel.
//
// The reference of a row is the largest score of the first tile in which it sees a key; it moves only when a later score is
// more than 2^14 above it (an fp16 probability carries 2^15): then, and in a row's first tile, the group of warps takes the
// slow path, which finds the tile's row maxima across lanes and rescales O and the sums.
#pragma once
#include "attend.cuh"
#include "cache_map.cuh"
#include "expand.cuh"
#include "umma.cuh"

namespace cda {
namespace tru {

using namespace umma;

constexpr int kKeys = 128, kTileBytes = 32768, kColBlock = 16384;
constexpr int kStageBytes = kKeys * 144;         // 128 slots side by side; their widths (144, 112, 80) are odd multiples of 16,
                                                 // so threads that read the same piece of 8 neighbouring slots meet no conflict
constexpr float kNoRef = 1.0e30f;                // stored negated reference of a row without one: any score exceeds it
constexpr float kSafe = 14.0f;

template <int NR>
struct Cfg {
  static constexpr int kGroups = NR == 128 ? 4 : 2;
  static constexpr int kCols = NR / kGroups;                     // rows of one softmax group = score columns of one thread
  static constexpr int kChunk = kCols < 16 ? kCols : 16;
  static constexpr int kChunks = kCols / kChunk;
  static constexpr int kSoftWarps = 4 * kGroups;
  static constexpr int kWarpK = kSoftWarps, kWarpV = kSoftWarps + 4, kWarpMma = kSoftWarps + 8, kWarpFeed = kWarpMma + 1;
  static constexpr int kThreads = (kWarpFeed + 1) * 32;
  static constexpr int kPStages = NR == 128 ? 1 : 2;
  static constexpr int kPBytes = kColBlock * (NR == 128 ? 2 : 1);
  static constexpr int kRing = NR == 128 ? 3 : NR == 64 ? 5 : 6;
  static constexpr int kTmemCols = NR <= 32 ? 256 : 512;
  static constexpr int kColK = 0, kColS = 128, kColO = 128 + 2 * NR;
  // shared memory (bytes from a 1024-aligned base)
  static constexpr int kOffV = 0, kOffP = 2 * kTileBytes, kOffQ = kOffP + kPStages * kPBytes, kOffRing = kOffQ + NR * 512;
  static constexpr int kOffRef = kOffRing + kRing * kStageBytes;  // NR floats: negated references
  static constexpr int kOffFac = kOffRef + 4 * NR;                // NR floats: factors of a slow path
  static constexpr int kOffPos = kOffFac + 4 * NR;                // NR ints: positions of the rows
  static constexpr int kOffSlope = kOffPos + 4 * NR;              // NR floats: slopes x log2 e
  static constexpr int kOffMask = kOffSlope + 4 * NR;             // NR 64-bit ancestor masks
  static constexpr int kOffMax = kOffMask + 8 * NR;               // 4 warps x NR floats
  static constexpr int kOffLevels = kOffMax + 16 * NR;            // 2 x 16 floats
  static constexpr int kOffBar = kOffLevels + 128;                // barriers, TMEM address, wait state, plan
  static constexpr int kSmemBytes = kOffBar + 320 + 1024;
  static_assert(kSmemBytes <= 232448, "one CTA's shared memory");
};
constexpr int kKFull = 0, kVFull = 2, kSFull = 4, kSEmpty = 6, kPFull = 8, kPvDone = 10, kQFull = 12, kDrained = 13, kRingFull = 14, kRingEmpty = 20;
constexpr int kOffTmemAddr = 208, kOffWait = 216, kOffPlan = 232, kOffValid = 256;   // inside kOffBar; valid: keys of each ring stage

// ---- shared memory access -----------------------------------------------------------------------------------------------
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void sts_f(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory"); }
__device__ __forceinline__ void sts64(uint32_t a, uint32_t x, uint32_t y) {
  asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint32_t sw128(uint32_t row, uint32_t chunk) {   // byte offset inside a block of 128-byte rows
  return (row >> 3) * 1024u + (row & 7u) * 128u + ((chunk ^ (row & 7u)) << 4);
}
__device__ __forceinline__ void group_barrier(int group) { asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory"); }
__device__ __forceinline__ bool group_any(int group, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(mine ? 1u : 0u), "r"(group + 1)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[N]) {
  if constexpr (N == 8) tmem_ld8(addr, v);
  else tmem_ld16(addr, v);
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&v)[N]) {
  if constexpr (N == 8) tmem_st8(addr, v);
  else tmem_st16(addr, v);
}

// A bounded wait for a barrier phase.  An attempt lets the hardware park the warp for up to kParkNs, so that waiting warps
// leave the issue slots to the working ones (attempts without the hint, with the timer read between them, cost the
// working warps three quarters of their speed).  Once a wait of the CTA has given up, every later one returns after one
// attempt: all roles then run their loops to the end (so nobody is left at a named barrier) without issuing or writing.
constexpr uint32_t kParkNs = 20000;
__device__ __forceinline__ bool park_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(kParkNs)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile WaitState* ws) {
  if (park_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!ws->abort && global_timer_ns() - t0 < ws->limit_ns)
    if (park_wait(bar, parity)) return true;
  ws->abort = 1;
  return false;
}

// ---- the walk over segments ---------------------------------------------------------------------------------------------
// Entry e = (sequence b, row block rb); its H_kv segments follow one another.  Tiles hold the keys that some row of the block
// may see.
struct Entry { int b, rb, q_begin, q_len, ctx, seq_len, t0, first, tiles; };
template <int NR>
__device__ __forceinline__ Entry entry_of(const AttendParams& p, int e) {
  Entry x;
  x.b = e / p.row_blocks;
  x.rb = e - x.b * p.row_blocks;
  const SequenceView s = sequence_view(p, x.b);
  x.q_begin = s.q_begin; x.q_len = s.q_len; x.seq_len = s.seq_len;
  x.ctx = s.seq_len - s.q_len;
  x.first = x.tiles = 0;
  x.t0 = x.rb * NR / p.group;
  if (x.rb * NR >= s.q_len * p.group) return x;
  const int t1 = min(s.q_len, (x.rb * NR + NR + p.group - 1) / p.group) - 1;
  const int hi = p.tree_mask ? s.seq_len : x.ctx + t1 + 1;
  const int lo = p.window > 0 ? max(0, x.ctx + (p.tree_mask ? 0 : x.t0) - p.window + 1) : 0;
  x.first = lo / kKeys;
  x.tiles = (hi + kKeys - 1) / kKeys - x.first;
  return x;
}
struct Piece { Entry x; int e, head, tile0, n; bool starts, ends; };
template <int NR>
struct Walk {
  int e, h, j, left, entries;
  __device__ __forceinline__ bool next(const AttendParams& p, Piece& q) {
    while (left > 0 && e < entries) {
      q.x = entry_of<NR>(p, e);
      if (q.x.tiles == 0) { ++e; continue; }
      q.e = e; q.head = h;
      q.tile0 = q.x.first + j;
      q.n = min(left, q.x.tiles - j);
      q.starts = j == 0;
      left -= q.n;
      j += q.n;
      q.ends = j == q.x.tiles;
      if (q.ends) { j = 0; if (++h == p.H_kv) { h = 0; ++e; } }
      return true;
    }
    return false;
  }
};

// What a CTA left for the merge: the segment that starts here and goes on (tail_e < 0: none), and whether the piece of a
// segment from before ends here (2), goes on (1) or does not exist (0); 3: this CTA gave up.
struct Record { int tail_e, tail_head, head_state, pad; };

// Workspace: one Record per CTA, then (m, l) of the 2 x CTAs x NR rows of pieces, then their O rows.
template <int NR>
struct Space {
  Record* rec;
  float2* ml;
  float* o;
  __device__ __forceinline__ Space(void* ws, int ctas) {
    rec = static_cast<Record*>(ws);
    ml = reinterpret_cast<float2*>(rec + ctas);
    o = reinterpret_cast<float*>(ml + static_cast<int64_t>(2) * ctas * NR);
  }
};

// Share of this CTA: finds its first segment and tile.  Every thread takes part.
template <int NR, int THREADS>
__device__ __forceinline__ void find_share(const AttendParams& p, int* s_scan, int* s_plan) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, entries = p.B * p.row_blocks;
  const int per = (entries + THREADS - 1) / THREADS, e0 = min(tid * per, entries), e1 = min(e0 + per, entries);
  int sum = 0;
  for (int e = e0; e < e1; ++e) {
    sum += entry_of<NR>(p, e).tiles * p.H_kv;
    if (blockIdx.x == 0 && e % p.row_blocks == 0 && sequence_view(p, e / p.row_blocks).bad) atomicOr(&g_tree_status, kStatusLengths);
  }
  int x = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  if (lane == 31) s_scan[warp] = x;
  if (tid == 0) s_plan[3] = 0;
  __syncthreads();
  int before = x - sum, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  // the first `busy` CTAs take equal shares of at least one tile, so the pieces of a segment lie in consecutive CTAs
  const int busy = min(static_cast<int>(gridDim.x), total), cta = min(static_cast<int>(blockIdx.x), busy);
  const int lo = busy ? static_cast<int>(static_cast<int64_t>(total) * cta / busy) : 0;
  const int hi = cta < busy ? static_cast<int>(static_cast<int64_t>(total) * (cta + 1) / busy) : lo;
  if (hi > lo && before <= lo && lo < before + sum) {
    int at = before;
    for (int e = e0; e < e1; ++e) {
      const int tiles = entry_of<NR>(p, e).tiles;
      if (lo < at + tiles * p.H_kv) {
        s_plan[0] = e;
        s_plan[1] = (lo - at) / tiles;
        s_plan[2] = (lo - at) % tiles;
        s_plan[3] = hi - lo;
        break;
      }
      at += tiles * p.H_kv;
    }
  }
  __syncthreads();
}

// ---- copies ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// 16 slots of one head (a box of 16 rows x slot_bytes at byte x of row y) -> shared memory; x is head * slot_bytes, a multiple
// of 16, the destination a multiple of 128.
__device__ __forceinline__ void copy_group(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
               : "memory");
}

template <int NR>
__global__ void __launch_bounds__(Cfg<NR>::kThreads, 1) tree_attention_kernel(const AttendParams p, void* ws,
                                                                                   const __grid_constant__ CUtensorMap map) {
  using C = Cfg<NR>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Space<NR> space(ws, gridDim.x);
  int* s_plan = reinterpret_cast<int*>(sm + C::kOffBar + kOffPlan);
  volatile WaitState* wait = reinterpret_cast<volatile WaitState*>(sm + C::kOffBar + kOffWait);
  const uint32_t bar0 = base + C::kOffBar;
  auto bar = [&](int i) { return bar0 + 8u * i; };

  find_share<NR, C::kThreads>(p, reinterpret_cast<int*>(sm + C::kOffMax), s_plan);
  const int total = s_plan[3];
  if (total == 0) {
    if (tid == 0) space.rec[blockIdx.x] = Record{-1, 0, 0, 0};
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(kKFull + i), 4); mbar_init(bar(kVFull + i), 4); mbar_init(bar(kSFull + i), 1);
      mbar_init(bar(kSEmpty + i), C::kSoftWarps); mbar_init(bar(kPFull + i), C::kSoftWarps); mbar_init(bar(kPvDone + i), 1);
    }
    mbar_init(bar(kQFull), C::kSoftWarps);
    mbar_init(bar(kDrained), 1);
    for (int i = 0; i < C::kRing; ++i) { mbar_init(bar(kRingFull + i), 1); mbar_init(bar(kRingEmpty + i), 8); }
    wait->abort = 0;
    wait->limit_ns = kWaitLimitNs;
    mbar_init_fence();
  }
  if (tid < 32) {                                               // code levels: 16 or 4 of K, then of V
    const int side = tid >> 4, i = tid & 15, n = (side ? p.v_bits : p.k_bits) == 4 ? 16 : 4;
    reinterpret_cast<float*>(sm + C::kOffLevels)[tid] = i < n ? __ldg((side ? p.cb_v : p.cb_k) + i) : 0.f;
  }
  if (warp == C::kWarpMma) {
    tmem_alloc(base + C::kOffBar + kOffTmemAddr, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + C::kOffBar + kOffTmemAddr);
  Walk<NR> w{s_plan[0], s_plan[1], s_plan[2], total, p.B * p.row_blocks};
  Record rec{-1, 0, 0, 0};

  if (warp < C::kSoftWarps) {
    // ============ softmax: a thread is a key (TMEM lane), its group's rows are columns ======================================
    const int group = warp >> 2, key = (warp & 3) * 32 + lane, gtid = tid & 127, col0 = group * C::kCols;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t ref_a = base + C::kOffRef + 4 * col0, fac_a = base + C::kOffFac + 4 * col0, max_a = base + C::kOffMax + 16 * col0;
    const float kf = p.scale * kLog2e, cap2 = p.softcap * kLog2e, inv_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
    bool alive = true;
    int i = 0;                                                  // tiles so far, over all pieces
    Piece pc;
    while (w.next(p, pc)) {
      const Entry& x = pc.x;
      // ---- the group's query rows: rotate, split, store as the B operand; what the masks need of them
#pragma unroll 1
      for (int r0 = warp & 3; r0 < C::kCols; r0 += 16) {        // four rows at a time
        float q[4][4];
        int t[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = col0 + r0 + 4 * u, row = x.rb * NR + r;
          t[u] = row / p.group;
          q[u][0] = q[u][1] = q[u][2] = q[u][3] = 0.f;
          if (r0 + 4 * u < C::kCols && t[u] < x.q_len)
            load_half4(p.q + (static_cast<int64_t>(x.q_begin + t[u]) * p.H_q + pc.head * p.group + row % p.group) * kHeadDim + 4 * lane, q[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int r = col0 + r0 + 4 * u;
          if (r0 + 4 * u >= C::kCols) break;
          fht128_warp(q[u], lane);
          float lo[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            q[u][c] *= kRsqrtD;
            lo[c] = q[u][c] - round_to_half(q[u][c]);
          }
          const uint2 h = pack_half4(q[u]), l = pack_half4(lo);
          const uint32_t at = base + C::kOffQ + (lane >> 4) * (NR * 128) + sw128(r, (lane & 15) >> 1) + 8 * (lane & 1);
          sts64(at, h.x, h.y);
          sts64(at + NR * 256, l.x, l.y);
          if (lane == 0) {
            const bool real = t[u] < x.q_len;
            reinterpret_cast<int*>(sm + C::kOffPos)[r] = x.ctx + (real ? depth_of(p, x.q_begin, t[u]) : 0);
            reinterpret_cast<unsigned long long*>(sm + C::kOffMask)[r] =
                real && p.tree_mask ? static_cast<unsigned long long>(p.tree_mask[x.q_begin + t[u]]) : 0ull;
            reinterpret_cast<float*>(sm + C::kOffSlope)[r] =
                p.slopes ? p.slopes[pc.head * p.group + (x.rb * NR + r) % p.group] * kLog2e : 0.f;
            sts_f(ref_a + 4 * (r - col0), kNoRef);
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kQFull));
      group_barrier(group);                                     // the rows' words are read by the whole group
      uint64_t sum[C::kCols / 2];
#pragma unroll
      for (int c = 0; c < C::kCols / 2; ++c) sum[c] = f2_pack(0.f, 0.f);

#pragma unroll 1
      for (int k = 0; k < pc.n; ++k, ++i) {
        const int key0 = (pc.tile0 + k) * kKeys;
        alive = wait_for(bar(kSFull + (i & 1)), (i >> 1) & 1, wait) && alive;
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t s_col = lanes + C::kColS + (i & 1) * NR + col0;
        // some row may not see some key of this tile, or keys get a bias: the scores are finished here, one by one
        const bool rule = p.slopes != nullptr || key0 + kKeys > x.ctx + (p.tree_mask ? 0 : x.t0 + 1) ||
                          (p.window > 0 && key0 <= x.ctx + x.q_len - p.window);
        const bool finish = rule || p.softcap > 0.f;
        const float f = finish ? 1.0f : kf;
        const uint64_t ff = f2_pack(f, f);
        const int n = key0 + key;
        int pos_k = n;
        if (rule && p.tree_mask && n >= x.ctx && n < x.seq_len) pos_k = x.ctx + depth_of(p, x.q_begin, n - x.ctx);
        // pass 1: does any score exceed its row's reference by more than an fp16 probability can carry?
        float excess = -INFINITY;
#pragma unroll
        for (int ch = 0; ch < C::kChunks; ++ch) {
          uint32_t s[C::kChunk];
          tmem_load<C::kChunk>(s_col + ch * C::kChunk, s);
          tmem_wait_ld();
          if (finish) {
#pragma unroll
            for (int c = 0; c < C::kChunk; ++c) {
              const int r = col0 + ch * C::kChunk + c;
              float v = __uint_as_float(s[c]);
              v = p.softcap > 0.f ? cap2 * soft_tanh(v * inv_cap) : v * kf;
              if (rule) {
                const int pos_q = reinterpret_cast<const int*>(sm + C::kOffPos)[r];
                v = fmaf(reinterpret_cast<const float*>(sm + C::kOffSlope)[r], static_cast<float>(pos_k - pos_q), v);
                bool see = n < x.ctx;
                if (!see && n < x.seq_len)
                  see = p.tree_mask ? (reinterpret_cast<const unsigned long long*>(sm + C::kOffMask)[r] >> (n - x.ctx)) & 1ull : n <= pos_q;
                if (p.window > 0 && pos_q - pos_k >= p.window) see = false;
                v = see ? v : -INFINITY;
              }
              s[c] = __float_as_uint(v);
            }
            tmem_store<C::kChunk>(s_col + ch * C::kChunk, s);
          }
#pragma unroll
          for (int c = 0; c < C::kChunk; c += 4) {
            const uint4 r = lds128(ref_a + 4 * (ch * C::kChunk + c));
            float a0, a1, a2, a3;
            f2_unpack(f2_fma(f2_pack(s[c], s[c + 1]), ff, f2_pack(r.x, r.y)), a0, a1);
            f2_unpack(f2_fma(f2_pack(s[c + 2], s[c + 3]), ff, f2_pack(r.z, r.w)), a2, a3);
            excess = fmax3(excess, a0, a1);
            excess = fmax3(excess, a2, a3);
          }
        }
        if (finish) tmem_wait_st();
        if (group_any(group, excess > kSafe)) {
          // slow path: row maxima of the tile, new references, factors for what the rows hold already
#pragma unroll 1
          for (int ch = 0; ch < C::kChunks; ++ch) {
            uint32_t s[C::kChunk];
            tmem_load<C::kChunk>(s_col + ch * C::kChunk, s);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < C::kChunk; ++c) {
              const float m = warp_max(__uint_as_float(s[c]) * f);
              if (lane == 0) sts_f(max_a + 4 * ((warp & 3) * C::kCols + ch * C::kChunk + c), m);
            }
          }
          group_barrier(group);
          if (gtid < C::kCols) {
            float m = lds_f(max_a + 4 * gtid);
#pragma unroll
            for (int u = 1; u < 4; ++u) m = fmaxf(m, lds_f(max_a + 4 * (u * C::kCols + gtid)));
            const float old = lds_f(ref_a + 4 * gtid);
            float fac = 1.0f;
            if (m + old > kSafe) {
              fac = old == kNoRef ? 0.f : fast_exp2(-old - m);
              sts_f(ref_a + 4 * gtid, -m);
            }
            sts_f(fac_a + 4 * gtid, fac);
          }
          group_barrier(group);
#pragma unroll
          for (int c = 0; c < C::kCols; c += 4) {
            const uint4 r = lds128(fac_a + 4 * c);
            sum[c / 2] = f2_mul(sum[c / 2], f2_pack(r.x, r.y));
            sum[c / 2 + 1] = f2_mul(sum[c / 2 + 1], f2_pack(r.z, r.w));
          }
          if (k > 0) {                                          // O of the piece so far; P V of this tile waits for this group
            alive = wait_for(bar(kPvDone + ((i - 1) & 1)), ((i - 1) >> 1) & 1, wait) && alive;
            __syncwarp();
            tc_fence_after_sync();
            const uint32_t o_col = lanes + C::kColO + col0;
#pragma unroll 1
            for (int ch = 0; ch < C::kChunks; ++ch) {
              uint32_t o[C::kChunk];
              tmem_load<C::kChunk>(o_col + ch * C::kChunk, o);
              tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < C::kChunk; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * lds_f(fac_a + 4 * (ch * C::kChunk + c)));
              tmem_store<C::kChunk>(o_col + ch * C::kChunk, o);
            }
            tmem_wait_st();
          }
        }
        // pass 2: probabilities against the references, sums in fp32, P to shared memory once its buffer is free
        if (i >= C::kPStages) {
          const int j = i - C::kPStages;
          alive = wait_for(bar(kPvDone + (j & 1)), (j >> 1) & 1, wait) && alive;
          __syncwarp();
        }
        const uint32_t p_tile = base + C::kOffP + (C::kPStages == 2 ? (i & 1) * C::kPBytes : 0) + (col0 >> 6) * kColBlock;
#pragma unroll
        for (int ch = 0; ch < C::kChunks; ++ch) {
          uint32_t s[C::kChunk], pk[C::kChunk / 2];
          tmem_load<C::kChunk>(s_col + ch * C::kChunk, s);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < C::kChunk; c += 4) {
            const uint4 r = lds128(ref_a + 4 * (ch * C::kChunk + c));
            float a[4];
            f2_unpack(f2_fma(f2_pack(s[c], s[c + 1]), ff, f2_pack(r.x, r.y)), a[0], a[1]);
            f2_unpack(f2_fma(f2_pack(s[c + 2], s[c + 3]), ff, f2_pack(r.z, r.w)), a[2], a[3]);
#pragma unroll
            for (int u = 0; u < 4; ++u) a[u] = fast_exp2(a[u]);
            const int g = (ch * C::kChunk + c) / 2;
            sum[g] = f2_add(sum[g], f2_pack(a[0], a[1]));
            sum[g + 1] = f2_add(sum[g + 1], f2_pack(a[2], a[3]));
            pk[c / 2] = pack_half2(a[0], a[1]);
            pk[c / 2 + 1] = pack_half2(a[2], a[3]);
          }
#pragma unroll
          for (int c8 = 0; c8 < C::kChunk / 8; ++c8)
            sts128(p_tile + sw128(key, ((col0 & 63) + ch * C::kChunk) / 8 + c8), pk[4 * c8], pk[4 * c8 + 1], pk[4 * c8 + 2], pk[4 * c8 + 3]);
        }
        fence_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(kSEmpty + (i & 1)));
          mbar_arrive(bar(kPFull + (i & 1)));
        }
      }

      // ---- end of the piece: sums over the 128 keys, then O
      alive = wait_for(bar(kPvDone + ((i - 1) & 1)), ((i - 1) >> 1) & 1, wait) && alive;
      __syncwarp();
      tc_fence_after_sync();
#pragma unroll
      for (int c = 0; c < C::kCols; c += 2) {
        float a, b;
        f2_unpack(sum[c / 2], a, b);
        a = warp_sum(a);
        b = warp_sum(b);
        if (lane == 0) {
          sts_f(max_a + 4 * ((warp & 3) * C::kCols + c), a);
          sts_f(max_a + 4 * ((warp & 3) * C::kCols + c + 1), b);
        }
      }
      group_barrier(group);
      if (gtid < C::kCols) {
        float l = 0.f;
#pragma unroll
        for (int u = 0; u < 4; ++u) l += lds_f(max_a + 4 * (u * C::kCols + gtid));
        sts_f(fac_a + 4 * gtid, l);
      }
      group_barrier(group);
      const bool whole = pc.starts && pc.ends;
      const int64_t slot = static_cast<int64_t>(2) * blockIdx.x + (pc.starts ? 1 : 0);
      if (!whole) {
        if (pc.starts) { rec.tail_e = pc.e; rec.tail_head = pc.head; }
        else rec.head_state = pc.ends ? 2 : 1;
        if (gtid < C::kCols && alive) {
          const float nref = lds_f(ref_a + 4 * gtid);
          space.ml[slot * NR + col0 + gtid] = make_float2(nref == kNoRef ? -INFINITY : -nref, lds_f(fac_a + 4 * gtid));
        }
      }
#pragma unroll 1
      for (int ch = 0; ch < C::kChunks; ++ch) {
        uint32_t o[C::kChunk];
        tmem_load<C::kChunk>(lanes + C::kColO + col0 + ch * C::kChunk, o);
        tmem_wait_ld();
        if (!whole) {                                           // un-normalised, one row of 128 per column
          float* to = space.o + (slot * NR + col0 + ch * C::kChunk) * kHeadDim + key;
          if (alive) {
#pragma unroll
            for (int c = 0; c < C::kChunk; ++c) to[c * kHeadDim] = __uint_as_float(o[c]);
          }
          continue;
        }
        // transpose through the (idle) P buffer, rotate back in fp32, round once
        const uint32_t area = base + C::kOffP + group * (C::kChunk * 512);
#pragma unroll
        for (int c = 0; c < C::kChunk; ++c) sts_f(area + c * 512 + key * 4, __uint_as_float(o[c]));
        group_barrier(group);
#pragma unroll 1
        for (int c = warp & 3; c < C::kChunk; c += 4) {
          const int r = ch * C::kChunk + c, row = x.rb * NR + col0 + r, t = row / p.group;
          const float l = lds_f(fac_a + 4 * r), inv = l > 0.f ? kRsqrtD / l : (l == 0.f ? 0.f : l);
          const uint4 v4 = lds128(area + c * 512 + lane * 16);
          float v[4] = {__uint_as_float(v4.x) * inv, __uint_as_float(v4.y) * inv, __uint_as_float(v4.z) * inv, __uint_as_float(v4.w) * inv};
          fht128_warp(v, lane);
          if (t < x.q_len && alive) {
            const int64_t at = static_cast<int64_t>(x.q_begin + t) * p.H_q + pc.head * p.group + row % p.group;
            *reinterpret_cast<uint2*>(p.out + at * kHeadDim + 4 * lane) = pack_half4(v);
            if (p.lse_out && lane == 0) {
              const float nref = lds_f(ref_a + 4 * r);
              p.lse_out[at] = nref == kNoRef && l == 0.f ? -INFINITY : (log2f(l) - nref) * kLn2;
            }
          }
        }
        group_barrier(group);
      }
      group_barrier(group);                                     // the rows' words may be overwritten
    }
  } else if (warp < C::kWarpMma) {
    // ============ producers: slot -> exact fp16 row; K to tensor memory (lane = key), V to shared memory (row = key) ==========
    const bool is_v = warp >= C::kWarpV;
    const int key = (warp & 3) * 32 + lane, bits = is_v ? p.v_bits : p.k_bits;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + C::kColK;
    const uint32_t cell0 = base + C::kOffRing + key * p.slot_bytes, code_at = is_v ? 16 * p.k_bits : 0;
    const uint32_t norm_at = 16 * (p.k_bits + p.v_bits) + (is_v ? 4 : 0), row = base + C::kOffV;
    const float* levels = reinterpret_cast<const float*>(sm + C::kOffLevels) + (is_v ? 16 : 0);
    const int full = is_v ? kVFull : kKFull, freed = is_v ? kPvDone : kSFull;
    int stage = 0, turn = 0;
#pragma unroll 1
    for (int i = 0; i < total; ++i) {
      wait_for(bar(kRingFull + stage), turn, wait);
      const uint32_t cell = cell0 + stage * kStageBytes;
      const int valid = *reinterpret_cast<volatile int*>(sm + C::kOffBar + kOffValid + 4 * stage);
      const float norm = key < valid ? lds_f(cell + norm_at) : 0.f;       // keys past the end: zero rows
      const expand::Planes t = expand::make_planes(levels, bits == 4 ? 4 : 1, norm);
      if (i >= 2) wait_for(bar(freed + (i & 1)), ((i - 2) >> 1) & 1, wait);
      __syncwarp();
      tc_fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {                                        // 32 coordinates at a time
        uint32_t v[16];
        if (bits == 4) {
          expand::quarter4(t, lds128(cell + code_at + 16 * c), v);
        } else {
          const uint2 w = lds64(cell + code_at + 8 * c);
          expand::quarter2(t, w.x, w.y, v);
        }
        if (is_v) {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            sts128(row + (i & 1) * kTileBytes + (c >> 1) * kColBlock + sw128(key, (c & 1) * 4 + u), v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        } else {
          tmem_st16(lanes + (i & 1) * 64 + 16 * c, v);
        }
      }
      if (is_v) fence_async_smem();
      else tmem_wait_st();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(kRingEmpty + stage));
        mbar_arrive(bar(full + (i & 1)));
      }
      if (++stage == C::kRing) { stage = 0; turn ^= 1; }
    }
  } else if (warp == C::kWarpFeed) {
    // ============ feeder: one lane per 16-token group of a tile; block ids are read one tile ahead ============================
    Piece q;
    bool live = w.next(p, q), bad = false, alive = true;
    int tile = live ? q.tile0 : 0, stage = 0, turn = 0, issued = 0;
    auto block_id = [&]() {
      const int n = min(tile * kKeys + 16 * (lane & 7), q.x.seq_len - 1);
      return __ldg(p.block_table + static_cast<int64_t>(q.x.b) * p.bt_stride + (p.bs_shift >= 0 ? n >> p.bs_shift : n / p.block_size));
    };
    int id = live ? block_id() : 0;
#pragma unroll 1
    while (live && alive) {
      if (issued >= C::kRing) alive = wait_for(bar(kRingEmpty + stage), turn ^ 1, wait);
      if (!__all_sync(0xffffffffu, alive)) break;
      const int left = q.x.seq_len - tile * kKeys, groups = min(8, (left + 15) >> 4), n = tile * kKeys + 16 * lane;
      if (lane == 0) {
        *reinterpret_cast<volatile int*>(sm + C::kOffBar + kOffValid + 4 * stage) = min(left, kKeys);
        expect_bytes(bar(kRingFull + stage), groups * 16 * p.slot_bytes);
      }
      __syncwarp();
      if (lane < groups) {
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks)) { bad = true; id = 0; }
        const int in = p.bs_shift >= 0 ? n & (p.block_size - 1) : n % p.block_size;
        copy_group(base + C::kOffRing + stage * kStageBytes + lane * 16 * p.slot_bytes, &map, q.head * p.slot_bytes, id * p.block_size + in, bar(kRingFull + stage));
      }
      ++issued;
      if (++stage == C::kRing) { stage = 0; turn ^= 1; }
      if (++tile == q.tile0 + q.n) {
        live = w.next(p, q);
        if (live) tile = q.tile0;
      }
      if (live) id = block_id();
    }
    if (bad) atomicOr(&g_tree_status, kStatusBadBlock);
    // no copy may be in flight when the CTA ends, also after a wait elsewhere gave up
    const unsigned long long t0 = global_timer_ns();
    for (int k = max(0, issued - C::kRing); k < issued; ++k)
      while (!park_wait(bar(kRingFull + k % C::kRing), (k / C::kRing) & 1) && global_timer_ns() - t0 < kWaitLimitNs) { }
  } else if (lane == 0) {
    // ============ MMA issuer =================================================================================================
    constexpr uint32_t idesc_s = instr_desc_f16(kKeys, NR, false, false), idesc_o = instr_desc_f16(kHeadDim, NR, true, true);
    bool alive = true;
    int i = 0, pieces = 0;
    auto issue_s = [&](int x) {
      alive = wait_for(bar(kKFull + (x & 1)), (x >> 1) & 1, wait) && alive;
      if (x >= 2) alive = wait_for(bar(kSEmpty + (x & 1)), ((x - 2) >> 1) & 1, wait) && alive;
      if (!alive) return;
      tc_fence_after_sync();
      const uint32_t d = tmem + C::kColS + (x & 1) * NR, a = tmem + C::kColK + (x & 1) * 64;
#pragma unroll
      for (int term = 0; term < 2; ++term)
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint64_t b = smem_desc_sw128(base + C::kOffQ + term * (NR * 256) + (ks >> 2) * (NR * 128) + (ks & 3) * 32u, 16, 1024);
          if (term == 0 && ks == 0) mma_ts<false>(d, a, b, idesc_s);
          else mma_ts<true>(d, a + 8 * ks, b, idesc_s);
        }
      mma_commit(bar(kSFull + (x & 1)));
    };
    auto issue_o = [&](int x, bool first) {
      alive = wait_for(bar(kVFull + (x & 1)), (x >> 1) & 1, wait) && alive;
      alive = wait_for(bar(kPFull + (x & 1)), (x >> 1) & 1, wait) && alive;
      if (!alive) return;
      tc_fence_after_sync();
      const uint32_t v = base + C::kOffV + (x & 1) * kTileBytes, pt = base + C::kOffP + (C::kPStages == 2 ? (x & 1) * C::kPBytes : 0);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        mma_ss(tmem + C::kColO, smem_desc_sw128(v + ks * 2048u, kColBlock, 1024), smem_desc_sw128(pt + ks * 2048u, kColBlock, 1024),
               idesc_o, first && ks == 0 ? 0u : 1u);
      mma_commit(bar(kPvDone + (x & 1)));
    };
    Piece pc;
    while (w.next(p, pc)) {
      alive = wait_for(bar(kQFull), pieces & 1, wait) && alive;
      issue_s(i);
#pragma unroll 1
      for (int k = 0; k < pc.n; ++k, ++i) {
        if (k + 1 < pc.n) issue_s(i + 1);
        issue_o(i, k == 0);
      }
      ++pieces;
    }
    // nothing in flight when tensor memory is released: a commit behind everything issued, waited for (with a limit) even
    // after a wait elsewhere gave up
    mma_commit(bar(kDrained));
    const unsigned long long t0 = global_timer_ns();
    while (!mbar_try_wait(bar(kDrained), 0) && global_timer_ns() - t0 < kWaitLimitNs) { }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0) {
    if (wait->abort) { rec = Record{-1, 0, 3, 0}; atomicOr(&g_tree_status, kStatusWait); }
    space.rec[blockIdx.x] = rec;
  }
  if (warp == C::kWarpMma) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// ---- merge ----------------------------------------------------------------------------------------------------------------
// CTA (c, y): rows 8 y .. 8 y + 7 of the segment that starts in CTA c of the first kernel and goes on, one warp per row.
template <int NR>
__global__ void __launch_bounds__(256) tree_merge_kernel(const AttendParams p, void* ws, int ctas) {
  const Space<NR> space(ws, ctas);
  const int c = blockIdx.x, lane = threadIdx.x & 31, r = blockIdx.y * 8 + (threadIdx.x >> 5);
  const Record rec = space.rec[c];
  if (rec.tail_e < 0) return;
  const Entry x = entry_of<NR>(p, rec.tail_e);
  const int row = x.rb * NR + r, t = row / p.group;
  if (t >= x.q_len) return;
  int pieces = 0;                                               // CTA c's own, then those of the CTAs up to the one where it ends
  for (int k0 = c + 1; k0 < ctas; k0 += 32) {
    const int state = k0 + lane < ctas ? space.rec[k0 + lane].head_state : 3;
    const uint32_t stop = __ballot_sync(0xffffffffu, state != 1);
    if (stop) {
      const int at = __ffs(stop) - 1;
      if (__shfl_sync(0xffffffffu, state, at) != 2) return;     // a CTA gave up: the status word says so
      pieces = k0 + at - c + 1;
      break;
    }
  }
  if (pieces == 0) return;
  auto piece_row = [&](int k) { return (static_cast<int64_t>(2) * (c + k) + (k == 0 ? 1 : 0)) * NR + r; };
  float top = -INFINITY, l = 0.f;
  for (int k = lane; k < pieces; k += 32) top = fmaxf(top, space.ml[piece_row(k)].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < pieces; ++k) {
    const int64_t at = piece_row(k);
    const float2 ml = space.ml[at];
    const float4 v = reinterpret_cast<const float4*>(space.o + at * kHeadDim)[lane];
    if (ml.x == -INFINITY) {                                    // the row saw no key in this piece (its sum is 0, or NaN)
      l += ml.y;
      continue;
    }
    const float f = exp2f(ml.x - top);
    l = fmaf(f, ml.y, l);
    o[0] = fmaf(f, v.x, o[0]); o[1] = fmaf(f, v.y, o[1]); o[2] = fmaf(f, v.z, o[2]); o[3] = fmaf(f, v.w, o[3]);
  }
  const float inv = l > 0.f ? kRsqrtD / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int u = 0; u < 4; ++u) o[u] *= inv;
  fht128_warp(o, lane);
  const int64_t at = static_cast<int64_t>(x.q_begin + t) * p.H_q + rec.tail_head * p.group + row % p.group;
  *reinterpret_cast<uint2*>(p.out + at * kHeadDim + 4 * lane) = pack_half4(o);
  if (p.lse_out && lane == 0) p.lse_out[at] = l == 0.f ? -INFINITY : (log2f(l) + top) * kLn2;
}

}  // namespace tru
}  // namespace cda

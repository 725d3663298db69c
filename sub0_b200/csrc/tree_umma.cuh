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
// Warps: four softmax groups, two K producer groups (one for 128 rows) and a V producer group of four warps each (a thread is a key), two MMA
// issuers, and two feeders that bring the slots into a ring in shared memory with tensor-map copies of 16 slots of one head.  In
// a group that waits, one warp polls and the others are parked on a named barrier, where they take no issue slots (27 polling
// warps spent a third of the kernel's instructions).
// A CTA walks an equal share of all (sequence, row block, KV head) segments' tiles; a segment that starts and ends in one CTA
// is finished there, the pieces of the others are merged by tree_merge_kernel.
//
// The reference of a row lies 2^10 below the largest score of the first tile in which it sees a key; it moves only when a later
// score is more than 2^15.5 above it (an fp16 probability ends at 2^16): then, and in a row's first tile, the group of warps
// takes the slow path, which finds the tile's row maxima across lanes and rescales O and the sums.  The distance keeps keys
// down to 2^-24 of the largest (17 nats below it) in fp16's normal range: where one key draws nearly all attention and has a
// small value row, they are the output.  (With the reference at the maximum, such an output of 1500 keys was off by 2 %.)
//
// Both sides' rows are the format's own, fp16(level * norm), from byte permutes of a key's 16 (or 4) values.  (4-bit value rows from
// a table of fp16 levels, with the norm on the probability, are rounded in another way: 138 us against 145 in the batch below, as both
// stood then.)
//
// Measured (4-bit slots, 8 KV heads, pages of 16): 16 trees of 16 tokens x 4 heads over 16k keys 141 us (slots: 20 us at copy
// bandwidth); one tree of 32 x 4 rows over 131k keys 206 us; 4 trees of 64 x 8 rows over 32k keys, 2-bit values, 718 us, 383
// TFLOP/s.  What bounds it: blocks of up to 64 rows wait for the producers -- one V group expands every tile, each K group every
// second one -- while the tensor cores are busy 17% of the time and no pipe more than 55%; blocks of 128 rows for the softmax (a
// chain of some 4500 cycles a tile) and for the clock that the power limit leaves.  A new piece costs 12 to 16 us beside its
// tiles: query rows, references, the way back, in code that has to come out of L2.
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
constexpr float kBelow = 10.0f, kSafe = 15.5f;   // largest exponents: in the tile that sets a reference, in any other
constexpr int kFeeders = 2, kFeedIdBytes = 256;   // block ids: two chunks of four tiles for each feeder
// What starting and ending a piece costs, in tiles (the share of a CTA counts it): preparing and writing out few rows is quick.
// Chains of 16 rows: 61 us with 2, 66 with 5; trees of 64 rows: 143 us with 7, 158 with 3.
template <int NR>
constexpr int kPieceCost = NR == 16 ? 2 : 7;

constexpr int kKFull = 0, kKEmpty = 2, kVFull = 4, kSFull = 6, kSEmpty = 10, kPFull = 14, kPvDone = 16, kQFull = 18, kDrained = 19, kRingFull = 20, kRingEmpty = 24;
constexpr int kOffTmemAddr = 224, kOffWait = 232, kOffPlan = 248, kOffPlanEnd = 264, kOffValid = 272, kOffIds = 320;   // inside kOffBar; valid: keys of each ring stage

template <int NR>
struct Cfg {
  // up to 64 rows: two pairs of groups take tiles in turn (streams), each with its own references, sums and O; 128 rows: all
  // four share every tile, since two O of 128 columns do not fit the tensor memory
  static constexpr int kStreams = NR == 128 ? 1 : 2;
  static constexpr int kCols = NR * kStreams / 4;                // columns of a softmax group
  static constexpr int kSBuffers = 2 * kStreams, kSShift = kStreams;   // S tiles; log2 of it
  static constexpr int kBlock = kCols < 16 ? kCols : 16;         // columns worked on at a time
  static constexpr int kOwn = NR / 4;                            // rows that a group prepares and writes out,
  static constexpr int kChunk = kOwn < 16 ? kOwn : 16;           // so many at a time
  static constexpr int kSoftWarps = 16;                          // four softmax groups; two K groups and one V group follow
  static constexpr int kKGroups = NR == 128 ? 1 : 2, kWarpK = kSoftWarps, kWarpV = kWarpK + 4 * kKGroups, kWarpS = kWarpV + 4, kWarpO = kWarpS + 1, kWarpFeed = kWarpO + 1;
  static constexpr int kThreads = (kWarpFeed + kFeeders) * 32;   // 32 or 28 warps: registers are handed out by four
  // Registers a thread: softmax takes what the others give back.  32 warps start with 64 (16 x 80 + 16 x 48 a lane; with 88 and 40
  // producers have fewer look-ups in flight: 16 trees of 64 rows 143 us against 138); blocks of 128 rows, whose softmax has the
  // longest chain, do with one K group: 28 warps start with 72 (4 trees of 512 rows 705 us; with two K groups, 88 and 40, 763 us;
  // with 80 and 56 757 us, with 96 and 40 841 us; all with references at the maximum, 718 us as it stands)
  static constexpr int kRegsSoft = NR == 128 ? 88 : 80, kRegsOther = 48;
  static constexpr int kRegsAll = 32 * (kSoftWarps * kRegsSoft + (kThreads / 32 - kSoftWarps) * kRegsOther);   // may not exceed the launch's
  static constexpr int kRing = NR == 128 ? 2 : 4;
  static_assert(kRing % 2 == 0, "one K group reads a stage, and so sees every phase of its barrier");
  static constexpr int kTmemCols = 512;                          // tensor memory: two K, the S, one O for each stream
  static constexpr int kColK = 0, kColS = 128, kColO = kColS + kSBuffers * NR;
  // shared memory (bytes from a 1024-aligned base)
  static constexpr int kOffV = 0, kOffP = 2 * kTileBytes, kOffQ = kOffP + 2 * kColBlock,   // P: one of 64 rows for each stream, or one of 128
                        kOffRing = kOffQ + NR * 512;
  static constexpr int kOffRef = kOffRing + kRing * kStageBytes;  // words of the rows, of two pieces in turn: negated references
  static constexpr int kOffPos = kOffRef + 16 * NR;               //   (of both groups), position,
  static constexpr int kOffSlope = kOffPos + 8 * NR;              //   slope x log2 e,
  static constexpr int kOffMask = kOffSlope + 8 * NR;             //   64-bit ancestor mask
  static constexpr int kOffFac = kOffMask + 16 * NR;              // 2 x NR floats: factors of a slow path
  static constexpr int kOffMax = kOffFac + 8 * NR;                // 4 warps x (kStreams x NR) floats: maxima, sums
  static constexpr int kOffCmb = kOffMax + 16 * NR * kStreams;               // 4 x NR floats: how the groups' results are put together
  static constexpr int kOffBad = kOffCmb + 16 * NR;               // 8 tiles x 128 bits: keys whose value row is not finite
  static constexpr int kOffLevels = kOffBad + 128;                // 2 x 16 floats, and the largest of V
  static constexpr int kOffBox = kOffLevels + 144;               // two boxes for each softmax warp
  static constexpr int kOffBar = kOffBox + 128 * kSoftWarps;                // barriers, TMEM address, wait state, plan
  static constexpr int kSmemBytes = kOffBar + kOffIds + kFeeders * kFeedIdBytes + 1024;
  static_assert(kSmemBytes <= 232448, "one CTA's shared memory");
};

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
__device__ __forceinline__ uint32_t lds32(uint32_t a) {          // (not volatile: look-ups in a table that is complete)
  uint32_t v;
  asm("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds_u(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
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
// Named barriers: 1 .. 4 the softmax groups, 5 all of them; 6 the V producers; 7, 8 the K producers.
__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
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
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&v)[N]) {
  if constexpr (N == 4) tmem_ld4(addr, v);
  else if constexpr (N == 8) tmem_ld8(addr, v);
  else tmem_ld16(addr, v);
}
template <int N>
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t (&v)[N]) {
  if constexpr (N == 8) tmem_st8(addr, v);
  else tmem_st16(addr, v);
}

// A bounded wait for a barrier phase.  Attempts carry no time hint (with one, an attempt is a software loop that sleeps: it
// wakes late and takes issue slots), and abort flag and clock are read after every eight.  Once a wait of the CTA has given up,
// every later one does so after eight attempts: all roles then run their loops to the end (so nobody is left at a named
// barrier) without issuing or writing anything.
__device__ __forceinline__ bool try_eight(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra D;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "D:\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile WaitState* ws) {
  if (try_eight(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
#pragma unroll 1
  while (!ws->abort && global_timer_ns() - t0 <= ws->limit_ns)
    if (try_eight(bar, parity)) return true;
  ws->abort = 1;
  return false;
}

// Whether the value row of a key -- its codes at `codes` in shared memory -- holds a coordinate that fp16 cannot (it rounds what
// is 65520 or more to infinity).  The largest level, behind the 16 levels, decides nearly always.  Such a row would make NaN of
// the zero probabilities of the rows that do not see its key: it is taken as zeros, and the probabilities of the others are
// made NaN.
__device__ __forceinline__ bool row_not_finite(uint32_t codes, int bits, uint32_t levels, float norm) {
  if (lds_f(levels + 64) * fabsf(norm) < 65520.0f) return false;
  bool bad = false;
#pragma unroll 1
  for (int at = 0; at < 128 * bits; at += bits) {
    const uint32_t code = lds_u(codes + at / 32 * 4) >> (at & 31) & ((1u << bits) - 1u);
    bad = bad || !(fabsf(lds_f(levels + 4 * code) * norm) < 65520.0f);
  }
  return bad;
}

// Sums of M values per lane over the warp's 32 lanes: lane l returns the total of value l % M (M - 1 + log2(32 / M) exchanges
// where one butterfly per value would take 5 M).
template <int M>
__device__ __forceinline__ float transposed_sum(float (&v)[M], int lane) {
#pragma unroll
  for (int d = M / 2; d > 0; d >>= 1) {
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int j = 0; j < d; ++j) v[j] = (upper ? v[j + d] : v[j]) + __shfl_xor_sync(0xffffffffu, upper ? v[j] : v[j + d], d);
  }
#pragma unroll
  for (int d = M; d < 32; d <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
  return v[0];
}
template <int R>
__device__ __forceinline__ void raise_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void lower_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
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
// An entry without tiles is behind its sequence's last row: so are those up to the next sequence.  (A call that allows far more new
// tokens than a sequence brings has hundreds of thousands of them, longer to step through than a wait may take.)
__device__ __forceinline__ int after_empty(const AttendParams& p, int b) { return (b + 1) * p.row_blocks; }
struct Piece { Entry x; int e, head, tile0, n; bool starts, ends; };
// What a softmax warp needs of a piece at its start and end, and where its walk stands, in shared memory (a box for each warp):
// held in registers they were spilled, and every start and end of a piece waited for L2 (1024 threads' stacks fit no L1).
struct Box { int rb, q_begin, q_len, ctx, seq_len, t0, head, e, tile0, n, edges, walk_e, walk_h, walk_j, walk_left, pad; };
template <int NR>
struct Walk {
  int e, h, j, left, entries;
  __device__ __forceinline__ bool next(const AttendParams& p, Piece& q) {
    while (left > 0 && e < entries) {
      q.x = entry_of<NR>(p, e);
      if (q.x.tiles == 0) { e = after_empty(p, q.x.b); continue; }
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

// Share of this CTA.  All segments are laid end to end, each with kPieceCost empty positions in front of its tiles, and the line
// is cut into equal parts: CTAs that serve more segments get fewer tiles.  s_plan: first entry, head, tile; s_end: tiles.
template <int NR, int THREADS>
__device__ __forceinline__ void find_share(const AttendParams& p, int2* s_scan, int* s_plan, int* s_end) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, entries = p.B * p.row_blocks;
  const int per = (entries + THREADS - 1) / THREADS, e0 = min(tid * per, entries), e1 = e0 + min(per, entries - e0);
  int tiles = 0, used = 0;                                       // of this thread's entries, one head: tiles, entries with any
  for (int e = e0; e < e1;) {
    const Entry x = entry_of<NR>(p, e);
    tiles += x.tiles;
    used += x.tiles > 0;
    if (blockIdx.x == 0 && x.rb == 0 && sequence_view(p, x.b).bad) atomicOr(&g_tree_status, kStatusLengths);
    e = x.tiles > 0 ? e + 1 : after_empty(p, x.b);
  }
  int x = tiles, y = used;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) { x += u; y += v; }
  }
  if (lane == 31) s_scan[warp] = make_int2(x, y);
  __syncthreads();
  const int2 s = lane < THREADS / 32 ? s_scan[lane] : make_int2(0, 0);   // a lane for every warp's total
  const int tiles_before = x - tiles + __reduce_add_sync(0xffffffffu, lane < warp ? s.x : 0);
  const int used_before = y - used + __reduce_add_sync(0xffffffffu, lane < warp ? s.y : 0);
  const int all_tiles = __reduce_add_sync(0xffffffffu, s.x), all_used = __reduce_add_sync(0xffffffffu, s.y);
  const int64_t line = (all_tiles + static_cast<int64_t>(kPieceCost<NR>) * all_used) * p.H_kv;
  const int busy = static_cast<int>(line < gridDim.x ? line : gridDim.x), cta = min(static_cast<int>(blockIdx.x), busy);
  const int64_t each = busy ? line / busy : 0, over = line - each * busy;           // the first `over` CTAs take one more
  const int64_t lo = each * cta + min(static_cast<int64_t>(cta), over), hi = cta < busy ? lo + each + (cta < over ? 1 : 0) : lo;
  if (tid == 0) s_plan[3] = *s_end = 0;
  __syncthreads();
  int64_t at = (tiles_before + static_cast<int64_t>(kPieceCost<NR>) * used_before) * p.H_kv;
  const int64_t mine = (tiles + static_cast<int64_t>(kPieceCost<NR>) * used) * p.H_kv;
  if (hi > lo && hi > at && lo < at + mine) {                    // the line's positions lo or hi - 1 may lie in these entries
    int real = tiles_before * p.H_kv;
    for (int e = e0, after; e < e1; e = after) {
      const Entry x = entry_of<NR>(p, e);
      const int n = x.tiles, len = n + kPieceCost<NR>;
      after = n > 0 ? e + 1 : after_empty(p, x.b);
      if (n == 0) continue;
      const int64_t next = at + static_cast<int64_t>(len) * p.H_kv;
      if (at <= lo && lo < next) {
        const int h = static_cast<int>(lo - at) / len, j = max(static_cast<int>(lo - at) % len - kPieceCost<NR>, 0);
        s_plan[0] = e; s_plan[1] = h; s_plan[2] = j;
        s_plan[3] = real + h * n + j;
      }
      if (at < hi && hi <= next) {
        const int h = static_cast<int>(hi - at) / len, j = max(static_cast<int>(hi - at) % len - kPieceCost<NR>, 0);
        *s_end = real + h * n + j;
      }
      at = next;
      real += n * p.H_kv;
    }
  }
  __syncthreads();
  if (tid == 0) s_plan[3] = *s_end - s_plan[3];
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

// Tiles [tile0, tile0 + n) of a piece, as the feeders see it.
struct Feed { int b, head, seq_len, tile0, n; };
// A feeder warp: copies every kFeeders-th tile of the CTA's walk to the ring, one lane per 16-token group.  A lane's copy takes
// about 90 cycles to issue, eight of them and the stage's bookkeeping 1250: two warps, or the ring is never full
// (4 trees of 512 rows: 734 us with one, 703 with two).  Block ids
// come four tiles at a time (one a lane), asynchronously into shared memory while the chunk before them is copied -- a load into a
// register was waited for at once, 2000 cycles under load -- across the end of a piece too.  Each feeder sees every phase of its
// stages' barriers.
template <int RING, class Next>
__device__ __forceinline__ void feed_ring(const AttendParams& p, const CUtensorMap* map, Next next, int which, uint32_t ring, uint32_t full, uint32_t empty,
                                          volatile int* valid, int32_t* ids, volatile WaitState* wait) {
  static_assert(RING % kFeeders == 0, "one feeder for each stage");
  const int lane = threadIdx.x & 31;
  const uint32_t ids_at = smem_addr(ids) + kFeedIdBytes * which + 4 * lane;
  auto fetch_ids = [&](const Feed& f, int k, int half) {        // tokens past the end: the last one's block
    const int n = min((f.tile0 + k) * kKeys + 16 * lane, f.seq_len - 1);
    const int32_t* from = p.block_table + static_cast<int64_t>(f.b) * p.bt_stride + (p.bs_shift >= 0 ? n >> p.bs_shift : n / p.block_size);
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ids_at + 128 * half), "l"(from) : "memory");
  };
  Feed f, after;
  bool live = next(f), bad = false, alive = true;
  int issued = 0, half = 0, k = 0;
  if (live) fetch_ids(f, 0, 0);
  asm volatile("cp.async.commit_group;" ::: "memory");
  while (live && alive) {
    const bool more = k + 4 < f.n;
    if (more) fetch_ids(f, k + 4, half ^ 1);
    else {
      live = next(after);
      if (live) fetch_ids(after, 0, half ^ 1);
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;" ::: "memory");
    uint32_t id4;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(id4) : "r"(ids_at + 128 * half) : "memory");
#pragma unroll 1
    for (const int end = min(k + 4, f.n), k0 = k; k < end; ++k, ++issued) {
      if (issued % kFeeders != which) continue;
      const int tile = f.tile0 + k, stage = issued % RING, turn = issued / RING;
      // (after a wait elsewhere gave up, producers free stages whose copies may still be on the way: no copy may follow those)
      if (turn > 0) alive = wait_for(empty + 8 * stage, (turn - 1) & 1, wait) && !wait->abort;
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      const int left = f.seq_len - tile * kKeys, groups = min(8, (left + 15) >> 4), n = tile * kKeys + 16 * (lane & 7);
      int id = static_cast<int>(__shfl_sync(0xffffffffu, id4, 8 * (k - k0) + (lane & 7)));
      if (lane == 0) {
        valid[stage] = min(left, kKeys);
        expect_bytes(full + 8 * stage, groups * 16 * p.slot_bytes);
      }
      __syncwarp();
      if (lane < groups) {
        if (static_cast<unsigned>(id) >= static_cast<unsigned>(p.num_blocks)) { bad = true; id = 0; }
        const int in = p.bs_shift >= 0 ? n & (p.block_size - 1) : n % p.block_size;
        copy_group(ring + stage * kStageBytes + lane * 16 * p.slot_bytes, map, f.head * p.slot_bytes, id * p.block_size + in, full + 8 * stage);
      }
      __syncwarp();
    }
    half ^= 1;
    if (!more) { f = after; k = 0; }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (bad) atomicOr(&g_tree_status, kStatusBadBlock);
  // no copy may be in flight when the CTA ends, also after a wait elsewhere gave up
  const unsigned long long t0 = global_timer_ns();
  for (int i = max(0, issued - RING); i < issued; ++i)
    if (i % kFeeders == which)
      while (!mbar_try_wait(full + 8 * (i % RING), (i / RING) & 1) && global_timer_ns() - t0 < kWaitLimitNs) { }
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

  // (the lengths' way from memory is long: what does not need them goes first)
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {                               // counts: warps that arrive, or one commit
      mbar_init(bar(kKFull + i), 4 + withheld(p, i)); mbar_init(bar(kKEmpty + i), 1); mbar_init(bar(kVFull + i), 4);
      mbar_init(bar(kPFull + i), C::kSoftWarps / C::kStreams); mbar_init(bar(kPvDone + i), 1);
    }
    for (int i = 0; i < C::kSBuffers; ++i) { mbar_init(bar(kSFull + i), 1); mbar_init(bar(kSEmpty + i), C::kSoftWarps / C::kStreams); }
    mbar_init(bar(kQFull), C::kSoftWarps);
    mbar_init(bar(kDrained), 2);
    for (int i = 0; i < C::kRing; ++i) { mbar_init(bar(kRingFull + i), 1); mbar_init(bar(kRingEmpty + i), 8); }
    wait->abort = 0;
    wait->limit_ns = p.wait_limit_ns;
    mbar_init_fence();
  }
  if (tid < 32) {                                               // code levels: 16 or 4 of K, then of V
    const int side = tid >> 4, i = tid & 15, n = (side ? p.v_bits : p.k_bits) == 4 ? 16 : 4;
    const float level = i < n ? __ldg((side ? p.cb_v : p.cb_k) + i) : 0.f, top = warp_max(side ? fabsf(level) : 0.f);
    reinterpret_cast<float*>(sm + C::kOffLevels)[tid] = level;
    if (tid == 0) reinterpret_cast<float*>(sm + C::kOffLevels)[32] = top;
  }
  if (warp == C::kWarpS) {
    tmem_alloc(base + C::kOffBar + kOffTmemAddr, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  find_share<NR, C::kThreads>(p, reinterpret_cast<int2*>(sm + C::kOffP), s_plan, reinterpret_cast<int*>(sm + C::kOffBar + kOffPlanEnd));
  tc_fence_after_sync();
  const int total = s_plan[3];
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + C::kOffBar + kOffTmemAddr);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge may take its places; it waits for this kernel's end
  if (total == 0) {
    if (tid == 0) space.rec[blockIdx.x] = Record{-1, 0, 0, 0};
    if (warp == C::kWarpS) tmem_dealloc(tmem, C::kTmemCols);
    return;
  }
  Walk<NR> w{s_plan[0], s_plan[1], s_plan[2], total, p.B * p.row_blocks};
  Record rec{-1, 0, 0, 0};

  if (warp < C::kSoftWarps) {
    // ============ softmax: a thread is a key (tensor-memory lane), the rows of the block are columns.  Two groups share a tile,
    // half of the columns each, and the pairs take tiles in turn, each with its own references, sums and O: a group's chain of
    // waits and barriers spans two tiles =====================================================================================
    raise_registers<C::kRegsSoft>();
    const int group = warp >> 2, stream = C::kStreams == 2 ? group & 1 : 0, col0 = (C::kStreams == 2 ? group >> 1 : group) * C::kCols;
    const int own0 = col0 + stream * C::kOwn;
    const int key = (warp & 3) * 32 + lane, gtid = tid & 127;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t fac_a = base + C::kOffFac + 4 * C::kCols * group, max_a = base + C::kOffMax + 16 * C::kCols * group;
    const float kf = p.scale * kLog2e, cap2 = p.softcap * kLog2e, inv_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
    constexpr int kRowsWarp = C::kOwn / 4, kPair = kRowsWarp < 2 ? 1 : 2;
    volatile Box* boxes = reinterpret_cast<volatile Box*>(sm + C::kOffBox) + 2 * warp;   // the piece in work, the one after it
    auto next_piece = [&](int from, int into) {                 // the walk goes on from the state in one box; the piece into the other
      volatile Box &a = boxes[from], &b = boxes[into];
      Walk<NR> at{a.walk_e, a.walk_h, a.walk_j, a.walk_left, p.B * p.row_blocks};
      Piece q;
      const bool any = at.next(p, q);
      __syncwarp();
      if (any && lane == 0) {
        b.rb = q.x.rb; b.q_begin = q.x.q_begin; b.q_len = q.x.q_len; b.ctx = q.x.ctx; b.seq_len = q.x.seq_len; b.t0 = q.x.t0;
        b.head = q.head; b.e = q.e; b.tile0 = q.tile0; b.n = q.n; b.edges = (q.starts ? 2 : 0) + (q.ends ? 1 : 0);
        b.walk_e = at.e; b.walk_h = at.h; b.walk_j = at.j; b.walk_left = at.left;
      }
      __syncwarp();
      return any;
    };
    auto place = [&](const volatile Box& q, int r, int& t) {    // row r of the block: its token, and its index in (T, H_q)
      const int row = q.rb * NR + r;
      t = p.group == 1 ? row : static_cast<int>(__umulhi(static_cast<uint32_t>(row), p.group_magic));
      return static_cast<int64_t>(q.q_begin + t) * p.H_q + q.head * p.group + (row - t * p.group);
    };
    // The query rows and row words of a piece are prepared by the group that owns the rows: loads first, the rest later.
    auto load_rows = [&](const volatile Box& q, uint2 (&rows)[kRowsWarp]) {
#pragma unroll
      for (int u = 0; u < kRowsWarp; ++u) {
        int t;
        const int64_t at = place(q, own0 + 4 * u + (warp & 3), t);
        rows[u] = make_uint2(0u, 0u);
        if (t < q.q_len) rows[u] = __ldg(reinterpret_cast<const uint2*>(p.q + at * kHeadDim) + lane);
      }
    };
    auto prepare_rows = [&](const volatile Box& q, uint2 (&rows)[kRowsWarp], int set) {
      if (gtid < C::kOwn) {
        int t;
        const int64_t at = place(q, own0 + gtid, t);
        const bool real = t < q.q_len;
        const int r = set * NR + own0 + gtid;
        const unsigned long long m = real && p.tree_mask ? static_cast<unsigned long long>(p.tree_mask[q.q_begin + t]) : 0ull;
        reinterpret_cast<unsigned long long*>(sm + C::kOffMask)[r] = m;
        reinterpret_cast<int*>(sm + C::kOffPos)[r] = q.ctx + (!real ? 0 : p.tree_mask ? max(__popcll(m) - 1, 0) : t);
        reinterpret_cast<float*>(sm + C::kOffSlope)[r] = p.slopes && real ? p.slopes[at % p.H_q] * kLog2e : 0.f;
        float* ref = reinterpret_cast<float*>(sm + C::kOffRef) + 2 * set * NR + own0 + gtid;
        ref[0] = ref[NR] = kNoRef;
      }
      // two rows at a time, in a loop: what runs once a piece is kept short, or it comes out of L2 line by line each time
#pragma unroll 1
      for (int u = 0; u < kRowsWarp; u += kPair) {
        float f[kPair][4];
#pragma unroll
        for (int v = 0; v < kPair; ++v) {
          const __half2 a = *reinterpret_cast<const __half2*>(&rows[v].x), b = *reinterpret_cast<const __half2*>(&rows[v].y);
          f[v][0] = __low2float(a); f[v][1] = __high2float(a); f[v][2] = __low2float(b); f[v][3] = __high2float(b);
        }
#pragma unroll
        for (int v = 0; v + kPair < kRowsWarp; ++v) rows[v] = rows[v + kPair];
#pragma unroll
        for (int v = 0; v < kPair; ++v) fht128_warp(f[v], lane);
#pragma unroll
        for (int v = 0; v < kPair; ++v) {
          float lo[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            f[v][c] *= kRsqrtD;
            lo[c] = f[v][c] - round_to_half(f[v][c]);
          }
          const uint2 h = pack_half4(f[v]), l = pack_half4(lo);
          const uint32_t at = base + C::kOffQ + (lane >> 4) * (NR * 128) + sw128(own0 + 4 * (u + v) + (warp & 3), (lane & 15) >> 1) + 8 * (lane & 1);
          sts64(at, h.x, h.y);
          sts64(at + NR * 256, l.x, l.y);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kQFull));
    };
    const int my_o = C::kColO + stream * NR + col0;
    int done = 0, set = 0;                                      // tiles of the pieces so far; which set of row words
    uint2 rows[kRowsWarp];
    if (lane == 0) { boxes[1].walk_e = w.e; boxes[1].walk_h = w.h; boxes[1].walk_j = w.j; boxes[1].walk_left = w.left; }
    __syncwarp();
    bool more = next_piece(1, 0);
    if (more) {
      load_rows(boxes[0], rows);
      prepare_rows(boxes[0], rows, set);
    }
    while (more) {
      const volatile Box& pc = boxes[set];
      named_barrier(5, 512);                                    // the row words of both groups
      const int ctx = pc.ctx, seq_len = pc.seq_len, end = done + pc.n;
      const uint32_t ref_a = base + C::kOffRef + 4 * ((2 * set + stream) * NR + col0);
      const int* pos_w = reinterpret_cast<const int*>(sm + C::kOffPos) + set * NR + col0;
      const float* slope_w = reinterpret_cast<const float*>(sm + C::kOffSlope) + set * NR + col0;
      const uint32_t* mask_w = reinterpret_cast<const uint32_t*>(sm + C::kOffMask) + 2 * (set * NR + col0);
      // tiles (by their number in all pieces) whose keys every row sees: [see_lo, see_hi)
      const int tile_at = pc.tile0 - done;                      // key tile = number + tile_at
      const int see_hi = p.slopes ? done : (ctx + (p.tree_mask ? 0 : pc.t0 + 1)) / kKeys - tile_at;
      const int see_lo = p.window > 0 ? max(0, ctx + positions_of(p, pc.q_len) - p.window + kKeys) / kKeys - tile_at : done;
      uint64_t sum[C::kCols / 2];
#pragma unroll
      for (int c = 0; c < C::kCols / 2; ++c) sum[c] = f2_pack(0.f, 0.f);
      uint32_t s[C::kBlock];                                    // raw scores of the next tile's first block, in flight
      auto fetch = [&](int tile) {
        if ((warp & 3) == 0) wait_for(bar(kSFull + (tile & (C::kSBuffers - 1))), (tile >> C::kSShift) & 1, wait);
        if (C::kStreams == 2 && (warp & 3) == 1 && tile >= 2) wait_for(bar(kPvDone + stream), ((tile - 2) >> 1) & 1, wait);   // P and O of the stream's last tile are at rest
        group_barrier(group);
        tc_fence_after_sync();
        tmem_load<C::kBlock>(lanes + C::kColS + (tile & (C::kSBuffers - 1)) * NR + col0, s);
      };
      int i = C::kStreams == 2 ? done + ((done ^ stream) & 1) : done;     // this group's tiles: those of its parity, or all
      const bool any_tile = i < end;
      if (any_tile) fetch(i);

#pragma unroll 1
      for (bool first = true; i < end; i += C::kStreams, first = false) {
        const bool rule = i >= see_hi || i < see_lo, finish = rule || p.softcap > 0.f;
        if (finish) {                                           // cap, bias and masks, in the base-2 domain, eight columns at a time
          const int n = (i + tile_at) * kKeys + key, j = n - ctx;
          const int pos_k = rule && p.tree_mask && j >= 0 && n < seq_len ? ctx + depth_of(p, pc.q_begin, j) : n;
          const int word = (j >> 5) & 1, up = 31 - (j & 31);    // bit j of a row's mask to the sign
          const uint32_t all = j < 0 ? 0x80000000u : 0u, none = n < seq_len ? 0xffffffffu : 0u;
          const float f1 = p.softcap > 0.f ? inv_cap : kf;
#pragma unroll 1
          for (int c0 = 0; c0 < C::kCols; c0 += 8) {
            const uint32_t at = lanes + C::kColS + (i & (C::kSBuffers - 1)) * NR + col0 + c0;
            uint32_t x[8];
            tmem_load<8>(at, x);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 8; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * f1);
            if (p.softcap > 0.f) {
#pragma unroll
              for (int c = 0; c < 8; ++c) x[c] = __float_as_uint(cap2 * soft_tanh(__uint_as_float(x[c])));
            }
            if (rule) {
              if (p.slopes) {
#pragma unroll
                for (int c = 0; c < 8; ++c) x[c] = __float_as_uint(fmaf(slope_w[c0 + c], static_cast<float>(pos_k - pos_w[c0 + c]), __uint_as_float(x[c])));
              }
              if (p.window > 0) {
#pragma unroll
                for (int c = 0; c < 8; ++c) x[c] = pos_w[c0 + c] - pos_k >= p.window ? 0xff800000u : x[c];
              }
              if (p.tree_mask) {
#pragma unroll
                for (int c = 0; c < 8; ++c) x[c] = static_cast<int>(((mask_w[2 * (c0 + c) + word] << up) | all) & none) < 0 ? x[c] : 0xff800000u;
              } else {
#pragma unroll
                for (int c = 0; c < 8; ++c) x[c] = n > pos_w[c0 + c] || n >= seq_len ? 0xff800000u : x[c];
              }
            }
            tmem_store<8>(at, x);
          }
          tmem_wait_st();
          tmem_load<C::kBlock>(lanes + C::kColS + (i & (C::kSBuffers - 1)) * NR + col0, s);      // instead of the raw ones
        }
        const uint64_t ff = f2_pack(finish ? 1.0f : kf, finish ? 1.0f : kf);
        const uint32_t p_tile = base + C::kOffP + (C::kStreams == 2 ? stream : col0 >> 6) * kColBlock;
#pragma unroll
        for (int blk = 0; blk < C::kCols / C::kBlock; ++blk) {
          const int c0 = blk * C::kBlock;
          float e[C::kBlock];
#pragma unroll 1
          for (bool again = first;; again = true) {              // a first tile has no references: the slow path at once
            if (blk > 0 || again) tmem_load<C::kBlock>(lanes + C::kColS + (i & (C::kSBuffers - 1)) * NR + col0 + c0, s);
            tmem_wait_ld();
            if (again) {
              // slow path: row maxima of the tile, new references, factors for what the rows hold already
              float top = 0.f;
#pragma unroll
              for (int c = 0; c < C::kBlock; ++c) {
                const float m = warp_max(__uint_as_float(s[c]) * (finish ? 1.0f : kf));
                top = lane == c ? m : top;
              }
              if (lane < C::kBlock) sts_f(max_a + 4 * ((warp & 3) * C::kCols + lane), top);
              group_barrier(group);
              if (gtid < C::kBlock) {
                float m = lds_f(max_a + 4 * gtid);
#pragma unroll
                for (int u = 1; u < 4; ++u) m = fmaxf(m, lds_f(max_a + 4 * (u * C::kCols + gtid)));
                const float old = lds_f(ref_a + 4 * (c0 + gtid));
                float fac = 1.0f;
                if (m + old > kSafe) {
                  fac = old == kNoRef ? 0.f : fast_exp2(kBelow - m - old);
                  sts_f(ref_a + 4 * (c0 + gtid), kBelow - m);
                }
                sts_f(fac_a + 4 * (c0 + gtid), fac);
              }
              group_barrier(group);
            }
            // probabilities against the references as they are; `excess`: the largest exponent
            float excess = -INFINITY;
#pragma unroll
            for (int c = 0; c < C::kBlock; c += 4) {
              const uint4 r = lds128(ref_a + 4 * (c0 + c));
              float* a = e + c;
              f2_unpack(f2_fma(f2_pack(s[c], s[c + 1]), ff, f2_pack(r.x, r.y)), a[0], a[1]);
              f2_unpack(f2_fma(f2_pack(s[c + 2], s[c + 3]), ff, f2_pack(r.z, r.w)), a[2], a[3]);
              excess = fmax3(excess, a[0], a[1]);
              excess = fmax3(excess, a[2], a[3]);
#pragma unroll
              for (int u = 0; u < 4; ++u) a[u] = fast_exp2(a[u]);
            }
            if (C::kStreams == 1 && blk == 0 && again == first && i >= 1) {       // P and O of the last tile are at rest
              if ((warp & 3) == 0) wait_for(bar(kPvDone + ((i - 1) & 1)), ((i - 1) >> 1) & 1, wait);
              group_barrier(group);
              tc_fence_after_sync();
            }
#pragma unroll
            for (int c = 0; c < C::kBlock; c += 8)
              sts128(p_tile + sw128(key, ((col0 & 63) + c0 + c) / 8), pack_half2(e[c], e[c + 1]), pack_half2(e[c + 2], e[c + 3]),
                     pack_half2(e[c + 4], e[c + 5]), pack_half2(e[c + 6], e[c + 7]));
            if (again) {
#pragma unroll
              for (int c = 0; c < C::kBlock; c += 4) {
                const uint4 r = lds128(fac_a + 4 * (c0 + c));
                sum[(c0 + c) / 2] = f2_mul(sum[(c0 + c) / 2], f2_pack(r.x, r.y));
                sum[(c0 + c) / 2 + 1] = f2_mul(sum[(c0 + c) / 2 + 1], f2_pack(r.z, r.w));
              }
              if (!first) {                                     // O of the group's tiles so far (at rest, see fetch)
                uint32_t o[C::kBlock];
                tmem_load<C::kBlock>(lanes + my_o + c0, o);
                tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < C::kBlock; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * lds_f(fac_a + 4 * (c0 + c)));
                tmem_store<C::kBlock>(lanes + my_o + c0, o);
                tmem_wait_st();
              }
              break;
            }
            if (!group_any(group, excess > kSafe)) break;
          }
#pragma unroll
          for (int c = 0; c < C::kBlock; c += 2) sum[(c0 + c) / 2] = f2_add(sum[(c0 + c) / 2], f2_pack(e[c], e[c + 1]));
        }
        if (const uint32_t bad_keys = lds_u(base + C::kOffBad + 16 * (i & 7) + 4 * (warp & 3))) {
#pragma unroll 1
          for (int c0 = 0; c0 < C::kCols; c0 += 8) {            // a value row that is not finite: NaN for the rows that see the key
            uint32_t x[8];
            tmem_load<8>(lanes + C::kColS + (i & (C::kSBuffers - 1)) * NR + col0 + c0, x);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 8; ++c) x[c] = x[c] == 0xff800000u ? 0u : 0x7fffu;
            if (bad_keys >> lane & 1u)
              sts128(p_tile + sw128(key, ((col0 & 63) + c0) / 8), x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16);
          }
        }
        fence_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(kSEmpty + (i & (C::kSBuffers - 1))));
          mbar_arrive(bar(kPFull + (i & 1)));
        }
        if (i + C::kStreams < end) fetch(i + C::kStreams);
      }

      // ---- end of the piece.  The next piece's rows go first: its scores can then be computed while this one is written out
      more = next_piece(set, set ^ 1);
      if (more) load_rows(boxes[set ^ 1], rows);
      if (any_tile) {
#pragma unroll
        for (int c0 = 0; c0 < C::kCols; c0 += C::kBlock) {
          float v[C::kBlock];
#pragma unroll
          for (int c = 0; c < C::kBlock; c += 2) f2_unpack(sum[(c0 + c) / 2], v[c], v[c + 1]);
          const float l = transposed_sum<C::kBlock>(v, lane);
          if (lane < C::kBlock) sts_f(max_a + 4 * ((warp & 3) * C::kCols + c0 + lane), l);
        }
      }
      if ((warp & 3) == 0) {                                    // both S of this piece are done before Q is overwritten
        const int last = end - 1, before = end - 2;
        if (more) wait_for(bar(kSFull + (last & (C::kSBuffers - 1))), (last >> C::kSShift) & 1, wait);
        if (any_tile) {
          const int mine = C::kStreams == 1 || ((last ^ stream) & 1) == 0 ? last : before;
          wait_for(bar(kPvDone + (mine & 1)), (mine >> 1) & 1, wait);
        }
      }
      named_barrier(5, 512);
      tc_fence_after_sync();
      if (more) prepare_rows(boxes[set ^ 1], rows, set ^ 1);
      // the two streams of every own row: sums, common reference, factors
      const bool both = C::kStreams == 2 && pc.n > 1, only = C::kStreams == 2 && (done & 1) != 0;       // with a single tile one stream is empty
      float* cmb = reinterpret_cast<float*>(sm + C::kOffCmb);   // [factor 0, factor 1, sum, reference][NR]
      if (gtid < C::kOwn) {
        const int r = own0 + gtid;
        const float* ref = reinterpret_cast<const float*>(sm + C::kOffRef) + 2 * set * NR + r;
        float m[2], l[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          m[g] = -INFINITY;
          l[g] = 0.f;
          if (g < C::kStreams && (both || only == (g == 1))) {
            const float* part = reinterpret_cast<const float*>(sm + C::kOffMax) + 4 * C::kCols * (C::kStreams == 2 ? (group & 2) + g : group) + (r - col0);
            l[g] = part[0] + part[C::kCols] + part[2 * C::kCols] + part[3 * C::kCols];
            m[g] = ref[g * NR] == kNoRef ? -INFINITY : -ref[g * NR];
          }
        }
        const float top = fmaxf(m[0], m[1]);
        const float f0 = m[0] == -INFINITY ? 0.f : exp2f(m[0] - top), f1 = m[1] == -INFINITY ? 0.f : exp2f(m[1] - top);
        // (a row without a reference has the sum 0, or NaN from NaN scores, which the factor 0 keeps)
        cmb[r] = f0;
        cmb[NR + r] = f1;
        cmb[2 * NR + r] = (m[0] == -INFINITY ? l[0] : f0 * l[0]) + (m[1] == -INFINITY ? l[1] : f1 * l[1]);
        cmb[3 * NR + r] = top;
      }
      group_barrier(group);
      const int edges = pc.edges;
      const bool alive = wait->abort == 0, whole = edges == 3, starts = (edges & 2) != 0;
      const int64_t slot = static_cast<int64_t>(2) * blockIdx.x + (starts ? 1 : 0);
      if (!whole) {
        if (starts) { rec.tail_e = pc.e; rec.tail_head = pc.head; }
        else rec.head_state = (edges & 1) ? 2 : 1;
        if (gtid < C::kOwn && alive)
          space.ml[slot * NR + own0 + gtid] = make_float2(cmb[3 * NR + own0 + gtid], cmb[2 * NR + own0 + gtid]);
      }
#pragma unroll 1
      for (int ch = own0; ch < own0 + C::kOwn; ch += C::kChunk) {
        float o[C::kChunk];
        {
          uint32_t a[C::kChunk];
          tmem_load<C::kChunk>(lanes + C::kColO + (both || !only ? 0 : NR) + ch, a);
          tmem_wait_ld();
          const float* f = cmb + (both || !only ? 0 : NR) + ch;
#pragma unroll
          for (int c = 0; c < C::kChunk; ++c) o[c] = __uint_as_float(a[c]) * f[c];
          if (both) {
            tmem_load<C::kChunk>(lanes + C::kColO + NR + ch, a);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < C::kChunk; ++c) o[c] = fmaf(__uint_as_float(a[c]), cmb[NR + ch + c], o[c]);
          }
        }
        if (!whole) {                                           // un-normalised, one row of 128 per column
          float* to = space.o + (slot * NR + ch) * kHeadDim + key;
          if (alive) {
#pragma unroll
            for (int c = 0; c < C::kChunk; ++c) to[c * kHeadDim] = o[c];
          }
          continue;
        }
        // transpose through the (idle) P buffers, rotate back in fp32, round once
        const uint32_t area = base + C::kOffP + group * (C::kChunk * 512);
        constexpr int kRowsChunk = C::kChunk / 4;
        if (ch > own0) group_barrier(group);
#pragma unroll
        for (int c = 0; c < C::kChunk; ++c) sts_f(area + c * 512 + key * 4, o[c]);
        group_barrier(group);
        constexpr int kTwo = kRowsChunk < 2 ? 1 : 2;
#pragma unroll 1
        for (int u0 = 0; u0 < kRowsChunk; u0 += kTwo) {
          float v[kTwo][4];
#pragma unroll
          for (int u = 0; u < kTwo; ++u) {
            const int r = 4 * (u0 + u) + (warp & 3);
            const float l = cmb[2 * NR + ch + r], inv = l > 0.f ? kRsqrtD / l : (l == 0.f ? 0.f : l);
            const uint4 v4 = lds128(area + r * 512 + lane * 16);
            v[u][0] = __uint_as_float(v4.x) * inv; v[u][1] = __uint_as_float(v4.y) * inv;
            v[u][2] = __uint_as_float(v4.z) * inv; v[u][3] = __uint_as_float(v4.w) * inv;
          }
#pragma unroll
          for (int u = 0; u < kTwo; ++u) fht128_warp(v[u], lane);
#pragma unroll
          for (int u = 0; u < kTwo; ++u) {
            const int r = ch + 4 * (u0 + u) + (warp & 3);
            int t;
            const int64_t at = place(pc, r, t);
            if (t < pc.q_len && alive) {
              *reinterpret_cast<uint2*>(p.out + at * kHeadDim + 4 * lane) = pack_half4(v[u]);
              if (p.lse_out && lane == 0) {
                const float l = cmb[2 * NR + r];
                p.lse_out[at] = l == 0.f ? -INFINITY : (log2f(l) + cmb[3 * NR + r]) * kLn2;
              }
            }
          }
        }
      }
      tc_fence_before_sync();
      named_barrier(5, 512);                                    // O and the P buffers may be overwritten
      tc_fence_after_sync();
      done = end;
      set ^= 1;
    }
  } else if (warp < C::kWarpS) {
    // ============ producers: slot -> fp16 row; K to tensor memory (lane = key), V to shared memory (row = key).  Two groups of
    // four warps for K, each with every second tile, and one for V; a thread expands one row.  The loops are kept short: unrolled
    // over the row, they evict one another (and the softmax) from the instruction caches and everything runs 1.5 times slower ==
    const bool is_v = warp >= C::kWarpV;
    lower_registers<C::kRegsOther>();
    const int step = is_v ? 1 : C::kKGroups, begin = is_v || C::kKGroups == 1 ? 0 : (warp >> 2) & 1;
    const int key = (warp & 3) * 32 + lane, bits = is_v ? p.v_bits : p.k_bits;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + C::kColK;
    const uint32_t cell0 = base + C::kOffRing + key * p.slot_bytes, code_at = is_v ? 16 * p.k_bits : 0;
    const uint32_t norm_at = 16 * (p.k_bits + p.v_bits), row0 = base + C::kOffV;
    const float* levels = reinterpret_cast<const float*>(sm + C::kOffLevels) + (is_v ? 16 : 0);
    const int id = is_v ? 6 : 7 + begin;                        // named barriers: V 6; K 7, 8
    int stage = begin, wraps = 0;                               // of the ring
#pragma unroll 1
    for (int i = begin; i < total; i += step) {
      const int buffer = i & 1, slot = (is_v ? kVFull : kKFull) + buffer;               // its "full" barrier
      const uint32_t row = row0 + buffer * kTileBytes;
      if ((warp & 3) == 0) {                                    // the slots are there, and the buffer they go to is free
        wait_for(bar(kRingFull + stage), wraps & 1, wait);
        if (i >= 2) wait_for(bar((is_v ? kPvDone : kKEmpty) + buffer), ((i - 2) >> 1) & 1, wait);
      }
      named_barrier(id, 128);
      tc_fence_after_sync();
      const uint32_t cell = cell0 + stage * kStageBytes;
      const uint2 norms = lds64(cell + norm_at);
      const bool live = key < *reinterpret_cast<volatile int*>(sm + C::kOffBar + kOffValid + 4 * stage);
      const float norm = live ? __uint_as_float(is_v ? norms.y : norms.x) : 0.f;        // keys past the end: zero rows
      expand::Planes t = expand::make_planes(levels, bits == 4 ? 4 : 1, norm);
      if (is_v && t.any_not_finite() && row_not_finite(cell + code_at, bits, base + C::kOffLevels + 64, norm)) t = expand::Planes{};
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {                                     // 32 coordinates at a time
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
            sts128(row + (c >> 1) * kColBlock + sw128(key, (c & 1) * 4 + u), v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        } else {
          tmem_st16(lanes + buffer * 64 + 16 * c, v);
        }
      }
      if (is_v) {
        fence_async_smem();
      } else {                                                          // (eight tiles deep: read before S of tile i + 4 is written)
        const bool bad = live && row_not_finite(cell + 16 * p.k_bits, p.v_bits, base + C::kOffLevels + 64, __uint_as_float(norms.y));
        const uint32_t bad_keys = __ballot_sync(0xffffffffu, bad);
        if (lane == 0) *reinterpret_cast<uint32_t*>(sm + C::kOffBad + 16 * (i & 7) + 4 * (warp & 3)) = bad_keys;
        tmem_wait_st();
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(kRingEmpty + stage));
        mbar_arrive(bar(slot));
      }
      stage += step;
      if (stage >= C::kRing) { stage -= C::kRing; ++wraps; }
    }
  } else {
    lower_registers<C::kRegsOther>();
    if (warp >= C::kWarpFeed) {
      feed_ring<C::kRing>(p, &map, [&](Feed& f) {
        Piece q;
        if (!w.next(p, q)) return false;
        f = Feed{q.x.b, q.head, q.x.seq_len, q.tile0, q.n};
        return true;
      }, warp - C::kWarpFeed, base + C::kOffRing, bar(kRingFull), bar(kRingEmpty),
          reinterpret_cast<volatile int*>(sm + C::kOffBar + kOffValid), reinterpret_cast<int32_t*>(sm + C::kOffBar + kOffIds), wait);
    } else if (warp == C::kWarpS || warp == C::kWarpO) {
      // ============ MMA issuers: one warp for S = K Q^T, one for O += V^T P, so that neither waits for the other's operands ======
      constexpr uint32_t idesc_s = instr_desc_f16(kKeys, NR, false, false), idesc_o = instr_desc_f16(kHeadDim, NR, true, true);
      const bool leader = elect_one();
      bool alive = true;
      int i = 0, pieces = 0;
      Piece pc;
      if (warp == C::kWarpS) {
        const uint64_t q_desc = smem_desc_sw128(base + C::kOffQ, 16, 1024);
        while (w.next(p, pc)) {
          alive = wait_for(bar(kQFull), pieces & 1, wait) && alive;
#pragma unroll 1
          for (int k = 0; k < pc.n; ++k, ++i) {
            alive = wait_for(bar(kKFull + (i & 1)), (i >> 1) & 1, wait) && alive;
            if (i >= C::kSBuffers) alive = wait_for(bar(kSEmpty + (i & (C::kSBuffers - 1))), ((i >> C::kSShift) - 1) & 1, wait) && alive;
            __syncwarp();
            tc_fence_after_sync();
            const uint32_t d = tmem + C::kColS + (i & (C::kSBuffers - 1)) * NR, a = tmem + C::kColK + (i & 1) * 64;
            if (leader && alive) {
              // the small terms of the query go first: the accumulator is cut off, not rounded, in each of the 16 steps, always
              // towards zero, and behind the large terms that costs eight more cuts of the whole score (log-sum-exp off by 1.25e-6
              // on average, this way by 0.6e-6)
#pragma unroll
              for (int term = 0; term < 2; ++term)
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                  const uint64_t q = q_desc + (((1 - term) * (NR * 256) + (ks >> 2) * (NR * 128) + (ks & 3) * 32) >> 4);
                  if (term == 0 && ks == 0) mma_ts<false>(d, a, q, idesc_s);
                  else mma_ts<true>(d, a + 8 * ks, q, idesc_s);
                }
              mma_commit(bar(kSFull + (i & (C::kSBuffers - 1))));
              mma_commit(bar(kKEmpty + (i & 1)));
            }
            __syncwarp();
          }
          ++pieces;
        }
      } else {
        const uint64_t v_desc = smem_desc_sw128(base + C::kOffV, kColBlock, 1024), p_desc = smem_desc_sw128(base + C::kOffP, kColBlock, 1024);
        while (w.next(p, pc)) {
#pragma unroll 1
          for (int k = 0; k < pc.n; ++k, ++i) {
            alive = wait_for(bar(kVFull + (i & 1)), (i >> 1) & 1, wait) && alive;
            alive = wait_for(bar(kPFull + (i & 1)), (i >> 1) & 1, wait) && alive;
            __syncwarp();
            tc_fence_after_sync();
            if (leader && alive) {
              const uint64_t v = v_desc + (i & 1) * (kTileBytes >> 4), pt = p_desc + (C::kStreams == 2 ? (i & 1) * (kColBlock >> 4) : 0);
#pragma unroll
              for (int ks = 0; ks < 8; ++ks) mma_ss(tmem + C::kColO + (C::kStreams == 2 ? (i & 1) * NR : 0), v + ks * 128, pt + ks * 128, idesc_o, k < C::kStreams && ks == 0 ? 0u : 1u);
              mma_commit(bar(kPvDone + (i & 1)));
            }
            __syncwarp();
          }
        }
      }
      // nothing in flight when tensor memory is released: a commit behind everything issued, waited for (with a limit) even
      // after a wait elsewhere gave up
      if (leader) mma_commit(bar(kDrained));
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(bar(kDrained), 0) && global_timer_ns() - t0 < kWaitLimitNs) { }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0) {
    if (wait->abort) { rec = Record{-1, 0, 3, 0}; atomicOr(&g_tree_status, kStatusWait); }
    space.rec[blockIdx.x] = rec;
  }
  if (warp == C::kWarpS) {
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
  asm volatile("griddepcontrol.wait;" ::: "memory");            // launched while the first kernel still runs
  const Record rec = space.rec[c];
  const int state1 = c + 1 + lane < ctas ? space.rec[c + 1 + lane].head_state : 3;
  if (rec.tail_e < 0) return;
  const Entry x = entry_of<NR>(p, rec.tail_e);
  const int row = x.rb * NR + r, t = row / p.group;
  if (t >= x.q_len) return;
  int pieces = 0;                                               // CTA c's own, then those of the CTAs up to the one where it ends
  for (int k0 = c + 1; k0 < ctas; k0 += 32) {
    const int state = k0 == c + 1 ? state1 : k0 + lane < ctas ? space.rec[k0 + lane].head_state : 3;
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
#pragma unroll 8
  for (int k = 0; k < pieces; ++k) {
    const int64_t at = piece_row(k);
    const float2 ml = space.ml[at];
    const float4 v = reinterpret_cast<const float4*>(space.o + at * kHeadDim)[lane];
    const bool seen = ml.x != -INFINITY;                        // else the row saw no key in this piece (its sum is 0, or NaN)
    const float f = seen ? exp2f(ml.x - top) : 1.0f;
    l = fmaf(f, ml.y, l);
    o[0] = seen ? fmaf(f, v.x, o[0]) : o[0]; o[1] = seen ? fmaf(f, v.y, o[1]) : o[1];
    o[2] = seen ? fmaf(f, v.z, o[2]) : o[2]; o[3] = seen ? fmaf(f, v.w, o[3]) : o[3];
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

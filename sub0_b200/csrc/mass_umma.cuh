// The weight that the rows of a query chunk give to every cached key, on the tcgen05 tensor cores (same frame as
// tree_umma.cuh: keys on the M axis, K tiles through tensor memory).
//
//   S^T (128 keys x NR) = K . Q^T            w_n = sum_r weight_r exp2(S_nr - lse_r)            mass_n += w_n
//
// With lse given there is no maximum to find and nothing to rescale, and a lane of S^T is a key: its thread adds the row's terms
// in a fixed order, in registers, and owns the key's word of `mass` -- no atomics, no reduction across lanes.
//
// Warps: two weighing groups and four K producer groups of four warps (tiles in turn), one MMA issuer, two feeders.  Expanding
// codes is what takes longest here (about 23 byte-permute and logic instructions for eight coordinates), hence four groups.
// A CTA walks an equal share of all (sequence, KV head) segments' tiles; chunks of more than NR rows pass over the share's
// tiles once per block of NR rows.
//
// Measured (4-bit slots, 8 KV heads, 4 query heads each): one token of 32 sequences of 16k keys 167 us -- the slots' K half
// and norms are 49 us at copy bandwidth, whole slots 92 us; the integer pipe is busy 76% of the time and DRAM at 3.8 TB/s --
// the last 64 tokens of two 30k prompts 90 us (128-row blocks, where it is the exponentials and their sums).
#pragma once
#include "tree_umma.cuh"

namespace cda {
namespace msu {

using namespace tru;

constexpr int kMassPieceCost = 3;                // what a new piece costs, in tiles

template <int NR>
struct MassCfg {
  static constexpr int kGroups = 2, kKGroups = 4;
  static constexpr int kWarpK = 4 * kGroups, kWarpS = kWarpK + 4 * kKGroups, kWarpFeed = kWarpS + 1, kThreads = (kWarpFeed + kFeeders) * 32;
  static constexpr int kSBuffers = NR == 128 ? 2 : 4;
  // a multiple of the K groups: every stage is read by one group, which sees all phases of its barrier (a group that skipped one
  // would take the phase before it for the one it waits for)
  static constexpr int kRing = 8;
  static_assert(kRing % kKGroups == 0, "one reader for each stage");
  static constexpr int kColK = 0, kColS = 64 * kKGroups, kTmemCols = 512;
  static constexpr int kChunk = 16;
  static constexpr int kOffQ = 0, kOffRing = NR * 512;
  static constexpr int kOffLse = kOffRing + kRing * kStageBytes;  // words of the rows: lse x log2 e,
  static constexpr int kOffWeight = kOffLse + 4 * NR;             //   weight,
  static constexpr int kOffPos = kOffWeight + 4 * NR;             //   position,
  static constexpr int kOffSlope = kOffPos + 4 * NR;              //   slope x log2 e,
  static constexpr int kOffMask = kOffSlope + 4 * NR;             //   64-bit ancestor mask
  static constexpr int kOffLevels = kOffMask + 8 * NR;
  static constexpr int kOffScan = kOffLevels + 64;
  static constexpr int kOffBar = kOffScan + 512;
  static constexpr int kSmemBytes = kOffBar + 384 + kFeeders * kFeedIdBytes + 1024;
  static_assert(kColS + kSBuffers * NR <= kTmemCols && kSmemBytes <= 232448, "one CTA");
};
constexpr int kMKFull = 0, kMKEmpty = 4, kMSFull = 8, kMSEmpty = 12, kMQFull = 16, kMDrained = 17, kMRingFull = 18, kMRingEmpty = 26;   // 34
constexpr int kMOffTmem = 272, kMOffWait = 280, kMOffPlan = 296, kMOffEnd = 312, kMOffValid = 320, kMOffIds = 384;

// Sequence b: the key tiles that any of its rows may see, and its row blocks.
struct Seq { SequenceView v; int ctx, first, tiles, blocks; };
template <int NR>
__device__ __forceinline__ Seq seq_of(const AttendParams& p, int b) {
  Seq s;
  s.v = sequence_view(p, b);
  s.ctx = s.v.seq_len - s.v.q_len;
  s.blocks = (s.v.q_len * p.group + NR - 1) / NR;
  const int lo = p.window > 0 ? max(0, s.ctx - p.window + 1) : 0;
  s.first = lo / kKeys;
  s.tiles = s.v.q_len > 0 ? (s.v.seq_len + kKeys - 1) / kKeys - s.first : 0;
  return s;
}
// One block of rows over a piece of a segment: tiles tile0 .. tile0 + n - 1 (n > 0).
struct Sub { Seq s; int b, head, rb, t0, tile0, n; };
template <int NR>
struct MassWalk {
  int b, h, j, left, B;       // segment, tile inside it, tiles of this CTA that are left
  int piece0, piece_n, rb;    // piece in work
  Seq s;
  __device__ __forceinline__ bool next(const AttendParams& p, Sub& q) {
    for (;;) {
      if (rb < s.blocks && piece_n > 0) {
        const int t0 = rb * NR / p.group, t1 = min(s.v.q_len, (rb * NR + NR + p.group - 1) / p.group) - 1;
        const int hi = p.tree_mask ? s.v.seq_len : s.ctx + t1 + 1;
        const int lo = p.window > 0 ? max(0, s.ctx + (p.tree_mask ? 0 : t0) - p.window + 1) : 0;
        const int from = max(piece0, lo / kKeys), to = min(piece0 + piece_n, (hi + kKeys - 1) / kKeys);
        q.s = s; q.b = b; q.head = h; q.rb = rb; q.t0 = t0; q.tile0 = from; q.n = to - from;
        ++rb;
        if (q.n > 0) return true;
        continue;
      }
      if (piece_n > 0) {                                        // the piece is done
        j += piece_n;
        piece_n = 0;
        if (j == s.tiles) { j = 0; if ((h += p.side) >= p.H_kv) { h %= p.side; ++b; } }
      }
      if (left <= 0 || b >= B) return false;
      s = seq_of<NR>(p, b);
      if (s.tiles == 0) { ++b; continue; }
      piece0 = s.first + j;
      piece_n = min(left, s.tiles - j);
      left -= piece_n;
      rb = 0;
    }
  }
};

// Share of this CTA on the line of all segments, a tile of a sequence of several row blocks being as long as their number.  `side`
// neighbouring CTAs (the largest divisor of H_kv up to 8) walk the same share, each for its own KV head: the heads of a token lie
// side by side, in pieces that are no whole memory lines, so they have to be read at about the same time.  (With the heads one
// after the other on the line, 32 x 16k keys of 8 heads read 1.33 GB from memory, at 5.9 TB/s, where the slots hold 0.60 GB.)
template <int NR, int THREADS>
__device__ __forceinline__ void find_mass_share(const AttendParams& p, longlong2* s_scan, int* s_plan, int* s_end) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (p.B + THREADS - 1) / THREADS, b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  long long tiles = 0, len = 0;
  for (int b = b0; b < b1; ++b) {
    const Seq s = seq_of<NR>(p, b);
    tiles += s.tiles;
    len += s.tiles > 0 ? static_cast<long long>(s.tiles) * s.blocks + kMassPieceCost : 0;
    if (blockIdx.x == 0 && s.v.bad) atomicOr(&g_tree_status, kStatusLengths);
  }
  long long x = tiles, y = len;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) { x += u; y += v; }
  }
  if (lane == 31) s_scan[warp] = make_longlong2(x, y);
  __syncthreads();
  long long tiles_before = x - tiles, at = y - len, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) { tiles_before += s_scan[w].x; at += s_scan[w].y; }
    all += s_scan[w].y;
  }
  const int turns = p.H_kv / p.side;                            // heads that a CTA's segments of a sequence are of
  const unsigned teams = gridDim.x / p.side, team = blockIdx.x / p.side;
  at *= turns;
  const long long line = all * turns, busy = line < teams ? line : teams, cta = team < busy ? team : busy;
  const long long lo = busy ? line * cta / busy : 0, hi = cta < busy ? line * (cta + 1) / busy : lo;
  if (tid == 0) s_plan[3] = *s_end = 0;
  __syncthreads();
  long long real = tiles_before * turns;
  for (int b = b0; hi > lo && b < b1 && at < hi; ++b) {
    const Seq s = seq_of<NR>(p, b);
    if (s.tiles == 0) continue;
    const long long one = static_cast<long long>(s.tiles) * s.blocks + kMassPieceCost, next = at + one * turns;
    const auto tile_of = [&](long long off) { return static_cast<int>(off > kMassPieceCost ? (off - kMassPieceCost) / s.blocks : 0); };
    if (at <= lo && lo < next) {
      s_plan[0] = b; s_plan[1] = static_cast<int>((lo - at) / one); s_plan[2] = tile_of((lo - at) % one);
      s_plan[3] = static_cast<int>(real + static_cast<long long>(s_plan[1]) * s.tiles + s_plan[2]);
    }
    if (at < hi && hi <= next) *s_end = static_cast<int>(real + (hi - at) / one * s.tiles + tile_of((hi - at) % one));
    at = next;
    real += static_cast<long long>(s.tiles) * turns;
  }
  __syncthreads();
  if (tid == 0) s_plan[3] = *s_end - s_plan[3];
  __syncthreads();
}

template <int NR>
__global__ void __launch_bounds__(MassCfg<NR>::kThreads, 1) attention_mass_kernel(const AttendParams p, const __grid_constant__ CUtensorMap map) {
  using C = MassCfg<NR>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* sm = smem_raw + (base - raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* s_plan = reinterpret_cast<int*>(sm + C::kOffBar + kMOffPlan);
  volatile WaitState* wait = reinterpret_cast<volatile WaitState*>(sm + C::kOffBar + kMOffWait);
  const uint32_t bar0 = base + C::kOffBar;
  auto bar = [&](int i) { return bar0 + 8u * i; };

  if (tid == 0) {
    for (int i = 0; i < C::kKGroups; ++i) { mbar_init(bar(kMKFull + i), 4 + withheld(p, i)); mbar_init(bar(kMKEmpty + i), 1); }
    for (int i = 0; i < C::kSBuffers; ++i) { mbar_init(bar(kMSFull + i), 1); mbar_init(bar(kMSEmpty + i), 4); }
    mbar_init(bar(kMQFull), 4 * C::kGroups);
    mbar_init(bar(kMDrained), 1);
    for (int i = 0; i < C::kRing; ++i) { mbar_init(bar(kMRingFull + i), 1); mbar_init(bar(kMRingEmpty + i), 4); }
    wait->abort = 0;
    wait->limit_ns = p.wait_limit_ns;
    mbar_init_fence();
  }
  if (tid < 16) reinterpret_cast<float*>(sm + C::kOffLevels)[tid] = tid < (p.k_bits == 4 ? 16 : 4) ? __ldg(p.cb_k + tid) : 0.f;
  if (warp == C::kWarpS) {
    tmem_alloc(base + C::kOffBar + kMOffTmem, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  find_mass_share<NR, C::kThreads>(p, reinterpret_cast<longlong2*>(sm + C::kOffScan), s_plan, reinterpret_cast<int*>(sm + C::kOffBar + kMOffEnd));
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + C::kOffBar + kMOffTmem);
  if (s_plan[3] == 0) {
    if (warp == C::kWarpS) tmem_dealloc(tmem, C::kTmemCols);
    return;
  }
  MassWalk<NR> w;
  w.b = s_plan[0]; w.h = s_plan[1] * p.side + blockIdx.x % p.side; w.j = s_plan[2]; w.left = s_plan[3]; w.B = p.B; w.piece_n = 0; w.rb = 0; w.s.blocks = 0;
  Sub q;

  if (warp < C::kWarpK) {
    // ============ weighing: a thread is a key; the groups take tiles in turn ==================================================
    const int group = warp >> 2, key = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + C::kColS;
    const float kf = p.scale * kLog2e, cap2 = p.softcap * kLog2e, inv_cap = p.softcap > 0.f ? p.scale / p.softcap : 0.f;
    const float* lse_w = reinterpret_cast<const float*>(sm + C::kOffLse);
    const int* pos_w = reinterpret_cast<const int*>(sm + C::kOffPos);
    const float* slope_w = reinterpret_cast<const float*>(sm + C::kOffSlope);
    const float* weight_w = reinterpret_cast<const float*>(sm + C::kOffWeight);
    const uint32_t* mask_w = reinterpret_cast<const uint32_t*>(sm + C::kOffMask);
    int done = 0;
    while (w.next(p, q)) {
      named_barrier(5, 256);                                    // all S of the rows before are done: Q and the row words are free
      const int rows = min(NR, q.s.v.q_len * p.group - q.rb * NR);
      if (tid < NR) {
        const int row = q.rb * NR + tid, t = row / p.group;
        const bool real = tid < rows;
        const int64_t at = static_cast<int64_t>(q.s.v.q_begin + t) * p.H_q + q.head * p.group + row % p.group;
        const float z = real ? p.lse[at] : 0.f, wt = real ? (p.weights ? p.weights[q.s.v.q_begin + t] : 1.0f) : 0.f;
        const unsigned long long m = real && p.tree_mask ? static_cast<unsigned long long>(p.tree_mask[q.s.v.q_begin + t]) : 0ull;
        // a row that counts nothing or saw nothing: exp2(x - inf) = 0
        reinterpret_cast<float*>(sm + C::kOffLse)[tid] = wt == 0.f || z == -INFINITY ? INFINITY : z * kLog2e;
        reinterpret_cast<float*>(sm + C::kOffWeight)[tid] = wt;
        reinterpret_cast<unsigned long long*>(sm + C::kOffMask)[tid] = m;
        reinterpret_cast<int*>(sm + C::kOffPos)[tid] = q.s.ctx + (!real ? 0 : p.tree_mask ? max(__popcll(m) - 1, 0) : t);
        reinterpret_cast<float*>(sm + C::kOffSlope)[tid] = p.slopes && real ? p.slopes[q.head * p.group + row % p.group] * kLog2e : 0.f;
      }
#pragma unroll 1
      for (int r0 = warp; r0 < NR; r0 += 16) {                  // two rows at a time
        float f[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int r = r0 + 8 * u, row = q.rb * NR + r, t = row / p.group;
          f[u][0] = f[u][1] = f[u][2] = f[u][3] = 0.f;
          if (r < rows) load_half4(p.q + (static_cast<int64_t>(q.s.v.q_begin + t) * p.H_q + q.head * p.group + row % p.group) * kHeadDim + 4 * lane, f[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) fht128_warp(f[u], lane);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float lo[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            f[u][c] *= kRsqrtD;
            lo[c] = f[u][c] - round_to_half(f[u][c]);
          }
          const uint2 h = pack_half4(f[u]), l = pack_half4(lo);
          const uint32_t at = base + C::kOffQ + (lane >> 4) * (NR * 128) + sw128(r0 + 8 * u, (lane & 15) >> 1) + 8 * (lane & 1);
          sts64(at, h.x, h.y);
          sts64(at + NR * 256, l.x, l.y);
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kMQFull));
      named_barrier(5, 256);
      const int ctx = q.s.ctx, seq_len = q.s.v.seq_len, end = done + q.n, tile_at = q.tile0 - done;
      const int see_hi = p.slopes ? done : (ctx + (p.tree_mask ? 0 : q.t0 + 1)) / kKeys - tile_at;
      const int see_lo = p.window > 0 ? max(0, ctx + positions_of(p, q.s.v.q_len) - p.window + kKeys) / kKeys - tile_at : done;
      const int cols = (rows + C::kChunk - 1) / C::kChunk * C::kChunk;
      float* mass = p.mass + (static_cast<int64_t>(q.b) * p.H_kv + q.head) * p.mass_stride;
#pragma unroll 1
      for (int i = done + ((done ^ group) & 1); i < end; i += 2) {
        const int n = (i + tile_at) * kKeys + key, j = n - ctx, buffer = i & (C::kSBuffers - 1);
        const bool rule = i >= see_hi || i < see_lo, finish = rule || p.softcap > 0.f;
        const float old = n < seq_len ? mass[n] : 0.f;
        if ((warp & 3) == 0) wait_for(bar(kMSFull + buffer), (i / C::kSBuffers) & 1, wait);
        group_barrier(group);
        tc_fence_after_sync();
        uint64_t sum = f2_pack(0.f, 0.f);
        const int pos_k = rule && p.tree_mask && j >= 0 && n < seq_len ? ctx + depth_of(p, q.s.v.q_begin, j) : n;
        const int word = (j >> 5) & 1, up = 31 - (j & 31);      // bit j of a row's mask to the sign
        const uint32_t all = j < 0 ? 0x80000000u : 0u, none = n < seq_len ? 0xffffffffu : 0u;
        const float f1 = finish ? (p.softcap > 0.f ? inv_cap : kf) : 1.0f, f2 = finish ? 1.0f : kf;
#pragma unroll 1
        for (int c0 = 0; c0 < cols; c0 += C::kChunk) {
          uint32_t x[C::kChunk];
          tmem_load<C::kChunk>(lanes + buffer * NR + c0, x);
          tmem_wait_ld();
          if (finish) {                                         // cap, bias and masks, in the base-2 domain
#pragma unroll
            for (int c = 0; c < C::kChunk; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * f1);
            if (p.softcap > 0.f) {
#pragma unroll
              for (int c = 0; c < C::kChunk; ++c) x[c] = __float_as_uint(cap2 * soft_tanh(__uint_as_float(x[c])));
            }
            if (rule) {
              if (p.slopes) {
#pragma unroll
                for (int c = 0; c < C::kChunk; ++c) x[c] = __float_as_uint(fmaf(slope_w[c0 + c], static_cast<float>(pos_k - pos_w[c0 + c]), __uint_as_float(x[c])));
              }
              if (p.window > 0) {
#pragma unroll
                for (int c = 0; c < C::kChunk; ++c) x[c] = pos_w[c0 + c] - pos_k >= p.window ? 0xff800000u : x[c];
              }
              if (p.tree_mask) {
#pragma unroll
                for (int c = 0; c < C::kChunk; ++c) x[c] = static_cast<int>(((mask_w[2 * (c0 + c) + word] << up) | all) & none) < 0 ? x[c] : 0xff800000u;
              } else {
#pragma unroll
                for (int c = 0; c < C::kChunk; ++c) x[c] = n > pos_w[c0 + c] || n >= seq_len ? 0xff800000u : x[c];
              }
            }
          }
          const uint64_t ff = f2_pack(f2, f2);
#pragma unroll
          for (int c = 0; c < C::kChunk; c += 2) {
            const float2 z = *reinterpret_cast<const float2*>(lse_w + c0 + c), wt = *reinterpret_cast<const float2*>(weight_w + c0 + c);
            float a0, a1;
            f2_unpack(f2_fma(f2_pack(x[c], x[c + 1]), ff, f2_pack(-z.x, -z.y)), a0, a1);
            sum = f2_fma(f2_pack(fast_exp2(a0), fast_exp2(a1)), f2_pack(wt.x, wt.y), sum);
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kMSEmpty + buffer));
        float s0, s1;
        f2_unpack(sum, s0, s1);
        if (n < seq_len && wait->abort == 0) mass[n] = old + (s0 + s1);
      }
      done = end;
    }
  } else if (warp < C::kWarpS) {
    // ============ K producers: slot -> exact fp16 row -> tensor memory, lane = key; four groups, tiles in turn ==================
    const int begin = (warp - C::kWarpK) >> 2, key = (warp & 3) * 32 + lane;
    const uint32_t to = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + C::kColK + begin * 64;
    const uint32_t cell0 = base + C::kOffRing + key * p.slot_bytes, norm_at = 16 * (p.k_bits + p.v_bits);
    const float* levels = reinterpret_cast<const float*>(sm + C::kOffLevels);
    int done = 0, mine = 0;                                     // tiles so far, and of this group
    while (w.next(p, q)) {
#pragma unroll 1
      for (int i = done + ((begin - done) & 3); i < done + q.n; i += 4, ++mine) {
        const int stage = i % C::kRing;
        if ((warp & 3) == 0) {
          wait_for(bar(kMRingFull + stage), (i / C::kRing) & 1, wait);
          if (mine > 0) wait_for(bar(kMKEmpty + begin), (mine - 1) & 1, wait);
        }
        named_barrier(6 + begin, 128);
        tc_fence_after_sync();
        const uint32_t cell = cell0 + stage * kStageBytes;
        const bool live = key < *reinterpret_cast<volatile int*>(sm + C::kOffBar + kMOffValid + 4 * stage);
        const expand::Planes t = expand::make_planes(levels, p.k_bits == 4 ? 4 : 1, live ? lds_f(cell + norm_at) : 0.f);   // keys past the end: zero rows
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {                           // 32 coordinates at a time
          uint32_t v[16];
          if (p.k_bits == 4) {
            expand::quarter4(t, lds128(cell + 16 * c), v);
          } else {
            const uint2 x = lds64(cell + 8 * c);
            expand::quarter2(t, x.x, x.y, v);
          }
          tmem_st16(to + 16 * c, v);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(kMRingEmpty + stage));
          mbar_arrive(bar(kMKFull + begin));
        }
      }
      done += q.n;
    }
  } else if (warp == C::kWarpS) {
    // ============ MMA issuer ====================================================================================================
    constexpr uint32_t idesc = instr_desc_f16(kKeys, NR, false, false);
    const uint64_t q_desc = smem_desc_sw128(base + C::kOffQ, 16, 1024);
    const bool leader = elect_one();
    bool alive = true;
    int i = 0, subs = 0;
    while (w.next(p, q)) {
      alive = wait_for(bar(kMQFull), subs & 1, wait) && alive;
#pragma unroll 1
      for (int k = 0; k < q.n; ++k, ++i) {
        const int buffer = i & (C::kSBuffers - 1);
        alive = wait_for(bar(kMKFull + (i & 3)), (i >> 2) & 1, wait) && alive;
        if (i >= C::kSBuffers) alive = wait_for(bar(kMSEmpty + buffer), (i / C::kSBuffers - 1) & 1, wait) && alive;
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t d = tmem + C::kColS + buffer * NR, a = tmem + C::kColK + (i & 3) * 64;
        if (leader && alive) {                                  // (the small terms first, see tree_umma.cuh)
#pragma unroll
          for (int term = 0; term < 2; ++term)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
              const uint64_t qd = q_desc + (((1 - term) * (NR * 256) + (ks >> 2) * (NR * 128) + (ks & 3) * 32) >> 4);
              if (term == 0 && ks == 0) mma_ts<false>(d, a, qd, idesc);
              else mma_ts<true>(d, a + 8 * ks, qd, idesc);
            }
          mma_commit(bar(kMSFull + buffer));
          mma_commit(bar(kMKEmpty + (i & 3)));
        }
        __syncwarp();
      }
      ++subs;
    }
    if (leader) mma_commit(bar(kMDrained));                     // nothing in flight when tensor memory is released
    const unsigned long long t0 = global_timer_ns();
    while (!mbar_try_wait(bar(kMDrained), 0) && global_timer_ns() - t0 < kWaitLimitNs) { }
  } else {
    feed_ring<C::kRing>(p, &map, [&](Feed& f) {
      if (!w.next(p, q)) return false;
      f = Feed{q.b, q.head, q.s.v.seq_len, q.tile0, q.n};
      return true;
    }, warp - C::kWarpFeed, base + C::kOffRing, bar(kMRingFull), bar(kMRingEmpty),
        reinterpret_cast<volatile int*>(sm + C::kOffBar + kMOffValid), reinterpret_cast<int32_t*>(sm + C::kOffBar + kMOffIds), wait);
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && wait->abort) atomicOr(&g_tree_status, kStatusWait);
  if (warp == C::kWarpS) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

}  // namespace msu
}  // namespace cda

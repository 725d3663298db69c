// Codes -> the exact fp16 values of a key, from tables held in registers.
//
// A slot stands for rows fp16(level * norm) (fp32 product, one rounding; compression.py:337-361).  A key has only 16 (or 4) such
// values per side.  They are computed once per key and kept as byte planes: the low bytes of four levels in one register,
// their high bytes in another.  A code then selects its value with byte permutes, four codes per instruction.
#pragma once
#include "common.cuh"

namespace cda {
namespace expand {

__device__ __forceinline__ uint32_t permute(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}

// lo[k], hi[k]: the bytes of levels 4k .. 4k + 3 times the key's norm; a 2-bit side uses k = 0 only.
struct Planes {
  uint32_t lo[4], hi[4];
  // whether any value is infinite or NaN: the five bits of its exponent are ones
  __device__ __forceinline__ bool any_not_finite() const {
    uint32_t any = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) any |= (hi[k] & 0x7C7C7C7Cu) + 0x04040404u;
    return (any & 0x80808080u) != 0;
  }
};

__device__ __forceinline__ Planes make_planes(const float* levels, int groups, float norm) {
  Planes t;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= groups) { t.lo[k] = t.hi[k] = 0u; continue; }
    const float4 c = *reinterpret_cast<const float4*>(levels + 4 * k);
    const uint32_t h0 = pack_half2(c.x * norm, c.y * norm), h1 = pack_half2(c.z * norm, c.w * norm);
    t.lo[k] = permute(h0, h1, 0x6420u);
    t.hi[k] = permute(h0, h1, 0x7531u);
  }
  return t;
}

// One word of 4-bit codes -> 8 coordinates as four fp16 pairs.  A code byte holds coordinate 2j in its high nibble
// (compression.py:163-188).  The low three bits of a code pick one of eight bytes, its top bit the register pair.
__device__ __forceinline__ void word4(const Planes& t, uint32_t x, uint32_t* v) {
  const uint32_t m = x & 0x77777777u, y = x & 0x88888888u, a = y << 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t sel = h ? m >> 16 : m;
    const uint32_t upper = permute(a, y, h ? 0xFBEAu : 0xD9C8u);      // 0xFF in the bytes whose code is 8 .. 15
    const uint32_t la = permute(t.lo[0], t.lo[1], sel), lb = permute(t.lo[2], t.lo[3], sel);
    const uint32_t ha = permute(t.hi[0], t.hi[1], sel), hb = permute(t.hi[2], t.hi[3], sel);
    const uint32_t lo = (lb & upper) | (la & ~upper), hi = (hb & upper) | (ha & ~upper);
    v[2 * h] = permute(lo, hi, 0x4051u);
    v[2 * h + 1] = permute(lo, hi, 0x6273u);
  }
}

// Half a word (16 bits) of 2-bit codes -> 8 coordinates.  A code byte holds coordinates 4j .. 4j + 3 from its top bit pair
// down (compression.py:375-386); the codes are spread to nibbles, which select four value bytes at a time.
__device__ __forceinline__ void half_word2(const Planes& t, uint32_t s, uint32_t* v) {
  s = (s | (s << 8)) & 0x00FF00FFu;
  s = (s | (s << 4)) & 0x0F0F0F0Fu;
  s = (s | (s << 2)) & 0x33333333u;
  const uint32_t l0 = permute(t.lo[0], t.lo[0], s), h0 = permute(t.hi[0], t.hi[0], s);
  const uint32_t l1 = permute(t.lo[0], t.lo[0], s >> 16), h1 = permute(t.hi[0], t.hi[0], s >> 16);
  v[0] = permute(l0, h0, 0x6273u);
  v[1] = permute(l0, h0, 0x4051u);
  v[2] = permute(l1, h1, 0x6273u);
  v[3] = permute(l1, h1, 0x4051u);
}

// Coordinates 32 q .. 32 q + 31 of a key: from code words 4 q .. 4 q + 3 of a 4-bit side, 2 q and 2 q + 1 of a 2-bit side.
__device__ __forceinline__ void quarter4(const Planes& t, const uint4& w, uint32_t (&v)[16]) {
  word4(t, w.x, v);
  word4(t, w.y, v + 4);
  word4(t, w.z, v + 8);
  word4(t, w.w, v + 12);
}
__device__ __forceinline__ void quarter2(const Planes& t, uint32_t w0, uint32_t w1, uint32_t (&v)[16]) {
  half_word2(t, w0 & 0xFFFFu, v);
  half_word2(t, w0 >> 16, v + 4);
  half_word2(t, w1 & 0xFFFFu, v + 8);
  half_word2(t, w1 >> 16, v + 12);
}

}  // namespace expand
}  // namespace cda

// Philox4x32-10, the counter-based generator of J. Salmon, M. Moraes, R. Dror and D. Shaw, "Parallel random numbers: as
// easy as 1, 2, 3" (SC 2011), and the dropout mask made from it.
#pragma once
#include "common.h"

// Mask of a tensor read row by row: element i belongs to block b = i >> 3 and takes 16 bits of the block's 128,
// philox(counter = (b, offset), key = seed): word (i & 7) >> 1, the lower half where i is even.  Kept where the 16 bits
// are >= thr.  The mask is a function of (seed, offset, i) alone: not of the launch, the type, the strides or the vector
// width, so any kernel regenerates it and nothing is stored.  16 bits per element make one generator call serve eight
// elements (a 16-byte vector of bf16); the probability is rounded to a multiple of 2^-16 and the scale follows the rounded
// value, so the expectation is kept exactly.
struct DropKey {
  uint32_t k0, k1, o0, o1;   // seed, offset
  uint32_t thr;              // 0 = keep all, 65536 = drop all
  float scale;               // 65536 / (65536 - thr), 0 where all is dropped
};

static inline DropKey drop_key(double p, uint64_t seed, uint64_t offset) {
  DropKey d;
  d.k0 = (uint32_t)seed;
  d.k1 = (uint32_t)(seed >> 32);
  d.o0 = (uint32_t)offset;
  d.o1 = (uint32_t)(offset >> 32);
  d.thr = (uint32_t)(p * 65536.0 + 0.5);
  d.scale = d.thr < 65536u ? (float)(65536.0 / (65536.0 - d.thr)) : 0.f;
  return d;
}

__device__ __forceinline__ uint4 philox_block(uint64_t block, const DropKey& d) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = d.o0, c3 = d.o1, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// the eight elements of one block; dropped ones become 0 whatever they hold (a product would keep NaN and infinities)
__device__ __forceinline__ void drop_block(float (&v)[8], const uint4& w, const DropKey& d) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = (u[e] & 0xFFFFu) >= d.thr ? v[2 * e] * d.scale : 0.f;
    v[2 * e + 1] = (u[e] >> 16) >= d.thr ? v[2 * e + 1] * d.scale : 0.f;
  }
}

// For lanes that own single ELEMENTS (rows that cannot be read in vectors): the G lanes of a group cover 8 G consecutive
// elements first + j * G + l, j = 0..7.  Lane l makes block (first >> 3) + l, lane 0 also the block behind where `first` is
// not at a block border, the words go through `slot` (G + 1 blocks of LDS that only these lanes of one wave use), and
// lane l takes the 16 bits of its eight elements from there: one or two generator calls per lane instead of eight.
typedef uint16_t __attribute__((may_alias)) u16_alias;
template <int G>
__device__ __forceinline__ void drop_elements(float (&v)[8], uint64_t first, const DropKey& d, uint4* slot, int l) {
  const uint64_t block0 = first >> 3;
  const int mis = (int)(first & 7);
  __builtin_amdgcn_wave_barrier();
  slot[l] = philox_block(block0 + l, d);
  if (mis && l == 0) slot[G] = philox_block(block0 + G, d);
  // LDS serves the accesses of one wave in order, so the compiler's order is all that has to be held
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const u16_alias* h = reinterpret_cast<const u16_alias*>(slot) + mis + l;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = h[j * G] >= d.thr ? v[j] * d.scale : 0.f;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// For lanes that own eight consecutive elements first + 8 l .. + 7 where `first` need not be at a block border, so that
// they lie in two blocks: G lanes, each makes one block (lane 0 also the one behind the last), the words change lanes
// through `slot` (G + 1 blocks of LDS that only these lanes of one wave use).
typedef uint32_t __attribute__((may_alias)) u32_alias;
template <int G>
__device__ __forceinline__ void drop_straddling(float (&v)[8], uint64_t first, const DropKey& d, uint4* slot, int l) {
  const uint64_t block0 = first >> 3;
  const int mis = (int)(first & 7);
  uint4 w = philox_block(block0 + l, d);
  if (__ballot(mis != 0)) {   // (of any row of the wave)
    __builtin_amdgcn_wave_barrier();
    slot[l] = w;
    if (l == 0) slot[G] = philox_block(block0 + G, d);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const u32_alias* p = reinterpret_cast<const u32_alias*>(slot) + l * 4 + (mis >> 1);
    const int odd = (mis & 1) * 16;
    const uint32_t u[5] = {p[0], p[1], p[2], p[3], p[4]};
    w.x = (uint32_t)((((uint64_t)u[1] << 32) | u[0]) >> odd);
    w.y = (uint32_t)((((uint64_t)u[2] << 32) | u[1]) >> odd);
    w.z = (uint32_t)((((uint64_t)u[3] << 32) | u[2]) >> odd);
    w.w = (uint32_t)((((uint64_t)u[4] << 32) | u[3]) >> odd);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  drop_block(v, w, d);
}

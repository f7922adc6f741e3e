// Philox-4x32 with ten rounds, the counter-based generator of Salmon, Moraes,
// Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3" (SC 2011):
// each round multiplies two words of the 128-bit counter by fixed constants
// and mixes the halves of the products with the other two words and a key
// that grows by a fixed (Weyl) step. Nothing is stored: the same {counter,
// key} gives the same 128 bits in the forward and in the backward pass.
//
// Dropout takes 16 bits per element: element i of the array (C order) uses
// the counter {i / 8, offset} with the key `seed`, and of its four words the
// 16-bit half number i % 8, low halves first. 16 bits put a drop probability
// within 2^-17 of the one asked for (what is kept is scaled by the
// probability in use, so means stay right) and serve the eight elements of a
// 16-byte word of a 16-bit type with one evaluation; with 32 bits per element
// the integer multiplies, not the memory, would bound the kernels.
#pragma once
#include "common.cuh"

namespace mpb {

struct Dropper {
  uint32_t k0, k1, c2, c3;  // key (seed) and upper counter words (offset)
  uint32_t drop;            // dropped when the 16 bits, as the upper half of a word, are below this
  float up;                 // factor of what is kept
  int all;                  // everything is dropped
};

// floor(p * 65536 + 1/2); what is kept is multiplied by 65536 / (65536 - drop).
inline Dropper make_dropper(double p, uint64_t seed, uint64_t offset) {
  Dropper d;
  d.k0 = (uint32_t)seed;
  d.k1 = (uint32_t)(seed >> 32);
  d.c2 = (uint32_t)offset;
  d.c3 = (uint32_t)(offset >> 32);
  const uint32_t k = (uint32_t)(p * 65536.0 + 0.5);
  d.all = k >= 65536u;
  d.drop = d.all ? 0xffffffffu : k << 16;
  d.up = d.all ? 0.0f : (float)(65536.0 / (65536.0 - (double)k));
  return d;
}

// The four words of counter {block, offset}.
MPB_D uint4 philox(const Dropper& d, uint64_t block) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = d.c2, c3 = d.c3, k0 = d.k0, k1 = d.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// Whether element j (0..7) of a counter's words stays: its half against the
// threshold. The upper half of a word needs no shift, as the lower bits do not
// change whether the word reaches drop << 16.
MPB_D bool stays(const Dropper& d, const uint4& w, int j) {
  const uint32_t v = j < 4 ? (j < 2 ? w.x : w.y) : (j < 6 ? w.z : w.w);
  return ((j & 1) ? v : v << 16) >= d.drop;
}

// The words to compare: none reaches the threshold where everything is dropped.
MPB_D uint4 drop_words(const Dropper& d, uint64_t block) {
  const uint4 w = philox(d, block);
  return d.all ? make_uint4(0, 0, 0, 0) : w;
}

// Element i alone.
MPB_D bool keeps(const Dropper& d, uint64_t i) { return stays(d, drop_words(d, i >> 3), (int)(i & 7)); }

}  // namespace mpb

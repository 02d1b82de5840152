// Dropout from a counter: an element's random bits come from its place, a seed and
// an offset, so a mask is never stored and the gradient makes it again.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011) of the counter (chunk, offset), both 64 bits, and the seed as its key gives
// eight successive elements of a row sixteen bits each: the sixteen-bit probability is
// exact to 2^-17 and the ten rounds' twenty 32 x 32 -> 64 products are shared by eight
// elements, which leaves a kernel that reads and writes them bound by its bytes.
#pragma once
#include "f8_common.h"

namespace {

struct Drop {
  uint32_t threshold;        // of 65536: bits below it drop the element; 0: nothing is dropped
  uint32_t seed[2], offset[2];
  float scale;               // 65536 / (65536 - threshold)
};

__device__ __forceinline__ Drop drop_of(uint32_t threshold, const int64_t* rng) {
  Drop d{};
  d.threshold = threshold;
  d.scale = 65536.0f / (float)(65536u - threshold);
  if (threshold) {
    const uint64_t s = (uint64_t)rng[0], o = (uint64_t)rng[1];
    d.seed[0] = (uint32_t)s;
    d.seed[1] = (uint32_t)(s >> 32);
    d.offset[0] = (uint32_t)o;
    d.offset[1] = (uint32_t)(o >> 32);
  }
  return d;
}

// a ^ b ^ c in one instruction (0x96 is that function's truth table).
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
}

// Sixteen bits for each of a chunk's eight elements: element j's are half j % 2 of word j / 2.
__device__ __forceinline__ v4u random_bits(const Drop& d, uint64_t chunk) {
  uint32_t x0 = (uint32_t)chunk, x1 = (uint32_t)(chunk >> 32), x2 = d.offset[0], x3 = d.offset[1];
  uint32_t k0 = d.seed[0], k1 = d.seed[1];
  // (The ten rounds' keys anew for each chunk: kept from one to the next they and a kernel's pointers do
  // not fit the scalar registers.)
  asm("" : "+s"(k0), "+s"(k1) : "v"((uint32_t)chunk));
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)x0 * 0xd2511f53u, b = (uint64_t)x2 * 0xcd9e8d57u;
    x0 = xor3((uint32_t)(b >> 32), x1, k0);
    x1 = (uint32_t)b;
    x2 = xor3((uint32_t)(a >> 32), x3, k1);
    x3 = (uint32_t)a;
    k0 += 0x9e3779b9u;
    k1 += 0xbb67ae85u;
  }
  return v4u{x0, x1, x2, x3};
}

// A chunk's bits, and which of its elements stay: compared where they are, the higher half of a word as
// the whole word, which takes half the instructions of a mask of eight bits made first and asked later.
struct Kept {
  v4u w;
  uint32_t threshold;                        // in the higher half
  __device__ __forceinline__ Kept(const Drop& d, uint64_t chunk) : threshold(d.threshold << 16) {
    w = d.threshold ? random_bits(d, chunk) : v4u{0u, 0u, 0u, 0u};
  }
  __device__ __forceinline__ bool at(int j) const { return (j & 1 ? w[j >> 1] : w[j >> 1] << 16) >= threshold; }
};

// The same as a mask, a bit each, where it is kept from one use to the next.
__device__ __forceinline__ uint32_t kept_of(const Drop& d, uint64_t chunk) {
  if (d.threshold == 0) return 0xffu;
  const Kept k(d, chunk);
  uint32_t kept = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) kept |= (uint32_t)k.at(j) << j;
  return kept;
}

}  // namespace

// Dropout's mask, which is never stored: whoever needs it makes it again, from the seed and the
// elements' places.
//
// Element i of a tensor in row-major order belongs to group i / 8.  A group's 128 random bits are
// Philox4x32 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011) of
// the counter (group's low word, its high word, site, 0) under the key (seed's low word, its high word);
// element i has half i % 2, the low one first, of word i % 8 / 2.  It is dropped where these 16 bits
// are below T = 65536 p rounded, and what is kept is multiplied by 65536 / (65536 - T): p is a multiple
// of 2^-16, and the mean is kept exactly.  A select, no product: what is dropped is zero, infinite
// and undefined values as well.
//
// Seven rounds, the fewest with which the paper finds it to pass its tests.  Sixteen bits an element and
// eight to a group: a group is 16 bytes of 16-bit elements, a lane's piece of memory.
#pragma once
#include <hip/hip_runtime.h>

#include "w4a16_common.hpp"

namespace w4a16 {

struct DropArgs {
  const long long* seed_at;  // the seed in device memory, or null: `seed`
  unsigned long long seed;
  unsigned site, below;  // below = 0: nothing is dropped
  float factor;          // of what is kept
};

struct DropKey {
  unsigned lo, hi, site;
  __device__ __forceinline__ explicit DropKey(const DropArgs& a) : site(a.site) {
    const unsigned long long seed = a.seed_at ? (unsigned long long)*a.seed_at : a.seed;
    lo = (unsigned)seed;
    hi = (unsigned)(seed >> 32);
  }
};

constexpr int kDropRounds = 7;

// the random bits of a group, eight halves
__device__ __forceinline__ i4 drop_bits(unsigned long long group, const DropKey& key) {
  unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32), c2 = key.site, c3 = 0;
  unsigned k0 = key.lo, k1 = key.hi;
#pragma unroll
  for (int r = 0; r < kDropRounds; r++) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    const unsigned n0 = (unsigned)(b >> 32) ^ c1 ^ k0, n2 = (unsigned)(a >> 32) ^ c3 ^ k1;
    c0 = n0, c1 = (unsigned)b, c2 = n2, c3 = (unsigned)a;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return (i4){(int)c0, (int)c1, (int)c2, (int)c3};
}

// element e of the words that hold its bits
template <class Words>
__device__ __forceinline__ float drop_one(float v, const Words& bits, int e, const DropArgs& a) {
  const unsigned random = (unsigned)bits[e >> 1] >> (16 * (e & 1)) & 0xffffu;
  return random >= a.below ? v * a.factor : 0.f;
}

}  // namespace w4a16

// Masks of dropped values from a counter: Philox 4x32-10 (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).
//
// The eight values of columns 8 c .. 8 c + 7 of row r take one call: key the
// seed, counter (c, layer, low and high word of r), sixteen bits a value in
// ascending order.  A value is dropped where its bits are below
// `below` = round(65536 p).  The mask is a function of the value's place alone,
// so the gradient makes it anew and nothing is stored.  Sixteen bits make p good to
// 2^-17 and halve the rounds a value, twenty 32 x 32 bit products a call.
#pragma once

#include "common.h"

namespace ye3t {

struct Dropout {
  uint32_t below;       // 0: nothing is dropped
  uint32_t layer;
  uint64_t seed;
  const int64_t* from;  // the seed in device memory, or null
  float scale;          // of kept values, 65536 / (65536 - below)
};

inline Dropout dropout_of(int64_t below, uint32_t layer, uint64_t seed, const int64_t* from) {
  return {uint32_t(below), layer, seed, from, below < 65536 ? float(65536.0 / double(65536 - below)) : 0.0f};
}

__device__ inline uint64_t seed_of(const Dropout& d) { return d.from ? uint64_t(*d.from) : d.seed; }

struct Bits {
  uint32_t w[4];
  // of value q < 8
  __device__ uint32_t operator[](int q) const { return q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xFFFFu; }
};

__device__ inline Bits bits_of(uint64_t seed, uint32_t layer, int64_t row, uint32_t chunk) {
  uint32_t c0 = chunk, c1 = layer, c2 = uint32_t(row), c3 = uint32_t(uint64_t(row) >> 32);
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = uint64_t(c0) * 0xD2511F53u, q = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(q >> 32) ^ c1 ^ k0;
    c1 = uint32_t(q);
    c2 = uint32_t(p >> 32) ^ c3 ^ k1;
    c3 = uint32_t(p);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Eight values of a row, dropped ones zero whatever they held.
__device__ inline void drop(const Dropout& d, uint64_t seed, int64_t row, uint32_t chunk, float* v) {
  const Bits b = bits_of(seed, d.layer, row, chunk);
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = b[q] < d.below ? 0.0f : v[q] * d.scale;
}

}  // namespace ye3t

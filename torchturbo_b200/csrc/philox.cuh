// Dropout masks from a counter-based generator: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011).  Nothing is stored: whoever needs the mask of an element again draws it again from the element's place and the seed.
//   counter (g, 0, i mod 2^32, i div 2^32), key = the seed's two words; the eight 16-bit halves of the four words (low half first) belong
//   to columns 8 g .. 8 g + 7 of row i; a value stays where its half is at least t = round(65536 p), times 65536 / (65536 - t).
// Sixteen bits a value: half the draws of 32, and the factor above is that of the probability that is really drawn with, so that the mean
// is kept exactly however p was rounded.
#pragma once
#include <stdint.h>

namespace ttb {

struct DropoutParams {
  uint32_t t;                        // 0: nothing is dropped
  float scale;                       // of what stays
  uint64_t seed;
  const unsigned long long* seed_dev;   // the seed, where it is known on the device only (a captured step whose seed moves on)
  long long first_row;               // place of this tensor's first row among the rows of the whole
};

struct PhiloxKey {
  uint32_t k0, k1;
};
__device__ __forceinline__ PhiloxKey dropout_key(const DropoutParams& d) {
  const uint64_t s = d.seed_dev ? *d.seed_dev : d.seed;
  return PhiloxKey{static_cast<uint32_t>(s), static_cast<uint32_t>(s >> 32)};
}

__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, PhiloxKey k) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k.k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k.k1;
    c3 = static_cast<uint32_t>(a);
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// draws of columns 8 g .. 8 g + 7
__device__ __forceinline__ uint4 dropout_draws(long long row, uint32_t g, PhiloxKey k) {
  return philox(g, 0u, static_cast<uint32_t>(row), static_cast<uint32_t>(static_cast<uint64_t>(row) >> 32), k);
}
// eight values: what stays times the factor, the rest zero (whatever it was)
__device__ __forceinline__ void dropout8(float* f, const uint4& u, uint32_t t, float scale) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = (w[j] & 0xffffu) >= t ? f[2 * j] * scale : 0.f;
    f[2 * j + 1] = (w[j] >> 16) >= t ? f[2 * j + 1] * scale : 0.f;
  }
}

}  // namespace ttb

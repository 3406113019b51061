// Dropout masks from a counter-based generator: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", 2011).  Nothing is stored: whoever needs the mask of an element again draws it again from the element's place and the seed.
//   counter (g, 0, i mod 2^32, i div 2^32), key = the seed's two words; the eight 16-bit halves of the four words (low half first) belong
//   to columns 8 g .. 8 g + 7 of row i; a value stays where its half is at least t = round(65536 p), times 65536 / (65536 - t).
// Sixteen bits a value: half the draws of 32, and the factor above is that of the probability that is really drawn with, so that the mean
// is kept exactly however p was rounded.
//
// A round multiplies two words by constants, 32 x 32 -> 64 bits, at a quarter of the rate of its other instructions: ten rounds for every
// eight bf16 values, twenty products, take nearly as long as a copy of the values.  The products of the first two rounds depend on the
// column group alone or on the row alone: a thread that stays in a column, or in a row, makes its share of them once, and 16 of 20
// are left per group (backward of 16384 x 4096 with dropout 72 -> 60 us, with the walk of dropout.cu).  Products as two instructions of 32 bits
// take the same time.
#pragma once
#include <stdint.h>

namespace ttb {

struct DropoutParams {
  uint32_t t;                        // below 65536; 0: nothing is dropped
  float scale;                       // of what stays
  uint32_t key[20];                  // the rounds' keys
  const unsigned long long* seed_dev;   // the seed, where it is known on the device only (a captured step whose seed moves on)
  long long first_row;               // place of this tensor's first row among the rows of the whole
};
constexpr uint32_t PHILOX_W0 = 0x9E3779B9u, PHILOX_W1 = 0xBB67AE85u;
inline DropoutParams dropout_params(uint32_t t, float scale, uint64_t seed, const unsigned long long* seed_dev, long long first_row) {
  DropoutParams d{t, scale, {}, seed_dev, first_row};
  for (uint32_t i = 0; i < 10; ++i) {
    d.key[2 * i] = static_cast<uint32_t>(seed) + i * PHILOX_W0;
    d.key[2 * i + 1] = static_cast<uint32_t>(seed >> 32) + i * PHILOX_W1;
  }
  return d;
}

// Keys of the rounds: from the launch's parameters (operands of the rounds' instructions as they are) or from a seed in memory
struct KeysOfLaunch {
  const DropoutParams& d;
  __device__ __forceinline__ explicit KeysOfLaunch(const DropoutParams& p) : d(p) {}
  __device__ __forceinline__ uint32_t k0(int i) const { return d.key[2 * i]; }
  __device__ __forceinline__ uint32_t k1(int i) const { return d.key[2 * i + 1]; }
};
struct KeysOfSeed {
  uint32_t a, b;
  __device__ __forceinline__ explicit KeysOfSeed(const DropoutParams& p) {
    a = p.key[0];
    b = p.key[1];
    if (p.seed_dev) {
      const uint64_t s = *p.seed_dev;
      a = static_cast<uint32_t>(s);
      b = static_cast<uint32_t>(s >> 32);
    }
  }
  __device__ __forceinline__ uint32_t k0(int i) const { return a + i * PHILOX_W0; }
  __device__ __forceinline__ uint32_t k1(int i) const { return b + i * PHILOX_W1; }
};

__device__ __forceinline__ void philox_mul(uint32_t x, uint32_t m, uint32_t& hi, uint32_t& lo) {
  const uint64_t p = static_cast<uint64_t>(x) * m;
  hi = static_cast<uint32_t>(p >> 32);
  lo = static_cast<uint32_t>(p);
}
// what column group g, and row i, give to the first two rounds
struct PhiloxColumn {
  uint32_t lo, hi2, lo2;
};
struct PhiloxRow {
  uint32_t lo, hi2, lo2;
};
template <typename Keys>
__device__ __forceinline__ PhiloxColumn philox_column(uint32_t g, uint32_t row_hi, const Keys& k) {
  PhiloxColumn c;
  uint32_t hi;
  philox_mul(g, 0xD2511F53u, hi, c.lo);
  philox_mul(hi ^ row_hi ^ k.k1(0), 0xCD9E8D57u, c.hi2, c.lo2);
  return c;
}
template <typename Keys>
__device__ __forceinline__ PhiloxRow philox_row(uint32_t row_lo, const Keys& k) {
  PhiloxRow r;
  uint32_t hi;
  philox_mul(row_lo, 0xCD9E8D57u, hi, r.lo);
  philox_mul(hi ^ k.k0(0), 0xD2511F53u, r.hi2, r.lo2);
  return r;
}
// draws of a column group in a row
template <typename Keys>
__device__ __forceinline__ uint4 philox(const PhiloxColumn& c, const PhiloxRow& r, const Keys& k) {
  uint32_t c0 = c.hi2 ^ r.lo ^ k.k0(1), c1 = c.lo2, c2 = r.hi2 ^ c.lo ^ k.k1(1), c3 = r.lo2;
#pragma unroll
  for (int i = 2; i < 10; ++i) {
    uint32_t ah, al, bh, bl;
    philox_mul(c0, 0xD2511F53u, ah, al);
    philox_mul(c2, 0xCD9E8D57u, bh, bl);
    c0 = bh ^ c1 ^ k.k0(i);
    c1 = bl;
    c2 = ah ^ c3 ^ k.k1(i);
    c3 = al;
  }
  return make_uint4(c0, c1, c2, c3);
}
template <typename Keys>
__device__ __forceinline__ uint4 dropout_draws(long long row, uint32_t g, const Keys& k) {
  return philox(philox_column(g, static_cast<uint32_t>(static_cast<uint64_t>(row) >> 32), k), philox_row(static_cast<uint32_t>(row), k), k);
}

// Eight values: what stays times the factor, the rest zero (whatever it was).  `top` is t in the upper half of a word: an upper half is
// compared where it is, a lower one shifted up.
__device__ __forceinline__ void dropout8(float* f, const uint4& u, uint32_t top, float scale) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = (w[j] << 16) >= top ? f[2 * j] * scale : 0.f;
    f[2 * j + 1] = w[j] >= top ? f[2 * j + 1] * scale : 0.f;
  }
}

}  // namespace ttb

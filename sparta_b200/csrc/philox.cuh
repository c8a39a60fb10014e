// Counter-based random bits for dropout: Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011; seven rounds are the fewest that its authors report as passing BigCrush).
//
// A decision belongs to a position (batch element b, row r, column c) of a call, not to a thread or a layout:
//   counter = (c / 8, r, b, call)   key = seed   ->   128 bits = eight 16-bit values, the one of column c at place c % 8
//   keep    <=>   value >= threshold,   threshold = round(65536 p)
// so a dense tensor, block values in any block size, and the fused attention kernels (forward, and the backward
// passes that hold the scores one way round or the other) all drop the same positions, and nothing is kept between them.  Eight
// decisions per call of the generator: 16 bits resolve p to 1 / 65536, and the scale 65536 / (65536 - threshold) is
// that of the rounded probability, so the expectation is exact.
#pragma once

#include "common.cuh"

namespace sparta {

constexpr uint32_t kDropoutOne = 65536u;  // probability 1 as a threshold

struct DropoutParams {
  const int64_t* rng;   // device (seed, call number) or null: the two values below
  uint64_t seed;
  uint32_t call;
  uint32_t threshold;   // 0: nothing dropped, 65536: everything
  float scale;          // 65536 / (65536 - threshold); 0 when everything is dropped
};

// p in [0, 1] -> threshold and scale; false when p is no probability
inline bool make_dropout(DropoutParams* d, double p, const int64_t* rng, uint64_t seed, uint64_t call) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  d->rng = rng;
  d->seed = seed;
  d->call = static_cast<uint32_t>(call);
  d->threshold = static_cast<uint32_t>(p * 65536.0 + 0.5);
  d->scale = d->threshold >= kDropoutOne ? 0.f : 65536.f / static_cast<float>(kDropoutOne - d->threshold);
  return true;
}

struct PhiloxKey {
  uint32_t k0, k1, call;
};

__device__ __forceinline__ PhiloxKey load_philox_key(const DropoutParams& d) {
  uint64_t seed = d.seed;
  uint32_t call = d.call;
  if (d.rng) {
    seed = static_cast<uint64_t>(__ldg(d.rng));
    call = static_cast<uint32_t>(__ldg(d.rng + 1));
  }
  return {static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32), call};
}

// After two of the seven rounds two of the four words depend on (column, batch element) alone, and of the other two's
// product one factor on (row, batch element) alone: of fourteen products nine depend on both.  Kernels make the row's
// and the column's share once for as many positions as they can.
struct PhiloxRow {
  uint32_t hi, lo;          // of the second round's product, the key in `hi`
};
struct PhiloxCol {
  uint32_t w3, k0, k2, x3;  // round one's fourth word; what the third round's words are combined with; its fourth word
};
constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u, kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

__device__ __forceinline__ PhiloxRow philox_row(const PhiloxKey& key, uint32_t row, uint32_t batch) {
  const uint32_t x0 = __umulhi(kPhiloxM1, batch) ^ row ^ key.k0;
  const uint64_t a = static_cast<uint64_t>(kPhiloxM0) * x0;
  return {static_cast<uint32_t>(a >> 32) ^ (key.k1 + kPhiloxW1), static_cast<uint32_t>(a)};
}
__device__ __forceinline__ PhiloxCol philox_col(const PhiloxKey& key, uint32_t g, uint32_t batch) {
  const uint64_t a1 = static_cast<uint64_t>(kPhiloxM0) * g;
  const uint64_t b2 = static_cast<uint64_t>(kPhiloxM1) * (static_cast<uint32_t>(a1 >> 32) ^ key.call ^ key.k1);
  const uint64_t a3 = static_cast<uint64_t>(kPhiloxM0) * (static_cast<uint32_t>(b2 >> 32) ^ (kPhiloxM1 * batch) ^ (key.k0 + kPhiloxW0));
  return {static_cast<uint32_t>(a1), static_cast<uint32_t>(b2) ^ (key.k0 + 2 * kPhiloxW0),
          static_cast<uint32_t>(a3 >> 32) ^ (key.k1 + 2 * kPhiloxW1), static_cast<uint32_t>(a3)};
}
// eight 16-bit values of columns 8 g .. 8 g + 7, two per word, lower column in the lower half
__device__ __forceinline__ void philox8(const PhiloxKey& key, const PhiloxRow& r, const PhiloxCol& c, uint32_t (&w)[4]) {
  const uint64_t b3 = static_cast<uint64_t>(kPhiloxM1) * (r.hi ^ c.w3);
  uint32_t x0 = static_cast<uint32_t>(b3 >> 32) ^ c.k0, x1 = static_cast<uint32_t>(b3), x2 = c.k2 ^ r.lo, x3 = c.x3;
#pragma unroll
  for (int i = 3; i < 7; ++i) {
    const uint64_t a = static_cast<uint64_t>(kPhiloxM0) * x0, b = static_cast<uint64_t>(kPhiloxM1) * x2;
    x0 = static_cast<uint32_t>(b >> 32) ^ x1 ^ (key.k0 + i * kPhiloxW0);
    x1 = static_cast<uint32_t>(b);
    x2 = static_cast<uint32_t>(a >> 32) ^ x3 ^ (key.k1 + i * kPhiloxW1);
    x3 = static_cast<uint32_t>(a);
  }
  w[0] = x0; w[1] = x1; w[2] = x2; w[3] = x3;
}
// the same key in every lane, known to the compiler as such; every lane of the warp calls it
__device__ __forceinline__ PhiloxKey load_uniform_philox_key(const DropoutParams& d) {
  const PhiloxKey k = load_philox_key(d);
  return {__shfl_sync(0xffffffffu, k.k0, 0), __shfl_sync(0xffffffffu, k.k1, 0), __shfl_sync(0xffffffffu, k.call, 0)};
}

// Bits 15 and 31: the halves of w are not below the halves of t (a threshold below 65536 twice).  Side by side: with
// the top bits set aside, a subtraction of the lower 15 bits leaves its borrow in place of the top bit, and the result
// is decided by the top bits or, where they agree, by that.
__device__ __forceinline__ uint32_t not_below2(uint32_t w, uint32_t t) {
  const uint32_t d = (w | 0x80008000u) - (t & 0x7fff7fffu);
  return (w & ~t) | (~(w ^ t) & d);
}
// bits 15 and 31 over their halves
__device__ __forceinline__ uint32_t spread2(uint32_t x) {
  uint32_t m;
  asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(m) : "r"(x));  // sign of byte 1, byte 3 over two bytes each
  return m;
}
// bits 15 and 31 of two words, each over a byte, lower columns in lower bytes
__device__ __forceinline__ uint32_t spread4(uint32_t a, uint32_t b) {
  uint32_t m;
  asm("prmt.b32 %0, %1, %2, 0xfdb9;" : "=r"(m) : "r"(a), "r"(b));
  return m;
}
// The threshold in both halves.  "Everything dropped" (65536) becomes "nothing": its scale is 0.
__device__ __forceinline__ uint32_t threshold2(const DropoutParams& d) { return (d.threshold & 0xffffu) * 0x00010001u; }

}  // namespace sparta

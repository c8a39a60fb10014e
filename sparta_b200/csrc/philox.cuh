// Counter-based random bits for dropout: Philox4x32 with seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011; seven rounds are the fewest that its authors report as passing BigCrush).
//
// A decision belongs to a position (batch element b, row r, column c) of a call, not to a thread or a layout:
//   counter = (c / 8, r, b, call)   key = seed   ->   128 bits = eight 16-bit values, the one of column c at place c % 8
//   keep    <=>   value >= threshold,   threshold = round(65536 p)
// so a dense tensor, block values in any block size, and the fused attention kernels (forward, and the backward
// passes that hold the scores one way round or the other) all drop the same positions, and nothing is stored.  Eight
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

// eight 16-bit values of columns 8 g .. 8 g + 7, two per word, lower column in the lower half
__device__ __forceinline__ void philox8(const PhiloxKey& key, uint32_t g, uint32_t row, uint32_t batch, uint32_t (&w)[4]) {
  uint32_t x0 = g, x1 = row, x2 = batch, x3 = key.call, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * x0, b = static_cast<uint64_t>(0xCD9E8D57u) * x2;
    x0 = static_cast<uint32_t>(b >> 32) ^ x1 ^ k0;
    x1 = static_cast<uint32_t>(b);
    x2 = static_cast<uint32_t>(a >> 32) ^ x3 ^ k1;
    x3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = x0; w[1] = x1; w[2] = x2; w[3] = x3;
}

// bit c: column 8 g + c is kept.  cut = threshold << 16 (threshold < 65536): the upper half of a word is not below the
// threshold exactly when the word is not below `cut`, the lower half exactly when the word shifted up is not.
__device__ __forceinline__ uint32_t philox_keep8(const PhiloxKey& key, uint32_t cut, uint32_t g, uint32_t row, uint32_t batch) {
  uint32_t w[4], bits = 0;
  philox8(key, g, row, batch, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bits |= ((w[i] << 16) >= cut ? 1u : 0u) << (2 * i);
    bits |= (w[i] >= cut ? 1u : 0u) << (2 * i + 1);
  }
  return bits;
}

}  // namespace sparta

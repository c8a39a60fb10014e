// What the fused attention kernels share: their arguments, the bare exponential, packing, and words of 32 mask or
// dropout decisions.
#pragma once

#include "philox.cuh"

namespace sparta {

// Arguments of the fused attention entry points, checked by them (attn_tc.cu).
struct AttnArgs {
  const void* Q;
  const void* K;
  const void* V;
  void* O;
  float* lse;               // [heads, Nt]: written forward (may be null), read backward
  const void* dO;           // backward only, like the three below
  void* dQ;
  void* dK;
  void* dV;
  void* workspace;
  const int32_t* row_ptr;
  const int32_t* idx;
  const uint8_t* mask;      // [Nt, Ns] element mask or null
  float scale;
  int heads, kv_heads;      // heads / kv_heads query heads share a key / value head
  int Nt, Ns, D, dtype;
  long long nnz;            // kept blocks, 0 when unknown
};

// fused attention with two Q tiles per CTA (attn_tc2.cu): query lengths that are a multiple of 256
bool attn_tc2_supported(int Nt);
bool kv_exceeds_l2(int heads, int Ns, int D);
int attn_tc2_launch(const AttnArgs& a, const DropoutParams& drop, int32_t* status, void* const* copies, int n_copies,
                    cudaStream_t st);

// fused attention for head dim 64 with one K block per step and four CTAs per SM (attn_tc64.cu)
int attn_tc64_launch(const AttnArgs& a, const DropoutParams& drop, int32_t* status, cudaStream_t st);

// backward pass (attn_bwd.cu)
size_t attn_bwd_workspace(int heads, int kv_heads, int Nt, int Ns, int D, long long nnz);
int attn_bwd_launch(const AttnArgs& a, const DropoutParams& drop, int32_t* status, cudaStream_t st);

// 2^x by the special-function unit alone.  exp2f() wraps the same instruction in a range fix for
// results below the normal range (a compare, two multiplies); probabilities that small round to zero
// in fp16 / bf16 anyway, and the softmax warps are bound by the number of instructions they issue.
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// two values rounded to 16 bits (to nearest), the first in the lower half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float v0, float v1);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float v0, float v1) {
  const __half2 h = __floats2half2_rn(v0, v1);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float v0, float v1) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v0, v1);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ---- words of 32 decisions about consecutive columns ----
// In "split" order bit i is column 2 i and bit 16 + i column 2 i + 1: the two bits of a packed pair of 16-bit values are
// 16 apart, so that one shift and one byte permutation make the mask of the pair.
__device__ __forceinline__ uint32_t to_split32(uint32_t c) { return (c >> 1) | ((c & 1u) << 4); }        // column -> bit
__device__ __forceinline__ uint32_t from_split32(uint32_t i) { return ((i & 15u) << 1) | (i >> 4); }  // bit -> column

// ---- the generator for a row of the score matrix ----
// The counter is (column / 8, row, batch element, call).  After two of the seven rounds two of the four words depend on
// (column, batch element) alone and two on the row as well, so that of fourteen products nine are left that depend on
// both; a row's own product is made once, and those of the column are the same for a whole warp.
struct PhiloxRow {
  uint32_t hi, lo;  // of the second round's product, the key in `hi`
};
__device__ __forceinline__ PhiloxRow philox_row(const PhiloxKey& key, uint32_t row, uint32_t batch) {
  const uint32_t x0 = __umulhi(0xCD9E8D57u, batch) ^ row ^ key.k0;
  const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * x0;
  return {static_cast<uint32_t>(a >> 32) ^ (key.k1 + 0xBB67AE85u), static_cast<uint32_t>(a)};
}
__device__ __forceinline__ void philox8_row(const PhiloxKey& key, const PhiloxRow& r, uint32_t g, uint32_t batch, uint32_t (&w)[4]) {
  constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u, kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;
  const uint64_t a1 = static_cast<uint64_t>(kM0) * g;
  const uint64_t b2 = static_cast<uint64_t>(kM1) * (static_cast<uint32_t>(a1 >> 32) ^ key.call ^ key.k1);
  const uint64_t a3 = static_cast<uint64_t>(kM0) * (static_cast<uint32_t>(b2 >> 32) ^ (kM1 * batch) ^ (key.k0 + kW0));
  const uint64_t b3 = static_cast<uint64_t>(kM1) * (r.hi ^ static_cast<uint32_t>(a1));
  uint32_t x0 = static_cast<uint32_t>(b3 >> 32) ^ (static_cast<uint32_t>(b2) ^ (key.k0 + 2 * kW0));
  uint32_t x1 = static_cast<uint32_t>(b3);
  uint32_t x2 = (static_cast<uint32_t>(a3 >> 32) ^ (key.k1 + 2 * kW1)) ^ r.lo;
  uint32_t x3 = static_cast<uint32_t>(a3);
#pragma unroll
  for (int i = 3; i < 7; ++i) {
    const uint64_t a = static_cast<uint64_t>(kM0) * x0, b = static_cast<uint64_t>(kM1) * x2;
    x0 = static_cast<uint32_t>(b >> 32) ^ x1 ^ (key.k0 + i * kW0);
    x1 = static_cast<uint32_t>(b);
    x2 = static_cast<uint32_t>(a >> 32) ^ x3 ^ (key.k1 + i * kW1);
    x3 = static_cast<uint32_t>(a);
  }
  w[0] = x0; w[1] = x1; w[2] = x2; w[3] = x3;
}
// the same key in every lane, known to the compiler as such
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
// 0xffff in each half whose bit (i, 16 + i) is set
__device__ __forceinline__ uint32_t pair_mask(uint32_t word, int i) { return spread2(word << (15 - i)); }

// The threshold in both halves.  "Everything dropped" (65536) becomes "nothing": its scale is 0.
__device__ __forceinline__ uint32_t threshold2(const DropoutParams& d) { return (d.threshold & 0xffffu) * 0x00010001u; }

// 32 dropout decisions of columns 32 g .. of a row, split order
__device__ __forceinline__ uint32_t philox_split32(const PhiloxKey& key, const PhiloxRow& r, uint32_t t2, uint32_t g, uint32_t batch) {
  uint32_t bits = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[4];
    philox8_row(key, r, 4 * g + q, batch, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) bits = (bits >> 1) | (not_below2(w[i], t2) & 0x80008000u);
  }
  return bits;
}
// packed pairs of columns 32 g .. of a row: the dropped ones to zero
__device__ __forceinline__ void drop_packed32(uint32_t* packed, const PhiloxKey& key, const PhiloxRow& r, uint32_t t2, uint32_t g, uint32_t batch) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[4];
    philox8_row(key, r, 4 * g + q, batch, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) packed[4 * q + i] &= spread2(not_below2(w[i], t2));
  }
}

// 32 mask bytes (16-byte aligned) -> bit i set when byte i is not zero
__device__ __forceinline__ uint32_t mask_word32(const uint8_t* m) {
  const uint4 lo = __ldg(reinterpret_cast<const uint4*>(m)), hi = __ldg(reinterpret_cast<const uint4*>(m) + 1);
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // top bit of every byte: the byte is not zero; the product gathers the four of them in its highest four bits
    const uint32_t t = (((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) & 0x80808080u;
    bits |= (((t >> 7) * 0x10204080u) >> 28) << (4 * i);
  }
  return bits;
}

// the same in split order: the even bits gathered in the lower half, the odd ones in the upper
__device__ __forceinline__ uint32_t mask_split32(const uint8_t* m) {
  uint32_t x = mask_word32(m), t;
  t = (x ^ (x >> 1)) & 0x22222222u; x ^= t ^ (t << 1);
  t = (x ^ (x >> 2)) & 0x0c0c0c0cu; x ^= t ^ (t << 2);
  t = (x ^ (x >> 4)) & 0x00f000f0u; x ^= t ^ (t << 4);
  t = (x ^ (x >> 8)) & 0x0000ff00u; x ^= t ^ (t << 8);
  return x;
}

// 32 x 32 bits across a warp, lane l holding row l: afterwards lane l holds column l (bit i = bit l of row i).  Swaps
// the off-diagonal halves of ever smaller squares.
__device__ __forceinline__ uint32_t transpose_bits32(uint32_t x, int lane) {
  uint32_t low = 0x0000ffffu;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const uint32_t y = __shfl_xor_sync(0xffffffffu, x, s);
    x = (lane & s) == 0 ? ((x & low) | ((y & low) << s)) : (((y >> s) & low) | (x & ~low));
    low ^= low << (s >> 1);
  }
  return x;
}

}  // namespace sparta

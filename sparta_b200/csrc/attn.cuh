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
  size_t workspace_bytes;
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
size_t attn_bwd_dropout_workspace(int heads, long long nnz);
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
// 0xffff in each half whose bit (i, 16 + i) is set
__device__ __forceinline__ uint32_t pair_mask(uint32_t word, int i) { return spread2(word << (15 - i)); }

// 32 dropout decisions of columns 32 g .. of a row, column c at bit 7 - c / 4 of byte c % 4: shifted left by u, the signs of
// the four bytes are columns 4 u .. 4 u + 3.
__device__ __forceinline__ uint32_t philox_bits32(const PhiloxKey& key, const PhiloxRow& r, uint32_t t2, uint32_t g, uint32_t batch) {
  uint32_t part[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[4];
    philox8(key, r, philox_col(key, 4 * g + q, batch), w);
    part[q] = (spread4(not_below2(w[0], t2), not_below2(w[1], t2)) & (0x80808080u >> (2 * q))) |
              (spread4(not_below2(w[2], t2), not_below2(w[3], t2)) & (0x40404040u >> (2 * q)));
  }
  return (part[0] | part[1]) | (part[2] | part[3]);
}
// packed pairs of columns 32 g .. of a row: the dropped ones to zero
__device__ __forceinline__ void drop_packed32(uint32_t* packed, const PhiloxKey& key, const PhiloxRow& r, uint32_t t2, uint32_t g, uint32_t batch) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t w[4];
    philox8(key, r, philox_col(key, 4 * g + q, batch), w);
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

// the even bits gathered in the lower half, the odd ones in the upper
__device__ __forceinline__ uint32_t split_bits32(uint32_t x) {
  uint32_t t;
  t = (x ^ (x >> 1)) & 0x22222222u; x ^= t ^ (t << 1);
  t = (x ^ (x >> 2)) & 0x0c0c0c0cu; x ^= t ^ (t << 2);
  t = (x ^ (x >> 4)) & 0x00f000f0u; x ^= t ^ (t << 4);
  t = (x ^ (x >> 8)) & 0x0000ff00u; x ^= t ^ (t << 8);
  return x;
}
}  // namespace sparta

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
};

// fused attention with two Q tiles per CTA (attn_tc2.cu): query lengths that are a multiple of 256
bool attn_tc2_supported(int Nt);
bool kv_exceeds_l2(int heads, int Ns, int D);
int attn_tc2_launch(const AttnArgs& a, const DropoutParams& drop, int32_t* status, void* const* copies, int n_copies,
                    cudaStream_t st);

// fused attention for head dim 64 with one K block per step and four CTAs per SM (attn_tc64.cu)
int attn_tc64_launch(const AttnArgs& a, const DropoutParams& drop, int32_t* status, cudaStream_t st);

// backward pass (attn_bwd.cu)
size_t attn_bwd_workspace(int heads, int Nt, int Ns);
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

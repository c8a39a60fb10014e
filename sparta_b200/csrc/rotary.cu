// Rotary positions: each pair (a, b) of the first `rotary_dim` elements of a head is turned by the angle
// position * f_i,   a' = m (a cos - b sin),  b' = m (b cos + a sin),   the rest of the head is copied.
// Pairs are (2 i, 2 i + 1) (interleaved) or (i, i + rotary_dim / 2).  The backward pass turns the gradient by the
// negative angle: the same kernel with the sine's sign changed.
//
// The angle.  In 32-bit floating point position * f_i is off by whole radians at the far end of a long context, and
// 64-bit floating point is slow here, so f_i comes as an unsigned 64-bit fraction of a TURN, f_i / (2 pi) * 2^64: the
// product with the position, modulo 2^64, is the angle modulo one turn, exact to position * 2^-65 turns, and its upper
// half goes to sincospi.
//
// Bound by HBM: one read and one write of each element.  A thread holds the angles of the pairs in one 16-byte vector
// (interleaved) or in one vector of first and one of second elements of a token and walks over several heads with them, so that the sines cost a
// few instructions per element; few tokens (a decoding step) are spread over heads instead.  Queries and keys are
// two entries of one launch (blockIdx.z).  Inputs may have any batch / head / token stride, so the token-major tensor
// that a projection leaves is turned and brought into the attention's head-major order in one pass.
#include "common.cuh"

namespace sparta {
namespace {

constexpr int kThreads = 256;

struct RotaryTensor {
  const void* x;
  void* y;
  const void* positions;   // [n], or [batch, n] with pos_batched; null: 0, 1, 2 ...
  long long sb, sh, sn;    // strides of x in elements; y is [batch, heads, n, dim]
  int batch, heads, n;
  int pos_batched;
};
struct RotaryParams {
  RotaryTensor t[2];
  const uint64_t* turns;   // [rotary_dim / 2]
  float magnitude, sign;
  int dim, half, heads_per_thread;
  int pos64;
};

__device__ __forceinline__ void turn_of(uint64_t freq, int64_t pos, float magnitude, float sign, float& c, float& s) {
  const uint64_t angle = freq * static_cast<uint64_t>(pos);  // modulo one turn; negative positions wrap alike
  const float half_turns = static_cast<float>(static_cast<int32_t>(angle >> 32)) * 4.656612873077393e-10f;  // 2^-31: [-1, 1]
  sincospif(half_turns, &s, &c);
  c *= magnitude;
  s *= magnitude * sign;
}

__device__ __forceinline__ int64_t position_of(const RotaryTensor& t, int pos64, int b, int i) {
  if (!t.positions) return i;
  const long long k = (t.pos_batched ? (long long)b * t.n : 0ll) + i;
  return pos64 ? __ldg(static_cast<const long long*>(t.positions) + k)
               : static_cast<int64_t>(__ldg(static_cast<const int*>(t.positions) + k));
}

// 16-byte vectors: V elements; the turned part and the head whole vectors, addresses and strides multiples of one.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_vec_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int V = 16 / sizeof(T);
  const RotaryTensor& t = p.t[blockIdx.z];
  // Units of P pairs, then (in warps of their own) units of V copied elements.  Interleaved pairs take one vector per
  // unit: with two, a thread's stores were halves of 32-byte sectors (16384 tokens, 40 heads, 96 of 128: 68 us).
  constexpr int P = INTERLEAVED ? V / 2 : V, kVecs = INTERLEAVED ? 1 : 2, kBatch = 4;  // heads with loads in flight
  const int turned = p.half / P, copied = (p.dim - 2 * p.half) / V;
  const long long tokens = (long long)t.batch * t.n, pairs_end = (tokens * turned + 31) / 32 * 32;
  long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
  const bool copies = id >= pairs_end;
  const int units = copies ? copied : turned;
  if (copies) id -= pairs_end;
  const int h0 = blockIdx.y * p.heads_per_thread;
  if (id >= tokens * units || h0 >= t.heads) return;
  const int h1 = min(h0 + p.heads_per_thread, t.heads);
  const long long token = id / units;
  const int u = static_cast<int>(id - token * units);
  const int b = static_cast<int>(token / t.n), i = static_cast<int>(token - (long long)b * t.n);
  const T* x = static_cast<const T*>(t.x) + b * t.sb + i * t.sn + h0 * t.sh;
  const long long y_head = (long long)t.n * p.dim;
  T* y = static_cast<T*>(t.y) + ((long long)b * t.heads + h0) * y_head + (long long)i * p.dim;
  if (copies) {
    const int at = 2 * p.half + u * V;
    for (int h = h0; h < h1; h += kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (h + j < h1) v[j] = __ldg(reinterpret_cast<const uint4*>(x + (h - h0 + j) * t.sh + at));
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (h + j < h1) *reinterpret_cast<uint4*>(y + (h - h0 + j) * y_head + at) = v[j];
    }
    return;
  }
  const int at0 = u * V, at1 = at0 + p.half;
  float c[P], s[P];
  for (int h = h0; h < h1; h += kBatch) {
    __align__(16) T v[kBatch][kVecs * V];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (h + j < h1) {
        const T* src = x + (h - h0 + j) * t.sh;
        *reinterpret_cast<uint4*>(v[j]) = __ldg(reinterpret_cast<const uint4*>(src + at0));
        if constexpr (!INTERLEAVED) *reinterpret_cast<uint4*>(v[j] + V) = __ldg(reinterpret_cast<const uint4*>(src + at1));
      }
    if (h == h0) {  // under the first loads
      const int64_t pos = position_of(t, p.pos64, b, i);
#pragma unroll
      for (int k = 0; k < P; ++k) turn_of(__ldg(p.turns + u * P + k), pos, p.magnitude, p.sign, c[k], s[k]);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (h + j >= h1) break;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        T& e0 = v[j][INTERLEAVED ? 2 * k : k];
        T& e1 = v[j][INTERLEAVED ? 2 * k + 1 : V + k];
        const float f0 = to_float(e0), f1 = to_float(e1);
        e0 = from_float<T>(f0 * c[k] - f1 * s[k]);
        e1 = from_float<T>(f1 * c[k] + f0 * s[k]);
      }
      T* dst = y + (h - h0 + j) * y_head;
      *reinterpret_cast<uint4*>(dst + at0) = *reinterpret_cast<const uint4*>(v[j]);
      if constexpr (!INTERLEAVED) *reinterpret_cast<uint4*>(dst + at1) = *reinterpret_cast<const uint4*>(v[j] + V);
    }
  }
}

// Any sizes, strides and alignment: a thread turns one pair, or copies one element behind the turned part.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_pair_kernel(const __grid_constant__ RotaryParams p, int interleaved) {
  const RotaryTensor& t = p.t[blockIdx.z];
  const int units = p.dim - p.half;  // half pairs, dim - 2 half copies
  const long long id = (long long)blockIdx.x * kThreads + threadIdx.x;
  const long long tokens = (long long)t.batch * t.n;
  const int h0 = blockIdx.y * p.heads_per_thread;
  if (id >= tokens * units || h0 >= t.heads) return;
  const int h1 = min(h0 + p.heads_per_thread, t.heads);
  const long long token = id / units;
  const int u = static_cast<int>(id - token * units);
  const int b = static_cast<int>(token / t.n), i = static_cast<int>(token - (long long)b * t.n);
  const T* x = static_cast<const T*>(t.x) + b * t.sb + i * t.sn + h0 * t.sh;
  const long long y_head = (long long)t.n * p.dim;
  T* y = static_cast<T*>(t.y) + ((long long)b * t.heads + h0) * y_head + (long long)i * p.dim;
  if (u >= p.half) {
    const int at = p.half + u;
    for (int h = h0; h < h1; ++h, x += t.sh, y += y_head) y[at] = x[at];
    return;
  }
  float c, s;
  turn_of(__ldg(p.turns + u), position_of(t, p.pos64, b, i), p.magnitude, p.sign, c, s);
  const int at0 = interleaved ? 2 * u : u, at1 = interleaved ? at0 + 1 : at0 + p.half;
  for (int h = h0; h < h1; ++h, x += t.sh, y += y_head) {
    const float f0 = to_float(x[at0]), f1 = to_float(x[at1]);
    y[at0] = from_float<T>(f0 * c - f1 * s);
    y[at1] = from_float<T>(f1 * c + f0 * s);
  }
}

template <typename T>
int launch_rotary(RotaryParams& p, int count, int interleaved, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int pairs = interleaved ? V / 2 : V;  // of a thread
  bool vec = p.half % pairs == 0 && p.dim % V == 0;
  for (int k = 0; k < count; ++k) {
    const RotaryTensor& t = p.t[k];
    vec = vec && aligned(t.x, 16) && aligned(t.y, 16) && t.sb % V == 0 && t.sh % V == 0 && t.sn % V == 0;
  }
  const int units = vec ? p.half / pairs + (p.dim - 2 * p.half) / V : p.dim - p.half;
  long long threads = 0, most = 0;
  int heads = 0;
  for (int k = 0; k < count; ++k) {
    const long long one = (long long)p.t[k].batch * p.t[k].n * units;
    threads += one * p.t[k].heads;
    most = one + 31 > most ? one + 31 : most;  // the copies begin at a warp's first lane
    heads = p.t[k].heads > heads ? p.t[k].heads : heads;
  }
  // heads per thread: as many as leave half a thread for every resident slot of the GPU (2048 per SM), so that a token's
  // sines serve many heads; with four heads' loads in flight that many threads keep HBM busy (B4 H16 S4096 D64 fp16:
  // 28.4 us with up to 8 heads taken one after the other, 20.8 us = 99 % of the measured HBM rate)
  long long per = threads / (kNumSMs * 1024ll);
  if (per > 8) per = 8;  // longer loops leave the last wave of blocks half empty (16384 tokens, 40 heads: 71 us with up to 32, 55 us)
  per = per < 1 ? 1 : per > heads ? heads : per;
  per = (heads + (heads + per - 1) / per - 1) / ((heads + per - 1) / per);  // even shares
  while ((heads + per - 1) / per > 65535) per *= 2;  // grid.y
  p.heads_per_thread = static_cast<int>(per);
  const long long gx = (most + kThreads - 1) / kThreads;
  const int gy = (heads + p.heads_per_thread - 1) / p.heads_per_thread;
  if (gx > 0x7fffffffll) return SPARTA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy), static_cast<unsigned>(count));
  if (!vec) rotary_pair_kernel<T><<<grid, kThreads, 0, st>>>(p, interleaved);
  else if (interleaved) rotary_vec_kernel<T, true><<<grid, kThreads, 0, st>>>(p);
  else rotary_vec_kernel<T, false><<<grid, kThreads, 0, st>>>(p);
  return launch_status();
}

}  // namespace
}  // namespace sparta

using namespace sparta;

extern "C" int sparta_rotary(const sparta_rotary_tensor* h_tensors, int count, const uint64_t* turns, int dim, int rotary_dim,
                             int interleaved, float magnitude, int backward, int positions_are_64, int dtype, void* stream) {
  if (!h_tensors || count < 1 || count > 2 || !turns || dim <= 0 || rotary_dim <= 0) return SPARTA_ERR_BAD_ARG;
  if (dtype < SPARTA_F32 || dtype > SPARTA_BF16) return SPARTA_ERR_BAD_ARG;
  if (rotary_dim > dim || rotary_dim % 2 || dim > 65536) return SPARTA_ERR_SHAPE;
  if (!aligned(turns, 8)) return SPARTA_ERR_ALIGN;
  const size_t esz = dtype == SPARTA_F32 ? 4 : 2;
  RotaryParams p = {};
  for (int k = 0; k < count; ++k) {
    const sparta_rotary_tensor& a = h_tensors[k];
    if (!a.x || !a.y || a.batch <= 0 || a.heads <= 0 || a.n <= 0) return SPARTA_ERR_BAD_ARG;
    if (!aligned(a.x, esz) || !aligned(a.y, esz) || !aligned(a.positions, positions_are_64 ? 8 : 4)) return SPARTA_ERR_ALIGN;
    if ((long long)a.batch * a.n > 0x7fffffffffll / dim || (long long)a.batch * a.n * a.heads > 0x7fffffffffffll / dim)
      return SPARTA_ERR_SHAPE;
    p.t[k].x = a.x; p.t[k].y = a.y; p.t[k].positions = a.positions;
    p.t[k].sb = a.stride_batch; p.t[k].sh = a.stride_head; p.t[k].sn = a.stride_token;
    p.t[k].batch = a.batch; p.t[k].heads = a.heads; p.t[k].n = a.n;
    p.t[k].pos_batched = a.positions_per_batch != 0;
  }
  p.turns = turns;
  p.magnitude = magnitude;
  p.sign = backward ? -1.f : 1.f;
  p.dim = dim; p.half = rotary_dim / 2; p.pos64 = positions_are_64 != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SPARTA_F32) return launch_rotary<float>(p, count, interleaved, st);
  if (dtype == SPARTA_F16) return launch_rotary<__half>(p, count, interleaved, st);
  return launch_rotary<__nv_bfloat16>(p, count, interleaved, st);
}

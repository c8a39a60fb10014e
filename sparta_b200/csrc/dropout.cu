// Dropout whose decisions come from a counter and are never stored:  y = keep(b, r, c) ? x * scale : 0  (philox.cuh).
// The backward pass is the same function of the output gradient, so one kernel serves both directions.
//
// Bound by HBM: one read and one write per element.  A Philox call (about 45 instructions for 8 decisions) and its
// compares must stay below the ~20 instructions per 16-bit element that the SMs can issue while HBM moves it, so a
// call is made once per group of eight columns:
//   * a thread owns a 16-byte aligned piece of memory (8 elements, or two pieces for fp32) per step, four steps,
//     all loads issued first;
//   * rows whose length is a multiple of 8: the piece is one group, one call;
//   * other rows: the piece straddles two groups.  Each lane makes the call of its piece's LAST group; the bits of
//     the group before it are what the lane below (or lane 31 of the step before) has just made, and only the first
//     step of a warp, and pieces that hold a row's end, call twice.
#include "philox.cuh"

namespace sparta {
namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 4;   // pieces per thread
constexpr int kPiece = 8;   // elements per piece = decisions per generator call

template <typename T>
struct alignas(16) Piece {
  T v[kPiece];
};
template <typename T, bool VEC>
__device__ __forceinline__ Piece<T> load_piece(const T* p) {
  Piece<T> r;
  if constexpr (VEC) {
    constexpr int n = sizeof(T) * kPiece / 16;
#pragma unroll
    for (int i = 0; i < n; ++i) reinterpret_cast<uint4*>(r.v)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  } else {
#pragma unroll
    for (int i = 0; i < kPiece; ++i) r.v[i] = p[i];
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, const Piece<T>& r) {
  constexpr int n = sizeof(T) * kPiece / 16;
#pragma unroll
  for (int i = 0; i < n; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(r.v)[i];
}
template <typename T>
__device__ __forceinline__ T drop(T v, bool keep, float scale) {
  return keep ? from_float<T>(to_float(v) * scale) : from_float<T>(0.f);  // a select: NaN and infinities are dropped too
}

// Dense [batch, H, W]; y 16-byte aligned, VEC: x too.  EVEN: W % 8 == 0.
template <typename T, bool EVEN, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_dense_kernel(const T* __restrict__ x, T* __restrict__ y, long long n, int H, int W, DropoutParams d) {
  const int lane = threadIdx.x & 31;
  const long long warp0 = ((long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * (32 * kSteps * kPiece);
  if (warp0 >= n) return;  // whole warps only: the shuffles below need every lane
  const PhiloxKey key = load_philox_key(d);
  const bool none = d.threshold >= kDropoutOne;
  const uint32_t cut = d.threshold << 16;
  // position of the warp's first element; a lane's position is that plus a 32-bit offset
  const long long row0 = warp0 / W;
  const uint32_t col0 = static_cast<uint32_t>(warp0 - row0 * W);
  const long long b0 = row0 / H;
  const uint32_t r0 = static_cast<uint32_t>(row0 - b0 * H);

  Piece<T> in[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const long long e = warp0 + (s * 32 + lane) * kPiece;
    if (e + kPiece <= n) in[s] = load_piece<T, VEC>(x + e);
    else if (e < n)
      for (int i = 0; i < kPiece; ++i) in[s].v[i] = e + i < n ? x[e + i] : from_float<T>(0.f);
  }
  uint32_t carry = 0;  // bits of lane 31's last group in the step before
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const long long e = warp0 + (s * 32 + lane) * kPiece;
    const uint32_t off = col0 + (s * 32 + lane) * kPiece;
    const uint32_t over = off / static_cast<uint32_t>(W);
    uint32_t c = off - over * W;  // column, row and batch element of the piece's first element
    uint32_t r = r0 + over, b = static_cast<uint32_t>(b0);
    if (r >= static_cast<uint32_t>(H)) { b += r / H; r %= H; }
    uint32_t bits;
    if constexpr (EVEN) {
      bits = philox_keep8(key, cut, c >> 3, r, b);
    } else {
      const uint32_t a = c & 7u;  // the piece begins at place a of group c / 8
      const bool ends = c + kPiece > static_cast<uint32_t>(W);  // the row ends inside the piece
      const uint32_t own = philox_keep8(key, cut, (c + kPiece - 1) >> 3, r, b);
      uint32_t before = __shfl_up_sync(0xffffffffu, own, 1);
      if (lane == 0) before = carry;
      carry = __shfl_sync(0xffffffffu, own, 31);
      // the lane below made the call of group c / 8 unless its piece reached over a row's end (then c < 8)
      if (a != 0 && ((s == 0 && lane == 0) || c < 8)) before = philox_keep8(key, cut, c >> 3, r, b);
      bits = a == 0 ? own : ((before | (own << 8)) >> a);
      if (ends) {  // element by element across the row's end (rows shorter than a piece wrap several times)
        bits = 0;
        uint32_t grp = 0xffffffffu, g8 = 0;
        for (int i = 0; i < kPiece; ++i) {
          if ((c >> 3) != grp) { grp = c >> 3; g8 = philox_keep8(key, cut, grp, r, b); }
          bits |= ((g8 >> (c & 7u)) & 1u) << i;
          if (++c == static_cast<uint32_t>(W)) {
            c = 0; grp = 0xffffffffu;
            if (++r == static_cast<uint32_t>(H)) { r = 0; ++b; }
          }
        }
      }
    }
    if (none) bits = 0;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) in[s].v[i] = drop(in[s].v[i], (bits >> i) & 1u, d.scale);
    if (e + kPiece <= n) store_piece(y + e, in[s]);
    else if (e < n)
      for (int i = 0; i < kPiece; ++i)
        if (e + i < n) y[e + i] = in[s].v[i];
  }
}

// Block values [batch, stride blocks of BH x BW], BCSR order: the positions come from the index entry.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_blocks_kernel(const T* __restrict__ x, T* __restrict__ y, const int32_t* __restrict__ idx,
                      const int32_t* __restrict__ nnz, int log_bh, int log_bw, long long stride, long long pieces, DropoutParams d) {
  const PhiloxKey key = load_philox_key(d);
  const bool none = d.threshold >= kDropoutOne;
  const uint32_t cut = d.threshold << 16;
  const uint32_t batch = blockIdx.y;
  const int log_pb = log_bh + log_bw - 3;  // pieces per block
  const long long base = (long long)batch * (stride << (log_bh + log_bw));
  const int kept = __ldg(nnz);
  Piece<T> in[kSteps];
  const long long first = (long long)blockIdx.x * (kThreads * kSteps) + threadIdx.x;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const long long v = first + s * kThreads;
    if (v < pieces) in[s] = load_piece<T, VEC>(x + base + v * kPiece);
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const long long v = first + s * kThreads;
    if (v >= pieces) continue;
    const long long blk = v >> log_pb;
    const uint32_t in_blk = static_cast<uint32_t>(v - (blk << log_pb)) << 3;
    uint32_t bits = 0;
    if (blk < kept && !none) {  // values behind the last block of a mask come out as zeros
      const uint32_t entry = static_cast<uint32_t>(__ldg(idx + blk));
      const uint32_t row = ((entry >> 16) << log_bh) + (in_blk >> log_bw);
      const uint32_t col = ((entry & 0xffffu) << log_bw) + (in_blk & ((1u << log_bw) - 1u));
      bits = philox_keep8(key, cut, col >> 3, row, batch);
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i) in[s].v[i] = drop(in[s].v[i], (bits >> i) & 1u, d.scale);
    store_piece(y + base + v * kPiece, in[s]);
  }
}

template <typename T>
int launch_dense(const void* x, void* y, long long n, int H, int W, const DropoutParams& d, cudaStream_t st) {
  const long long per_cta = (long long)kThreads * kSteps * kPiece;
  const long long ctas = (n + per_cta - 1) / per_cta;
  if (ctas > 0x7fffffffll) return SPARTA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(ctas));
  const T* px = static_cast<const T*>(x);
  T* py = static_cast<T*>(y);
  const bool vec = aligned(x, 16), even = W % 8 == 0;
  if (even && vec) dropout_dense_kernel<T, true, true><<<grid, kThreads, 0, st>>>(px, py, n, H, W, d);
  else if (even) dropout_dense_kernel<T, true, false><<<grid, kThreads, 0, st>>>(px, py, n, H, W, d);
  else if (vec) dropout_dense_kernel<T, false, true><<<grid, kThreads, 0, st>>>(px, py, n, H, W, d);
  else dropout_dense_kernel<T, false, false><<<grid, kThreads, 0, st>>>(px, py, n, H, W, d);
  return launch_status();
}

template <typename T>
int launch_blocks(const void* x, void* y, const int32_t* idx, const int32_t* nnz, int batch, int BH, int BW, long long stride,
                  const DropoutParams& d, cudaStream_t st) {
  int lh = 0, lw = 0;
  while ((1 << lh) < BH) ++lh;
  while ((1 << lw) < BW) ++lw;
  const long long pieces = (stride << (lh + lw)) / kPiece;
  const long long ctas = (pieces + kThreads * kSteps - 1) / (kThreads * kSteps);
  if (ctas > 0x7fffffffll) return SPARTA_ERR_SHAPE;
  const T* px = static_cast<const T*>(x);
  T* py = static_cast<T*>(y);
  const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(batch));
  if (aligned(x, 16)) dropout_blocks_kernel<T, true><<<grid, kThreads, 0, st>>>(px, py, idx, nnz, lh, lw, stride, pieces, d);
  else dropout_blocks_kernel<T, false><<<grid, kThreads, 0, st>>>(px, py, idx, nnz, lh, lw, stride, pieces, d);
  return launch_status();
}

}  // namespace
}  // namespace sparta

using namespace sparta;

extern "C" int sparta_dropout(const void* x, void* y, int batch, int H, int W, double p, const int64_t* rng, uint64_t seed,
                              uint64_t call, int dtype, void* stream) {
  if (!x || !y || batch <= 0 || H <= 0 || W <= 0) return SPARTA_ERR_BAD_ARG;
  if (dtype < SPARTA_F32 || dtype > SPARTA_BF16) return SPARTA_ERR_BAD_ARG;
  if (W > (1 << 30) || (long long)batch * H > 0x7fffffffffffll / W) return SPARTA_ERR_SHAPE;
  if (!aligned(y, 16) || !aligned(x, dtype == SPARTA_F32 ? 4 : 2) || (rng && !aligned(rng, 8))) return SPARTA_ERR_ALIGN;
  DropoutParams d;
  if (!make_dropout(&d, p, rng, seed, call)) return SPARTA_ERR_BAD_ARG;
  const long long n = (long long)batch * H * W;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SPARTA_F32) return launch_dense<float>(x, y, n, H, W, d, st);
  if (dtype == SPARTA_F16) return launch_dense<__half>(x, y, n, H, W, d, st);
  return launch_dense<__nv_bfloat16>(x, y, n, H, W, d, st);
}

extern "C" int sparta_dropout_blocks(const void* x, void* y, const int32_t* bcsr_idx, const int32_t* nnz, int batch, int BH,
                                     int BW, int64_t val_stride_blocks, double p, const int64_t* rng, uint64_t seed,
                                     uint64_t call, int dtype, void* stream) {
  if (!x || !y || !bcsr_idx || !nnz || batch <= 0 || val_stride_blocks <= 0) return SPARTA_ERR_BAD_ARG;
  if (dtype < SPARTA_F32 || dtype > SPARTA_BF16) return SPARTA_ERR_BAD_ARG;
  if (!valid_bcs_block(BH) || !valid_bcs_block(BW) || BW < 8 || batch > 65535 || val_stride_blocks > (1ll << 32))
    return SPARTA_ERR_SHAPE;
  if (!aligned(y, 16) || !aligned(x, dtype == SPARTA_F32 ? 4 : 2) || (rng && !aligned(rng, 8))) return SPARTA_ERR_ALIGN;
  DropoutParams d;
  if (!make_dropout(&d, p, rng, seed, call)) return SPARTA_ERR_BAD_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SPARTA_F32) return launch_blocks<float>(x, y, bcsr_idx, nnz, batch, BH, BW, val_stride_blocks, d, st);
  if (dtype == SPARTA_F16) return launch_blocks<__half>(x, y, bcsr_idx, nnz, batch, BH, BW, val_stride_blocks, d, st);
  return launch_blocks<__nv_bfloat16>(x, y, bcsr_idx, nnz, batch, BH, BW, val_stride_blocks, d, st);
}

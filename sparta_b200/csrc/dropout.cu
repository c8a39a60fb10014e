// Dropout whose decisions come from a counter and are never stored:  y = keep(b, r, c) ? x * scale : 0  (philox.cuh).
// The backward pass is the same function of the output gradient, so one kernel serves both directions.
//
// Bound by HBM: one read and one write per element, which leaves the SMs about 20 instructions per 16-bit element.  A
// thread owns 16 bytes of 16-bit elements (32 of fp32), one call of the generator, at the same place of several rows:
// the column's share of the generator is made once for all of them, the row's share once per row, and the decisions
// are applied to packed pairs (134 M bf16 elements: 82 us, 100 % of the measured HBM rate, 13 instructions per element; with a
// full call and a compare and a select per element 119 us and 23).
// Rows whose length is no multiple of 8 begin anywhere in a 16-byte piece of memory.  Pieces stay aligned, so that a
// piece holds the end of one group of eight columns and the beginning of the next: each lane makes the decisions of the
// group that begins in its piece and takes those of the group before from the lane below (the lowest lane of a segment
// only makes them).  Pieces at either end of a row are stored element by element, in a loop of their own that has as many
// loads in flight (one after the other: 54 us instead of 50).
#include <type_traits>

#include "philox.cuh"

namespace sparta {
namespace {

constexpr int kThreads = 128;  // blocks of 256 wait longer for their last warp (58 M elements in rows of 4093: 49 us against 47.5)
template <typename T>
constexpr int kBatch = 8 / sizeof(T);  // rows whose loads are in flight together: 64 bytes per thread
constexpr int kMaxRows = 8; // rows per thread, or 1 where rows are few
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
// Scale a pair and keep what `mask` covers.  Masked bits, not a product with zero: NaN and infinities are dropped too.
// The product is taken in 32 bits and rounded once.
template <typename T>
__device__ __forceinline__ void drop_pair(Piece<T>& p, int i, uint32_t mask, float scale) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t lo = __byte_perm(mask, 0, 0x1010), hi = __byte_perm(mask, 0, 0x3232);
    p.v[2 * i] = __uint_as_float(__float_as_uint(p.v[2 * i] * scale) & lo);
    p.v[2 * i + 1] = __uint_as_float(__float_as_uint(p.v[2 * i + 1] * scale) & hi);
  } else {
    const T a = from_float<T>(to_float(p.v[2 * i]) * scale), b = from_float<T>(to_float(p.v[2 * i + 1]) * scale);
    T two[2] = {a, b};
    reinterpret_cast<uint32_t*>(p.v)[i] = *reinterpret_cast<const uint32_t*>(two) & mask;
  }
}

// The masks of a piece's four pairs.  Rows that are no multiple of 8 long begin `a` elements into a piece: the piece then
// holds the last `a` columns of the group before the lane's own (whose decisions the lane below made) and the first
// 8 - a of its own.  Every lane of the warp calls it.
template <bool EVEN>
__device__ __forceinline__ void piece_masks(const PhiloxKey& key, const PhiloxRow& row, const PhiloxCol& col, uint32_t t2, int a, int seg,
                                            uint32_t (&mask)[4]) {
  uint32_t w[4];
  philox8(key, row, col, w);
  if constexpr (EVEN) {
#pragma unroll
    for (int i = 0; i < 4; ++i) mask[i] = spread2(not_below2(w[i], t2));
  } else {
    // one byte per column, 0 or 255
    const uint32_t own0 = spread4(not_below2(w[0], t2), not_below2(w[1], t2)), own1 = spread4(not_below2(w[2], t2), not_below2(w[3], t2));
    const uint32_t before0 = __shfl_up_sync(0xffffffffu, own0, 1, seg), before1 = __shfl_up_sync(0xffffffffu, own1, 1, seg);
    // bytes 8 - a .. 15 - a of before0, before1, own0, own1: shifted left by a bytes, 4 of them as whole words
    const bool far = a >= 4;
    const uint32_t n0 = far ? before0 : before1, n1 = far ? before1 : own0, n2 = far ? own0 : own1;
    const uint32_t lo = __funnelshift_l(n0, n1, 8 * a), hi = __funnelshift_l(n1, n2, 8 * a);  // the shift is taken mod 32
    mask[0] = __byte_perm(lo, 0, 0x1100); mask[1] = __byte_perm(lo, 0, 0x3322);
    mask[2] = __byte_perm(hi, 0, 0x1100); mask[3] = __byte_perm(hi, 0, 0x3322);
  }
}

// Dense [rows, W], rows = batch * H; y 16-byte aligned, VEC: x too.  EVEN: W % 8 == 0.  A warp is 32 >> log_seg segments
// of 1 << log_seg lanes, each on a row of its own; rows longer than a segment reaches are cut into `chunks`.
template <typename T, bool EVEN, bool VEC>
__global__ void __launch_bounds__(kThreads, 8)  // 64 registers: the loads of many warps hide each other
dropout_dense_kernel(const T* __restrict__ x, T* __restrict__ y, long long rows, int H, int W, int log_seg, int chunks,
                     int per_thread, DropoutParams d) {
  const PhiloxKey key = load_uniform_philox_key(d);
  const uint32_t t2 = threshold2(d);
  const int lane = threadIdx.x & 31, seg = 1 << log_seg, at = lane & (seg - 1), per_warp = 32 >> log_seg;
  const long long warp = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const long long group = warp / chunks;
  const int chunk = static_cast<int>(warp - group * chunks);
  const long long row0 = group * per_thread * per_warp;
  if (row0 >= rows) return;  // whole warps only: the shuffles need every lane
  // the group of columns whose decisions this lane makes, which begins in (or, EVEN, is) its piece of every row
  const int m0 = EVEN ? chunk * seg : chunk * (seg - 1) - 1, m = m0 + at;
  const bool makes_only = !EVEN && at == 0;
  long long row = row0 + (lane >> log_seg);
  uint32_t b = static_cast<uint32_t>(row / H), r = static_cast<uint32_t>(row - (long long)b * H);
  PhiloxCol col = philox_col(key, m, b);
  auto next_row = [&] {
    r += per_warp;
    if (r >= static_cast<uint32_t>(H)) {
      b += r / H;
      r %= H;
      col = philox_col(key, m, b);
    }
  };
  const bool inside = (EVEN || m0 >= 0) && m0 + seg <= W / kPiece;  // no piece of the warp holds an end of a row
  if (d.threshold < kDropoutOne && (inside || (!EVEN && W >= kPiece)) && per_thread >= kBatch<T> && W <= (1 << 24) &&
      (row0 + per_thread * per_warp < rows || (inside && row0 + per_thread * per_warp == rows))) {
    // ---- all rows are there, and pieces may be read whole: loads of four rows in flight ----
    // rows that begin anywhere: 32-bit offsets from the first one (58 M fp16 elements in rows of 4093: 61 -> 55 us when it was measured); the
    // other rows measured faster with 64-bit ones (134 M bf16 elements: 85 us against 93)
    using Offset = typename std::conditional<EVEN, long long, uint32_t>::type;
    const Offset step = static_cast<Offset>(per_warp) * static_cast<Offset>(W);
    const long long first = row * W;
    Offset start0 = EVEN ? 0 : static_cast<Offset>(first & 7);
    const long long base = ((first >> 3) + m) * kPiece;
    const T* px = x + base;
    T* py = y + base;
    auto run = [&](auto ends) {
      Offset start = start0;
#pragma unroll 1
      for (int k0 = 0; k0 < per_thread; k0 += kBatch<T>) {
        Piece<T> in[kBatch<T>];
#pragma unroll
        for (int k = 0; k < kBatch<T>; ++k) {
          const Offset s = start + k * step;
          const bool read = !makes_only && (!ends || kPiece * m - static_cast<int>(s & 7) < W);
          if (read) in[k] = load_piece<T, VEC>(px + (EVEN ? s : s / kPiece * kPiece));
        }
#pragma unroll
        for (int k = 0; k < kBatch<T>; ++k) {
          uint32_t mask[4];
          piece_masks<EVEN>(key, philox_row(key, r, b), col, t2, static_cast<int>(start) & 7, seg, mask);
#pragma unroll
          for (int i = 0; i < 4; ++i) drop_pair(in[k], i, mask[i], d.scale);
          T* out = py + (EVEN ? start : start / kPiece * kPiece);
          const int c0 = kPiece * m - static_cast<int>(start & 7);  // column of the piece's first element
          if (!ends || (c0 >= 0 && c0 + kPiece <= W)) {
            if (!makes_only) store_piece(out, in[k]);
          } else if (!makes_only) {
#pragma unroll
            for (int i = 0; i < kPiece; ++i)
              if (c0 + i >= 0 && c0 + i < W) out[i] = in[k].v[i];
          }
          start += step;
          next_row();
        }
      }
    };
    if (EVEN || inside) run(std::false_type{});
    else run(std::true_type{});
    return;
  }
  // ---- the last rows, few rows, and p = 1: piece by piece, whole or in part ----
#pragma unroll 1
  for (int k = 0; k < per_thread; ++k, row += per_warp) {
    const long long start = row * W;
    const int a = EVEN ? 0 : static_cast<int>(start & 7), c0 = kPiece * m - a;  // column of the piece's first element
    uint32_t mask[4];
    piece_masks<EVEN>(key, philox_row(key, r, b), col, t2, a, seg, mask);
    if (d.threshold >= kDropoutOne) mask[0] = mask[1] = mask[2] = mask[3] = 0;
    const int lo = max(0, -c0), hi = makes_only || row >= rows ? 0 : min(kPiece, W - c0);
    if (lo < hi) {
      Piece<T> in;
      const long long e0 = start + c0;
      if (e0 >= 0 && e0 + kPiece <= rows * W) {  // a piece may be read across a row's ends, but not across the tensor's
        in = load_piece<T, VEC>(x + e0);
      } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) in.v[i] = i >= lo && i < hi ? x[e0 + i] : from_float<T>(0.f);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) drop_pair(in, i, mask[i], d.scale);
      if (hi - lo == kPiece) {
        store_piece(y + e0, in);
      } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i)
          if (i >= lo && i < hi) y[e0 + i] = in.v[i];
      }
    }
    next_row();
  }
}

// Block values [batch, stride blocks of BH x BW], BCSR order: the positions come from the index entry.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads)
dropout_blocks_kernel(const T* __restrict__ x, T* __restrict__ y, const int32_t* __restrict__ idx,
                      const int32_t* __restrict__ nnz, int log_bh, int log_bw, long long stride, long long pieces, DropoutParams d) {
  const PhiloxKey key = load_uniform_philox_key(d);
  const uint32_t t2 = threshold2(d);
  const bool none = d.threshold >= kDropoutOne;
  const uint32_t batch = blockIdx.y;
  const int log_pb = log_bh + log_bw - 3;  // pieces per block
  const long long base = (long long)batch * (stride << (log_bh + log_bw));
  const int kept = __ldg(nnz);
  Piece<T> in[kBatch<T>];
  const long long first = (long long)blockIdx.x * (kThreads * kBatch<T>) + threadIdx.x;
#pragma unroll
  for (int s = 0; s < kBatch<T>; ++s) {
    const long long v = first + s * kThreads;
    if (v < pieces) in[s] = load_piece<T, VEC>(x + base + v * kPiece);
  }
#pragma unroll
  for (int s = 0; s < kBatch<T>; ++s) {
    const long long v = first + s * kThreads;
    if (v >= pieces) continue;
    const long long blk = v >> log_pb;
    const uint32_t in_blk = static_cast<uint32_t>(v - (blk << log_pb)) << 3;
    uint32_t w[4] = {0, 0, 0, 0};
    const bool there = blk < kept && !none;  // values behind the last block of a mask come out as zeros
    if (there) {
      const uint32_t entry = static_cast<uint32_t>(__ldg(idx + blk));
      const uint32_t row = ((entry >> 16) << log_bh) + (in_blk >> log_bw);
      const uint32_t col = ((entry & 0xffffu) << log_bw) + (in_blk & ((1u << log_bw) - 1u));
      philox8(key, philox_row(key, row, batch), philox_col(key, col >> 3, batch), w);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) drop_pair(in[s], i, there ? spread2(not_below2(w[i], t2)) : 0u, d.scale);
    store_piece(y + base + v * kPiece, in[s]);
  }
}

template <typename T>
int launch_dense(const void* x, void* y, long long rows, int H, int W, const DropoutParams& d, cudaStream_t st) {
  const bool even = W % kPiece == 0;
  const int pieces = even ? W / kPiece : (W + 2 * kPiece - 2) / kPiece;  // of a row, wherever in a piece it begins
  int log_seg = even ? 0 : 1;
  while (log_seg < 5 && (1 << log_seg) - (even ? 0 : 1) < pieces) ++log_seg;
  const int reach = (1 << log_seg) - (even ? 0 : 1), chunks = (pieces + reach - 1) / reach;
  // several rows per thread share the column's part of the generator and have their loads in flight together; with fewer
  // than 16 warps per SM it is the latency of one row that counts
  const int per_thread = (rows >> (5 - log_seg)) * chunks / kMaxRows >= 16 * kNumSMs ? kMaxRows : 1;
  const long long per_group = (long long)per_thread * (32 >> log_seg);
  const long long warps = (rows + per_group - 1) / per_group * chunks;
  const long long ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (ctas > 0x7fffffffll) return SPARTA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(ctas));
  const T* px = static_cast<const T*>(x);
  T* py = static_cast<T*>(y);
  const bool vec = aligned(x, 16);
  if (even && vec) dropout_dense_kernel<T, true, true><<<grid, kThreads, 0, st>>>(px, py, rows, H, W, log_seg, chunks, per_thread, d);
  else if (even) dropout_dense_kernel<T, true, false><<<grid, kThreads, 0, st>>>(px, py, rows, H, W, log_seg, chunks, per_thread, d);
  else if (vec) dropout_dense_kernel<T, false, true><<<grid, kThreads, 0, st>>>(px, py, rows, H, W, log_seg, chunks, per_thread, d);
  else dropout_dense_kernel<T, false, false><<<grid, kThreads, 0, st>>>(px, py, rows, H, W, log_seg, chunks, per_thread, d);
  return launch_status();
}

template <typename T>
int launch_blocks(const void* x, void* y, const int32_t* idx, const int32_t* nnz, int batch, int BH, int BW, long long stride,
                  const DropoutParams& d, cudaStream_t st) {
  int lh = 0, lw = 0;
  while ((1 << lh) < BH) ++lh;
  while ((1 << lw) < BW) ++lw;
  const long long pieces = (stride << (lh + lw)) / kPiece;
  const long long ctas = (pieces + kThreads * kBatch<T> - 1) / (kThreads * kBatch<T>);
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
  const long long rows = (long long)batch * H;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SPARTA_F32) return launch_dense<float>(x, y, rows, H, W, d, st);
  if (dtype == SPARTA_F16) return launch_dense<__half>(x, y, rows, H, W, d, st);
  return launch_dense<__nv_bfloat16>(x, y, rows, H, W, d, st);
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

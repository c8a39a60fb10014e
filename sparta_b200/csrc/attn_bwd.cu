// Backward pass of the fused block-sparse attention (fp16 / bf16, head dim 64 or 128, 64 x 64 mask blocks).  The
// probabilities are recomputed from Q, K and the forward pass's row log-sum-exp; nothing of size Nt x Ns is stored
// but, with dropout and for the time of the call, a bit per kept score.
//
//   S = Q K^T    P = exp(scale S - lse)            on kept elements, 0 elsewhere
//   P' = P keep up                                  (dropout: keep in {0, 1}, up = 1 / (1 - p))
//   dV = P'^T dO     dP = (dO V^T) keep up     delta_i = sum_d dO_id O_id = sum_j P_ij dP_ij
//   dS = P (dP - delta)      dQ = scale dS K       dK = scale dS^T Q        (K, V shared by heads: summed over them)
//
// Two passes over the kept blocks, each with its sums in tensor memory from the first block to the last, so that every
// gradient is written once, in a fixed order of additions: one pass owns 128 query rows and walks the kept key blocks
// (dQ), the other owns 128 key rows and walks the query blocks of every head that shares them (dK, dV).  That is seven products per kept block instead of the five of a single pass,
// which would have to add 128 x D 32-bit partial sums of dQ per block to global memory (in an order that changes from
// run to run): 32 to 64 KB of atomic traffic per 128 x 128 scores, more than L2 takes at the rate of the products.
//
// Both passes are one kernel.  A CTA holds two resident tiles A1, A2 of 128 rows and streams pairs of 64-row blocks
// B1, B2 through shared memory; the tile's rows are the lanes of tensor memory:
//                      A1   A2   B1   B2
//   dQ pass            Q    dO   K    V        S = A1 B1^T   dP = A2 B2^T   acc1 += dS B1
//   dK, dV pass        K    V    Q    dO       S^T, dP^T likewise, acc1 = dK += dS^T B1, acc2 = dV += P'^T B2
// P' and dS go back into tensor memory, over the columns that their own thread has just read, as the A operand of the
// last products; B1 and B2 serve twice, K-major for S and dP, MN-major (the head dim contiguous) for the sums.
//
// Schedule.  A step is 128 columns of scores (two blocks) for head dim 128, 64 (one) for head dim 64, for 128 rows, in
// two phases: P from S, then dS from P and dP; one warp for every 32 rows x 32 columns.  Another warp issues every MMA:
// when P of step j is in place, P'^T dO of j and then S of a later step; when dS of j is in place, dS B1 of j and then
// dP of the next step.  MMAs of one thread execute in order, so S of a later step may take the columns that P' is being
// read from, and the tensor pipe works on one half of a step while the threads work on the other.
//   Head dim 128: tensor memory is full with S, dP (128 columns each) and the sums; one CTA of 18 warps per SM.  With
//   steps of one block an MMA reads 6 KB of shared memory for 32 cycles of math, and there are twice as many to issue at
//   one per 60 to 80 cycles: 1.4 times the time (H16 S8192 on 4 key heads, both passes: 1012 us against 705).
//   Head dim 64: half the tensor memory per CTA (S twice in the dQ pass), so that two CTAs of 10 warps share an SM and
//   one computes while the other waits or starts up: steps of two blocks with one CTA measured 595 us against 490 us
//   (B4 H16 S4096, both passes).
//   The warp number and what MMAs are addressed with go through a shuffle: the compiler then knows them to be uniform
//   and keeps descriptors in uniform registers (dK, dV of B4 H16 S4096 D64 335 -> 305 us before the other steps).
// What bounds it now: the chain of a step -- scores, exponentials, hand-over, products -- of the tiles in flight: the
// tensor pipe is occupied 60 % of the time, issue slots 44 % (D64) and 28 % (D128).  420 us for both passes of B4 H16
// S4096 D64 with 31 % of the blocks kept (510 TFLOP/s on five products), 420 us for H16 S8192 D128 on 4 key heads with
// 19 % kept (607 TFLOP/s).
//
// The dK, dV pass needs the statistics of its columns, the query rows.  Read by threads that each own a row they were 16
// vector loads of shared memory per warp and step, all lanes at one address, and took 45 % of its bandwidth; that pass
// therefore reads and writes tensor memory in the fragment layout, where a thread has four rows and eight columns.
//
// Masks and dropout are words of 32 decisions per row of the score matrix (query): in the dQ pass each thread's own, in
// the dK, dV pass each lane has one and the threads fetch those of their eight columns from the lanes that have them.
// Dropout decisions are made once, by the first kernel, for both passes, if the workspace has room (B4 H16 S4096 D64,
// p = 0.1: 716 us with the generator in the steps of both; 610 us now, of which 94 the first kernel, 515 the passes).
// The forward pass it belongs to: SparseAttention.forward (sparta/specializer/operators/sparse_attention.py:76-80),
// whose gradients the reference takes through its three operators.
#include <type_traits>

#include "attn.cuh"
#include "bsmm.cuh"
#include "tc_common.cuh"

namespace sparta {
namespace {

using namespace tc;

constexpr int kBlk = 64;        // mask block edge
constexpr int kTileM = 128;     // rows of A1, A2 per CTA (two blocks)
constexpr int kMaxBlocks = 1024;  // blocks along the streamed side (65536 rows)

struct BwdParams {
  const uint8_t* mask;      // [Nt, Ns] or null
  const uint8_t* present;   // [Nt / 64, present_pitch]: block kept (made by the first kernel)
  const float* neg_lse;     // [heads, Nt]: -lse * log2(e), -inf for a row without any score
  const float* neg_delta;   // [heads, Nt]
  int Nt, Ns, heads, kv_heads, group;
  int present_pitch;
  float scale, scale_log2;
  int32_t* status;
  DropoutParams drop;
  const int32_t* position;  // [Nt / 64, present_pitch]: place of a kept block in the index (dropout only)
  const uint32_t* bits;     // [heads, bits_blocks, 2, 64]: decisions by place in the index, made by the first
  int bits_blocks;          // kernel; 32 columns of a query row per word
  const int32_t* blocks;    // kept blocks: where they are more than bits_blocks, decisions are made in the steps
};
constexpr int kBitWords = kBlk * kBlk / 32;  // of a block

struct PassParams {         // of one of the two passes
  void* out1;               // dQ, or dK
  void* out2;               // dV
  int by_head;              // launch order: tiles of a head together
  int split;                // CTAs per tile at most
  int split_steps;          // steps that one of them should take
  float* partial;           // [heads, tiles, split, columns of the sums, 128], where a tile is split
  uint32_t* tickets;        // [heads, tiles], zero
};

template <bool DKV, int D>
struct BwdCfg {
  static constexpr int kBlocks = D == 64 ? 1 : 2;      // blocks per step
  static constexpr int kCols = kBlocks * kBlk;         // columns of a step
  static constexpr int kCtasPerSM = D == 64 ? 2 : 1;
  static constexpr int kScoreWarps = 4 * (kCols / 32); // one per tensor-memory lane quadrant for each 32 columns of a step
  static constexpr int kWarpLoad = kScoreWarps, kWarpMma = kScoreWarps + 1;
  static constexpr int kThreads = 32 * (kScoreWarps + 2);
  static constexpr int kSBuf = D == 64 && !DKV ? 2 : 1;      // score buffers in tensor memory
  static constexpr int kStages = D == 64 ? 4 : 2;      // step j + kSBuf is read while j still is
  static constexpr int kChunks = D / 64;               // 64-element (128-byte) chunks of the head dim
  static constexpr int kABytes = kTileM * D * 2;
  static constexpr int kBBytes = kCols * D * 2;
  static constexpr int kStatFloats = DKV ? 2 * kCols : 0;  // neg_lse and neg_delta of the streamed query rows
  static constexpr uint32_t kDpCol = kSBuf * kCols;
  static constexpr uint32_t kAcc1 = kDpCol + kCols, kAcc2 = kAcc1 + D;
  static constexpr uint32_t kTmemCols = 512 / kCtasPerSM;
  static_assert(kAcc2 + (DKV ? D : 0) <= kTmemCols, "tensor memory budget");
  static constexpr int smem_bytes(bool drop) {
    return 2 * kABytes + kStages * (2 * kBBytes + kStatFloats * 4) + (drop ? 2 * kMaxBlocks * 4 : 0) + kMaxBlocks * 3 + 512 + 1024;
  }
};

// two 32-bit operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)), "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}

// Decisions about two columns (8 n + 2 (lane % 4) and the next) and the thread's four rows (lane / 4 + 8 r), at the top
// of byte r; lane c of the warp holds the word of column c, bit = row.  A byte permutation spreads the tops into masks.
struct ColumnMasks {
  uint32_t c0, c1;
};
__device__ __forceinline__ ColumnMasks column_masks(uint32_t word, int n, int lane) {
  const int c = 8 * n + 2 * (lane & 3), up = 7 - (lane >> 2);
  return {__shfl_sync(0xffffffffu, word, c) << up, __shfl_sync(0xffffffffu, word, c + 1) << up};
}
__device__ __forceinline__ uint32_t permute_signs(uint32_t a, uint32_t b, uint32_t selector) {  // selector nibbles 8 + byte: its sign
  uint32_t m;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(m) : "r"(a), "r"(b), "r"(selector));
  return m;
}
__device__ __forceinline__ uint32_t packed_mask(const ColumnMasks& m, int r) {  // of a pair of 16-bit values in row r
  return permute_signs(m.c0, m.c1, 0xcc88u + r * 0x1111u);
}
__device__ __forceinline__ float2 mask_pair(float2 v, const ColumnMasks& m, int r) {
  return make_float2(__uint_as_float(__float_as_uint(v.x) & permute_signs(m.c0, 0, 0x8888u + r * 0x1111u)),
                     __uint_as_float(__float_as_uint(v.y) & permute_signs(m.c1, 0, 0x8888u + r * 0x1111u)));
}

// Dropout decisions of a 32 x 32 region for a thread of the fragment layout, from the lanes' words of a column each
// (philox_bits32, its columns the region's rows): column pair n in byte n, rows lane / 4 + 8 r at bits 7 - 2 r of the first
// column and 6 - 2 r of the second.  A shift by 2 r thus has row r's decisions at the tops of the bytes.
__device__ __forceinline__ uint32_t fragment_bits(uint32_t word, int lane) {
  const int g = lane >> 2, turn = 8 * (g & 3) - (g >> 2);  // brings row 8 r + g to bit 7 - 2 r
  uint32_t pair[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const uint32_t c0 = __shfl_sync(0xffffffffu, word, 8 * n + 2 * (lane & 3)), c1 = __shfl_sync(0xffffffffu, word, 8 * n + 2 * (lane & 3) + 1);
    pair[n] = (__funnelshift_r(c0, c0, turn) & 0xaau) | (__funnelshift_r(c1, c1, turn + 1) & 0x55u);
  }
  return __byte_perm(__byte_perm(pair[0], pair[1], 0x0040), __byte_perm(pair[2], pair[3], 0x0040), 0x5410);
}

__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// The dropout decisions of all blocks of the index and all heads, if there is room.  A warp makes a block's, two rows
// per lane, so that the columns' share of the generator serves both.  Bound by the integer instructions, about 45 per call
// of the generator: 334 M decisions in 83 us.
__device__ void make_dropout_bits(const DropoutParams& drop, const int32_t* __restrict__ idx, int blocks, int bits_blocks, int heads,
                                  uint32_t* __restrict__ bits, uint32_t warp, uint32_t warps) {
  const int lane = threadIdx.x & 31;
  const PhiloxKey key = load_uniform_philox_key(drop);
  const uint32_t t2 = threshold2(drop);
  if (blocks > bits_blocks) return;  // they will be made in the steps
  const uint32_t n = max(0, blocks);
  for (uint64_t item = warp; item < static_cast<uint64_t>(n) * heads; item += warps) {
    const uint32_t head = static_cast<uint32_t>(item / n), e = static_cast<uint32_t>(item - static_cast<uint64_t>(head) * n);
    const uint32_t entry = static_cast<uint32_t>(__ldg(idx + e));
    const uint32_t row = (entry >> 16) * kBlk + lane, word = (entry & 0xffffu) * (kBlk / 32);
    uint32_t* dst = bits + (static_cast<uint64_t>(head) * bits_blocks + e) * kBitWords + lane;
    const PhiloxRow r0 = philox_row(key, row, head), r1 = philox_row(key, row + 32, head);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      dst[w * kBlk] = philox_bits32(key, r0, t2, word + w, head);
      dst[w * kBlk + 32] = philox_bits32(key, r1, t2, word + w, head);
    }
  }
}

// The negated delta and log-sum-exp of every query row; the blocks kept, as bytes, for the pass that walks columns; their
// places in the index and their dropout decisions.  The latter are arithmetic, for which the first `bits_ctas` CTAs are
// there; the rest is bound by the read of O and dO.  A row is D / 8 lanes of 16 bytes; four rows' loads are in flight per
// thread.
constexpr int kPrepRows = 4;
struct PrepBits {
  DropoutParams drop;
  int32_t* position;
  uint32_t* bits;
  int blocks, heads, ctas;
};
template <typename T, int D, bool DROP>
__global__ void __launch_bounds__(256)
attn_bwd_prep_kernel(const T* __restrict__ O, const T* __restrict__ dO, const float* __restrict__ lse, float* __restrict__ neg_lse,
                     float* __restrict__ neg_delta, uint8_t* __restrict__ present, const int32_t* __restrict__ row_ptr,
                     const int32_t* __restrict__ idx, long long rows, int nbr, int nbc, int pitch,
                     uint32_t* __restrict__ tickets, long long n_tickets, const __grid_constant__ PrepBits make) {
  int block = blockIdx.x, grid = gridDim.x;
  if constexpr (DROP) {
    if (block < make.ctas) {
      make_dropout_bits(make.drop, idx, __ldg(row_ptr + nbr), make.blocks, make.heads, make.bits, block * 8 + (threadIdx.x >> 5), make.ctas * 8);
      return;
    }
    block -= make.ctas;
    grid -= make.ctas;
  }
  constexpr int kLanes = D / 8, kStep = 256 / kLanes;
  const int lane = threadIdx.x % kLanes;
  const long long row0 = (long long)block * (kPrepRows * kStep) + threadIdx.x / kLanes;
  uint4 a[kPrepRows], b[kPrepRows];
#pragma unroll
  for (int k = 0; k < kPrepRows; ++k) {
    const long long row = row0 + k * kStep;
    a[k] = b[k] = make_uint4(0, 0, 0, 0);
    if (row < rows) {
      a[k] = __ldg(reinterpret_cast<const uint4*>(O + row * D) + lane);
      b[k] = __ldg(reinterpret_cast<const uint4*>(dO + row * D) + lane);
    }
  }
#pragma unroll
  for (int k = 0; k < kPrepRows; ++k) {
    const long long row = row0 + k * kStep;
    const T* x = reinterpret_cast<const T*>(&a[k]);
    const T* y = reinterpret_cast<const T*>(&b[k]);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(to_float(x[i]), to_float(y[i]), sum);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (row < rows && lane == 0) {
      neg_delta[row] = -sum;
      // (a NaN stays one, so that it reaches the gradients)
      neg_lse[row] = lse[row] == -INFINITY ? -INFINITY : lse[row] * -1.4426950408889634f;
    }
  }
  for (long long i = (long long)block * 256 + threadIdx.x; i < n_tickets; i += (long long)grid * 256) tickets[i] = 0;
  __shared__ uint8_t kept[kMaxBlocks];
  for (int r = block; r < nbr; r += grid) {  // block rows of the mask
    __syncthreads();
    for (int c = threadIdx.x; c < pitch; c += 256) kept[c] = 0;
    __syncthreads();
    for (int e = row_ptr[r] + threadIdx.x; e < row_ptr[r + 1]; e += 256) {
      const int c = __ldg(idx + e) & 0xffff;
      if (c < nbc) {  // index arrays come from the caller: never index shared memory with them unchecked
        kept[c] = 1;
        if constexpr (DROP) make.position[(long long)r * pitch + c] = max(0, min(e, make.blocks - 1));  // (nor the workspace)
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < pitch; c += 256) present[(long long)r * pitch + c] = kept[c];
  }
}

// SPLIT: several CTAs may share a tile.  A variant of its own, because the other one keeps its registers for the steps
// (B4 H16 S4096 D64, which does not split: 509 us with the code for it, 483 us without).
// READY: the first kernel has made every block's dropout decisions (otherwise they are made in the steps).
template <bool DKV, int D, int FMT, bool MASK, bool DROP, bool READY, bool SPLIT>
__device__ __forceinline__ void bwd_pass(const CUtensorMap& tm_a1, const CUtensorMap& tm_a2, const CUtensorMap& tm_b1,
                                         const CUtensorMap& tm_b2, const BwdParams& p, const PassParams& pass, int block) {
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  using C = BwdCfg<DKV, D>;
  constexpr int kSBuf = C::kSBuf, kStages = C::kStages, kChunks = C::kChunks, kThreads = C::kThreads;
  constexpr int kScoreWarps = C::kScoreWarps, kWarpLoad = C::kWarpLoad, kWarpMma = C::kWarpMma;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a1_s = smem;
  uint8_t* a2_s = a1_s + C::kABytes;
  uint8_t* b1_s = a2_s + C::kABytes;                        // [kStages]
  uint8_t* b2_s = b1_s + kStages * C::kBBytes;              // [kStages]
  float* stat_s = reinterpret_cast<float*>(b2_s + kStages * C::kBBytes);  // [kStages][neg_lse, neg_delta of the step's columns]
  int32_t* pos_s = reinterpret_cast<int32_t*>(stat_s + kStages * C::kStatFloats);    // [2][kMaxBlocks] offsets of decisions
  uint16_t* ulist = reinterpret_cast<uint16_t*>(pos_s + (DROP ? 2 * kMaxBlocks : 0));  // (block << 2) | presence bits
  uint8_t* kmask = reinterpret_cast<uint8_t*>(ulist + kMaxBlocks);
  uint64_t* a1_full = reinterpret_cast<uint64_t*>(kmask + kMaxBlocks);
  uint64_t* a2_full = a1_full + 1;
  uint64_t* full1 = a2_full + 1;        // [kStages] B1 (and the statistics) of a step have landed
  uint64_t* empty1 = full1 + kStages;   // [kStages] the MMAs that read it are done
  uint64_t* full2 = empty1 + kStages;   // [kStages] B2 likewise
  uint64_t* empty2 = full2 + kStages;
  uint64_t* s_full = empty2 + kStages;  // [kSBuf] S complete
  uint64_t* dp_full = s_full + kSBuf;   // dP complete
  uint64_t* p_full = dp_full + 1;       // [kSBuf] S consumed (and P' in its place); one for each buffer, since a warp
                                        // may be done with the next S before another is with this one
  uint64_t* ds_full = p_full + kSBuf;       // dS in place of dP
  uint64_t* done = ds_full + 1;         // the sums are complete
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);
  int* s_count = reinterpret_cast<int*>(tmem_holder + 1);
  int* s_last = s_count + 1;            // this CTA finishes the tile

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rows = DKV ? p.Ns : p.Nt;                  // of the resident side
  const int heads = DKV ? p.kv_heads : p.heads;
  const int tiles = (rows + kTileM - 1) / kTileM;
  int head, tile;                                      // and the CTA's part of the tile
  if (!pass.by_head) {  // the first tiles of all heads first: with global tokens they are the longest
    tile = block / heads;
    head = block - tile * heads;
  } else {
    const int per_head = SPLIT ? tiles * pass.split : tiles;
    head = block / per_head;
    tile = block - head * per_head;
  }
  int part = 0;
  if constexpr (SPLIT) {
    part = tile % pass.split;
    tile /= pass.split;
  }
  const int blk0 = tile * 2;                           // first of the tile's two blocks
  const int nbr = p.Nt / kBlk, nbc = p.Ns / kBlk;
  const int nstream = DKV ? nbr : nbc;

  // ------------------------------ prologue ------------------------------
  if (threadIdx.x == 0) {
    mbar_init(a1_full, 1);
    mbar_init(a2_full, 1);
    for (int st = 0; st < kStages; ++st) {
      mbar_init(&full1[st], 1);
      mbar_init(&empty1[st], 1);
      mbar_init(&full2[st], 1);
      mbar_init(&empty2[st], 1);
    }
    for (int b = 0; b < kSBuf; ++b) { mbar_init(&s_full[b], 1); mbar_init(&p_full[b], kScoreWarps); }
    mbar_init(dp_full, 1);
    mbar_init(ds_full, kScoreWarps);
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == kWarpLoad && lane == 0) {
    prefetch_tensormap(&tm_a1);
    prefetch_tensormap(&tm_a2);
    prefetch_tensormap(&tm_b1);
    prefetch_tensormap(&tm_b2);
  }
  if (warp == kWarpMma) tmem_alloc<C::kTmemCols>(tmem_holder);
  if constexpr (DKV) {
    for (int r = threadIdx.x; r < nbr; r += kThreads) {  // pitch is even: the two block columns are one 16-bit word
      const uint32_t two = __ldg(reinterpret_cast<const uint16_t*>(p.present + (long long)r * p.present_pitch + blk0));
      kmask[r] = static_cast<uint8_t>((two & 1u) | ((two >> 7) & 2u));
    }
  } else {
    const uint8_t* row0 = p.present + (long long)blk0 * p.present_pitch;
    const bool second = blk0 + 1 < nbr;                // the last tile may be one block row high
    for (int k = threadIdx.x; k < nbc; k += kThreads)
      kmask[k] = static_cast<uint8_t>(__ldg(row0 + k) | (second ? __ldg(row0 + p.present_pitch + k) << 1 : 0));
  }
  __syncthreads();
  if (warp == 0) {  // ordered compaction of the merged list
    int n = 0;
    for (int base = 0; base < nstream; base += 32) {
      const int k = base + lane;
      const int m = k < nstream ? kmask[k] : 0;
      const unsigned bal = __ballot_sync(0xffffffffu, m != 0);
      if (m) ulist[n + __popc(bal & ((1u << lane) - 1u))] = static_cast<uint16_t>((k << 2) | m);
      n += __popc(bal);
    }
    if (lane == 0) *s_count = n;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_holder, 0);
  const int count = __shfl_sync(0xffffffffu, *s_count, 0);
  if constexpr (READY) {
    for (int i = threadIdx.x; i < 2 * count; i += kThreads) {
      const int half = i & 1, e = ulist[i >> 1], blk = e >> 2;
      if ((e >> half) & 1) {
        const int pos = __ldg(p.position + (DKV ? (long long)blk * p.present_pitch + blk0 + half
                                                : (long long)(blk0 + half) * p.present_pitch + blk));
        pos_s[half * kMaxBlocks + (i >> 1)] = pos * kBitWords;
      }
    }
    __syncthreads();
  }
  const int pairs = (count + C::kBlocks - 1) / C::kBlocks;  // steps through the list
  const int all_steps = DKV ? pairs * p.group : pairs;  // dK, dV: the list once for every head that shares the keys
  // A tile whose steps would take one CTA far longer than the others (global tokens, heads that share their keys), or
  // that is one of few, is shared by several CTAs, each with a range of the steps.  They leave 32-bit partial sums; the
  // last one to finish adds them in their order.
  int parts = 1, step0 = 0, steps = all_steps, h0 = 0, k0 = 0;  // step = h * pairs + k
  if constexpr (SPLIT) {
    parts = min(pass.split, max(1, (all_steps + pass.split_steps / 2) / pass.split_steps));
    if (part >= parts) {
      if (warp == kWarpMma) tmem_dealloc<C::kTmemCols>(tmem_base);
      return;
    }
    step0 = static_cast<int>((long long)all_steps * part / parts);
    steps = static_cast<int>((long long)all_steps * (part + 1) / parts) - step0;
    h0 = pairs > 0 ? step0 / pairs : 0;
    k0 = step0 - h0 * pairs;
  }
  const long long a_row0 = (long long)head * rows + (long long)tile * kTileM;

  bool failed = false;  // a bounded wait of this thread gave up
  if (warp == kWarpLoad) {
    // ------------------------------ producer ------------------------------
    if (lane == 0 && steps > 0) {
      auto resident = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar) {
        mbar_arrive_expect_tx(bar, C::kABytes);
        for (int c = 0; c < kChunks; ++c) tma_load_2d(dst + c * (kTileM * 128), map, c * 64, (int)a_row0, bar);
      };
      resident(a1_s, &tm_a1, a1_full);  // with the first B1: the first S needs nothing else
      bool ok = true;
      int h = h0, k = k0;
      for (int j = 0; j < steps; ++j) {
        const int st = j % kStages, nblk = min(C::kBlocks, count - C::kBlocks * k);
        const uint32_t par = ((j / kStages) & 1) ^ 1;
        const long long row0 = DKV ? ((long long)head * p.group + h) * p.Nt : (long long)(head / p.group) * p.Ns;
        if (!mbar_wait(&empty1[st], par)) { ok = false; break; }
        mbar_arrive_expect_tx(&full1[st], nblk * (kBlk * D * 2 + (DKV ? 2 * kBlk * 4 : 0)));
        for (int b = 0; b < nblk; ++b) {
          const long long row = row0 + (ulist[C::kBlocks * k + b] >> 2) * kBlk;
          for (int c = 0; c < kChunks; ++c)
            tma_load_2d(b1_s + st * C::kBBytes + c * (C::kCols * 128) + b * (kBlk * 128), &tm_b1, c * 64, (int)row, &full1[st]);
          if constexpr (DKV) {
            bulk_load(stat_s + st * C::kStatFloats + b * kBlk, p.neg_lse + row, kBlk * 4, &full1[st]);
            bulk_load(stat_s + st * C::kStatFloats + C::kCols + b * kBlk, p.neg_delta + row, kBlk * 4, &full1[st]);
          }
        }
        if (j == 0) resident(a2_s, &tm_a2, a2_full);
        if (!mbar_wait(&empty2[st], par)) { ok = false; break; }
        mbar_arrive_expect_tx(&full2[st], nblk * kBlk * D * 2);
        for (int b = 0; b < nblk; ++b) {
          const long long row = row0 + (ulist[C::kBlocks * k + b] >> 2) * kBlk;
          for (int c = 0; c < kChunks; ++c)
            tma_load_2d(b2_s + st * C::kBBytes + c * (C::kCols * 128) + b * (kBlk * 128), &tm_b2, c * 64, (int)row, &full2[st]);
        }
        if (++k == pairs) { k = 0; ++h; }
      }
      failed |= !ok;
      if (!ok) atomicExch(&p.status[0], 1);
    }
  } else if (warp == kWarpMma) {
    // ------------------------------ MMA issue ------------------------------
    // K-major operands: 128-byte rows, 128-byte swizzle.  P', dS: A operands in tensor memory, lane = row, two 16-bit
    // values per column, eight columns per K = 16 slab, the two slabs of each 32 columns at the first 16 of them.
    // B1, B2 as right operands of the sums: MN-major (head dim contiguous), eight rows per 1024-byte group, 64-element
    // chunks C::kCols * 128 bytes apart.
    const uint64_t desc_k = make_smem_desc(0, 16, 1024, SW_128B), desc_mn = make_smem_desc(0, C::kCols * 128, 1024, SW_128B);
    const uint32_t hi_k = static_cast<uint32_t>(desc_k >> 32), hi_mn = static_cast<uint32_t>(desc_mn >> 32);
    const uint32_t flags_k = static_cast<uint32_t>(desc_k) & 0xffff0000u, flags_mn = static_cast<uint32_t>(desc_mn) & 0xffff0000u;
    const uint32_t a1 = flags_k | (smem_u32(a1_s) >> 4), a2 = flags_k | (smem_u32(a2_s) >> 4);
    const uint32_t b1 = smem_u32(b1_s) >> 4, b2 = smem_u32(b2_s) >> 4;
    constexpr uint32_t idesc_1 = make_idesc_f16(kTileM, kBlk, FMT, 0, 0), idesc_2 = make_idesc_f16(kTileM, 2 * kBlk, FMT, 0, 0);
    constexpr uint32_t idesc_acc = make_idesc_f16(kTileM, D, FMT, 0, 1);
    auto scores = [&](uint32_t d, uint32_t a, uint32_t b, int nblk) {  // d = A B^T
      const uint32_t idesc = nblk == 2 ? idesc_2 : idesc_1;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off_a = ((kk / 4) * (kTileM * 128) + (kk % 4) * 32) >> 4;
        const uint32_t off_b = ((kk / 4) * (C::kCols * 128) + (kk % 4) * 32) >> 4;
        umma_ss_lohi(d, a + off_a, hi_k, flags_k | (b + off_b), hi_k, idesc, kk > 0 ? 1u : 0u);
      }
    };
    auto accumulate = [&](uint32_t d, uint32_t a, uint32_t b, int nblk, bool first) {  // d += A (tensor memory) B
#pragma unroll
      for (int kk = 0; kk < C::kCols / 16; ++kk)
        if (kk < nblk * (kBlk / 16))
          umma_ts_lohi(d, a + (kk / 2) * 32 + (kk % 2) * 8, flags_mn | (b + ((kk * 16 * 128) >> 4)), hi_mn, idesc_acc,
                       (!first || kk > 0) ? 1u : 0u);
    };
    // the last pair of the list may be a single block
    auto blocks_of = [&](int j) { return C::kBlocks == 2 && !((count & 1) && (step0 + j + 1) % pairs == 0) ? 2 : 1; };
    bool ok = steps == 0 || mbar_wait_warp(a1_full, 0);
#pragma unroll
    for (int j = 0; j < kSBuf; ++j) {  // the first scores
      if (j >= steps || !ok) break;
      const int nblk = blocks_of(j);
      if (!mbar_wait_warp(&full1[j], 0)) { ok = false; break; }
      tc_fence_after_sync();
      if (elect_one()) {
        scores(tmem_base + j * C::kCols, a1, b1 + ((j * C::kBBytes) >> 4), nblk);
        umma_commit(&s_full[j]);
      }
      __syncwarp();
    }
    if (ok && steps > 0) {
      ok = mbar_wait_warp(a2_full, 0) && mbar_wait_warp(&full2[0], 0);
      if (ok) {
        tc_fence_after_sync();
        if (elect_one()) {
          scores(tmem_base + C::kDpCol, a2, b2, blocks_of(0));
          umma_commit(dp_full);
          if constexpr (!DKV) umma_commit(&empty2[0]);
        }
        __syncwarp();
      }
    }
    // (unrolled over the stages, so that every descriptor is a compile-time offset from a base register)
    for (int j0 = 0; j0 < steps && ok; j0 += kStages) {
#pragma unroll
      for (int st = 0; st < kStages; ++st) {
        const int j = j0 + st, round = j0 / kStages;
        if (j >= steps) break;
        const uint32_t par = j & 1;
        constexpr int kRing = kStages;
        const int nx = (st + kSBuf) % kRing, nx2 = (st + 1) % kRing;
        const uint32_t d = tmem_base + (j % kSBuf) * C::kCols, dp = tmem_base + C::kDpCol;
        const uint32_t off = (st * C::kBBytes) >> 4;
        const int nblk = blocks_of(j);
        // ---- P of this step is in place: P' B2, then S of a later step ----
        const bool more_s = j + kSBuf < steps;
        if (!mbar_wait_warp(&p_full[j % kSBuf], (j / kSBuf) & 1)) { ok = false; break; }
        tc_fence_after_sync();
        if constexpr (DKV) {
          if (elect_one()) {
            accumulate(tmem_base + C::kAcc2, d, b2 + off, nblk, j == 0);
            umma_commit(&empty2[st]);
          }
          __syncwarp();
        }
        if (more_s) {
          if (!mbar_wait_warp(&full1[nx], (round + (st + kSBuf) / kRing) & 1)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            scores(d, a1, b1 + ((nx * C::kBBytes) >> 4), blocks_of(j + kSBuf));
            umma_commit(&s_full[j % kSBuf]);
          }
          __syncwarp();
        }
        // ---- dS of this step is in place: dS B1, then dP of the next step ----
        const bool more = j + 1 < steps;
        if (!mbar_wait_warp(ds_full, par)) { ok = false; break; }
        tc_fence_after_sync();
        if (elect_one()) {
          accumulate(tmem_base + C::kAcc1, dp, b1 + off, nblk, j == 0);
          umma_commit(&empty1[st]);
          if (!more) umma_commit(done);
        }
        __syncwarp();
        if (more) {
          if (!mbar_wait_warp(&full2[nx2], (round + (st + 1) / kRing) & 1)) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            scores(dp, a2, b2 + ((nx2 * C::kBBytes) >> 4), blocks_of(j + 1));
            umma_commit(dp_full);
            if constexpr (!DKV) umma_commit(&empty2[nx2]);
          }
          __syncwarp();
        }
      }
    }
    failed |= !ok;
    if (!ok && lane == 0) atomicExch(&p.status[1], 1);
  } else {
    // ------------------------------ scores and epilogue ------------------------------
    const int quad = warp & 3, quarter = warp >> 2;    // lane quadrant, 32-column quarter of the step
    const int row = quad * 32 + lane;                  // of the tile == tensor-memory lane
    const int half = quad >> 1;                        // which of the tile's two blocks
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_base = tmem_base + lane_base + quarter * 32, dp_addr = s_base + C::kDpCol;
    const int grow = tile * kTileM + row;              // row inside the head
    const bool inside = grow < rows;
    float2 nl = make_float2(0.f, 0.f), nd = nl;
    if (!DKV && inside) {
      nl.x = nl.y = __ldg(p.neg_lse + a_row0 + row);
      nd.x = nd.y = __ldg(p.neg_delta + a_row0 + row);
    }
    const float up = p.drop.scale;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    int h = h0, k = k0;
    // READY: the list entry of a step and the decisions of its 32 x 32 scores, a step ahead
    const uint32_t* bits = nullptr;  // of the head, for this thread
    uint32_t next_bits = 0;
    int next_e = 0;
    auto look_ahead = [&] {
      const int at = C::kBlocks * k + (quarter >> 1);
      next_e = __shfl_sync(0xffffffffu, at < count ? ulist[at] : 0, 0);
      if ((next_e >> half) & 1) next_bits = __ldg(bits + pos_s[half * kMaxBlocks + at]);
    };
    PhiloxKey key = {};
    PhiloxRow key_row = {};
    if constexpr (DROP && !READY) {
      key = load_uniform_philox_key(p.drop);
      if constexpr (!DKV) key_row = philox_row(key, grow, head);
    }
    if constexpr (READY) {
      const int q_head = DKV ? head * p.group + h : head;
      bits = p.bits + (long long)q_head * p.bits_blocks * kBitWords + lane +
             (DKV ? (quad & 1) * kBlk + (quarter & 1) * 32 : (quarter & 1) * kBlk + (quad & 1) * 32);
      if (steps > 0) look_ahead();
    }
    for (int j = 0; j < steps; ++j) {
      const int st = j % kStages, at = C::kBlocks * k + (quarter >> 1);
      int e = next_e;
      if constexpr (!READY) e = __shfl_sync(0xffffffffu, at < count ? ulist[at] : 0, 0);
      const bool there = at < count;                   // the pair has this block
      const bool mine = (e >> half) & 1;               // it is kept for this warp's rows
      const int blk = e >> 2;
      const uint32_t s_addr = s_base + (j % kSBuf) * C::kCols;
      // words of decisions over the warp's 32 x 32 scores, made for rows of the score matrix: for this thread's own over
      // its columns (the mask's in split order), or for query `lane` of the block over the warp's keys
      uint32_t mask_w = 0xffffffffu, keep_w = 0xffffffffu;
      if ((MASK || DROP) && mine) {
        const int q_row = DKV ? blk * kBlk + (quarter & 1) * 32 + lane : grow;
        const int word = DKV ? tile * (kTileM / 32) + quad : blk * (kBlk / 32) + (quarter & 1);
        if constexpr (MASK) {
          mask_w = mask_word32(p.mask + (long long)q_row * p.Ns + word * 32);
          if constexpr (!DKV) mask_w = split_bits32(mask_w);
        }
        if constexpr (DROP) {
          if constexpr (READY) {
            keep_w = next_bits;
          } else {
            const int q_head = DKV ? head * p.group + h : head;
            if constexpr (DKV) key_row = philox_row(key, q_row, q_head);
            keep_w = philox_bits32(key, key_row, threshold2(p.drop), word, q_head);
          }
          if constexpr (DKV) keep_w = fragment_bits(keep_w, lane);
        }
      }
      if (++k == pairs) {
        k = 0; ++h;
        if constexpr (DKV && READY) bits += (long long)p.bits_blocks * kBitWords;
      }
      if constexpr (READY) {
        if (j + 1 < steps) look_ahead();
      }
      if (ok && DKV && !mbar_wait_warp(&full1[st], (j / kStages) & 1)) ok = false;  // the statistics are read here
      if (ok && !mbar_wait_warp(&s_full[j % kSBuf], (j / kSBuf) & 1)) ok = false;
      if (!ok) continue;
      tc_fence_after_sync();
      // ---- P = exp2(scale log2(e) S - lse log2(e)) ----
      const float* stat = stat_s + st * C::kStatFloats + quarter * 32 + 2 * (lane & 3);  // of this thread's columns
      float2 prob[16];
      uint32_t packed[16];
      if (mine) {
        uint32_t s[32];
        if constexpr (DKV) {
          tmem_ld_16x256b_x4(s_addr, s);
          tmem_ld_16x256b_x4(s_addr + (16u << 16), s + 16);
        } else {
          tmem_ld_x32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(s));
        }
        tmem_ld_wait();
        auto exp_pair = [&](int i, float2 n) {  // scores 2 i, 2 i + 1
          const float2 v = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, n);
          return make_float2(ex2_approx(v.x), ex2_approx(v.y));
        };
        if constexpr (DKV) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 stats = *reinterpret_cast<const float2*>(stat + 8 * n);
            const ColumnMasks m = MASK ? column_masks(mask_w, n, lane) : ColumnMasks{};
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // rows lane / 4 + 8 r
              const int i = (r >> 1) * 8 + 2 * n + (r & 1);
              float2 v = exp_pair(i, stats);
              if constexpr (MASK) v = mask_pair(v, m, r);
              prob[i] = v;
              packed[i] = pack2<T>(v.x, v.y);
              if constexpr (DROP) packed[i] &= packed_mask({keep_w << (2 * r), keep_w << (2 * r + 1)}, n);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 v = exp_pair(i, nl);
            if constexpr (MASK) {
              v.x = (mask_w >> i) & 1u ? v.x : 0.f;
              v.y = (mask_w >> (i + 16)) & 1u ? v.y : 0.f;
            }
            prob[i] = v;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[i] = 0;
      }
      if constexpr (DKV) {
        if (there) {  // over columns that this warp has read
          tmem_st_16x128b_x4(s_addr, packed);
          tmem_st_16x128b_x4(s_addr + (16u << 16), packed + 8);
          tmem_st_wait();
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      mbar_arrive_if(&p_full[j % kSBuf], lane == 0);
      // ---- dS = P (dP - delta) ----
      if (!mbar_wait_warp(dp_full, j & 1)) { ok = false; continue; }
      tc_fence_after_sync();
      if (mine) {
        uint32_t s[32];
        if constexpr (DKV) {
          tmem_ld_16x256b_x4(dp_addr, s);
          tmem_ld_16x256b_x4(dp_addr + (16u << 16), s + 16);
        } else {
          tmem_ld_x32(dp_addr, *reinterpret_cast<uint32_t(*)[32]>(s));
        }
        tmem_ld_wait();
        const float2 up2 = make_float2(up, up);
        if constexpr (DKV) {
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 stats = *reinterpret_cast<const float2*>(stat + C::kCols + 8 * n);
            const ColumnMasks m = MASK ? column_masks(mask_w, n, lane) : ColumnMasks{};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int i = (r >> 1) * 8 + 2 * n + (r & 1);
              float2 v = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
              v = DROP ? fma2(mask_pair(v, {keep_w << (2 * r), keep_w << (2 * r + 1)}, n), up2, stats) : add2(v, stats);
              v = mul2(prob[i], v);
              packed[i] = pack2<T>(v.x, v.y);
              // a masked score's probability is zero, and so is its dS whatever stands in V
              if constexpr (MASK) packed[i] &= packed_mask(m, r);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 v = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
            if constexpr (DROP) {
              const uint32_t four = keep_w << (i >> 1);  // columns 2 i, 2 i + 1 at the tops of bytes 2 (i & 1) and the next
              v.x = __uint_as_float(__float_as_uint(v.x) & permute_signs(four, 0, 0x8888u + (i & 1) * 0x2222u));
              v.y = __uint_as_float(__float_as_uint(v.y) & permute_signs(four, 0, 0x9999u + (i & 1) * 0x2222u));
            }
            v = mul2(prob[i], DROP ? fma2(v, up2, nd) : add2(v, nd));
            packed[i] = pack2<T>(v.x, v.y);
            if constexpr (MASK) packed[i] &= pair_mask(mask_w, i);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[i] = 0;
      }
      if (there) {
        if constexpr (DKV) {
          tmem_st_16x128b_x4(dp_addr, packed);
          tmem_st_16x128b_x4(dp_addr + (16u << 16), packed + 8);
        } else {
          tmem_st_x16(dp_addr, packed);
        }
        tmem_st_wait();
      }
      tc_fence_before_sync();
      __syncwarp();
      mbar_arrive_if(ds_full, lane == 0);
    }
    // ---- epilogue: the sums -> global, one row per thread, 32-column pieces dealt to the threads of a row ----
    if (ok && steps > 0 && !mbar_wait_warp(done, 0)) ok = false;
    failed |= !ok;
    if (!ok && lane == 0) atomicExch(&p.status[3], 1);
    tc_fence_after_sync();
    constexpr int kPieces = (DKV ? 2 : 1) * D / 32;
    const long long tile_id = (long long)head * tiles + tile;
    // partial sums: [piece][float4 of the piece][row], so that a warp's accesses are contiguous
    auto partial_at = [&](int of, int piece) {
      return reinterpret_cast<float4*>(pass.partial) + ((tile_id * pass.split + of) * kPieces + piece) * (8 * kTileM) + row;
    };
    auto load_piece = [&](int piece, float (&v)[32]) {
      if (steps > 0 && ok) {
        uint32_t r[32];
        tmem_ld_x32(tmem_base + lane_base + C::kAcc1 + piece * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
      }
    };
    auto store_piece = [&](int piece, const float (&v)[32]) {
      const bool second = piece >= D / 32;             // dV
      const float f = second ? (DROP ? up : 1.f) : p.scale;
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(second ? pass.out2 : pass.out1) + (a_row0 + row) * D + (piece % (D / 32)) * 32);
      if (inside) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          dst[q] = make_uint4(pack2<T>(v[8 * q] * f, v[8 * q + 1] * f), pack2<T>(v[8 * q + 2] * f, v[8 * q + 3] * f),
                              pack2<T>(v[8 * q + 4] * f, v[8 * q + 5] * f), pack2<T>(v[8 * q + 6] * f, v[8 * q + 7] * f));
      }
    };
    if (!SPLIT || parts == 1) {
      for (int piece = quarter; piece < kPieces; piece += kScoreWarps / 4) {
        float v[32];
        load_piece(piece, v);
        store_piece(piece, v);
      }
    } else {
      for (int piece = quarter; piece < kPieces; piece += kScoreWarps / 4) {
        float v[32];
        load_piece(piece, v);
        float4* dst = partial_at(part, piece);
#pragma unroll
        for (int q = 0; q < 8; ++q) __stcg(dst + q * kTileM, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
      }
      __threadfence();
      named_barrier_sync(1, kScoreWarps * 32);
      if (threadIdx.x == 0) *s_last = atomicAdd(pass.tickets + tile_id, 1u) == static_cast<uint32_t>(parts - 1);
      named_barrier_sync(1, kScoreWarps * 32);
      if (*s_last) {  // the others' sums are in L2
        __threadfence();
        for (int piece = quarter; piece < kPieces; piece += kScoreWarps / 4) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
          for (int of = 0; of < parts; ++of) {
            const float4* src = partial_at(of, piece);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 x = __ldcg(src + q * kTileM);
              v[4 * q] += x.x; v[4 * q + 1] += x.y; v[4 * q + 2] += x.z; v[4 * q + 3] += x.w;
            }
          }
          store_piece(piece, v);
        }
      }
    }
  }
  tc_fence_before_sync();
  sync_and_drain(failed);
  if (warp == kWarpMma) {
    tc_fence_after_sync();
    tmem_dealloc<C::kTmemCols>(tmem_base);
  }
}

// Tensor maps by tensor and box height: as resident tiles and as streamed blocks.
struct BwdMaps {
  CUtensorMap q_tile, do_tile, k_tile, v_tile, q_block, do_block, k_block, v_block;
};

// Both passes in one launch, the blocks of the dK, dV pass first (its tiles take longer): nothing of one needs anything
// of the other, and the last blocks of the first run beside the first of the second.
template <int D, int FMT, bool MASK, bool DROP, bool SPLIT>
__global__ void __launch_bounds__(BwdCfg<true, D>::kThreads, BwdCfg<true, D>::kCtasPerSM)
attn_bwd_kernel(const __grid_constant__ BwdMaps m, const __grid_constant__ BwdParams p, const __grid_constant__ PassParams kv,
                const __grid_constant__ PassParams q, int kv_blocks) {
  static_assert(BwdCfg<true, D>::kThreads == BwdCfg<false, D>::kThreads, "one launch, one block size");
  const int block = blockIdx.x;
  auto pass = [&](auto ready) {
    constexpr bool kReady = decltype(ready)::value;
    if (block < kv_blocks) bwd_pass<true, D, FMT, MASK, DROP, kReady, SPLIT>(m.k_tile, m.v_tile, m.q_block, m.do_block, p, kv, block);
    else bwd_pass<false, D, FMT, MASK, DROP, kReady, SPLIT>(m.q_tile, m.do_tile, m.k_block, m.v_block, p, q, block - kv_blocks);
  };
  // All of them or none, decided once: a choice in every step cost the steps that have their decisions 40 to 100 us of
  // 520 (B4 H16 S4096 D64, both passes).  Only the device knows how many blocks there are: `nnz` is a hint.
  if constexpr (DROP) {
    if (__ldg(p.blocks) <= p.bits_blocks) pass(std::true_type{});
    else pass(std::false_type{});
  } else {
    pass(std::false_type{});
  }
}

int rows_map(CUtensorMap* map, const void* base, int dtype, int D, long long rows, uint32_t box_rows) {
  const uint64_t dims[2] = {(uint64_t)D, (uint64_t)rows}, strides[1] = {(uint64_t)D * 2};
  const uint32_t box[2] = {64, box_rows};
  return make_tensor_map(map, base, dtype, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Tiles, CTAs per tile and steps per CTA of a pass.  Splitting aims at CTAs of half of what a resident CTA would have to
// do if the work were dealt out evenly; `nnz` (kept blocks, 0 when unknown: no splitting) says how much there is, 0.65 of
// it being what merging two block rows typically leaves.  A CTA takes kMinSteps steps at least: below that its fixed
// costs and its partial sums (written once, read once) outweigh the balance.
struct PassPlan {
  int tiles, split, split_steps;
  size_t partial_bytes;
};
constexpr int kMinSteps = 12, kMaxSplit = 16;
constexpr size_t kMaxPartialBytes = size_t(128) << 20;  // of a pass
constexpr size_t kMaxBitsBytes = size_t(1) << 30;       // a bit per kept score of every head: as much as Q (D 64) at 16 blocks a row

template <bool DKV, int D>
PassPlan plan_pass(int heads, int kv_heads, int Nt, int Ns, long long nnz) {
  using C = BwdCfg<DKV, D>;
  const int h = DKV ? kv_heads : heads, rows = DKV ? Ns : Nt, stream = DKV ? Nt : Ns;
  PassPlan plan;
  plan.tiles = (rows + kTileM - 1) / kTileM;
  const long long ctas = (long long)h * plan.tiles;
  const long long most = (long long)((stream / kBlk + C::kBlocks - 1) / C::kBlocks) * (DKV ? heads / kv_heads : 1);  // steps of a tile
  const double even = 0.65 * static_cast<double>(nnz) * heads / C::kBlocks / (kNumSMs * C::kCtasPerSM);
  long long steps = static_cast<long long>(even / 2) + 1;
  if (steps < kMinSteps) steps = kMinSteps;
  const size_t bytes = sizeof(float) * kTileM * D * (DKV ? 2 : 1);
  long long split = nnz > 0 ? (most + steps / 2) / steps : 1;
  if (split > kMaxSplit) split = kMaxSplit;
  while (split > 1 && ctas * split * bytes > kMaxPartialBytes) --split;
  plan.split = split < 1 ? 1 : static_cast<int>(split);
  if (plan.split == kMaxSplit) steps = (most + plan.split - 1) / plan.split > steps ? (most + plan.split - 1) / plan.split : steps;
  plan.split_steps = static_cast<int>(steps > 0x3fffffff ? 0x3fffffff : steps);
  plan.partial_bytes = plan.split > 1 ? ctas * plan.split * bytes : 0;
  return plan;
}

int present_pitch(int Ns) { return (Ns / kBlk + 1) & ~1; }
size_t round16(size_t n) { return (n + 15) & ~size_t(15); }

struct Workspace {
  size_t neg_lse, neg_delta, present, position, tickets_q, tickets_kv, partial_q, partial_kv, total;  // total: decisions begin
  long long n_tickets;
  PassPlan q, kv;
};
template <int D>
Workspace lay_out(int heads, int kv_heads, int Nt, int Ns, long long nnz) {
  Workspace w;
  w.q = plan_pass<false, D>(heads, kv_heads, Nt, Ns, nnz);
  w.kv = plan_pass<true, D>(heads, kv_heads, Nt, Ns, nnz);
  w.n_tickets = (long long)heads * w.q.tiles + (long long)kv_heads * w.kv.tiles;
  w.neg_lse = 0;
  w.neg_delta = w.neg_lse + round16(sizeof(float) * (size_t)heads * Nt);
  w.present = w.neg_delta + round16(sizeof(float) * (size_t)heads * Nt);
  w.position = w.present + round16((size_t)(Nt / kBlk) * present_pitch(Ns));
  w.tickets_q = w.position + round16(sizeof(int32_t) * (size_t)(Nt / kBlk) * present_pitch(Ns));
  w.tickets_kv = w.tickets_q + sizeof(uint32_t) * (size_t)heads * w.q.tiles;
  w.partial_q = w.tickets_q + round16(sizeof(uint32_t) * (size_t)w.n_tickets);
  w.partial_kv = w.partial_q + w.q.partial_bytes;
  w.total = w.partial_kv + w.kv.partial_bytes;
  return w;
}

template <int D, int FMT, bool MASK, bool DROP>
int launch_bwd(const AttnArgs& a, BwdParams p, cudaStream_t st) {
  using T = typename std::conditional<FMT == 0, __half, __nv_bfloat16>::type;
  const Workspace w = lay_out<D>(a.heads, a.kv_heads, a.Nt, a.Ns, a.nnz);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  float* neg_lse = reinterpret_cast<float*>(ws + w.neg_lse);
  float* neg_delta = reinterpret_cast<float*>(ws + w.neg_delta);
  uint32_t* tickets_q = reinterpret_cast<uint32_t*>(ws + w.tickets_q);
  p.neg_lse = neg_lse; p.neg_delta = neg_delta; p.present = ws + w.present;
  p.present_pitch = present_pitch(a.Ns);
  const long long q_rows = (long long)a.heads * a.Nt, k_rows = (long long)a.kv_heads * a.Ns;
  constexpr int kRowsPerBlock = kPrepRows * 2048 / D;
  const long long prep_ctas = (q_rows + kRowsPerBlock - 1) / kRowsPerBlock;
  PrepBits make = {};
  if constexpr (DROP) {
    make.drop = p.drop;
    make.heads = a.heads;
    make.position = reinterpret_cast<int32_t*>(ws + w.position);
    make.bits = reinterpret_cast<uint32_t*>(ws + w.total);
    const size_t room = (a.workspace_bytes - w.total) / (sizeof(uint32_t) * kBitWords * (size_t)a.heads);
    const size_t most = (size_t)(a.Nt / kBlk) * (a.Ns / kBlk);
    make.blocks = static_cast<int>(room < most ? room : most);
    p.position = make.position; p.bits = make.bits; p.bits_blocks = make.blocks;
    const long long items = (long long)make.blocks * a.heads, ctas = (items + 7) / 8;
    make.ctas = static_cast<int>(ctas < 8 * kNumSMs ? ctas : 8 * kNumSMs);
  }
  attn_bwd_prep_kernel<T, D, DROP><<<static_cast<unsigned>(prep_ctas + make.ctas), 256, 0, st>>>(
      static_cast<const T*>(a.O), static_cast<const T*>(a.dO), a.lse, neg_lse, neg_delta, ws + w.present, a.row_ptr, a.idx, q_rows,
      a.Nt / kBlk, a.Ns / kBlk, p.present_pitch, tickets_q, w.n_tickets, make);
  if (int rc = launch_status(); rc != SPARTA_OK) return rc;
  BwdMaps m;
  int rc = rows_map(&m.q_tile, a.Q, a.dtype, D, q_rows, kTileM);
  if (rc == SPARTA_OK) rc = rows_map(&m.do_tile, a.dO, a.dtype, D, q_rows, kTileM);
  if (rc == SPARTA_OK) rc = rows_map(&m.k_tile, a.K, a.dtype, D, k_rows, kTileM);
  if (rc == SPARTA_OK) rc = rows_map(&m.v_tile, a.V, a.dtype, D, k_rows, kTileM);
  if (rc == SPARTA_OK) rc = rows_map(&m.q_block, a.Q, a.dtype, D, q_rows, kBlk);
  if (rc == SPARTA_OK) rc = rows_map(&m.do_block, a.dO, a.dtype, D, q_rows, kBlk);
  if (rc == SPARTA_OK) rc = rows_map(&m.k_block, a.K, a.dtype, D, k_rows, kBlk);
  if (rc == SPARTA_OK) rc = rows_map(&m.v_block, a.V, a.dtype, D, k_rows, kBlk);
  if (rc != SPARTA_OK) return rc;
  PassParams kv = {}, q = {};
  kv.out1 = a.dK; kv.out2 = a.dV;
  kv.by_head = kv_exceeds_l2(a.heads, a.Nt, D);
  kv.split = w.kv.split; kv.split_steps = w.kv.split_steps;
  kv.partial = reinterpret_cast<float*>(ws + w.partial_kv);
  kv.tickets = reinterpret_cast<uint32_t*>(ws + w.tickets_kv);
  q.out1 = a.dQ;
  q.by_head = kv_exceeds_l2(a.kv_heads, a.Ns, D);
  q.split = w.q.split; q.split_steps = w.q.split_steps;
  q.partial = reinterpret_cast<float*>(ws + w.partial_q);
  q.tickets = tickets_q;
  const long long kv_ctas = a.dK ? (long long)a.kv_heads * w.kv.tiles * w.kv.split : 0;
  const long long q_ctas = a.dQ ? (long long)a.heads * w.q.tiles * w.q.split : 0;
  if (kv_ctas + q_ctas > 0x7fffffffll) return SPARTA_ERR_SHAPE;
  auto launch = [&](auto kern, SmemAttrOnce& attr) {
    constexpr int kKv = BwdCfg<true, D>::smem_bytes(DROP), kQ = BwdCfg<false, D>::smem_bytes(DROP), kSmem = kKv > kQ ? kKv : kQ;
    static_assert((kSmem + 1024) * BwdCfg<true, D>::kCtasPerSM <= 228 * 1024, "shared memory budget");
    if (cudaError_t e = attr.ensure(kern, kSmem); e != cudaSuccess) return static_cast<int>(e);
    kern<<<static_cast<unsigned>(kv_ctas + q_ctas), BwdCfg<true, D>::kThreads, kSmem, st>>>(m, p, kv, q, static_cast<int>(kv_ctas));
    return launch_status();
  };
  static SmemAttrOnce attr_whole, attr_split;
  return w.kv.split > 1 || w.q.split > 1 ? launch(attn_bwd_kernel<D, FMT, MASK, DROP, true>, attr_split)
                                         : launch(attn_bwd_kernel<D, FMT, MASK, DROP, false>, attr_whole);
}

template <int D, int FMT>
int launch_variant(const AttnArgs& a, const BwdParams& p, cudaStream_t st) {
  const bool drop = p.drop.threshold > 0;
  if (a.mask) return drop ? launch_bwd<D, FMT, true, true>(a, p, st)
                          : launch_bwd<D, FMT, true, false>(a, p, st);
  return drop ? launch_bwd<D, FMT, false, true>(a, p, st)
              : launch_bwd<D, FMT, false, false>(a, p, st);
}

}  // namespace

size_t attn_bwd_workspace(int heads, int kv_heads, int Nt, int Ns, int D, long long nnz) {
  return D == 64 ? lay_out<64>(heads, kv_heads, Nt, Ns, nnz).total : lay_out<128>(heads, kv_heads, Nt, Ns, nnz).total;
}

// Room for the dropout decisions of `nnz` blocks for every head, up to kMaxBitsBytes.
size_t attn_bwd_dropout_workspace(int heads, long long nnz) {
  const size_t block = sizeof(uint32_t) * kBitWords * (size_t)heads;
  const size_t fit = kMaxBitsBytes / block;
  return block * ((size_t)nnz < fit ? (size_t)nnz : fit);
}

int attn_bwd_launch(const AttnArgs& a, const DropoutParams& drop, int32_t* status, cudaStream_t st) {
  if (a.Ns / kBlk > kMaxBlocks || a.Nt / kBlk > kMaxBlocks) return SPARTA_ERR_UNSUPPORTED;
  BwdParams p = {};
  p.mask = a.mask;
  p.Nt = a.Nt; p.Ns = a.Ns; p.heads = a.heads; p.kv_heads = a.kv_heads; p.group = a.heads / a.kv_heads;
  p.scale = a.scale; p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = status;
  p.drop = drop;
  p.blocks = a.row_ptr + a.Nt / kBlk;
  if (a.D == 64) return a.dtype == SPARTA_F16 ? launch_variant<64, 0>(a, p, st) : launch_variant<64, 1>(a, p, st);
  return a.dtype == SPARTA_F16 ? launch_variant<128, 0>(a, p, st) : launch_variant<128, 1>(a, p, st);
}

}  // namespace sparta

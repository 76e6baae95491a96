// Tensor-core engine of the expert block (tcgen05.mma.cta_group::2, sm_100a):
// four ragged grouped products on one kernel, over segments
// [offsets[e], offsets[e+1]) of grouped rows.
//
//   kGated  h = act(x Wg[e]) * (x Wu[e])             contraction over hidden
//   kDx     dx = dg Wg[e]^T + du Wu[e]^T             contraction over 2 x output
//   kDw     dWg[e] = x_e^T dg_e, dWu[e] = x_e^T du_e contraction over the rows
//   kInt8   y = (xq . wq[e]^T) * xs[row] * ws[e][n]  contraction over hidden
//
// A pair of CTAs computes a 256-row tile whose 256 accumulator columns are 256
// output columns (kDx, kInt8) or 128 columns of each of two products that
// share their A operand (kGated: gate and up; kDw: the two weight gradients),
// so one MMA of N = 256 advances both products and x is read once for both.
// Each CTA holds half of B: in kDw one gradient each, in kGated 64 columns of
// gate and the same 64 of up, which then lie 64 accumulator columns apart in
// one thread's row, where the activation and the product are applied.
//
// A tile with at most 128 rows left (the end of a segment, or an expert with
// few rows) is issued with M = 128, 64 rows per CTA, at half the tensor time.
// Its accumulator is folded: TMEM lanes 0-63 hold the even CTA's half of the
// columns, lanes 64-127 the odd CTA's, both for the CTA's 64 rows.
//
// Operands reach shared memory by TMA in 128-byte-swizzled boxes of 16 KB per
// operand, part and k-block (64 bfloat16 or 128 int8 deep). Whatever layout
// the tensors have in memory is used as it is: K-major where the contraction
// is the contiguous axis (x in kGated, everything in kDx and kInt8), MN-major
// where it is not (the weights in kGated, both operands of kDw), so no tensor
// is transposed.
//
// FP32 (three parts per operand): each operand is the exact sum of three bfloat16 parts
// (8 + 8 + 8 significand bits, each part rounded to nearest: at most 1, 2^-8 and
// 2^-17 of it), and the product sums the six part products of weight 2^-17 and above;
// what is left out is at most 2^-24 of |a||b| and has either sign. The
// tensor core truncates when it accumulates, with a bias that grows with the
// number of steps taken at full magnitude, so every k-block is its own
// accumulation, small products first (four full-magnitude steps), and the
// epilogue warps add the blocks in FP32 registers while the next block runs
// in the other half of TMEM.
//
// Roles (384 threads per CTA): warp 0 TMA producer (both CTAs' loads complete
// on the even CTA's barriers); warp 1 MMA issuer (even CTA); warp 2, in kDw,
// clears the rows of a segment's last block that belong to other segments and
// hands that block over; warps 4-11 epilogue. TMEM holds two 256-column accumulators, so a tile's
// epilogue runs beside the next tile's products. Waits are bounded as in the
// other pair engine (gemm_pair.cu), with the same exit protocol.
//
// Bound by the tensor pipe, busy 86% of the time at 8 experts, 16384 rows, K=4096,
// N=1408 (kGated, bfloat16: 243 us, DRAM 334 MB read, 41 MB written). 128 experts of 1024
// rows: 2.12 ms in a burst (1.42 PFLOP/s), 2.51 ms back to back (1.21), where the power
// limit sets the clock. FP32 (six products): 64 experts, 32768 rows, K=N=1024: 0.73
// ms of 1.08 with the packing. Taller tiles (512 rows, two accumulators sharing B) took
// 844 against 912 us for one dense 8192^3 product but 2.68 against 2.41 ms over ragged
// segments, whose tails grow and whose epilogue no longer runs beside the products;
// FP32 blocks 32 deep took 757 against 727 us.
#include <cuda.h>

#include <mutex>

#include "expert_block.cuh"
#include "sm100.cuh"

namespace rrb {
namespace {

using namespace sm100;

enum Mode { kGated, kDx, kDw, kInt8 };

constexpr int kRowsCta = 128;
constexpr int kTileM = 2 * kRowsCta;
constexpr int kTileN = 256;
constexpr int kBoxBytes = 8192;            // 64 lines of 128 bytes
constexpr int kOperandBytes = 2 * kBoxBytes;
constexpr int kBand = 8;
constexpr int kTmemCols = 512;
constexpr int kEpiWarp0 = 4;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarp0 + kEpiWarps) * 32;
constexpr uint64_t kDrainNs = 2000000;
constexpr int kPolls = 256;
// What a k-block may take beyond the limit of a wait (0.4 us where the tensor pipe is
// full), for the waits that last as long as a tile's contraction.
constexpr uint64_t kBlockLimitNs = 4000;
constexpr int kStagingBytes = 32 * 64;  // 64 bytes of 32 rows, per epilogue warp

// A stage holds one k-block: kPa parts of A and kPb parts of B, 16 KB each.
template <int kPa, int kPb>
struct Config {
  static constexpr int kOffB = kPa * kOperandBytes;
  static constexpr int kStageBytes = kOffB + kPb * kOperandBytes;
  static constexpr int kStages = 12 * kOperandBytes / kStageBytes;  // 192 KB
};

struct EngineArgs {
  const int32_t* offsets;
  void* out0;
  void* out1;
  float* gate_up;
  const float* row_scale;
  const float* col_scale;
  unsigned* err;
  int experts, rows;
  int hidden;   // contraction of kGated and kInt8; output columns of kDx, rows of kDw's tiles
  int output;   // output columns of kGated, kDw, kInt8; contraction (twice) of kDx
  int activation;
  int vec;          // 16-byte stores of out0 / out1 allowed
  int vec_gate_up;  // and of gate_up
};

template <typename Cfg>
struct alignas(1024) EngineSmem {
  uint8_t stage[Cfg::kStages][Cfg::kStageBytes];
  uint8_t staging[kEpiWarps][kStagingBytes];  // output rows on their way out
  uint64_t empty[Cfg::kStages];  // the pair's MMAs have read the stage
  uint64_t ready[Cfg::kStages];  // even CTA: both CTAs' halves are in place
  uint64_t tail[Cfg::kStages];   // kDw: this CTA's half of a short block landed
  uint64_t tmem_full[2];         // accumulator finished (both CTAs)
  uint64_t tmem_empty[2];        // even CTA: both CTAs have read it
  uint64_t mma_done;
  uint32_t tmem_base;
  int failed;
  int prefix[kMaxExperts + 1];
  int scratch[33];
};

// kind::f16 with bfloat16 operands and FP32 accumulation.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn) << 15) |
         (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// kind::i8 with signed operands and 32-bit integer accumulation.
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct Tile {
  int expert;
  int m0, m_end;  // rows of the output (kDw: of the weight matrix)
  int m_mma;      // rows of the instruction: 256, or 128 when at most 128 are left
  int c0, ncols;  // columns of each product
  int n_mma;      // accumulator columns, a multiple of 32
  int own;        // kGated: gate (and up) columns of each CTA
  int k_blocks;   // of the contraction
  int row0, row_end;  // the segment (kDw's contraction)
};

__device__ __forceinline__ int tiles_of(int2 s, int n_tiles) {
  return ((s.y - s.x + kTileM - 1) / kTileM) * n_tiles;
}

// Exclusive prefix of the experts' tile counts (all threads); the total.
__device__ __forceinline__ int build_prefix(const EngineArgs& p, int n_tiles, int* prefix,
                                            int* scratch) {
  const int per = (p.experts + kThreads - 1) / kThreads;
  const int e0 = min(p.experts, static_cast<int>(threadIdx.x) * per);
  const int e1 = min(p.experts, e0 + per);
  int local = 0;
  for (int e = e0; e < e1; ++e) local += tiles_of(segment(p.offsets, e, p.rows), n_tiles);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = local;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  int run = incl - local;
  for (int w = 0; w < warp; ++w) run += scratch[w];
  for (int e = e0; e < e1; ++e) {
    prefix[e] = run;
    run += tiles_of(segment(p.offsets, e, p.rows), n_tiles);
  }
  if (threadIdx.x == kThreads - 1) prefix[p.experts] = run;
  __syncthreads();
  return prefix[p.experts];
}

template <int kMode>
__device__ __forceinline__ Tile tile_at(const EngineArgs& p, int t, const int* prefix,
                                        int n_tiles) {
  constexpr bool kTwo = kMode == kGated || kMode == kDw;  // two products side by side
  Tile g;
  int local;
  if constexpr (kMode == kDw) {
    const int per = ((p.hidden + kTileM - 1) / kTileM) * n_tiles;
    g.expert = t / per;
    local = t - g.expert * per;
  } else {
    int lo = 0, hi = p.experts - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (prefix[mid] <= t) lo = mid; else hi = mid - 1;
    }
    g.expert = lo;
    local = t - prefix[lo];
  }
  const int2 s = segment(p.offsets, g.expert, p.rows);
  g.row0 = s.x;
  g.row_end = s.y;
  // Bands of kBand row tiles, column by column: the tiles in flight then touch
  // about as many row blocks as column blocks, so few bytes feed them all.
  const int m_tiles = kMode == kDw ? (p.hidden + kTileM - 1) / kTileM : tiles_of(s, 1);
  const int band = local / (kBand * n_tiles);
  const int in_band = local - band * kBand * n_tiles;
  const int band_tiles = min(kBand, m_tiles - band * kBand);
  const int nt = in_band / band_tiles;
  const int mt = band * kBand + in_band - nt * band_tiles;
  const int width = kTwo ? kTileN / 2 : kTileN;
  const int total = kMode == kDx ? p.hidden : p.output;
  g.c0 = nt * width;
  g.ncols = min(width, total - g.c0);
  // kGated: a CTA's up columns follow a whole box of 64 gate columns.
  g.own = min(64, (((g.ncols + 1) >> 1) + 15) & ~15);
  if constexpr (kMode == kGated) g.n_mma = 2 * (64 + g.own);
  else g.n_mma = kTwo ? 2 * ((g.ncols + 15) & ~15) : (g.ncols + 31) & ~31;
  if constexpr (kMode == kDw) {
    g.m0 = mt * kTileM;
    g.m_end = p.hidden;
    g.k_blocks = (s.y - s.x + 63) >> 6;
  } else {
    g.m0 = s.x + mt * kTileM;
    g.m_end = s.y;
    if constexpr (kMode == kDx) g.k_blocks = 2 * ((p.output + 63) >> 6);
    else if constexpr (kMode == kInt8) g.k_blocks = (p.hidden + 127) >> 7;
    else g.k_blocks = (p.hidden + 63) >> 6;
  }
  g.m_mma = g.m_end - g.m0 <= kRowsCta ? kRowsCta : kTileM;
  return g;
}

// Writes 64 bytes of each of a warp's 32 output rows; lane r holds row r in v.
// An accumulator row belongs to one thread, so storing from registers would
// touch 32 lines with 16 bytes each; through shared memory a warp writes whole
// 64-byte pieces of eight rows at a time (or, where rows are not 16-byte
// aligned or the piece is cut, consecutive elements). Chunk c of row r sits at
// c ^ (r / 2 mod 4): no bank conflicts in either direction.
// kUnroll: of the element-wise form (whole, where registers allow).
template <typename T, int kUnroll>
__device__ __forceinline__ void store_rows(uint8_t* staging, const float* v, T* base, long long ld,
                                           int rows, int cols, bool vec) {
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kCols = 4 * kPer;
  const int lane = threadIdx.x & 31;
  __syncwarp();  // the previous piece has been read
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    *reinterpret_cast<uint4*>(staging + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
        pack16<T>(v + kPer * c);
  }
  __syncwarp();
  if (vec && cols >= kCols) {
    const int c = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2);
      if (r < rows) {
        *reinterpret_cast<uint4*>(base + r * ld + kPer * c) = *reinterpret_cast<const uint4*>(
            staging + r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
      }
    }
  } else {
    const int col = lane % kCols;
    const int c = col / kPer;
    if (col < cols) {
      T* out = base + lane / kCols * ld + col;
#pragma unroll kUnroll
      for (int i = 0; i < kCols; ++i, out += 32 / kCols * ld) {
        const int r = lane / kCols + i * (32 / kCols);
        if (r < rows) {
          *out = *reinterpret_cast<const T*>(staging + r * 64 + ((c ^ ((r >> 1) & 3)) << 4) +
                                             (col % kPer) * sizeof(T));
        }
      }
    }
  }
}

// 32 columns of a warp's rows: one piece of bfloat16 or two of float.
template <typename T, int kUnroll>
__device__ __forceinline__ void store_rows32(uint8_t* staging, const float* v, T* base,
                                             long long ld, int rows, int cols, bool vec) {
  constexpr int kCols = 64 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 32 / kCols; ++i) {
    if (cols > i * kCols) {
      store_rows<T, kUnroll>(staging, v + i * kCols, base + i * kCols, ld, rows, cols - i * kCols, vec);
    }
  }
}

template <int kMode, int kPa, int kPb, typename T>
__global__ void __launch_bounds__(kThreads, 1) expert_gemm_kernel(
    const __grid_constant__ CUtensorMap map_a0, const __grid_constant__ CUtensorMap map_a1,
    const __grid_constant__ CUtensorMap map_b0, const __grid_constant__ CUtensorMap map_b1,
    const EngineArgs p) {
  using Cfg = Config<kPa, kPb>;
  constexpr bool kTwo = kMode == kGated || kMode == kDw;
  constexpr bool kMnA = kMode == kDw;
  constexpr bool kMnB = kMode == kGated || kMode == kDw;
  constexpr bool kFp32 = kPa == 3;  // every k-block its own accumulation
  constexpr int kUnroll = kFp32 ? 8 : 32;
  constexpr int kStages = Cfg::kStages;
  constexpr int kOffB = Cfg::kOffB;
  // Byte step of one K = 16 (bfloat16) or 32 (int8) MMA inside a box, and the
  // descriptors' offsets: K-major tiles repeat every 8 rows of 128 bytes;
  // MN-major ones every 8 k-lines of 128 bytes, the next 64 columns one box on.
  constexpr uint32_t kStepA = kMnA ? 2048 : 32, kStepB = kMnB ? 2048 : 32;
  constexpr uint32_t kLboA = kMnA ? kBoxBytes : 16, kLboB = kMnB ? kBoxBytes : 16;
  // Part products (a, b) in rising magnitude. Three parts: 2^-16 three times,
  // 2^-8 twice, 1.
  constexpr int kProducts = kFp32 ? 6 : kPa * kPb;
  constexpr int kProductA[6] = {kFp32 ? 2 : kPa - 1, 0, 1, 1, 0, 0};
  constexpr int kProductB[6] = {kFp32 ? 0 : kPb - 1, kFp32 ? 2 : 0, 1, 0, 1, 0};

  extern __shared__ uint8_t smem_raw[];
  auto& s = *reinterpret_cast<EngineSmem<Cfg>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = rank == 0;
  const int unit = static_cast<int>(blockIdx.x >> 1);
  const int units = static_cast<int>(gridDim.x >> 1);
  constexpr int kWidth = kTwo ? kTileN / 2 : kTileN;
  const int n_tiles = ((kMode == kDx ? p.hidden : p.output) + kWidth - 1) / kWidth;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&s.empty[i], 1);
      mbar_init(&s.ready[i], kMode == kDw ? 2 : 1);
      mbar_init(&s.tail[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.tmem_full[i], 1);
      mbar_init(&s.tmem_empty[i], 2 * kEpiWarps);
    }
    mbar_init(&s.mma_done, 1);
    s.failed = 0;
    fence_mbar_init();
  }
  // Tensor memory is taken only once the kernel before has ended, and the next
  // kernel may come only once it is taken: no block waits with what another needs.
  wait_for_previous();
  if (warp == 1) {
    tmem_alloc_pair(&s.tmem_base, kTmemCols);
    tmem_relinquish_pair();
  }
  int total;
  if constexpr (kMode == kDw) {
    total = p.experts * ((p.hidden + kTileM - 1) / kTileM) * n_tiles;
  } else {
    total = build_prefix(p, n_tiles, s.prefix, s.scratch);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  let_next_start();
  const uint32_t tmem = s.tmem_base;
  volatile int* failed = &s.failed;
  const uint32_t peer_failed = mapa_shared(smem_u32(&s.failed), rank ^ 1);
  auto wait = [&](uint64_t* bar, uint32_t parity, int blocks = 0) {
    // Most waits end within microseconds: poll before reading any clock.
#pragma unroll 1
    for (int i = 0; i < kPolls; ++i) {
      if (mbar_try_wait(bar, parity)) return true;
    }
    return mbar_wait_pair(bar, parity, p.err, failed, peer_failed,
                          kWaitLimitNs + static_cast<uint64_t>(blocks) * kBlockLimitNs);
  };
  auto tile = [&](int t) { return tile_at<kMode>(p, t, s.prefix, n_tiles); };

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    int stage = 0;
    uint32_t phase = 0;
    for (int t = unit; t < total && !*failed; t += units) {
      const Tile g = tile(t);
      const int half = g.n_mma >> 1;
      const int m = g.m0 + rank * (g.m_mma >> 1);
      for (int kb = 0; kb < g.k_blocks; ++kb) {
        if (!wait(&s.empty[stage], phase ^ 1u)) break;
        if (elect_one()) {
          // Both CTAs' bytes complete on the even CTA's barrier. A short last
          // block of kDw completes on each CTA's own: its relay warp hands it
          // over once it has cleared the lines past the segment.
          const bool cut = kMode == kDw && g.row_end - g.row0 - kb * 64 < 64;
          uint32_t bar;
          if (cut) {
            bar = smem_u32(&s.tail[stage]);
            mbar_arrive_expect_tx(&s.tail[stage], Cfg::kStageBytes);
          } else {
            bar = mapa_shared(smem_u32(&s.ready[stage]), 0u);
            if (leader) mbar_arrive_expect_tx(&s.ready[stage], 2 * Cfg::kStageBytes);
            else if (kMode == kDw) mbar_arrive_remote(bar);
          }
          // The contraction's first element; kDx passes over two pairs of operands.
          const int pass = g.k_blocks >> 1;
          const bool second = kMode == kDx && kb >= pass;
          const int k = kMode == kDw ? g.row0 + kb * 64
                                     : (second ? kb - pass : kb) * (kMode == kInt8 ? 128 : 64);
          uint8_t* a = s.stage[stage];
#pragma unroll
          for (int q = 0; q < kPa; ++q, a += kOperandBytes) {
            if constexpr (kMode == kDw) {
              tma_load_3d_pair(a, &map_a0, bar, m, k, q);
              tma_load_3d_pair(a + kBoxBytes, &map_a0, bar, m + 64, k, q);
            } else {
              tma_load_3d_pair(a, second ? &map_a1 : &map_a0, bar, k, m, q);
            }
          }
          uint8_t* b = a;
#pragma unroll
          for (int q = 0; q < kPb; ++q, b += kOperandBytes) {
            const int z = q * p.experts + g.expert;
            if constexpr (kMode == kGated) {
              const int c = g.c0 + rank * g.own;
              tma_load_3d_pair(b, &map_b0, bar, c, k, z);
              tma_load_3d_pair(b + kBoxBytes, &map_b1, bar, c, k, z);
            } else if constexpr (kMode == kDw) {
              const CUtensorMap* mb = leader ? &map_b0 : &map_b1;
              tma_load_3d_pair(b, mb, bar, g.c0, k, q);
              tma_load_3d_pair(b + kBoxBytes, mb, bar, g.c0 + 64, k, q);
            } else {
              tma_load_3d_pair(b, second ? &map_b1 : &map_b0, bar, k, g.c0 + rank * half, z);
            }
          }
        }
        __syncwarp();
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    // Wait for the MMAs' last use of every stage: nothing may read or signal
    // this CTA's shared memory after it exits.
    for (int i = 0; i < kStages && !*failed; ++i) {
      if (!wait(&s.empty[stage], phase ^ 1u)) break;
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (even CTA) ----------------
    if (leader) {
      int stage = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = unit; t < total && ok && !*failed; t += units) {
        const Tile g = tile(t);
        const uint32_t idesc = kMode == kInt8 ? idesc_i8(g.m_mma, g.n_mma)
                                              : idesc_f16(g.m_mma, g.n_mma, kMnA, kMnB);
        for (int kb = 0; kb < g.k_blocks; ++kb) {
          if (((kFp32 || kb == 0) && !wait(&s.tmem_empty[buf], acc_phase ^ 1u)) ||
              !wait(&s.ready[stage], phase)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const bool last = kFp32 || kb + 1 == g.k_blocks;
          if (elect_one()) {
            const uint32_t d = tmem + static_cast<uint32_t>(buf) * kTileN;
            const uint32_t base = smem_u32(s.stage[stage]);
            const uint64_t a0 = smem_desc(base, kLboA, 1024, Swizzle::k128B);
            const uint64_t b0 = smem_desc(base + kOffB, kLboB, 1024, Swizzle::k128B);
#pragma unroll
            for (int q = 0; q < kProducts; ++q) {
              const uint64_t aq = a0 + kProductA[q] * (kOperandBytes >> 4);
              const uint64_t bq = b0 + kProductB[q] * (kOperandBytes >> 4);
#pragma unroll
              for (uint32_t ks = 0; ks < 4; ++ks) {
                const uint64_t ad = aq + ks * (kStepA >> 4), bd = bq + ks * (kStepB >> 4);
                const uint32_t add = ((!kFp32 && kb > 0) || q > 0 || ks > 0) ? 1u : 0u;
                if constexpr (kMode == kInt8) mma_i8_pair(d, ad, bd, idesc, add);
                else mma_bf16_pair(d, ad, bd, idesc, add);
              }
            }
            mma_commit_pair_both(smem_u32(&s.empty[stage]));
            if (last) mma_commit_pair_both(smem_u32(&s.tmem_full[buf]));
          }
          __syncwarp();
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (last) {
            buf ^= 1;
            if (buf == 0) acc_phase ^= 1u;
          }
        }
      }
      if (elect_one()) mma_commit_pair_to(smem_u32(&s.mma_done));
      __syncwarp();
      int dummy = 0;
      mbar_wait(&s.mma_done, 0, p.err, &dummy);
    }
  } else if (warp == 2) {
    // ---------------- relay (kDw): short last blocks ----------------
    if constexpr (kMode == kDw) {
      int at = 0;           // k-blocks so far: stage at % kStages
      uint32_t phases = 0;  // per stage, of its tail barrier
      for (int t = unit; t < total && !*failed; t += units) {
        const Tile g = tile(t);
        at = (at + g.k_blocks) % kStages;
        const int valid = (g.row_end - g.row0) & 63;
        if (valid == 0) continue;
        const int stage = (at + kStages - 1) % kStages;  // of the last block
        if (!wait(&s.tail[stage], (phases >> stage) & 1u, g.k_blocks)) break;
        phases ^= 1u << stage;
        // Lines past the segment's end hold other segments' rows (or
        // anything): both operands become zero there. A line is one row of a
        // box, so the swizzle inside it does not matter.
        for (int bx = 0; bx < 2 * (kPa + kPb); ++bx) {
          uint8_t* box = s.stage[stage] + bx * kBoxBytes;
          for (int i = valid * 8 + lane; i < 512; i += 32) {
            reinterpret_cast<uint4*>(box)[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&s.ready[stage]), 0u));
      }
    }
  } else if (warp >= kEpiWarp0) {
    // ---------------- epilogue ----------------
    const int quarter = warp & 3;  // the TMEM lanes this warp may read
    const int hw = (warp - kEpiWarp0) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    uint8_t* staging = s.staging[warp - kEpiWarp0];
    int buf = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = unit; t < total && ok && !*failed; t += units) {
      const Tile g = tile(t);
      const int half = g.n_mma >> 1;
      const bool folded = g.m_mma < kTileM;
      const int side = quarter >> 1;  // folded: the half of the columns in these lanes
      const int row0 = g.m0 + rank * (g.m_mma >> 1) +
                       (folded ? quarter & 1 : quarter) * 32;  // of the warp
      const int rows = max(0, min(32, g.m_end - row0));
      // This warp's groups of 32 accumulator columns, q = 0 .. groups - 1:
      // TMEM column, first output column, and output columns left from there
      // on (none: the group is skipped; warp-uniform). In kGated a group's
      // up columns lie 64 TMEM columns after its gate columns.
      const int groups = (kMode == kGated ? 2 : 4) >> (folded ? 1 : 0);
      auto group_col = [&](int q) {
        if constexpr (kMode == kGated) return folded ? 32 * hw : hw * half + 32 * q;
        else if constexpr (kMode == kDw) return folded ? hw * 64 + 32 * q : hw * half + 32 * q;
        else return folded ? hw * 64 + 32 * q : hw * 128 + 32 * q;
      };
      auto group_out = [&](int q) {
        if constexpr (kMode == kGated) {
          return folded ? side * g.own + 32 * hw : hw * g.own + 32 * q;
        } else if constexpr (kMode == kDw) {
          return folded ? hw * 64 + 32 * q : 32 * q;
        } else {
          return folded ? side * half + hw * 64 + 32 * q : hw * 128 + 32 * q;
        }
      };
      auto group_left = [&](int q) {
        const int out = group_out(q);
        if constexpr (kMode == kGated) {
          return min(g.ncols, ((folded ? side : hw) + 1) * g.own) - out;
        } else if constexpr (kMode == kDw) {
          return g.ncols - out;
        } else {
          return min(g.ncols, folded ? (side + 1) * half : g.ncols) - out;
        }
      };
      // kInt8: the scales of this lane's row and, of each group, of column `lane`,
      // read while the products run.
      float row_scale = 0.0f, col_scale[4] = {};
      if constexpr (kMode == kInt8) {
        if (lane < rows) row_scale = __ldg(p.row_scale + row0 + lane);
        const float* scales = p.col_scale + static_cast<long long>(g.expert) * p.output + g.c0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (q < groups && lane < group_left(q)) col_scale[q] = __ldg(scales + group_out(q) + lane);
        }
      }
      // Stores group q: v, in kGated with its up columns v2.
      auto put = [&](int q, const float* v, const float* v2) {
        const int c = group_out(q);
        const int cols = group_left(q);
        if (rows == 0 || cols <= 0) return;  // warp-uniform
        if constexpr (kMode == kGated) {
          float h[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) h[i] = activate<T>(p.activation, v[i]) * v2[i];
          const long long at = static_cast<long long>(row0) * p.output + g.c0 + c;
          store_rows32<T, kUnroll>(staging, h, static_cast<T*>(p.out0) + at, p.output, rows, cols,
                          p.vec != 0);
          if (p.gate_up != nullptr) {
            float* gu = p.gate_up + 2LL * row0 * p.output + g.c0 + c;
            store_rows32<float, kUnroll>(staging, v, gu, 2LL * p.output, rows, cols,
                                p.vec_gate_up != 0);
            store_rows32<float, kUnroll>(staging, v2, gu + p.output, 2LL * p.output, rows, cols,
                                p.vec_gate_up != 0);
          }
        } else if constexpr (kMode == kDw) {
          T* out = static_cast<T*>((folded ? side : hw) == 0 ? p.out0 : p.out1) +
                   (static_cast<long long>(g.expert) * p.hidden + row0) * p.output + g.c0 + c;
          store_rows32<T, kUnroll>(staging, v, out, p.output, rows, cols, p.vec != 0);
        } else {
          const int ld = kMode == kDx ? p.hidden : p.output;
          T* out = static_cast<T*>(p.out0) + static_cast<long long>(row0) * ld + g.c0 + c;
          if constexpr (kMode == kInt8) {
            const float ws = q < 2 ? (q == 0 ? col_scale[0] : col_scale[1])
                                   : (q == 2 ? col_scale[2] : col_scale[3]);
            float y[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              y[i] = static_cast<float>(__float_as_int(v[i])) * row_scale *
                     __shfl_sync(0xffffffffu, ws, i);
            }
            store_rows32<T, kUnroll>(staging, y, out, ld, rows, cols, p.vec != 0);
          } else {
            store_rows32<T, kUnroll>(staging, v, out, ld, rows, cols, p.vec != 0);
          }
        }
      };
      auto take = [&]() {  // the accumulator is finished
        if (!wait(&s.tmem_full[buf], acc_phase, g.k_blocks)) return false;
        tc_fence_after();
        return true;
      };
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(mapa_shared(smem_u32(&s.tmem_empty[buf]), 0u));
        buf ^= 1;
        if (buf == 0) acc_phase ^= 1u;
      };
      if constexpr (kMode == kDw) {
        if (g.k_blocks == 0) {  // no rows: a zero gradient
          const float zero[32] = {};
#pragma unroll 1
          for (int q = 0; q < groups; ++q) put(q, zero, zero);
          continue;
        }
      }
      if constexpr (!kFp32) {
        if (!take()) break;
        auto load = [&](int col, float* v) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(tmem + static_cast<uint32_t>(buf * kTileN + col) + lane_addr, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        };
#pragma unroll 1
        for (int q = 0; q < groups; ++q) {
          if (group_left(q) <= 0) break;
          float v[32];
          load(group_col(q), v);
          if constexpr (kMode == kGated) {
            float v2[32];
            load(group_col(q) + 64, v2);
            put(q, v, v2);
          } else {
            put(q, v, v);
          }
        }
        release();
      } else {
        float sum[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) sum[i] = 0.0f;
        for (int kb = 0; kb < g.k_blocks; ++kb) {
          if (!take()) {
            ok = false;
            break;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // 16 columns; kGated: 0-3 gate, 4-7 up
            const int q = kMode == kGated ? (i >> 1) & 1 : i >> 1;
            if (q < groups && group_left(q) > 0) {
              uint32_t r[16];
              const int col =
                  group_col(q) + 16 * (i & 1) + (kMode == kGated ? 64 * (i >> 2) : 0);
              tmem_ld_32x32b_x16(tmem + static_cast<uint32_t>(buf * kTileN + col) + lane_addr,
                                 r);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 16; ++c) sum[16 * i + c] += __uint_as_float(r[c]);
            }
          }
          release();
        }
        if (!ok) break;
#pragma unroll
        for (int q = 0; q < (kMode == kGated ? 2 : 4); ++q) {
          if (q < groups) put(q, sum + 32 * q, sum + (32 * q + (kMode == kGated ? 64 : 0)));
        }
      }
    }
  }

  __syncthreads();
  if (threadIdx.x == 0 && *failed) {
    // After a wait that ran out: give this CTA's loads in flight (microseconds
    // each) time to land before its shared memory is given up.
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < kDrainNs) {
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the pair's MMAs are done; no arrivals into either CTA remain
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, kTmemCols);
}

// ---- host side -----------------------------------------------------------------

// [d2][d1][d0] elements with row stride ld (elements) and plane stride d1 * ld.
bool encode_map(CUtensorMap* map, const void* base, bool int8, long long d0, long long d1,
                long long d2, long long ld, int box0, int box1) {
  EncodeTiledFn encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t size = int8 ? 1 : 2;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d0), static_cast<cuuint64_t>(d1),
                              static_cast<cuuint64_t>(d2)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * size,
                                 static_cast<cuuint64_t>(ld) * size * dims[1]};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box0), static_cast<cuuint32_t>(box1), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode(map, int8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;

// CTA pairs the device can hold at once, per kernel and device; 0 when the
// kernel cannot be configured there.
template <int kMode, int kPa, int kPb, typename T>
int engine_units(std::size_t smem) {
  static std::mutex mutex;
  static int known[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  std::lock_guard<std::mutex> lock(mutex);
  if (known[dev] == 0) {
    auto* kernel = expert_gemm_kernel<kMode, kPa, kPb, T>;
    int n = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) == cudaSuccess) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(2 * sm_count(), 1, 1);
      cfg.blockDim = dim3(kThreads, 1, 1);
      cfg.dynamicSmemBytes = smem;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
    }
    if (n <= 0) {
      cudaGetLastError();
      return 0;
    }
    known[dev] = n;
  }
  return known[dev];
}

template <int kMode, int kPa, int kPb, typename T>
cudaError_t launch_engine(const CUtensorMap (&maps)[4], EngineArgs args, long long tiles,
                          cudaStream_t stream) {
  constexpr std::size_t smem = sizeof(EngineSmem<Config<kPa, kPb>>) + 1024;
  static_assert(smem <= 227 * 1024, "over the shared memory a CTA may use");
  int units = engine_units<kMode, kPa, kPb, T>(smem);
  if (units <= 0) return cudaErrorNotSupported;
  if (tiles < units) units = static_cast<int>(tiles);
  if (units <= 0) return cudaSuccess;
  args.err = device_error_word();
  return launch_following(expert_gemm_kernel<kMode, kPa, kPb, T>, dim3(2 * units), kThreads, smem, 2,
                          stream, maps[0], maps[1], maps[2], maps[3], args);
}

// Output tiles of the row modes, at most: every expert with rows may end in a
// partial one.
long long row_tiles(int rows, int experts, int columns, int width) {
  const long long m = rows / kTileM + (experts < rows ? experts : rows);
  return m * ceil_div(columns, width);
}

bool vec_ok(const void* p, int ld, Dtype t) {
  return p == nullptr || (aligned_to(p, 16) && (ld * dtype_bytes(t)) % 16 == 0);
}

}  // namespace

cudaError_t launch_gated_gemm(const GatedOperands& in, const int32_t* offsets, void* h,
                              float* gate_up, int rows, int experts, int hidden, int output,
                              Activation activation, Dtype dtype, cudaStream_t stream) {
  CUtensorMap maps[4] = {};
  const long long planes = static_cast<long long>(in.terms) * experts;
  if (!encode_map(&maps[0], in.x, false, hidden, rows, in.terms, in.ldk, 64, kRowsCta) ||
      !encode_map(&maps[2], in.wg, false, output, hidden, planes, in.ldn, 64, 64) ||
      !encode_map(&maps[3], in.wu, false, output, hidden, planes, in.ldn, 64, 64)) {
    return cudaErrorInvalidValue;
  }
  maps[1] = maps[0];
  EngineArgs a{};
  a.offsets = offsets;
  a.out0 = h;
  a.gate_up = gate_up;
  a.experts = experts;
  a.rows = rows;
  a.hidden = hidden;
  a.output = output;
  a.activation = static_cast<int>(activation);
  a.vec = vec_ok(h, output, dtype);
  a.vec_gate_up = vec_ok(gate_up, output, Dtype::kFp32);
  const long long tiles = row_tiles(rows, experts, output, kTileN / 2);
  return dtype == Dtype::kBf16
             ? launch_engine<kGated, 1, 1, __nv_bfloat16>(maps, a, tiles, stream)
             : launch_engine<kGated, 3, 3, float>(maps, a, tiles, stream);
}

cudaError_t launch_gated_dx(const GatedOperands& in, const __nv_bfloat16* dg,
                            const __nv_bfloat16* du, int parts, const int32_t* offsets, void* dx,
                            int rows, int experts, int hidden, int output, Dtype dtype,
                            cudaStream_t stream) {
  CUtensorMap maps[4] = {};
  const long long planes = static_cast<long long>(in.terms) * experts;
  if (!encode_map(&maps[0], dg, false, output, rows, parts, in.ldn, 64, kRowsCta) ||
      !encode_map(&maps[1], du, false, output, rows, parts, in.ldn, 64, kRowsCta) ||
      !encode_map(&maps[2], in.wg, false, output, hidden, planes, in.ldn, 64, kRowsCta) ||
      !encode_map(&maps[3], in.wu, false, output, hidden, planes, in.ldn, 64, kRowsCta)) {
    return cudaErrorInvalidValue;
  }
  EngineArgs a{};
  a.offsets = offsets;
  a.out0 = dx;
  a.experts = experts;
  a.rows = rows;
  a.hidden = hidden;
  a.output = output;
  a.vec = vec_ok(dx, hidden, dtype);
  const long long tiles = row_tiles(rows, experts, hidden, kTileN);
  if (dtype == Dtype::kFp32) return launch_engine<kDx, 3, 3, float>(maps, a, tiles, stream);
  if (parts == 2) return launch_engine<kDx, 2, 1, __nv_bfloat16>(maps, a, tiles, stream);
  return launch_engine<kDx, 1, 1, __nv_bfloat16>(maps, a, tiles, stream);
}

cudaError_t launch_gated_dw(const GatedOperands& in, const __nv_bfloat16* dg,
                            const __nv_bfloat16* du, int parts, const int32_t* offsets, void* dwg,
                            void* dwu, int rows, int experts, int hidden, int output, Dtype dtype,
                            cudaStream_t stream) {
  CUtensorMap maps[4] = {};
  if (!encode_map(&maps[0], in.x, false, hidden, rows, in.terms, in.ldk, 64, 64) ||
      !encode_map(&maps[2], dg, false, output, rows, parts, in.ldn, 64, 64) ||
      !encode_map(&maps[3], du, false, output, rows, parts, in.ldn, 64, 64)) {
    return cudaErrorInvalidValue;
  }
  maps[1] = maps[0];
  EngineArgs a{};
  a.offsets = offsets;
  a.out0 = dwg;
  a.out1 = dwu;
  a.experts = experts;
  a.rows = rows;
  a.hidden = hidden;
  a.output = output;
  a.vec = vec_ok(dwg, output, dtype) && vec_ok(dwu, output, dtype);
  const long long tiles = static_cast<long long>(experts) * ceil_div(hidden, kTileM) *
                          ceil_div(output, kTileN / 2);
  if (dtype == Dtype::kFp32) return launch_engine<kDw, 3, 3, float>(maps, a, tiles, stream);
  if (parts == 2) return launch_engine<kDw, 1, 2, __nv_bfloat16>(maps, a, tiles, stream);
  return launch_engine<kDw, 1, 1, __nv_bfloat16>(maps, a, tiles, stream);
}

cudaError_t launch_int8_gemm(const int8_t* xq, const float* x_scale, const int8_t* wq,
                             const float* w_scale, const int32_t* offsets, void* y, int rows,
                             int experts, int ld, int output, Dtype dtype, cudaStream_t stream) {
  CUtensorMap maps[4] = {};
  if (!encode_map(&maps[0], xq, true, ld, rows, 1, ld, 128, kRowsCta) ||
      !encode_map(&maps[2], wq, true, ld, output, experts, ld, 128, kRowsCta)) {
    return cudaErrorInvalidValue;
  }
  maps[1] = maps[0];
  maps[3] = maps[2];
  EngineArgs a{};
  a.offsets = offsets;
  a.out0 = y;
  a.row_scale = x_scale;
  a.col_scale = w_scale;
  a.experts = experts;
  a.rows = rows;
  a.hidden = ld;
  a.output = output;
  a.vec = vec_ok(y, output, dtype);
  const long long tiles = row_tiles(rows, experts, output, kTileN);
  return dtype == Dtype::kBf16 ? launch_engine<kInt8, 1, 1, __nv_bfloat16>(maps, a, tiles, stream)
                               : launch_engine<kInt8, 1, 1, float>(maps, a, tiles, stream);
}

}  // namespace rrb

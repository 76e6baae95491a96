// The parts of the gated expert projection around the tensor-core engine
// (expert_gemm.cu): the form for a few rows, the packing of operands the
// engine cannot read as they are, and the pointwise half of the gradient.
#include <climits>

#include "expert_block.cuh"
#include "sm100.cuh"

namespace rrb {
namespace {

// ---- few rows --------------------------------------------------------------------
//
// h[r, c] = act(sum_k x[r, k] Wg[e][k, c]) * sum_k x[r, k] Wu[e][k, c] for a
// handful of rows: bound by reading the weights of the experts that have
// rows, 2 K N elements each, once. A cluster takes 128 bytes of columns of up to
// kFewRows rows of one expert, 16 bytes of each matrix per thread and k-step, with the
// contraction spread over its blocks and their threads; the partial sums
// (FP32) meet by shuffles, in shared memory and in the first block of the
// cluster, in a fixed order. (Two rows of 128 experts, K=4096, N=1408, bfloat16: 46 MB in
// 11.5 us, 4.0 TB/s; the rest is its start and the join.) The cluster grows (to 8 blocks) until every SM has
// work to keep its loads in flight: one row of a narrow layer is a few dozen
// column groups.

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewMaxCols = 64;
template <typename T>
constexpr int kFewCols = 128 / static_cast<int>(sizeof(T));  // a line of the weights
constexpr int kFewRows = 4;
constexpr int kMaxSplit = 8;

struct FewSmem {
  float warps[kFewWarps][kFewRows][2][kFewMaxCols];      // gate and up sums of each warp
  float parts[kMaxSplit - 1][kFewRows][2][kFewMaxCols];  // and of the cluster's other blocks
};

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// kVec consecutive elements as loaded, and as floats.
template <typename T, int kVec>
struct Raw {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = ld_stream16(p); }
  __device__ __forceinline__ void get(float* f) const { unpack16<T>(v, f); }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(p); }
  __device__ __forceinline__ void get(float* f) const { f[0] = to_f32(v); }
};

template <typename T, int kVec, int kR>
__device__ __forceinline__ void few_rows(const T* __restrict__ x, const T* __restrict__ wg,
                                         const T* __restrict__ wu, T* __restrict__ h,
                                         float* __restrict__ gate_up, int row, int nrows,
                                         int hidden, int output, int c0, int activation,
                                         int split, FewSmem& s) {
  constexpr int kCols = kFewCols<T>;
  constexpr int kLanes = kCols / kVec;           // threads across the columns
  constexpr int kGroups = kFewThreads / kLanes;  // contraction groups of a block
  constexpr int kUnroll = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // Partial sums that meet in shared memory: one per warp, or (a scalar row of
  // 64 bfloat16 takes two warps) one per pair of warps.
  constexpr int kWide = kLanes > 32 ? kLanes / 32 : 1;
  constexpr int kSums = kFewWarps / kWide;
  const int sum_row = warp / kWide;
  const int part = static_cast<int>(sm100::cluster_ctarank());
  const int stride = split * kGroups;
  // A block's shared memory may be written by its cluster only once it runs: each
  // says so here, and the others wait for that behind the weights, for nothing.
  if (split > 1) sm100::cluster_arrive();
  const int col = (threadIdx.x % kLanes) * kVec;
  const int kg = threadIdx.x / kLanes;
  float g[kR][kVec], u[kR][kVec];
#pragma unroll
  for (int i = 0; i < kR; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) g[i][j] = u[i][j] = 0.0f;
  }
  if (c0 + col < output) {
    const T* pg = wg + c0 + col;
    const T* pu = wu + c0 + col;
    const T* px[kR];
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      px[i] = x + static_cast<long long>(row + min(i, nrows - 1)) * hidden;
    }
    auto step = [&](int k, const Raw<T, kVec>& wa, const Raw<T, kVec>& wb) {
      float a[kVec], b[kVec];
      wa.get(a);
      wb.get(b);
#pragma unroll
      for (int i = 0; i < kR; ++i) {
        const float v = to_f32(__ldg(px[i] + k));
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          g[i][j] = fmaf(v, a[j], g[i][j]);
          u[i][j] = fmaf(v, b[j], u[i][j]);
        }
      }
    };
    int k = part * kGroups + kg;
    for (; k + (kUnroll - 1) * stride < hidden; k += kUnroll * stride) {
      Raw<T, kVec> a[kUnroll], b[kUnroll];
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) {
        const long long at = static_cast<long long>(k + q * stride) * output;
        a[q].load(pg + at);
        b[q].load(pu + at);
      }
#pragma unroll
      for (int q = 0; q < kUnroll; ++q) step(k + q * stride, a[q], b[q]);
    }
    for (; k < hidden; k += stride) {
      Raw<T, kVec> a, b;
      const long long at = static_cast<long long>(k) * output;
      a.load(pg + at);
      b.load(pu + at);
      step(k, a, b);
    }
  }
  // Sum over the contraction groups: lanes of a warp, then warps.
#pragma unroll
  for (int i = 0; i < kR; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
#pragma unroll
      for (int d = kLanes; d < 32; d <<= 1) {  // (none where a row takes a warp or more)
        g[i][j] += __shfl_xor_sync(0xffffffffu, g[i][j], d);
        u[i][j] += __shfl_xor_sync(0xffffffffu, u[i][j], d);
      }
      if (lane < kLanes) {
        s.warps[sum_row][i][0][col + j] = g[i][j];
        s.warps[sum_row][i][1][col + j] = u[i][j];
      }
    }
  }
  __syncthreads();
  const int i = threadIdx.x / kCols, c = threadIdx.x % kCols;
  float sg = 0.0f, su = 0.0f;
  if (i < kR) {
#pragma unroll
    for (int w = 0; w < kSums; ++w) {
      sg += s.warps[w][i][0][c];
      su += s.warps[w][i][1][c];
    }
  }
  if (split > 1) {
    sm100::cluster_wait();
    if (part > 0 && i < kR) {
      const uint32_t to = sm100::mapa_shared(sm100::smem_u32(&s.parts[part - 1][i][0][c]), 0u);
      sm100::st_shared_cluster_u32(to, __float_as_uint(sg));
      sm100::st_shared_cluster_u32(to + kFewMaxCols * 4, __float_as_uint(su));
    }
    sm100::cluster_sync();
    if (part > 0) return;
    if (i < kR) {
      for (int q = 0; q < split - 1; ++q) {
        sg += s.parts[q][i][0][c];
        su += s.parts[q][i][1][c];
      }
    }
  }
  if (i < nrows && i < kR && c0 + c < output) {
    const long long r = row + i;
    h[r * output + c0 + c] = from_f32<T>(activate<T>(activation, sg) * su);
    if (gate_up != nullptr) {
      gate_up[2 * r * output + c0 + c] = sg;
      gate_up[(2 * r + 1) * output + c0 + c] = su;
    }
  }
}

// The expert whose segment holds `row` (the block's threads look at all of them),
// or `experts`.
__device__ __forceinline__ int expert_of(const int32_t* __restrict__ offsets, int row, int rows,
                                         int experts) {
  __shared__ int owner;
  if (threadIdx.x == 0) owner = experts;
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kFewThreads) {
    const int2 s = segment(offsets, e, rows);
    if (s.x <= row && row < s.y) atomicMin(&owner, e);
  }
  __syncthreads();
  return owner;
}

// kR rows of an expert share a reading of its weights. One row at a time needs
// half the registers, so twice the loads are in flight.
template <typename T, int kVec, int kR>
__global__ void __launch_bounds__(kFewThreads, kR == 1 ? 4 : 2) gated_few_kernel(
    const T* __restrict__ x, const T* __restrict__ wg, const T* __restrict__ wu,
    const int32_t* __restrict__ offsets, T* __restrict__ h, float* __restrict__ gate_up, int rows,
    int experts, int hidden, int output, int activation, int split) {
  __shared__ FewSmem smem;
  follow_previous();
  const int row = blockIdx.y;
  const int e = expert_of(offsets, row, rows, experts);
  // Uniform over a cluster, whose blocks share the row.
  if (e == experts) return;  // a row outside every segment
  const int2 s = segment(offsets, e, rows);
  if ((row - s.x) % kR != 0) return;  // an earlier block's row
  const long long at = static_cast<long long>(e) * hidden * output;
  few_rows<T, kVec, kR>(x, wg + at, wu + at, h, gate_up, row, min(kR, s.y - row), hidden, output,
                        blockIdx.x / split * kFewCols<T>, activation, split, smem);
}

template <typename T>
cudaError_t few(const void* x, const void* wg, const void* wu, const int32_t* offsets, void* h,
                float* gate_up, int rows, int experts, int hidden, int output, int activation,
                cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  const bool vec = output % kVec == 0 && aligned_to(wg, 16) && aligned_to(wu, 16);
  const int groups = ceil_div(output, kFewCols<T>);
  // With rows scarce among the experts hardly any two share one, and rows are
  // taken one at a time; more may share an expert.
  const bool single = rows <= 2 || 2 * rows <= experts;
  // Contraction steps of a thread without a split; a split leaves four.
  const int steps = hidden / (kFewThreads / (kFewCols<T> / (vec ? kVec : 1)));
  int split = 1;
  while (split < kMaxSplit &&
         static_cast<long long>(groups) * rows * split < (single ? 4 : 2) * kNumSms &&
         steps >= 8 * split) {
    split *= 2;
  }
  auto* kernel = vec ? (single ? gated_few_kernel<T, kVec, 1> : gated_few_kernel<T, kVec, kFewRows>)
                     : (single ? gated_few_kernel<T, 1, 1> : gated_few_kernel<T, 1, kFewRows>);
  return launch_following(kernel, dim3(groups * split, rows), kFewThreads, 0, split, stream,
                          static_cast<const T*>(x), static_cast<const T*>(wg),
                          static_cast<const T*>(wu), offsets, static_cast<T*>(h), gate_up, rows,
                          experts, hidden, output, activation, split);
}

// ---- gradients of few rows ------------------------------------------------------------
//
// From dg and du in FP32 (no rounding before the sums). The input gradient reads
// the weights of the experts that have rows once, along their rows:
//   dx[r, k] = sum_n dg[r, n] Wg[e][k, n] + du[r, n] Wu[e][k, n];
// a warp takes kDxRows weight rows of up to kFewRows rows of one expert (46 MB as
// above: 16.9 us with the pointwise half).

constexpr int kDxRows = 4;

template <typename T, int kVec, int kR>
__device__ __forceinline__ void few_dx(const float* __restrict__ dg, const float* __restrict__ du,
                                       const T* __restrict__ wg, const T* __restrict__ wu,
                                       T* __restrict__ dx, int row, int nrows, int hidden,
                                       int output, int k0) {
  const int lane = threadIdx.x & 31;
  float acc[kR][kDxRows] = {};
  for (int n = lane * kVec; n < output; n += 32 * kVec) {  // kVec divides output
    Raw<T, kVec> a[kDxRows], b[kDxRows];
#pragma unroll
    for (int j = 0; j < kDxRows; ++j) {
      const long long at = static_cast<long long>(min(k0 + j, hidden - 1)) * output + n;
      a[j].load(wg + at);
      b[j].load(wu + at);
    }
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const long long at = static_cast<long long>(row + min(i, nrows - 1)) * output + n;
      float g[kVec], u[kVec];
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        g[v] = __ldg(dg + at + v);
        u[v] = __ldg(du + at + v);
      }
#pragma unroll
      for (int j = 0; j < kDxRows; ++j) {
        float wa[kVec], wb[kVec];
        a[j].get(wa);
        b[j].get(wb);
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
          acc[i][j] = fmaf(g[v], wa[v], acc[i][j]);
          acc[i][j] = fmaf(u[v], wb[v], acc[i][j]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kR; ++i) {
#pragma unroll
    for (int j = 0; j < kDxRows; ++j) {
      float s = acc[i][j];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      if (lane == i * kDxRows + j && i < nrows && k0 + j < hidden) {
        dx[static_cast<long long>(row + i) * hidden + k0 + j] = from_f32<T>(s);
      }
    }
  }
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kFewThreads) gated_few_dx_kernel(
    const float* __restrict__ dg, const float* __restrict__ du, const T* __restrict__ wg,
    const T* __restrict__ wu, const int32_t* __restrict__ offsets, T* __restrict__ dx, int rows,
    int experts, int hidden, int output) {
  follow_previous();
  const int row = blockIdx.y;
  const int e = expert_of(offsets, row, rows, experts);
  if (e == experts) return;
  const int2 s = segment(offsets, e, rows);
  if ((row - s.x) % kFewRows != 0) return;
  const int k0 = (blockIdx.x * kFewWarps + (threadIdx.x >> 5)) * kDxRows;
  if (k0 >= hidden) return;
  const long long at = static_cast<long long>(e) * hidden * output;
  const int nrows = min(kFewRows, s.y - row);
  if (nrows == 1) {
    few_dx<T, kVec, 1>(dg, du, wg + at, wu + at, dx, row, nrows, hidden, output, k0);
  } else {
    few_dx<T, kVec, kFewRows>(dg, du, wg + at, wu + at, dx, row, nrows, hidden, output, k0);
  }
}

// The weight gradients are written once, zeros for experts without rows: bound
// by those bytes (128 experts, 4096 x 1408, bfloat16: 2.95 GB in 404 us, 7.3 TB/s).
// dW[e][k, n] = sum_r x[r, k] d[r, n]; a warp takes kDwRows
// weight rows of 32 vectors of columns, both gradients.
template <int kVec>
constexpr int kDwRows = kVec == 1 ? 16 : 4;  // 32 and 64 sums per thread

template <typename T>
__device__ __forceinline__ void zero_range(T* p, T* end) {  // by the whole block
  if (p >= end) return;
  const auto up = [](T* q, uintptr_t d) {
    return reinterpret_cast<T*>((reinterpret_cast<uintptr_t>(q) + d) & ~static_cast<uintptr_t>(15));
  };
  T* mid = up(p, 15) < end ? up(p, 15) : end;
  T* last = up(end, 0) > mid ? up(end, 0) : mid;
  for (T* q = p + threadIdx.x; q < mid; q += kFewThreads) *q = from_f32<T>(0.0f);
  for (auto* q = reinterpret_cast<uint4*>(mid) + threadIdx.x; q < reinterpret_cast<uint4*>(last);
       q += kFewThreads) {
    *q = make_uint4(0u, 0u, 0u, 0u);
  }
  for (T* q = last + threadIdx.x; q < end; q += kFewThreads) *q = from_f32<T>(0.0f);
}

template <typename T, int kVec>
__global__ void __launch_bounds__(kFewThreads) gated_few_dw_kernel(
    const T* __restrict__ x, const float* __restrict__ dg, const float* __restrict__ du,
    const int32_t* __restrict__ offsets, T* __restrict__ dwg, T* __restrict__ dwu, int rows,
    int hidden, int output, int k_blocks, long long part) {
  follow_previous();
  // Experts and blocks of k share the y axis of the grid; part: a block's share of
  // an expert's elements.
  const int e = blockIdx.y / k_blocks;
  const int lane = threadIdx.x & 31;
  const int n = (blockIdx.x * 32 + lane) * kVec;
  const int kb = blockIdx.y - e * k_blocks;
  const int k0 = (kb * kFewWarps + (threadIdx.x >> 5)) * kDwRows<kVec>;
  const int2 s = segment(offsets, e, rows);
  if (kVec == 1 && s.x >= s.y) {
    // An idle expert's gradients are one run of zeros each: whole granules, also
    // where rows start anywhere.
    const long long size = static_cast<long long>(hidden) * output;
    const long long from = part * (kb * gridDim.x + blockIdx.x);
    const long long to = from + part < size ? from + part : size;
    zero_range(dwg + e * size + from, dwg + e * size + to);
    zero_range(dwu + e * size + from, dwu + e * size + to);
    return;
  }
  if (k0 >= hidden || n >= output) return;
  float g[kDwRows<kVec>][kVec] = {}, u[kDwRows<kVec>][kVec] = {};
  for (int r = s.x; r < s.y; ++r) {
    float a[kVec], b[kVec];
    const long long at = static_cast<long long>(r) * output + n;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
      a[v] = __ldg(dg + at + v);
      b[v] = __ldg(du + at + v);
    }
#pragma unroll
    for (int j = 0; j < kDwRows<kVec>; ++j) {
      const float xv =
          to_f32(__ldg(x + static_cast<long long>(r) * hidden + min(k0 + j, hidden - 1)));
#pragma unroll
      for (int v = 0; v < kVec; ++v) {
        g[j][v] = fmaf(xv, a[v], g[j][v]);
        u[j][v] = fmaf(xv, b[v], u[j][v]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kDwRows<kVec>; ++j) {
    if (k0 + j < hidden) {
      const long long at =
          (static_cast<long long>(e) * hidden + k0 + j) * output + n;
      if constexpr (kVec == 1) {
        dwg[at] = from_f32<T>(g[j][0]);
        dwu[at] = from_f32<T>(u[j][0]);
      } else {
        *reinterpret_cast<uint4*>(dwg + at) = pack16<T>(g[j]);
        *reinterpret_cast<uint4*>(dwu + at) = pack16<T>(u[j]);
      }
    }
  }
}

// ---- operand parts -----------------------------------------------------------------

// Two values as sums of three bfloat16 values each (a in the low halves), exact from
// 2^-110 on, below within 2^-134: each part is what is left, rounded to nearest, so
// that the parts have either sign and the products of them that are left out do not
// lean one way (cut off instead, the parts have the value's sign, and what is left out
// of a product reaches 2^-21 of it, always towards zero).
__device__ __forceinline__ void split3(float a, float b, uint32_t (&w)[3]) {
  w[0] = pack_bf16x2(a, b);
  if ((((w[0] & 0x7F807F80u) + 0x00800080u) & 0x80008000u) != 0) {
    // Not finite, or rounded up to infinity: the first part cuts off. Infinity and NaN
    // stay in it.
    auto first = [](float v) {
      const uint32_t bits = __float_as_uint(v);
      return (bits & 0xFFFF0000u) | ((bits & 0x7FFFFFFFu) > 0x7F800000u ? 0x400000u : 0u);
    };
    w[0] = (first(a) >> 16) | first(b);
  }
  auto rest = [](float v, uint32_t part) {
    return (part & 0x7F800000u) == 0x7F800000u ? 0.0f : v - __uint_as_float(part);
  };
  a = rest(a, w[0] << 16);
  b = rest(b, w[0] & 0xFFFF0000u);
  w[1] = pack_bf16x2(a, b);
  w[2] = pack_bf16x2(a - __uint_as_float(w[1] << 16), b - __uint_as_float(w[1] & 0xFFFF0000u));
}

// Eight values as one 16-byte store per part; planes `plane` elements apart. One
// part: rounded to nearest. Two: what the first leaves, rounded again (16
// significand bits). Three: the FP32 value (split3).
template <int kTerms>
__device__ __forceinline__ void store_parts(__nv_bfloat16* dst, long long plane,
                                            const float (&v)[8]) {
  if constexpr (kTerms == 1) {
    *reinterpret_cast<uint4*>(dst) = pack16<__nv_bfloat16>(v);
  } else if constexpr (kTerms == 2) {
    float hi[8], lo[8];
    const uint4 top = pack16<__nv_bfloat16>(v);
    unpack16<__nv_bfloat16>(top, hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = isfinite(hi[i]) ? v[i] - hi[i] : 0.0f;
    }
    *reinterpret_cast<uint4*>(dst) = top;
    *reinterpret_cast<uint4*>(dst + plane) = pack16<__nv_bfloat16>(lo);
  } else {
    uint32_t w[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) split3(v[2 * i], v[2 * i + 1], w[i]);
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      *reinterpret_cast<uint4*>(dst + q * plane) = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
    }
  }
}

constexpr int kPackThreads = 256;

// Eight values as they lie in memory.
template <typename T>
struct Raw8 {
  static constexpr int kPer = 16 / sizeof(T), kPieces = 8 / kPer;
  uint4 w[kPieces];
  __device__ __forceinline__ void load_aligned(const T* p) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) w[j] = __ldg(reinterpret_cast<const uint4*>(p) + j);
  }
  __device__ __forceinline__ void load(const T* p, const T* begin, const T* end, int count) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) w[j] = load16<T>(p + kPer * j, begin, end, count - kPer * j);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) unpack16<T>(w[j], v + kPer * j);
  }
};

// One thread packs eight columns: bound by the bytes (FP32: 4 read, 6 written
// per element; 6.2 TB/s at 64 x 1024 x 1024). Runs only for FP32 operands and
// for row strides that are no multiple of 16 bytes, which TMA cannot read.
// The operands of a call are packed by one launch.
template <typename T, int kTerms>
__global__ void __launch_bounds__(kPackThreads) pack_terms_kernel(const PackJobs jobs) {
  follow_previous();
  const int index = static_cast<int>(blockIdx.x) * kPackThreads + static_cast<int>(threadIdx.x);
  const int step = static_cast<int>(gridDim.x) * kPackThreads;
  for (int q = 0; q < jobs.count; ++q) {
    const PackJob& job = jobs.job[q];
    const int groups = job.ld >> 3;
    const long long total = job.rows * groups;
    const long long plane = job.rows * job.ld;
    const T* src = static_cast<const T*>(job.src);
    const T* end = src + job.rows * job.cols;
    const bool vec = (job.cols * sizeof(T)) % 16 == 0;  // such rows are 16-byte aligned
    // A job goes on where the one before it left the grid. Row and group of an
    // item are carried along: a division for each costs more than its bytes.
    const int first = index < job.shift ? index - job.shift + step : index - job.shift;
    int c = first % groups;
    long long r = first / groups;
    for (long long i = first; i < total; i += step) {
      const T* p = src + r * job.cols + 8 * c;
      const int count = job.cols - 8 * c;
      Raw8<T> raw;
      if (vec && count >= 8) raw.load_aligned(p);
      else raw.load(p, src, end, count);
      __nv_bfloat16* dst = job.dst + 8 * i;  // ld is 8 * groups
      if constexpr (sizeof(T) == 2 && kTerms == 1) {
        *reinterpret_cast<uint4*>(dst) = raw.w[0];
      } else {
        float v[8];
        raw.get(v);
        store_parts<kTerms>(dst, plane, v);
      }
      r += job.step_rows;
      c += job.step_groups;
      if (c >= groups) {
        c -= groups;
        ++r;
      }
    }
  }
}

// ---- pointwise gradient --------------------------------------------------------------
//
// From the saved FP32 products g, u and the incoming dh:
//   dg = dh * u * act'(g), du = dh * act(g).
// Written as the engine's operand parts: for bfloat16 one rounding, which every
// tensor-core operand takes, or two parts (see gradient_parts in block_api.cpp);
// for FP32 three parts (split3). Bound by its bytes.
template <typename T, int kTerms, bool kVec>
__global__ void __launch_bounds__(kPackThreads) gated_pointwise_backward_kernel(
    const float* __restrict__ gate_up, const T* __restrict__ dh, __nv_bfloat16* __restrict__ dg,
    __nv_bfloat16* __restrict__ du, int rows, int output, int ld, int activation) {
  follow_previous();
  const int groups = ld >> 3;
  const long long total = static_cast<long long>(rows) * groups;
  const long long plane = static_cast<long long>(rows) * ld;
  for (long long i = static_cast<long long>(blockIdx.x) * kPackThreads + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * kPackThreads) {
    const long long r = total <= INT_MAX ? static_cast<int>(i) / groups : i / groups;
    const int c = static_cast<int>(i - r * groups) << 3;
    const float* pg = gate_up + 2 * r * output + c;
    const float* pu = pg + output;
    const T* pd = dh + r * output + c;
    float g[8], u[8], d[8];
    Raw8<float> rg, ru;
    Raw8<T> rd;
    if (kVec && c + 8 <= output) {
      rg.load_aligned(pg);
      ru.load_aligned(pu);
      rd.load_aligned(pd);
    } else {
      const float* end = gate_up + 2LL * rows * output;
      rg.load(pg, gate_up, end, output - c);
      ru.load(pu, gate_up, end, output - c);
      rd.load(pd, dh, dh + static_cast<long long>(rows) * output, output - c);
    }
    rg.get(g);
    ru.get(u);
    rd.get(d);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float slope;
      const float a = activate<T>(activation, g[j], &slope);
      g[j] = d[j] * u[j] * slope;
      u[j] = d[j] * a;
    }
    store_parts<kTerms>(dg + r * ld + c, plane, g);
    store_parts<kTerms>(du + r * ld + c, plane, u);
  }
}

// The same for the few-row forms, in FP32.
template <typename T>
__global__ void __launch_bounds__(kPackThreads) gated_pointwise_backward_f32_kernel(
    const float* __restrict__ gate_up, const T* __restrict__ dh, float* __restrict__ dg,
    float* __restrict__ du, long long total, int output, int activation) {
  follow_previous();
  for (long long i = static_cast<long long>(blockIdx.x) * kPackThreads + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * kPackThreads) {
    const long long r = total <= INT_MAX ? static_cast<int>(i) / output : i / output;
    const long long at = i + r * output;  // gate_up rows are 2 * output long
    float slope;
    const float a = activate<T>(activation, __ldg(gate_up + at), &slope);
    const float d = to_f32(__ldg(dh + i));
    dg[i] = d * __ldg(gate_up + at + output) * slope;
    du[i] = d * a;
  }
}

int pack_blocks(long long total) {
  const long long want = (total + kPackThreads - 1) / kPackThreads;
  const long long cap = 8LL * sm_count();
  return static_cast<int>(want < cap ? want : cap);
}

}  // namespace

cudaError_t launch_gated_few(const void* x, const void* wg, const void* wu,
                             const int32_t* offsets, void* h, float* gate_up, int rows,
                             int experts, int hidden, int output, Activation activation,
                             Dtype dtype, cudaStream_t stream) {
  const int act = static_cast<int>(activation);
  return dtype == Dtype::kBf16 ? few<__nv_bfloat16>(x, wg, wu, offsets, h, gate_up, rows, experts,
                                                    hidden, output, act, stream)
                               : few<float>(x, wg, wu, offsets, h, gate_up, rows, experts, hidden,
                                            output, act, stream);
}

cudaError_t launch_pack_terms(PackJobs jobs, Dtype dtype, cudaStream_t stream) {
  long long total = 0;
  for (int q = 0; q < jobs.count; ++q) total += jobs.job[q].rows * (jobs.job[q].ld >> 3);
  const int blocks = pack_blocks(total);
  if (blocks == 0) return cudaSuccess;
  const int step = blocks * kPackThreads;
  long long before = 0;
  for (int q = 0; q < jobs.count; ++q) {
    PackJob& job = jobs.job[q];
    const int groups = job.ld >> 3;
    job.shift = static_cast<int>(before % step);
    job.step_rows = step / groups;
    job.step_groups = step % groups;
    before += job.rows * groups;
  }
  auto* kernel = dtype == Dtype::kBf16 ? pack_terms_kernel<__nv_bfloat16, 1>
                                       : pack_terms_kernel<float, 3>;
  return launch_following(kernel, dim3(blocks), kPackThreads, 0, 0, stream, jobs);
}

cudaError_t launch_gated_pointwise_backward(const float* gate_up, const void* dh,
                                            __nv_bfloat16* dg, __nv_bfloat16* du, int rows,
                                            int output, int ld, int parts, Activation activation,
                                            Dtype dtype, cudaStream_t stream) {
  const int blocks = pack_blocks(static_cast<long long>(rows) * (ld >> 3));
  if (blocks == 0) return cudaSuccess;
  const int act = static_cast<int>(activation);
  const bool vec = output % 8 == 0 && aligned_to(gate_up, 16) && aligned_to(dh, 16);
  if (dtype == Dtype::kBf16) {
    auto* kernel = parts == 2
                       ? (vec ? gated_pointwise_backward_kernel<__nv_bfloat16, 2, true>
                              : gated_pointwise_backward_kernel<__nv_bfloat16, 2, false>)
                       : (vec ? gated_pointwise_backward_kernel<__nv_bfloat16, 1, true>
                              : gated_pointwise_backward_kernel<__nv_bfloat16, 1, false>);
    return launch_following(kernel, dim3(blocks), kPackThreads, 0, 0, stream, gate_up,
                            static_cast<const __nv_bfloat16*>(dh), dg, du, rows, output, ld, act);
  }
  auto* kernel = vec ? gated_pointwise_backward_kernel<float, 3, true>
                     : gated_pointwise_backward_kernel<float, 3, false>;
  return launch_following(kernel, dim3(blocks), kPackThreads, 0, 0, stream, gate_up,
                          static_cast<const float*>(dh), dg, du, rows, output, ld, act);
}

cudaError_t launch_gated_pointwise_backward_f32(const float* gate_up, const void* dh, float* dg,
                                                float* du, int rows, int output,
                                                Activation activation, Dtype dtype,
                                                cudaStream_t stream) {
  const long long total = static_cast<long long>(rows) * output;
  const int blocks = pack_blocks(total);
  const int act = static_cast<int>(activation);
  if (dtype == Dtype::kBf16) {
    return launch_following(gated_pointwise_backward_f32_kernel<__nv_bfloat16>, dim3(blocks),
                            kPackThreads, 0, 0, stream, gate_up,
                            static_cast<const __nv_bfloat16*>(dh), dg, du, total, output, act);
  }
  return launch_following(gated_pointwise_backward_f32_kernel<float>, dim3(blocks), kPackThreads, 0,
                          0, stream, gate_up, static_cast<const float*>(dh), dg, du, total, output,
                          act);
}

namespace {

template <typename T>
cudaError_t few_dx_launch(const float* dg, const float* du, const void* wg, const void* wu,
                          const int32_t* offsets, void* dx, int rows, int experts, int hidden,
                          int output, cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  const bool vec = output % kVec == 0 && aligned_to(wg, 16) && aligned_to(wu, 16);
  auto* kernel = vec ? gated_few_dx_kernel<T, kVec> : gated_few_dx_kernel<T, 1>;
  return launch_following(kernel, dim3(ceil_div(hidden, kFewWarps * kDxRows), rows), kFewThreads, 0,
                          0, stream, dg, du, static_cast<const T*>(wg), static_cast<const T*>(wu),
                          offsets, static_cast<T*>(dx), rows, experts, hidden, output);
}

template <typename T>
cudaError_t few_dw_launch(const void* x, const float* dg, const float* du, const int32_t* offsets,
                          void* dwg, void* dwu, int rows, int experts, int hidden, int output,
                          cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  const bool vec = output % kVec == 0 && aligned_to(dwg, 16) && aligned_to(dwu, 16);
  const int k_blocks = ceil_div(hidden, kFewWarps * (vec ? kDwRows<kVec> : kDwRows<1>));
  auto* kernel = vec ? gated_few_dw_kernel<T, kVec> : gated_few_dw_kernel<T, 1>;
  const int columns = ceil_div(output, 32 * (vec ? kVec : 1));
  const long long blocks = static_cast<long long>(columns) * k_blocks;
  const long long part = (static_cast<long long>(hidden) * output + blocks - 1) / blocks;
  // The y axis holds 65535 blocks: experts in slices that fit.
  const int slice = k_blocks < 65535 ? 65535 / k_blocks : 0;
  if (slice == 0) return cudaErrorInvalidConfiguration;
  for (int e = 0; e < experts; e += slice) {
    const int count = experts - e < slice ? experts - e : slice;
    const long long at = static_cast<long long>(e) * hidden * output;
    const cudaError_t err = launch_following(
        kernel, dim3(columns, count * k_blocks), kFewThreads, 0, 0, stream,
        static_cast<const T*>(x), dg, du, offsets + e, static_cast<T*>(dwg) + at,
        static_cast<T*>(dwu) + at, rows, hidden, output, k_blocks, part);
    if (err != cudaSuccess) return err;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_gated_few_dx(const float* dg, const float* du, const void* wg, const void* wu,
                                const int32_t* offsets, void* dx, int rows, int experts,
                                int hidden, int output, Dtype dtype, cudaStream_t stream) {
  return dtype == Dtype::kBf16
             ? few_dx_launch<__nv_bfloat16>(dg, du, wg, wu, offsets, dx, rows, experts, hidden,
                                            output, stream)
             : few_dx_launch<float>(dg, du, wg, wu, offsets, dx, rows, experts, hidden, output,
                                    stream);
}

cudaError_t launch_gated_few_dw(const void* x, const float* dg, const float* du,
                                const int32_t* offsets, void* dwg, void* dwu, int rows,
                                int experts, int hidden, int output, Dtype dtype,
                                cudaStream_t stream) {
  return dtype == Dtype::kBf16
             ? few_dw_launch<__nv_bfloat16>(x, dg, du, offsets, dwg, dwu, rows, experts, hidden,
                                            output, stream)
             : few_dw_launch<float>(x, dg, du, offsets, dwg, dwu, rows, experts, hidden, output,
                                    stream);
}

}  // namespace rrb

// 8-bit integer operands of the grouped product: quantisation of rows and of
// expert weights, and the product for a few rows (more rows run on the
// tensor-core engine, expert_gemm.cu).
//
//   rows     top = max |x|, q = rint(x * (127 / top)), scale = top / 127
//   weights  the same for every output channel W[e][:, n], written K-major
//   product  y[r, n] = (sum_k xq[r, k] wq[e][n, k]) * x_scale[r] * w_scale[e, n]
//
// The integer sum is exact. A row or channel whose largest magnitude is below
// 2^-120 (where 127 / top overflows) counts as zero: q = 0, scale = 0. With an
// infinity or a NaN in it the scale is that infinity or NaN and its products
// come out NaN.
#include "expert_block.cuh"

namespace rrb {
namespace {

constexpr uint32_t kTinyBits = 0x03800000u;  // 2^-120

struct Scale {
  float scale, inverse;
};

// From the bit pattern of the largest magnitude (integer order equals float
// order for magnitudes, with NaN on top).
__device__ __forceinline__ Scale scale_of(uint32_t top_bits) {
  if (top_bits < kTinyBits) return {0.0f, 0.0f};
  const float top = __uint_as_float(top_bits);
  return {__fdiv_rn(top, 127.0f), __fdiv_rn(127.0f, top)};
}

__device__ __forceinline__ int quantize(float v, float inverse) {
  // NaN (0 * inf of a row with an infinity) converts to 0.
  return max(-127, min(127, __float2int_rn(__fmul_rn(v, inverse))));
}

__device__ __forceinline__ uint32_t pack_i8x4(int a, int b, int c, int d) {
  return (a & 0xFF) | ((b & 0xFF) << 8) | ((c & 0xFF) << 16) | (static_cast<uint32_t>(d) << 24);
}

// ---- rows ------------------------------------------------------------------------
//
// Bound by the bytes in and out (131072 x 4096, bfloat16: 230 us, 7.0 TB/s; rows of
// 1181, which no vector load fits: 27040 in 31 us, 3.1 TB/s, against 34 and more with
// a warp that shifts 16-byte granules). Long or unaligned rows take one block each: the
// row is read once into registers (up to kHeld steps per thread; what is longer
// is read again, from L2).

constexpr int kRowThreads = 128;
constexpr int kHeld = 4;

template <typename T, bool kVec>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(
    const T* __restrict__ x, int8_t* __restrict__ xq, float* __restrict__ x_scale, int cols,
    int ld) {
  constexpr int kPer = kVec ? 16 / sizeof(T) : 4;  // values per thread and step
  __shared__ uint32_t tops[kRowThreads / 32];
  follow_previous();
  const long long row = blockIdx.x;
  const T* src = x + row * cols;
  int8_t* dst = xq + row * ld;
  const int steps = ld / kPer;
  auto load = [&](int i, float* v) {
    const int c = i * kPer;
    if constexpr (kVec) {
      if (c < cols) {  // cols is a multiple of kPer
        unpack16<T>(__ldg(reinterpret_cast<const uint4*>(src) + i), v);
        return;
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = 0.0f;
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[j] = c + j < cols ? to_f32(__ldg(src + c + j)) : 0.0f;
    }
  };
  uint32_t top = 0;
  float held[kHeld][kPer];
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const int i = threadIdx.x + h * kRowThreads;
    if (i < steps) {
      load(i, held[h]);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        top = max(top, __float_as_uint(held[h][j]) & 0x7FFFFFFFu);
      }
    }
  }
  for (int i = threadIdx.x + kHeld * kRowThreads; i < steps; i += kRowThreads) {
    float v[kPer];
    load(i, v);
#pragma unroll
    for (int j = 0; j < kPer; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) top = max(top, tops[w]);
  const Scale s = scale_of(top);
  if (threadIdx.x == 0) x_scale[row] = s.scale;
  auto store = [&](int i, const float* v) {
    uint32_t w[kPer / 4];
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) {
      w[j] = pack_i8x4(quantize(v[4 * j], s.inverse), quantize(v[4 * j + 1], s.inverse),
                       quantize(v[4 * j + 2], s.inverse), quantize(v[4 * j + 3], s.inverse));
    }
    if constexpr (kPer == 8) {
      reinterpret_cast<uint2*>(dst)[i] = make_uint2(w[0], w[1]);
    } else {
      reinterpret_cast<uint32_t*>(dst)[i] = w[0];
    }
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const int i = threadIdx.x + h * kRowThreads;
    if (i < steps) store(i, held[h]);
  }
  for (int i = threadIdx.x + kHeld * kRowThreads; i < steps; i += kRowThreads) {
    float v[kPer];
    load(i, v);
    store(i, v);
  }
}

// Rows of up to 32 * 16 * kHeld bytes, 16-byte aligned: a warp per row, the row
// held as loaded, no barrier. Rounding adds 1.5 * 2^23, whose sum rounds to the
// nearest integer with ties to even and holds it in its low bits (the
// conversion instruction issues at a quarter of that rate).
constexpr int kRowWarps = 8;

__device__ __forceinline__ uint32_t quantize4(float a, float b, float c, float d, float inverse) {
  constexpr float kRound = 12582912.0f;
  const uint32_t ia = __float_as_uint(__fadd_rn(__fmul_rn(a, inverse), kRound));
  const uint32_t ib = __float_as_uint(__fadd_rn(__fmul_rn(b, inverse), kRound));
  const uint32_t ic = __float_as_uint(__fadd_rn(__fmul_rn(c, inverse), kRound));
  const uint32_t id = __float_as_uint(__fadd_rn(__fmul_rn(d, inverse), kRound));
  return __byte_perm(__byte_perm(ia, ib, 0x0040), __byte_perm(ic, id, 0x0040), 0x5410);
}

template <typename T, int kWarpHeld>
__global__ void __launch_bounds__(32 * kRowWarps) quantize_rows_warp_kernel(
    const T* __restrict__ x, int8_t* __restrict__ xq, float* __restrict__ x_scale, int rows,
    int cols, int ld) {
  constexpr int kPer = 16 / sizeof(T);
  follow_previous();
  const int lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * cols);
  const int chunks = cols / kPer, places = ld / kPer;
  uint4 held[kWarpHeld];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < kWarpHeld; ++h) {
    const int i = lane + 32 * h;
    held[h] = i < chunks ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int h = 0; h < kWarpHeld; ++h) {
    const uint32_t w[4] = {held[h].x, held[h].y, held[h].z, held[h].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // Magnitudes order as integers, also two bfloat16 at a time.
      if constexpr (sizeof(T) == 2) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
      else top = max(top, w[j] & 0x7FFFFFFFu);
    }
  }
  if constexpr (sizeof(T) == 2) top = max(top & 0xFFFF0000u, top << 16);
  top = __reduce_max_sync(0xffffffffu, top);
  Scale s = scale_of(top);
  if (lane == 0) x_scale[row] = s.scale;
  const bool finite = top < 0x7F800000u;  // otherwise the scale says it: q = 0
  int8_t* dst = xq + row * ld;
#pragma unroll
  for (int h = 0; h < kWarpHeld; ++h) {
    const int i = lane + 32 * h;
    if (i < places) {
      float v[kPer];
      unpack16<T>(held[h], v);
      uint32_t q[kPer / 4];
#pragma unroll
      for (int j = 0; j < kPer / 4; ++j) {
        q[j] = finite ? quantize4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], s.inverse)
                      : 0u;
      }
      if constexpr (kPer == 8) reinterpret_cast<uint2*>(dst)[i] = make_uint2(q[0], q[1]);
      else reinterpret_cast<uint32_t*>(dst)[i] = q[0];
    }
  }
}

template <typename T>
cudaError_t quantize_rows(const T* x, int8_t* xq, float* x_scale, int rows, int cols, int ld,
                          cudaStream_t stream) {
  constexpr int kPer = 16 / sizeof(T);
  const bool vec = aligned_to(x, 16) && cols % kPer == 0;
  const int places = ld / kPer;  // 16-byte pieces of a row
  if (vec && places <= 32 * 16) {
    auto* kernel = places <= 32 * 4 ? quantize_rows_warp_kernel<T, 4>
                                    : quantize_rows_warp_kernel<T, 16>;
    return launch_following(kernel, dim3(ceil_div(rows, kRowWarps)), 32 * kRowWarps, 0, 0, stream,
                            x, xq, x_scale, rows, cols, ld);
  }
  auto* kernel = vec ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>;
  return launch_following(kernel, dim3(rows), kRowThreads, 0, 0, stream, x, xq, x_scale, cols, ld);
}

// ---- weights -----------------------------------------------------------------------
//
// W[e] is [hidden][output] and wq[e] is [output][ld]: a block takes 64
// channels of one expert, finds their scales in one pass over K and transposes
// 64 x 64 tiles through shared memory in a second. Done once per weight set (128 x 4096
// x 1408, bfloat16: 1.2 ms; the second pass reads from DRAM again).

constexpr int kChan = 64;
constexpr int kWeightThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kWeightThreads) quantize_weights_kernel(
    const T* __restrict__ w, int8_t* __restrict__ wq, float* __restrict__ w_scale, int hidden,
    int output, int ld) {
  __shared__ uint32_t tops[kWeightThreads / kChan][kChan];
  __shared__ float inverse[kChan];
  __shared__ __align__(16) int8_t tile[kChan][kChan + 16];
  const int e = blockIdx.y;
  const int n0 = blockIdx.x * kChan;
  const int c = threadIdx.x % kChan;
  const int g = threadIdx.x / kChan;
  constexpr int kGroups = kWeightThreads / kChan;
  const T* src = w + static_cast<long long>(e) * hidden * output;
  const bool in = n0 + c < output;
  uint32_t top = 0;
  if (in) {
    for (int k = g; k < hidden; k += kGroups) {
      const float v = to_f32(__ldg(src + static_cast<long long>(k) * output + n0 + c));
      top = max(top, __float_as_uint(v) & 0x7FFFFFFFu);
    }
  }
  tops[g][c] = top;
  __syncthreads();
  if (threadIdx.x < kChan) {
#pragma unroll
    for (int i = 1; i < kGroups; ++i) top = max(top, tops[i][c]);
    const Scale s = scale_of(top);
    inverse[c] = s.inverse;
    if (in) w_scale[static_cast<long long>(e) * output + n0 + c] = s.scale;
  }
  __syncthreads();
  for (int k0 = 0; k0 < ld; k0 += kChan) {
    for (int i = g; i < kChan; i += kGroups) {
      const int k = k0 + i;
      const float v =
          in && k < hidden ? to_f32(__ldg(src + static_cast<long long>(k) * output + n0 + c))
                           : 0.0f;
      tile[c][i] = static_cast<int8_t>(quantize(v, inverse[c]));
    }
    __syncthreads();
    const int ch = threadIdx.x >> 2, q = threadIdx.x & 3;  // 16 bytes each
    if (n0 + ch < output && k0 + 16 * q < ld) {
      *reinterpret_cast<uint4*>(wq + (static_cast<long long>(e) * output + n0 + ch) * ld + k0 +
                                16 * q) = *reinterpret_cast<const uint4*>(&tile[ch][16 * q]);
    }
    __syncthreads();
  }
}

// ---- few rows ------------------------------------------------------------------------
//
// Bound by reading the weights of the experts that have rows, K bytes per
// channel, once: a warp takes kCols channels of up to kFewRows rows of one
// expert, 16 bytes per lane and channel, four-way integer dot products. (Two rows of
// 128 experts, K=4096, N=1408: 11.5 MB in 3.3 us, of which 2 are its start.)

constexpr int kFewThreads = 256;
constexpr int kCols = 4;
constexpr int kFewRows = 4;

__device__ __forceinline__ int dot16(const int4 a, const int4 b, int acc) {
  acc = __dp4a(a.x, b.x, acc);
  acc = __dp4a(a.y, b.y, acc);
  acc = __dp4a(a.z, b.z, acc);
  return __dp4a(a.w, b.w, acc);
}

template <typename T, int kR>
__device__ __forceinline__ void int8_few_rows(const int8_t* __restrict__ xq,
                                              const float* __restrict__ x_scale,
                                              const int8_t* __restrict__ wq,
                                              const float* __restrict__ w_scale,
                                              T* __restrict__ y, int row, int nrows, int ld,
                                              int output, int n0) {
  const int lane = threadIdx.x & 31;
  const int chunks = ld >> 4;
  int acc[kR][kCols] = {};
  const int4* px[kR];
  const int4* pw[kCols];
#pragma unroll
  for (int i = 0; i < kR; ++i) {
    px[i] = reinterpret_cast<const int4*>(xq + static_cast<long long>(row + min(i, nrows - 1)) *
                                                   ld);
  }
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    pw[j] = reinterpret_cast<const int4*>(wq + static_cast<long long>(min(n0 + j, output - 1)) *
                                                   ld);
  }
#pragma unroll 2
  for (int c = lane; c < chunks; c += 32) {
    int4 w[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) w[j] = __ldg(pw[j] + c);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int4 v = __ldg(px[i] + c);
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[i][j] = dot16(v, w[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < kR; ++i) {
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int sum = __reduce_add_sync(0xffffffffu, acc[i][j]);
      if (lane == i * kCols + j && i < nrows && n0 + j < output) {
        y[static_cast<long long>(row + i) * output + n0 + j] = from_f32<T>(
            static_cast<float>(sum) * __ldg(x_scale + row + i) * __ldg(w_scale + n0 + j));
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kFewThreads) int8_few_kernel(
    const int8_t* __restrict__ xq, const float* __restrict__ x_scale,
    const int8_t* __restrict__ wq, const float* __restrict__ w_scale,
    const int32_t* __restrict__ offsets, T* __restrict__ y, int rows, int experts, int ld,
    int output) {
  __shared__ int owner;
  follow_previous();
  if (threadIdx.x == 0) owner = experts;
  __syncthreads();
  const int row = blockIdx.y;
  for (int e = threadIdx.x; e < experts; e += kFewThreads) {
    const int2 s = segment(offsets, e, rows);
    if (s.x <= row && row < s.y) atomicMin(&owner, e);
  }
  __syncthreads();
  const int e = owner;
  if (e == experts) return;
  const int2 s = segment(offsets, e, rows);
  if ((row - s.x) % kFewRows != 0) return;
  const int nrows = min(kFewRows, s.y - row);
  const int n0 = (blockIdx.x * (kFewThreads / 32) + (threadIdx.x >> 5)) * kCols;
  if (n0 >= output) return;
  const int8_t* we = wq + static_cast<long long>(e) * output * ld;
  const float* se = w_scale + static_cast<long long>(e) * output;
  if (nrows == 1) {
    int8_few_rows<T, 1>(xq, x_scale, we, se, y, row, nrows, ld, output, n0);
  } else {
    int8_few_rows<T, kFewRows>(xq, x_scale, we, se, y, row, nrows, ld, output, n0);
  }
}

}  // namespace

cudaError_t launch_quantize_rows_int8(const void* x, int8_t* xq, float* x_scale, int rows,
                                      int cols, int ld, Dtype dtype, cudaStream_t stream) {
  return dtype == Dtype::kBf16
             ? quantize_rows(static_cast<const __nv_bfloat16*>(x), xq, x_scale, rows, cols, ld,
                             stream)
             : quantize_rows(static_cast<const float*>(x), xq, x_scale, rows, cols, ld, stream);
}

cudaError_t launch_quantize_expert_weights_int8(const void* w, int8_t* wq, float* w_scale,
                                                int experts, int hidden, int output, int ld,
                                                Dtype dtype, cudaStream_t stream) {
  const dim3 grid(ceil_div(output, kChan), experts);
  if (dtype == Dtype::kBf16) {
    quantize_weights_kernel<<<grid, kWeightThreads, 0, stream>>>(
        static_cast<const __nv_bfloat16*>(w), wq, w_scale, hidden, output, ld);
  } else {
    quantize_weights_kernel<<<grid, kWeightThreads, 0, stream>>>(static_cast<const float*>(w), wq,
                                                                 w_scale, hidden, output, ld);
  }
  note_launch();
  return cudaGetLastError();
}

cudaError_t launch_int8_few(const int8_t* xq, const float* x_scale, const int8_t* wq,
                            const float* w_scale, const int32_t* offsets, void* y, int rows,
                            int experts, int ld, int output, Dtype dtype, cudaStream_t stream) {
  const dim3 grid(ceil_div(output, kCols * (kFewThreads / 32)), rows);
  if (dtype == Dtype::kBf16) {
    return launch_following(int8_few_kernel<__nv_bfloat16>, grid, kFewThreads, 0, 0, stream, xq,
                            x_scale, wq, w_scale, offsets, static_cast<__nv_bfloat16*>(y), rows,
                            experts, ld, output);
  }
  return launch_following(int8_few_kernel<float>, grid, kFewThreads, 0, 0, stream, xq, x_scale, wq,
                          w_scale, offsets, static_cast<float*>(y), rows, experts, ld, output);
}

}  // namespace rrb

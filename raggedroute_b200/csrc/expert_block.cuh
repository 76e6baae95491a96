// Internal interface of the expert-block operators: the gated expert
// projection and its gradients (expert_gemm.cu, gated.cu), the 8-bit integer
// grouped product (expert_gemm.cu, int8.cu) and the weighted combine with the
// norms, gate and residual around the block (unpermute_norm.cu). Launchers
// enqueue on the stream and return the launch status, as in common.cuh.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace rrb {

// Values of RR_DTYPE_* and RR_ACTIVATION_* in the C ABI.
enum class Dtype : int { kFp32 = 0, kBf16 = 2 };
enum class Activation : int { kSilu = 0, kGeluTanh = 1, kRelu = 2 };

inline std::size_t dtype_bytes(Dtype t) { return t == Dtype::kBf16 ? 2 : 4; }

// ---- launches one behind another -----------------------------------------------
//
// A kernel of a few microseconds costs as much again to start. Kernels launched
// with launch_following() are set up and placed on the SMs while the kernel before
// them in the stream still runs; every block calls follow_previous() before it
// touches global memory, which waits until that kernel (whatever it is) has ended
// and its writes are visible. Only then may the next kernel start the same way, so
// at most one waits. Back to back, K=4096, N=1408, one token: unpermute_norm 3.6
// against 6.2 us, quantize_rows_int8 and grouped_gemm_int8 5.9 against 10.2.

__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void follow_previous() {
  wait_for_previous();
  let_next_start();
}

template <typename... P, typename... A>
cudaError_t launch_following(void (*kernel)(P...), dim3 grid, dim3 block, std::size_t smem,
                             int cluster, cudaStream_t stream, const A&... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return e;
  }
  note_launch();
  return cudaSuccess;
}

// ---- element conversions and activations ------------------------------------

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(v);
  else return v;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(v);
  else return v;
}

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// 16 bytes of T as floats: 8 bfloat16 or 4 float values.
template <typename T>
__device__ __forceinline__ void unpack16(const uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      f[i] = __uint_as_float(w[i]);
    }
  }
}

// Bytes skip to skip + 15 of two 16-byte granules (skip < 16, a multiple of
// sizeof(T)); values from the `count`th on become zero.
template <typename T>
__device__ __forceinline__ uint4 shift16(const uint4 a, const uint4 b, uint32_t skip, int count) {
  constexpr int kPer = 4 / sizeof(T);  // values in a word
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  const bool two = skip & 8u, one = skip & 4u;
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = two ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = one ? w[i + 1] : w[i];
  if constexpr (sizeof(T) == 2) {
    const uint32_t bits = (skip & 3u) * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
  }
  if (count < 4 * kPer) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int left = count - kPer * i;
      w[i] = left >= kPer ? w[i] : (left > 0 ? w[i] & 0xFFFFu : 0u);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A granule at `at` of which only the values in [begin, end) exist; the others
// read as zero.
template <typename T>
__device__ __forceinline__ uint4 part16(uintptr_t at, const T* begin, const T* end) {
  uint32_t w[4];
  auto value = [&](int byte) -> uint32_t {
    const T* p = reinterpret_cast<const T*>(at + byte);
    if (p < begin || p >= end) return 0u;
    if constexpr (sizeof(T) == 2) return __ldg(reinterpret_cast<const unsigned short*>(p));
    else return __ldg(reinterpret_cast<const unsigned*>(p));
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = value(4 * i);
    if constexpr (sizeof(T) == 2) w[i] |= value(4 * i + 2) << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The 16 bytes from p on, wherever p lies: the two granules around them are loaded
// whole (neighbouring threads share them in L1), or, where one reaches past the
// buffer [begin, end), the `count` values that exist.
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p, const T* begin, const T* end, int count) {
  const auto at = reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(15);
  const auto skip = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
  uint4 a, b;
  if (at >= reinterpret_cast<uintptr_t>(begin) && at + 32 <= reinterpret_cast<uintptr_t>(end)) {
    a = __ldg(reinterpret_cast<const uint4*>(at));
    b = __ldg(reinterpret_cast<const uint4*>(at) + 1);
  } else {
    a = part16<T>(at, begin, end);
    b = part16<T>(at + 16, begin, end);
  }
  return shift16<T>(a, b, skip, count);
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* f) {
  if constexpr (sizeof(T) == 2) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  } else {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
}

// Logistic function; exp(-g) = inf gives 0. For FP32 results in full float
// precision; a result that is rounded to bfloat16 takes the hardware's exp and
// division: the exp is off by up to 2 + 1.2 |g| units in the last place (CUDA's bound),
// so within 2^-16 before it leaves the floats' range at |g| = 88.
template <typename T>
__device__ __forceinline__ float sigmoid_f32(float g) {
  if constexpr (sizeof(T) == 2) return __fdividef(1.0f, 1.0f + __expf(-g));
  else return __fdiv_rn(1.0f, 1.0f + expf(-g));
}

constexpr float kGeluC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// act(g) and, if derivative != nullptr, act'(g), for a result of type T.
template <typename T>
__device__ __forceinline__ float activate(int activation, float g, float* derivative = nullptr) {
  if (activation == static_cast<int>(Activation::kSilu)) {
    const float s = sigmoid_f32<T>(g);
    if (derivative != nullptr) *derivative = s * (1.0f + g * (1.0f - s));
    return g * s;
  }
  if (activation == static_cast<int>(Activation::kGeluTanh)) {
    const float t = tanhf(kGeluC * (g + kGeluA * g * g * g));
    if (derivative != nullptr) {
      // t is 1 or -1 long before 32, and the second term zero; beyond, its square would
      // overflow against that zero. NaN passes.
      const float c = g > 32.0f ? 32.0f : (g < -32.0f ? -32.0f : g);
      *derivative = 0.5f * (1.0f + t) +
                    0.5f * c * (1.0f - t * t) * kGeluC * (1.0f + 3.0f * kGeluA * c * c);
    }
    return 0.5f * g * (1.0f + t);
  }
  // ReLU; NaN stays NaN, and the derivative at 0 is 0.
  if (derivative != nullptr) *derivative = g > 0.0f ? 1.0f : 0.0f;
  return g < 0.0f ? 0.0f : g;
}

// Rows of segment e, clipped to [0, rows): offsets come from the device and
// nothing else bounds them.
__device__ __forceinline__ int2 segment(const int32_t* __restrict__ offsets, int e, int rows) {
  const int a = min(max(__ldg(offsets + e), 0), rows);
  const int b = min(max(__ldg(offsets + e + 1), a), rows);
  return make_int2(a, b);
}

// ---- tensor-core engine (expert_gemm.cu) -------------------------------------

// Operands of the engine are bfloat16 in `terms` parts that sum to the value
// (1 for bfloat16 inputs, 3 for FP32), part-major, row strides a multiple of
// 8 elements.
struct GatedOperands {
  const __nv_bfloat16* x = nullptr;   // [terms][rows][ldk]
  const __nv_bfloat16* wg = nullptr;  // [terms][experts][hidden][ldn]
  const __nv_bfloat16* wu = nullptr;
  int ldk = 0;
  int ldn = 0;
  int terms = 1;
};

// h[r] = act(x[r] Wg[e]) * (x[r] Wu[e]), gate_up (optional, [rows][2 output])
// the two products.
cudaError_t launch_gated_gemm(const GatedOperands& in, const int32_t* offsets, void* h,
                              float* gate_up, int rows, int experts, int hidden, int output,
                              Activation activation, Dtype dtype, cudaStream_t stream);
// dx[r] = dg[r] Wg[e]^T + du[r] Wu[e]^T; dg, du are [parts][rows][ldn] (parts =
// terms, or 2 for bfloat16).
cudaError_t launch_gated_dx(const GatedOperands& in, const __nv_bfloat16* dg,
                            const __nv_bfloat16* du, int parts, const int32_t* offsets, void* dx,
                            int rows, int experts, int hidden, int output, Dtype dtype,
                            cudaStream_t stream);
// dwg[e] = x_e^T dg_e, dwu[e] = x_e^T du_e; zero for an empty segment.
cudaError_t launch_gated_dw(const GatedOperands& in, const __nv_bfloat16* dg,
                            const __nv_bfloat16* du, int parts, const int32_t* offsets, void* dwg,
                            void* dwu, int rows, int experts, int hidden, int output, Dtype dtype,
                            cudaStream_t stream);
// y[r, n] = (xq[r] . wq[e][n]) * x_scale[r] * w_scale[e][n]; xq [rows][ld],
// wq [experts][output][ld], ld a multiple of 16.
cudaError_t launch_int8_gemm(const int8_t* xq, const float* x_scale, const int8_t* wq,
                             const float* w_scale, const int32_t* offsets, void* y, int rows,
                             int experts, int ld, int output, Dtype dtype, cudaStream_t stream);

// ---- gated.cu ------------------------------------------------------------------

// Few rows: one pass over the weights of the experts that have rows.
cudaError_t launch_gated_few(const void* x, const void* wg, const void* wu,
                             const int32_t* offsets, void* h, float* gate_up, int rows,
                             int experts, int hidden, int output, Activation activation,
                             Dtype dtype, cudaStream_t stream);
// src [rows][cols] -> dst [terms][rows][ld] bfloat16 (columns past cols zero),
// for up to three tensors in one launch.
struct PackJob {
  const void* src = nullptr;
  __nv_bfloat16* dst = nullptr;
  long long rows = 0;
  int cols = 0;
  int ld = 0;
  int shift = 0, step_rows = 0, step_groups = 0;  // filled in by the launch
};
struct PackJobs {
  PackJob job[3];
  int count = 0;
};
cudaError_t launch_pack_terms(PackJobs jobs, Dtype dtype, cudaStream_t stream);
// dg = dh u act'(g), du = dh act(g) from gate_up [rows][2 output], written as
// [parts][rows][ld] bfloat16 parts.
cudaError_t launch_gated_pointwise_backward(const float* gate_up, const void* dh,
                                            __nv_bfloat16* dg, __nv_bfloat16* du, int rows,
                                            int output, int ld, int parts, Activation activation,
                                            Dtype dtype, cudaStream_t stream);

// The same with dg and du in FP32, [rows][output] each, for the few-row forms.
cudaError_t launch_gated_pointwise_backward_f32(const float* gate_up, const void* dh, float* dg,
                                                float* du, int rows, int output,
                                                Activation activation, Dtype dtype,
                                                cudaStream_t stream);
cudaError_t launch_gated_few_dx(const float* dg, const float* du, const void* wg, const void* wu,
                                const int32_t* offsets, void* dx, int rows, int experts,
                                int hidden, int output, Dtype dtype, cudaStream_t stream);
cudaError_t launch_gated_few_dw(const void* x, const float* dg, const float* du,
                                const int32_t* offsets, void* dwg, void* dwu, int rows,
                                int experts, int hidden, int output, Dtype dtype,
                                cudaStream_t stream);

// ---- int8.cu -------------------------------------------------------------------

cudaError_t launch_quantize_rows_int8(const void* x, int8_t* xq, float* x_scale, int rows,
                                      int cols, int ld, Dtype dtype, cudaStream_t stream);
cudaError_t launch_quantize_expert_weights_int8(const void* w, int8_t* wq, float* w_scale,
                                                int experts, int hidden, int output, int ld,
                                                Dtype dtype, cudaStream_t stream);
cudaError_t launch_int8_few(const int8_t* xq, const float* x_scale, const int8_t* wq,
                            const float* w_scale, const int32_t* offsets, void* y, int rows,
                            int experts, int ld, int output, Dtype dtype, cudaStream_t stream);

// ---- unpermute_norm.cu -----------------------------------------------------------

struct UnpermuteNorm {
  const void* y_permuted = nullptr;        // [tokens * top_k][output]
  const int32_t* route_pos = nullptr;      // [tokens][top_k]
  const float* route_weights = nullptr;    // [tokens][top_k]
  const void* residual = nullptr;          // [tokens][output]
  const float* post_gamma = nullptr;       // [output]; null: no norm before the gate
  const float* gate = nullptr;             // [output]; null: ones
  const float* pre_gamma = nullptr;        // [output]; null: ones
  float eps = 0.0f;
  float residual_scale = 1.0f;
  int tokens = 0;
  int top_k = 0;
  int output = 0;
};
cudaError_t launch_unpermute_norm(const UnpermuteNorm& in, void* residual_out, void* normed,
                                  float* inv_rms, Dtype dtype, cudaStream_t stream);
struct UnpermuteNormGrads {
  const float* inv_rms = nullptr;          // [tokens][2] of the forward pass
  const void* d_residual_out = nullptr;    // null: zero
  const void* d_normed = nullptr;          // null: zero
  void* d_residual = nullptr;
  void* d_y_permuted = nullptr;
  float* d_route_weights = nullptr;
  float* d_post_gamma = nullptr;           // each may be null
  float* d_gate = nullptr;
  float* d_pre_gamma = nullptr;
};
std::size_t unpermute_norm_backward_workspace_bytes(int tokens, int output);
cudaError_t launch_unpermute_norm_backward(const UnpermuteNorm& in, const UnpermuteNormGrads& g,
                                           float* workspace, Dtype dtype, cudaStream_t stream);

}  // namespace rrb

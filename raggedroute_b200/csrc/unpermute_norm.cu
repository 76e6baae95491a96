// The end of an expert block in one pass: weighted unpermute, norm, gate,
// scaled residual, and the norm that opens the next block; and its gradient.
//
//   c  = sum_k w[t,k] * y_permuted[pos[t,k]]      (routes outside the buffer skipped)
//   b  = c * i1 * post,  i1 = 1/sqrt(mean(c^2) + eps)   (b = c without post)
//   r' = scale * residual + gate * b
//   n  = r' * i2 * pre,  i2 = 1/sqrt(mean(r'^2) + eps)  (optional)
//
// Everything is FP32 between loading and the one rounding of each output.
//
// One block holds one token's row in registers, 16 columns per thread, so the
// route rows and the residual are read once and r', n written once: bound by
// those bytes. The two means are block reductions in a fixed order. The
// gradient recomputes c and r' from its inputs instead of reading rounded
// copies, walks tokens with a persistent grid, keeps its share of the three
// column sums (post, gate, pre) in registers and writes it once; a second
// kernel adds the shares in block order. No atomics, so results repeat.
#include "expert_block.cuh"

namespace rrb {
namespace {

constexpr int kElems = 16;  // columns per thread
constexpr int kMaxTopK = 64;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sum over the block in every thread; `parts` holds 32 floats and is free
// again after the next barrier.
__device__ __forceinline__ float block_sum(float v, float* parts) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < warps ? parts[lane] : 0.0f);
}

// kPer consecutive columns.
template <typename T, int kPer>
__device__ __forceinline__ void load_cols(const T* p, float* v) {
  if constexpr (kPer == 1) v[0] = to_f32(__ldg(p));
  else unpack16<T>(__ldg(reinterpret_cast<const uint4*>(p)), v);
}

// The same through an ordinary load, for a row that the kernel may overwrite
// (residual_out may be residual, d_residual may be d_residual_out).
template <typename T, int kPer>
__device__ __forceinline__ void load_own_cols(const T* p, float* v) {
  if constexpr (kPer == 1) v[0] = to_f32(*p);
  else unpack16<T>(*reinterpret_cast<const uint4*>(p), v);
}

template <int kPer>
__device__ __forceinline__ void load_gamma(const float* p, float* v) {
  if constexpr (kPer == 1) {
    v[0] = __ldg(p);
  } else {
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p) + i);
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
  }
}

template <typename T, int kPer>
__device__ __forceinline__ void store_cols(T* p, const float* v) {
  if constexpr (kPer == 1) p[0] = from_f32<T>(v[0]);
  else *reinterpret_cast<uint4*>(p) = pack16<T>(v);
}

// c of this thread's columns of token t (zero past the row's end).
template <typename T, int kPer>
__device__ __forceinline__ void combine_cols(const UnpermuteNorm& in, long long t,
                                             float (&c)[kElems]) {
#pragma unroll
  for (int i = 0; i < kElems; ++i) c[i] = 0.0f;
  const long long routes = static_cast<long long>(in.tokens) * in.top_k;
#pragma unroll 2
  for (int k = 0; k < in.top_k; ++k) {
    const long long r = t * in.top_k + k;
    const int pos = __ldg(in.route_pos + r);
    if (pos < 0 || pos >= routes) continue;
    const float w = __ldg(in.route_weights + r);
    const T* row = static_cast<const T*>(in.y_permuted) + static_cast<long long>(pos) * in.output;
#pragma unroll
    for (int q = 0; q < kElems / kPer; ++q) {
      const int col = (q * blockDim.x + threadIdx.x) * kPer;
      if (col < in.output) {
        float v[kPer];
        load_cols<T, kPer>(row + col, v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) c[q * kPer + i] = fmaf(w, v[i], c[q * kPer + i]);
      }
    }
  }
}

template <typename T, int kPer, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) unpermute_norm_kernel(const UnpermuteNorm in,
                                                                     T* residual_out, T* normed,
                                                                     float* inv_rms) {
  __shared__ float parts[2][32];
  const long long t = blockIdx.x;
  const long long row = t * in.output;
  const float per_col = 1.0f / static_cast<float>(in.output);
  float res[kElems];
#pragma unroll
  for (int q = 0; q < kElems / kPer; ++q) {
    const int col = (q * blockDim.x + threadIdx.x) * kPer;
    if (col < in.output) {
      load_own_cols<T, kPer>(static_cast<const T*>(in.residual) + row + col, res + q * kPer);
    }
  }
  float c[kElems];
  combine_cols<T, kPer>(in, t, c);
  float i1 = 1.0f;
  if (in.post_gamma != nullptr) {
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < kElems; ++i) sq = fmaf(c[i], c[i], sq);
    i1 = rsqrtf(block_sum(sq, parts[0]) * per_col + in.eps);
  }
  float sq = 0.0f;
#pragma unroll
  for (int q = 0; q < kElems / kPer; ++q) {
    const int col = (q * blockDim.x + threadIdx.x) * kPer;
    if (col < in.output) {
      float* r = c + q * kPer;
      float g[kPer];
      if (in.post_gamma != nullptr) {
        load_gamma<kPer>(in.post_gamma + col, g);
#pragma unroll
        for (int i = 0; i < kPer; ++i) r[i] *= i1 * g[i];
      }
      if (in.gate != nullptr) {
        load_gamma<kPer>(in.gate + col, g);
#pragma unroll
        for (int i = 0; i < kPer; ++i) r[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        r[i] = fmaf(in.residual_scale, res[q * kPer + i], r[i]);
        sq = fmaf(r[i], r[i], sq);
      }
      store_cols<T, kPer>(residual_out + row + col, r);
    }
  }
  float i2 = 1.0f;
  if (in.pre_gamma != nullptr) {
    i2 = rsqrtf(block_sum(sq, parts[1]) * per_col + in.eps);
#pragma unroll
    for (int q = 0; q < kElems / kPer; ++q) {
      const int col = (q * blockDim.x + threadIdx.x) * kPer;
      if (col < in.output) {
        float* r = c + q * kPer;
        float g[kPer];
        load_gamma<kPer>(in.pre_gamma + col, g);
#pragma unroll
        for (int i = 0; i < kPer; ++i) r[i] *= i2 * g[i];
        store_cols<T, kPer>(normed + row + col, r);
      }
    }
  }
  if (inv_rms != nullptr && threadIdx.x == 0) {
    inv_rms[2 * t] = i1;
    inv_rms[2 * t + 1] = i2;
  }
}

// ---- gradient ---------------------------------------------------------------------
//
//   rn = r' i2, v = dn pre:  dr = dro + i2 (v - rn mean(v rn))
//   cn = c i1, db = dr gate, v = db post:  dc = i1 (v - cn mean(v cn))
//   d_residual = scale dr, dy_permuted[pos_k] = w_k dc, dw_k = <dc, y_permuted[pos_k]>
//   d_gate = sum_t dr b, d_post = sum_t db cn, d_pre = sum_t dn rn

template <typename T, int kPer, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) unpermute_norm_backward_kernel(
    const UnpermuteNorm in, const UnpermuteNormGrads g, float* partial) {
  __shared__ float parts[2][32];
  __shared__ float dots[kMaxTopK][32];
  const long long routes = static_cast<long long>(in.tokens) * in.top_k;
  const float per_col = 1.0f / static_cast<float>(in.output);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool post = in.post_gamma != nullptr, pre = in.pre_gamma != nullptr;
  float s_post[kElems], s_gate[kElems], s_pre[kElems];
#pragma unroll
  for (int i = 0; i < kElems; ++i) s_post[i] = s_gate[i] = s_pre[i] = 0.0f;

  for (long long t = blockIdx.x; t < in.tokens; t += gridDim.x) {
    const long long row = t * in.output;
    const float i1 = post ? __ldg(g.inv_rms + 2 * t) : 1.0f;
    const float i2 = pre ? __ldg(g.inv_rms + 2 * t + 1) : 0.0f;
    float c[kElems];   // c, then cn
    float dr[kElems];  // incoming gradient, then dr, then dc
    float rn[kElems];  // normalised r'
    float v2[kElems];  // dn * pre
    combine_cols<T, kPer>(in, t, c);
    float dot = 0.0f;
#pragma unroll
    for (int q = 0; q < kElems / kPer; ++q) {
      const int col = (q * blockDim.x + threadIdx.x) * kPer;
      const int o = q * kPer;
      if (col < in.output) {
        float a[kPer], res[kPer];
        load_cols<T, kPer>(static_cast<const T*>(in.residual) + row + col, res);
        if (g.d_residual_out != nullptr) {
          load_own_cols<T, kPer>(static_cast<const T*>(g.d_residual_out) + row + col, dr + o);
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) dr[o + i] = 0.0f;
        }
        float b[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          c[o + i] *= i1;
          b[i] = c[o + i];
        }
        if (post) {
          load_gamma<kPer>(in.post_gamma + col, a);
#pragma unroll
          for (int i = 0; i < kPer; ++i) b[i] *= a[i];
        }
        if (in.gate != nullptr) {
          load_gamma<kPer>(in.gate + col, a);
#pragma unroll
          for (int i = 0; i < kPer; ++i) b[i] *= a[i];
        }
        if (pre) {
          float dn[kPer];
          load_cols<T, kPer>(static_cast<const T*>(g.d_normed) + row + col, dn);
          load_gamma<kPer>(in.pre_gamma + col, a);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            rn[o + i] = fmaf(in.residual_scale, res[i], b[i]) * i2;
            s_pre[o + i] = fmaf(dn[i], rn[o + i], s_pre[o + i]);
            v2[o + i] = dn[i] * a[i];
            dot = fmaf(v2[o + i], rn[o + i], dot);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) rn[o + i] = v2[o + i] = 0.0f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) dr[o + i] = rn[o + i] = v2[o + i] = 0.0f;
      }
    }
    const float m2 = pre ? block_sum(dot, parts[0]) * per_col : 0.0f;
    dot = 0.0f;
#pragma unroll
    for (int q = 0; q < kElems / kPer; ++q) {
      const int col = (q * blockDim.x + threadIdx.x) * kPer;
      const int o = q * kPer;
      if (col < in.output) {
        float a[kPer], out[kPer], gp[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          dr[o + i] += i2 * (v2[o + i] - rn[o + i] * m2);
          out[i] = in.residual_scale * dr[o + i];
        }
        store_cols<T, kPer>(static_cast<T*>(g.d_residual) + row + col, out);
        if (post) {
          load_gamma<kPer>(in.post_gamma + col, gp);
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) gp[i] = 1.0f;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          s_gate[o + i] = fmaf(dr[o + i], c[o + i] * gp[i], s_gate[o + i]);
        }
        if (in.gate != nullptr) {
          load_gamma<kPer>(in.gate + col, a);
#pragma unroll
          for (int i = 0; i < kPer; ++i) dr[o + i] *= a[i];
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          s_post[o + i] = fmaf(dr[o + i], c[o + i], s_post[o + i]);
          dr[o + i] *= gp[i];
          dot = fmaf(dr[o + i], c[o + i], dot);
        }
      }
    }
    if (post) {
      const float m1 = block_sum(dot, parts[1]) * per_col;
#pragma unroll
      for (int i = 0; i < kElems; ++i) dr[i] = i1 * (dr[i] - c[i] * m1);
    }
    // Routes: the gradient rows and the weights' dot products.
    for (int k = 0; k < in.top_k; ++k) {
      const long long r = t * in.top_k + k;
      const int pos = __ldg(in.route_pos + r);
      float d = 0.0f;
      if (pos >= 0 && pos < routes) {
        const float w = __ldg(in.route_weights + r);
        const long long at = static_cast<long long>(pos) * in.output;
#pragma unroll
        for (int q = 0; q < kElems / kPer; ++q) {
          const int col = (q * blockDim.x + threadIdx.x) * kPer;
          if (col < in.output) {
            float v[kPer], out[kPer];
            load_cols<T, kPer>(static_cast<const T*>(in.y_permuted) + at + col, v);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              d = fmaf(dr[q * kPer + i], v[i], d);
              out[i] = w * dr[q * kPer + i];
            }
            store_cols<T, kPer>(static_cast<T*>(g.d_y_permuted) + at + col, out);
          }
        }
      }
      d = warp_sum(d);
      if (lane == 0) dots[k][warp] = d;
    }
    __syncthreads();
    const int warps = blockDim.x >> 5;
    for (int k = threadIdx.x; k < in.top_k; k += blockDim.x) {
      float d = 0.0f;
      for (int w = 0; w < warps; ++w) d += dots[k][w];
      g.d_route_weights[t * in.top_k + k] = d;
    }
    __syncthreads();
  }
  // This block's shares of the column sums: [block][3][output].
  float* p = partial + 3LL * blockIdx.x * in.output;
#pragma unroll
  for (int q = 0; q < kElems / kPer; ++q) {
    const int col = (q * blockDim.x + threadIdx.x) * kPer;
    if (col < in.output) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        p[col + i] = s_post[q * kPer + i];
        p[in.output + col + i] = s_gate[q * kPer + i];
        p[2 * in.output + col + i] = s_pre[q * kPer + i];
      }
    }
  }
}

constexpr int kSumThreads = 256;
constexpr int kSumCols = 32;

__global__ void __launch_bounds__(kSumThreads) column_sums_kernel(
    const float* __restrict__ partial, int blocks, int output, float* d_post, float* d_gate,
    float* d_pre) {
  __shared__ float parts[kSumThreads / kSumCols][kSumCols];
  float* out = blockIdx.y == 0 ? d_post : (blockIdx.y == 1 ? d_gate : d_pre);
  if (out == nullptr) return;
  const int lane = threadIdx.x % kSumCols, group = threadIdx.x / kSumCols;
  const int col = blockIdx.x * kSumCols + lane;
  float sum = 0.0f;
  if (col < output) {
    for (int b = group; b < blocks; b += kSumThreads / kSumCols) {
      sum += __ldg(partial + (3LL * b + blockIdx.y) * output + col);
    }
  }
  parts[group][lane] = sum;
  __syncthreads();
  if (group == 0 && col < output) {
#pragma unroll
    for (int i = 1; i < kSumThreads / kSumCols; ++i) sum += parts[i][lane];
    out[col] = sum;
  }
}

// Threads so that each holds at most `per` columns; at least a warp.
int row_threads(int output, int per) {
  int threads = 32;
  while (threads < 1024 && threads * per < output) threads *= 2;
  return threads;
}

// One resident wave of the gradient kernel (about 128 registers per thread).
int backward_blocks(int tokens, int output) {
  const int threads = row_threads(output, kElems);
  int per_sm = 512 / threads;
  if (per_sm > 16) per_sm = 16;
  if (per_sm < 1) per_sm = 1;
  const int most = kNumSms * per_sm;
  return tokens < most ? tokens : most;
}

bool aligned_rows(const UnpermuteNorm& in, Dtype dtype) {
  return (in.output * dtype_bytes(dtype)) % 16 == 0 && aligned_to(in.y_permuted, 16) &&
         aligned_to(in.residual, 16) && aligned_to(in.post_gamma, 16) &&
         aligned_to(in.gate, 16) && aligned_to(in.pre_gamma, 16);
}

template <typename T, int kPer>
cudaError_t forward(const UnpermuteNorm& in, void* residual_out, void* normed, float* inv_rms,
                    cudaStream_t stream) {
  // Eight columns per thread while the block stays at 512 threads.
  int threads = row_threads(in.output, 8);
  if (threads > 512) threads = row_threads(in.output, kElems);
  auto* kernel = threads <= 512 ? unpermute_norm_kernel<T, kPer, 512>
                                : unpermute_norm_kernel<T, kPer, 1024>;
  kernel<<<in.tokens, threads, 0, stream>>>(in, static_cast<T*>(residual_out),
                                            static_cast<T*>(normed), inv_rms);
  note_launch();
  return cudaGetLastError();
}

template <typename T, int kPer>
cudaError_t backward(const UnpermuteNorm& in, const UnpermuteNormGrads& g, float* workspace,
                     cudaStream_t stream) {
  const int threads = row_threads(in.output, kElems);
  const int blocks = backward_blocks(in.tokens, in.output);
  auto* kernel = threads <= 512 ? unpermute_norm_backward_kernel<T, kPer, 512>
                                : unpermute_norm_backward_kernel<T, kPer, 1024>;
  kernel<<<blocks, threads, 0, stream>>>(in, g, workspace);
  note_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (g.d_post_gamma != nullptr || g.d_gate != nullptr || g.d_pre_gamma != nullptr) {
    column_sums_kernel<<<dim3(ceil_div(in.output, kSumCols), 3), kSumThreads, 0, stream>>>(
        workspace, blocks, in.output, g.d_post_gamma, g.d_gate, g.d_pre_gamma);
    note_launch();
  }
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_unpermute_norm(const UnpermuteNorm& in, void* residual_out, void* normed,
                                  float* inv_rms, Dtype dtype, cudaStream_t stream) {
  const bool vec =
      aligned_rows(in, dtype) && aligned_to(residual_out, 16) && aligned_to(normed, 16);
  if (dtype == Dtype::kBf16) {
    return vec ? forward<__nv_bfloat16, 8>(in, residual_out, normed, inv_rms, stream)
               : forward<__nv_bfloat16, 1>(in, residual_out, normed, inv_rms, stream);
  }
  return vec ? forward<float, 4>(in, residual_out, normed, inv_rms, stream)
             : forward<float, 1>(in, residual_out, normed, inv_rms, stream);
}

std::size_t unpermute_norm_backward_workspace_bytes(int tokens, int output) {
  return 12ull * static_cast<std::size_t>(backward_blocks(tokens, output)) * output;
}

cudaError_t launch_unpermute_norm_backward(const UnpermuteNorm& in, const UnpermuteNormGrads& g,
                                           float* workspace, Dtype dtype, cudaStream_t stream) {
  const bool vec = aligned_rows(in, dtype) && aligned_to(g.d_residual_out, 16) &&
                   aligned_to(g.d_normed, 16) && aligned_to(g.d_residual, 16) &&
                   aligned_to(g.d_y_permuted, 16);
  if (dtype == Dtype::kBf16) {
    return vec ? backward<__nv_bfloat16, 8>(in, g, workspace, stream)
               : backward<__nv_bfloat16, 1>(in, g, workspace, stream);
  }
  return vec ? backward<float, 4>(in, g, workspace, stream)
             : backward<float, 1>(in, g, workspace, stream);
}

}  // namespace rrb

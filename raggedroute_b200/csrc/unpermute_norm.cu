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
// A token's row is held in registers, 16 columns per thread, so the route rows
// and the residual are read once and r', n written once: bound by those bytes.
// The two means are reductions in a fixed order. The gradient recomputes c and
// r' from its inputs instead of reading rounded copies, keeps its share of the
// three column sums (post, gate, pre) in registers and writes it once; a
// second kernel adds the shares in block order. No atomics, so results repeat.
//
// Two forms of each kernel. A token passes several dependent steps (positions,
// rows, one or two reductions, stores), and with loads issued by the threads
// that wait for them too few bytes are in flight. From a few tokens per SM up,
// teams of 32 to 512 threads of one persistent block per SM therefore take a
// token each, and each team streams the rows of its next tokens into a ring in
// shared memory with bulk copies; rows of any alignment are copied as the
// 16-byte granules they touch. Fewer tokens, and rows too wide for the ring,
// take plain blocks (forward_streams and backward_streams say when).
//
// Top 2, both norms and the gate: bf16, 32768 tokens, N=4096 forward 253 us (5.3
// TB/s), gradient 470 (4.6; latency: the 16 warps per SM that its registers allow
// issue 47% of the time, and DRAM is not full either); FP32, 16384 tokens, N=1024 60 and 95 (5.5 and
// 5.7 TB/s); rows that are no multiple of 16 bytes 1.7 to 2.3 TB/s, their columns taken
// singly or in pairs (bf16, N=1491, 2340). Tried for the gradient at N=4096 and slower:
// two tokens per step (spills), sixteen columns per thread; a warp that only
// copies was faster there and slower in all other widths.
#include <mutex>

#include "expert_block.cuh"
#include "sm100.cuh"

namespace rrb {
namespace {

constexpr int kElems = 16;  // columns per thread
constexpr int kMaxTopK = 64;
constexpr int kMaxDevices = 64;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

// Sum over a token's threads (the block's x axis) in each of them; `parts` holds 32 floats and is free
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
  follow_previous();
  const long long t = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (t >= in.tokens) return;  // only where warps share a block, and then no barrier
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
  follow_previous();
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

// ---- streamed form ------------------------------------------------------------------

constexpr int kStreamThreads = 512;  // per block, at most
constexpr int kStreamTopK = 16;
constexpr int kMaxStages = 4;
constexpr int kMaxTeams = kStreamThreads / 32;
constexpr std::size_t kRingBytes = 204 * 1024;

// A team's ring has one token's rows per stage: the route rows, the residual,
// and for the gradient d_residual_out and d_normed.
struct Stream {
  int team = 0;      // threads per token
  int teams = 0;     // of a block
  int sources = 0;   // rows per token
  int stride = 0;    // bytes of a row's place
  int padded = 0;    // gradient: columns of a factor kept behind the rings
  int factors = 0;   // gradient: factors kept there: post * gate, and pre if it fits
  int stages = 0;
  int blocks = 0;
};

struct StreamSmem {
  uint64_t full[kMaxTeams][kMaxStages];
  int failed;
  // Of each token in a ring: where its rows start (-1: a skipped route), and
  // the routes' weights (behind them the gradient's two 1/rms) and positions.
  int start[kMaxTeams][kMaxStages][kStreamTopK + 3];
  float weight[kMaxTeams][kMaxStages][kStreamTopK + 2];
  int pos[kMaxTeams][kMaxStages][kStreamTopK];
};

// The threads of one team (a barrier of its own each; one warp needs none).
__device__ __forceinline__ void team_sync(int team, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

struct Sources {
  const void* row[3] = {};         // residual, d_residual_out, d_normed; null ones left out
  const float* inv_rms = nullptr;  // [tokens][2], for the gradient
};

// Fills a team's ring; called by its first warp, a lane per row (sources <= 32).
// kAligned: rows are whole 16-byte granules.
template <typename T, bool kAligned>
struct Filler {
  const UnpermuteNorm& in;
  const Stream& st;
  StreamSmem& s;
  uint32_t ring;     // this team's
  int team;
  const char* base;  // of this lane's rows
  long long rows;    // how many there are
  const float* inv_rms;
  int pos;  // of the next token's row, fetched ahead
  float weight;

  __device__ __forceinline__ Filler(const UnpermuteNorm& in, const Stream& st, StreamSmem& s,
                                    const Sources& src, uint32_t ring, int team)
      : in(in), st(st), s(s), ring(ring), team(team), inv_rms(src.inv_rms) {
    const int lane = threadIdx.x & 31;
    const bool route = lane < in.top_k;
    base = route ? static_cast<const char*>(in.y_permuted)
                 : (lane < st.sources ? static_cast<const char*>(src.row[lane - in.top_k])
                                      : nullptr);
    rows = route ? static_cast<long long>(in.tokens) * in.top_k
                 : (lane < st.sources ? in.tokens : 0);
  }
  __device__ __forceinline__ void fetch(long long t) {
    const int lane = threadIdx.x & 31;
    pos = -1;
    weight = 0.0f;
    if (lane < in.top_k && t < in.tokens) {
      pos = __ldg(in.route_pos + t * in.top_k + lane);
      weight = __ldg(in.route_weights + t * in.top_k + lane);
    } else if (inv_rms != nullptr && lane < in.top_k + 2 && t < in.tokens) {
      weight = __ldg(inv_rms + 2 * t + lane - in.top_k);
    }
  }
  // Starts token t's rows (position and weight fetched) into `stage`, and fetches
  // those of token `next`.
  __device__ __forceinline__ void fill(long long t, int stage, long long next) {
    using namespace sm100;
    if (t >= in.tokens) return;
    const int lane = threadIdx.x & 31;
    const long long bytes = static_cast<long long>(in.output) * sizeof(T);
    const bool route = lane < in.top_k;
    const long long row = route ? pos : t;
    const bool there = row >= 0 && row < rows;
    const int place = (stage * st.sources + lane) * st.stride;
    const long long at = row * bytes;
    // The granules of the row. The buffers start on a 16-byte boundary, so only
    // the last row's last granule can reach past one; its elements are copied
    // one by one.
    long long a0 = at, a1 = at + bytes;
    bool past = false;
    if constexpr (!kAligned) {
      a0 = at & ~15LL;
      a1 = (a1 + 15) & ~15LL;
      past = a1 > rows * bytes;
      if (past) a1 -= 16;
    }
    const uint32_t size = there && a1 > a0 ? static_cast<uint32_t>(a1 - a0) : 0u;
    if (lane < st.sources) {
      s.start[team][stage][lane] = there ? static_cast<int>(place + (at - a0)) : -1;
    }
    if (lane < in.top_k + 2) s.weight[team][stage][lane] = weight;
    if (route) s.pos[team][stage][lane] = pos;
    uint32_t total;
    if constexpr (kAligned) {
      total = __popc(__ballot_sync(0xffffffffu, there)) * static_cast<uint32_t>(bytes);
    } else {
      if (there && past) {
        for (long long b = a1 > at ? a1 : at; b < at + bytes; b += sizeof(T)) {
          const uint32_t to = ring + place + static_cast<uint32_t>(b - a0);
          if constexpr (sizeof(T) == 2) {
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(to),
                         "h"(__ldg(reinterpret_cast<const unsigned short*>(base + b)))
                         : "memory");
          } else {
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(to),
                         "r"(__ldg(reinterpret_cast<const unsigned*>(base + b)))
                         : "memory");
          }
        }
        // This lane's later copies into the same place come after these stores.
        fence_proxy_async_smem();
      }
      total = __reduce_add_sync(0xffffffffu, size);
    }
    uint64_t* full = &s.full[team][stage];
    __syncwarp();  // the lanes' notes come before the arrival
    if (lane == 0) mbar_arrive_expect_tx(full, total);
    __syncwarp();
    if (size > 0) bulk_load(ring + place, base + a0, size, full);
    fetch(next);
  }
};

// kPer columns of a staged row.
template <typename T, int kPer>
__device__ __forceinline__ void staged_cols(const char* p, float* v) {
  if constexpr (kPer == 1) {
    v[0] = to_f32(*reinterpret_cast<const T*>(p));
  } else if constexpr (kPer * sizeof(T) == 16) {
    unpack16<T>(*reinterpret_cast<const uint4*>(p), v);
  } else {
    static_assert(kPer == 2 && sizeof(T) == 2, "pairs of bfloat16");
    const uint32_t w = *reinterpret_cast<const uint32_t*>(p);
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xFFFF0000u);
  }
}

template <typename T, int kPer>
__device__ __forceinline__ void put_cols(T* p, const float* v) {
  if constexpr (kPer == 2) *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(v[0], v[1]);
  else store_cols<T, kPer>(p, v);
}

// kPer floats of shared memory.
template <int kPer>
__device__ __forceinline__ void shared_cols(const float* p, float* v) {
  if constexpr (kPer % 4 == 0) {
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) {
      const float4 f = reinterpret_cast<const float4*>(p)[i];
      v[4 * i] = f.x;
      v[4 * i + 1] = f.y;
      v[4 * i + 2] = f.z;
      v[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = p[i];
  }
}

// post * gate and pre of kPer columns (1 for what is left out, 0 past the row).
template <int kPer>
__device__ __forceinline__ void column_factors(const UnpermuteNorm& in, int col, float* pg,
                                               float* pr) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool there = col + i < in.output;
    pg[i] = there ? (in.post_gamma != nullptr ? __ldg(in.post_gamma + col + i) : 1.0f) *
                        (in.gate != nullptr ? __ldg(in.gate + col + i) : 1.0f)
                  : 0.0f;
    pr[i] = there && in.pre_gamma != nullptr ? __ldg(in.pre_gamma + col + i) : 0.0f;
  }
}

// c of this thread's columns from the staged route rows.
template <typename T, int kPer>
__device__ __forceinline__ void staged_combine(const UnpermuteNorm& in, const Stream& st,
                                               const char* ring, const int* start,
                                               const float* weight, int tid,
                                               float (&c)[kElems]) {
#pragma unroll
  for (int i = 0; i < kElems; ++i) c[i] = 0.0f;
#pragma unroll 2
  for (int k = 0; k < in.top_k; ++k) {
    if (start[k] < 0) continue;
    const float w = weight[k];
    const char* row = ring + start[k];
#pragma unroll
    for (int q = 0; q < kElems / kPer; ++q) {
      const int col = (q * st.team + tid) * kPer;
      if (col < in.output) {
        float v[kPer];
        staged_cols<T, kPer>(row + col * sizeof(T), v);
#pragma unroll
        for (int i = 0; i < kPer; ++i) c[q * kPer + i] = fmaf(w, v[i], c[q * kPer + i]);
      }
    }
  }
}

__device__ __forceinline__ void stream_setup(const Stream& st, int top_k, StreamSmem& s) {
  using namespace sm100;
  if (threadIdx.x == 0) {
    for (int i = 0; i < st.teams; ++i) {
      for (int j = 0; j < st.stages; ++j) mbar_init(&s.full[i][j], 1);
    }
    s.failed = 0;
    fence_mbar_init();
  }
  // What a token finds after a wait that ran out: nothing, at a valid place.
  for (int i = threadIdx.x; i < kMaxTeams * kMaxStages * (kStreamTopK + 3); i += blockDim.x) {
    (&s.start[0][0][0])[i] = i % (kStreamTopK + 3) < top_k ? -1 : 0;
  }
  __syncthreads();
}

// Ends a streamed kernel: after a wait that ran out, copies in flight
// (microseconds each) get time to land before the shared memory is given up.
__device__ __forceinline__ void stream_end(StreamSmem& s) {
  __syncthreads();
  if (*static_cast<volatile int*>(&s.failed)) {
    const uint64_t start = sm100::global_timer_ns();
    while (sm100::global_timer_ns() - start < 2000000u) {
    }
  }
}

// The tokens of a team. step() waits for the next token's rows; refill(), called
// after a barrier of the team inside that token, starts the rows that go where
// the token before it was. A wait that runs out raises the error word and lets
// the loop run on (further waits return at once): the team's barriers stay
// matched, and what is computed is reported as wrong.
template <typename T, bool kAligned>
struct TokenLoop {
  Filler<T, kAligned> filler;
  unsigned* err;
  long long t, stride;
  int stage;
  uint32_t phase;
  bool filling, first_token;

  __device__ __forceinline__ TokenLoop(const UnpermuteNorm& in, const Stream& st, StreamSmem& s,
                                       const Sources& src, uint32_t ring, int team, unsigned* err)
      : filler(in, st, s, src, ring, team), err(err) {
    t = static_cast<long long>(blockIdx.x) * st.teams + team;
    stride = static_cast<long long>(gridDim.x) * st.teams;
    stage = -1;
    phase = 0;
    first_token = true;
    filling = threadIdx.x % st.team < 32;
    if (filling) {
      filler.fetch(t);
      for (int i = 0; i < st.stages; ++i) filler.fill(t + i * stride, i, t + (i + 1) * stride);
    }
    t -= stride;
  }
  __device__ __forceinline__ bool step() {
    t += stride;
    if (t >= filler.in.tokens) return false;  // uniform over a team
    if (++stage == filler.st.stages) {
      stage = 0;
      phase ^= 1u;
    }
    sm100::mbar_wait(&filler.s.full[filler.team][stage], phase, err, &filler.s.failed);
    return true;
  }
  __device__ __forceinline__ void refill() {
    if (filling && !first_token) {
      const int stages = filler.st.stages;
      filler.fill(t + (stages - 1) * stride, stage == 0 ? stages - 1 : stage - 1,
                  t + stages * stride);
    }
    first_token = false;
  }
};

template <typename T, int kPer>
__global__ void __launch_bounds__(kStreamThreads, 1) unpermute_norm_stream_kernel(
    const UnpermuteNorm in, const Stream st, T* residual_out, T* normed, float* inv_rms,
    unsigned* err) {
  using namespace sm100;
  extern __shared__ __align__(16) char rings[];
  __shared__ StreamSmem s;
  __shared__ float parts[2][kMaxTeams];  // each warp's share of a sum
  stream_setup(st, in.top_k, s);
  follow_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = threadIdx.x / st.team, tid = threadIdx.x % st.team;
  const int team_warps = st.team >> 5, warp0 = team * team_warps;
  const char* ring = rings + team * st.stages * st.sources * st.stride;
  const float per_col = 1.0f / static_cast<float>(in.output);
  float pg[kElems], pr[kElems];  // post * gate and pre of this thread's columns
#pragma unroll
  for (int q = 0; q < kElems / kPer; ++q) {
    column_factors<kPer>(in, (q * st.team + tid) * kPer, pg + q * kPer, pr + q * kPer);
  }
  // Sums take the rows of `parts` in turn, across tokens too: between a sum's reads
  // and the writes of the next one in its row lies the barrier of the sum between
  // them, whatever other barriers a token has.
  int turn = 0;
  auto team_sum = [&](float v) {
    v = warp_sum(v);
    if (team_warps == 1) {
      __syncwarp();
      return v;
    }
    float* shares = parts[turn];
    turn ^= 1;
    if (lane == 0) shares[warp] = v;
    team_sync(team, st.team);
    float sum = 0.0f;
    for (int w = 0; w < team_warps; ++w) sum += shares[warp0 + w];
    return sum;
  };
  Sources src;
  src.row[0] = in.residual;
  TokenLoop<T, kPer * sizeof(T) == 16> loop(in, st, s, src, smem_u32(ring), team, err);
  while (loop.step()) {
    const long long t = loop.t;
    const int* start = s.start[team][loop.stage];
    float c[kElems];
    staged_combine<T, kPer>(in, st, ring, start, s.weight[team][loop.stage], tid, c);
    float i1 = 1.0f;
    if (in.post_gamma != nullptr) {
      float sq = 0.0f;
#pragma unroll
      for (int i = 0; i < kElems; ++i) sq = fmaf(c[i], c[i], sq);
      i1 = rsqrtf(team_sum(sq) * per_col + in.eps);
    } else {
      team_sync(team, st.team);
    }
    loop.refill();
    const char* res_row = ring + start[in.top_k];
    float sq = 0.0f;
#pragma unroll
    for (int q = 0; q < kElems / kPer; ++q) {
      const int col = (q * st.team + tid) * kPer;
      if (col < in.output) {
        float* r = c + q * kPer;
        float res[kPer];
        staged_cols<T, kPer>(res_row + col * sizeof(T), res);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          r[i] = fmaf(in.residual_scale, res[i], r[i] * i1 * pg[q * kPer + i]);
          sq = fmaf(r[i], r[i], sq);
        }
        put_cols<T, kPer>(residual_out + t * in.output + col, r);
      }
    }
    float i2 = 1.0f;
    if (in.pre_gamma != nullptr) {
      i2 = rsqrtf(team_sum(sq) * per_col + in.eps);
#pragma unroll
      for (int q = 0; q < kElems / kPer; ++q) {
        const int col = (q * st.team + tid) * kPer;
        if (col < in.output) {
          float* r = c + q * kPer;
#pragma unroll
          for (int i = 0; i < kPer; ++i) r[i] *= i2 * pr[q * kPer + i];
          put_cols<T, kPer>(normed + t * in.output + col, r);
        }
      }
    }
    if (inv_rms != nullptr && tid == 0) {
      inv_rms[2 * t] = i1;
      inv_rms[2 * t + 1] = i2;
    }
  }
  stream_end(s);
}

// The gradient, in one pass over a token's inputs and one reduction. With
// a = dro + i2 v (v = dn pre) and f = post * gate:
//   dr = a - i2 m2 rn,  v1 = f dr,  m2 = mean(v rn)
//   P_k = <v1, y_k> = <f a, y_k> - i2 m2 <f rn, y_k>
//   m1 = mean(v1 cn) = i1 sum_k w_k P_k / N
//   dw_k = <dc, y_k> = i1 (P_k - m1 <cn, y_k>)
// (without the norm of c: i1 = 1, m1 = 0), so a token's 1 + 3 top_k sums are
// known together, before any of its results. The gradients of post and gate
// are one column sum, of dr cn, times the other factor. post * gate and pre
// lie in shared memory behind the ring: read from the caller's buffers for
// every token they would be as many bytes as its rows. Two columns share an
// instruction (packed FP32 arithmetic, which rounds each half as the plain
// instruction does).

struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ F2 f2(float x) { return f2(x, x); }
__device__ __forceinline__ void split(F2 a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float sum2(F2 a) {
  float lo, hi;
  split(a, lo, hi);
  return lo + hi;
}

// This thread's columns of a staged row in pairs. Columns past the row's end take
// the row's first ones: the caller's factors are zero there, which costs less
// than a test around every load.
template <typename T, int kPer, int kPairs>
__device__ __forceinline__ void staged_row(const char* row, int output, int team, int tid,
                                           F2 (&v)[kPairs]) {
  float f[2 * kPairs];
#pragma unroll
  for (int q = 0; q < 2 * kPairs / kPer; ++q) {
    const int col = (q * team + tid) * kPer;
    staged_cols<T, kPer>(row + (col < output ? col : 0) * sizeof(T), f + q * kPer);
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}

// The same of a row of factors, whose column `past` stands for those past the end.
template <int kPer, int kPairs>
__device__ __forceinline__ void factor_row(const float* row, int output, int past, int team,
                                           int tid, F2 (&v)[kPairs]) {
  float f[2 * kPairs];
#pragma unroll
  for (int q = 0; q < 2 * kPairs / kPer; ++q) {
    const int col = (q * team + tid) * kPer;
    shared_cols<kPer>(row + (col < output ? col : past), f + q * kPer);
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}

template <typename T, int kPer, int kPairs>
__device__ __forceinline__ void put_row(T* row, int output, int team, int tid,
                                        const F2 (&v)[kPairs]) {
  float f[2 * kPairs];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) split(v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int q = 0; q < 2 * kPairs / kPer; ++q) {
    const int col = (q * team + tid) * kPer;
    if (col < output) put_cols<T, kPer>(row + col, f + q * kPer);
  }
}

// Eight sums over a warp with nine shuffles: halves of the warp exchange halves
// of the sums until each lane holds one; lane l ends with the sum l / 4.
__device__ __forceinline__ float warp_sum8(const float (&v)[8]) {
  const int lane = threadIdx.x & 31;
  float a[4], b[2];
  const bool h4 = lane & 16, h3 = lane & 8, h2 = lane & 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float keep = h4 ? v[4 + i] : v[i], give = h4 ? v[i] : v[4 + i];
    a[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float keep = h3 ? a[2 + i] : a[i], give = h3 ? a[i] : a[2 + i];
    b[i] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
  }
  float c = (h2 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, h2 ? b[0] : b[1], 4);
  c += __shfl_xor_sync(0xffffffffu, c, 2);
  return c + __shfl_xor_sync(0xffffffffu, c, 1);
}

template <typename T, int kPer, int kCols, bool kTwo>
__global__ void __launch_bounds__(kStreamThreads, 1) unpermute_norm_backward_stream_kernel(
    const UnpermuteNorm in, const Stream st, const UnpermuteNormGrads g, float* partial,
    unsigned* err) {
  using namespace sm100;
  constexpr int kPairs = kCols / 2;
  constexpr int kSets = kTwo ? 1 : kStreamTopK / 2;
  extern __shared__ __align__(16) char rings[];
  __shared__ StreamSmem s;
  // Of each warp, by parity of the token: for two routes at a time
  // <f a, y>, <f rn, y>, <cn, y> of the first, the same of the second, and
  // (with the first two) <v, rn>.
  __shared__ float sums[2][kMaxTeams][kSets][8];
  const bool post = in.post_gamma != nullptr, pre = in.pre_gamma != nullptr;
  const bool has_dro = g.d_residual_out != nullptr;
  const int n = in.output;
  const int ring_size = st.stages * st.sources * st.stride;
  float* pg = reinterpret_cast<float*>(rings + st.teams * ring_size);
  float* shared_pre = pg + st.padded;
  follow_previous();
  for (int c = threadIdx.x; c < st.padded; c += blockDim.x) {
    float f, p;  // zero from column n on; column padded - 8 is past the end
    column_factors<1>(in, c, &f, &p);
    pg[c] = f;
    if (st.factors > 1) shared_pre[c] = p;
  }
  const float* pr = st.factors > 1 ? shared_pre : in.pre_gamma;
  const int past = st.padded - 8;
  stream_setup(st, in.top_k, s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = threadIdx.x / st.team, tid = threadIdx.x % st.team;
  const int team_warps = st.team >> 5, warp0 = team * team_warps;
  const char* ring = rings + team * ring_size;
  const float per_col = 1.0f / static_cast<float>(n);
  const int at_res = in.top_k, at_dro = in.top_k + 1, at_dn = in.top_k + 1 + (has_dro ? 1 : 0);
  F2 s_dc[kPairs], s_pre[kPairs];  // sums over tokens of dr cn and dn rn
#pragma unroll
  for (int i = 0; i < kPairs; ++i) s_dc[i] = s_pre[i] = f2(0.0f);
  Sources src;
  src.row[0] = in.residual;
  src.row[1] = has_dro ? g.d_residual_out : g.d_normed;
  src.row[2] = g.d_normed;
  src.inv_rms = post || pre ? g.inv_rms : nullptr;
  int parity = 0;
  TokenLoop<T, kPer * sizeof(T) == 16> loop(in, st, s, src, smem_u32(ring), team, err);
  while (loop.step()) {
    const long long t = loop.t;
    const int* start = s.start[team][loop.stage];
    const float* weight = s.weight[team][loop.stage];
    const float i1 = post ? weight[in.top_k] : 1.0f;
    const float i2 = pre ? weight[in.top_k + 1] : 0.0f;
    // Zero for columns past the end, whose c and rn then are zero as well.
    F2 i12[kPairs], i22[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const bool in0 = ((2 * i / kPer) * st.team + tid) * kPer < n;
      const bool in1 = (((2 * i + 1) / kPer) * st.team + tid) * kPer < n;
      i12[i] = f2(in0 ? i1 : 0.0f, in1 ? i1 : 0.0f);
      i22[i] = f2(in0 ? i2 : 0.0f, in1 ? i2 : 0.0f);
    }
    const F2 scale = f2(in.residual_scale);
    F2 c[kPairs], a[kPairs], rn[kPairs];
    F2 y0[kTwo ? kPairs : 1], y1[kTwo ? kPairs : 1];  // the routes' rows, if there are two at most
    F2 f[kPairs];                                     // post * gate
    F2 dot = f2(0.0f);                                // <v, rn>
    auto route_row = [&](int k, F2 (&y)[kPairs]) {
      staged_row<T, kPer>(ring + start[k], n, st.team, tid, y);
    };
    {
      F2 x[kPairs];
      if constexpr (kTwo) {
        const bool there0 = start[0] >= 0, there1 = in.top_k > 1 && start[1] >= 0;
#pragma unroll
        for (int i = 0; i < kPairs; ++i) y0[i] = y1[i] = f2(0.0f);
        if (there0) route_row(0, y0);
        if (there1) route_row(1, y1);
        const F2 w0 = f2(there0 ? weight[0] : 0.0f), w1 = f2(there1 ? weight[1] : 0.0f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) c[i] = fma2(w1, y1[i], mul2(w0, y0[i]));
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) c[i] = f2(0.0f);
        for (int k = 0; k < in.top_k; ++k) {
          if (start[k] < 0) continue;
          route_row(k, x);
          const F2 w = f2(weight[k]);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) c[i] = fma2(w, x[i], c[i]);
        }
      }
      factor_row<kPer>(pg, n, past, st.team, tid, f);
      staged_row<T, kPer>(ring + start[at_res], n, st.team, tid, x);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        c[i] = mul2(i12[i], c[i]);
        // Without the second norm r' takes no part, whatever it holds.
        rn[i] = pre ? mul2(i22[i], fma2(scale, x[i], mul2(c[i], f[i]))) : f2(0.0f);
      }
      if (has_dro) {
        staged_row<T, kPer>(ring + start[at_dro], n, st.team, tid, a);
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) a[i] = f2(0.0f);
      }
      if (pre) {
        F2 p[kPairs];
        staged_row<T, kPer>(ring + start[at_dn], n, st.team, tid, x);
        factor_row<kPer>(pr, n, 0, st.team, tid, p);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          s_pre[i] = fma2(x[i], rn[i], s_pre[i]);
          const F2 v = mul2(x[i], p[i]);
          dot = fma2(v, rn[i], dot);
          a[i] = fma2(i22[i], v, a[i]);
        }
      }
    }
    // The sums of two routes at a time, reduced over the warp.
    float mine = 0.0f;
    auto reduce_pair = [&](int k) {
      float v8[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        F2 fa = f2(0.0f), fr = f2(0.0f), cy = f2(0.0f);
        if (kTwo || (k + h < in.top_k && start[k + h] >= 0)) {
          F2 y[kPairs];
          if constexpr (kTwo) {
#pragma unroll
            for (int i = 0; i < kPairs; ++i) y[i] = h == 0 ? y0[i] : y1[i];
          } else {
            route_row(k + h, y);
          }
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            cy = fma2(c[i], y[i], cy);
            y[i] = mul2(f[i], y[i]);
            fa = fma2(a[i], y[i], fa);
            fr = fma2(rn[i], y[i], fr);
          }
        }
        v8[3 * h] = sum2(fa);
        v8[3 * h + 1] = sum2(fr);
        v8[3 * h + 2] = sum2(cy);
      }
      v8[6] = k == 0 ? sum2(dot) : 0.0f;
      v8[7] = 0.0f;
      mine = warp_sum8(v8);
      if ((team_warps > 1 || !kTwo) && (lane & 3) == 0) {
        sums[parity][warp][k >> 1][lane >> 2] = mine;
      }
    };
    if constexpr (kTwo) {
      reduce_pair(0);
    } else {
      for (int k = 0; k < in.top_k; k += 2) reduce_pair(k);
    }
    // Over the team: lane l ends with sum l / 4 of routes k and k + 1.
    team_sync(team, st.team);
    loop.refill();
    auto team_sums = [&](int k) {
      if (kTwo && team_warps == 1) return mine;
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < kMaxTeams; i += 4) {
        const int w = (lane & 3) + i;
        if (w < team_warps) v += sums[parity][warp0 + w][k >> 1][lane >> 2];
      }
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      return v + __shfl_xor_sync(0xffffffffu, v, 2);
    };
    auto sum_of = [&](float v, int j) { return __shfl_sync(0xffffffffu, v, 4 * j); };
    const float sums01 = team_sums(0);
    const float im2 = i2 * (sum_of(sums01, 6) * per_col);
    // Terms of a norm that is left out are not added as zero times something: a row
    // that is not finite would spread to the token's other results.
    auto p_of = [&](float v, int h) {
      const float p = sum_of(v, 3 * h), r = sum_of(v, 3 * h + 1);
      return pre ? p - im2 * r : p;
    };
    float m1 = 0.0f;
    for (int k = 0; k < (kTwo ? 1 : in.top_k); k += 2) {
      const float v = k == 0 ? sums01 : team_sums(k);
      const float p0 = p_of(v, 0), p1 = p_of(v, 1);
      if (start[k] >= 0) m1 = fmaf(weight[k], p0, m1);
      if (k + 1 < in.top_k && start[k + 1] >= 0) m1 = fmaf(weight[k + 1], p1, m1);
    }
    m1 = post ? i1 * m1 * per_col : 0.0f;
    // The last warp's lane 0 writes the routes' gradients (the first one fills the ring).
    for (int k = 0; warp - warp0 == team_warps - 1 && k < (kTwo ? 1 : in.top_k); k += 2) {
      const float v = k == 0 ? sums01 : team_sums(k);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float p = p_of(v, h), cy = sum_of(v, 3 * h + 2);
        const float d = post ? i1 * (p - m1 * cy) : p;
        if (lane == 0 && k + h < in.top_k) {
          g.d_route_weights[t * in.top_k + k + h] = start[k + h] >= 0 ? d : 0.0f;
        }
      }
    }
    parity ^= 1;
    F2 x[kPairs];
    const F2 nim2 = f2(-im2), nm1 = f2(-m1);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      a[i] = fma2(nim2, rn[i], a[i]);  // dr
      s_dc[i] = fma2(a[i], c[i], s_dc[i]);
      x[i] = mul2(scale, a[i]);
    }
    put_row<T, kPer>(static_cast<T*>(g.d_residual) + t * n, n, st.team, tid, x);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {  // dc
      a[i] = mul2(f[i], a[i]);
      if (post) a[i] = mul2(i12[i], fma2(nm1, c[i], a[i]));
    }
    auto put_route = [&](int k) {
      if (start[k] < 0) return;
      const F2 w = f2(weight[k]);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) x[i] = mul2(w, a[i]);
      put_row<T, kPer>(static_cast<T*>(g.d_y_permuted) +
                           static_cast<long long>(s.pos[team][loop.stage][k]) * n,
                       n, st.team, tid, x);
    };
    if constexpr (kTwo) {
      put_route(0);
      if (in.top_k > 1) put_route(1);
    } else {
      for (int k = 0; k < in.top_k; ++k) put_route(k);
    }
  }
  // The block's shares of the column sums, [block][3][output]: its teams' add up
  // in the rings, of which every load has been used by now.
  __syncthreads();
  float* shared = reinterpret_cast<float*>(rings);
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    const int col = ((i / kPer) * st.team + tid) * kPer + i % kPer;
    if (col < n) {
      float lo, hi;
      split(s_dc[i / 2], lo, hi);
      shared[(2 * team) * n + col] = i % 2 ? hi : lo;
      split(s_pre[i / 2], lo, hi);
      shared[(2 * team + 1) * n + col] = i % 2 ? hi : lo;
    }
  }
  __syncthreads();
  float* p = partial + 3LL * blockIdx.x * n;
  for (int col = threadIdx.x; col < n; col += blockDim.x) {
    float d = 0.0f, e = 0.0f;
    for (int q = 0; q < st.teams; ++q) {
      d += shared[(2 * q) * n + col];
      e += shared[(2 * q + 1) * n + col];
    }
    p[col] = in.gate != nullptr ? d * __ldg(in.gate + col) : d;
    p[n + col] = post ? d * __ldg(in.post_gamma + col) : d;
    p[2 * n + col] = e;
  }
  stream_end(s);
}

constexpr int kSumCols = 32;
constexpr int kSumGroups = 32;

// Adds the blocks' shares in a fixed order: a warp of columns, 32 blocks at a time.
__global__ void __launch_bounds__(kSumCols* kSumGroups) column_sums_kernel(
    const float* __restrict__ partial, int blocks, int output, float* d_post, float* d_gate,
    float* d_pre) {
  __shared__ float parts[kSumGroups][kSumCols];
  follow_previous();
  float* out = blockIdx.y == 0 ? d_post : (blockIdx.y == 1 ? d_gate : d_pre);
  if (out == nullptr) return;
  const int lane = threadIdx.x % kSumCols, group = threadIdx.x / kSumCols;
  const int col = blockIdx.x * kSumCols + lane;
  float sum = 0.0f;
  if (col < output) {
#pragma unroll 8
    for (int b = group; b < blocks; b += kSumGroups) {
      sum += __ldg(partial + (3LL * b + blockIdx.y) * output + col);
    }
  }
  parts[group][lane] = sum;
  __syncthreads();
  if (group == 0 && col < output) {
#pragma unroll
    for (int i = 1; i < kSumGroups; ++i) sum += parts[i][lane];
    out[col] = sum;
  }
}

// Threads so that each holds at most `per` columns; at least a warp.
int row_threads(int output, int per) {
  int threads = 32;
  while (threads < 1024 && threads * per < output) threads *= 2;
  return threads;
}

// The streamed form's layout, or blocks = 0 where it has none: more routes than a
// ring keeps track of, or rows of which two stages do not fit.
Stream stream_plan(int tokens, int top_k, int output, int extra_rows, bool gradient, int elems,
                   std::size_t size) {
  Stream st;
  if (top_k > kStreamTopK || output > kStreamThreads * elems) return st;
  st.team = row_threads(output, elems);
  st.teams = kStreamThreads / st.team;
  st.sources = top_k + extra_rows;
  // A row's granules: up to 15 bytes before and after it.
  st.stride = static_cast<int>((output * size + 15) / 16 * 16 + 16);
  if (gradient) {
    st.padded = (output + 7) / 8 * 8 + 8;  // and eight zeros
    st.factors = 2;
  }
  // Two stages have to fit: with pre left in its own buffer, or with half the
  // teams, if need be.
  for (;;) {
    const std::size_t stage = static_cast<std::size_t>(st.teams) * st.sources * st.stride;
    st.stages = static_cast<int>((kRingBytes - 4 * st.factors * st.padded) / stage);
    if (st.stages >= 2) break;
    if (st.teams > 1) st.teams /= 2;
    else if (st.factors == 2) st.factors = 1;
    else return st;
  }
  if (st.stages > kMaxStages) st.stages = kMaxStages;
  st.blocks = ceil_div(tokens, st.teams);
  if (st.blocks > kNumSms) st.blocks = kNumSms;
  return st;
}

std::size_t ring_bytes(const Stream& st) {
  return static_cast<std::size_t>(st.stages) * st.teams * st.sources * st.stride +
         4 * st.factors * st.padded;
}

// Columns per thread of the streamed gradient: eight, so that a token's c, a, rn
// and the thread's column sums stay in registers with sixteen warps per SM;
// rows wider than that covers take sixteen.
int gradient_elems(int output) { return output <= kStreamThreads * 8 ? 8 : 16; }

// One resident wave of the plain gradient kernel (about 128 registers per
// thread).
int backward_blocks(int tokens, int output) {
  const int threads = row_threads(output, kElems);
  int per_sm = 512 / threads;
  if (per_sm > 16) per_sm = 16;
  if (per_sm < 1) per_sm = 1;
  const int most = kNumSms * per_sm;
  return tokens < most ? tokens : most;
}

// Shared memory of a streamed kernel, granted once per device.
template <auto kKernel>
bool allow_ring() {
  static std::mutex mutex;
  static bool done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
  std::lock_guard<std::mutex> lock(mutex);
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kRingBytes)) != cudaSuccess) {
      cudaGetLastError();
      return false;
    }
    done[dev] = true;
  }
  return true;
}

// Where the rings pay in the forward pass: they have to fill first, and rows that
// still lie in L2 come as fast without them. Crossovers in bytes moved: aligned
// rows 50 to 100 MB (top 2, plain against streamed: bf16, N=2048, 2400 tokens 14.4
// against 16.4 us, 4800 33 against 27; FP32, N=4096, 600 tokens 9.8 against 12.5, 1200
// 22 against 21), others, which the plain form reads in single elements, earlier: bf16
// at 6 MB (N=1027, 600 tokens 13.2 against 12.9; N=2051, 300 tokens 16.6 against 12.5), FP32
// at 32 MB (N=1027, 1200 tokens 14.4 against 15.4, 2400 24 against 23); always with two
// tokens per SM (bf16, N=4095, 148 tokens 8.4 against 11.5). Short aligned rows are a
// warp's work with one load per thread and row, and stay so (32768 tokens, N=256: FP32
// 35 against 50 us).
bool forward_streams(const UnpermuteNorm& in, std::size_t unit, std::size_t size) {
  if (in.output <= 256 && unit == 16) return false;
  const double moved = (in.top_k + 3.0) * in.tokens * in.output * size;
  return in.tokens >= 2 * kNumSms && moved >= (unit == 16 ? 64e6 : size == 4 ? 32e6 : 6e6);
}

// In the gradient the streamed form needs one reduction where the plain one needs
// two and reads a token's rows once, so it pays from about a token per SM (N=512, 148
// tokens: FP32 8.8 us either way, 600 tokens 12.8 against 9.6; N=4096, 148 tokens: bf16
// 26 against 17, 37 tokens 16.6 against 15.0), for rows of single elements always
// (N=1027, one token: bf16 12.9 against 9.0), for rows of a few elements per thread
// later (N=64: 600 tokens 7.9 against 9.0, 1200 10.7 against 9.2), and for those that
// take sixteen from two tokens per SM (bf16, N=6363: 148 tokens 25 against 34, 600
// 89 against 72).
bool backward_streams(const UnpermuteNorm& in, std::size_t unit) {
  if (in.output <= 128) return in.tokens >= 8 * kNumSms;
  if (in.output > kStreamThreads * 8) return in.tokens >= 2 * kNumSms;
  return unit < 16 || in.tokens >= kNumSms;
}

// Columns handled together by the streamed form: 16 bytes where rows are a
// multiple of that, pairs of bfloat16 in rows of even length, else one.
int stream_columns(int output, Dtype dtype) {
  if (output * dtype_bytes(dtype) % 16 == 0) return static_cast<int>(16 / dtype_bytes(dtype));
  return dtype == Dtype::kBf16 && output % 2 == 0 ? 2 : 1;
}

bool aligned_gammas(const UnpermuteNorm& in, int columns) {
  return columns < 4 || (aligned_to(in.post_gamma, 16) && aligned_to(in.gate, 16) &&
                         aligned_to(in.pre_gamma, 16));
}

bool aligned_rows(const UnpermuteNorm& in, Dtype dtype) {
  return (in.output * dtype_bytes(dtype)) % 16 == 0 && aligned_to(in.y_permuted, 16) &&
         aligned_to(in.residual, 16) && aligned_gammas(in, 4);
}

template <typename T, int kPer>
cudaError_t forward(const UnpermuteNorm& in, void* residual_out, void* normed, float* inv_rms,
                    cudaStream_t stream) {
  // Eight columns per thread while the block stays at 512 threads; four where short rows
  // are read in single elements and there is a token per SM at most (one token, FP32:
  // N=333 4.5 against 5.6 us, N=1027 4.9 against 5.3, N=2051 6.6 against 5.8).
  const bool spread = kPer == 1 && in.output <= 1536 && in.tokens <= kNumSms;
  int threads = row_threads(in.output, spread ? 4 : 8);
  if (threads > 512) threads = row_threads(in.output, kElems);
  auto* kernel = threads <= 512 ? unpermute_norm_kernel<T, kPer, 512>
                                : unpermute_norm_kernel<T, kPer, 1024>;
  // Tokens of one warp share blocks once there are several per SM: starting a
  // block takes longer than such a row (bf16, 65536 tokens: N=256 56 against 71 us, N=64 36
  // against 69).
  const int share = threads == 32 && in.tokens > 4 * kNumSms ? 8 : 1;
  return launch_following(kernel, dim3(ceil_div(in.tokens, share)), dim3(threads, share), 0, 0,
                          stream, in, static_cast<T*>(residual_out), static_cast<T*>(normed),
                          inv_rms);
}

cudaError_t column_sums(const float* workspace, int parts, int output,
                        const UnpermuteNormGrads& g, cudaStream_t stream) {
  if (g.d_post_gamma == nullptr && g.d_gate == nullptr && g.d_pre_gamma == nullptr) {
    return cudaSuccess;
  }
  return launch_following(column_sums_kernel, dim3(ceil_div(output, kSumCols), 3),
                          kSumCols * kSumGroups, 0, 0, stream, workspace, parts, output,
                          g.d_post_gamma, g.d_gate, g.d_pre_gamma);
}

template <typename T, int kPer>
cudaError_t backward(const UnpermuteNorm& in, const UnpermuteNormGrads& g, float* workspace,
                     cudaStream_t stream) {
  const int threads = row_threads(in.output, kElems);
  const int blocks = backward_blocks(in.tokens, in.output);
  auto* kernel = threads <= 512 ? unpermute_norm_backward_kernel<T, kPer, 512>
                                : unpermute_norm_backward_kernel<T, kPer, 1024>;
  const cudaError_t e =
      launch_following(kernel, dim3(blocks), threads, 0, 0, stream, in, g, workspace);
  if (e != cudaSuccess) return e;
  return column_sums(workspace, blocks, in.output, g, stream);
}

template <typename T, int kPer>
cudaError_t forward_stream(const UnpermuteNorm& in, const Stream& st, void* residual_out,
                           void* normed, float* inv_rms, cudaStream_t stream) {
  constexpr auto kernel = unpermute_norm_stream_kernel<T, kPer>;
  if (!allow_ring<kernel>()) return cudaErrorNotSupported;
  return launch_following(kernel, dim3(st.blocks), st.team * st.teams, ring_bytes(st), 0, stream,
                          in, st, static_cast<T*>(residual_out), static_cast<T*>(normed), inv_rms,
                          device_error_word());
}

template <typename T, int kPer>
cudaError_t backward_stream(const UnpermuteNorm& in, const Stream& st, const UnpermuteNormGrads& g,
                            float* workspace, cudaStream_t stream) {
  constexpr auto narrow2 = unpermute_norm_backward_stream_kernel<T, kPer, 8, true>;
  constexpr auto narrow = unpermute_norm_backward_stream_kernel<T, kPer, 8, false>;
  constexpr auto wide = unpermute_norm_backward_stream_kernel<T, kPer, 16, false>;
  const bool eight = gradient_elems(in.output) == 8, two = in.top_k <= 2;
  if (!(eight ? (two ? allow_ring<narrow2>() : allow_ring<narrow>()) : allow_ring<wide>())) {
    return cudaErrorNotSupported;
  }
  auto* kernel = eight ? (two ? narrow2 : narrow) : wide;
  const cudaError_t e = launch_following(kernel, dim3(st.blocks), st.team * st.teams,
                                         ring_bytes(st), 0, stream, in, st, g, workspace,
                                         device_error_word());
  if (e != cudaSuccess) return e;
  return column_sums(workspace, st.blocks, in.output, g, stream);
}

}  // namespace

cudaError_t launch_unpermute_norm(const UnpermuteNorm& in, void* residual_out, void* normed,
                                  float* inv_rms, Dtype dtype, cudaStream_t stream) {
  const Stream st = stream_plan(in.tokens, in.top_k, in.output, 1, false, kElems, dtype_bytes(dtype));
  const int per = stream_columns(in.output, dtype);
  const std::size_t unit = per * dtype_bytes(dtype);
  if (st.blocks > 0 && forward_streams(in, unit, dtype_bytes(dtype)) &&
      aligned_to(in.y_permuted, 16) && aligned_to(in.residual, 16) && aligned_gammas(in, per) &&
      aligned_to(residual_out, unit) && aligned_to(normed, unit)) {
    if (dtype == Dtype::kBf16) {
      auto* run = per == 8   ? forward_stream<__nv_bfloat16, 8>
                  : per == 2 ? forward_stream<__nv_bfloat16, 2>
                             : forward_stream<__nv_bfloat16, 1>;
      return run(in, st, residual_out, normed, inv_rms, stream);
    }
    auto* run = per == 4 ? forward_stream<float, 4> : forward_stream<float, 1>;
    return run(in, st, residual_out, normed, inv_rms, stream);
  }
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
  // Shares of the column sums: of the plain form's blocks or the streamed
  // form's, whichever are more.
  std::size_t parts = static_cast<std::size_t>(backward_blocks(tokens, output));
  if (parts < kNumSms && tokens >= kNumSms) parts = kNumSms;
  return 12 * parts * output;
}

cudaError_t launch_unpermute_norm_backward(const UnpermuteNorm& in, const UnpermuteNormGrads& g,
                                           float* workspace, Dtype dtype, cudaStream_t stream) {
  const int extra = 1 + (g.d_residual_out != nullptr) + (in.pre_gamma != nullptr);
  const Stream st = stream_plan(in.tokens, in.top_k, in.output, extra, true,
                                gradient_elems(in.output), dtype_bytes(dtype));
  const int per = stream_columns(in.output, dtype);
  const std::size_t unit = per * dtype_bytes(dtype);
  if (st.blocks > 0 && backward_streams(in, unit) && aligned_to(in.y_permuted, 16) &&
      aligned_to(in.residual, 16) && aligned_to(g.d_residual_out, 16) &&
      aligned_to(g.d_normed, 16) && aligned_gammas(in, per) && aligned_to(g.d_residual, unit) && aligned_to(g.d_y_permuted, unit)) {
    if (dtype == Dtype::kBf16) {
      auto* run = per == 8   ? backward_stream<__nv_bfloat16, 8>
                  : per == 2 ? backward_stream<__nv_bfloat16, 2>
                             : backward_stream<__nv_bfloat16, 1>;
      return run(in, st, g, workspace, stream);
    }
    auto* run = per == 4 ? backward_stream<float, 4> : backward_stream<float, 1>;
    return run(in, st, g, workspace, stream);
  }
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

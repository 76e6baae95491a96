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
// one persistent block per SM therefore streams the rows of the next tokens
// into shared memory with bulk copies (a producer warp, a ring of stages)
// while teams of 32 to 512 threads work on the current ones; rows of any
// alignment are copied as the 16-byte granules they touch. Fewer tokens, and
// rows too wide for the ring, take one plain block per token.
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

// ---- streamed form ------------------------------------------------------------------

constexpr int kWorkers = 512;                   // worker threads per block, at most
constexpr int kStreamThreads = kWorkers + 32;   // and the producer warp
constexpr int kStreamTopK = 16;
constexpr int kMaxStages = 4;
constexpr int kRounds = 3;                      // rows of a stage per producer lane
constexpr int kMaxTeams = kWorkers / 32;
constexpr std::size_t kRingBytes = 200 * 1024;

// A stage holds the rows of one token per team: the route rows, the residual,
// and for the gradient d_residual_out and d_normed.
struct Stream {
  int team = 0;      // threads per token
  int teams = 0;     // tokens per stage
  int sources = 0;   // rows per token
  int stride = 0;    // bytes of a row's place
  int padded = 0;    // gradient: columns of the factors behind the ring
  int stages = 0;
  int blocks = 0;
};

struct StreamSmem {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  int failed;
  // What the producer knows of each token: where in its place a row starts
  // (-1: a skipped route), and the route weights.
  int start[kMaxStages][kMaxTeams][kStreamTopK + 3];
  float weight[kMaxStages][kMaxTeams][kStreamTopK];
  int pos[kMaxStages][kMaxTeams][kStreamTopK];
  float parts[2][kMaxTeams][kStreamTopK + 1];  // of each warp, two reductions
};

// The threads of one team (a barrier of its own each; one warp needs none).
__device__ __forceinline__ void team_sync(int team, int threads) {
  if (threads == 32) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(threads) : "memory");
}

// Whether `ok` holds in every thread of the team.
__device__ __forceinline__ bool team_all(int team, int threads, bool ok) {
  if (threads == 32) return __all_sync(0xffffffffu, ok);
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "bar.red.and.pred q, %1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(team + 1), "r"(threads), "r"(static_cast<int>(ok))
      : "memory");
  return r != 0;
}

struct Sources {
  const void* row[3] = {};  // residual, d_residual_out, d_normed; null ones left out
  int count = 0;
};

// Streams the rows of this block's tokens. Lanes share the rows of a stage, up
// to kRounds each; a route's position and weight are fetched one stage ahead.
template <typename T>
__device__ __forceinline__ void produce(const UnpermuteNorm& in, const Sources& src,
                                        const Stream& st, StreamSmem& s, uint32_t ring,
                                        unsigned* err) {
  using namespace sm100;
  const int lane = threadIdx.x & 31;
  const long long routes = static_cast<long long>(in.tokens) * in.top_k;
  const long long bytes = static_cast<long long>(in.output) * sizeof(T);
  const int items = st.teams * st.sources;
  const long long step = static_cast<long long>(gridDim.x) * st.teams;
  int team[kRounds], r[kRounds], pos[kRounds];
  float weight[kRounds];
#pragma unroll
  for (int j = 0; j < kRounds; ++j) {
    team[j] = (lane + 32 * j) / st.sources;
    r[j] = lane + 32 * j - team[j] * st.sources;
  }
  auto fetch = [&](long long first) {
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      const long long t = first + team[j];
      pos[j] = -1;
      weight[j] = 0.0f;
      if (lane + 32 * j < items && r[j] < in.top_k && t < in.tokens) {
        pos[j] = __ldg(in.route_pos + t * in.top_k + r[j]);
        weight[j] = __ldg(in.route_weights + t * in.top_k + r[j]);
      }
    }
  };
  int stage = 0;
  uint32_t phase = 0;
  long long first = static_cast<long long>(blockIdx.x) * st.teams;
  fetch(first);
  for (; first < in.tokens; first += step) {
    if (!mbar_wait(&s.empty[stage], phase ^ 1u, err, &s.failed)) return;
    const char* from[kRounds];
    uint32_t size[kRounds], place[kRounds], total = 0;
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      size[j] = 0;
      const int i = lane + 32 * j;
      const long long t = first + team[j];
      if (i >= items || t >= in.tokens) continue;
      long long row = t, rows = in.tokens;
      const char* base;
      if (r[j] < in.top_k) {
        row = pos[j];
        rows = routes;
        base = static_cast<const char*>(in.y_permuted);
        s.weight[stage][team[j]][r[j]] = weight[j];
        s.pos[stage][team[j]][r[j]] = pos[j];
        if (row < 0 || row >= routes) {
          s.start[stage][team[j]][r[j]] = -1;
          continue;
        }
      } else {
        base = static_cast<const char*>(src.row[r[j] - in.top_k]);
      }
      // The granules of the row. The buffers start on a 16-byte boundary, so
      // only the last row's last granule can reach past one; its elements are
      // copied one by one.
      const long long at = row * bytes;
      const long long a0 = at & ~15LL;
      long long a1 = (at + bytes + 15) & ~15LL;
      const bool past = a1 > rows * bytes;
      if (past) a1 -= 16;
      place[j] = (stage * items + i) * st.stride;
      s.start[stage][team[j]][r[j]] = static_cast<int>(place[j] + (at - a0));
      from[j] = base + a0;
      size[j] = a1 > a0 ? static_cast<uint32_t>(a1 - a0) : 0u;
      total += size[j];
      if (past) {
        for (long long b = a1 > at ? a1 : at; b < at + bytes; b += sizeof(T)) {
          const uint32_t to = ring + place[j] + static_cast<uint32_t>(b - a0);
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
      }
    }
    total = __reduce_add_sync(0xffffffffu, total);
    __syncwarp();  // the lanes' notes come before the arrival
    if (lane == 0) mbar_arrive_expect_tx(&s.full[stage], total);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kRounds; ++j) {
      if (size[j] > 0) bulk_load(ring + place[j], from[j], size[j], &s.full[stage]);
    }
    fetch(first + step);
    if (++stage == st.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
}

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

__device__ __forceinline__ void stream_setup(const Stream& st, StreamSmem& s) {
  using namespace sm100;
  if (threadIdx.x == 0) {
    for (int i = 0; i < st.stages; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], st.team * st.teams / 32);
    }
    s.failed = 0;
    fence_mbar_init();
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

template <typename T, int kPer>
__global__ void __launch_bounds__(kStreamThreads, 1) unpermute_norm_stream_kernel(
    const UnpermuteNorm in, const Stream st, T* residual_out, T* normed, float* inv_rms,
    unsigned* err) {
  using namespace sm100;
  extern __shared__ __align__(16) char ring[];
  __shared__ StreamSmem s;
  stream_setup(st, s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x >= st.team * st.teams) {
    Sources src;
    src.row[0] = in.residual;
    produce<T>(in, src, st, s, smem_u32(ring), err);
    stream_end(s);
    return;
  }
  const int team = threadIdx.x / st.team, tid = threadIdx.x % st.team;
  const int team_warps = st.team >> 5, warp0 = team * team_warps;
  const float per_col = 1.0f / static_cast<float>(in.output);
  float pg[kElems], pr[kElems];  // post * gate and pre of this thread's columns
#pragma unroll
  for (int q = 0; q < kElems / kPer; ++q) {
    column_factors<kPer>(in, (q * st.team + tid) * kPer, pg + q * kPer, pr + q * kPer);
  }
  int stage = 0;
  uint32_t phase = 0;
  const long long step = static_cast<long long>(gridDim.x) * st.teams;
  for (long long first = static_cast<long long>(blockIdx.x) * st.teams; first < in.tokens;
       first += step) {
    const bool ok = mbar_wait(&s.full[stage], phase, err, &s.failed);
    if (!team_all(team, st.team, ok)) break;
    const long long t = first + team;
    if (t < in.tokens) {  // uniform over a team
      const int* start = s.start[stage][team];
      float c[kElems];
      staged_combine<T, kPer>(in, st, ring, start, s.weight[stage][team], tid, c);
      auto team_sum = [&](float v, int which) {
        v = warp_sum(v);
        if (team_warps == 1) return v;
        if (lane == 0) s.parts[which][warp][0] = v;
        team_sync(team, st.team);
        float sum = 0.0f;
        for (int w = 0; w < team_warps; ++w) sum += s.parts[which][warp0 + w][0];
        return sum;
      };
      float i1 = 1.0f;
      if (in.post_gamma != nullptr) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < kElems; ++i) sq = fmaf(c[i], c[i], sq);
        i1 = rsqrtf(team_sum(sq, 0) * per_col + in.eps);
      }
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
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[stage]);
      float i2 = 1.0f;
      if (in.pre_gamma != nullptr) {
        i2 = rsqrtf(team_sum(sq, 1) * per_col + in.eps);
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
    } else {
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.empty[stage]);
    }
    if (++stage == st.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  stream_end(s);
}

// The gradient, with two reductions per token: the first of <v, rn> and of
// Q_k = <cn, y_k>, the second of <v1, cn> and of P_k = <v1, y_k>, where
// v1 = db post; then dw_k = <dc, y_k> = i1 (P_k - mean(v1 cn) Q_k) needs no
// third (without the norm of c: dc = v1, dw_k = P_k). The gradients of post and
// gate are one column sum, of dr cn, times the other factor. post * gate and
// pre lie in shared memory behind the ring: read from the caller's buffers for
// every token they would be as many bytes as its rows.
template <typename T, int kPer>
__global__ void __launch_bounds__(kStreamThreads, 1) unpermute_norm_backward_stream_kernel(
    const UnpermuteNorm in, const Stream st, const UnpermuteNormGrads g, float* partial,
    unsigned* err) {
  using namespace sm100;
  extern __shared__ __align__(16) char ring[];
  __shared__ StreamSmem s;
  const bool post = in.post_gamma != nullptr, pre = in.pre_gamma != nullptr;
  const bool has_dro = g.d_residual_out != nullptr;
  float* pg = reinterpret_cast<float*>(ring + st.stages * st.teams * st.sources * st.stride);
  float* pr = pg + st.padded;
  for (int c = threadIdx.x; c < st.padded; c += blockDim.x) {
    column_factors<1>(in, c, pg + c, pr + c);
  }
  stream_setup(st, s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x >= st.team * st.teams) {
    Sources src;
    src.row[src.count++] = in.residual;
    if (has_dro) src.row[src.count++] = g.d_residual_out;
    if (pre) src.row[src.count++] = g.d_normed;
    produce<T>(in, src, st, s, smem_u32(ring), err);
    stream_end(s);
    return;
  }
  const int team = threadIdx.x / st.team, tid = threadIdx.x % st.team;
  const int team_warps = st.team >> 5, warp0 = team * team_warps;
  const float per_col = 1.0f / static_cast<float>(in.output);
  const int at_res = in.top_k, at_dro = in.top_k + 1, at_dn = in.top_k + 1 + (has_dro ? 1 : 0);
  float s_dc[kElems], s_pre[kElems];  // sums over tokens of dr cn and dn rn
#pragma unroll
  for (int i = 0; i < kElems; ++i) s_dc[i] = s_pre[i] = 0.0f;
  int stage = 0;
  uint32_t phase = 0;
  const long long step = static_cast<long long>(gridDim.x) * st.teams;
  for (long long first = static_cast<long long>(blockIdx.x) * st.teams; first < in.tokens;
       first += step) {
    const bool ok = mbar_wait(&s.full[stage], phase, err, &s.failed);
    if (!team_all(team, st.team, ok)) break;
    const long long t = first + team;
    if (t < in.tokens) {  // uniform over a team
      const int* start = s.start[stage][team];
      const float* weight = s.weight[stage][team];
      // Sums of the team's warps are kept as parts[which][warp][j].
      auto part = [&](float v, int which, int j) {
        v = warp_sum(v);
        if (lane == 0) s.parts[which][warp][j] = v;
      };
      auto total = [&](int which, int j) {
        float sum = 0.0f;
        for (int w = 0; w < team_warps; ++w) sum += s.parts[which][warp0 + w][j];
        return sum;
      };
      // <x, y_k> of this thread's columns.
      auto route_dot = [&](const float (&x)[kElems], int k) {
        float d = 0.0f;
        if (start[k] >= 0) {
#pragma unroll
          for (int q = 0; q < kElems / kPer; ++q) {
            const int col = (q * st.team + tid) * kPer;
            if (col < in.output) {
              float v[kPer];
              staged_cols<T, kPer>(ring + start[k] + col * sizeof(T), v);
#pragma unroll
              for (int i = 0; i < kPer; ++i) d = fmaf(x[q * kPer + i], v[i], d);
            }
          }
        }
        return d;
      };
      const float i1 = post ? __ldg(g.inv_rms + 2 * t) : 1.0f;
      const float i2 = pre ? __ldg(g.inv_rms + 2 * t + 1) : 0.0f;
      float c[kElems];  // cn
      staged_combine<T, kPer>(in, st, ring, start, weight, tid, c);
#pragma unroll
      for (int i = 0; i < kElems; ++i) c[i] *= i1;
      // rn of kPer columns, from the staged residual and cn.
      auto normalised = [&](int q, int col, const float* f, float* rn) {
        staged_cols<T, kPer>(ring + start[at_res] + col * sizeof(T), rn);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          rn[i] = fmaf(in.residual_scale, rn[i], c[q * kPer + i] * f[i]) * i2;
        }
      };
      float dot = 0.0f;
      if (pre) {
#pragma unroll
        for (int q = 0; q < kElems / kPer; ++q) {
          const int col = (q * st.team + tid) * kPer;
          if (col < in.output) {
            float f[kPer], rn[kPer], v[kPer];
            shared_cols<kPer>(pg + col, f);
            normalised(q, col, f, rn);
            staged_cols<T, kPer>(ring + start[at_dn] + col * sizeof(T), v);
            shared_cols<kPer>(pr + col, f);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              s_pre[q * kPer + i] = fmaf(v[i], rn[i], s_pre[q * kPer + i]);
              dot = fmaf(v[i] * f[i], rn[i], dot);
            }
          }
        }
      }
      part(dot, 0, 0);
      if (post) {
        for (int k = 0; k < in.top_k; ++k) part(route_dot(c, k), 0, k + 1);
      }
      team_sync(team, st.team);
      const float m2 = total(0, 0) * per_col;
      float dr[kElems];  // v1
      dot = 0.0f;
#pragma unroll
      for (int q = 0; q < kElems / kPer; ++q) {
        const int col = (q * st.team + tid) * kPer;
        float* d = dr + q * kPer;
#pragma unroll
        for (int i = 0; i < kPer; ++i) d[i] = 0.0f;
        if (col < in.output) {
          float f[kPer], out[kPer];
          if (has_dro) staged_cols<T, kPer>(ring + start[at_dro] + col * sizeof(T), d);
          shared_cols<kPer>(pg + col, f);
          if (pre) {
            float rn[kPer], v[kPer], a[kPer];
            normalised(q, col, f, rn);
            staged_cols<T, kPer>(ring + start[at_dn] + col * sizeof(T), v);
            shared_cols<kPer>(pr + col, a);
#pragma unroll
            for (int i = 0; i < kPer; ++i) d[i] += i2 * (v[i] * a[i] - rn[i] * m2);
          }
#pragma unroll
          for (int i = 0; i < kPer; ++i) out[i] = in.residual_scale * d[i];
          put_cols<T, kPer>(static_cast<T*>(g.d_residual) + t * in.output + col, out);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            s_dc[q * kPer + i] = fmaf(d[i], c[q * kPer + i], s_dc[q * kPer + i]);
            d[i] *= f[i];
            dot = fmaf(d[i], c[q * kPer + i], dot);
          }
        }
      }
      part(dot, 1, 0);
      for (int k = 0; k < in.top_k; ++k) part(route_dot(dr, k), 1, k + 1);
      team_sync(team, st.team);
      const float m1 = post ? total(1, 0) * per_col : 0.0f;
#pragma unroll
      for (int i = 0; i < kElems; ++i) dr[i] = i1 * (dr[i] - c[i] * m1);
      for (int k = 0; k < in.top_k; ++k) {
        const bool there = start[k] >= 0;
        if (tid == k) {
          const float p = total(1, k + 1);
          g.d_route_weights[t * in.top_k + k] =
              !there ? 0.0f : (post ? i1 * (p - m1 * total(0, k + 1)) : p);
        }
        if (!there) continue;
        const float w = weight[k];
        T* row = static_cast<T*>(g.d_y_permuted) +
                 static_cast<long long>(s.pos[stage][team][k]) * in.output;
#pragma unroll
        for (int q = 0; q < kElems / kPer; ++q) {
          const int col = (q * st.team + tid) * kPer;
          if (col < in.output) {
            float out[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) out[i] = w * dr[q * kPer + i];
            put_cols<T, kPer>(row + col, out);
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.empty[stage]);
    if (++stage == st.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // This team's shares of the column sums: [block * teams + team][3][output].
  float* p = partial + 3LL * (static_cast<long long>(blockIdx.x) * st.teams + team) * in.output;
#pragma unroll
  for (int q = 0; q < kElems / kPer; ++q) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int col = (q * st.team + tid) * kPer + i;
      if (col < in.output) {
        const float d = s_dc[q * kPer + i];
        p[col] = in.gate != nullptr ? d * __ldg(in.gate + col) : d;
        p[in.output + col] = post ? d * __ldg(in.post_gamma + col) : d;
        p[2 * in.output + col] = s_pre[q * kPer + i];
      }
    }
  }
  stream_end(s);
}

// ---- the gradient for one or two routes per token ----------------------------------
//
// The same in one pass over the inputs and one reduction. With a = dro + i2 v
// (v = dn pre) and f = post * gate:
//   dr = a - i2 m2 rn,  v1 = f dr,  m2 = mean(v rn)
//   P_k = <v1, y_k> = <f a, y_k> - i2 m2 <f rn, y_k>
//   mean(v1 cn) = i1 sum_k w_k P_k / N,  Q_k = <cn, y_k> = i1 sum_j w_j <y_j, y_k>
// so a token's eight sums are known together, before any of its results. Two
// columns share an instruction (packed FP32 arithmetic, which rounds each half
// as the plain instruction does).

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

// Eight columns per thread: a token's c, a and rn and the thread's column sums
// then stay in registers with sixteen warps per SM (sixteen columns spilled,
// and eight warps leave too little to overlap).
constexpr int kPairElems = 8;
constexpr int kPairs = kPairElems / 2;

// This thread's columns of a staged row in pairs, zero past the row's end.
template <typename T, int kPer>
__device__ __forceinline__ void staged_row(const char* row, int output, int team, int tid,
                                           F2 (&v)[kPairs]) {
  float f[kPairElems];
#pragma unroll
  for (int q = 0; q < kPairElems / kPer; ++q) {
    const int col = (q * team + tid) * kPer;
    if (col < output) {
      staged_cols<T, kPer>(row + col * sizeof(T), f + q * kPer);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) f[q * kPer + i] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}

template <int kPer>
__device__ __forceinline__ void shared_row(const float* row, int output, int team, int tid,
                                           F2 (&v)[kPairs]) {
  float f[kPairElems];
#pragma unroll
  for (int q = 0; q < kPairElems / kPer; ++q) {
    const int col = (q * team + tid) * kPer;
    if (col < output) {
      shared_cols<kPer>(row + col, f + q * kPer);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) f[q * kPer + i] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}

template <typename T, int kPer>
__device__ __forceinline__ void put_row(T* row, int output, int team, int tid,
                                        const F2 (&v)[kPairs]) {
  float f[kPairElems];
#pragma unroll
  for (int i = 0; i < kPairs; ++i) split(v[i], f[2 * i], f[2 * i + 1]);
#pragma unroll
  for (int q = 0; q < kPairElems / kPer; ++q) {
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

template <typename T, int kPer>
__global__ void __launch_bounds__(kStreamThreads, 1) unpermute_norm_backward_pair_kernel(
    const UnpermuteNorm in, const Stream st, const UnpermuteNormGrads g, float* partial,
    unsigned* err) {
  using namespace sm100;
  extern __shared__ __align__(16) char ring[];
  __shared__ StreamSmem s;
  __shared__ float sums[2][kMaxTeams][8];  // of each warp, by parity of the token
  const bool post = in.post_gamma != nullptr, pre = in.pre_gamma != nullptr;
  const bool has_dro = g.d_residual_out != nullptr;
  float* pg = reinterpret_cast<float*>(ring + st.stages * st.teams * st.sources * st.stride);
  float* pr = pg + st.padded;
  for (int c = threadIdx.x; c < st.padded; c += blockDim.x) {
    column_factors<1>(in, c, pg + c, pr + c);
  }
  stream_setup(st, s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x >= st.team * st.teams) {
    Sources src;
    src.row[src.count++] = in.residual;
    if (has_dro) src.row[src.count++] = g.d_residual_out;
    if (pre) src.row[src.count++] = g.d_normed;
    produce<T>(in, src, st, s, smem_u32(ring), err);
    stream_end(s);
    return;
  }
  const int team = threadIdx.x / st.team, tid = threadIdx.x % st.team;
  const int team_warps = st.team >> 5, warp0 = team * team_warps;
  const int n = in.output;
  const float per_col = 1.0f / static_cast<float>(n);
  const int at_res = in.top_k, at_dro = in.top_k + 1, at_dn = in.top_k + 1 + (has_dro ? 1 : 0);
  F2 s_dc[kPairs], s_pre[kPairs];  // sums over tokens of dr cn and dn rn
#pragma unroll
  for (int i = 0; i < kPairs; ++i) s_dc[i] = s_pre[i] = f2(0.0f);
  int stage = 0, parity = 0;
  uint32_t phase = 0;
  const long long step = static_cast<long long>(gridDim.x) * st.teams;
  for (long long first = static_cast<long long>(blockIdx.x) * st.teams; first < in.tokens;
       first += step) {
    const bool ok = mbar_wait(&s.full[stage], phase, err, &s.failed);
    if (!team_all(team, st.team, ok)) break;
    const long long t = first + team;
    if (t < in.tokens) {  // uniform over a team
      const int* start = s.start[stage][team];
      const bool there0 = start[0] >= 0, there1 = in.top_k > 1 && start[1] >= 0;
      const float w0 = there0 ? s.weight[stage][team][0] : 0.0f;
      const float w1 = there1 ? s.weight[stage][team][1] : 0.0f;
      const float i1 = post ? __ldg(g.inv_rms + 2 * t) : 1.0f;
      const float i2 = pre ? __ldg(g.inv_rms + 2 * t + 1) : 0.0f;
      F2 c[kPairs], a[kPairs], rn[kPairs];
      float v8[8];  // <v, rn>, <f a, y0>, <f a, y1>, <f rn, y0>, <f rn, y1>, <y0, y0>, ...
      {
        F2 y0[kPairs], y1[kPairs], x[kPairs], f[kPairs], sum[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] = f2(0.0f);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) y0[i] = y1[i] = f2(0.0f);
        if (there0) staged_row<T, kPer>(ring + start[0], n, st.team, tid, y0);
        if (there1) staged_row<T, kPer>(ring + start[1], n, st.team, tid, y1);
        shared_row<kPer>(pg, n, st.team, tid, f);
        staged_row<T, kPer>(ring + start[at_res], n, st.team, tid, x);
        const F2 w02 = f2(w0), w12 = f2(w1), i12 = f2(i1), i22 = f2(i2);
        const F2 scale = f2(in.residual_scale);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          c[i] = mul2(i12, fma2(w12, y1[i], mul2(w02, y0[i])));
          rn[i] = mul2(i22, fma2(scale, x[i], mul2(c[i], f[i])));
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
          shared_row<kPer>(pr, n, st.team, tid, p);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            s_pre[i] = fma2(x[i], rn[i], s_pre[i]);
            const F2 v = mul2(x[i], p[i]);
            sum[0] = fma2(v, rn[i], sum[0]);
            a[i] = fma2(i22, v, a[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const F2 fa = mul2(f[i], a[i]), fr = mul2(f[i], rn[i]);
          sum[1] = fma2(fa, y0[i], sum[1]);
          sum[2] = fma2(fa, y1[i], sum[2]);
          sum[3] = fma2(fr, y0[i], sum[3]);
          sum[4] = fma2(fr, y1[i], sum[4]);
          sum[5] = fma2(y0[i], y0[i], sum[5]);
          sum[6] = fma2(y0[i], y1[i], sum[6]);
          sum[7] = fma2(y1[i], y1[i], sum[7]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v8[j] = sum2(sum[j]);
      }
      // The team's sums: lane l of every warp ends with the sum l / 4.
      float mine = warp_sum8(v8);
      if (team_warps > 1) {
        if ((lane & 3) == 0) sums[parity][warp][lane >> 2] = mine;
        team_sync(team, st.team);
        mine = 0.0f;
        for (int w = lane & 3; w < team_warps; w += 4) mine += sums[parity][warp0 + w][lane >> 2];
        mine += __shfl_xor_sync(0xffffffffu, mine, 1);
        mine += __shfl_xor_sync(0xffffffffu, mine, 2);
        parity ^= 1;
      }
      auto total = [&](int j) { return __shfl_sync(0xffffffffu, mine, 4 * j); };
      const float im2 = i2 * (total(0) * per_col);
      const float p0 = total(1) - im2 * total(3), p1 = total(2) - im2 * total(4);
      const float g00 = total(5), g01 = total(6), g11 = total(7);
      const float m1 = post ? i1 * (w0 * p0 + w1 * p1) * per_col : 0.0f;
      if (tid == 0) {
        const float q0 = i1 * (w0 * g00 + w1 * g01), q1 = i1 * (w0 * g01 + w1 * g11);
        float* dw = g.d_route_weights + t * in.top_k;
        dw[0] = there0 ? i1 * (p0 - m1 * q0) : 0.0f;
        if (in.top_k > 1) dw[1] = there1 ? i1 * (p1 - m1 * q1) : 0.0f;
      }
      {
        F2 x[kPairs];
        const F2 nim2 = f2(-im2), scale = f2(in.residual_scale);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          a[i] = fma2(nim2, rn[i], a[i]);  // dr
          s_dc[i] = fma2(a[i], c[i], s_dc[i]);
          x[i] = mul2(scale, a[i]);
        }
        put_row<T, kPer>(static_cast<T*>(g.d_residual) + t * n, n, st.team, tid, x);
        shared_row<kPer>(pg, n, st.team, tid, x);
        const F2 i12 = f2(i1), nm1 = f2(-m1);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          a[i] = mul2(i12, fma2(nm1, c[i], mul2(x[i], a[i])));  // dc
        }
        T* rows = static_cast<T*>(g.d_y_permuted);
        if (there0) {
          const F2 w = f2(w0);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) x[i] = mul2(w, a[i]);
          put_row<T, kPer>(rows + static_cast<long long>(s.pos[stage][team][0]) * n, n, st.team,
                           tid, x);
        }
        if (there1) {
          const F2 w = f2(w1);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) x[i] = mul2(w, a[i]);
          put_row<T, kPer>(rows + static_cast<long long>(s.pos[stage][team][1]) * n, n, st.team,
                           tid, x);
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&s.empty[stage]);
    if (++stage == st.stages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // This team's shares of the column sums: [block * teams + team][3][output].
  float* p = partial + 3LL * (static_cast<long long>(blockIdx.x) * st.teams + team) * n;
#pragma unroll
  for (int i = 0; i < kPairElems; ++i) {
    const int col = ((i / kPer) * st.team + tid) * kPer + i % kPer;
    if (col < n) {
      float lo, hi;
      split(s_dc[i / 2], lo, hi);
      const float d = i % 2 ? hi : lo;
      split(s_pre[i / 2], lo, hi);
      p[col] = in.gate != nullptr ? d * __ldg(in.gate + col) : d;
      p[n + col] = post ? d * __ldg(in.post_gamma + col) : d;
      p[2 * n + col] = i % 2 ? hi : lo;
    }
  }
  stream_end(s);
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

// The streamed form's layout, or blocks = 0 where the plain one runs: few
// tokens (the ring has to fill before it pays: two stages per SM), more routes
// than a stage keeps track of, or rows of which two stages do not fit.
Stream stream_plan(int tokens, int top_k, int output, int extra_rows, bool gradient, int elems,
                   std::size_t size) {
  Stream st;
  if (top_k > kStreamTopK || output > kWorkers * elems) return st;
  st.team = row_threads(output, elems);
  st.teams = kWorkers / st.team;
  st.sources = top_k + extra_rows;
  if (st.teams * st.sources > 32 * kRounds) return st;
  // A row's granules: up to 15 bytes before and after it.
  st.stride = static_cast<int>((output * size + 15) / 16 * 16 + 16);
  if (gradient) st.padded = (output + 3) / 4 * 4;
  for (;; st.teams /= 2) {  // two stages have to fit: halve the teams until they do
    const std::size_t stage = static_cast<std::size_t>(st.teams) * st.sources * st.stride;
    st.stages = static_cast<int>((kRingBytes - 8 * st.padded) / stage);
    if (st.stages >= 2 || st.teams == 1) break;
  }
  if (st.stages > kMaxStages) st.stages = kMaxStages;
  const int fill = 2 * kNumSms * st.teams;
  if (st.stages >= 2 && tokens >= fill) st.blocks = kNumSms;
  return st;
}

std::size_t ring_bytes(const Stream& st) {
  return static_cast<std::size_t>(st.stages) * st.teams * st.sources * st.stride + 8 * st.padded;
}

// Columns per thread of the streamed gradient: one or two routes per token have
// a kernel of their own, up to the width its teams cover.
int gradient_elems(int top_k, int output) {
  return top_k <= 2 && output <= kWorkers * kPairElems ? kPairElems : kElems;
}

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

cudaError_t column_sums(const float* workspace, int parts, int output,
                        const UnpermuteNormGrads& g, cudaStream_t stream) {
  if (g.d_post_gamma != nullptr || g.d_gate != nullptr || g.d_pre_gamma != nullptr) {
    column_sums_kernel<<<dim3(ceil_div(output, kSumCols), 3), kSumThreads, 0, stream>>>(
        workspace, parts, output, g.d_post_gamma, g.d_gate, g.d_pre_gamma);
    note_launch();
  }
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
  return column_sums(workspace, blocks, in.output, g, stream);
}

template <typename T, int kPer>
cudaError_t forward_stream(const UnpermuteNorm& in, const Stream& st, void* residual_out,
                           void* normed, float* inv_rms, cudaStream_t stream) {
  constexpr auto kernel = unpermute_norm_stream_kernel<T, kPer>;
  if (!allow_ring<kernel>()) return cudaErrorNotSupported;
  kernel<<<st.blocks, st.team * st.teams + 32, ring_bytes(st), stream>>>(
      in, st, static_cast<T*>(residual_out), static_cast<T*>(normed), inv_rms,
      device_error_word());
  note_launch();
  return cudaGetLastError();
}

template <typename T, int kPer>
cudaError_t backward_stream(const UnpermuteNorm& in, const Stream& st, const UnpermuteNormGrads& g,
                            float* workspace, cudaStream_t stream) {
  constexpr auto any = unpermute_norm_backward_stream_kernel<T, kPer>;
  constexpr auto pair = unpermute_norm_backward_pair_kernel<T, kPer>;
  const bool two = gradient_elems(in.top_k, in.output) == kPairElems;
  if (!(two ? allow_ring<pair>() : allow_ring<any>())) return cudaErrorNotSupported;
  (two ? pair : any)<<<st.blocks, st.team * st.teams + 32, ring_bytes(st), stream>>>(
      in, st, g, workspace, device_error_word());
  note_launch();
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return column_sums(workspace, st.blocks * st.teams, in.output, g, stream);
}

}  // namespace

cudaError_t launch_unpermute_norm(const UnpermuteNorm& in, void* residual_out, void* normed,
                                  float* inv_rms, Dtype dtype, cudaStream_t stream) {
  const Stream st = stream_plan(in.tokens, in.top_k, in.output, 1, false, kElems, dtype_bytes(dtype));
  const int per = stream_columns(in.output, dtype);
  const std::size_t unit = per * dtype_bytes(dtype);
  if (st.blocks > 0 && aligned_to(in.y_permuted, 16) && aligned_to(in.residual, 16) &&
      aligned_gammas(in, per) && aligned_to(residual_out, unit) && aligned_to(normed, unit)) {
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
  // form's teams, whichever is more.
  std::size_t parts = static_cast<std::size_t>(backward_blocks(tokens, output));
  const int elems = gradient_elems(1, output);
  if (output <= kWorkers * kElems) {
    const std::size_t teams = static_cast<std::size_t>(kNumSms) *
                              (kWorkers / row_threads(output, kElems));
    const std::size_t narrow = static_cast<std::size_t>(kNumSms) *
                               (kWorkers / row_threads(output, elems));
    const std::size_t most = teams > narrow ? teams : narrow;
    if (most > parts && tokens >= static_cast<long long>(narrow)) parts = most;
  }
  return 12 * parts * output;
}

cudaError_t launch_unpermute_norm_backward(const UnpermuteNorm& in, const UnpermuteNormGrads& g,
                                           float* workspace, Dtype dtype, cudaStream_t stream) {
  const int extra = 1 + (g.d_residual_out != nullptr) + (in.pre_gamma != nullptr);
  const Stream st = stream_plan(in.tokens, in.top_k, in.output, extra, true,
                                gradient_elems(in.top_k, in.output), dtype_bytes(dtype));
  const int per = stream_columns(in.output, dtype);
  const std::size_t unit = per * dtype_bytes(dtype);
  if (st.blocks > 0 && aligned_to(in.y_permuted, 16) && aligned_to(in.residual, 16) &&
      aligned_to(g.d_residual_out, 16) && aligned_to(g.d_normed, 16) && aligned_gammas(in, per) &&
      aligned_to(g.d_residual, unit) && aligned_to(g.d_y_permuted, unit)) {
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

// C ABI of the expert-block operators: rr_grouped_gated_gemm and its backward
// pass, the 8-bit integer operators, and rr_unpermute_norm and its backward
// pass. As in api.cpp, every argument is checked before any launch, nothing
// allocates or synchronises, and errors come back as an rr_status.
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <initializer_list>

#include "../../include/raggedroute/runtime.h"
#include "../../include/raggedroute/status.h"
#include "../../include/raggedroute_b200.h"
#include "expert_block.cuh"

namespace raggedroute {
__attribute__((visibility("hidden"))) Status detail_resolve_sm100(
    const RuntimeContext& context) noexcept;
}

namespace {

using rrb::Activation;
using rrb::Dtype;

rr_status fail(int32_t code, const char* message, cudaError_t e = cudaSuccess) {
  return {code, static_cast<int32_t>(e), message};
}
rr_status ok() { return fail(RR_SUCCESS, "success"); }
rr_status invalid(const char* message) { return fail(RR_INVALID_ARGUMENT, message); }
rr_status launched(cudaError_t e, const char* message) {
  return e == cudaSuccess ? ok() : fail(RR_CUDA_ERROR, message, e);
}

// The checks every entry point shares: a context, a known dtype, a B200.
rr_status check_call(const rr_context* ctx, int dtype) {
  if (ctx == nullptr) return invalid("rr_context must not be null");
  if (dtype != RR_DTYPE_FP32 && dtype != RR_DTYPE_BF16) {
    return fail(RR_UNSUPPORTED_DATA_TYPE, "the data type must be RR_DTYPE_FP32 or RR_DTYPE_BF16");
  }
  return ok();
}

rr_status check_device(const rr_context* ctx) {
  raggedroute::RuntimeContext r;
  r.stream = static_cast<cudaStream_t>(ctx->stream);
  r.workspace = ctx->workspace;
  r.workspace_bytes = ctx->workspace_bytes;
  r.architecture = static_cast<raggedroute::DeviceArchitecture>(ctx->architecture);
  const raggedroute::Status s = raggedroute::detail_resolve_sm100(r);
  if (s.ok()) return ok();
  return fail(static_cast<int32_t>(s.code), s.message, s.cuda_error);
}

cudaStream_t stream_of(const rr_context* ctx) { return static_cast<cudaStream_t>(ctx->stream); }

rr_status check_workspace(const rr_context* ctx, std::size_t bytes) {
  if (bytes == 0) return ok();
  if (ctx->workspace == nullptr || ctx->workspace_bytes < bytes) {
    return fail(RR_INSUFFICIENT_WORKSPACE, "the workspace is smaller than the operator needs");
  }
  if (!rrb::aligned_to(ctx->workspace, 256)) {
    return invalid("the workspace must be 256-byte aligned");
  }
  return ok();
}

// Column counts: an index and a few strides past it stay an int.
constexpr int kMaxDim = 1 << 30;

std::size_t up256(std::size_t n) { return (n + 255) / 256 * 256; }
long long up8(long long n) { return (n + 7) / 8 * 8; }
int up16(int n) { return (n + 15) / 16 * 16; }

struct Range {
  const void* p;
  std::size_t bytes;
};

bool overlap(const Range& a, const Range& b) {
  if (a.p == nullptr || b.p == nullptr || a.bytes == 0 || b.bytes == 0) return false;
  const auto a0 = reinterpret_cast<std::uintptr_t>(a.p);
  const auto b0 = reinterpret_cast<std::uintptr_t>(b.p);
  return a0 < b0 + b.bytes && b0 < a0 + a.bytes;
}

// No output (the workspace counts as one) may touch an input or another output.
bool outputs_clash(std::initializer_list<Range> outputs, std::initializer_list<Range> inputs) {
  for (auto o = outputs.begin(); o != outputs.end(); ++o) {
    for (const Range& i : inputs) {
      if (overlap(*o, i)) return true;
    }
    for (auto q = o + 1; q != outputs.end(); ++q) {
      if (overlap(*o, *q)) return true;
    }
  }
  return false;
}

// Rows of a multiple of 16 bytes are read and written 16 bytes at a time, so
// their buffer starts on such a boundary; other rows need the element's own.
bool rows_aligned(const void* p, long long cols, std::size_t size) {
  return rrb::aligned_to(p, cols * size % 16 == 0 ? 16 : size);
}

// ---- gated projection ----------------------------------------------------------

// Few rows run without the tensor cores, straight from the caller's weights.
// BF16: where hardly any two rows share an expert both forms read the weights
// once, and the plain one spreads them over all SMs (64 experts, 16 rows,
// K=2048, N=1408 37 against 49 us; 8 experts, 4 rows, K=N=1024 5 against 10);
// sharing experts, the engine's tiles reuse them (one row per expert: 154 against
// 121, 14 against 13). FP32: the engine first writes the weights of every expert as
// three bfloat16 parts and then takes a microsecond per 64 of K and round of tiles; the
// plain form does 18 TFLOP/s (half of it in single elements) and pays for each block.
// The smaller estimate, in microseconds, decides; it is within a fifth of what was
// measured (plain against engine: 64 experts, K=N=1024: 16 rows each 312 against 467; K=256,
// N=128: 20 against 21, 24 each 28 against 22; 8 experts, 4096 x 128: 64 each 62 against
// 95, 128 each 116 against 102; 8 experts, 1784 x 126: 48 each 50 against 57, 64 each 71
// against 57; 32 experts, 1024 x 128: 32 each 40 against 41).
bool gated_few(int rows, int experts, int hidden, int output, Dtype dtype) {
  if (rows <= 4) return true;
  if (dtype == Dtype::kBf16) return 2LL * rows <= experts;
  if (rows > 65535) return false;  // the y axis of its grid
  const double weights = static_cast<double>(hidden) * output;
  const double blocks = ((rows + 3) / 4) * ((output + 31LL) / 32);
  const double plain = 4e-6 * rows * weights / 18 + 0.0072 * blocks;
  const long long tiles = ((rows + 256LL * experts - 1) / (256LL * experts)) * experts *
                          ((output + 127) / 128);
  const double engine = 9 + static_cast<double>((hidden + 63) / 64) * ((tiles + 73) / 74) +
                        4.5e-6 * experts * weights;
  return 3 + (output % 4 != 0 ? 2 * plain : plain) <= engine;
}

// The backward pass takes its few-row forms where they beat the engine. BF16:
// up to half a row per expert (64 experts, K=2048, N=1408: 16 rows 186 against 212 us,
// 32 rows 266 against 267, 64 rows 397 against 381; 8 experts, K=N=1024: 4 rows 15
// against 32), and, as the engine then packs its operands, up to two for sizes that are
// no multiple of 8 (1001 x 333: 17 experts, 34 rows 33 against 44, 64 experts, 128 rows
// 121 against 123; four each 44 against 42 and 149 against 123). FP32, where it always
// packs: 8 rows per expert (64 experts, K=N=1024: 547 against 629 us, 12 each 759 against
// 640; K=256, N=128: 32 against 33). The grid of the weight gradients limits K.
bool gated_few_backward(int rows, int experts, int hidden, int output, Dtype dtype) {
  if (hidden > (1 << 20)) return false;
  if (rows <= 4) return true;
  if (dtype == Dtype::kFp32) return rows <= 8LL * experts;
  return hidden % 8 != 0 || output % 8 != 0 ? rows <= 2LL * experts : 2LL * rows <= experts;
}

// Parts of dg and du in a bfloat16 backward pass. One rounding to bfloat16 is
// what any tensor-core operand takes, and over many rows its errors average out
// against the result's own: the gradients are 0.0023 off normwise where a single
// rounding is 0.0017, and a second part everywhere would take that to 0.0017 at half
// again the time (32768 rows, 16 experts, 4096 x 1408, forward and backward: 2.05
// against 3.15 ms). With few rows per expert an element of a weight
// gradient is a sum of few products and carries the rounding whole, and the
// products are bound by the weights' bytes: there a second part (16 significand
// bits) doubles tensor work that is hidden behind them.
int gradient_parts(int rows, int experts, Dtype dtype) {
  if (dtype == Dtype::kFp32) return 3;
  return rows <= 32LL * experts ? 2 : 1;
}

// Where the operands of one call lie in the workspace; an offset of 0 bytes
// with packed == false means that the caller's buffer is used as it is.
struct GatedPlan {
  bool pack_x = false, pack_w = false, few = false;
  int terms = 1, parts = 1, ldk = 0, ldn = 0;
  std::size_t x = 0, wg = 0, wu = 0, dg = 0, du = 0, total = 0;
};

GatedPlan gated_plan(int rows, int experts, int hidden, int output, Dtype dtype, bool backward) {
  GatedPlan p;
  p.terms = dtype == Dtype::kFp32 ? 3 : 1;
  p.ldk = static_cast<int>(up8(hidden));
  p.ldn = static_cast<int>(up8(output));
  if (rows <= 0 || (!backward && gated_few(rows, experts, hidden, output, dtype))) return p;
  if (backward && gated_few_backward(rows, experts, hidden, output, dtype)) {  // dg and du in FP32
    p.few = true;
    p.du = up256(4ull * rows * output);
    p.total = 2 * p.du;
    return p;
  }
  p.pack_x = p.terms == 3 || hidden % 8 != 0;
  p.pack_w = p.terms == 3 || output % 8 != 0;
  p.parts = gradient_parts(rows, experts, dtype);
  auto take = [&p](bool used, std::size_t elements, int parts) {
    const std::size_t at = p.total;
    if (used) p.total += up256(2 * elements * parts);
    return at;
  };
  const std::size_t r = rows, w = static_cast<std::size_t>(experts) * hidden * p.ldn;
  p.x = take(p.pack_x, r * p.ldk, p.terms);
  p.wg = take(p.pack_w, w, p.terms);
  p.wu = take(p.pack_w, w, p.terms);
  p.dg = take(backward, r * p.ldn, p.parts);
  p.du = take(backward, r * p.ldn, p.parts);
  return p;
}

// Workspace bytes that serve any number of rows up to `rows`. A call's own need
// (gated_plan) falls where more rows take a form that needs less: from the engine to
// the plain form in FP32, whose estimate steps with the tiles, and from two parts of dg
// and du to one.
std::size_t gated_workspace(int rows, int experts, int hidden, int output, Dtype dtype,
                            bool backward) {
  auto need = [&](long long r) {
    return gated_plan(static_cast<int>(r), experts, hidden, output, dtype, backward).total;
  };
  std::size_t most = need(rows);
  auto also = [&](long long r) {
    if (r < rows && need(r) > most) most = need(r);
  };
  if (backward) {
    also(32LL * experts);  // the most rows with two parts
  } else if (dtype == Dtype::kFp32) {
    // Within a step the rows of the plain form come first, so the engine's largest need
    // up to `rows` is at `rows` or at a step's end.
    const long long step = 256LL * experts;
    const long long last = rows < 65535 ? rows : 65535;
    for (long long r = step; r <= last; r += step) also(r);
  }
  return most;
}

rr_status check_gated(int route_pairs, int experts, int hidden, int output, int activation) {
  if (experts <= 0 || experts > RR_MAX_EXPERTS || route_pairs < 0 || hidden <= 0 || output <= 0 ||
      hidden > kMaxDim || output > kMaxDim / 2 || route_pairs > INT_MAX - 512) {
    return invalid("grouped_gated_gemm requires 1<=E<=1024, R>=0, 1<=K<=2^30 and 1<=N<=2^29");
  }
  if (activation < RR_ACTIVATION_SILU || activation > RR_ACTIVATION_RELU) {
    return invalid("grouped_gated_gemm received an unknown activation");
  }
  return ok();
}

// Packs what the engine cannot read in place and names the operands.
cudaError_t gated_operands(const GatedPlan& plan, const void* x, const void* wg, const void* wu,
                           char* ws, int rows, int experts, int hidden, int output, Dtype dtype,
                           bool need_w, cudaStream_t stream, rrb::GatedOperands* out) {
  out->terms = plan.terms;
  out->ldk = plan.ldk;
  out->ldn = plan.ldn;
  rrb::PackJobs jobs;
  auto place = [&](bool pack, const void* src, std::size_t at, long long r, int cols, int ld) {
    if (!pack) return static_cast<const __nv_bfloat16*>(src);
    auto* to = reinterpret_cast<__nv_bfloat16*>(ws + at);
    jobs.job[jobs.count++] = {src, to, r, cols, ld};
    return static_cast<const __nv_bfloat16*>(to);
  };
  out->x = place(plan.pack_x, x, plan.x, rows, hidden, plan.ldk);
  const long long wrows = static_cast<long long>(experts) * hidden;
  if (need_w) {
    out->wg = place(plan.pack_w, wg, plan.wg, wrows, output, plan.ldn);
    out->wu = place(plan.pack_w, wu, plan.wu, wrows, output, plan.ldn);
  }
  return jobs.count > 0 ? rrb::launch_pack_terms(jobs, dtype, stream) : cudaSuccess;
}

}  // namespace

extern "C" {

size_t rr_grouped_gated_gemm_workspace_size(int route_pairs, int experts, int hidden, int output,
                                            int dtype) {
  if (check_gated(route_pairs, experts, hidden, output, RR_ACTIVATION_SILU).code != RR_SUCCESS ||
      (dtype != RR_DTYPE_FP32 && dtype != RR_DTYPE_BF16)) {
    return 0;
  }
  return gated_workspace(route_pairs, experts, hidden, output, static_cast<Dtype>(dtype), false);
}

size_t rr_grouped_gated_gemm_backward_workspace_size(int route_pairs, int experts, int hidden,
                                                     int output, int dtype) {
  if (check_gated(route_pairs, experts, hidden, output, RR_ACTIVATION_SILU).code != RR_SUCCESS ||
      (dtype != RR_DTYPE_FP32 && dtype != RR_DTYPE_BF16)) {
    return 0;
  }
  return gated_workspace(route_pairs, experts, hidden, output, static_cast<Dtype>(dtype), true);
}

rr_status rr_grouped_gated_gemm(const void* x_permuted, const void* gate_weights,
                                const void* up_weights, const int32_t* offsets, void* h,
                                float* gate_up, int route_pairs, int experts, int hidden,
                                int output, int activation, int dtype, const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  s = check_gated(route_pairs, experts, hidden, output, activation);
  if (s.code != RR_SUCCESS) return s;
  if (route_pairs == 0) return ok();
  const Dtype t = static_cast<Dtype>(dtype);
  const std::size_t size = rrb::dtype_bytes(t);
  if (x_permuted == nullptr || gate_weights == nullptr || up_weights == nullptr ||
      offsets == nullptr || h == nullptr) {
    return invalid("grouped_gated_gemm received a null buffer");
  }
  if (!rows_aligned(x_permuted, hidden, size) || !rows_aligned(gate_weights, output, size) ||
      !rows_aligned(up_weights, output, size) || !rows_aligned(h, output, size) ||
      !rows_aligned(gate_up, output, 4) || !rrb::aligned_to(offsets, 4)) {
    return invalid("grouped_gated_gemm: rows of a multiple of 16 bytes need 16-byte aligned buffers");
  }
  const std::size_t rows = route_pairs, weights = size * experts * hidden * output;
  const GatedPlan plan = gated_plan(route_pairs, experts, hidden, output, t, false);
  if (outputs_clash({{h, rows * output * size},
                     {gate_up, rows * output * 8},
                     {ctx->workspace, plan.total}},
                    {{x_permuted, rows * hidden * size},
                     {gate_weights, weights},
                     {up_weights, weights},
                     {offsets, 4ull * (experts + 1)}})) {
    return invalid("grouped_gated_gemm: an output overlaps another buffer");
  }
  s = check_workspace(ctx, plan.total);
  if (s.code != RR_SUCCESS) return s;
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  const Activation act = static_cast<Activation>(activation);
  const char* what = "grouped_gated_gemm launch failed";
  if (gated_few(route_pairs, experts, hidden, output, t)) {
    return launched(rrb::launch_gated_few(x_permuted, gate_weights, up_weights, offsets, h,
                                          gate_up, route_pairs, experts, hidden, output, act, t,
                                          stream_of(ctx)),
                    what);
  }
  rrb::GatedOperands in;
  const cudaError_t e =
      gated_operands(plan, x_permuted, gate_weights, up_weights,
                     static_cast<char*>(ctx->workspace), route_pairs, experts, hidden, output, t,
                     true, stream_of(ctx), &in);
  if (e != cudaSuccess) return launched(e, what);
  return launched(rrb::launch_gated_gemm(in, offsets, h, gate_up, route_pairs, experts, hidden,
                                         output, act, t, stream_of(ctx)),
                  what);
}

rr_status rr_grouped_gated_gemm_backward(const void* x_permuted, const void* gate_weights,
                                         const void* up_weights, const int32_t* offsets,
                                         const float* gate_up, const void* dh, void* dx,
                                         void* d_gate_weights, void* d_up_weights,
                                         int route_pairs, int experts, int hidden, int output,
                                         int activation, int dtype, const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  s = check_gated(route_pairs, experts, hidden, output, activation);
  if (s.code != RR_SUCCESS) return s;
  const Dtype t = static_cast<Dtype>(dtype);
  const std::size_t size = rrb::dtype_bytes(t);
  if ((d_gate_weights == nullptr) != (d_up_weights == nullptr) ||
      (dx == nullptr && d_gate_weights == nullptr)) {
    return invalid("grouped_gated_gemm_backward needs dx, both weight gradients, or all three");
  }
  const std::size_t weights = size * experts * hidden * output;
  const char* what = "grouped_gated_gemm_backward launch failed";
  if (route_pairs == 0) {
    if (d_gate_weights == nullptr) return ok();
    s = check_device(ctx);
    if (s.code != RR_SUCCESS) return s;
    const cudaError_t e = cudaMemsetAsync(d_gate_weights, 0, weights, stream_of(ctx));
    if (e != cudaSuccess) return launched(e, what);
    return launched(cudaMemsetAsync(d_up_weights, 0, weights, stream_of(ctx)), what);
  }
  const bool need_w = dx != nullptr, need_dw = d_gate_weights != nullptr;
  if (x_permuted == nullptr || gate_weights == nullptr || up_weights == nullptr ||
      offsets == nullptr || gate_up == nullptr || dh == nullptr) {
    return invalid("grouped_gated_gemm_backward received a null buffer");
  }
  if (!rows_aligned(x_permuted, hidden, size) || !rows_aligned(gate_weights, output, size) ||
      !rows_aligned(up_weights, output, size) || !rows_aligned(dh, output, size) ||
      !rows_aligned(gate_up, output, 4) || !rows_aligned(dx, hidden, size) ||
      !rows_aligned(d_gate_weights, output, size) || !rows_aligned(d_up_weights, output, size) ||
      !rrb::aligned_to(offsets, 4)) {
    return invalid(
        "grouped_gated_gemm_backward: rows of a multiple of 16 bytes need 16-byte aligned buffers");
  }
  const std::size_t rows = route_pairs;
  const GatedPlan plan = gated_plan(route_pairs, experts, hidden, output, t, true);
  if (outputs_clash({{dx, rows * hidden * size},
                     {d_gate_weights, weights},
                     {d_up_weights, weights},
                     {ctx->workspace, plan.total}},
                    {{x_permuted, rows * hidden * size},
                     {gate_weights, weights},
                     {up_weights, weights},
                     {gate_up, rows * output * 8},
                     {dh, rows * output * size},
                     {offsets, 4ull * (experts + 1)}})) {
    return invalid("grouped_gated_gemm_backward: an output overlaps another buffer");
  }
  s = check_workspace(ctx, plan.total);
  if (s.code != RR_SUCCESS) return s;
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  char* ws = static_cast<char*>(ctx->workspace);
  cudaStream_t stream = stream_of(ctx);
  if (plan.few) {
    auto* fg = reinterpret_cast<float*>(ws + plan.dg);
    auto* fu = reinterpret_cast<float*>(ws + plan.du);
    cudaError_t f = rrb::launch_gated_pointwise_backward_f32(
        gate_up, dh, fg, fu, route_pairs, output, static_cast<Activation>(activation), t, stream);
    if (f == cudaSuccess && need_w) {
      f = rrb::launch_gated_few_dx(fg, fu, gate_weights, up_weights, offsets, dx, route_pairs,
                                   experts, hidden, output, t, stream);
    }
    if (f == cudaSuccess && need_dw) {
      f = rrb::launch_gated_few_dw(x_permuted, fg, fu, offsets, d_gate_weights, d_up_weights,
                                   route_pairs, experts, hidden, output, t, stream);
    }
    return launched(f, what);
  }
  auto* dg = reinterpret_cast<__nv_bfloat16*>(ws + plan.dg);
  auto* du = reinterpret_cast<__nv_bfloat16*>(ws + plan.du);
  cudaError_t e = rrb::launch_gated_pointwise_backward(gate_up, dh, dg, du, route_pairs, output,
                                                       plan.ldn, plan.parts,
                                                       static_cast<Activation>(activation), t,
                                                       stream);
  rrb::GatedOperands in;
  if (e == cudaSuccess) {
    GatedPlan used = plan;
    used.pack_x = plan.pack_x && need_dw;
    e = gated_operands(used, x_permuted, gate_weights, up_weights, ws, route_pairs, experts,
                       hidden, output, t, need_w, stream, &in);
  }
  if (e == cudaSuccess && need_w) {
    e = rrb::launch_gated_dx(in, dg, du, plan.parts, offsets, dx, route_pairs, experts, hidden, output, t,
                             stream);
  }
  if (e == cudaSuccess && need_dw) {
    e = rrb::launch_gated_dw(in, dg, du, plan.parts, offsets, d_gate_weights, d_up_weights, route_pairs,
                             experts, hidden, output, t, stream);
  }
  return launched(e, what);
}

// ---- 8-bit integers --------------------------------------------------------------

int rr_int8_row_stride(int hidden) {
  return hidden <= 0 || hidden > RR_MAX_INT8_HIDDEN ? 0 : up16(hidden);
}

rr_status rr_quantize_rows_int8(const void* x, int8_t* xq, float* x_scale, int rows, int hidden,
                                int dtype, const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  if (rows < 0 || hidden <= 0 || hidden > RR_MAX_INT8_HIDDEN) {
    return invalid("quantize_rows_int8 requires rows>=0 and 1<=K<=131072");
  }
  if (rows == 0) return ok();
  const std::size_t size = dtype == RR_DTYPE_BF16 ? 2 : 4;
  if (x == nullptr || xq == nullptr || x_scale == nullptr || !rrb::aligned_to(xq, 16) ||
      !rrb::aligned_to(x, size) || !rrb::aligned_to(x_scale, 4)) {
    return invalid("quantize_rows_int8 received a null buffer or xq is not 16-byte aligned");
  }
  const int ld = up16(hidden);
  const std::size_t r = rows;
  if (outputs_clash({{xq, r * ld}, {x_scale, 4 * r}}, {{x, r * hidden * size}})) {
    return invalid("quantize_rows_int8: an output overlaps another buffer");
  }
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  return launched(rrb::launch_quantize_rows_int8(x, xq, x_scale, rows, hidden, ld,
                                                 static_cast<Dtype>(dtype), stream_of(ctx)),
                  "quantize_rows_int8 launch failed");
}

rr_status rr_quantize_expert_weights_int8(const void* expert_weights, int8_t* wq, float* w_scale,
                                          int experts, int hidden, int output, int dtype,
                                          const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  if (experts <= 0 || experts > RR_MAX_EXPERTS || hidden <= 0 || hidden > RR_MAX_INT8_HIDDEN ||
      output <= 0 || output > kMaxDim) {
    return invalid(
        "quantize_expert_weights_int8 requires 1<=E<=1024, 1<=K<=131072 and 1<=N<=2^30");
  }
  const std::size_t size = dtype == RR_DTYPE_BF16 ? 2 : 4;
  if (expert_weights == nullptr || wq == nullptr || w_scale == nullptr ||
      !rrb::aligned_to(wq, 16) || !rrb::aligned_to(expert_weights, size) ||
      !rrb::aligned_to(w_scale, 4)) {
    return invalid(
        "quantize_expert_weights_int8 received a null buffer or wq is not 16-byte aligned");
  }
  const int ld = up16(hidden);
  const std::size_t channels = static_cast<std::size_t>(experts) * output;
  if (outputs_clash({{wq, channels * ld}, {w_scale, 4 * channels}},
                    {{expert_weights, channels * hidden * size}})) {
    return invalid("quantize_expert_weights_int8: an output overlaps another buffer");
  }
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  return launched(
      rrb::launch_quantize_expert_weights_int8(expert_weights, wq, w_scale, experts, hidden,
                                               output, ld, static_cast<Dtype>(dtype),
                                               stream_of(ctx)),
      "quantize_expert_weights_int8 launch failed");
}

rr_status rr_grouped_gemm_int8(const int8_t* xq, const float* x_scale, const int8_t* wq,
                               const float* w_scale, const int32_t* offsets, void* y_permuted,
                               int route_pairs, int experts, int hidden, int output, int dtype,
                               const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  if (experts <= 0 || experts > RR_MAX_EXPERTS || route_pairs < 0 ||
      route_pairs > INT_MAX - 512 || hidden <= 0 || hidden > RR_MAX_INT8_HIDDEN || output <= 0 ||
      output > kMaxDim) {
    return invalid("grouped_gemm_int8 requires 1<=E<=1024, R>=0, 1<=K<=131072 and 1<=N<=2^30");
  }
  if (route_pairs == 0) return ok();
  const Dtype t = static_cast<Dtype>(dtype);
  const std::size_t size = rrb::dtype_bytes(t);
  if (xq == nullptr || x_scale == nullptr || wq == nullptr || w_scale == nullptr ||
      offsets == nullptr || y_permuted == nullptr) {
    return invalid("grouped_gemm_int8 received a null buffer");
  }
  if (!rrb::aligned_to(xq, 16) || !rrb::aligned_to(wq, 16) || !rrb::aligned_to(x_scale, 4) ||
      !rrb::aligned_to(w_scale, 4) || !rrb::aligned_to(offsets, 4) ||
      !rows_aligned(y_permuted, output, size)) {
    return invalid("grouped_gemm_int8: xq, wq and rows of a multiple of 16 bytes need 16-byte "
                   "aligned buffers");
  }
  const int ld = up16(hidden);
  const std::size_t rows = route_pairs, channels = static_cast<std::size_t>(experts) * output;
  if (outputs_clash({{y_permuted, rows * output * size}}, {{xq, rows * ld},
                                                           {x_scale, 4 * rows},
                                                           {wq, channels * ld},
                                                           {w_scale, 4 * channels},
                                                           {offsets, 4ull * (experts + 1)}})) {
    return invalid("grouped_gemm_int8: the output overlaps another buffer");
  }
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  // Few rows: the weights are read once either way, and the plain kernel
  // spreads a single row over the whole GPU and starts faster (128 experts,
  // K=4096, N=1408: 2 rows 3.2 against 13 us, 128 rows 88 against 95, 256 rows
  // 138 against 130; 8 experts, K=N=1024: 32 rows 6.2 against 7.6, 64 rows 9.6
  // against 7.6).
  const bool few = route_pairs <= 32 || route_pairs <= experts;
  const cudaError_t e =
      few ? rrb::launch_int8_few(xq, x_scale, wq, w_scale, offsets, y_permuted, route_pairs,
                                 experts, ld, output, t, stream_of(ctx))
          : rrb::launch_int8_gemm(xq, x_scale, wq, w_scale, offsets, y_permuted, route_pairs,
                                  experts, ld, output, t, stream_of(ctx));
  return launched(e, "grouped_gemm_int8 launch failed");
}

// ---- combine, norms, gate, residual ------------------------------------------------

namespace {

rr_status check_norm(int tokens, int top_k, int output) {
  if (tokens < 0 || top_k < 1 || top_k > RR_MAX_NORM_TOP_K || output < 1 ||
      output > RR_MAX_NORM_OUTPUT || static_cast<long long>(tokens) * top_k > INT_MAX) {
    return invalid("unpermute_norm requires T>=0, 1<=top_k<=64 and 1<=N<=16384");
  }
  return ok();
}

bool floats_aligned(std::initializer_list<const void*> ps) {
  for (const void* p : ps) {
    if (!rrb::aligned_to(p, 4)) return false;
  }
  return true;
}

}  // namespace

rr_status rr_unpermute_norm(const void* y_permuted, const int32_t* route_pos,
                            const float* route_weights, const void* residual,
                            const float* post_gamma, const float* gate, const float* pre_gamma,
                            void* residual_out, void* normed, float* inv_rms, float eps,
                            float residual_scale, int tokens, int top_k, int output, int dtype,
                            const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  s = check_norm(tokens, top_k, output);
  if (s.code != RR_SUCCESS) return s;
  if (!(eps >= 0.0f)) return invalid("unpermute_norm requires eps >= 0");
  if ((pre_gamma == nullptr) != (normed == nullptr)) {
    return invalid("unpermute_norm: normed goes with pre_gamma");
  }
  if (tokens == 0) return ok();
  const Dtype t = static_cast<Dtype>(dtype);
  const std::size_t size = rrb::dtype_bytes(t);
  if (y_permuted == nullptr || route_pos == nullptr || route_weights == nullptr ||
      residual == nullptr || residual_out == nullptr) {
    return invalid("unpermute_norm received a null buffer");
  }
  if (!floats_aligned({route_pos, route_weights, post_gamma, gate, pre_gamma, inv_rms}) ||
      !rrb::aligned_to(y_permuted, size) || !rrb::aligned_to(residual, size) ||
      !rrb::aligned_to(residual_out, size) || !rrb::aligned_to(normed, size)) {
    return invalid("unpermute_norm received a misaligned buffer");
  }
  const std::size_t rows = tokens, routes = rows * top_k, cols = output;
  const Range out{residual_out, rows * cols * size}, res{residual, rows * cols * size};
  if (outputs_clash({out, {normed, rows * cols * size}, {inv_rms, 8 * rows}},
                    {{y_permuted, routes * cols * size},
                     {route_pos, 4 * routes},
                     {route_weights, 4 * routes},
                     {post_gamma, 4 * cols},
                     {gate, 4 * cols},
                     {pre_gamma, 4 * cols}}) ||
      (residual_out != residual && overlap(out, res)) ||
      outputs_clash({{normed, rows * cols * size}, {inv_rms, 8 * rows}}, {res})) {
    return invalid("unpermute_norm: an output overlaps another buffer");
  }
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  rrb::UnpermuteNorm in;
  in.y_permuted = y_permuted;
  in.route_pos = route_pos;
  in.route_weights = route_weights;
  in.residual = residual;
  in.post_gamma = post_gamma;
  in.gate = gate;
  in.pre_gamma = pre_gamma;
  in.eps = eps;
  in.residual_scale = residual_scale;
  in.tokens = tokens;
  in.top_k = top_k;
  in.output = output;
  return launched(rrb::launch_unpermute_norm(in, residual_out, normed, inv_rms, t, stream_of(ctx)),
                  "unpermute_norm launch failed");
}

size_t rr_unpermute_norm_backward_workspace_size(int tokens, int output) {
  if (check_norm(tokens, 1, output).code != RR_SUCCESS || tokens == 0) return 0;
  return rrb::unpermute_norm_backward_workspace_bytes(tokens, output);
}

rr_status rr_unpermute_norm_backward(
    const void* y_permuted, const int32_t* route_pos, const float* route_weights,
    const void* residual, const float* post_gamma, const float* gate, const float* pre_gamma,
    const float* inv_rms, const void* d_residual_out, const void* d_normed, void* d_residual,
    void* d_y_permuted, float* d_route_weights, float* d_post_gamma, float* d_gate,
    float* d_pre_gamma, float residual_scale, int tokens, int top_k, int output, int dtype,
    const rr_context* ctx) {
  rr_status s = check_call(ctx, dtype);
  if (s.code != RR_SUCCESS) return s;
  s = check_norm(tokens, top_k, output);
  if (s.code != RR_SUCCESS) return s;
  if ((d_post_gamma != nullptr && post_gamma == nullptr) ||
      (d_gate != nullptr && gate == nullptr) ||
      (d_pre_gamma != nullptr && pre_gamma == nullptr)) {
    return invalid("unpermute_norm_backward: a parameter gradient needs its parameter");
  }
  if (d_normed != nullptr && pre_gamma == nullptr) {
    return invalid("unpermute_norm_backward: d_normed goes with pre_gamma");
  }
  const std::size_t rows = tokens, routes = rows * top_k, cols = output;
  const char* what = "unpermute_norm_backward launch failed";
  if (tokens == 0) {
    s = check_device(ctx);
    if (s.code != RR_SUCCESS) return s;
    for (float* g : {d_post_gamma, d_gate, d_pre_gamma}) {
      if (g == nullptr) continue;
      const cudaError_t e = cudaMemsetAsync(g, 0, 4 * cols, stream_of(ctx));
      if (e != cudaSuccess) return launched(e, what);
    }
    return ok();
  }
  const Dtype t = static_cast<Dtype>(dtype);
  const std::size_t size = rrb::dtype_bytes(t);
  const bool norms = post_gamma != nullptr || d_normed != nullptr;
  if (y_permuted == nullptr || route_pos == nullptr || route_weights == nullptr ||
      residual == nullptr || (norms && inv_rms == nullptr) || d_residual == nullptr ||
      d_y_permuted == nullptr || d_route_weights == nullptr) {
    return invalid("unpermute_norm_backward received a null buffer");
  }
  if (!floats_aligned({route_pos, route_weights, post_gamma, gate, pre_gamma, inv_rms,
                       d_route_weights, d_post_gamma, d_gate, d_pre_gamma}) ||
      !rrb::aligned_to(y_permuted, size) || !rrb::aligned_to(residual, size) ||
      !rrb::aligned_to(d_residual_out, size) || !rrb::aligned_to(d_normed, size) ||
      !rrb::aligned_to(d_residual, size) || !rrb::aligned_to(d_y_permuted, size)) {
    return invalid("unpermute_norm_backward received a misaligned buffer");
  }
  const std::size_t grid = rows * cols * size, wide = routes * cols * size;
  const Range work{ctx->workspace, rrb::unpermute_norm_backward_workspace_bytes(tokens, output)};
  const Range dro{d_residual_out, grid}, dres{d_residual, grid};
  if (outputs_clash({dres,
                     work,
                     {d_y_permuted, wide},
                     {d_route_weights, 4 * routes},
                     {d_post_gamma, 4 * cols},
                     {d_gate, 4 * cols},
                     {d_pre_gamma, 4 * cols}},
                    {{y_permuted, wide},
                     {route_pos, 4 * routes},
                     {route_weights, 4 * routes},
                     {residual, grid},
                     {post_gamma, 4 * cols},
                     {gate, 4 * cols},
                     {pre_gamma, 4 * cols},
                     {inv_rms, 8 * rows},
                     {d_normed, grid}}) ||
      (d_residual != d_residual_out && overlap(dres, dro)) ||
      outputs_clash({work,
                     {d_y_permuted, wide},
                     {d_route_weights, 4 * routes},
                     {d_post_gamma, 4 * cols},
                     {d_gate, 4 * cols},
                     {d_pre_gamma, 4 * cols}},
                    {dro})) {
    return invalid("unpermute_norm_backward: an output overlaps another buffer");
  }
  s = check_workspace(ctx, work.bytes);
  if (s.code != RR_SUCCESS) return s;
  s = check_device(ctx);
  if (s.code != RR_SUCCESS) return s;
  rrb::UnpermuteNorm in;
  in.y_permuted = y_permuted;
  in.route_pos = route_pos;
  in.route_weights = route_weights;
  in.residual = residual;
  in.post_gamma = post_gamma;
  in.gate = gate;
  // Without a gradient into normed its norm takes no part.
  in.pre_gamma = d_normed != nullptr ? pre_gamma : nullptr;
  in.residual_scale = residual_scale;
  in.tokens = tokens;
  in.top_k = top_k;
  in.output = output;
  rrb::UnpermuteNormGrads g;
  g.inv_rms = inv_rms;
  g.d_residual_out = d_residual_out;
  g.d_normed = d_normed;
  g.d_residual = d_residual;
  g.d_y_permuted = d_y_permuted;
  g.d_route_weights = d_route_weights;
  g.d_post_gamma = d_post_gamma;
  g.d_gate = d_gate;
  g.d_pre_gamma = d_pre_gamma;
  return launched(rrb::launch_unpermute_norm_backward(
                      in, g, static_cast<float*>(ctx->workspace), t, stream_of(ctx)),
                  what);
}

}  // extern "C"

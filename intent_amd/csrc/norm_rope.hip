// Norm and rotation of query and key heads (forward and backward), for gfx950. No reference counterpart.
//
// A row is one (token, head): y = x * rsqrt(mean(x^2) + eps) * w in f32, whose first 2R dimensions are R pairs turned by
// the token's angles. Backward: g = the gradient turned back; u = x r; grad_x = r (g w - u mean(g w u)); grad_w = the sum
// of g u over rows, through f32 partial sums per workgroup that a second kernel adds in order.
#include "common.hpp"

namespace intent_hip {
namespace {

constexpr int kMaxWidth = 1024;       // head width: a wave holds a row in 16 registers a lane
constexpr int kRowRegisters = kMaxWidth / kWave;
constexpr int kWaves = 4;

struct NormRope {
  const uint16_t *x[2], *dy[2];       // queries, keys
  uint16_t *out[2];
  const float *w[2];
  const int32_t *positions;
  const float *cos, *sin;
  int64_t xs[2][2], dys[2][2], outs[2][2];   // token and head strides
  int64_t coss, sins, table;
  int64_t tokens;
  int heads[2];
  int d, pairs, interleaved;
  float eps;
};

__device__ __forceinline__ int64_t table_row(const NormRope &p, int64_t token) {
  const int64_t at = p.positions[token];
  return at < 0 ? 0 : (at >= p.table ? p.table - 1 : at);
}

// The other dimension of d's pair (d itself where none is turned), the pair, and the sign of the partner's sine.
struct Partner {
  int other, pair;
  float sign;
};
__device__ __forceinline__ Partner partner(const NormRope &p, int d) {
  if (d >= 2 * p.pairs) return {d, 0, 0.0f};
  if (p.interleaved) return {d ^ 1, d >> 1, d & 1 ? 1.0f : -1.0f};
  return d < p.pairs ? Partner{d + p.pairs, d, -1.0f} : Partner{d - p.pairs, d - p.pairs, 1.0f};
}

// ---------------------------------------------------------------- any width, any layout of rows
// One wave per row, a lane every 64th dimension; the partner's value is read again (it is in the L1).
template <typename E>
__global__ __launch_bounds__(kWaves * kWave) void norm_rope_any(NormRope p) {
  const int lane = threadIdx.x & 63;
  const int heads = p.heads[0] + p.heads[1];
  const int64_t row = static_cast<int64_t>(grid_block()) * kWaves + (threadIdx.x >> 6);
  if (row >= p.tokens * heads) return;
  const int64_t token = row / heads;
  int head = static_cast<int>(row % heads);
  const int which = head >= p.heads[0];
  if (which) head -= p.heads[0];
  const E *x = reinterpret_cast<const E *>(p.x[which]) + token * p.xs[which][0] + head * p.xs[which][1];
  E *out = reinterpret_cast<E *>(p.out[which]) + token * p.outs[which][0] + head * p.outs[which][1];
  const float *w = p.w[which];
  const int64_t at = p.pairs ? table_row(p, token) : 0;
  float v[kRowRegisters], sum = 0.0f;
#pragma unroll
  for (int j = 0; j < kRowRegisters; ++j) {
    const int d = j * kWave + lane;
    v[j] = d < p.d ? to_f32(x[d]) : 0.0f;
    sum += v[j] * v[j];
  }
  const float r = rsqrtf(wave_sum(sum) / p.d + p.eps);
#pragma unroll
  for (int j = 0; j < kRowRegisters; ++j) {
    const int d = j * kWave + lane;
    if (d >= p.d) continue;
    float y = v[j] * r * w[d];
    const Partner q = partner(p, d);
    if (q.other != d) {
      const float other = to_f32(x[q.other]) * r * w[q.other];
      y = y * p.cos[at * p.coss + q.pair] + q.sign * other * p.sin[at * p.sins + q.pair];
    }
    out[d] = from_f32<E>(y);
  }
}

// The backward of the same: waves walk rows of the queries (blocks below `split`) or of the keys, and keep their share
// of the weight's gradient in registers until the end.
template <typename E>
__global__ __launch_bounds__(kWaves * kWave) void norm_rope_backward_any(NormRope p, int split, float *partial) {
  __shared__ float sums[kWaves][kMaxWidth];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int which = static_cast<int>(blockIdx.x) >= split;
  const int block = which ? blockIdx.x - split : blockIdx.x, blocks = which ? gridDim.x - split : split;
  const int heads = p.heads[which];
  const int64_t rows = p.tokens * heads;
  const float *w = p.w[which];
  float dw[kRowRegisters];
#pragma unroll
  for (int j = 0; j < kRowRegisters; ++j) dw[j] = 0.0f;
  for (int64_t row = static_cast<int64_t>(block) * kWaves + wave; row < rows; row += static_cast<int64_t>(blocks) * kWaves) {
    const int64_t token = row / heads;
    const int head = static_cast<int>(row % heads);
    const E *x = reinterpret_cast<const E *>(p.x[which]) + token * p.xs[which][0] + head * p.xs[which][1];
    const E *dy = reinterpret_cast<const E *>(p.dy[which]) + token * p.dys[which][0] + head * p.dys[which][1];
    E *out = reinterpret_cast<E *>(p.out[which]) + token * p.outs[which][0] + head * p.outs[which][1];
    const int64_t at = p.pairs ? table_row(p, token) : 0;
    float v[kRowRegisters], g[kRowRegisters], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kRowRegisters; ++j) {
      const int d = j * kWave + lane;
      v[j] = d < p.d ? to_f32(x[d]) : 0.0f;
      sum += v[j] * v[j];
    }
    const float r = rsqrtf(wave_sum(sum) / p.d + p.eps);
    float along = 0.0f;
#pragma unroll
    for (int j = 0; j < kRowRegisters; ++j) {
      const int d = j * kWave + lane;
      g[j] = 0.0f;
      if (d < p.d) {
        g[j] = to_f32(dy[d]);
        const Partner q = partner(p, d);
        if (q.other != d)
          g[j] = g[j] * p.cos[at * p.coss + q.pair] - q.sign * to_f32(dy[q.other]) * p.sin[at * p.sins + q.pair];
        v[j] *= r;
        dw[j] += g[j] * v[j];
        g[j] *= w[d];
        along += g[j] * v[j];
      }
    }
    along = wave_sum(along) / p.d;
#pragma unroll
    for (int j = 0; j < kRowRegisters; ++j) {
      const int d = j * kWave + lane;
      if (d < p.d) out[d] = from_f32<E>(r * (g[j] - v[j] * along));
    }
  }
#pragma unroll
  for (int j = 0; j < kRowRegisters; ++j) {
    const int d = j * kWave + lane;
    if (d < p.d) sums[wave][d] = dw[j];
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.d; d += kWaves * kWave) {
    float total = 0.0f;
    for (int i = 0; i < kWaves; ++i) total += sums[i][d];
    partial[static_cast<int64_t>(blockIdx.x) * p.d + d] = total;
  }
}

// grad_w[which][d]: the workgroups' partial sums, in a fixed order. One workgroup per 16 dimensions of the queries' or the
// keys' weight; 16 threads share a dimension.
__global__ __launch_bounds__(256) void norm_rope_fold(const float *partial, int split, int blocks, int d, float *dq, float *dk) {
  __shared__ float sums[16][17];
  const int column = threadIdx.x & 15, part = threadIdx.x >> 4, at = blockIdx.x * 16 + column;
  const int which = blockIdx.y, first = which ? split : 0, last = which ? blocks : split;
  float total = 0.0f;
  if (at < d)
    for (int i = first + part; i < last; i += 16) total += partial[static_cast<int64_t>(i) * d + at];
  sums[part][column] = total;
  __syncthreads();
  if (part == 0 && at < d) {
    for (int i = 1; i < 16; ++i) total += sums[i][column];
    (which ? dk : dq)[at] = total;
  }
}

// Workgroups of the backward pass and how many of them walk the queries' rows.
struct Blocks {
  int split, total;
};
Blocks backward_blocks(int64_t tokens, int64_t q_heads, int64_t kv_heads) {
  const int64_t most = 1024, rows = tokens * (q_heads + kv_heads);
  const auto share = [&](int64_t heads) -> int {
    if (tokens * heads == 0) return 0;
    const int64_t wanted = (tokens * heads + kWaves - 1) / kWaves, fair = (most * tokens * heads + rows - 1) / rows;
    return static_cast<int>(wanted < fair ? wanted : fair);
  };
  const int split = share(q_heads);
  return {split, split + share(kv_heads)};
}

int check(int dtype, const NormRope &p, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t d, int64_t table,
          int64_t pairs, const int64_t *strides, int views) {
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || d < 0 || table < 0 || pairs < 0)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "qk_norm_rope dtype must be F16 or BF16, got %d", dtype);
  if (2 * pairs > d)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "%lld rotated pairs do not fit a head of width %lld",
                static_cast<long long>(pairs), static_cast<long long>(d));
  if (d > kMaxWidth)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "qk_norm_rope takes heads of up to %d dimensions, got %lld", kMaxWidth,
                static_cast<long long>(d));
  if (q_heads > INT32_MAX / 2 || kv_heads > INT32_MAX / 2) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  if (q_heads + kv_heads > 0 && tokens > (int64_t{1} << 40) / (q_heads + kv_heads))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  if (tokens == 0 || d == 0 || q_heads + kv_heads == 0) return INTENT_HIP_OK;
  if (strides == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  for (int i = 0; i < views; ++i)
    if (strides[i] < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (pairs > 0) {
    if (p.positions == nullptr || p.cos == nullptr || p.sin == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
    if (table < 1) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "the rotation tables hold no position");
  }
  const int64_t heads[2] = {q_heads, kv_heads};
  for (int i = 0; i < 2; ++i)
    if (heads[i] > 0 && (p.x[i] == nullptr || p.out[i] == nullptr || p.w[i] == nullptr))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  return INTENT_HIP_OK;
}

// Rows one wave each. Widths, strides and alignments are free.
int launch_forward(int dtype, const NormRope &p, hipStream_t s) {
  const int64_t rows = p.tokens * (p.heads[0] + p.heads[1]), blocks = (rows + kWaves - 1) / kWaves;
  if (blocks > INT32_MAX) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  const dim3 grid = tile_grid(blocks, 1);
  if (dtype == INTENT_HIP_F16)
    norm_rope_any<f16_t><<<grid, kWaves * kWave, 0, s>>>(p);
  else
    norm_rope_any<bf16_t><<<grid, kWaves * kWave, 0, s>>>(p);
  return hipPeekAtLastError() != hipSuccess ? launch_status("norm_rope") : INTENT_HIP_OK;
}

}  // namespace

int norm_rope_resources(int dtype, int backward, IntentHipKernelResources *out) {
  const bool half = dtype == INTENT_HIP_F16;
  if (backward)
    return half ? describe_kernel(reinterpret_cast<const void *>(norm_rope_backward_any<f16_t>), "norm_rope_backward_any<f16>", kWaves * kWave, out)
                : describe_kernel(reinterpret_cast<const void *>(norm_rope_backward_any<bf16_t>), "norm_rope_backward_any<bf16>", kWaves * kWave, out);
  return half ? describe_kernel(reinterpret_cast<const void *>(norm_rope_any<f16_t>), "norm_rope_any<f16>", kWaves * kWave, out)
              : describe_kernel(reinterpret_cast<const void *>(norm_rope_any<bf16_t>), "norm_rope_any<bf16>", kWaves * kWave, out);
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_qk_norm_rope(int dtype, const void *q, const void *k, const float *q_weight, const float *k_weight,
                                       const int32_t *positions, const float *cos, const float *sin, void *q_out, void *k_out,
                                       int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t d, int64_t table,
                                       int64_t pairs, const int64_t *strides, float eps, int interleaved, void *stream) {
  NormRope p{};
  p.x[0] = static_cast<const uint16_t *>(q), p.x[1] = static_cast<const uint16_t *>(k);
  p.out[0] = static_cast<uint16_t *>(q_out), p.out[1] = static_cast<uint16_t *>(k_out);
  p.w[0] = q_weight, p.w[1] = k_weight;
  p.positions = positions, p.cos = cos, p.sin = sin;
  if (int rc = check(dtype, p, tokens, q_heads, kv_heads, d, table, pairs, strides, 16)) return rc;
  if (tokens == 0 || d == 0 || q_heads + kv_heads == 0) return INTENT_HIP_OK;
  for (int i = 0; i < 2; ++i) {
    p.xs[i][0] = strides[3 * i], p.xs[i][1] = strides[3 * i + 1];
    p.outs[i][0] = strides[10 + 3 * i], p.outs[i][1] = strides[11 + 3 * i];
    if (d > 1 && (strides[3 * i + 2] != 1 || strides[12 + 3 * i] != 1))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows need unit inner stride");
  }
  if (pairs > 1 && (strides[7] != 1 || strides[9] != 1)) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "tables need unit inner stride");
  p.coss = strides[6], p.sins = strides[8], p.table = table;
  p.tokens = tokens, p.heads[0] = static_cast<int>(q_heads), p.heads[1] = static_cast<int>(kv_heads);
  p.d = static_cast<int>(d), p.pairs = static_cast<int>(pairs), p.interleaved = interleaved != 0, p.eps = eps;
  return launch_forward(dtype, p, as_stream(stream));
}

extern "C" int intent_hip_qk_norm_rope_backward_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t d,
                                                                size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || d < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (q_heads > INT32_MAX / 2 || kv_heads > INT32_MAX / 2 || d > kMaxWidth ||
      (q_heads + kv_heads > 0 && tokens > (int64_t{1} << 40) / (q_heads + kv_heads)))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  *bytes = static_cast<size_t>(backward_blocks(tokens, q_heads, kv_heads).total) * d * sizeof(float);
  return INTENT_HIP_OK;
}

extern "C" int intent_hip_qk_norm_rope_backward(int dtype, const void *q, const void *k, const float *q_weight,
                                                const float *k_weight, const int32_t *positions, const float *cos,
                                                const float *sin, const void *grad_q_out, const void *grad_k_out, void *grad_q,
                                                void *grad_k, float *grad_q_weight, float *grad_k_weight, int64_t tokens,
                                                int64_t q_heads, int64_t kv_heads, int64_t d, int64_t table, int64_t pairs,
                                                const int64_t *strides, float eps, int interleaved, void *workspace,
                                                size_t workspace_bytes, void *stream) {
  NormRope p{};
  p.x[0] = static_cast<const uint16_t *>(q), p.x[1] = static_cast<const uint16_t *>(k);
  p.dy[0] = static_cast<const uint16_t *>(grad_q_out), p.dy[1] = static_cast<const uint16_t *>(grad_k_out);
  p.out[0] = static_cast<uint16_t *>(grad_q), p.out[1] = static_cast<uint16_t *>(grad_k);
  p.w[0] = q_weight, p.w[1] = k_weight;
  p.positions = positions, p.cos = cos, p.sin = sin;
  if (int rc = check(dtype, p, tokens, q_heads, kv_heads, d, table, pairs, strides, 22)) return rc;
  if (d == 0) return INTENT_HIP_OK;
  if (grad_q_weight == nullptr || grad_k_weight == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  const Blocks blocks = backward_blocks(tokens, q_heads, kv_heads);
  float *partial = static_cast<float *>(workspace);
  if (blocks.total > 0) {
    if ((q_heads > 0 && grad_q_out == nullptr) || (kv_heads > 0 && grad_k_out == nullptr))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
    if (workspace == nullptr || workspace_bytes < static_cast<size_t>(blocks.total) * d * sizeof(float) || !aligned(workspace, 16))
      return fail(INTENT_HIP_ERR_WORKSPACE, "qk_norm_rope_backward needs %lld workspace bytes",
                  static_cast<long long>(blocks.total) * d * 4);
    for (int i = 0; i < 2; ++i) {
      p.xs[i][0] = strides[3 * i], p.xs[i][1] = strides[3 * i + 1];
      p.dys[i][0] = strides[10 + 3 * i], p.dys[i][1] = strides[11 + 3 * i];
      p.outs[i][0] = strides[16 + 3 * i], p.outs[i][1] = strides[17 + 3 * i];
      if (d > 1 && (strides[3 * i + 2] != 1 || strides[12 + 3 * i] != 1 || strides[18 + 3 * i] != 1))
        return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows need unit inner stride");
    }
    if (pairs > 1 && (strides[7] != 1 || strides[9] != 1))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "tables need unit inner stride");
    p.coss = strides[6], p.sins = strides[8], p.table = table;
    p.tokens = tokens, p.heads[0] = static_cast<int>(q_heads), p.heads[1] = static_cast<int>(kv_heads);
    p.d = static_cast<int>(d), p.pairs = static_cast<int>(pairs), p.interleaved = interleaved != 0, p.eps = eps;
    const dim3 grid(static_cast<unsigned>(blocks.total));
    if (dtype == INTENT_HIP_F16)
      norm_rope_backward_any<f16_t><<<grid, kWaves * kWave, 0, as_stream(stream)>>>(p, blocks.split, partial);
    else
      norm_rope_backward_any<bf16_t><<<grid, kWaves * kWave, 0, as_stream(stream)>>>(p, blocks.split, partial);
    if (hipPeekAtLastError() != hipSuccess) return launch_status("norm_rope_backward");
  }
  norm_rope_fold<<<dim3(static_cast<unsigned>((d + 15) / 16), 2), 256, 0, as_stream(stream)>>>(
      partial, blocks.split, blocks.total, static_cast<int>(d), grad_q_weight, grad_k_weight);
  return hipPeekAtLastError() != hipSuccess ? launch_status("norm_rope_fold") : INTENT_HIP_OK;
}

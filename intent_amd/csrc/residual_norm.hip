// The residual stream after a block's output has joined it, and its norm (forward, forward with 8-bit rows, backward), for gfx950.
// No reference counterpart.
//
// For a token's rows x (the block's output) and s (the stream before it), in f32:
//   u = x * rsqrt(mean(x^2) + eps) * wp   (x itself where the block has no norm of its own)
//   h = residual_scale * s + block_scale * gate * u,  y = h * rsqrt(mean(h^2) + eps) * w
// stored once rounded each; y is formed from h before its rounding. Its 8-bit form stores round(127 y / max|y|) and max|y| / 127; the
// factor rsqrt(..) cancels out of the first, so the largest |h w| comes with the sum of h^2.
// Backward, from x and the stored h, with r_x, r_h the reciprocal roots:
//   dh = grad_h + r_h (gy w - h r_h mean(gy w h r_h)),   grad_s = residual_scale dh,   grad_w = sum over tokens of gy h r_h
//   S = sum of dh u,  grad_gate = block_scale S,  du = block_scale gate dh
//   grad_x = r_x (du wp - x r_x mean(du wp x r_x)) (du without a norm),  grad_wp = sum over tokens of du x r_x
// where the mean of du wp x r_x is block_scale gate S / D.
//
// Bound by the rows' bytes, so each is read and written once: a row stays in the registers of its threads, one or two pieces of 16
// bytes each, 16384 elements in all. Measured, bf16 with both norms and a gate, forward, 8-bit and backward: 16384 x 4096 100.5, 90, 184 us
// (5.3, 5.2, 4.4 TB/s), 16384 x 1024 27, 29, 53, 8192 x 8192 103, 92, 184, 4096 x 16384 103, 96, 305 (the backward's rows no longer fit the
// registers of 16 waves, and 140 bytes a lane go by memory), 8192 x 8191 133, 122, 263, whose rows begin anywhere (two bytes at a time: 334,
// 324, 1003).
#include <stdio.h>

#include <algorithm>

#include "rows.hpp"

namespace intent_hip {
namespace {

constexpr int kWaveRows = 4;           // rows of a workgroup where a wave holds a row
constexpr int kFoldParts = 64;
constexpr int kBackwardWaves = 8;      // of a workgroup of the backward, but for rows that take more

struct Norm {
  const uint16_t *block, *residual;    // backward: residual is the stored sum
  const float *gate, *post, *weight;
  uint16_t *sum, *out;                 // backward: grad_residual, grad_block
  int8_t *q;
  float *scales;
  const uint16_t *grad_sum, *grad_out;
  float *grad_gate, *partial;          // partial: [slot][weight, post][d]
  int64_t bs, rs, ss, os, gss, gos, gs, ggs;     // strides of a token
  int64_t tokens;
  int d, waves, slots;
  float residual_scale, block_scale, eps, inverse_d;
};

__device__ __forceinline__ float gate_of(const Norm &p, int64_t token) {
  return p.gate == nullptr ? p.block_scale : p.block_scale * p.gate[token * p.gs];
}

template <typename E, int P, int W, bool kPieces, bool kPost, bool kI8>
__global__ __launch_bounds__(W *kWave) void residual_norm_rows(Norm p) {
  __shared__ RowSlots<1> first;
  __shared__ RowSlots<2> second;
  const int wave_rows = p.waves == 1 ? kWaveRows : 1;
  const int64_t token = static_cast<int64_t>(grid_block()) * wave_rows + (p.waves == 1 ? threadIdx.x >> 6 : 0);
  if (token >= p.tokens) return;       // of a whole wave; of a row of several waves the whole workgroup
  const RowPlace<kPieces> at{p.d, p.waves * kWave, static_cast<int>(p.waves == 1 ? threadIdx.x & 63 : threadIdx.x)};
  uint4 block[P], residual[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    block[j] = load_piece(p.block + token * p.bs, at, j);
    residual[j] = load_piece(p.residual + token * p.rs, at, j);
  }
  const float factor = gate_of(p, token);
  float w[P][kPiece], h[P][kPiece];
#pragma unroll
  for (int j = 0; j < P; ++j) load_weights(p.weight, at, j, w[j]);
#pragma unroll
  for (int j = 0; j < P; ++j) block[j] = settled(block[j], at, j), residual[j] = settled(residual[j], at, j);
  float r = 1.0f;
  if constexpr (kPost) {
    float sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float x[kPiece];
      widen_piece<E>(block[j], x);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) sum[0] += x[i] * x[i];
    }
    row_reduce(sum, p.waves, first);
    r = rsqrtf(sum[0] * p.inverse_d + p.eps);
  }
  float sum[1] = {0.0f};
  uint32_t most[1] = {0};
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float x[kPiece], s[kPiece], wp[kPiece];
    widen_piece<E>(block[j], x);
    widen_piece<E>(residual[j], s);
    if constexpr (kPost) load_weights(p.post, at, j, wp);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const float u = kPost ? x[i] * r * wp[i] : x[i];
      h[j][i] = fmaf(p.residual_scale, s[i], factor * u);
      sum[0] += h[j][i] * h[j][i];
      if constexpr (kI8) most[0] = max(most[0], at.holds(j, i) ? magnitude(h[j][i] * w[j][i]) : 0u);
    }
    store_piece(p.sum + token * p.ss, at, j, narrow_piece<E>(h[j]));
  }
  if constexpr (kI8) {
    row_reduce(sum, most, p.waves, second);
    const float unit = rsqrtf(sum[0] * p.inverse_d + p.eps);
    // max|y| says what the row is; where the root is 0 or infinite it is not what max|h w| would say. Elements of 0 go without a quotient.
    const uint32_t top = magnitude(__uint_as_float(most[0]) * unit);
    const RowQuant quant(top > 0 && top < kInfinity ? most[0] : kInfinity);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float v[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) v[i] = h[j][i] * w[j][i];
      store_piece(p.q + token * p.os, at, j, quant.piece(v));
    }
    if (at.thread == 0) p.scales[token] = row_scale(top);
  } else {
    RowSlots<1> &slots = *reinterpret_cast<RowSlots<1> *>(&second);
    row_reduce(sum, p.waves, slots);
    const float unit = rsqrtf(sum[0] * p.inverse_d + p.eps);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float y[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) y[i] = h[j][i] * unit * w[j][i];
      store_piece(p.out + token * p.os, at, j, narrow_piece<E>(y));
    }
  }
}

// A workgroup takes `rows` tokens at a time, and keeps its share of the weights' gradients in registers until its end. The rows of the
// next tokens are on their way while these ones' sums are formed, where registers allow.
template <typename E, int P, int W, bool kPieces, bool kPost>
__global__ __launch_bounds__(W *kWave) void residual_norm_backward_rows(Norm p) {
  __shared__ RowSlots<3> first[2];
  __shared__ RowSlots<1> second[2];
  constexpr int kWeights = kPost ? 2 : 1;
  constexpr bool kShared = W == kBackwardWaves;      // by several rows
  __shared__ float4 shares[kShared ? kWeights * P * W * kWave * kPiece / 4 : 1];     // [row][weight, post][d]
  const int row = kShared ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / p.waves : 0, row_wave = row * p.waves;
  const int rows = kShared ? static_cast<int>(blockDim.x) / (p.waves * kWave) : 1, thread = static_cast<int>(threadIdx.x) - row_wave * kWave;
  struct Rows {
    uint4 x, h, gh, gy;
  };
  // Behind the last token: rows without elements.
  const auto place = [&](int64_t token) { return RowPlace<kPieces>{!kShared || token < p.tokens ? p.d : 0, p.waves * kWave, thread}; };
  const auto load = [&](int64_t token, Rows (&to)[P]) {
    const auto at = place(token);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      to[j].h = load_piece(p.residual + token * p.rs, at, j);
      to[j].gy = load_piece(p.grad_out + token * p.gos, at, j);
      to[j].x = load_piece(p.block + token * p.bs, at, j);
      to[j].gh = load_piece(p.grad_sum + token * p.gss, at, j);
    }
  };
  float dw[P][kPiece] = {}, dwp[P][kPiece] = {};
  constexpr bool kAhead = P == 1;
  Rows next[P];
  int64_t at_once = static_cast<int64_t>(blockIdx.x) * rows;
  if constexpr (kAhead) load(at_once + row, next);
  int turn = 0;
  for (; at_once < p.tokens; at_once += static_cast<int64_t>(p.slots) * rows, turn ^= 1) {
    const int64_t token = at_once + row;
    const auto at = place(token);
    const bool live = !kShared || token < p.tokens;
    Rows now[P];
    if constexpr (kAhead) {
#pragma unroll
      for (int j = 0; j < P; ++j) now[j] = next[j];
      if (at_once + static_cast<int64_t>(p.slots) * rows < p.tokens) load(token + static_cast<int64_t>(p.slots) * rows, next);
    } else {
      load(token, now);
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
      for (uint4 *v : {&now[j].x, &now[j].h, &now[j].gh, &now[j].gy}) *v = settled(*v, at, j);
    const float factor = live ? gate_of(p, token) : 0.0f;
    float sums[3] = {0.0f, 0.0f, 0.0f};              // of h^2, gy w h, x^2
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float h[kPiece], gy[kPiece], x[kPiece], w[kPiece];
      widen_piece<E>(now[j].h, h);
      widen_piece<E>(now[j].gy, gy);
      if constexpr (kPost) widen_piece<E>(now[j].x, x);
      load_weights(p.weight, at, j, w);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        sums[0] += h[i] * h[i];
        sums[1] += gy[i] * w[i] * h[i];
        if constexpr (kPost) sums[2] += x[i] * x[i];
      }
    }
    row_reduce(sums, p.waves, first[turn], row_wave);
    const float rh = live ? rsqrtf(sums[0] * p.inverse_d + p.eps) : 0.0f, along = sums[1] * rh * p.inverse_d;
    const float rx = !live ? 0.0f : kPost ? rsqrtf(sums[2] * p.inverse_d + p.eps) : 1.0f;
    float dh[P][kPiece], inner[1] = {0.0f};          // sum of dh u
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float h[kPiece], gy[kPiece], gh[kPiece], x[kPiece], w[kPiece], wp[kPiece];
      widen_piece<E>(now[j].h, h);
      widen_piece<E>(now[j].gy, gy);
      widen_piece<E>(now[j].gh, gh);
      widen_piece<E>(now[j].x, x);
      load_weights(p.weight, at, j, w);
      if constexpr (kPost) load_weights(p.post, at, j, wp);
      float grad[kPiece];
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        const float unit = h[i] * rh;
        dw[j][i] += gy[i] * unit;
        dh[j][i] = gh[i] + rh * (gy[i] * w[i] - unit * along);
        inner[0] += dh[j][i] * (kPost ? x[i] * rx * wp[i] : x[i]);
        grad[i] = p.residual_scale * dh[j][i];
      }
      store_piece(p.sum + token * p.ss, at, j, narrow_piece<E>(grad));
    }
    if (kPost || p.grad_gate != nullptr) {
      row_reduce(inner, p.waves, second[turn], row_wave);
      if (p.grad_gate != nullptr && live && thread == 0) p.grad_gate[token * p.ggs] = p.block_scale * inner[0];
    }
    const float back = factor * inner[0] * p.inverse_d;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float x[kPiece], wp[kPiece], grad[kPiece];
      if constexpr (kPost) {
        widen_piece<E>(now[j].x, x);
        load_weights(p.post, at, j, wp);
      }
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        const float du = factor * dh[j][i];
        if constexpr (kPost) {
          const float unit = x[i] * rx;
          dwp[j][i] += du * unit;
          grad[i] = rx * (du * wp[i] - unit * back);
        } else {
          grad[i] = du;
        }
      }
      store_piece(p.out + token * p.os, at, j, narrow_piece<E>(grad));
    }
  }
  const auto at = RowPlace<kPieces>{p.d, p.waves * kWave, thread};
  float *const to = p.partial + static_cast<int64_t>(blockIdx.x) * kWeights * p.d;
  float *const mine = rows == 1 ? to : reinterpret_cast<float *>(shares) + row * kWeights * p.d;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    store_weights(mine, at, j, dw[j]);
    if constexpr (kPost) store_weights(mine + p.d, at, j, dwp[j]);
  }
  if (rows == 1) return;
  __syncthreads();
  for (int i = threadIdx.x; i < kWeights * p.d; i += blockDim.x) {
    float total = 0.0f;
    for (int r = 0; r < rows; ++r) total += reinterpret_cast<const float *>(shares)[r * kWeights * p.d + i];
    to[i] = total;
  }
}

// The weights' gradients: the slots' shares, in a fixed order. One workgroup per 16 dimensions; 64 threads share a dimension.
__global__ __launch_bounds__(16 * kFoldParts) void residual_norm_fold(const float *partial, int slots, int d, int weights, float *dw,
                                                                      float *dpost) {
  __shared__ float sums[kFoldParts][17];
  const int column = threadIdx.x & 15, part = threadIdx.x >> 4, at = blockIdx.x * 16 + column;
  float total = 0.0f;
  if (at < d) {
#pragma unroll 8
    for (int i = part; i < slots; i += kFoldParts) total += partial[(static_cast<int64_t>(i) * weights + blockIdx.y) * d + at];
  }
  sums[part][column] = total;
  __syncthreads();
#pragma unroll
  for (int half = kFoldParts / 2; half >= 1; half /= 2) {
    if (part < half) sums[part][column] += sums[part + half][column];
    __syncthreads();
  }
  if (part == 0 && at < d) (blockIdx.y ? dpost : dw)[at] = sums[0][column];
}

// How a row lies over threads: pieces of a thread, and the waves that its kernel is built for.
struct Layout {
  int pieces, most;
};
// Forward: 16384 x 2048 takes 50.9 us in one piece a thread, 53.0 in two, and 16384 x 4096 99.7 in two, 97.1 in one; 8-bit rows 90.2 in two, 91.8
// in one. One rule for both kinds, so plain rows of 4096 take 3% longer than they could.
// Backward: one piece leaves registers for the rows of the next token (8192 x 8192 184 us; two pieces of 8 waves 191).
Layout forward_layout(int64_t d) { return row_waves(d, 1) <= 4 ? Layout{1, 4} : Layout{2, 16}; }
Layout backward_layout(int64_t d) { return row_waves(d, 1) <= 8 ? Layout{1, 8} : row_waves(d, 1) <= 16 ? Layout{1, 16} : Layout{2, 16}; }
int layout_waves(int64_t d, Layout layout) { return std::max(1, row_waves(d, layout.pieces)); }

// Of the backward: tokens that a workgroup takes at a time, and workgroups, as many as there is room for: registers leave a SIMD four
// waves, and a workgroup of five waves takes the room of eight (16384 x 2056 with three of them for a CU: 157 us, with two 123).
int backward_rows(int64_t d) { return std::max(1, kBackwardWaves / layout_waves(d, backward_layout(d))); }
int backward_slots(int64_t tokens, int64_t d) {
  const int64_t rows = backward_rows(d);
  return static_cast<int>(std::min<int64_t>((tokens + rows - 1) / rows, (backward_layout(d).most == kBackwardWaves ? 2 : 1) * int64_t{device_cus()}));
}

int check(const char *name, int dtype, int64_t tokens, int64_t d, int64_t gates, int64_t post) {
  if (tokens < 0 || d < 0 || gates < 0 || post < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "%s dtype must be F16 or BF16, got %d", name, dtype);
  if (gates != 0 && gates != tokens)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "%lld gates for %lld tokens", static_cast<long long>(gates), static_cast<long long>(tokens));
  if (post != 0 && post != d)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "a norm of the block has %lld weights, rows of %lld", static_cast<long long>(post),
                static_cast<long long>(d));
  if (d > kMaxRow) return fail(INTENT_HIP_ERR_UNSUPPORTED, "%s takes rows of up to %d elements, got %lld", name, kMaxRow, static_cast<long long>(d));
  if (tokens > (1 << 30)) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");        // blocks count in 32 bits
  return INTENT_HIP_OK;
}

// Every address and every stride in bytes, or-ed.
uint64_t mixed_rows(std::initializer_list<const void *> views, std::initializer_list<int64_t> strides, int64_t tokens) {
  uint64_t all = 0;
  for (const void *a : views) all |= static_cast<uint64_t>(reinterpret_cast<uintptr_t>(a));
  if (tokens > 1)
    for (const int64_t s : strides) all |= 2 * static_cast<uint64_t>(s);
  return all;
}

// Whether rows and weights come in 16-byte pieces (rows of 8-bit integers in pieces of 8, so `narrow`, the same of those, counts twice).
bool in_pieces(int64_t d, uint64_t mixed, uint64_t narrow) { return d % kPiece == 0 && (mixed | 2 * narrow) % 16 == 0; }

template <typename F>
auto with_flag(bool flag, F f) {
  return flag ? f(std::true_type{}) : f(std::false_type{});
}
// f with the kernel of a call.
template <typename F>
int with_forward(int dtype, int64_t d, bool in_pieces, bool post, bool i8, F f) {
  return with_flag(forward_layout(d).pieces == 1, [&](auto one) {
    return with_flag(in_pieces, [&](auto whole) {
      return with_flag(post, [&](auto norm) {
        return with_flag(i8, [&](auto eight) {
          constexpr int P = one.value ? 1 : 2, W = one.value ? 4 : 16;
          return f(dtype == INTENT_HIP_F16 ? residual_norm_rows<f16_t, P, W, whole.value, norm.value, eight.value>
                                           : residual_norm_rows<bf16_t, P, W, whole.value, norm.value, eight.value>);
        });
      });
    });
  });
}

template <typename F>
int with_backward(int dtype, int64_t d, bool in_pieces, bool post, F f) {
  const Layout layout = backward_layout(d);
  return with_flag(in_pieces, [&](auto whole) {
    return with_flag(post, [&](auto norm) {
      const auto of = [&](auto pieces, auto waves) {
        return f(dtype == INTENT_HIP_F16 ? residual_norm_backward_rows<f16_t, pieces.value, waves.value, whole.value, norm.value>
                                         : residual_norm_backward_rows<bf16_t, pieces.value, waves.value, whole.value, norm.value>);
      };
      const std::integral_constant<int, 1> one;
      const std::integral_constant<int, 2> two;
      const std::integral_constant<int, 8> eight;
      const std::integral_constant<int, 16> sixteen;
      return layout.most == 8 ? of(one, eight) : layout.pieces == 1 ? of(one, sixteen) : of(two, sixteen);
    });
  });
}

int backward_threads(int64_t d) { return layout_waves(d, backward_layout(d)) * backward_rows(d) * kWave; }
unsigned row_threads(int waves) { return static_cast<unsigned>((waves == 1 ? kWaveRows : waves) * kWave); }

}  // namespace

int residual_norm_resources(int dtype, int kind, int64_t d, int64_t post, uint64_t mix, IntentHipKernelResources *out) {
  if (d < 0 || d > kMaxRow) return fail(INTENT_HIP_ERR_UNSUPPORTED, "residual_norm takes rows of up to %d elements", kMaxRow);
  const bool whole = in_pieces(d, mix, 0);
  const Layout layout = kind == 2 ? backward_layout(d) : forward_layout(d);
  char name[96];
  snprintf(name, sizeof(name), "residual_norm_%srows<%s,%d,%s,%s%s>", kind == 2 ? "backward_" : "", dtype == INTENT_HIP_F16 ? "f16" : "bf16", layout.pieces,
           whole ? "true" : "false", post ? "true" : "false", kind == 2 ? "" : kind == 1 ? ",true" : ",false");
  const auto describe = [&](void (*kernel)(Norm)) {
    return describe_kernel(reinterpret_cast<const void *>(kernel), name, kind == 2 ? backward_threads(d) : static_cast<int>(row_threads(layout_waves(d, layout))), out);
  };
  return kind == 2 ? with_backward(dtype, d, whole, post != 0, describe) : with_forward(dtype, d, whole, post != 0, kind == 1, describe);
}

namespace {

int forward(const char *name, bool i8, int dtype, const void *block, const void *residual, const float *gate, const float *post,
            const float *weight, void *sum, void *out, float *scales, int64_t tokens, int64_t d, int64_t gates, int64_t posts,
            const int64_t *strides, float residual_scale, float block_scale, float eps, void *stream) {
  if (int rc = check(name, dtype, tokens, d, gates, posts)) return rc;
  if (tokens == 0) return INTENT_HIP_OK;
  if (strides == nullptr || (i8 && scales == nullptr)) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  for (int i = 0; i < 5; ++i)
    if (strides[i] < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (d == 0 && !i8) return INTENT_HIP_OK;
  if (d > 0 && (block == nullptr || residual == nullptr || weight == nullptr || sum == nullptr || out == nullptr ||
                (gates > 0 && gate == nullptr) || (posts > 0 && post == nullptr)))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  Norm p{};
  p.block = static_cast<const uint16_t *>(block), p.residual = static_cast<const uint16_t *>(residual);
  p.gate = gates > 0 ? gate : nullptr, p.post = post, p.weight = weight, p.sum = static_cast<uint16_t *>(sum);
  (i8 ? reinterpret_cast<void *&>(p.q) : reinterpret_cast<void *&>(p.out)) = out;
  p.scales = scales;
  p.bs = strides[0], p.rs = strides[1], p.gs = strides[2], p.ss = strides[3], p.os = strides[4];
  p.tokens = tokens, p.d = static_cast<int>(d), p.residual_scale = residual_scale, p.block_scale = block_scale, p.eps = eps;
  p.inverse_d = d > 0 ? 1.0f / static_cast<float>(d) : 0.0f;
  p.waves = layout_waves(d, forward_layout(d));
  const uint64_t wide = mixed_rows({block, residual, sum, weight, posts > 0 ? post : nullptr, i8 ? nullptr : out}, {p.bs, p.rs, p.ss, i8 ? 0 : p.os}, tokens);
  const uint64_t narrow = i8 ? reinterpret_cast<uintptr_t>(out) | (tokens > 1 ? static_cast<uint64_t>(p.os) : 0) : 0;
  const int rows = p.waves == 1 ? kWaveRows : 1;
  with_forward(dtype, d, in_pieces(d, wide, narrow), posts > 0, i8, [&](void (*kernel)(Norm)) {
    kernel<<<tile_grid((tokens + rows - 1) / rows, 1), row_threads(p.waves), 0, as_stream(stream)>>>(p);
    return 0;
  });
  return hipPeekAtLastError() != hipSuccess ? launch_status(name) : INTENT_HIP_OK;
}

}  // namespace
}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_residual_norm(int dtype, const void *block, const void *residual, const float *gate, const float *post_weight,
                                        const float *weight, void *sum, void *output, int64_t tokens, int64_t d, int64_t gates,
                                        int64_t post, const int64_t *strides, float residual_scale, float block_scale, float eps,
                                        void *stream) {
  return forward("residual_norm", false, dtype, block, residual, gate, post_weight, weight, sum, output, nullptr, tokens, d, gates, post, strides,
                 residual_scale, block_scale, eps, stream);
}

extern "C" int intent_hip_residual_norm_i8(int dtype, const void *block, const void *residual, const float *gate, const float *post_weight,
                                           const float *weight, void *sum, int8_t *output, float *scales, int64_t tokens, int64_t d,
                                           int64_t gates, int64_t post, const int64_t *strides, float residual_scale, float block_scale,
                                           float eps, void *stream) {
  return forward("residual_norm_i8", true, dtype, block, residual, gate, post_weight, weight, sum, output, scales, tokens, d, gates, post, strides,
                 residual_scale, block_scale, eps, stream);
}

extern "C" int intent_hip_residual_norm_backward_workspace_bytes(int64_t tokens, int64_t d, int64_t post, size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (int rc = check("residual_norm_backward", INTENT_HIP_F16, tokens, d, 0, post)) return rc;
  if (d > 0) *bytes = static_cast<size_t>(backward_slots(tokens, d)) * (post > 0 ? 2 : 1) * d * sizeof(float);
  return INTENT_HIP_OK;
}

extern "C" int intent_hip_residual_norm_backward(int dtype, const void *block, const void *sum, const float *gate, const float *post_weight,
                                                 const float *weight, const void *grad_sum, const void *grad_output, void *grad_block,
                                                 void *grad_residual, float *grad_gate, float *grad_post_weight, float *grad_weight,
                                                 int64_t tokens, int64_t d, int64_t gates, int64_t post, const int64_t *strides,
                                                 float residual_scale, float block_scale, float eps, void *workspace,
                                                 size_t workspace_bytes, void *stream) {
  if (int rc = check("residual_norm_backward", dtype, tokens, d, gates, post)) return rc;
  if (d == 0 && gates == 0) return INTENT_HIP_OK;
  if ((d > 0 && grad_weight == nullptr) || (post > 0 && grad_post_weight == nullptr) || (gates > 0 && (gate == nullptr || grad_gate == nullptr)))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  const int slots = backward_slots(tokens, d);
  const int weights = post > 0 ? 2 : 1;
  const size_t bytes = static_cast<size_t>(slots) * weights * d * sizeof(float);
  if (slots > 0) {
    if (strides == nullptr || (d > 0 && (block == nullptr || sum == nullptr || weight == nullptr || grad_sum == nullptr || grad_output == nullptr ||
                                         grad_block == nullptr || grad_residual == nullptr || (post > 0 && post_weight == nullptr))))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
    for (int i = 0; i < 8; ++i)
      if (strides[i] < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
    if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16)))
      return fail(INTENT_HIP_ERR_WORKSPACE, "residual_norm_backward needs %zu workspace bytes, 16-byte aligned", bytes);
    Norm p{};
    p.block = static_cast<const uint16_t *>(block), p.residual = static_cast<const uint16_t *>(sum);
    p.grad_sum = static_cast<const uint16_t *>(grad_sum), p.grad_out = static_cast<const uint16_t *>(grad_output);
    p.gate = gates > 0 ? gate : nullptr, p.post = post_weight, p.weight = weight;
    p.out = static_cast<uint16_t *>(grad_block), p.sum = static_cast<uint16_t *>(grad_residual);
    p.grad_gate = gates > 0 ? grad_gate : nullptr, p.partial = static_cast<float *>(workspace);
    p.bs = strides[0], p.rs = strides[1], p.gs = strides[2], p.gss = strides[3], p.gos = strides[4], p.os = strides[5], p.ss = strides[6], p.ggs = strides[7];
    p.tokens = tokens, p.d = static_cast<int>(d), p.residual_scale = residual_scale, p.block_scale = block_scale, p.eps = eps;
    p.inverse_d = d > 0 ? 1.0f / static_cast<float>(d) : 0.0f;
    p.waves = layout_waves(d, backward_layout(d)), p.slots = slots;
    const uint64_t wide = mixed_rows({block, sum, grad_sum, grad_output, grad_block, grad_residual, weight, post > 0 ? post_weight : nullptr},
                                     {p.bs, p.rs, p.gss, p.gos, p.os, p.ss}, tokens);
    with_backward(dtype, d, in_pieces(d, wide, 0), post > 0, [&](void (*kernel)(Norm)) {
      kernel<<<static_cast<unsigned>(slots), static_cast<unsigned>(backward_threads(d)), 0, as_stream(stream)>>>(p);
      return 0;
    });
    if (hipPeekAtLastError() != hipSuccess) return launch_status("residual_norm_backward");
  }
  if (d == 0) return INTENT_HIP_OK;
  residual_norm_fold<<<dim3(static_cast<unsigned>((d + 15) / 16), static_cast<unsigned>(weights)), 16 * kFoldParts, 0, as_stream(stream)>>>(
      static_cast<const float *>(workspace), slots, static_cast<int>(d), weights, grad_weight, grad_post_weight);
  return hipPeekAtLastError() != hipSuccess ? launch_status("residual_norm_fold") : INTENT_HIP_OK;
}

// Norm and rotation of query and key heads (forward and backward), for gfx950. No reference counterpart.
//
// A row is one (token, head): y = x * rsqrt(mean(x^2) + eps) * w in f32, whose first 2R dimensions are R pairs turned by
// the token's angles. Backward: g = the gradient turned back; u = x r; grad_x = r (g w - u mean(g w u)); grad_w = the sum
// of g u over rows, through f32 partial sums per workgroup that a second kernel adds in order.
//
// Bound by the rows' bytes, so each is read and written once, in whole 16-byte pieces (bf16, 16384 tokens of 32 + 8 heads of 128:
// forward 67 us, 5.1 TB/s; backward 102 us, 5.0 TB/s, and 4 for the sums); with few tokens by latency and launches (8 tokens: 3.1
// and 7.2 us). Layouts without such pieces (D no multiple of 16, R no multiple of 8, odd strides) take two bytes a lane: 342 and
// 999 us; heads of 80 with 10 pairs turned 276 and 916, all 40 turned 55 and 95.
#include <stdio.h>

#include <algorithm>

#include "common.hpp"

namespace intent_hip {
namespace {

constexpr int kMaxWidth = 1024;       // head width: a wave holds a row in 16 registers a lane
constexpr int kRowRegisters = kMaxWidth / kWave;
constexpr int kWaves = 4;
constexpr int kMaxHeads = INT32_MAX / 4;        // of queries, of keys: a walk over both, and a step past its end, stay within 32 bits

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

// The backward of the same: waves walk rows of the queries, then of the keys, and keep their share of the weight's gradient
// in registers until the end. partial: [workgroup][queries, keys][d].
template <typename E>
__global__ __launch_bounds__(kWaves * kWave) void norm_rope_backward_any(NormRope p, float *partial) {
  __shared__ float sums[kWaves][kMaxWidth];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int which = 0; which < 2; ++which) {
    const int heads = p.heads[which];
    const int64_t rows = p.tokens * heads;
    const float *w = p.w[which];
    float dw[kRowRegisters];
#pragma unroll
    for (int j = 0; j < kRowRegisters; ++j) dw[j] = 0.0f;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + wave; row < rows; row += static_cast<int64_t>(gridDim.x) * kWaves) {
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
      partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.d + d] = total;
    }
    __syncthreads();
  }
}

// grad_w[which][d]: the workgroups' partial sums, in a fixed order. One workgroup per 16 dimensions of the queries' or the
// keys' weight; 64 threads share a dimension (a row's 16 values are half a line), so few loads wait for each other.
constexpr int kFoldParts = 64;
__global__ __launch_bounds__(16 * kFoldParts) void norm_rope_fold(const float *partial, int blocks, int d, float *dq, float *dk) {
  __shared__ float sums[kFoldParts][17];
  const int column = threadIdx.x & 15, part = threadIdx.x >> 4, at = blockIdx.x * 16 + column;
  const int which = blockIdx.y;
  float total = 0.0f;
  if (at < d) {
#pragma unroll 8
    for (int i = part; i < blocks; i += kFoldParts) total += partial[(static_cast<int64_t>(i) * 2 + which) * d + at];
  }
  sums[part][column] = total;
  __syncthreads();
#pragma unroll
  for (int half = kFoldParts / 2; half >= 1; half /= 2) {
    if (part < half) sums[part][column] += sums[part + half][column];
    __syncthreads();
  }
  if (part == 0 && at < d) (which ? dk : dq)[at] = sums[0][column];
}

// ---------------------------------------------------------------- rows of 16-byte pieces
// Widths of a multiple of 16 with R a multiple of 8, aligned rows. G lanes hold a row, a lane eight pairs: dimensions
// 8 c .. and 8 c + R .. (rotated), or R + 8 c .. and D / 2 + 8 c .. (the rest, paired the same way), or 16 c .. 16 c + 15
// where pairs lie side by side. A pair's two values are then a lane's own, and a wave reads and writes whole rows in 16-byte
// pieces. A wave takes one token, 64 / G heads at a time, queries then keys, so its angles are read once.
template <bool kInterleaved>
struct Piece {
  int a, b;                            // offsets of the two runs of 8
  bool live, turned;
  __device__ __forceinline__ Piece(const NormRope &p, int c) {
    live = 16 * c < p.d;
    turned = 8 * c < p.pairs;
    a = kInterleaved ? 16 * c : turned ? 8 * c : p.pairs + 8 * c;
    b = kInterleaved ? 16 * c + 8 : turned ? 8 * c + p.pairs : p.d / 2 + 8 * c;
  }
};

// Firsts and seconds of the eight pairs from two runs of 8, and back.
template <bool kInterleaved, typename T>
__device__ __forceinline__ void apart(const T (&u)[8], const T (&v)[8], T (&first)[8], T (&second)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    first[j] = kInterleaved ? (j < 4 ? u[2 * j] : v[2 * j - 8]) : u[j];
    second[j] = kInterleaved ? (j < 4 ? u[2 * j + 1] : v[2 * j - 7]) : v[j];
  }
}
template <bool kInterleaved, typename T>
__device__ __forceinline__ void together(const T (&first)[8], const T (&second)[8], T (&u)[8], T (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    u[j] = kInterleaved ? (j & 1 ? second[j / 2] : first[j / 2]) : first[j];
    v[j] = kInterleaved ? (j & 1 ? second[4 + j / 2] : first[4 + j / 2]) : second[j];
  }
}

template <typename E>
__device__ __forceinline__ void widen(uint4 raw, float (&out)[8]) {
  const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) out[j] = to_f32(E{static_cast<uint16_t>(words[j / 2] >> (16 * (j & 1)))});
}
template <typename E>
__device__ __forceinline__ uint4 narrow(const float (&v)[8]) {
  uint32_t words[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    words[j] = from_f32<E>(v[2 * j]).bits | static_cast<uint32_t>(from_f32<E>(v[2 * j + 1]).bits) << 16;
  return make_uint4(words[0], words[1], words[2], words[3]);
}

__device__ __forceinline__ void read8(const float *at, float (&out)[8]) {
  const float4 u = *reinterpret_cast<const float4 *>(at), v = *reinterpret_cast<const float4 *>(at + 4);
  out[0] = u.x, out[1] = u.y, out[2] = u.z, out[3] = u.w, out[4] = v.x, out[5] = v.y, out[6] = v.z, out[7] = v.w;
}

// Sum over the G lanes of a row, in every one of them.
template <int G>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  if constexpr (G >= 8) v += dpp_move<0x141>(v);
  if constexpr (G >= 16) v += dpp_move<0x140>(v);
  if constexpr (G >= 32) v += __shfl_xor(v, 16);
  if constexpr (G >= 64) v += __shfl_xor(v, 32);
  return v;
}

// What a lane keeps for a token: its eight pairs' cosines and sines (1 and 0 where they are not turned).
template <bool kInterleaved>
__device__ __forceinline__ void angles(const NormRope &p, const Piece<kInterleaved> &at, int c, int64_t token, float (&cs)[8],
                                       float (&sn)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = 1.0f, sn[j] = 0.0f;
  if (at.live && at.turned) {
    const int64_t row = table_row(p, token);
    read8(p.cos + row * p.coss + 8 * c, cs);
    read8(p.sin + row * p.sins + 8 * c, sn);
  }
}

// The weights of a lane's pairs.
template <bool kInterleaved>
__device__ __forceinline__ void weights(const float *w, const Piece<kInterleaved> &at, float (&first)[8], float (&second)[8]) {
  float u[8] = {}, v[8] = {};
  if (at.live && w != nullptr) read8(w + at.a, u), read8(w + at.b, v);
  apart<kInterleaved>(u, v, first, second);
}

// `waves` waves share a token's heads.
template <typename E, int G, bool kInterleaved>
__global__ __launch_bounds__(kWaves * kWave) void norm_rope_rows(NormRope p, int waves) {
  constexpr int kRows = kWave / G;
  const int lane = threadIdx.x & 63, c = lane % G;
  const int64_t job = static_cast<int64_t>(grid_block()) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = job / waves;
  if (token >= p.tokens) return;
  const int heads = p.heads[0] + p.heads[1];
  const Piece<kInterleaved> at(p, c);
  float wq[2][8], wk[2][8], cs[8], sn[8];
  struct Row {
    uint4 a, b;
    bool live;
  };
  const auto load = [&](int f) {
    Row x{make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0), at.live && f < heads};
    if (x.live) {
      const int which = f >= p.heads[0];
      const uint16_t *from = p.x[which] + token * p.xs[which][0] + (f - (which ? p.heads[0] : 0)) * p.xs[which][1];
      x.a = *reinterpret_cast<const uint4 *>(from + at.a);
      x.b = *reinterpret_cast<const uint4 *>(from + at.b);
    }
    return x;
  };
  int f0 = static_cast<int>(job % waves) * kRows;
  Row next = load(f0 + lane / G);
  angles(p, at, c, token, cs, sn);
  weights(p.w[0], at, wq[0], wq[1]);
  weights(p.w[1], at, wk[0], wk[1]);
  for (; f0 < heads; f0 += waves * kRows) {
    const int f = f0 + lane / G, which = f >= p.heads[0];
    const Row x = next;
    if (f0 + waves * kRows < heads) next = load(f + waves * kRows);
    float u[8], v[8], first[8], second[8], sum = 0.0f;
    widen<E>(x.a, u);
    widen<E>(x.b, v);
    apart<kInterleaved>(u, v, first, second);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += first[j] * first[j] + second[j] * second[j];
    const float r = rsqrtf(row_sum<G>(sum) / p.d + p.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = first[j] * r * (which ? wk[0][j] : wq[0][j]), b = second[j] * r * (which ? wk[1][j] : wq[1][j]);
      first[j] = at.turned ? a * cs[j] - b * sn[j] : a;
      second[j] = at.turned ? b * cs[j] + a * sn[j] : b;
    }
    if (!x.live) continue;
    together<kInterleaved>(first, second, u, v);
    uint16_t *to = p.out[which] + token * p.outs[which][0] + (f - (which ? p.heads[0] : 0)) * p.outs[which][1];
    *reinterpret_cast<uint4 *>(to + at.a) = narrow<E>(u);
    *reinterpret_cast<uint4 *>(to + at.b) = narrow<E>(v);
  }
}

// The backward of the same; waves walk tokens (`waves` of them share one's heads) and keep their share of the weights'
// gradients in registers.
template <typename E, int G, bool kInterleaved>
__global__ __launch_bounds__(kWaves * kWave) void norm_rope_backward_rows(NormRope p, float *partial, int waves) {
  constexpr int kRows = kWave / G;
  __shared__ float sums[kWaves][2][16 * G];
  const int lane = threadIdx.x & 63, c = lane % G, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = p.heads[0] + p.heads[1];
  const Piece<kInterleaved> at(p, c);
  float wq[2][8], wk[2][8], dq[2][8], dk[2][8];
  weights(p.w[0], at, wq[0], wq[1]);
  weights(p.w[1], at, wk[0], wk[1]);
#pragma unroll
  for (int j = 0; j < 8; ++j) dq[0][j] = dq[1][j] = dk[0][j] = dk[1][j] = 0.0f;
  struct Row {
    uint4 a, b, da, db;
    bool live;
  };
  const auto load = [&](int64_t token, int f) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    Row x{zero, zero, zero, zero, at.live && f < heads};
    if (x.live) {
      const int which = f >= p.heads[0], head = f - (which ? p.heads[0] : 0);
      const uint16_t *from = p.x[which] + token * p.xs[which][0] + head * p.xs[which][1];
      const uint16_t *grad = p.dy[which] + token * p.dys[which][0] + head * p.dys[which][1];
      x.a = *reinterpret_cast<const uint4 *>(from + at.a);
      x.b = *reinterpret_cast<const uint4 *>(from + at.b);
      x.da = *reinterpret_cast<const uint4 *>(grad + at.a);
      x.db = *reinterpret_cast<const uint4 *>(grad + at.b);
    }
    return x;
  };
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kWaves, jobs = p.tokens * waves;
  for (int64_t job = static_cast<int64_t>(blockIdx.x) * kWaves + wave; job < jobs; job += stride) {
    const int64_t token = waves == 1 ? job : job / waves;
    float cs[8], sn[8];
    int f0 = static_cast<int>(job - token * waves) * kRows;
    Row next = load(token, f0 + lane / G);
    angles(p, at, c, token, cs, sn);
    for (; f0 < heads; f0 += waves * kRows) {
      const int f = f0 + lane / G, which = f >= p.heads[0];
      const Row x = next;
      if (f0 + waves * kRows < heads) next = load(token, f + waves * kRows);
      float u[8], v[8], first[8], second[8], ga[8], gb[8], sum = 0.0f, along = 0.0f;
      widen<E>(x.a, u);
      widen<E>(x.b, v);
      apart<kInterleaved>(u, v, first, second);
      widen<E>(x.da, u);
      widen<E>(x.db, v);
      apart<kInterleaved>(u, v, ga, gb);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += first[j] * first[j] + second[j] * second[j];
      // A place without a row adds nothing, also where the rows need no eps.
      const float mean = row_sum<G>(sum) / p.d, r = f < heads ? rsqrtf(mean + p.eps) : 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = at.turned ? ga[j] * cs[j] + gb[j] * sn[j] : ga[j], b = at.turned ? gb[j] * cs[j] - ga[j] * sn[j] : gb[j];
        first[j] *= r, second[j] *= r;
        const float da = a * first[j], db = b * second[j];
        dq[0][j] += which ? 0.0f : da, dq[1][j] += which ? 0.0f : db;
        dk[0][j] += which ? da : 0.0f, dk[1][j] += which ? db : 0.0f;
        ga[j] = a * (which ? wk[0][j] : wq[0][j]), gb[j] = b * (which ? wk[1][j] : wq[1][j]);
        along += ga[j] * first[j] + gb[j] * second[j];
      }
      along = row_sum<G>(along) / p.d;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        first[j] = r * (ga[j] - first[j] * along);
        second[j] = r * (gb[j] - second[j] * along);
      }
      if (!x.live) continue;
      together<kInterleaved>(first, second, u, v);
      uint16_t *to = p.out[which] + token * p.outs[which][0] + (f - (which ? p.heads[0] : 0)) * p.outs[which][1];
      *reinterpret_cast<uint4 *>(to + at.a) = narrow<E>(u);
      *reinterpret_cast<uint4 *>(to + at.b) = narrow<E>(v);
    }
  }
  // Over the rows of a wave, then over the waves.
  const auto put = [&](int which, float (&first)[8], float (&second)[8]) {
    float u[8], v[8];
#pragma unroll
    for (int step = G; step < kWave; step *= 2)
#pragma unroll
      for (int j = 0; j < 8; ++j) first[j] += __shfl_xor(first[j], step), second[j] += __shfl_xor(second[j], step);
    together<kInterleaved>(first, second, u, v);
    if (lane < G && at.live)
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[wave][which][at.a + j] = u[j], sums[wave][which][at.b + j] = v[j];
  };
  put(0, dq[0], dq[1]);
  put(1, dk[0], dk[1]);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.d; i += kWaves * kWave) {
    const int which = i / p.d, d = i % p.d;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += sums[w][which][d];
    partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * p.d + d] = total;
  }
}

// Workgroups of the backward pass: as many as the chip holds at once (16384 tokens: 106 us; half as many 145, twice as many
// 107), fewer where a wave would have no row.
int backward_blocks(int64_t tokens, int64_t q_heads, int64_t kv_heads) {
  const int64_t rows = tokens * (q_heads + kv_heads), wanted = (rows + kWaves - 1) / kWaves, most = 2 * device_cus();
  return static_cast<int>(wanted < most ? wanted : most);
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
  if (q_heads > kMaxHeads || kv_heads > kMaxHeads) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  if (q_heads + kv_heads > 0 && tokens > (int64_t{1} << 32) / (q_heads + kv_heads))
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

// Whether rows, weights and tables can be read in 16-byte pieces: `mixed` is every address and every stride in bytes, or-ed.
bool in_pieces(int64_t d, int64_t pairs, uint64_t mixed) { return d % 16 == 0 && pairs % 8 == 0 && mixed % 16 == 0; }

uint64_t mixed(const NormRope &p, bool backward) {
  const auto at = [](const void *a) { return static_cast<uint64_t>(reinterpret_cast<uintptr_t>(a)); };
  uint64_t all = p.pairs == 0 ? 0 : at(p.cos) | at(p.sin) | 4 * static_cast<uint64_t>(p.coss | p.sins);
  for (int i = 0; i < 2; ++i) {
    if (p.heads[i] == 0) continue;
    all |= at(p.x[i]) | at(p.out[i]) | at(p.w[i]) | 2 * static_cast<uint64_t>(p.xs[i][0] | p.xs[i][1] | p.outs[i][0] | p.outs[i][1]);
    if (backward) all |= at(p.dy[i]) | 2 * static_cast<uint64_t>(p.dys[i][0] | p.dys[i][1]);
  }
  return all;
}

// Lanes of a row: the power of two that covers its pieces of 16 (at least a quad).
int row_lanes(int d) {
  int g = 4;
  while (16 * g < d) g *= 2;
  return g;
}

// Waves of a token: more than one where tokens alone leave CUs idle (forward, 40 heads of 128: 8 tokens 3.1 us, a wave each 5.6;
// 512 tokens 4.8 and 6.4; backward with its second kernel 7.2 and 11.1, 10.4 and 12.3).
int token_waves(const NormRope &p) {
  const int rows = kWave / row_lanes(p.d), steps = (p.heads[0] + p.heads[1] + rows - 1) / rows;
  const int64_t spare = (8 * static_cast<int64_t>(device_cus()) + p.tokens - 1) / p.tokens;
  return static_cast<int>(spare < steps ? spare : steps);
}

template <typename E, int G>
void launch_rows(const NormRope &p, hipStream_t s) {
  const int waves = token_waves(p);
  const dim3 grid = tile_grid((p.tokens * waves + kWaves - 1) / kWaves, 1);
  if (p.interleaved)
    norm_rope_rows<E, G, true><<<grid, kWaves * kWave, 0, s>>>(p, waves);
  else
    norm_rope_rows<E, G, false><<<grid, kWaves * kWave, 0, s>>>(p, waves);
}

template <typename E, int G>
void launch_backward_rows(const NormRope &p, int blocks, float *partial, hipStream_t s) {
  if (p.interleaved)
    norm_rope_backward_rows<E, G, true><<<blocks, kWaves * kWave, 0, s>>>(p, partial, token_waves(p));
  else
    norm_rope_backward_rows<E, G, false><<<blocks, kWaves * kWave, 0, s>>>(p, partial, token_waves(p));
}

template <typename E>
void launch_forward(const NormRope &p, hipStream_t s) {
  if (!in_pieces(p.d, p.pairs, mixed(p, false))) {
    const int64_t rows = p.tokens * (p.heads[0] + p.heads[1]);
    norm_rope_any<E><<<tile_grid((rows + kWaves - 1) / kWaves, 1), kWaves * kWave, 0, s>>>(p);
    return;
  }
  switch (row_lanes(p.d)) {
    case 4: return launch_rows<E, 4>(p, s);
    case 8: return launch_rows<E, 8>(p, s);
    case 16: return launch_rows<E, 16>(p, s);
    case 32: return launch_rows<E, 32>(p, s);
    default: return launch_rows<E, 64>(p, s);
  }
}

template <typename E>
void launch_backward(const NormRope &p, int blocks, float *partial, hipStream_t s) {
  if (!in_pieces(p.d, p.pairs, mixed(p, true))) {
    norm_rope_backward_any<E><<<blocks, kWaves * kWave, 0, s>>>(p, partial);
    return;
  }
  switch (row_lanes(p.d)) {
    case 4: return launch_backward_rows<E, 4>(p, blocks, partial, s);
    case 8: return launch_backward_rows<E, 8>(p, blocks, partial, s);
    case 16: return launch_backward_rows<E, 16>(p, blocks, partial, s);
    case 32: return launch_backward_rows<E, 32>(p, blocks, partial, s);
    default: return launch_backward_rows<E, 64>(p, blocks, partial, s);
  }
}

}  // namespace

int norm_rope_resources(int dtype, int backward, int64_t d, int64_t pairs, int interleaved, uint64_t mix,
                        IntentHipKernelResources *out) {
  if (d < 0 || d > kMaxWidth) return fail(INTENT_HIP_ERR_UNSUPPORTED, "qk_norm_rope takes heads of up to %d dimensions", kMaxWidth);
  const char *const type = dtype == INTENT_HIP_F16 ? "f16" : "bf16";
  char name[64];
  const auto describe = [&](const void *half, const void *brain) {
    return describe_kernel(dtype == INTENT_HIP_F16 ? half : brain, name, kWaves * kWave, out);
  };
  if (!in_pieces(d, pairs, mix)) {
    snprintf(name, sizeof(name), "norm_rope_%sany<%s>", backward ? "backward_" : "", type);
    return backward ? describe(reinterpret_cast<const void *>(norm_rope_backward_any<f16_t>),
                               reinterpret_cast<const void *>(norm_rope_backward_any<bf16_t>))
                    : describe(reinterpret_cast<const void *>(norm_rope_any<f16_t>),
                               reinterpret_cast<const void *>(norm_rope_any<bf16_t>));
  }
  const int g = row_lanes(static_cast<int>(d));
  snprintf(name, sizeof(name), "norm_rope_%srows<%s,%d,%s>", backward ? "backward_" : "", type, g, interleaved ? "true" : "false");
#define INTENT_HIP_ROWS(G)                                                                                                      \
  case G:                                                                                                                       \
    if (backward)                                                                                                               \
      return interleaved ? describe(reinterpret_cast<const void *>(norm_rope_backward_rows<f16_t, G, true>),                    \
                                    reinterpret_cast<const void *>(norm_rope_backward_rows<bf16_t, G, true>))                   \
                         : describe(reinterpret_cast<const void *>(norm_rope_backward_rows<f16_t, G, false>),                   \
                                    reinterpret_cast<const void *>(norm_rope_backward_rows<bf16_t, G, false>));                 \
    return interleaved ? describe(reinterpret_cast<const void *>(norm_rope_rows<f16_t, G, true>),                               \
                                  reinterpret_cast<const void *>(norm_rope_rows<bf16_t, G, true>))                              \
                       : describe(reinterpret_cast<const void *>(norm_rope_rows<f16_t, G, false>),                              \
                                  reinterpret_cast<const void *>(norm_rope_rows<bf16_t, G, false>))
  switch (g) {
    INTENT_HIP_ROWS(4);
    INTENT_HIP_ROWS(8);
    INTENT_HIP_ROWS(16);
    INTENT_HIP_ROWS(32);
    INTENT_HIP_ROWS(64);
  }
#undef INTENT_HIP_ROWS
  return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "qk_norm_rope takes heads of up to %d dimensions", kMaxWidth);
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
  p.tokens = tokens, p.heads[0] = static_cast<int>(q_heads), p.heads[1] = static_cast<int>(kv_heads);
  for (int i = 0; i < 2; ++i) {
    p.xs[i][0] = strides[3 * i], p.xs[i][1] = strides[3 * i + 1];
    p.outs[i][0] = strides[10 + 3 * i], p.outs[i][1] = strides[11 + 3 * i];
    if (p.heads[i] > 0 && d > 1 && (strides[3 * i + 2] != 1 || strides[12 + 3 * i] != 1))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows need unit inner stride");
  }
  if (pairs > 1 && (strides[7] != 1 || strides[9] != 1)) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "tables need unit inner stride");
  p.coss = strides[6], p.sins = strides[8], p.table = table;
  p.d = static_cast<int>(d), p.pairs = static_cast<int>(pairs), p.interleaved = interleaved != 0, p.eps = eps;
  if (dtype == INTENT_HIP_F16)
    launch_forward<f16_t>(p, as_stream(stream));
  else
    launch_forward<bf16_t>(p, as_stream(stream));
  return hipPeekAtLastError() != hipSuccess ? launch_status("norm_rope") : INTENT_HIP_OK;
}

extern "C" int intent_hip_qk_norm_rope_backward_workspace_bytes(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t d,
                                                                size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || d < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (q_heads > kMaxHeads || kv_heads > kMaxHeads || d > kMaxWidth ||
      (q_heads + kv_heads > 0 && tokens > (int64_t{1} << 32) / (q_heads + kv_heads)))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  *bytes = static_cast<size_t>(backward_blocks(tokens, q_heads, kv_heads)) * 2 * d * sizeof(float);
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
  int blocks = backward_blocks(tokens, q_heads, kv_heads);
  const size_t bytes = static_cast<size_t>(blocks) * 2 * d * sizeof(float);
  float *partial = static_cast<float *>(workspace);
  if (blocks > 0) {
    if ((q_heads > 0 && grad_q_out == nullptr) || (kv_heads > 0 && grad_k_out == nullptr))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
    if (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16))
      return fail(INTENT_HIP_ERR_WORKSPACE, "qk_norm_rope_backward needs %zu workspace bytes, 16-byte aligned", bytes);
    p.tokens = tokens, p.heads[0] = static_cast<int>(q_heads), p.heads[1] = static_cast<int>(kv_heads);
    for (int i = 0; i < 2; ++i) {
      p.xs[i][0] = strides[3 * i], p.xs[i][1] = strides[3 * i + 1];
      p.dys[i][0] = strides[10 + 3 * i], p.dys[i][1] = strides[11 + 3 * i];
      p.outs[i][0] = strides[16 + 3 * i], p.outs[i][1] = strides[17 + 3 * i];
      if (p.heads[i] > 0 && d > 1 && (strides[3 * i + 2] != 1 || strides[12 + 3 * i] != 1 || strides[18 + 3 * i] != 1))
        return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows need unit inner stride");
    }
    if (pairs > 1 && (strides[7] != 1 || strides[9] != 1))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "tables need unit inner stride");
    p.coss = strides[6], p.sins = strides[8], p.table = table;
    p.d = static_cast<int>(d), p.pairs = static_cast<int>(pairs), p.interleaved = interleaved != 0, p.eps = eps;
    if (in_pieces(d, pairs, mixed(p, true)))
      blocks = static_cast<int>(std::min<int64_t>(blocks, (tokens * token_waves(p) + kWaves - 1) / kWaves));      // none without a job
    if (dtype == INTENT_HIP_F16)
      launch_backward<f16_t>(p, blocks, partial, as_stream(stream));
    else
      launch_backward<bf16_t>(p, blocks, partial, as_stream(stream));
    if (hipPeekAtLastError() != hipSuccess) return launch_status("norm_rope_backward");
  }
  norm_rope_fold<<<dim3(static_cast<unsigned>((d + 15) / 16), 2), 16 * kFoldParts, 0, as_stream(stream)>>>(
      partial, blocks, static_cast<int>(d), grad_q_weight, grad_k_weight);
  return hipPeekAtLastError() != hipSuccess ? launch_status("norm_rope_fold") : INTENT_HIP_OK;
}

// Attention of one new token per sequence over a prefix that all sequences share and over the pages of each, for gfx950. No reference
// counterpart; the cache is the paged one of 16-bit rows that paged_gqa_decode_partials reads.
//
// For query head h of sequence s, over the prefix's tokens and the sequence's own:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp2(scale * log2(e) * (q . k_j) - peak)        0 where there is no token
// Products are summed in f32. Weights enter the second product as two numbers of the queries' type each: two of f16 hold 21 bits, at 2^11
// times their share of the largest, which leaves out no more than 2^-36 of that; two of bf16 hold 16. The sum that divides is of the
// weights as they were rounded, so a rounding moves a weight and no more.
//
// Design. One launch does two kinds of jobs, whose states (peak, sum of weights, weighted sum of values) a second kernel joins:
//   * the prefix: the query heads of all sequences that share a key head are the rows of one product, so the prefix is read once for 64
//     NQ of them instead of once for each sequence. A workgroup's 4 waves take 16 NQ rows each and walk the same run of the prefix,
//     whose keys and values pass through the LDS 32 tokens at a time;
//   * a sequence's own tokens: a job is a run of its pages for one key head; the 4 waves take 32 tokens in turn, straight to registers.
// Scores are formed with 16 keys as rows and 16 query rows as columns (v_mfma_f32_16x16x32), which leaves the weights of keys 4 g .. 4 g
// + 3 in lane (r, g), where the second product wants them: columns of the values as rows, 32 keys (4 of each 16 a lane) summed over. A
// lane reads D / 16 columns of its eight keys and pairs them with v_perm. The peak is raised only when a score passes it by 2^4.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace intent_hip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kStep = 32;              // tokens of a step: two tiles of 16
constexpr float kSlack = 4.0f;
constexpr float kNoToken = -1.0f;      // the sum of a state without a token (weights are not negative)
constexpr int kSets = 4;               // LDS stages of a prefix job

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void_t;

struct Decode {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int32_t *prefix, *prefix_length, *offsets, *indices, *lengths;
  int64_t qs[2], ks[3], vs[3], outs[2];          // strides: sequence, head; page, token, head
  int64_t pages;
  int prefix_positions, positions, ps, shift;    // shift: log2 of ps, -1 where it is no power of two
  int batch, kv_heads, group;
  int row_tiles, parts, prefix_blocks;           // of the prefix: tiles of query rows, parts of its tokens
  int head_tiles, job_pages, jobs;               // of the sequences
  float scale;
  // States: of the prefix [parts][batch][q_heads] (and [D]), then of the jobs [jobs][q_heads] (and [D]).
  float *peak, *total, *sums;
};

#define INTENT_WAIT_VMCNT(n) __builtin_amdgcn_s_waitcnt((((n) & 0xF) | (((n) >> 4) << 14) | (0x7 << 4) | (0xF << 8)))

// s_barrier with an acquire fence alone: a release fence would wait for every load into the LDS that is on its way.
__device__ __forceinline__ void stage_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  __builtin_amdgcn_sched_barrier(0);
}

template <typename E>
__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same_v<E, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

constexpr int kParts = 2;              // numbers of a weight
// Weights are held at this power of two (times 2^kSlack they stay below the largest f16).
template <typename E>
constexpr float kRaise = std::is_same_v<E, f16_t> ? 11.0f : 0.0f;

// Two weights as kParts numbers each, and what these add up to. No part of a weight that counts is 0, so that an infinite value gives an
// infinity and not 0 times it: of f16 the first number is cut off below the weight, which leaves a second of 2^-10 of it at least (for
// weights from 2^-25 of the largest on); of bf16 a number of 0 becomes 2^-126.
template <typename E>
__device__ __forceinline__ void rounded(float &a, float &b, uint32_t (&part)[kParts]) {
  if constexpr (std::is_same_v<E, f16_t>) {
    constexpr float kBelow = 1.0f - 0x1p-10f;
    const f16x2_t high = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_cvt_pkrtz(a * kBelow, b * kBelow));
    const float high_a = static_cast<float>(high[0]), high_b = static_cast<float>(high[1]);
    const f16x2_t low = __builtin_convertvector(f32x2_t{a - high_a, b - high_b}, f16x2_t);
    part[0] = __builtin_bit_cast(uint32_t, high), part[1] = __builtin_bit_cast(uint32_t, low);
    a = high_a + static_cast<float>(low[0]), b = high_b + static_cast<float>(low[1]);
  } else {
    // The first 8 bits cut off, the rest rounded to 8.
    constexpr uint32_t kTiny = 0x00800080u;
    const auto raised = [=](uint32_t pair) {
      return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, pair), __builtin_bit_cast(u16x2_t, kTiny)));
    };
    const uint32_t u = __float_as_uint(a), v = __float_as_uint(b);
    const float high_a = __uint_as_float(u & 0xFFFF0000u), high_b = __uint_as_float(v & 0xFFFF0000u);
    const bf16x2_t low = __builtin_convertvector(f32x2_t{a - high_a, b - high_b}, bf16x2_t);
    part[0] = raised(__builtin_amdgcn_perm(v, u, 0x07060302)), part[1] = raised(__builtin_bit_cast(uint32_t, low));
    a = high_a + __uint_as_float(part[1] << 16), b = high_b + __uint_as_float(part[1] & 0xFFFF0000u);
  }
}

// The state of 16 query rows: lane (r, g) has the peak of row r, its own share of the sum of weights, and columns 4 C g .. of the
// weighted values, C = D / 16: product j gives column C (4 g + i) + j in sums[j][i].
template <int D>
struct State {
  static constexpr int C = D / 16;
  float peak, total;
  f32x4_t sums[C];
  __device__ __forceinline__ void clear() {
    peak = -INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) sums[j] = f32x4_t{0, 0, 0, 0};
  }
};

// Largest and sum over the four lanes of a query row.
__device__ __forceinline__ float largest_of_row(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_of_row(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// The weights of 32 keys for 16 query rows, from their scores: key 16 t + 4 g + i of the step in s[t][i]. `live` keys count.
template <typename E, int D>
__device__ __forceinline__ void weigh(State<D> &state, f32x4_t (&s)[2], float scale, int live, int g, uint4 (&weights)[kParts]) {
  float most = -INFINITY;
  float z[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[t][i] = s[t][i] * scale;
      if (live < kStep && t * 16 + g * 4 + i >= live) z[t][i] = -INFINITY;
      most = fmaxf(most, z[t][i]);
    }
  if (__builtin_amdgcn_ballot_w64(most > state.peak + kSlack)) {
    const float peak = fmaxf(state.peak, largest_of_row(most));
    const float down = peak == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(state.peak - peak);
    state.peak = peak;
    state.total *= down;
#pragma unroll
    for (int j = 0; j < State<D>::C; ++j) state.sums[j] *= down;
  }
  // A row all of whose scores are -inf so far has no peak; its weights are 0.
  const float base = state.peak == -INFINITY ? 0.0f : kRaise<E> - state.peak;
  uint32_t words[4][kParts];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      float a = __builtin_amdgcn_exp2f(z[t][i] + base), b = __builtin_amdgcn_exp2f(z[t][i + 1] + base);
      rounded<E>(a, b, words[t * 2 + i / 2]);
      state.total += a + b;
    }
#pragma unroll
  for (int n = 0; n < kParts; ++n) weights[n] = make_uint4(words[0][n], words[1][n], words[2][n], words[3][n]);
}

// Column j of a lane's eight keys, from the D / 16 columns of each.
template <int C>
__device__ __forceinline__ uint4 column(const uint32_t (&rows)[8][C / 2], int j) {
  const uint32_t pick = j & 1 ? 0x07060302u : 0x05040100u;
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_perm(rows[2 * i + 1][j / 2], rows[2 * i][j / 2], pick);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ int page_of(const Decode &p, int token) { return p.shift >= 0 ? token >> p.shift : token / p.ps; }

// The physical page of entry `at` of a table: entries outside the table and pages outside the cache read the nearest.
__device__ __forceinline__ int physical(const Decode &p, const int32_t *table, int entries, int at) {
  const int page = table[min(max(at, 0), entries - 1)];
  return static_cast<int>(min<int64_t>(max(page, 0), p.pages - 1));
}

// Writes the state of a query row (its four lanes together) to row `at` of the states.
template <int D>
__device__ __forceinline__ void keep(const Decode &p, const State<D> &state, int64_t at, int g, bool any) {
  constexpr int C = D / 16;
  const float total = sum_of_row(state.total);
  if (g == 0) p.peak[at] = state.peak, p.total[at] = any ? total : kNoToken;
  if (!any) return;
  float *to = p.sums + at * D + 4 * C * g;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < C; j += 4)
      *reinterpret_cast<float4 *>(to + C * i + j) = make_float4(state.sums[j][i], state.sums[j + 1][i], state.sums[j + 2][i], state.sums[j + 3][i]);
}

// ---------------------------------------------------------------- the prefix
// Unit (16 bytes) u of row `row` of a stage lies at u ^ place(row): the 16 rows of a read of keys are then in different banks.
template <int D>
__device__ __forceinline__ int place(int row) {
  return D == 128 ? row & 15 : (row >> 1) & 7;
}

// kTiles: pages hold whole tiles of 16 tokens, so a tile's page is the wave's to look up.
template <typename E, int D, int NQ, bool kTiles>
__device__ __forceinline__ void prefix_job(const Decode &p, int block, uint4 *set_0, uint4 *set_1, uint4 *set_2, uint4 *set_3) {
  constexpr int kRowUnits = D / 8, kUnits = kStep * kRowUnits, kLoads = kUnits / kThreads, kChunks = D / 32, C = D / 16;
  constexpr int kIssued = 2 * kLoads;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Blocks of one part and key head follow each other: their rows' tiles read the same run.
  const int tile = block % p.row_tiles, kh = block / p.row_tiles % p.kv_heads, part = block / p.row_tiles / p.kv_heads;
  const int rows = p.batch * p.group, q_heads = p.kv_heads * p.group;
  const int64_t held = p.pages > 0 ? static_cast<int64_t>(p.prefix_positions) * p.ps : 0;
  const int tokens = static_cast<int>(min<int64_t>(max(p.prefix_length[0], 0), held));
  const int steps = (tokens + kStep - 1) / kStep, of_part = (steps + p.parts - 1) / p.parts;
  const int first = part * of_part * kStep, last = min(tokens, first + of_part * kStep);
  const int row0 = (tile * kWaves + wave) * 16 * NQ;
  State<D> state[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) state[n].clear();
  if (first < last) {
    const int count = (last - first + kStep - 1) / kStep;
    uint4 q[NQ][kChunks];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int row = min(row0 + n * 16 + r, rows - 1), b = row / p.group, h = kh * p.group + row % p.group;
      const uint16_t *from = p.q + b * p.qs[0] + h * p.qs[1];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) q[n][c] = *reinterpret_cast<const uint4 *>(from + (c * 4 + g) * 8);
    }
    const float scale = p.scale * kLog2e;
    const auto set_of = [&](int u) -> uint4 * { return u == 0 ? set_0 : u == 1 ? set_1 : u == 2 ? set_2 : set_3; };
    const auto issue = [&](int t, int set) {           // step t (the last again behind it)
      uint4 *stage = set_of(set);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int slot = (i * kWaves + wave) * kWave + lane, row = slot / kRowUnits;
        const int at = first + min(t, count - 1) * kStep;
        const int token = min(at + row, last - 1);
        int page, in;
        if constexpr (kTiles) {                        // rows of one tile of 16: this wave's
          const int base = min(at + __builtin_amdgcn_readfirstlane(row) / 16 * 16, last - 1) & ~15, entry = page_of(p, base);
          page = physical(p, p.prefix, p.prefix_positions, entry);
          in = token - entry * p.ps;
        } else {
          const int entry = page_of(p, token);
          page = physical(p, p.prefix, p.prefix_positions, entry);
          in = token - entry * p.ps;
        }
        const int unit = slot % kRowUnits ^ place<D>(row);
        const uint16_t *k = p.k + page * p.ks[0] + in * p.ks[1] + kh * p.ks[2] + unit * 8;
        const uint16_t *v = p.v + page * p.vs[0] + in * p.vs[1] + kh * p.vs[2] + unit * 8;
        __builtin_amdgcn_global_load_lds(k, (lds_void_t *)(stage + (i * kWaves + wave) * kWave), 16, 0, 0);
        __builtin_amdgcn_global_load_lds(v, (lds_void_t *)(stage + kUnits + (i * kWaves + wave) * kWave), 16, 0, 0);
      }
    };
#pragma unroll
    for (int u = 0; u < kSets - 1; ++u) issue(u, u);
    for (int t0 = 0; t0 < count; t0 += kSets) {
#pragma unroll
      for (int u = 0; u < kSets; ++u) {
        if (t0 + u >= count) break;
        INTENT_WAIT_VMCNT((kSets - 2) * kIssued);      // this wave's loads of the step have come
        stage_barrier();                               // everybody's have, and nobody reads the set that is filled next
        issue(t0 + u + kSets - 1, (u + kSets - 1) % kSets);
        const uint4 *keys = set_of(u), *values = keys + kUnits;
        f32x4_t s[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const uint4 key = keys[(t * 16 + r) * kRowUnits + ((c * 4 + g) ^ place<D>(t * 16 + r))];
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[n][t] = mfma<E>(key, q[n][c], s[n][t]);
          }
        }
        uint4 weights[NQ][kParts];
        const int live = last - first - (t0 + u) * kStep;
#pragma unroll
        for (int n = 0; n < NQ; ++n) weigh<E, D>(state[n], s[n], scale, live, g, weights[n]);
        uint32_t own[8][C / 2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i / 4 * 16 + g * 4 + i % 4;
          if constexpr (D == 128) {
            const uint4 v = values[row * kRowUnits + (r ^ place<D>(row))];
            own[i][0] = v.x, own[i][1] = v.y, own[i][2] = v.z, own[i][3] = v.w;
          } else {
            const uint2 v = reinterpret_cast<const uint2 *>(values + row * kRowUnits + ((r >> 1) ^ place<D>(row)))[r & 1];
            own[i][0] = v.x, own[i][1] = v.y;
          }
        }
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const uint4 v = column<C>(own, j);
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int k = 0; k < kParts; ++k) state[n].sums[j] = mfma<E>(v, weights[n][k], state[n].sums[j]);
        }
      }
    }
    INTENT_WAIT_VMCNT(0);                              // nothing is on its way into the LDS of an ended workgroup
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int row = row0 + n * 16 + r;
    if (row0 + n * 16 >= rows) break;
    const int b = min(row, rows - 1) / p.group, h = kh * p.group + min(row, rows - 1) % p.group;
    // Lanes behind the last row hold its state too and write the same.
    keep<D>(p, state[n], (static_cast<int64_t>(part) * p.batch + b) * q_heads + h, g, first < last);
  }
}

// ---------------------------------------------------------------- a sequence's own tokens
// A sequence: its first entry of the page indices, and its tokens: what its length and its pages both have.
struct Sequence {
  int s, first, tokens;
};

__device__ __forceinline__ int held_tokens(const Decode &p, int first, int next, int length) {
  const int64_t held = static_cast<int64_t>(max(0, min(next, p.positions) - max(first, 0))) * p.ps;
  return p.pages <= 0 || length < 0 ? 0 : static_cast<int>(min<int64_t>(length, held));
}

// The sequence of job `job` (the wave's): the last whose jobs, from offsets[s] / job_pages + s on, begin at or before it. Found by all
// lanes of the wave, 64 candidates at a time.
__device__ __forceinline__ Sequence job_sequence(const Decode &p, int job) {
  const int lane = threadIdx.x & 63;
  int first = 0, count = p.batch - 1;                  // it is one of first .. first + count
  while (count >= kWave) {
    const int step = (count + 63) / 64, at = (lane + 1) * step;
    const bool past = at <= count && static_cast<int64_t>(p.offsets[first + at] / p.job_pages) + first + at <= job;
    const int steps = __popcll(__ballot(past));
    first += steps * step;
    count = min(step - 1, count - steps * step);
  }
  const bool in = lane <= count;
  const int s = first + (in ? lane : 0), begin = p.offsets[s], next = p.offsets[s + 1], length = p.lengths[s];
  const bool past = lane > 0 && in && static_cast<int64_t>(begin / p.job_pages) + s <= job;
  const int at = __popcll(__ballot(past));
  const int from = __builtin_amdgcn_readlane(begin, at);
  return Sequence{first + at, from, held_tokens(p, from, __builtin_amdgcn_readlane(next, at), __builtin_amdgcn_readlane(length, at))};
}

template <typename E, int D, bool kTiles>
__device__ __forceinline__ void own_job(const Decode &p, int block, float *sums, float *peaks) {
  constexpr int kChunks = D / 32, C = D / 16;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = block % p.head_tiles, kh = block / p.head_tiles % p.kv_heads, job = block / p.head_tiles / p.kv_heads;
  const int q_heads = p.kv_heads * p.group;
  const Sequence sequence = job_sequence(p, job);
  const int64_t turn = job - (static_cast<int64_t>(sequence.first / p.job_pages) + sequence.s);
  const int64_t from = turn * p.job_pages * p.ps;
  const int first = static_cast<int>(min<int64_t>(max<int64_t>(from, 0), sequence.tokens));
  const int last = static_cast<int>(min<int64_t>(sequence.tokens, first + static_cast<int64_t>(p.job_pages) * p.ps));
  const int head = min(tile * 16 + r, p.group - 1);
  const int64_t at = static_cast<int64_t>(p.parts) * p.batch * q_heads + static_cast<int64_t>(job) * q_heads + kh * p.group + head;
  if (first >= last) {                                 // of the whole workgroup
    if (wave == 0 && g == 0) p.total[at] = kNoToken;
    return;
  }
  State<D> state;
  state.clear();
  uint4 q[kChunks];
  {
    const uint16_t *row = p.q + sequence.s * p.qs[0] + (kh * p.group + head) * p.qs[1];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) q[c] = *reinterpret_cast<const uint4 *>(row + (c * 4 + g) * 8);
  }
  const float scale = p.scale * kLog2e;
  struct Tokens {
    uint4 keys[2][kChunks];
    uint32_t values[8][C / 2];
  };
  // Offsets of a token's row in the caches.
  const auto load = [&](int t, Tokens &to) {           // step t of the wave
    const int base = first + t * kStep;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      int whole_page = 0, whole_entry = 0;
      if constexpr (kTiles) {
        whole_entry = page_of(p, min(base + half * 16, last - 1) & ~15);
        whole_page = physical(p, p.indices, p.positions, sequence.first + whole_entry);
      }
      const auto find = [&](int token, int &page, int &in) {
        token = min(token, last - 1);
        if constexpr (kTiles) {
          page = whole_page, in = token - whole_entry * p.ps;
        } else {
          const int entry = page_of(p, token);
          page = physical(p, p.indices, p.positions, sequence.first + entry), in = token - entry * p.ps;
        }
      };
      int page, in;
      find(base + half * 16 + r, page, in);
      const uint16_t *key = p.k + page * p.ks[0] + in * p.ks[1] + kh * p.ks[2];
#pragma unroll
      for (int c = 0; c < kChunks; ++c) to.keys[half][c] = *reinterpret_cast<const uint4 *>(key + (c * 4 + g) * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        find(base + half * 16 + g * 4 + i, page, in);
        const uint16_t *value = p.v + page * p.vs[0] + in * p.vs[1] + kh * p.vs[2] + r * C;
        uint32_t(&row)[C / 2] = to.values[half * 4 + i];
        if constexpr (D == 128) {
          const uint4 v = *reinterpret_cast<const uint4 *>(value);
          row[0] = v.x, row[1] = v.y, row[2] = v.z, row[3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2 *>(value);
          row[0] = v.x, row[1] = v.y;
        }
      }
    }
  };
  const int count = (last - first + kStep - 1) / kStep;
  Tokens next;
  if (wave < count) load(wave, next);
  for (int t = wave; t < count; t += kWaves) {
    const Tokens now = next;
    if (t + kWaves < count) load(t + kWaves, next);
    f32x4_t s[2] = {f32x4_t{0, 0, 0, 0}, f32x4_t{0, 0, 0, 0}};
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) s[half] = mfma<E>(now.keys[half][c], q[c], s[half]);
    uint4 weights[kParts];
    weigh<E, D>(state, s, scale, last - first - t * kStep, g, weights);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const uint4 v = column<C>(now.values, j);
#pragma unroll
      for (int k = 0; k < kParts; ++k) state.sums[j] = mfma<E>(v, weights[k], state.sums[j]);
    }
  }
  // The waves' states, through the LDS: peaks and sums of weights, then the weighted values at the common peak, half of each lane's
  // columns at a time.
  const float total = sum_of_row(state.total);
  if (g == 0) peaks[wave * 16 + r] = state.peak;
  __syncthreads();
  float peak = -INFINITY;
  for (int i = 0; i < min(kWaves, count); ++i) peak = fmaxf(peak, peaks[i * 16 + r]);
  const float share = wave >= count ? 0.0f : peak == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(state.peak - peak);
  if (g == 0) peaks[(kWaves + wave) * 16 + r] = wave < count ? total * share : 0.0f;
  // Wave w joins rows 4 w .. 4 w + 3, a lane the D / 16 columns of one from r D / 16 on.
  const int row = wave * 4 + g, of_group = tile * 16 + row;
  float joined[C];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < C / 2; ++j)
        sums[((wave * 16 + r) * 16 + 4 * g + i) * (C / 2) + j] = wave < count ? state.sums[h * (C / 2) + j][i] * share : 0.0f;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
      float of_all = 0.0f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) of_all += sums[((i * 16 + row) * 16 + r) * (C / 2) + j];
      joined[h * (C / 2) + j] = of_all;
    }
  }
  if (of_group >= p.group) return;
  const int64_t to = static_cast<int64_t>(p.parts) * p.batch * q_heads + static_cast<int64_t>(job) * q_heads + kh * p.group + of_group;
  float weight = 0.0f, most = -INFINITY;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    weight += peaks[(kWaves + i) * 16 + row];
    if (i < count) most = fmaxf(most, peaks[i * 16 + row]);
  }
  if (r == 0) p.peak[to] = most, p.total[to] = weight;
#pragma unroll
  for (int j = 0; j < C; j += 4)
    *reinterpret_cast<float4 *>(p.sums + to * D + r * C + j) = make_float4(joined[j], joined[j + 1], joined[j + 2], joined[j + 3]);
}

template <typename E, int D, int NQ, bool kTiles>
__global__ __launch_bounds__(kThreads, 2) void prefix_decode_jobs(Decode p) {
  constexpr int kStage = 2 * kStep * D / 8;           // keys and values of a step; each has an array of its own, so that the compiler
  __shared__ uint4 set_0[kStage], set_1[kStage], set_2[kStage], set_3[kStage];      // knows which loads a read has to wait for
  static_assert(kSets == 4 && kStage * sizeof(uint4) >= kWaves * 16 * (D / 2) * sizeof(float), "the waves' states fit a set");
  const int block = grid_block();
  if (block < p.prefix_blocks)
    prefix_job<E, D, NQ, kTiles>(p, block, set_0, set_1, set_2, set_3);
  else if (block - p.prefix_blocks < p.jobs * p.kv_heads * p.head_tiles)
    own_job<E, D, kTiles>(p, block - p.prefix_blocks, reinterpret_cast<float *>(set_0), reinterpret_cast<float *>(set_1));
}

// The states of a query head's parts of the prefix and of its sequence's jobs, joined: a wave per head.
template <typename E, int D>
__global__ __launch_bounds__(kThreads) void prefix_decode_join(Decode p) {
  constexpr int kOwn = D / kWave;
  const int lane = threadIdx.x & 63, q_heads = p.kv_heads * p.group;
  const int64_t row = static_cast<int64_t>(grid_block()) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(p.batch) * q_heads) return;
  const int b = static_cast<int>(row / q_heads), h = static_cast<int>(row % q_heads);
  const int begin = p.offsets[b], next = p.offsets[b + 1];
  const int tokens = held_tokens(p, begin, next, p.lengths[b]);
  const int64_t own = static_cast<int64_t>(begin / p.job_pages) + b, of_job = static_cast<int64_t>(p.job_pages) * p.ps;
  const int jobs = tokens > 0 && own >= 0 && own < p.jobs ? static_cast<int>(min<int64_t>((tokens + of_job - 1) / of_job, p.jobs - own)) : 0;
  const int64_t of_prefix = static_cast<int64_t>(p.batch) * q_heads;
  // State i of this head: the parts of the prefix, then its jobs.
  const auto state = [&](int i) -> int64_t {
    return i < p.parts ? i * of_prefix + row : p.parts * of_prefix + (own + i - p.parts) * q_heads + h;
  };
  const int count = p.parts + jobs;
  float peak = -INFINITY;
  for (int i = lane; i < count; i += kWave)
    if (p.total[state(i)] >= 0.0f || p.total[state(i)] != p.total[state(i)]) peak = fmaxf(peak, p.peak[state(i)]);
  peak = wave_max(peak);
  float total = 0.0f, sums[kOwn] = {};
  bool any = false;
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const int64_t at = state(i);
    const float held = p.total[at];
    if (held == kNoToken) continue;
    any = true;
    const float share = peak == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(p.peak[at] - peak);
    total += held * share;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) sums[j] += p.sums[at * D + lane * kOwn + j] * share;
  }
  uint16_t *out = p.out + b * p.outs[0] + h * p.outs[1] + lane * kOwn;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) out[j] = from_f32<E>(any ? sums[j] / total : 0.0f).bits;
}

// How a call is cut.
struct Cut {
  int nq, row_tiles, parts, head_tiles, job_pages, jobs;
};

Cut cut(int64_t batch, int64_t kv_heads, int64_t group, int64_t ps, int64_t prefix_positions, int64_t positions) {
  Cut c{};
  const int64_t rows = batch * group, cus = device_cus();
  c.nq = rows <= 64 ? 1 : 2;
  c.row_tiles = static_cast<int>((rows + kWaves * 16 * c.nq - 1) / (kWaves * 16 * c.nq));
  const int64_t tokens = prefix_positions * ps, tiles = std::max<int64_t>(c.row_tiles * kv_heads, 1);
  const int64_t most = (tokens + 127) / 128;           // a part walks four steps at least
  c.parts = static_cast<int>(tokens == 0 ? 0 : std::max<int64_t>(1, std::min<int64_t>(most, 2 * cus / tiles)));
  c.head_tiles = static_cast<int>((group + 15) / 16);
  // Jobs of about 256 tokens, longer where there are many.
  const int64_t own = positions * ps, aim = 4 * cus / std::max<int64_t>(kv_heads * c.head_tiles, 1);
  const int64_t of_job = std::max<int64_t>(256, (own + std::max<int64_t>(aim, 1) - 1) / std::max<int64_t>(aim, 1));
  c.job_pages = ps > 0 ? static_cast<int>(std::max<int64_t>(1, (of_job + ps - 1) / ps)) : 1;
  c.jobs = static_cast<int>(positions / c.job_pages + batch);
  return c;
}

size_t states_of(const Cut &c, int64_t batch, int64_t q_heads) { return (static_cast<size_t>(c.parts) * batch + c.jobs) * q_heads; }

template <typename E, typename F>
int with_kernel(int64_t d, int nq, bool tiles, F f) {
  const auto of = [&](auto width, auto rows) {
    return tiles ? f(prefix_decode_jobs<E, width.value, rows.value, true>, prefix_decode_join<E, width.value>)
                 : f(prefix_decode_jobs<E, width.value, rows.value, false>, prefix_decode_join<E, width.value>);
  };
  const std::integral_constant<int, 64> narrow;
  const std::integral_constant<int, 128> wide;
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, 2> two;
  if (d == 64) return nq == 1 ? of(narrow, one) : of(narrow, two);
  return nq == 1 ? of(wide, one) : of(wide, two);
}

int check(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t group, int64_t d, int64_t pages, int64_t ps, int64_t prefix_positions,
          int64_t positions) {
  if (batch < 0 || q_heads < 0 || kv_heads < 0 || d < 0 || pages < 0 || ps < 0 || prefix_positions < 0 || positions < 0)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (group < 1 || q_heads != kv_heads * group)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "query heads (%lld) must equal key/value heads (%lld) * HEAD_GROUP (%lld)",
                static_cast<long long>(q_heads), static_cast<long long>(kv_heads), static_cast<long long>(group));
  if (d != 64 && d != 128)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "paged_gqa_decode_prefix takes heads of 64 or 128 dimensions, got %lld", static_cast<long long>(d));
  // Tokens of a table and rows of queries are counted in 32 bits, and so are blocks.
  if (batch > (1 << 20) || q_heads > (1 << 16) || pages > INT32_MAX || ps > (1 << 20) || prefix_positions > (1 << 28) || positions > (1 << 28) ||
      prefix_positions * ps > INT32_MAX - 64 || positions * ps > (int64_t{1} << 40) || batch * q_heads > (1 << 28))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}

}  // namespace

int prefix_decode_resources(int dtype, int64_t batch, int64_t kv_heads, int64_t group, int64_t d, int64_t ps, int64_t prefix_positions,
                            int64_t positions, IntentHipKernelResources *out) {
  if (int rc = check(batch, kv_heads * group, kv_heads, group, d, 1, ps, prefix_positions, positions)) return rc;
  const Cut c = cut(batch, kv_heads, group, ps, prefix_positions, positions);
  const bool tiles = ps % 16 == 0;
  char name[64];
  snprintf(name, sizeof(name), "prefix_decode_jobs<%s,%lld,%d,%s>", dtype == INTENT_HIP_F16 ? "f16" : "bf16", static_cast<long long>(d), c.nq,
           tiles ? "true" : "false");
  const auto describe = [&](void (*kernel)(Decode), void (*)(Decode)) {
    return describe_kernel(reinterpret_cast<const void *>(kernel), name, kThreads, out);
  };
  return dtype == INTENT_HIP_F16 ? with_kernel<f16_t>(d, c.nq, tiles, describe) : with_kernel<bf16_t>(d, c.nq, tiles, describe);
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_paged_gqa_decode_prefix_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_group,
                                                                  int64_t d, int64_t ps, int64_t prefix_positions, int64_t positions,
                                                                  size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (int rc = check(batch, q_heads, kv_heads, head_group, d, 0, ps, prefix_positions, positions)) return rc;
  if (batch == 0 || q_heads == 0) return INTENT_HIP_OK;
  *bytes = states_of(cut(batch, kv_heads, head_group, ps, prefix_positions, positions), batch, q_heads) * (d + 2) * sizeof(float);
  return INTENT_HIP_OK;
}

extern "C" int intent_hip_paged_gqa_decode_prefix(int dtype, const void *q, const void *key_cache, const void *value_cache,
                                                  const int32_t *prefix_indices, const int32_t *prefix_length, const int32_t *page_offsets,
                                                  const int32_t *page_indices, const int32_t *lengths, void *output, int64_t batch,
                                                  int64_t q_heads, int64_t kv_heads, int64_t head_group, int64_t d, int64_t pages, int64_t ps,
                                                  int64_t prefix_positions, int64_t positions, const int64_t *strides, float scale,
                                                  void *workspace, size_t workspace_bytes, void *stream) {
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "paged_gqa_decode_prefix dtype must be F16 or BF16, got %d", dtype);
  if (int rc = check(batch, q_heads, kv_heads, head_group, d, pages, ps, prefix_positions, positions)) return rc;
  if (batch == 0 || q_heads == 0) return INTENT_HIP_OK;
  const bool shared = prefix_positions > 0, own = positions > 0, any = pages > 0 && ps > 0 && (shared || own);
  if (strides == nullptr || q == nullptr || output == nullptr || prefix_length == nullptr || page_offsets == nullptr || lengths == nullptr ||
      (any && (key_cache == nullptr || value_cache == nullptr)) || (shared && prefix_indices == nullptr) || (own && page_indices == nullptr))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  // strides: q[3], key_cache[4], value_cache[4], output[3]
  for (int i = 0; i < 14; ++i)
    if (strides[i] < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (strides[2] != 1 || (any && (strides[6] != 1 || strides[10] != 1)) || strides[13] != 1)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows need unit inner stride");
  uint64_t mixed = reinterpret_cast<uintptr_t>(q);
  if (batch > 1) mixed |= 2 * static_cast<uint64_t>(strides[0]);
  if (q_heads > 1) mixed |= 2 * static_cast<uint64_t>(strides[1]);
  if (any) {
    mixed |= reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache);
    for (int i = 0; i < 2; ++i) {
      if (pages > 1) mixed |= 2 * static_cast<uint64_t>(strides[3 + 4 * i]);
      if (ps > 1) mixed |= 2 * static_cast<uint64_t>(strides[4 + 4 * i]);
      if (kv_heads > 1) mixed |= 2 * static_cast<uint64_t>(strides[5 + 4 * i]);
    }
  }
  if (mixed % 16) return fail(INTENT_HIP_ERR_UNSUPPORTED, "rows of q and of the caches must be 16-byte aligned, their strides multiples of 8");
  const Cut c = cut(batch, kv_heads, head_group, ps, prefix_positions, positions);
  const size_t states = states_of(c, batch, q_heads), bytes = states * (d + 2) * sizeof(float);
  if (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16))
    return fail(INTENT_HIP_ERR_WORKSPACE, "paged_gqa_decode_prefix needs %zu workspace bytes, 16-byte aligned", bytes);
  Decode p{};
  p.q = static_cast<const uint16_t *>(q), p.k = static_cast<const uint16_t *>(key_cache), p.v = static_cast<const uint16_t *>(value_cache);
  p.out = static_cast<uint16_t *>(output);
  p.prefix = prefix_indices, p.prefix_length = prefix_length, p.offsets = page_offsets, p.indices = page_indices, p.lengths = lengths;
  p.qs[0] = strides[0], p.qs[1] = strides[1], p.outs[0] = strides[11], p.outs[1] = strides[12];
  for (int i = 0; i < 3; ++i) p.ks[i] = strides[3 + i], p.vs[i] = strides[7 + i];
  p.pages = ps > 0 ? pages : 0, p.ps = static_cast<int>(ps), p.shift = -1;
  for (int i = 0; i < 21; ++i)
    if (ps == int64_t{1} << i) p.shift = i;
  p.prefix_positions = static_cast<int>(prefix_positions), p.positions = static_cast<int>(positions);
  p.batch = static_cast<int>(batch), p.kv_heads = static_cast<int>(kv_heads), p.group = static_cast<int>(head_group);
  p.row_tiles = c.row_tiles, p.parts = c.parts, p.prefix_blocks = static_cast<int>(c.row_tiles * kv_heads * c.parts);
  p.head_tiles = c.head_tiles, p.job_pages = c.job_pages, p.jobs = c.jobs, p.scale = scale;
  p.sums = static_cast<float *>(workspace), p.peak = p.sums + states * d, p.total = p.peak + states;
  const int64_t blocks = p.prefix_blocks + static_cast<int64_t>(c.jobs) * kv_heads * c.head_tiles;
  const auto run = [&](void (*jobs)(Decode), void (*join)(Decode)) {
    jobs<<<tile_grid(blocks, 1), kThreads, 0, as_stream(stream)>>>(p);
    join<<<tile_grid((batch * q_heads + kWaves - 1) / kWaves, 1), kThreads, 0, as_stream(stream)>>>(p);
    return 0;
  };
  if (dtype == INTENT_HIP_F16)
    with_kernel<f16_t>(d, c.nq, ps % 16 == 0, run);
  else
    with_kernel<bf16_t>(d, c.nq, ps % 16 == 0, run);
  return hipPeekAtLastError() != hipSuccess ? launch_status("paged_gqa_decode_prefix") : INTENT_HIP_OK;
}

// Attention of one new token per sequence over a prefix that all sequences share and over the pages of each, for gfx950. No reference
// counterpart; the cache is the paged one of 16-bit rows that paged_gqa_decode_partials reads.
//
// For query head h of sequence s, over the prefix's tokens and the sequence's own:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp2(scale * log2(e) * (q . k_j) - peak)        0 where there is no token
// Products are summed in f32. Weights are f32 and enter the second product whole, as three numbers of the queries' type each, but for what
// 2^-36 of the largest in f16.
//
// Design. One launch does two kinds of jobs, whose states (peak, sum of weights, weighted sum of values) a second kernel joins:
//   * the prefix: the query heads of all sequences that share a key head are the rows of one product, so the prefix is read once for 64
//     NQ of them instead of once for each sequence. A workgroup's 4 waves take 16 NQ rows each and walk the same run of the prefix,
//     whose keys and values pass through the LDS 32 tokens at a time;
//   * a sequence's own tokens: a job is a run of its pages for one key head; the 4 waves take 32 tokens in turn, straight to registers.
// Scores are formed with 16 keys as rows and 16 query rows as columns (v_mfma_f32_16x16x32), which leaves the weights of keys 4 g .. 4 g
// + 3 in lane (r, g), where the second product wants them: columns of the values as rows, 32 keys (4 of each 16 a lane) summed over. The
// LDS gives those columns turned (ds_read_b64_tr_b16); from memory a lane reads D / 16 columns of its eight keys and pairs them with
// v_perm. The peak is raised only when a score passes it by 2^4.
// Measured: 64 sequences behind 16384 tokens, up to 1000 of their own, 64 heads on 8, bf16, 111 us (matrix pipe 32% busy, vector pipe 33%: two
// or three waves a SIMD, each of whose steps waits for its own LDS reads, products and weights in turn); the prefix alone 94, the own tokens
// alone 47 (2.8 TB/s), the join 12 of each; own jobs between those of the prefix instead of behind them 130, before weights were whole. 8
// sequences behind 8191 tokens, up to 512, 32 heads on 8, f16, 19.6 us, of which the join is 5. Weights of two numbers, 16 bits in bf16: 101 and 18.8.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "stages.hpp"

namespace intent_hip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4, kThreads = kWaves * kWave;
constexpr int kStep = 32;              // tokens of a step: two tiles of 16
constexpr float kSlack = 4.0f;
constexpr float kNoToken = -1.0f;      // the sum of a state without a token (weights are not negative)
constexpr int kSets = 3;               // LDS stages of a prefix job

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

struct Decode {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  const int32_t *prefix, *prefix_length, *offsets, *indices, *lengths;
  int64_t qs[2], ks[3], vs[3], outs[2];          // strides: sequence, head; page, token, head
  int64_t pages;
  int prefix_positions, positions, ps;
  uint32_t magic, shift;                         // a token's place over ps: (high half of magic times it, plus it) >> shift
  uint32_t of_page[2], of_token[2];              // bytes, of keys and of values, where they and a page stay below 2^32 (kTile)
  int batch, kv_heads, group;
  int row_tiles, parts, prefix_blocks;           // of the prefix: tiles of query rows, parts of its tokens
  int head_tiles, job_pages, jobs;               // of the sequences
  float scale;
  // States: of the prefix [parts][batch][q_heads] (and [D]), then of the jobs [jobs][q_heads] (and [D]).
  float *peak, *total, *sums;
};

template <typename E>
__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same_v<E, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

constexpr int kParts = 3;              // numbers of a weight
// The largest weight is held at this power of two, and 2^kSlack times that before the peak is raised: just below the largest f16.
template <typename E>
constexpr float kRaise = std::is_same_v<E, f16_t> ? 11.9375f : 0.0f;

// Two weights as kParts numbers each, every one what those before it leave, cut off: three of bf16 hold all 24 bits of a weight, and so do
// three of f16 down to f16's last, 2^-24, which is about 2^-36 of the largest weight. No number of a weight that counts is 0, so that an
// infinite value gives an infinity and not 0 times it: the second and third are the least of their type at least (2^-126 in bf16). In f16,
// whose least is 2^-24, only where the first has all its bits (2^-13, 2^-25 of the largest): smaller weights would move by more than the cut.
template <typename E>
__device__ __forceinline__ void rounded(float a, float b, uint32_t (&part)[kParts]) {
  constexpr bool kHalf = std::is_same_v<E, f16_t>;
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    if constexpr (kHalf) {
      const f16x2_t h = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_cvt_pkrtz(a, b));
      part[i] = __builtin_bit_cast(uint32_t, h);
      a = fmaf(static_cast<float>(h[0]), -1.0f, a), b = fmaf(static_cast<float>(h[1]), -1.0f, b);
    } else {
      const uint32_t u = __float_as_uint(a), v = __float_as_uint(b);
      part[i] = __builtin_amdgcn_perm(v, u, 0x07060302);
      a -= __uint_as_float(u & 0xFFFF0000u), b -= __uint_as_float(v & 0xFFFF0000u);
    }
  }
  const u16x2_t first = __builtin_bit_cast(u16x2_t, part[0]);
  const u16x2_t least = kHalf ? __builtin_elementwise_min(first >> u16x2_t{11, 11}, u16x2_t{1, 1})
                              : __builtin_elementwise_min(first, u16x2_t{0x0080, 0x0080});
#pragma unroll
  for (int i = 1; i < kParts; ++i)
    part[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, part[i]), least));
}

// The state of 16 query rows, weights being exp2(score + base): lane (r, g) has row r's base (+inf before any score has counted), the sum
// of the weights that it formed (a quarter of the row's), and in sums[j][i] the weighted values of row 4 g + i of product j, C = D / 16
// products: column 16 j + 4 g + i of the prefix's, whose values come through the LDS, column C (4 g + i) + j of a sequence's own.
template <int D>
struct State {
  static constexpr int C = D / 16;
  float base, total;
  f32x4_t sums[C];
  __device__ __forceinline__ void clear() {
    base = INFINITY, total = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) sums[j] = f32x4_t{0, 0, 0, 0};
  }
};

// Largest over the four lanes of a query row.
__device__ __forceinline__ float largest_of_row(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ float sum_of_row(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

__device__ __forceinline__ float largest(float a, float b, float c) {
  float v;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(v) : "v"(a), "v"(b), "v"(c));       // (fmaxf first makes each of its operands quiet)
  return v;
}

// The weights of 32 keys for 16 query rows, from their scores: key 16 t + 4 g + i of the step in s[n][t][i], for NQ tiles of rows. First
// the powers z of two that they are, of the keys of which `live` count: the base is looked at once for all tiles.
template <typename E, int D, int NQ>
__device__ __forceinline__ void powers(State<D> (&state)[NQ], const f32x4_t (&s)[NQ][2], float scale, int live, int g, float (&z)[NQ][8]) {
  bool low = true;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[n][i] = fmaf(s[n][i / 4][i % 4], scale, state[n].base);
    const float half = largest(z[n][0], z[n][1], z[n][2]), rest = largest(z[n][3], z[n][4], z[n][5]);
    low = low && largest(half, rest, largest(z[n][6], z[n][7], z[n][7])) <= kRaise<E> + kSlack;
  }
  // Also where no score of a lane is a number (a row without a base whose scores are -inf), and where not all keys count.
  if (live >= kStep && !__builtin_amdgcn_ballot_w64(!low)) return;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float largest = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      z[n][i] = i / 4 * 16 + g * 4 + i % 4 >= live ? -INFINITY : s[n][i / 4][i % 4] * scale;
      largest = fmaxf(largest, z[n][i]);
    }
    const float base = fminf(state[n].base, kRaise<E> - largest_of_row(largest));      // +inf while every score is -inf
    const float down = base == INFINITY ? 1.0f : __builtin_amdgcn_exp2f(base - state[n].base);
    state[n].base = base;
    state[n].total *= down;
#pragma unroll
    for (int j = 0; j < State<D>::C; ++j) state[n].sums[j] *= down;
#pragma unroll
    for (int i = 0; i < 8; ++i) z[n][i] += base == INFINITY ? 0.0f : base;
  }
}

// The weights as the second product takes them; their sum is added to `total`.
template <typename E>
__device__ __forceinline__ void weigh(const float (&z)[8], uint4 (&weights)[kParts], float &total) {
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_exp2f(z[i]);
  total += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  uint32_t words[4][kParts];
#pragma unroll
  for (int i = 0; i < 4; ++i) rounded<E>(w[2 * i], w[2 * i + 1], words[i]);
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

// token / ps of tokens below 2^31.
__device__ __forceinline__ int page_of(const Decode &p, int token) {
  return static_cast<int>((__umulhi(p.magic, static_cast<uint32_t>(token)) + static_cast<uint32_t>(token)) >> p.shift);
}

// The physical page of entry `at` of a table: entries outside the table and pages outside the cache read the nearest.
__device__ __forceinline__ int physical(const Decode &p, const int32_t *table, int entries, int at) {
  const int page = table[min(max(at, 0), entries - 1)];
  return static_cast<int>(min<int64_t>(max(page, 0), p.pages - 1));
}

// The page of an entry that is the wave's (clamped to `entries`, if any), as the table has it, through the scalar cache: a vector load here
// would be waited for together with every load of keys and values before it.
typedef const __attribute__((address_space(4))) int32_t *table_t;
__device__ __forceinline__ int page_of_wave(const int32_t *table, int entries, int at) {
  return ((table_t)(table))[entries > 0 ? min(max(at, 0), entries - 1) : at];
}

// T tokens of one page, the wave's: the page as the table has it, the first one's place in it, and the last that counts.
template <int T>
struct WaveTile {
  int page, in, most;
  // `entries`: of the table; 0 where the entry is known to be one of its.
  __device__ __forceinline__ void find(const Decode &p, const int32_t *table, int entries, int begin, uint32_t token, int last) {
    const int base = static_cast<int>(min(token, static_cast<uint32_t>(last - 1))) & ~(T - 1), entry = page_of(p, base);
    page = page_of_wave(table, entries, begin + entry);
    in = base - entry * p.ps, most = last - 1 - base;
    if (token >= static_cast<uint32_t>(last)) in += most, most = 0;           // a tile behind the last token reads that one alone
  }
  // Its first row, of keys (0) or of values (1).
  __device__ __forceinline__ const uint16_t *rows(const Decode &p, const uint16_t *cache, int which) const {
    const uint32_t at = static_cast<uint32_t>(min(max(page, 0), static_cast<int>(p.pages) - 1));
    return reinterpret_cast<const uint16_t *>(reinterpret_cast<const char *>(cache) + static_cast<uint64_t>(at) * p.of_page[which] +
                                              static_cast<uint32_t>(in) * p.of_token[which]);
  }
};

// ---------------------------------------------------------------- the prefix
// Unit (16 bytes) u of row `row` of a stage lies at u ^ place(row): the 16 rows of a read of keys are then in different banks.
template <int D>
__device__ __forceinline__ int place(int row) {
  return D == 128 ? row & 15 : (row >> 1) & 7;
}

// Writes the state of a query row of the prefix (its four lanes together) to row `at` of the states.
template <int D>
__device__ __forceinline__ void keep(const Decode &p, const State<D> &state, int64_t at, int g, bool any) {
  constexpr int C = D / 16;
  const float total = sum_of_row(state.total);
  if (g == 0) p.peak[at] = -state.base, p.total[at] = any ? total : kNoToken;
  if (!any) return;
  float *to = p.sums + at * D + 4 * g;
#pragma unroll
  for (int j = 0; j < C; ++j) *reinterpret_cast<f32x4_t *>(to + 16 * j) = state.sums[j];
}

// kTile: pages hold whole tiles of so many tokens (16 or 32), so a tile's page is the wave's to look up; 0: any pages.
template <typename E, int D, int NQ, int kTile>
__device__ __forceinline__ void prefix_job(const Decode &p, int block, const uint16_t *__restrict__ key_cache, const uint16_t *__restrict__ value_cache,
                                           uint4 *lds) {
  constexpr int kRowUnits = D / 8, kUnits = kStep * kRowUnits, kLoads = kUnits / kThreads, kChunks = D / 32, C = D / 16;
  constexpr int kIssued = 2 * kLoads;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Jobs of one part and key head follow each other, on one XCD: their rows' tiles read the same run, which its L2 then holds (64
  // sequences, a prefix of 16384, 64 heads on 8: 410 MB read where the workgroups of a run lay on four XCDs).
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
    const uint16_t *const keys_of = key_cache + kh * p.ks[2], *const values_of = value_cache + kh * p.vs[2];      // this head's
    constexpr int T = kTile > 0 ? kTile : 16;
    WaveTile<T> next[kLoads];                          // of the next step to be issued
    const auto find = [&](int t) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if (T == kStep && i > 0) {
          next[i] = next[0];
          continue;
        }
        const int row = __builtin_amdgcn_readfirstlane((i * kWaves + wave) * kWave / kRowUnits);
        next[i].find(p, p.prefix, 0, 0, static_cast<uint32_t>(first + min(t, count - 1) * kStep + row / T * T), last);
      }
    };
    // Where this lane's unit of each load lies from its tile's first row on.
    int row_of[kLoads], unit_of[kLoads];
    uint32_t near_key[kLoads], near_value[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int slot = (i * kWaves + wave) * kWave + lane, row = slot / kRowUnits;
      row_of[i] = row, unit_of[i] = (slot % kRowUnits ^ place<D>(row)) * 8;
      near_key[i] = (row % T) * p.of_token[0] + unit_of[i] * 2, near_value[i] = (row % T) * p.of_token[1] + unit_of[i] * 2;
    }
    const auto issue = [&](int t, int set) {           // step t (the last again behind it)
      uint4 *stage = lds + set * 2 * kUnits;
      const int begin = first + min(t, count - 1) * kStep;
      const uint16_t *const zeros = reinterpret_cast<const uint16_t *>(&kZeroUnit);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint16_t *k, *v;
        if constexpr (kTile > 0) {
          k = next[i].rows(p, keys_of, 0), v = next[i].rows(p, values_of, 1);
          // A tile that not all of counts: the last row again, as values zeros (a weight of 0 times that row's own, were they infinite, would
          // not be 0).
          if (next[i].most < T - 1) {
            const uint32_t row = min(row_of[i] % T, next[i].most);
            k += (row * p.of_token[0] + unit_of[i] * 2) / 2;
            v = begin + row_of[i] < last ? v + (row * p.of_token[1] + unit_of[i] * 2) / 2 : zeros;
          } else {
            k += near_key[i] / 2, v += near_value[i] / 2;
          }
        } else {
          const int token = min(begin + row_of[i], last - 1), entry = page_of(p, token);
          const int page = physical(p, p.prefix, p.prefix_positions, entry), in = token - entry * p.ps;
          k = keys_of + page * p.ks[0] + in * p.ks[1] + unit_of[i];
          v = begin + row_of[i] < last ? values_of + page * p.vs[0] + in * p.vs[1] + unit_of[i] : zeros;
        }
        __builtin_amdgcn_global_load_lds(k, (lds_void_t *)(stage + (i * kWaves + wave) * kWave), 16, 0, 0);
        __builtin_amdgcn_global_load_lds(v, (lds_void_t *)(stage + kUnits + (i * kWaves + wave) * kWave), 16, 0, 0);
      }
      if constexpr (kTile > 0) find(t + 1);
    };
    if constexpr (kTile > 0) find(0);
#pragma unroll
    for (int t = 0; t < kSets - 1; ++t) issue(t, t);
    for (int step = 0, set = 0; step < count; ++step, set = set == kSets - 1 ? 0 : set + 1) {
      INTENT_WAIT_VMCNT((kSets - 2) * kIssued);        // this wave's loads of the step have come
      stage_barrier();                                 // everybody's have, and nobody reads the set that is filled next
      issue(step + kSets - 1, set == 0 ? kSets - 1 : set - 1);
      const uint4 *keys = lds + set * 2 * kUnits, *values = keys + kUnits;
      uint4 key[2][kChunks];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < kChunks; ++c) key[t][c] = keys[(t * 16 + r) * kRowUnits + ((c * 4 + g) ^ place<D>(t * 16 + r))];
      __builtin_amdgcn_sched_barrier(0);               // all of them asked for before the first product
      f32x4_t s[NQ][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][t] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][t] = mfma<E>(key[t][c], q[n][c], s[n][t]);
      }
      // Columns 16 j + r of keys 4 g .. 4 g + 3 of each tile: lane m of a group of 16 points at four columns of key m / 4, and lane i
      // gets column i of all four.
      uint4 column[C];
      const auto ask = [&](int j) {
        u32x2_t half[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int row = t * 16 + g * 4 + (r >> 2), unit = (j * 2 + ((r >> 1) & 1)) ^ place<D>(row);
          const uint16_t *at = reinterpret_cast<const uint16_t *>(values + row * kRowUnits + unit) + (r & 1) * 4;
          half[t] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t *)(at)));
        }
        column[j] = make_uint4(half[0][0], half[0][1], half[1][0], half[1][1]);
      };
#pragma unroll
      for (int j = 0; j < C; ++j) ask(j);
      uint4 weights[NQ][kParts];
      float z[NQ][8];
      powers<E, D, NQ>(state, s, scale, last - first - step * kStep, g, z);
      weigh<E>(z[0], weights[0], state[0].total);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {                   // the next tile's weights beside this one's products
        if (n + 1 < NQ) weigh<E>(z[n + 1], weights[n + 1], state[n + 1].total);
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
          for (int k = 0; k < kParts; ++k) state[n].sums[j] = mfma<E>(column[j], weights[n][k], state[n].sums[j]);
        __builtin_amdgcn_sched_barrier(0);
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

template <typename E, int D, int kTile>
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
  State<D> of_row[1];
  State<D> &state = of_row[0];
  state.clear();
  uint4 q[kChunks];
  {
    const uint16_t *row = p.q + sequence.s * p.qs[0] + (kh * p.group + head) * p.qs[1];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) q[c] = *reinterpret_cast<const uint4 *>(row + (c * 4 + g) * 8);
  }
  const float scale = p.scale * kLog2e;
  // The tiles of a step, where a tile's page is the wave's: of the step at hand, of the next, whose keys are on their way, and of the one
  // after it, whose page is.
  constexpr int T = kTile > 0 ? kTile : 16, kHalves = kStep / T;
  struct Step {
    WaveTile<T> tile[kHalves];
  };
  // A token's place behind the last step may pass 2^31, so it is counted without a sign until it is clamped.
  const auto token_at = [&](int t, int row) { return static_cast<uint32_t>(first) + static_cast<uint32_t>(t) * kStep + row; };
  const auto find = [&](int t) {
    Step found{};
    if constexpr (kTile > 0) {
#pragma unroll
      for (int i = 0; i < kHalves; ++i)
        found.tile[i].find(p, p.indices, p.positions, sequence.first, token_at(t, i * T), last);
    }
    return found;
  };
  const uint16_t *const keys_of = p.k + kh * p.ks[2], *const values_of = p.v + kh * p.vs[2];
  // Row `row` of 32 of step t, its element `at`, of keys (0) or of values (1).
  const auto row_of = [&](const Step &step, int t, int row, int at, int which) {
    const uint16_t *const cache = which ? values_of : keys_of;
    if constexpr (kTile > 0) {
      const WaveTile<T> &tile = step.tile[row / 16 * 16 / T];
      return tile.rows(p, cache, which) + (static_cast<uint32_t>(min(row % T, tile.most)) * p.of_token[which] + at * 2) / 2;
    } else {
      const int64_t(&strides)[3] = which ? p.vs : p.ks;
      const int token = static_cast<int>(min(token_at(t, row), static_cast<uint32_t>(last - 1))), entry = page_of(p, token);
      return cache + physical(p, p.indices, p.positions, sequence.first + entry) * strides[0] + (token - entry * p.ps) * strides[1] + at;
    }
  };
  const auto load_keys = [&](const Step &step, int t, uint4 (&to)[2][kChunks]) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint16_t *const key = row_of(step, t, half * 16 + r, g * 8, 0);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) to[half][c] = *reinterpret_cast<const uint4 *>(key + c * 32);
    }
  };
  const int count = static_cast<int>((static_cast<uint32_t>(last - first) + kStep - 1) / kStep);
  uint4 next_keys[2][kChunks];
  Step next = find(wave), after = find(wave + kWaves);
  if (wave < count) load_keys(next, wave, next_keys);
  for (int t = wave; t < count; t += kWaves) {
    const Step now = next;
    uint4 keys[2][kChunks];
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) keys[half][c] = next_keys[half][c];
    uint32_t values[8][C / 2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t *const value = row_of(now, t, i / 4 * 16 + g * 4 + i % 4, r * C, 1);
      if constexpr (D == 128) {
        const uint4 v = *reinterpret_cast<const uint4 *>(value);
        values[i][0] = v.x, values[i][1] = v.y, values[i][2] = v.z, values[i][3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2 *>(value);
        values[i][0] = v.x, values[i][1] = v.y;
      }
    }
    next = after;
    if (t + kWaves < count) load_keys(next, t + kWaves, next_keys);
    after = find(t + 2 * kWaves);
    f32x4_t s[1][2] = {{f32x4_t{0, 0, 0, 0}, f32x4_t{0, 0, 0, 0}}};
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) s[0][half] = mfma<E>(keys[half][c], q[c], s[0][half]);
    float z[1][8];
    const int live = last - first - t * kStep;
    powers<E, D, 1>(of_row, s, scale, live, g, z);
    uint4 weights[kParts];
    weigh<E>(z[0], weights, state.total);
    if (live < kStep) {                                // values of keys behind the last token: zeros
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < C / 2; ++c) values[i][c] = i / 4 * 16 + g * 4 + i % 4 < live ? values[i][c] : 0;
    }
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const uint4 v = column<C>(values, j);
#pragma unroll
      for (int k = 0; k < kParts; ++k) state.sums[j] = mfma<E>(v, weights[k], state.sums[j]);
    }
  }
  // The waves' states, through the LDS: peaks and sums of weights, then the weighted values at the common peak, half of each lane's
  // columns at a time.
  if (g == 0) peaks[wave * 16 + r] = -state.base;
  __syncthreads();
  float peak = -INFINITY;
  for (int i = 0; i < min(kWaves, count); ++i) peak = fmaxf(peak, peaks[i * 16 + r]);
  const float share = wave >= count ? 0.0f : peak == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(-state.base - peak);
  const float total = sum_of_row(state.total);
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

template <typename E, int D, int NQ, int kTile>
__global__ __launch_bounds__(kThreads, 2) void prefix_decode_jobs(Decode p) {
  constexpr int kStage = 2 * kStep * D / 8;            // keys and values of a step
  static_assert(kSets * kStage * sizeof(uint4) >= kWaves * 16 * (D / 2) * sizeof(float) + kStage * sizeof(uint4), "the waves' states fit behind the first set");
  __shared__ uint4 lds[kSets * kStage];
  const int block = grid_block(), own_blocks = p.jobs * p.kv_heads * p.head_tiles;
  const int first_own = (p.prefix_blocks + 7) / 8 * 8, at = block - first_own;
  if (at < 0) {
    const int job = xcd_tile(block, p.prefix_blocks);
    if (job >= 0) prefix_job<E, D, NQ, kTile>(p, job, p.k, p.v, lds);
  } else if (at < own_blocks) {
    own_job<E, D, kTile>(p, at, reinterpret_cast<float *>(lds + kStage), reinterpret_cast<float *>(lds));
  }
}

// The states of a query head's parts of the prefix and of its sequence's jobs, joined: a workgroup per head, whose waves take a quarter
// of the states each, 64 peaks and sums at a time, a lane each.
template <typename E, int D>
__global__ __launch_bounds__(kThreads) void prefix_decode_join(Decode p) {
  constexpr int kOwn = D / kWave;
  __shared__ float joined[kWaves][D + 2];
  __shared__ bool live_of[kWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q_heads = p.kv_heads * p.group;
  const int64_t row = grid_block();
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
  float peak = -INFINITY, total = 0.0f, sums[kOwn] = {};
  bool any = false;
  constexpr int kAhead = 5;                            // states on their way: a wave has 5 of 20 (8 took the 64 sequences 1% longer)
  float held[kAhead][kOwn];
  const int of_wave = (count + kWaves - 1) / kWaves, last = min(count, (wave + 1) * of_wave);
  // The values of states first .. of this wave (of the last again behind it); not all of them were written.
  const auto ask = [&](int first) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float *from = p.sums + state(min(first + i, last - 1)) * D + lane * kOwn;
#pragma unroll
      for (int j = 0; j < kOwn; ++j) held[i][j] = from[j];
    }
  };
  for (int first = wave * of_wave; first < last; first += kWave) {
    const int at = min(first + lane, last - 1);
    const float of_state = p.total[state(at)], peak_of = p.peak[state(at)];
    ask(first);
    const bool live = first + lane < last && of_state != kNoToken;
    const float most = fmaxf(peak, wave_max(live ? peak_of : -INFINITY));
    const float down = most == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(peak - most);
    const float share = !live ? 0.0f : most == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(peak_of - most);
    any = any || __builtin_amdgcn_ballot_w64(live);
    total = total * down + wave_sum(live ? of_state * share : 0.0f);
#pragma unroll
    for (int j = 0; j < kOwn; ++j) sums[j] *= down;
    peak = most;
    const int here = min(last - first, kWave);
    for (int i0 = 0; i0 < here; i0 += kAhead) {
      if (i0 > 0) ask(first + i0);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const bool counts = i0 + i < here && __builtin_amdgcn_readlane(live, (i0 + i) & 63);
        const float weight = lane_value(share, (i0 + i) & 63);
#pragma unroll
        for (int j = 0; j < kOwn; ++j) sums[j] += counts ? held[i][j] * weight : 0.0f;
      }
    }
  }
  // The waves' own, at the common peak.
#pragma unroll
  for (int j = 0; j < kOwn; ++j) joined[wave][lane * kOwn + j] = sums[j];
  if (lane == 0) joined[wave][D] = peak, joined[wave][D + 1] = total, live_of[wave] = any;
  __syncthreads();
  if (wave > 0) return;
  float of_all = -INFINITY, weight = 0.0f, out[kOwn] = {};
  any = false;
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    if (live_of[w]) any = true, of_all = fmaxf(of_all, joined[w][D]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (!live_of[w]) continue;
    const float share = of_all == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(joined[w][D] - of_all);
    weight += joined[w][D + 1] * share;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) out[j] += joined[w][lane * kOwn + j] * share;
  }
  uint16_t *to = p.out + b * p.outs[0] + h * p.outs[1] + lane * kOwn;
#pragma unroll
  for (int j = 0; j < kOwn; ++j) to[j] = from_f32<E>(any ? out[j] / weight : 0.0f).bits;
}

// How a call is cut.
struct Cut {
  int nq, row_tiles, parts, head_tiles, job_pages, jobs;
};

// NQ = 2 reads the LDS half as often, NQ = 1 leaves room for more waves, which the own tokens' jobs need too. us with NQ = 1 and 2, of 128
// dimensions, bf16, 8 key heads: 128 rows for a key head behind 8192 tokens, up to 512 of their own, 28.1 and 37.3; 512 rows 65 and 70, behind
// 16384 with up to 1000 110 and 113, with 1 92 and 85; 768 rows behind 8192 88 and 87, behind 16384 alone 136 and 122; of 64 dimensions, 256 rows
// 27.0 and 30.3, 512 rows 42.7 and 42.7, behind 16384 alone 65 and 60, 1024 rows 73 and 70. Parts of the prefix for three workgroups a CU in
// place of two: 23.5 for 21.5 (one sequence, 16384 tokens), 118 for 113 (512 rows, 16384 + 1000).
Cut cut(int64_t batch, int64_t kv_heads, int64_t group, int64_t d, int64_t ps, int64_t prefix_positions, int64_t positions) {
  Cut c{};
  const int64_t rows = batch * group, cus = device_cus();
  c.nq = rows <= 4 * d ? 1 : 2;
  c.row_tiles = static_cast<int>((rows + kWaves * 16 * c.nq - 1) / (kWaves * 16 * c.nq));
  const int64_t tokens = prefix_positions * ps, tiles = std::max<int64_t>(c.row_tiles * kv_heads, 1);
  const int64_t most = (tokens + 127) / 128;           // a part walks four steps at least
  c.parts = static_cast<int>(tokens == 0 ? 0 : std::max<int64_t>(1, std::min<int64_t>(most, 2 * cus / tiles)));
  c.head_tiles = static_cast<int>((group + 15) / 16);
  // Jobs of 128 tokens, of more where that makes over two a CU: 8 sequences behind 8191 tokens 19.6 us (256: 20.2), 16 24.6 (25.3); of 64
  // dimensions 256 would take less where there are many (32 sequences behind 8192 20.5 for 23.2) and more where there are few (one 14.5 for 13.7).
  const int64_t own = positions * ps, aim = 2 * cus / std::max<int64_t>(kv_heads * c.head_tiles, 1);
  const int64_t of_job = std::max<int64_t>(128, (own + std::max<int64_t>(aim, 1) - 1) / std::max<int64_t>(aim, 1));
  c.job_pages = ps > 0 ? static_cast<int>(std::max<int64_t>(1, (of_job + ps - 1) / ps)) : 1;
  c.jobs = static_cast<int>((ps > 0 ? positions / c.job_pages : 0) + batch);
  return c;
}

// The tiles of tokens that pages come in; `reach`: the largest stride of a page, or elements from a page's first token to behind its last,
// which are counted in 32 bits of bytes then.
int tile_of(int64_t ps, int64_t reach) { return reach >= int64_t{1} << 31 || ps == 0 || ps % 16 ? 0 : ps % 32 ? 16 : 32; }

size_t states_of(const Cut &c, int64_t batch, int64_t q_heads) { return (static_cast<size_t>(c.parts) * batch + c.jobs) * q_heads; }

template <typename E, typename F>
int with_kernel(int64_t d, int nq, int tile, F f) {
  const auto of = [&](auto width, auto rows) {
    return tile == 32   ? f(prefix_decode_jobs<E, width.value, rows.value, 32>, prefix_decode_join<E, width.value>)
           : tile == 16 ? f(prefix_decode_jobs<E, width.value, rows.value, 16>, prefix_decode_join<E, width.value>)
                        : f(prefix_decode_jobs<E, width.value, rows.value, 0>, prefix_decode_join<E, width.value>);
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
  // Tokens of a table (to behind the last part of them) and rows of queries are counted in 32 bits, and so are blocks.
  if (batch > (1 << 20) || q_heads > (1 << 16) || pages > INT32_MAX || ps > (1 << 20) || prefix_positions > (1 << 28) || positions > (1 << 28) ||
      prefix_positions * ps > INT32_MAX - (1 << 20) || positions * ps > (int64_t{1} << 40) || batch * q_heads > (1 << 28))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}

}  // namespace

int prefix_decode_resources(int dtype, int64_t batch, int64_t kv_heads, int64_t group, int64_t d, int64_t ps, int64_t prefix_positions,
                            int64_t positions, int64_t reach, IntentHipKernelResources *out) {
  if (int rc = check(batch, kv_heads * group, kv_heads, group, d, 1, ps, prefix_positions, positions)) return rc;
  const Cut c = cut(batch, kv_heads, group, d, ps, prefix_positions, positions);
  const int tile = tile_of(ps, reach);
  char name[64];
  snprintf(name, sizeof(name), "prefix_decode_jobs<%s,%lld,%d,%d>", dtype == INTENT_HIP_F16 ? "f16" : "bf16", static_cast<long long>(d), c.nq, tile);
  const auto describe = [&](void (*kernel)(Decode), void (*)(Decode)) {
    return describe_kernel(reinterpret_cast<const void *>(kernel), name, kThreads, out);
  };
  return dtype == INTENT_HIP_F16 ? with_kernel<f16_t>(d, c.nq, tile, describe) : with_kernel<bf16_t>(d, c.nq, tile, describe);
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
  *bytes = states_of(cut(batch, kv_heads, head_group, d, ps, prefix_positions, positions), batch, q_heads) * (d + 2) * sizeof(float);
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
  const Cut c = cut(batch, kv_heads, head_group, d, ps, prefix_positions, positions);
  const size_t states = states_of(c, batch, q_heads), bytes = states * (d + 2) * sizeof(float);
  if (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16))
    return fail(INTENT_HIP_ERR_WORKSPACE, "paged_gqa_decode_prefix needs %zu workspace bytes, 16-byte aligned", bytes);
  Decode p{};
  p.q = static_cast<const uint16_t *>(q), p.k = static_cast<const uint16_t *>(key_cache), p.v = static_cast<const uint16_t *>(value_cache);
  p.out = static_cast<uint16_t *>(output);
  p.prefix = prefix_indices, p.prefix_length = prefix_length, p.offsets = page_offsets, p.indices = page_indices, p.lengths = lengths;
  p.qs[0] = strides[0], p.qs[1] = strides[1], p.outs[0] = strides[11], p.outs[1] = strides[12];
  for (int i = 0; i < 3; ++i) p.ks[i] = strides[3 + i], p.vs[i] = strides[7 + i];
  p.pages = ps > 0 ? pages : 0, p.ps = static_cast<int>(ps);
  if (ps > 0) {
    while (int64_t{1} << p.shift < ps) ++p.shift;
    p.magic = static_cast<uint32_t>(((((uint64_t{1} << p.shift) - ps) << 32) / ps) + 1);
  }
  p.prefix_positions = static_cast<int>(prefix_positions), p.positions = static_cast<int>(positions);
  p.batch = static_cast<int>(batch), p.kv_heads = static_cast<int>(kv_heads), p.group = static_cast<int>(head_group);
  p.row_tiles = c.row_tiles, p.parts = c.parts, p.prefix_blocks = static_cast<int>(c.row_tiles * kv_heads * c.parts);
  p.head_tiles = c.head_tiles, p.job_pages = c.job_pages, p.jobs = c.jobs, p.scale = scale;
  p.sums = static_cast<float *>(workspace), p.peak = p.sums + states * d, p.total = p.peak + states;
  const int64_t blocks = (static_cast<int64_t>(p.prefix_blocks) + 7) / 8 * 8 + static_cast<int64_t>(c.jobs) * kv_heads * c.head_tiles;
  const auto run = [&](void (*jobs)(Decode), void (*join)(Decode)) {
    jobs<<<tile_grid(blocks, 1), kThreads, 0, as_stream(stream)>>>(p);
    join<<<tile_grid(batch * q_heads, 1), kThreads, 0, as_stream(stream)>>>(p);
    return 0;
  };
  int64_t reach = 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t *const of = i == 0 ? p.ks : p.vs;
    reach = std::max({reach, of[0], of[1] >= int64_t{1} << 31 ? of[1] : of[1] * ps});
    p.of_page[i] = static_cast<uint32_t>(of[0] * 2), p.of_token[i] = static_cast<uint32_t>(of[1] * 2);
  }
  const int tile = tile_of(ps, reach);
  if (dtype == INTENT_HIP_F16)
    with_kernel<f16_t>(d, c.nq, tile, run);
  else
    with_kernel<bf16_t>(d, c.nq, tile, run);
  return hipPeekAtLastError() != hipSuccess ? launch_status("paged_gqa_decode_prefix") : INTENT_HIP_OK;
}

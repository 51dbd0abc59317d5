// Attention of one new token per sequence over a paged cache of e4m3 elements with a shared power of two per 32, for gfx950.
// No reference counterpart; the cache and its tables are those of mx_cache.hip.
//
// For query head h of sequence s, over the positions j below lengths[s] that the tables have a page for:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp2(scale * log2(e) * (q . k_j) - peak)        0 where there is none
// Keys and values are taken in the query's type (element * 2^e, one rounding) and products are summed in f32. Weights are f32
// and enter the second product whole, as three bf16 numbers of 8 bits each: f16 numbers end at 2^-24, and the sum that the
// products are divided by holds the weights below. Two bf16 numbers would leave out 2^-16 of a weight; the third costs up to 4 %
// where jobs are few (one sequence of 512, f16: 8.1 us, two 7.8; 8 of 8191: 34.5 and 34.3) and nothing where they are many (64
// ragged sequences up to 8191, bf16: 135.2 and 135.4). The values are bf16 numbers exactly: e4m3 has four bits.
// Where their exponents are such that f16 rounds or does not reach them, f16 calls convert them by way of f16 (35.9 -> 37.8).
//
// Design. The page range of a sequence is cut into jobs of `job_pages` pages; job j of the flat list belongs to the last
// sequence s with page_offsets[s] / job_pages + s <= j, which every wave finds by itself, so no table of work is made and
// lengths may change under a captured graph. A workgroup takes a job of one key head, its waves 32 keys in turn; only their
// final states go through the LDS, and the states of a sequence's jobs through the workspace to mx_decode_merge:
//   * scores: v_mfma_f32_16x16x32 with 16 keys as rows and 16 query heads as columns. The sum over a head's dimensions may
//     run in any order, so lane (r, g) takes dimensions g D / 4 .. of key r as they lie in memory, converts them with its
//     blocks' scales, and the query is laid out to match.
//   * weights: the result leaves keys 4 g .. 4 g + 3 of head r in lane (r, g), which is where the second product wants
//     them: heads as rows, 32 keys (4 of each 16 per lane) summed over.
//   * values: lane (c, g) loads its columns of its own 8 keys and pairs them with v_perm, for 16 columns a product.
//     Their exponents come a key a lane and go to the lanes that use them by a permutation (8 sequences of 8191: 34.9 us with a
//     byte a lane and key, 33.9 so).
//   * the running maximum is raised (and the sums scaled down) only when a score passes it by 2^8, so most steps have no
//     cross-lane move at all; weights up to 2^8 are far inside bf16.
// Bound by the cache's bytes once there are many jobs (64 sequences of 8191, 8 key heads of 128: 191 us, 5.1 TB/s; the loads
// alone take as long); with few jobs by a step's chain of instructions, about 470 of a wave. Where a tile of 16 keys may cross pages
// (PS no multiple of 16) every lane looks up the pages of its own keys: 8 sequences of 8191 take 82 us with pages of 1, 80 with 8,
// 39 with 16, 35 with 64.
#include <stdio.h>

#include <algorithm>
#include <type_traits>

#include "mx.hpp"

namespace intent_hip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kParts = 3;              // bf16 numbers of a weight
constexpr int kStep = 32;              // keys of a wave's step: two tiles of 16
constexpr float kSlack = 8.0f;
constexpr float kNoToken = -1.0f;      // the sum of a state without a token (weights are not negative)
constexpr uint32_t kSigns = 0x80008000u;
constexpr uint32_t kTiny = 0x00800080u;          // 2^-126 in bf16, twice
constexpr int kMany = 6, kFew = 2;     // workgroups a CU is given
constexpr int kLong = 256;            // tokens of a job: from here on it is one of many
constexpr int kLeast = 128;
constexpr int kWhole = 2048, kWholeOne = 768;   // tokens of all sequences and of one, up to here each is one job

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct Decode {
  const uint16_t *q;
  const uint8_t *k, *ke, *v, *ve;
  uint16_t *out;
  const int32_t *lengths;
  PageTable table;
  int64_t qs[2], ks[3], kes[3], vs[3], ves[3], outs[2];
  int batch, kv_heads, group, head_tiles, job_pages, jobs;
  float scale;
  float *peak, *total, *sums;          // states of the jobs: [jobs][q_heads] twice, [jobs][q_heads][D]; null: one job a sequence
};

template <typename E>
__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same_v<E, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Two f32 in bf16, rounded to nearest even.
__device__ __forceinline__ uint32_t in_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{a, b}, bfloat2_t));
}

// Two weights as sums of kParts bf16 numbers each: 8 bits of what the numbers before leave, cut off, so that three hold all 24
// and none is negative.
__device__ __forceinline__ void parts(float a, float b, uint32_t (&part)[kParts]) {
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const uint32_t u = __float_as_uint(a), v = __float_as_uint(b);
    part[i] = __builtin_amdgcn_perm(v, u, 0x07060302);
    a -= __uint_as_float(u & 0xFFFF0000u), b -= __uint_as_float(v & 0xFFFF0000u);
  }
}

// A sequence: its first entry of the page indices, and its tokens: what its length and its pages both have; none in a cache
// without a page.
struct Sequence {
  int s, first, tokens;
  __device__ __forceinline__ void settle(const Decode &p, int next, int length) {
    const int64_t held = static_cast<int64_t>(max(0, next - first)) * p.table.ps;
    tokens = p.table.pages == 0 || length < 0 ? 0 : length < held ? length : static_cast<int>(held);
  }
};

// The sequence of job `job` (the wave's): the last whose jobs, from offsets[s] / job_pages + s on, begin at or before it.
// Found by all lanes of the wave, who then hold what is known of 64 candidates.
__device__ __forceinline__ Sequence job_sequence(const Decode &p, int job) {
  const int lane = threadIdx.x & 63;
  int first = 0, count = p.batch - 1;          // it is one of first .. first + count
  while (count >= kWave) {
    const int step = (count + 63) / 64;
    const int at = (lane + 1) * step;
    const bool past = at <= count && static_cast<int64_t>(p.table.offsets[first + at] / p.job_pages) + first + at <= job;
    const int steps = __popcll(__ballot(past));
    first += steps * step;
    count = min(step - 1, count - steps * step);
  }
  const bool in = lane <= count;
  const int s = first + (in ? lane : 0), begin = p.table.offsets[s], next = p.table.offsets[s + 1], length = p.lengths[s];
  const bool past = lane > 0 && in && static_cast<int64_t>(begin / p.job_pages) + s <= job;
  const int at = __popcll(__ballot(past));
  Sequence found{first + at, __builtin_amdgcn_readlane(begin, at), 0};
  found.settle(p, __builtin_amdgcn_readlane(next, at), __builtin_amdgcn_readlane(length, at));
  return found;
}

// How a lane's columns of the values lie: `kWide` runs of 128 columns (8 bytes a lane), then one of 64 (4) and one of 32 (2).
template <int D>
struct Columns {
  static constexpr int kWide = D / 128, kRest = D % 128;
  static constexpr bool kHalf = kRest >= 64, kQuarter = kRest % 64 != 0;
  static constexpr int kRuns = kWide + kHalf + kQuarter;
  static constexpr int kTiles = D / 16;          // products of 16 columns
  // Column of lane r in product j.
  static __device__ __forceinline__ int column(int j, int r) {
    if (j < kWide * 8) return j / 8 * 128 + r * 8 + j % 8;
    if (kHalf && j < kWide * 8 + 4) return kWide * 128 + r * 4 + (j - kWide * 8);
    return D - 32 + r * 2 + (j - (kTiles - 2));
  }
};

// Waves of a SIMD: what the accumulators, the query and a step's loads leave room for.
constexpr int waves_per_simd(int width) { return width <= 64 ? 4 : width <= 128 ? 3 : width <= 256 ? 2 : 1; }

template <int D>
struct Step {                                     // what a lane loads for 32 keys
  uint2 k[2][D / 32];                             // [tile][8 dimensions]
  uint8_t ke[2][D / 32];
  uint2 v[8][Columns<D>::kRuns];                  // [key][run]
  uint8_t ve[8][Columns<D>::kRuns];               // its block's exponent; with kUniform instead:
  uint32_t powers[2][Columns<D>::kRuns];          // [tile][run]: all exponents of key r of the tile
  int valid[2];                                   // kUniform: how many keys of a tile have a token
  unsigned live;                                  // else: a bit for each of the lane's keys of the values
};

// kUniform: a tile of 16 keys lies in one page (PS is a multiple of 16), so its address is the wave's, and a lane's place in
// it stays the same.
template <typename E, int D, int QT, bool kUniform, int W>
__global__ __launch_bounds__(W *kWave) __attribute__((amdgpu_waves_per_eu(waves_per_simd(D * QT)))) void mx_decode(Decode p) {
  using C = Columns<D>;
  constexpr int kChunks = D / 32;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ float sums_s[W][C::kTiles * 4][kWave], peak_s[W][16], total_s[W][16];
  // Key heads of a job run on one XCD at about the same time: pages with their heads side by side share lines.
  const int n = static_cast<int>(gridDim.x), xcd = static_cast<int>(blockIdx.x) % 8;
  const int item = xcd * (n / 8) + (xcd < n % 8 ? xcd : n % 8) + static_cast<int>(blockIdx.x) / 8;
  const int ht = item % p.head_tiles, kh = item / p.head_tiles % p.kv_heads, job = item / p.head_tiles / p.kv_heads;
  const Sequence sequence = job_sequence(p, job);
  const int s = sequence.s, place = job - (sequence.first / p.job_pages + s);        // of the job among the sequence's
  const int64_t begin = static_cast<int64_t>(place) * p.job_pages * p.table.ps, size = static_cast<int64_t>(p.job_pages) * p.table.ps;
  // A sequence without a token is its first job's, which writes the 0 itself where no states are joined.
  if (place < 0 || (begin >= sequence.tokens && (place > 0 || p.peak != nullptr))) return;
  const int tokens = static_cast<int>(sequence.tokens - begin < size ? sequence.tokens - begin : size);      // of the job
  const int index0 = sequence.first + place * p.job_pages;           // its first entry of the page indices
  const int head0 = kh * p.group + ht * QT * 16, heads = min(QT * 16, p.group - ht * QT * 16);

  uint4 q[QT][kChunks];
#pragma unroll
  for (int t = 0; t < QT; ++t)
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      q[t][c] = make_uint4(0, 0, 0, 0);
      if (t * 16 + r < heads)
        q[t][c] = *reinterpret_cast<const uint4 *>(p.q + s * p.qs[0] + (head0 + t * 16 + r) * p.qs[1] + g * (D / 4) + c * 8);
    }
  // The sign of the scale goes to the query, so that scores order as their products do.
  const float c1 = fabsf(p.scale) * kLog2e;
  if (p.scale < 0.0f)
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        q[t][c] = make_uint4(q[t][c].x ^ kSigns, q[t][c].y ^ kSigns, q[t][c].z ^ kSigns, q[t][c].w ^ kSigns);
  f32x4_t acc[QT][C::kTiles];
  float peak[QT], total[QT];
  bool any = false;                    // a token so far
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    peak[t] = -INFINITY;
    total[t] = 0.0f;
#pragma unroll
    for (int j = 0; j < C::kTiles; ++j) acc[t][j] = f32x4_t{0, 0, 0, 0};
  }

  // A key's elements and exponents, and a value's, from a row's start and this lane's offset in it.
  const auto key = [&](Step<D> &x, int u, const uint8_t *k, const uint8_t *ke, unsigned ko, unsigned keo) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      x.k[u][c] = *reinterpret_cast<const uint2 *>(k + ko + g * (D / 4) + c * 8);
      x.ke[u][c] = ke[keo + (g * (D / 4) + c * 8) / 32];
    }
  };
  const auto value = [&](Step<D> &x, int i, const uint8_t *v, unsigned vo) {
#pragma unroll
    for (int w = 0; w < C::kWide; ++w) x.v[i][w] = *reinterpret_cast<const uint2 *>(v + vo + w * 128 + r * 8);
    if constexpr (C::kHalf) x.v[i][C::kWide].x = *reinterpret_cast<const uint32_t *>(v + vo + C::kWide * 128 + r * 4);
    if constexpr (C::kQuarter) x.v[i][C::kRuns - 1].x = *reinterpret_cast<const uint16_t *>(v + vo + D - 32 + r * 2);
  };
  const auto value_power = [&](Step<D> &x, int i, const uint8_t *ve) {
#pragma unroll
    for (int w = 0; w < C::kWide; ++w) x.ve[i][w] = ve[w * 4 + r / 4];
    if constexpr (C::kHalf) x.ve[i][C::kWide] = ve[C::kWide * 4 + r / 8];
    if constexpr (C::kQuarter) x.ve[i][C::kRuns - 1] = ve[D / 32 - 1];
  };
  // A tile's value exponents, key r's in lane (r, g): a load a run, where the lanes that use them would take one a key, and
  // each touch as many lines.
  const auto value_powers = [&](Step<D> &x, int u, const uint8_t *ve) {
#pragma unroll
    for (int w = 0; w < C::kWide; ++w) __builtin_memcpy(&x.powers[u][w], ve + w * 4, 4);
    if constexpr (C::kHalf) {
      uint16_t two;
      __builtin_memcpy(&two, ve + C::kWide * 4, 2);
      x.powers[u][C::kWide] = two;
    }
    if constexpr (C::kQuarter) x.powers[u][C::kRuns - 1] = ve[D / 32 - 1];
  };

  const auto fold = [&](Step<D> &x) {
    // Scores of keys 16 u + 4 g + i against head 16 t + r.
    f32x4_t sc[QT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int t = 0; t < QT; ++t) sc[t][u] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const float ks = mx_scale(x.ke[u][c]);
        const uint4 k = make_uint4(mx_pair_e4m3<E, false>(x.k[u][c].x, ks), mx_pair_e4m3<E, true>(x.k[u][c].x, ks),
                                   mx_pair_e4m3<E, false>(x.k[u][c].y, ks), mx_pair_e4m3<E, true>(x.k[u][c].y, ks));
#pragma unroll
        for (int t = 0; t < QT; ++t) sc[t][u] = mfma<E>(k, q[t][c], sc[t][u]);
      }
    }
    bool live[8];
    bool whole = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      live[i] = kUniform ? g * 4 + (i & 3) < x.valid[i >> 2] : (x.live >> i & 1) != 0;
      whole = whole && live[i];
    }
    const bool all = kUniform ? x.valid[0] == 16 && x.valid[1] == 16 : __all(whole);
    float vs[8][C::kRuns];                          // scales of the lane's columns of its keys
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int w = 0; w < C::kRuns; ++w) {
        if constexpr (kUniform) {
          const uint32_t word = __builtin_amdgcn_ds_bpermute((g * 4 + (i & 3)) * 4, static_cast<int>(x.powers[i >> 2][w]));
          vs[i][w] = mx_scale(word >> (w < C::kWide ? r / 4 * 8 : C::kHalf && w == C::kWide ? r / 8 * 8 : 0) & 0xFF);
        } else {
          vs[i][w] = mx_scale(x.ve[i][w]);
        }
      }
    // Whether a value may be one that its type rounds or holds as infinity: exponents outside -15 .. 7 (f16) or above 119 (bf16);
    // asked of all exponents in a few comparisons of bits, which take -15 .. 0 and up to 0 as certain.
    constexpr bool kF16 = std::is_same_v<E, f16_t>;
    constexpr uint32_t kSure = kF16 ? 0x70707070u : 0u, kAsked = kF16 ? 0xF0F0F0F0u : 0x80808080u;
    uint32_t odd = 0;
#pragma unroll
    for (int w = 0; w < C::kRuns; ++w) {
      if constexpr (kUniform) {
        const uint32_t bytes = w < C::kWide ? ~0u : C::kHalf && w == C::kWide ? 0xFFFFu : 0xFFu;
        odd |= ((x.powers[0][w] ^ kSure) | (x.powers[1][w] ^ kSure)) & bytes;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) odd |= x.ve[i][w] ^ (kSure & 0xFFu);
      }
    }
    const bool extreme = __any((odd & kAsked) != 0);
    if (!all) {
      // What lies in places without a token has no weight, and must not turn a zero weight into NaN.
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < C::kRuns; ++w)
          if (!live[i]) x.v[i][w] = make_uint2(0, 0), vs[i][w] = 1.0f;
    }
    uint4 wp[QT][kParts];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float z[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = all || live[i] ? sc[t][i >> 2][i & 3] : -INFINITY;
      float most = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7]))) * c1;
      if (__any(most > peak[t] + kSlack)) {
        most = fmaxf(most, __shfl_xor(most, 16));
        most = fmaxf(most, __shfl_xor(most, 32));
        const float next = fmaxf(peak[t], most);
        const float shrink = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(peak[t] - next);
        peak[t] = next;
        total[t] *= shrink;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = __shfl(shrink, g * 4 + i);
#pragma unroll
          for (int j = 0; j < C::kTiles; ++j) acc[t][j][i] *= f;
        }
      }
      const float base = peak[t] == -INFINITY ? 0.0f : -peak[t];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i], c1, base));
      if (!all)                                     // (-inf times a scale of 0 is NaN)
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = live[i] ? w[i] : 0.0f;
      total[t] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      uint32_t part[4][kParts];
#pragma unroll
      for (int i = 0; i < 4; ++i) parts(w[2 * i], w[2 * i + 1], part[i]);
      if (__builtin_expect(extreme, 0))             // infinity by a number of 0 is NaN; none is 0 where the first is not
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 1; j < kParts; ++j) part[i][j] = mx_larger(part[i][j], mx_smaller(part[i][0], kTiny));
#pragma unroll
      for (int i = 0; i < kParts; ++i) wp[t][i] = make_uint4(part[0][i], part[1][i], part[2][i], part[3][i]);
    }
    // Values: pairs of columns of each key, paired again over the keys.
    const auto columns = [&](int run, int tile, auto upper, auto half) {
      uint32_t pair[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t word = upper.value ? x.v[i][run].y : x.v[i][run].x;
        pair[i] = mx_pair_e4m3<bf16_t, half.value>(word, vs[i][run]);
      }
      if constexpr (kF16)
        if (__builtin_expect(extreme, 0))           // by way of f16
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t word = upper.value ? x.v[i][run].y : x.v[i][run].x;
            const half2_t h = __builtin_bit_cast(half2_t, mx_pair_e4m3<f16_t, half.value>(word, vs[i][run]));
            pair[i] = in_bf16(static_cast<float>(h[0]), static_cast<float>(h[1]));
          }
      uint32_t even[4], odd[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        even[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100);
        odd[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302);
      }
      const uint4 v0 = make_uint4(even[0], even[1], even[2], even[3]), v1 = make_uint4(odd[0], odd[1], odd[2], odd[3]);
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          acc[t][tile] = mfma<bf16_t>(wp[t][i], v0, acc[t][tile]);
          acc[t][tile + 1] = mfma<bf16_t>(wp[t][i], v1, acc[t][tile + 1]);
        }
    };
    constexpr std::integral_constant<bool, false> no{};
    constexpr std::integral_constant<bool, true> yes{};
#pragma unroll
    for (int w = 0; w < C::kWide; ++w) {
      columns(w, w * 8, no, no);
      columns(w, w * 8 + 2, no, yes);
      columns(w, w * 8 + 4, yes, no);
      columns(w, w * 8 + 6, yes, yes);
    }
    if constexpr (C::kHalf) {
      columns(C::kWide, C::kWide * 8, no, no);
      columns(C::kWide, C::kWide * 8 + 2, no, yes);
    }
    if constexpr (C::kQuarter) columns(C::kRuns - 1, C::kTiles - 2, no, no);
  };

  if constexpr (kUniform) {
    // The wave's tiles: the first token of each, its page among the job's and its place there.
    const int ps = p.table.ps, pages_on = W * kStep / ps, places_on = W * kStep - pages_on * ps;
    int at[2], logical[2], slot[2], raw[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      at[u] = wave * kStep + u * 16;
      logical[u] = at[u] / ps, slot[u] = at[u] - logical[u] * ps;
    }
    const auto look = [&](int u) {                 // the page index of a tile, on its way a step early
      const int index = index0 + logical[u];
      raw[u] = at[u] < tokens && index >= 0 && index < p.table.positions ? p.table.indices[index] : -1;
    };
    look(0), look(1);
    // Of this key head, and of this lane's places in a tile.
    const uint8_t *const k0 = p.k + kh * p.ks[2], *const ke0 = p.ke + kh * p.kes[2];
    const uint8_t *const v0 = p.v + kh * p.vs[2], *const ve0 = p.ve + kh * p.ves[2];
    const uint64_t ks0 = p.ks[0], kes0 = p.kes[0], vs0 = p.vs[0], ves0 = p.ves[0];
    const unsigned ks1 = static_cast<unsigned>(p.ks[1]), kes1 = static_cast<unsigned>(p.kes[1]);
    const unsigned vs1 = static_cast<unsigned>(p.vs[1]), ves1 = static_cast<unsigned>(p.ves[1]);
    const unsigned ko = r * ks1, keo = r * kes1;
    const unsigned veo = r * ves1;
    unsigned vo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vo[i] = (g * 4 + i) * vs1;
    const auto load = [&](Step<D> &x) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // A tile without a page reads any 16 rows of the cache: their weights are 0.
        const bool none = raw[u] < 0 || raw[u] >= p.table.pages;
        const uint64_t page = static_cast<unsigned>(none ? 0 : raw[u]), in = static_cast<unsigned>(none ? 0 : slot[u]);
        x.valid[u] = none ? 0 : min(tokens - at[u], 16);
        at[u] += W * kStep;
        logical[u] += pages_on, slot[u] += places_on;
        if (slot[u] >= ps) slot[u] -= ps, ++logical[u];
        look(u);
        key(x, u, k0 + (page * ks0 + in * ks1), ke0 + (page * kes0 + in * kes1), ko, keo);
        const uint8_t *const v = v0 + (page * vs0 + in * vs1), *const ve = ve0 + (page * ves0 + in * ves1);
        value_powers(x, u, ve + veo);
#pragma unroll
        for (int i = 0; i < 4; ++i) value(x, u * 4 + i, v, vo[i]);
      }
    };
    while (at[0] < tokens) {
      Step<D> x;
      load(x);
      any = any || x.valid[0] > 0 || x.valid[1] > 0;
      fold(x);
    }
  } else {
    // Any page size: every lane finds its own keys.
    for (int at = wave * kStep; at < tokens; at += W * kStep) {
      Step<D> x;
      x.live = 0;
      const auto find = [&](int token, int64_t &page, int64_t &in) {
        const int logical = token / p.table.ps, index = index0 + logical;
        const int raw = token < tokens && index >= 0 && index < p.table.positions ? p.table.indices[index] : -1;
        const bool none = raw < 0 || raw >= p.table.pages;
        page = none ? 0 : raw, in = none ? 0 : token - logical * p.table.ps;
        return !none;
      };
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        int64_t page, in;
        find(at + u * 16 + r, page, in);
        key(x, u, p.k + page * p.ks[0] + in * p.ks[1] + kh * p.ks[2], p.ke + page * p.kes[0] + in * p.kes[1] + kh * p.kes[2], 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x.live |= static_cast<unsigned>(find(at + u * 16 + g * 4 + i, page, in)) << (u * 4 + i);
          value(x, u * 4 + i, p.v + page * p.vs[0] + in * p.vs[1] + kh * p.vs[2], 0);
          value_power(x, u * 4 + i, p.ve + page * p.ves[0] + in * p.ves[1] + kh * p.ves[2]);
        }
      }
      any = any || __any(x.live != 0);
      fold(x);
    }
  }

  // The waves' states, a tile of query heads at a time: brought to the common maximum and added in wave order. Wave w takes
  // rows 4 g + w % 4 of the tile and, of eight waves, half of their columns.
  const int q_heads = p.kv_heads * p.group;
  constexpr int kMine = C::kTiles * 4 / W;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    total[t] += __shfl_xor(total[t], 16);
    total[t] += __shfl_xor(total[t], 32);
    if (t > 0) __syncthreads();
    if (g == 0) peak_s[wave][r] = peak[t], total_s[wave][r] = any ? total[t] : kNoToken;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < C::kTiles; ++j) sums_s[wave][i * C::kTiles + j][lane] = acc[t][j][i];
    __syncthreads();
    const int i = wave & 3, j0 = wave / 4 * kMine, in = g * 4 + i, head = t * 16 + in;
    float whole = -INFINITY, sum = 0.0f, row[kMine] = {};
    bool token = false;
#pragma unroll
    for (int w = 0; w < W; ++w) whole = fmaxf(whole, peak_s[w][in]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float own = peak_s[w][in];
      const float f = own == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(own - whole);      // a wave without a score has sums of 0, or NaN
      const bool none = total_s[w][in] < 0.0f;
      sum += none ? 0.0f : total_s[w][in] * f;
      token = token || !none;
#pragma unroll
      for (int j = 0; j < kMine; ++j) row[j] += sums_s[w][i * C::kTiles + j0 + j][lane] * f;
    }
    if (head >= heads) continue;
    const int64_t state = static_cast<int64_t>(job) * q_heads + head0 + head;
    if (p.peak != nullptr && r == 0 && j0 == 0) p.peak[state] = whole, p.total[state] = token ? sum : kNoToken;
    const float share = p.peak != nullptr ? 1.0f : token ? 1.0f / sum : 0.0f;
    float *const sums = p.sums + state * D;
    uint16_t *const out = p.out + s * p.outs[0] + (head0 + head) * p.outs[1];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int column = C::column(j0 + j, r);
      if (p.peak != nullptr)
        sums[column] = row[j];
      else
        out[column] = from_f32<E>(row[j] * share).bits;
    }
  }
}

// Output rows from the states of a sequence's jobs: a workgroup per (sequence, query head), its W waves every W-th job each.
// A lane weighs one job in 64 of its wave's, then the lanes take columns and add the jobs' sums in order, eight on their way
// at once.
template <typename E, int D, int W>
__global__ __launch_bounds__(W *kWave) void mx_decode_merge(Decode p) {
  constexpr int kColumns = (D + kWave - 1) / kWave, kTogether = 8;
  __shared__ float sums_s[W][kColumns * kWave], peak_s[W], total_s[W];
  const int q_heads = p.kv_heads * p.group, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = static_cast<int>(blockIdx.x) / q_heads, head = static_cast<int>(blockIdx.x) - s * q_heads;
  Sequence sequence{s, p.table.offsets[s], 0};
  sequence.settle(p, p.table.offsets[s + 1], p.lengths[s]);
  const int64_t size = static_cast<int64_t>(p.job_pages) * p.table.ps;
  const int first = sequence.first / p.job_pages + s;
  int jobs = static_cast<int>((sequence.tokens + size - 1) / size);
  if (first < 0 || static_cast<int64_t>(first) + jobs > p.jobs) jobs = 0;
  const int mine = (jobs - wave + W - 1) / W;              // jobs wave, wave + W, ..
  const int64_t row0 = static_cast<int64_t>(first + wave) * q_heads + head, stride = static_cast<int64_t>(W) * q_heads;
  float peak = -INFINITY;
  for (int j = lane; j < mine; j += kWave) peak = fmaxf(peak, p.peak[row0 + j * stride]);
  peak = wave_max(peak);
  float total = 0.0f, out[kColumns] = {};
  bool token = false;
  for (int j0 = 0; j0 < mine; j0 += kWave) {
    const int count = min(mine - j0, kWave);
    float weight = 0.0f;
    if (lane < count) {
      const float own = p.peak[row0 + (j0 + lane) * stride];
      weight = own == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(own - peak);        // a job without a score has sums of 0, or NaN
      const float sum = p.total[row0 + (j0 + lane) * stride];
      token = token || !(sum < 0.0f);
      total += sum < 0.0f ? 0.0f : sum * weight;
    }
    for (int j = 0; j < count; j += kTogether) {
      float from[kTogether][kColumns] = {};
#pragma unroll
      for (int i = 0; i < kTogether; ++i)
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
          if (j + i < count && (D % kWave == 0 || c * kWave + lane < D))
            from[i][c] = p.sums[(row0 + (j0 + j + i) * stride) * D + c * kWave + lane];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const float w = j + i < count ? lane_value(weight, j + i) : 0.0f;
#pragma unroll
        for (int c = 0; c < kColumns; ++c) out[c] += from[i][c] * w;
      }
    }
  }
  total = wave_sum(total);
  token = __any(token);
  if (lane == 0) peak_s[wave] = peak, total_s[wave] = token ? total : kNoToken;
#pragma unroll
  for (int c = 0; c < kColumns; ++c) sums_s[wave][c * kWave + lane] = out[c];
  __syncthreads();
  float whole = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) whole = fmaxf(whole, peak_s[w]);
  for (int column = threadIdx.x; column < D; column += W * kWave) {
    float sum = 0.0f, value = 0.0f;
    bool held = false;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = peak_s[w] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(peak_s[w] - whole);
      sum += total_s[w] < 0.0f ? 0.0f : total_s[w] * f;
      held = held || !(total_s[w] < 0.0f);
      value += sums_s[w][column] * f;
    }
    p.out[s * p.outs[0] + head * p.outs[1] + column] = from_f32<E>(value * (held ? 1.0f / sum : 0.0f)).bits;
  }
}

// How a call is cut, from what the host knows: the pages that the table holds for all sequences. Measured with 8 key heads of
// 128, 4 query heads each, us:
//   * few tokens in all and per sequence: a workgroup of eight waves takes a whole sequence, and nothing is joined (4
//     sequences of 300: 7.0, in jobs 10.7; one of 1024 11.2 and 10.3, one of 2048 17.8 and 10.1);
//   * else jobs of four waves, 6 workgroups a CU where that leaves a job 256 tokens, so that a job's start and end hide behind
//     others (64 sequences of 8191: 191; 2 a CU 204, 3 210), or 2, which are on the chip at once;
//   * a job has 128 tokens at least (one sequence of 2048: 10.1; 256 11.4, 512 13.4).
struct Cut {
  int job_pages, jobs, head_tiles, qt, waves;
  bool merge;
  int64_t blocks;
};
Cut cut(int64_t batch, int64_t kv_heads, int64_t group, int64_t positions, int64_t ps) {
  Cut c{};
  c.qt = group > 16 ? 2 : 1;
  c.head_tiles = static_cast<int>((group + 16 * c.qt - 1) / (16 * c.qt));
  const int64_t all = positions * ps, heads = kv_heads * c.head_tiles;
  int64_t tokens = all * heads / (kMany * device_cus());
  if (tokens < kLong) tokens = all * heads / (kFew * device_cus());
  tokens = tokens < kLeast ? kLeast : tokens;
  int64_t pages = (tokens + ps - 1) / ps;
  if ((all <= kWhole && all <= kWholeOne * batch) || pages >= positions) pages = positions;
  c.job_pages = static_cast<int>(pages < 1 ? 1 : pages);
  c.merge = c.job_pages < positions;
  c.waves = !c.merge && c.qt == 1 && ps % 16 == 0 ? 8 : 4;
  const int64_t jobs = positions / c.job_pages + batch;
  c.jobs = static_cast<int>(jobs);
  c.blocks = jobs * heads;
  return c;
}

int check_extents(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_group, int64_t d, int64_t pages, int64_t ps,
                  int64_t positions) {
  if (batch < 0 || q_heads < 0 || kv_heads < 0 || d < 0 || pages < 0 || ps < 0 || positions < 0)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (head_group < 1 || head_group > INT32_MAX || kv_heads > INT32_MAX || q_heads != kv_heads * head_group)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "query heads (%lld) must equal key heads (%lld) * HEAD_GROUP (%lld)",
                static_cast<long long>(q_heads), static_cast<long long>(kv_heads), static_cast<long long>(head_group));
  if (batch > INT32_MAX / 64 || q_heads > (1 << 20) || ps > INT32_MAX / 64 || positions > INT32_MAX / 64 ||
      positions * ps > int64_t{1} << 40 || pages > INT32_MAX)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}

size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
size_t state_bytes(const Cut &c, int64_t q_heads, int64_t d) {
  if (!c.merge) return 0;
  const size_t rows = static_cast<size_t>(c.jobs) * q_heads;
  return 2 * rounded(rows * 4) + rows * d * 4;
}

template <typename E, int D>
void launch(const Decode &p, const Cut &c, bool uniform, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(c.blocks));
  if (c.qt == 1) {
    if (!uniform)
      mx_decode<E, D, 1, false, 4><<<grid, 4 * kWave, 0, s>>>(p);
    else if (c.waves == 4)
      mx_decode<E, D, 1, true, 4><<<grid, 4 * kWave, 0, s>>>(p);
    else
      mx_decode<E, D, 1, true, 8><<<grid, 8 * kWave, 0, s>>>(p);
  } else {
    if (uniform)
      mx_decode<E, D, 2, true, 4><<<grid, 4 * kWave, 0, s>>>(p);
    else
      mx_decode<E, D, 2, false, 4><<<grid, 4 * kWave, 0, s>>>(p);
  }
  if (!c.merge) return;
  // Few rows: four waves share one's jobs (one sequence of 8000, 32 heads: 12.4 us in all, one wave a row 15.8; 64 sequences, 64
  // heads: 135 with one, 142 with four).
  const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_heads * p.group;
  if (rows < 4 * device_cus())
    mx_decode_merge<E, D, 4><<<dim3(static_cast<unsigned>(rows)), 4 * kWave, 0, s>>>(p);
  else
    mx_decode_merge<E, D, 1><<<dim3(static_cast<unsigned>(rows)), kWave, 0, s>>>(p);
}

template <typename E>
void launch(const Decode &p, const Cut &c, bool uniform, int64_t d, hipStream_t s) {
  switch (d) {
    case 64: return launch<E, 64>(p, c, uniform, s);
    case 96: return launch<E, 96>(p, c, uniform, s);
    case 128: return launch<E, 128>(p, c, uniform, s);
    case 192: return launch<E, 192>(p, c, uniform, s);
    case 256: return launch<E, 256>(p, c, uniform, s);
  }
}

// Whether a tile of 16 keys lies in one page and a lane's place in it within 32 bits; reach: the largest stride of a token.
bool is_uniform(int64_t ps, int64_t reach) { return ps % 16 == 0 && reach < INT32_MAX / 32; }

bool width_ok(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

}  // namespace

int mx_decode_resources(int dtype, int64_t batch, int64_t kv_heads, int64_t group, int64_t d, int64_t ps, int64_t positions,
                        int64_t reach, IntentHipKernelResources *out) {
  if (group < 1 || !width_ok(d)) return fail(INTENT_HIP_ERR_UNSUPPORTED, "mx decode has no head width %lld", static_cast<long long>(d));
  if (int rc = check_extents(batch, kv_heads * group, kv_heads, group, d, 0, ps, positions)) return rc;
  if (ps == 0) ps = 1;                             // a cache without a token
  const Cut c = cut(batch, kv_heads, group, positions, ps);
  const bool uniform = is_uniform(ps, reach);
  char name[64];
  snprintf(name, sizeof(name), "mx_decode<%s,%d,%d,%s,%d>", dtype == INTENT_HIP_F16 ? "f16" : "bf16", static_cast<int>(d), c.qt,
           uniform ? "true" : "false", uniform ? c.waves : 4);
  const auto describe = [&](const void *half, const void *brain) {
    return describe_kernel(dtype == INTENT_HIP_F16 ? half : brain, name, (uniform ? c.waves : 4) * kWave, out);
  };
#define INTENT_HIP_MX_DECODE(W)                                                                                          \
  case W:                                                                                                                \
    if (c.qt == 2)                                                                                                       \
      return uniform ? describe(reinterpret_cast<const void *>(mx_decode<f16_t, W, 2, true, 4>),                         \
                                reinterpret_cast<const void *>(mx_decode<bf16_t, W, 2, true, 4>))                        \
                     : describe(reinterpret_cast<const void *>(mx_decode<f16_t, W, 2, false, 4>),                        \
                                reinterpret_cast<const void *>(mx_decode<bf16_t, W, 2, false, 4>));                      \
    if (!uniform)                                                                                                        \
      return describe(reinterpret_cast<const void *>(mx_decode<f16_t, W, 1, false, 4>),                                  \
                      reinterpret_cast<const void *>(mx_decode<bf16_t, W, 1, false, 4>));                                \
    return c.waves == 4 ? describe(reinterpret_cast<const void *>(mx_decode<f16_t, W, 1, true, 4>),                      \
                                   reinterpret_cast<const void *>(mx_decode<bf16_t, W, 1, true, 4>))                     \
                        : describe(reinterpret_cast<const void *>(mx_decode<f16_t, W, 1, true, 8>),                      \
                                   reinterpret_cast<const void *>(mx_decode<bf16_t, W, 1, true, 8>))
  switch (d) {
    INTENT_HIP_MX_DECODE(64);
    INTENT_HIP_MX_DECODE(96);
    INTENT_HIP_MX_DECODE(128);
    INTENT_HIP_MX_DECODE(192);
    default: INTENT_HIP_MX_DECODE(256);
  }
#undef INTENT_HIP_MX_DECODE
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_paged_gqa_decode_mx_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                              int64_t head_group, int64_t d, int64_t ps, int64_t positions,
                                                              size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (int rc = check_extents(batch, q_heads, kv_heads, head_group, d, 1, ps, positions)) return rc;
  if (batch == 0 || q_heads == 0) return INTENT_HIP_OK;
  if (ps == 0) ps = 1;
  *bytes = state_bytes(cut(batch, kv_heads, head_group, positions, ps), q_heads, d);
  return INTENT_HIP_OK;
}

extern "C" int intent_hip_paged_gqa_decode_mx(int dtype, const void *q, const void *key_cache, const uint8_t *key_exponents,
                                              const void *value_cache, const uint8_t *value_exponents,
                                              const int32_t *page_offsets, const int32_t *page_indices, const int32_t *lengths,
                                              void *output, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                              int64_t head_group, int64_t d, int64_t pages, int64_t ps, int64_t positions,
                                              const int64_t *strides, float scale, void *workspace, size_t workspace_bytes,
                                              void *stream) {
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "decode queries must be F16 or BF16, got %d", dtype);
  if (int rc = check_extents(batch, q_heads, kv_heads, head_group, d, pages, ps, positions)) return rc;
  if (batch == 0 || q_heads == 0) return INTENT_HIP_OK;
  if (!width_ok(d))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "mx decode takes head widths of 64, 96, 128, 192 and 256 (got %lld)",
                static_cast<long long>(d));
  if (ps == 0) pages = 0, ps = 1;                  // as the workspace's size has it; without a page no sequence has a token
  if (q == nullptr || page_offsets == nullptr || lengths == nullptr || output == nullptr || strides == nullptr ||
      (positions > 0 && page_indices == nullptr) ||
      (pages > 0 && (key_cache == nullptr || key_exponents == nullptr || value_cache == nullptr || value_exponents == nullptr)))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  for (int i = 0; i < 22; ++i)
    if (strides[i] < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (strides[2] != 1 || strides[6] != 1 || strides[10] != 1 || strides[14] != 1 || strides[18] != 1 || strides[21] != 1)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows, elements and exponents need unit inner stride");
  if (strides[0] % 8 || strides[1] % 8 || !aligned(q, 16))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "queries must be 16-byte aligned, their strides multiples of 8 elements");
  for (int i = 0; i < 3; ++i)
    if (strides[3 + i] % 16 || strides[11 + i] % 16)
      return fail(INTENT_HIP_ERR_UNSUPPORTED, "cache strides must be multiples of 16 elements");
  if (!aligned(key_cache, 16) || !aligned(value_cache, 16))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "cache elements must be 16-byte aligned");
  const Cut c = cut(batch, kv_heads, head_group, positions, ps);
  if (c.blocks > INT32_MAX / 512) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  const size_t bytes = state_bytes(c, q_heads, d);
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16)))
    return fail(INTENT_HIP_ERR_WORKSPACE, "mx decode needs %zu workspace bytes, 16-byte aligned", bytes);
  Decode p{};
  p.q = static_cast<const uint16_t *>(q);
  p.k = static_cast<const uint8_t *>(key_cache), p.ke = key_exponents;
  p.v = static_cast<const uint8_t *>(value_cache), p.ve = value_exponents;
  p.out = static_cast<uint16_t *>(output);
  p.lengths = lengths;
  p.table = {page_offsets, page_indices, positions, pages, static_cast<int>(ps)};
  for (int i = 0; i < 2; ++i) p.qs[i] = strides[i], p.outs[i] = strides[19 + i];
  for (int i = 0; i < 3; ++i)
    p.ks[i] = strides[3 + i], p.kes[i] = strides[7 + i], p.vs[i] = strides[11 + i], p.ves[i] = strides[15 + i];
  p.batch = static_cast<int>(batch), p.kv_heads = static_cast<int>(kv_heads), p.group = static_cast<int>(head_group);
  p.head_tiles = c.head_tiles, p.job_pages = c.job_pages, p.jobs = c.jobs;
  p.scale = scale;
  if (c.merge) {
    const size_t rows = static_cast<size_t>(c.jobs) * q_heads;
    p.peak = static_cast<float *>(workspace);
    p.total = p.peak + rounded(rows * 4) / 4;
    p.sums = p.total + rounded(rows * 4) / 4;
  }
  hipStream_t s = as_stream(stream);
  const bool uniform = is_uniform(ps, std::max({strides[4], strides[8], strides[12], strides[16]}));
  if (dtype == INTENT_HIP_F16)
    launch<f16_t>(p, c, uniform, d, s);
  else
    launch<bf16_t>(p, c, uniform, d, s);
  return hipPeekAtLastError() != hipSuccess ? launch_status("mx_decode") : INTENT_HIP_OK;
}

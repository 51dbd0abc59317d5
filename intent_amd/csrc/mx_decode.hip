// Attention of one new token per sequence over a paged cache of e4m3 elements with a shared power of two per 32, for gfx950.
// No reference counterpart; the cache and its tables are those of mx_cache.hip.
//
// For query head h of sequence s, over the positions j below lengths[s] that the tables have a page for:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp2(scale * log2(e) * (q . k_j) - peak)        0 where there is none
// Keys and values are taken in the query's type (element * 2^e, one rounding), products are summed in f32, weights enter
// the second product in two parts (the 16-bit rounding of w and of what it left), so its rounding is below f32's.
//
// Design. The page range of a sequence is cut into jobs of `job_pages` pages; job j of the flat list belongs to the last
// sequence s with page_offsets[s] / job_pages + s <= j, which every wave finds by itself, so no table of work is made and
// lengths may change under a captured graph. A workgroup takes a job of one key head, its waves 32 keys in turn; nothing
// but the waves' final states goes through the LDS:
//   * scores: v_mfma_f32_16x16x32 with 16 keys as rows and 16 query heads as columns. The sum over a head's dimensions may
//     run in any order, so lane (r, g) takes dimensions g D / 4 .. of key r as they lie in memory, converts them with its
//     blocks' scales, and the query is laid out to match.
//   * weights: the result leaves keys 4 g .. 4 g + 3 of head r in lane (r, g), which is where the second product wants
//     them: heads as rows, 32 keys (4 of each 16 per lane) summed over.
//   * values: lane (c, g) loads its columns of its own 8 keys and pairs them with v_perm, for 16 columns a product.
//   * the running maximum is raised (and the sums scaled down) only when a score passes it by 2^8, so most steps have no
//     cross-lane move at all; weights up to 2^8 are far inside either type.
// Bound by the cache's bytes.
#include <type_traits>

#include "mx.hpp"

namespace intent_hip {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;
constexpr int kStep = 32;              // keys of a wave's step: two tiles of 16
constexpr float kSlack = 8.0f;

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

// Two values rounded to E, the first in the low half.
template <typename E>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  return static_cast<uint32_t>(from_f32<E>(a).bits) | static_cast<uint32_t>(from_f32<E>(b).bits) << 16;
}
template <typename E>
__device__ __forceinline__ float unpack(uint32_t word, int half) {
  return to_f32(E{static_cast<uint16_t>(half ? word >> 16 : word)});
}

// The sequence of job `job`: sequence s's jobs begin at offsets[s] / job_pages + s.
__device__ __forceinline__ int job_sequence(const Decode &p, int job) {
  const int lane = threadIdx.x & 63;
  int first = 0, count = p.batch;
  while (count > 0) {
    const int step = (count + 63) / 64;
    const int at = (lane + 1) * step;
    const bool past = at <= count && static_cast<int64_t>(p.table.offsets[first + at] / p.job_pages) + first + at <= job;
    const int steps = __popcll(__ballot(past));
    first += steps * step;
    count = step == 1 ? 0 : min(step - 1, count - steps * step);
  }
  return first;
}

// Tokens of sequence s: what its length and its pages both have; none in a cache without a page.
__device__ __forceinline__ int64_t sequence_tokens(const Decode &p, int s) {
  if (p.table.pages == 0) return 0;
  const int64_t pages = static_cast<int64_t>(p.table.offsets[s + 1]) - p.table.offsets[s];
  const int64_t held = (pages < 0 ? 0 : pages) * p.table.ps, length = p.lengths[s];
  return length < held ? (length < 0 ? 0 : length) : held;
}

// How a lane's columns of the values lie: `kWide` runs of 128 columns (8 bytes a lane), then one of 64 (4) and one of 32 (2).
template <int D>
struct Columns {
  static constexpr int kWide = D / 128, kRest = D % 128;
  static constexpr bool kHalf = kRest >= 64, kQuarter = kRest % 64 != 0;
  static constexpr int kRuns = kWide + kHalf + kQuarter;
  static constexpr int kTiles = D / 16;          // products of 16 columns
};

template <int D>
struct Step {                                     // what a lane loads for 32 keys
  uint2 k[2][D / 32];                             // [tile][8 dimensions]
  uint8_t ke[2][D / 32];
  uint2 v[8][Columns<D>::kRuns];                  // [key][run]
  uint8_t ve[8][Columns<D>::kRuns];
};

// kUniform: a tile of 16 keys lies in one page (PS is a multiple of 16), so its address is the wave's.
template <typename E, int D, int QT, bool kUniform>
__global__ __launch_bounds__(kWaves *kWave) void mx_decode(Decode p) {
  using C = Columns<D>;
  constexpr int kChunks = D / 32;
  constexpr int kState = QT * C::kTiles * 4;      // accumulators of a lane
  __shared__ float sums_s[kWaves / 2][kState][kWave];
  __shared__ float peak_s[kWaves][QT * 16], total_s[kWaves][QT * 16];

  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Key heads of a job run on one XCD, close in time: pages with their heads side by side share lines.
  const int n = static_cast<int>(gridDim.x), xcd = static_cast<int>(blockIdx.x) % 8;
  const int item = xcd * (n / 8) + (xcd < n % 8 ? xcd : n % 8) + static_cast<int>(blockIdx.x) / 8;
  const int ht = item % p.head_tiles, kh = item / p.head_tiles % p.kv_heads, job = item / p.head_tiles / p.kv_heads;
  const int s = job_sequence(p, job);
  if (s >= p.batch) return;
  const int64_t tokens = sequence_tokens(p, s);
  const int64_t begin = static_cast<int64_t>(job - (p.table.offsets[s] / p.job_pages + s)) * p.job_pages * p.table.ps;
  int64_t end = begin + static_cast<int64_t>(p.job_pages) * p.table.ps;
  end = end < tokens ? end : tokens;
  // A sequence without a token is its first job's, which writes the 0 itself where no states are merged.
  if (begin < 0 || (begin >= end && (begin > 0 || p.peak != nullptr))) return;
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
  const float c1 = p.scale * kLog2e;
  f32x4_t acc[QT][C::kTiles];
  float peak[QT], total[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    peak[t] = -INFINITY;
    total[t] = 0.0f;
#pragma unroll
    for (int j = 0; j < C::kTiles; ++j) acc[t][j] = f32x4_t{0, 0, 0, 0};
  }

  // Row addresses of a key: page * stride + place * stride. `valid`: how many of a tile's keys count (kUniform), or a bit
  // per key of the lane (bits 0, 1: its keys of the scores; 8 + i: its keys of the values).
  const auto load = [&](Step<D> &x, int64_t p0, int(&valid)[2], unsigned &bits) {
    const auto keys = [&](int u, const uint8_t *k, const uint8_t *ke) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        x.k[u][c] = *reinterpret_cast<const uint2 *>(k + g * (D / 4) + c * 8);
        x.ke[u][c] = ke[(g * (D / 4) + c * 8) / 32];
      }
    };
    const auto values = [&](int i, const uint8_t *v, const uint8_t *ve) {
#pragma unroll
      for (int w = 0; w < C::kWide; ++w) {
        x.v[i][w] = *reinterpret_cast<const uint2 *>(v + w * 128 + r * 8);
        x.ve[i][w] = ve[w * 4 + r / 4];
      }
      if constexpr (C::kHalf) {
        x.v[i][C::kWide].x = *reinterpret_cast<const uint32_t *>(v + C::kWide * 128 + r * 4);
        x.ve[i][C::kWide] = ve[C::kWide * 4 + r / 8];
      }
      if constexpr (C::kQuarter) {
        x.v[i][C::kRuns - 1].x = *reinterpret_cast<const uint16_t *>(v + D - 32 + r * 2);
        x.ve[i][C::kRuns - 1] = ve[D / 32 - 1];
      }
    };
    bits = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if constexpr (kUniform) {
        const int64_t at = p0 + u * 16;
        int64_t page = at < end ? p.table.page(p.table.offsets[s], p.table.offsets[s + 1] - static_cast<int64_t>(p.table.offsets[s]), at / p.table.ps) : -1;
        int64_t slot = at % p.table.ps;
        valid[u] = page < 0 ? 0 : static_cast<int>(end - at < 16 ? end - at : 16);
        if (page < 0) page = slot = 0;             // any 16 rows of the cache: their weights are 0
        keys(u, p.k + page * p.ks[0] + (slot + r) * p.ks[1] + kh * p.ks[2], p.ke + page * p.kes[0] + (slot + r) * p.kes[1] + kh * p.kes[2]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t at_slot = slot + g * 4 + i;
          values(u * 4 + i, p.v + page * p.vs[0] + at_slot * p.vs[1] + kh * p.vs[2], p.ve + page * p.ves[0] + at_slot * p.ves[1] + kh * p.ves[2]);
        }
      } else {
        const auto find = [&](int64_t at, int64_t &page, int64_t &slot) {
          page = at < end ? p.table.page(p.table.offsets[s], p.table.offsets[s + 1] - static_cast<int64_t>(p.table.offsets[s]), at / p.table.ps) : -1;
          slot = at % p.table.ps;
          const bool live = page >= 0;
          if (!live) page = slot = 0;
          return live;
        };
        int64_t page, slot;
        bits |= static_cast<unsigned>(find(p0 + u * 16 + r, page, slot)) << u;
        keys(u, p.k + page * p.ks[0] + slot * p.ks[1] + kh * p.ks[2], p.ke + page * p.kes[0] + slot * p.kes[1] + kh * p.kes[2]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bits |= static_cast<unsigned>(find(p0 + u * 16 + g * 4 + i, page, slot)) << (8 + u * 4 + i);
          values(u * 4 + i, p.v + page * p.vs[0] + slot * p.vs[1] + kh * p.vs[2], p.ve + page * p.ves[0] + slot * p.ves[1] + kh * p.ves[2]);
        }
      }
    }
  };

  const auto fold = [&](Step<D> &x, const int(&valid)[2], unsigned bits) {
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
      live[i] = kUniform ? g * 4 + (i & 3) < valid[i >> 2] : (bits >> (8 + i) & 1) != 0;
      whole = whole && live[i];
    }
    const bool all = kUniform ? valid[0] == 16 && valid[1] == 16 : __all(whole);
    if (!all) {
      // What lies in places without a token has no weight, and must not turn a zero weight into NaN.
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < C::kRuns; ++w)
          if (!live[i]) x.v[i][w] = make_uint2(0, 0), x.ve[i][w] = 127;
    }
    uint4 hi[QT], lo[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float z[8], most = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        z[i] = sc[t][i >> 2][i & 3] * c1;
        if (!all && !live[i]) z[i] = -INFINITY;
        most = fmaxf(most, z[i]);
      }
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
      const float base = peak[t] == -INFINITY ? 0.0f : peak[t];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(z[i] - base);
        total[t] += w[i];
      }
      uint32_t h[4], l[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        h[i] = pack<E>(w[2 * i], w[2 * i + 1]);
        l[i] = pack<E>(w[2 * i] - unpack<E>(h[i], 0), w[2 * i + 1] - unpack<E>(h[i], 1));
      }
      hi[t] = make_uint4(h[0], h[1], h[2], h[3]);
      lo[t] = make_uint4(l[0], l[1], l[2], l[3]);
    }
    // Values: pairs of columns of each key, paired again over the keys.
    const auto columns = [&](int run, int tile, auto upper, auto half) {
      uint32_t pair[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float vs = mx_scale(x.ve[i][run]);
        pair[i] = mx_pair_e4m3<E, half.value>(upper.value ? x.v[i][run].y : x.v[i][run].x, vs);
      }
      uint32_t even[4], odd[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        even[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100);
        odd[i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302);
      }
      const uint4 v0 = make_uint4(even[0], even[1], even[2], even[3]), v1 = make_uint4(odd[0], odd[1], odd[2], odd[3]);
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        acc[t][tile] = mfma<E>(hi[t], v0, acc[t][tile]);
        acc[t][tile + 1] = mfma<E>(hi[t], v1, acc[t][tile + 1]);
        acc[t][tile] = mfma<E>(lo[t], v0, acc[t][tile]);
        acc[t][tile + 1] = mfma<E>(lo[t], v1, acc[t][tile + 1]);
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

  Step<D> x;
  int valid[2];
  unsigned bits;
  for (int64_t p0 = begin + wave * kStep; p0 < end; p0 += kWaves * kStep) {
    load(x, p0, valid, bits);
    fold(x, valid, bits);
  }

  // The waves' states: to the common maximum, then added, two waves at a time.
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    total[t] += __shfl_xor(total[t], 16);
    total[t] += __shfl_xor(total[t], 32);
    if (g == 0) peak_s[wave][t * 16 + r] = peak[t], total_s[wave][t * 16 + r] = total[t];
  }
  __syncthreads();
  float whole_peak[QT], whole_total[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float m = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, peak_s[w][t * 16 + r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float other = peak_s[w][t * 16 + r], part = total_s[w][t * 16 + r];
      // A wave without a score has no weight; one whose weights are NaN keeps them.
      sum += other == -INFINITY ? part : part * __builtin_amdgcn_exp2f(other - m);
    }
    whole_peak[t] = m, whole_total[t] = sum;
    const float shrink = peak[t] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(peak[t] - m);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = __shfl(shrink, g * 4 + i);
#pragma unroll
      for (int j = 0; j < C::kTiles; ++j) acc[t][j][i] *= f;
    }
  }
#pragma unroll
  for (int half = kWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int j = 0; j < C::kTiles; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) sums_s[wave - half][(t * C::kTiles + j) * 4 + i][lane] = acc[t][j][i];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int j = 0; j < C::kTiles; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][j][i] += sums_s[wave][(t * C::kTiles + j) * 4 + i][lane];
    __syncthreads();
  }
  if (wave != 0) return;

  const int q_heads = p.kv_heads * p.group;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (p.peak != nullptr && g == 0 && t * 16 + r < heads) {
      p.peak[static_cast<int64_t>(job) * q_heads + head0 + t * 16 + r] = whole_peak[t];
      p.total[static_cast<int64_t>(job) * q_heads + head0 + t * 16 + r] = whole_total[t];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int head = t * 16 + g * 4 + i;
      const float sum = __shfl(whole_total[t], g * 4 + i);
      if (head >= heads) continue;
      const float share = end > begin ? 1.0f / sum : 0.0f;
      float *state = p.sums + (static_cast<int64_t>(job) * q_heads + head0 + head) * D;
      uint16_t *out = p.out + s * p.outs[0] + (head0 + head) * p.outs[1];
#pragma unroll
      for (int j = 0; j < C::kTiles; ++j) {
        const int wide = j / 8;
        const int column = wide < C::kWide ? wide * 128 + r * 8 + j % 8
                           : C::kHalf && j < C::kWide * 8 + 4 ? C::kWide * 128 + r * 4 + (j - C::kWide * 8)
                                                              : D - 32 + r * 2 + (j - (C::kTiles - 2));
        if (p.peak != nullptr)
          state[column] = acc[t][j][i];
        else
          out[column] = from_f32<E>(acc[t][j][i] * share).bits;
      }
    }
  }
}

// Output rows from the states of a sequence's jobs: one wave per (sequence, query head), lanes over columns.
template <typename E>
__global__ __launch_bounds__(kWaves *kWave) void mx_decode_merge(Decode p, int d) {
  const int q_heads = p.kv_heads * p.group, lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(p.batch) * q_heads) return;
  const int s = static_cast<int>(row / q_heads), head = static_cast<int>(row % q_heads);
  const int64_t tokens = sequence_tokens(p, s), size = static_cast<int64_t>(p.job_pages) * p.table.ps;
  const int64_t first = static_cast<int64_t>(p.table.offsets[s] / p.job_pages) + s;
  int64_t jobs = (tokens + size - 1) / size;
  if (first < 0 || first + jobs > p.jobs) jobs = 0;
  float peak = -INFINITY, total = 0.0f;
  for (int64_t j = 0; j < jobs; ++j) peak = fmaxf(peak, p.peak[(first + j) * q_heads + head]);
  uint16_t *out = p.out + s * p.outs[0] + head * p.outs[1];
  for (int64_t j = 0; j < jobs; ++j) {
    const int64_t at = (first + j) * q_heads + head;
    total += p.peak[at] == -INFINITY ? p.total[at] : p.total[at] * __builtin_amdgcn_exp2f(p.peak[at] - peak);
  }
  const float share = jobs > 0 ? 1.0f / total : 0.0f;
  for (int c = lane; c < d; c += kWave) {
    float sum = 0.0f;
    for (int64_t j = 0; j < jobs; ++j) {
      const int64_t at = (first + j) * q_heads + head;
      const float f = p.peak[at] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(p.peak[at] - peak);
      sum += p.sums[at * d + c] * f;
    }
    out[c] = from_f32<E>(sum * share).bits;
  }
}

// How a call is cut. Jobs of at least 256 tokens, as many as fill the chip a few times over.
struct Cut {
  int job_pages, jobs, head_tiles, qt;
  bool merge;
  int64_t blocks;
};
Cut cut(int64_t batch, int64_t kv_heads, int64_t group, int64_t positions, int64_t ps) {
  Cut c{};
  c.qt = group > 16 ? 2 : 1;
  c.head_tiles = static_cast<int>((group + 16 * c.qt - 1) / (16 * c.qt));
  const int64_t wanted = 4 * device_cus();
  int64_t tokens = positions * ps * kv_heads * c.head_tiles / wanted;
  tokens = tokens < 256 ? 256 : tokens;
  int64_t pages = (tokens + ps - 1) / ps;
  if (pages >= positions) pages = positions;
  c.job_pages = static_cast<int>(pages < 1 ? 1 : pages);
  c.merge = c.job_pages < positions;
  c.jobs = static_cast<int>(c.merge ? positions / c.job_pages + batch : 0);
  c.blocks = (positions / c.job_pages + batch) * kv_heads * c.head_tiles;
  return c;
}

int check_extents(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_group, int64_t d, int64_t pages, int64_t ps,
                  int64_t positions) {
  if (batch < 0 || q_heads < 0 || kv_heads < 0 || d < 0 || pages < 0 || ps < 0 || positions < 0)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (head_group < 1 || head_group > INT32_MAX || kv_heads > INT32_MAX || q_heads != kv_heads * head_group)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "query heads (%lld) must equal key heads (%lld) * HEAD_GROUP (%lld)",
                static_cast<long long>(q_heads), static_cast<long long>(kv_heads), static_cast<long long>(head_group));
  if (batch > INT32_MAX / 64 || q_heads > INT32_MAX / 64 || ps > INT32_MAX / 64 || positions > INT32_MAX / 64 ||
      pages > INT32_MAX)
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
  const dim3 grid(static_cast<unsigned>(c.blocks)), block(kWaves * kWave);
  if (c.qt == 1) {
    if (uniform)
      mx_decode<E, D, 1, true><<<grid, block, 0, s>>>(p);
    else
      mx_decode<E, D, 1, false><<<grid, block, 0, s>>>(p);
  } else {
    if (uniform)
      mx_decode<E, D, 2, true><<<grid, block, 0, s>>>(p);
    else
      mx_decode<E, D, 2, false><<<grid, block, 0, s>>>(p);
  }
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

bool width_ok(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

}  // namespace

int mx_decode_resources(int dtype, int64_t group, int64_t d, IntentHipKernelResources *out) {
  const bool half = dtype == INTENT_HIP_F16, two = group > 16;
#define INTENT_HIP_MX_DECODE(W)                                                                                             \
  case W:                                                                                                                   \
    return half ? two ? describe_kernel(reinterpret_cast<const void *>(mx_decode<f16_t, W, 2, true>), "mx_decode<f16," #W ",2>", kWaves * kWave, out)  \
                      : describe_kernel(reinterpret_cast<const void *>(mx_decode<f16_t, W, 1, true>), "mx_decode<f16," #W ",1>", kWaves * kWave, out)  \
                : two ? describe_kernel(reinterpret_cast<const void *>(mx_decode<bf16_t, W, 2, true>), "mx_decode<bf16," #W ",2>", kWaves * kWave, out) \
                      : describe_kernel(reinterpret_cast<const void *>(mx_decode<bf16_t, W, 1, true>), "mx_decode<bf16," #W ",1>", kWaves * kWave, out)
  switch (d) {
    INTENT_HIP_MX_DECODE(64);
    INTENT_HIP_MX_DECODE(96);
    INTENT_HIP_MX_DECODE(128);
    INTENT_HIP_MX_DECODE(192);
    INTENT_HIP_MX_DECODE(256);
  }
#undef INTENT_HIP_MX_DECODE
  return fail(INTENT_HIP_ERR_UNSUPPORTED, "mx decode has no head width %lld", static_cast<long long>(d));
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
  if (pages == 0 || ps == 0) pages = 0, ps = 1;
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
  if (c.blocks > INT32_MAX / 256) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
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
  const bool uniform = ps % 16 == 0;
  if (dtype == INTENT_HIP_F16)
    launch<f16_t>(p, c, uniform, d, s);
  else
    launch<bf16_t>(p, c, uniform, d, s);
  if (hipPeekAtLastError() != hipSuccess) return launch_status("mx_decode");
  if (!c.merge) return INTENT_HIP_OK;
  const dim3 grid(static_cast<unsigned>((batch * q_heads + kWaves - 1) / kWaves));
  if (dtype == INTENT_HIP_F16)
    mx_decode_merge<f16_t><<<grid, kWaves * kWave, 0, s>>>(p, static_cast<int>(d));
  else
    mx_decode_merge<bf16_t><<<grid, kWaves * kWave, 0, s>>>(p, static_cast<int>(d));
  return hipPeekAtLastError() != hipSuccess ? launch_status("mx_decode_merge") : INTENT_HIP_OK;
}

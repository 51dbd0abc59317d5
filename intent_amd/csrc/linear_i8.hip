// Products of 8-bit integers with a scale for each row of x and each row of the weight, for gfx950. No reference counterpart.
//
//   y[m, n] = (sum_k x[m, k] w[n, k]) * x_scale[m] * w_scale[n] + bias[n]
// The sums are int32 and exact (K below 2^17, so they cannot leave 32 bits): no order, cut or tile changes them, and a result is rounded
// once to f32 by each factor and the bias, and once to its type.
//
// Design. x [M, K] and w [N, K] both lie along K, as the matrix instructions take them. Products are formed transposed, weight rows as
// rows, so that a lane ends with consecutive columns of one row of y. Few rows are bound by the weights' bytes, many by the matrix pipe.
//   * linear_few, up to 16 rows: K over the 16 waves of a workgroup, weights and x straight to registers. 1 x 14336 x 4096 14.0 us (4.2
//     TB/s), 1 x 4096 x 14336 12.7 (4.6), 16 rows 17.9 and 18.0: what a launch's start and end leave of a burst of two to four steps a wave.
//   * linear_tiles, 64 or 128 x 128 results: x through the LDS, weights to registers, K over several workgroups. 32 x 4096 x 14336 20 us, of
//     which the fold is 4; 128 x 14336 x 4096 30.5, 256 40.
//   * linear_big, 256 or 128 x 256 results of four waves: both operands through the LDS. 4096 x 14336 x 4096 247 us, 8192^3 510 (2160
//     TOP/s), 1024 x 14336 x 4096 73, 512 51; 1021 x 4096 x 14336 97, K in two parts, 11 of them the fold. The matrix pipe is busy in 52%
//     of the cycles at 4096 x 14336 x 4096, in 64% at 8192^3 (a library's product without scales: 72%), at clocks that fall to 1.6 .. 1.75 GHz under
//     this load; what the other cycles wait for has not been found.
#include <stdio.h>

#include <type_traits>

#include "stages.hpp"

namespace intent_hip {
namespace {

constexpr int kUnit = 16;              // bytes of a lane's load; K is a multiple of it
constexpr int kFewWaves = 16;

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

struct Linear {
  const int8_t *x, *w;
  const float *xs, *ws, *bias;         // bias: null for none
  uint16_t *y;
  int32_t *sums;                       // [parts][m][pitch] where K is divided, pitch: n in whole fours
  int64_t ldx, ldw, ldy;
  int m, n, pitch, units;              // units: K / 16
  int m_tiles, n_tiles, parts, stages; // tiles; stages of a part (or of a wave)
  int full;                            // linear_big: tiles of I = 4
  int wide;                            // y takes stores of so many elements (1, 4 or 8)
};

__device__ __forceinline__ i32x4_t mfma(uint4 a, uint4 b, i32x4_t c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float scaled(const Linear &p, int sum, float xs, int n) {
  const float y = static_cast<float>(sum) * xs * p.ws[n];
  return p.bias != nullptr ? y + p.bias[n] : y;
}

// kCount consecutive results of one row of y, from column n on.
template <typename E, int kCount>
__device__ __forceinline__ void store(const Linear &p, int m, int n, const int (&sum)[kCount]) {
  if (m >= p.m || n >= p.n) return;
  uint16_t *y = p.y + m * p.ldy + n;
  const float xs = p.xs[m];
  if (p.wide >= 4) {
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
      if (n + i >= p.n) break;
      uint32_t words[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        words[j] = from_f32<E>(scaled(p, sum[i + 2 * j], xs, n + i + 2 * j)).bits |
                   static_cast<uint32_t>(from_f32<E>(scaled(p, sum[i + 2 * j + 1], xs, n + i + 2 * j + 1)).bits) << 16;
      *reinterpret_cast<uint2 *>(y + i) = make_uint2(words[0], words[1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      if (n + i < p.n) y[i] = from_f32<E>(scaled(p, sum[i], xs, n + i)).bits;
  }
}

// ---------------------------------------------------------------- few rows of x
// A wave's word of its row of 16 lanes, from lane kFirst on: four of them.
template <int kFirst>
__device__ __forceinline__ uint4 words_of_row(uint32_t own) {
  const int v = static_cast<int>(own);
  return make_uint4(__builtin_amdgcn_update_dpp(0, v, 0x150 + kFirst, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, v, 0x151 + kFirst, 0xF, 0xF, false),
                    __builtin_amdgcn_update_dpp(0, v, 0x152 + kFirst, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, v, 0x153 + kFirst, 0xF, 0xF, false));
}

// Up to 16 rows of x by 16 NT weight rows a workgroup; its 16 waves take a run of K each and add their sums through the LDS. A step is
// 128 bytes of K, of which lane (r, g) takes 32 of weight row r and, of its row of x, the same; kAhead steps are on their way at once.
// Columns of the product behind the rows of x are never stored, so their lanes read any row. kOne: x is one row, whose 32 bytes of a
// lane are spread over the 16 lanes that want them, eight words of which every lane takes by moves within its row of lanes.
template <typename E, int NT, bool kOne>
__global__ __launch_bounds__(kFewWaves *kWave) void linear_few(Linear p) {
  constexpr int kAhead = NT == 1 ? 4 : 2, kSums = NT * 4;
  __shared__ int sums[kFewWaves][kSums][kWave];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = grid_block() * 16 * NT;
  if (n0 >= p.n) return;
  const int8_t *w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)         // rows behind the last are not stored
    w[j] = p.w + static_cast<int64_t>(min(n0 + r * NT + j, p.n - 1)) * p.ldw + g * 32;
  const int8_t *x = kOne ? p.x + g * 32 + (r & 7) * 4 : p.x + min(r, p.m - 1) * p.ldx + g * 32;
  i32x4_t acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = i32x4_t{0, 0, 0, 0};
  const int first = min(wave * p.stages * 8, p.units), last = min(first + p.stages * 8, p.units);
  for (int u0 = first; u0 < last; u0 += kAhead * 8) {
    uint4 raw[kAhead][NT][2], v[kAhead][2];
    uint32_t one[kAhead];
    const bool whole = u0 + kAhead * 8 <= last;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int u = u0 + i * 8 + g * 2;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          raw[i][j][c] = make_uint4(0, 0, 0, 0);
          if (whole || u + c < last) raw[i][j][c] = *reinterpret_cast<const uint4 *>(w[j] + (u0 + i * 8) * kUnit + c * kUnit);
        }
      if constexpr (kOne) {
        one[i] = 0;
        if (whole || u + ((r >> 2) & 1) < last) one[i] = *reinterpret_cast<const uint32_t *>(x + (u0 + i * 8) * kUnit);
      } else {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          v[i][c] = make_uint4(0, 0, 0, 0);
          if (whole || u + c < last) v[i][c] = *reinterpret_cast<const uint4 *>(x + (u0 + i * 8) * kUnit + c * kUnit);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if constexpr (kOne) v[i][0] = words_of_row<0>(one[i]), v[i][1] = words_of_row<4>(one[i]);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[j] = mfma(raw[i][j][c], v[i][c], acc[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][i * NT + j][lane] = acc[j][i];
  __syncthreads();
  if (wave >= kSums || r >= p.m) return;
  int total = 0;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) total += sums[i][wave][lane];
  const int n = n0 + g * kSums + wave;
  if (n < p.n) p.y[r * p.ldy + n] = from_f32<E>(scaled(p, total, p.xs[r], n)).bits;
}

// ---------------------------------------------------------------- tiles whose weights go to registers
// 16 MT rows of x by 16 NT weight rows for each of W waves; S stages of B bytes of K are on their way or in use. x passes through the
// LDS (unit u of row r at another place for each of 16 rows, so that a read's rows lie in different banks), weights go straight to
// registers: no wave needs another's. Each stage has an LDS array of its own, and the loop is unrolled by S: the compiler then knows
// which loads into the LDS a read has to wait for.
template <typename E, int MT, int NT, int S, int W, int B>
__global__ __launch_bounds__(W *kWave, 2) void linear_tiles(Linear p) {
  constexpr int kRows = 16 * MT, kRowUnits = B / kUnit, kUnits = kRows * kRowUnits, kLoads = kUnits / (W * kWave);
  constexpr int kOwn = kRowUnits / 4;                  // units of a stage that a lane multiplies
  constexpr int kIssued = kLoads + NT * kOwn;          // loads of a wave per stage, always as many
  static_assert(S == 4 && kLoads >= 1, "one LDS array per stage");
  __shared__ uint4 x_0[kUnits], x_1[kUnits], x_2[kUnits], x_3[kUnits];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.m_tiles * p.n_tiles;
  int tile = xcd_tile(grid_block(), tiles * p.parts);
  if (tile < 0) return;
  const int part = tile / tiles;
  tile -= part * tiles;
  const int m0 = tile % p.m_tiles * kRows, n0 = (tile / p.m_tiles * W + wave) * 16 * NT;
  const int first = min(part * p.stages * kRowUnits, p.units), last = min(p.units, first + p.stages * kRowUnits);     // units of this part
  const int stages = (last - first + kRowUnits - 1) / kRowUnits;
  static_assert(kRowUnits == 8, "the 16 rows of a read lie in different banks");
  const auto place = [](int row) { return (row >> 1) & 7; };
  const int8_t *from[kLoads];
  int unit[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int slot = (i * W + wave) * kWave + lane, row = slot / kRowUnits;
    unit[i] = slot % kRowUnits ^ place(row);
    from[i] = p.x + static_cast<int64_t>(min(m0 + row, p.m - 1)) * p.ldx + unit[i] * kUnit;      // rows behind the last are not stored
  }
  const int8_t *w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) w[j] = p.w + static_cast<int64_t>(min(n0 + r * NT + j, p.n - 1)) * p.ldw;
  uint4 raw[S][NT][kOwn];
  const auto array = [&](int u) -> uint4 * { return u == 0 ? x_0 : u == 1 ? x_1 : u == 2 ? x_2 : x_3; };
  const auto issue = [&](int t, int set) {             // stage t (the last again behind it) into a set
    const int u0 = first + min(t, stages - 1) * kRowUnits;
    const bool whole = u0 + kRowUnits <= last;
    uint4 *stage = array(set);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int8_t *src = whole || u0 + unit[i] < last ? from[i] + static_cast<int64_t>(u0) * kUnit : reinterpret_cast<const int8_t *>(&kZeroUnit);
      __builtin_amdgcn_global_load_lds(src, (lds_void_t *)(stage + (i * W + wave) * kWave), 16, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < kOwn; ++c)                   // behind K any: x is 0 there
        raw[set][j][c] = *reinterpret_cast<const uint4 *>(w[j] + static_cast<int64_t>(min(u0 + g * kOwn + c, last - 1)) * kUnit);
  };
  i32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = i32x4_t{0, 0, 0, 0};
  if (stages > 0) {
#pragma unroll
    for (int u = 0; u < S - 1; ++u) issue(u, u);
    for (int t0 = 0; t0 < stages; t0 += S) {
#pragma unroll
      for (int u = 0; u < S; ++u) {
        if (t0 + u >= stages) break;
        INTENT_WAIT_VMCNT((S - 2) * kIssued);          // this wave's loads of the stage have come
        stage_barrier();                               // everybody's have, and nobody reads the set that is filled next
        issue(t0 + u + S - 1, (u + S - 1) % S);
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
          uint4 v[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i) v[i] = array(u)[(i * 16 + r) * kRowUnits + ((g * kOwn + c) ^ place(r))];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mfma(raw[u][j][c], v[i], acc[i][j]);
        }
      }
    }
    INTENT_WAIT_VMCNT(0);                              // nothing is on its way into the LDS of an ended workgroup
  }
  // A lane's results: row m0 + 16 i + r of y, columns n0 + (4 g + k) NT + j.
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    int row[4 * NT];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < NT; ++j) row[k * NT + j] = acc[i][j][k];
    const int m = m0 + i * 16 + r, n = n0 + g * 4 * NT;
    if (p.parts == 1) {
      store<E>(p, m, n, row);
    } else if (m < p.m) {
      int32_t *to = p.sums + (static_cast<int64_t>(part) * p.m + m) * p.pitch + n;
#pragma unroll
      for (int k = 0; k < 4 * NT; k += 4)
        if (n + k < p.pitch) *reinterpret_cast<i32x4_t *>(to + k) = i32x4_t{row[k], row[k + 1], row[k + 2], row[k + 3]};
    }
  }
}

// y from the parts' sums, four columns a thread.
template <typename E>
__global__ __launch_bounds__(256) void linear_fold(Linear p) {
  const int64_t all = static_cast<int64_t>(p.m) * p.pitch, at = (static_cast<int64_t>(grid_block()) * 256 + threadIdx.x) * 4;
  if (at >= all) return;
  i32x4_t total = {0, 0, 0, 0};
#pragma unroll 8
  for (int i = 0; i < p.parts; ++i) total += *reinterpret_cast<const i32x4_t *>(p.sums + i * all + at);
  const int m = static_cast<int>(at / p.pitch), n = static_cast<int>(at - static_cast<int64_t>(m) * p.pitch);
  const int sum[4] = {total[0], total[1], total[2], total[3]};
  store<E>(p, m, n, sum);
}

// ---------------------------------------------------------------- large tiles, both operands through the LDS
// 64 I rows of x by 256 weight rows, 4 waves of 32 I x 128 = I x 4 products of 32 x 32 x 32 (I = 4: a byte read from the LDS meets 128
// others). A stage is 64 bytes of K of both; stages arrive by loads into the LDS, as many as it holds. A wave has its SIMD to itself and
// hides its reads behind its own products: while the 4 I products of half a stage run, the operands of the next half are read.
// Whole rounds of tiles over the CUs have I = 4; where at most half a round is left, or less than that is all there is, that is done by
// twice as many tiles of I = 2 (4096 x 14336 x 4096, three rounds and a half: 273 us without).
constexpr int kBN = 256, kBK = 64, kBigWaves = 4, kBigThreads = kBigWaves * kWave;
constexpr int kGroupM = 8;             // tiles of x that share a walk along the weight rows
constexpr int big_rows(int i) { return 64 * i; }
constexpr int big_stages(int i) { return i == 4 ? 5 : 6; }
constexpr int kBigUnits = big_stages(4) * (big_rows(4) + kBN) * kBK / kUnit;      // 160 KB
static_assert(big_stages(2) * (big_rows(2) + kBN) * kBK / kUnit <= kBigUnits, "all kinds of tiles share one array");

// Tiles in groups of kGroupM rows of tiles, walked column by column: those that run at one time share rows and columns.
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int &tm, int &tn) {
  const int per_group = kGroupM * n_tiles, group = t / per_group, first = group * kGroupM;
  const int rows = min(m_tiles - first, kGroupM), in = t - group * per_group;
  tm = first + in % rows, tn = in / rows;
}

// The tile from row m0 of x and weight row n0 on, over the part of K that is `part` if kDivided.
template <typename E, int I, bool kDivided>
__device__ __forceinline__ void big_tile(const Linear &p, int m0, int n0, int part, uint4 *lds) {
  constexpr int kStages = big_stages(I), kXUnits = big_rows(I) * kBK / kUnit, kWUnits = kBN * kBK / kUnit, kStageUnits = kXUnits + kWUnits;
  constexpr int kXLoads = kXUnits / kBigThreads, kWLoads = kWUnits / kBigThreads, kLoads = kXLoads + kWLoads, kReads = I + 4, kProducts = 4 * I;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int first = kDivided ? part * p.stages * 4 : 0, units = kDivided ? max(0, min(p.units - first, p.stages * 4)) : p.units;
  // Unit c of row r lies at place c ^ (r / 4) % 4 of its four.
  const int8_t *src[kLoads];                           // of x, then of the weight
  int unit[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int slot = (wave * (i < kXLoads ? kXLoads : kWLoads) + (i < kXLoads ? i : i - kXLoads)) * kWave + lane, row = slot >> 2;
    unit[i] = (slot & 3) ^ ((row >> 2) & 3);
    src[i] = (i < kXLoads ? p.x + static_cast<int64_t>(min(m0 + row, p.m - 1)) * p.ldx : p.w + static_cast<int64_t>(min(n0 + row, p.n - 1)) * p.ldw) + (unit[i] + first) * kUnit;
  }
  const auto place = [&](int i) { return i < kXLoads ? (wave * kXLoads + i) * kWave : kXUnits + (wave * kWLoads + i - kXLoads) * kWave; };
  const int stages = units / 4, rest = units % 4;      // whole ones; units behind them
  const auto issue = [&](int t, int i) {               // load i of stage t (the last again behind it, so that as many are always on their way)
    const int64_t k0 = static_cast<int64_t>(min(t, stages - 1)) * kBK;
    __builtin_amdgcn_global_load_lds(src[i] + k0, (lds_void_t *)(lds + (t % kStages) * kStageUnits + place(i)), 16, 0, 0);
  };
  i32x16_t acc[I][4];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  const int row = lane & 31, half = lane >> 5, turn = (row >> 2) & 3;
  i32x4_t xf[2][I], wf[2][4];
  const auto read = [&](int t, int k, int i) {         // of half k of stage t: operand i of the weight, then of x
    const uint4 *sx = lds + (t % kStages) * kStageUnits, *sw = sx + kXUnits;
    const int at = ((i < 4 ? i : i - 4) * 32 + row) * 4 + ((k * 2 + half) ^ turn);
    if (i < 4)
      wf[k][i] = __builtin_bit_cast(i32x4_t, sw[wn * 128 * 4 + at]);
    else
      xf[k][i - 4] = __builtin_bit_cast(i32x4_t, sx[wm * 32 * I * 4 + at]);
  };
  const auto multiply = [&](int k, int at) {           // product `at` of half k
    acc[at / 4][at % 4] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[k][at % 4], xf[k][at / 4], acc[at / 4][at % 4], 0, 0, 0);
  };
  constexpr int kEach = kProducts / 8;                 // products behind each of eight reads (and loads)
  if (stages > 0) {
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) issue(t, i);
    INTENT_WAIT_VMCNT((kStages - 2) * kLoads);
    stage_barrier();
#pragma unroll
    for (int i = 0; i < kReads; ++i) read(0, 0, i);
    for (int t = 0; t < stages; ++t) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {                    // a read and some products at a time, in this order
        if (i < kReads) read(t, 1, i);
#pragma unroll
        for (int j = 0; j < kEach; ++j) multiply(0, kEach * i + j);
        __builtin_amdgcn_sched_barrier(0);
      }
      INTENT_WAIT_VMCNT((kStages - 3) * kLoads);       // this wave's loads of the next stage have come
      stage_barrier();                                 // everybody's have, and everybody has read the stage that is filled next
#pragma unroll
      for (int i = 0; i < 8; ++i) {                    // and a load
        if (i < kReads) read(t + 1, 0, i);             // behind the last stage: the last again, never used
        if (i < kLoads) issue(t + kStages - 1, i);
#pragma unroll
        for (int j = 0; j < kEach; ++j) multiply(1, kEach * i + j);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    INTENT_WAIT_VMCNT(0);                              // nothing is on its way into the LDS of an ended workgroup
  }
  if (rest > 0) {                                      // the end of K, zeros behind it
    stage_barrier();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int8_t *const from = unit[i] < rest ? src[i] + static_cast<int64_t>(stages) * kBK : reinterpret_cast<const int8_t *>(&kZeroUnit);
      __builtin_amdgcn_global_load_lds(from, (lds_void_t *)(lds + place(i)), 16, 0, 0);
    }
    INTENT_WAIT_VMCNT(0);
    stage_barrier();
#pragma unroll
    for (int i = 0; i < 2 * kReads; ++i) read(0, i / kReads, i % kReads);
#pragma unroll
    for (int i = 0; i < 2 * kProducts; ++i) multiply(i / kProducts, i % kProducts);
  }
  // acc[i][j][4 q + e] is row 32 i + (lane % 32) of x with weight row 32 j + 8 q + 4 half + e.
  if constexpr (kDivided) {
    int m = m0 + wm * I * 32 + row;
    const int n = n0 + wn * 128 + 4 * half;
    int32_t *to = p.sums + (static_cast<int64_t>(part) * p.m + m) * p.pitch + n;
#pragma unroll
    for (int i = 0; i < I; ++i, m += 32, to += static_cast<int64_t>(32) * p.pitch) {
      if (m >= p.m) break;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + j * 32 + 8 * q < p.pitch)
            *reinterpret_cast<i32x4_t *>(to + j * 32 + 8 * q) = i32x4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    }
    return;
  }
  // The results of 32 rows go through the wave's own part of the LDS, from where whole rows of 128 are written (straight from registers, 8 bytes a lane and row with a load of
  // their scales: 39 us a tile, as long as K = 2700 takes).
  __syncthreads();
  constexpr int kRowUnits = 17;                        // 128 results and 16 bytes, so that rows lie in different banks
  float *const scales = reinterpret_cast<float *>(lds + kBigWaves * 32 * kRowUnits);      // of the tile's weight rows, then their biases
  for (int i = tid; i < kBN; i += kBigThreads) {
    const int n = min(n0 + i, p.n - 1);
    scales[i] = p.ws[n], scales[kBN + i] = p.bias != nullptr ? p.bias[n] : 0.0f;
  }
  float xs[I];
#pragma unroll
  for (int i = 0; i < I; ++i) xs[i] = p.xs[min(m0 + (wm * I + i) * 32 + row, p.m - 1)];
  __syncthreads();
  uint4 *const own = lds + wave * 32 * kRowUnits;
#pragma unroll
  for (int i = 0; i < I; ++i) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = wn * 128 + j * 32 + 8 * q + 4 * half;
        const float4 ws = *reinterpret_cast<const float4 *>(scales + at), bias = *reinterpret_cast<const float4 *>(scales + kBN + at);
        const auto result = [&](int e, float w, float b) {
          const float y = static_cast<float>(acc[i][j][4 * q + e]) * xs[i] * w;
          return static_cast<uint32_t>(from_f32<E>(p.bias != nullptr ? y + b : y).bits);
        };
        reinterpret_cast<uint2 *>(own + row * kRowUnits)[j * 8 + 2 * q + half] =
            make_uint2(result(0, ws.x, bias.x) | result(1, ws.y, bias.y) << 16, result(2, ws.z, bias.z) | result(3, ws.w, bias.w) << 16);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int of = k * 4 + (lane >> 4), m = m0 + (wm * I + i) * 32 + of, n = n0 + wn * 128 + (lane & 15) * 8;
      const uint4 v = own[of * kRowUnits + (lane & 15)];
      if (m >= p.m || n >= p.n) continue;
      uint16_t *const y = p.y + m * p.ldy + n;
      if (p.wide == 8) {
        *reinterpret_cast<uint4 *>(y) = v;
      } else {
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < p.n) y[e] = static_cast<uint16_t>(words[e / 2] >> (16 * (e & 1)));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// full: tiles of I = 4, the first of the order of tiles; the others are halved.
template <typename E>
__global__ __launch_bounds__(kBigThreads, 1) void linear_big(Linear p) {
  __shared__ uint4 lds[kBigUnits];
  const int tiles = p.m_tiles * p.n_tiles, full_blocks = (p.full + 7) / 8 * 8;
  int tm, tn;
  if (const int block = grid_block(); block < full_blocks) {
    const int tile = xcd_tile(block, p.full);
    if (tile < 0) return;
    tile_at(tile, p.m_tiles, p.n_tiles, tm, tn);
    big_tile<E, 4, false>(p, tm * big_rows(4), tn * kBN, 0, lds);
  } else {
    const int tile = xcd_tile(block - full_blocks, 2 * (tiles - p.full));
    if (tile < 0) return;
    tile_at(p.full + tile / 2, p.m_tiles, p.n_tiles, tm, tn);
    const int m0 = tm * big_rows(4) + tile % 2 * big_rows(2);
    if (m0 < p.m) big_tile<E, 2, false>(p, m0, tn * kBN, 0, lds);
  }
}

// Tiles of one kind over parts of K, one part after the other. A kernel of its own: with both ends in one registers spilled, and 4096 x
// 4096 x 4096 took 80 us for 77.
template <typename E, int I>
__global__ __launch_bounds__(kBigThreads, 1) void linear_big_part(Linear p) {
  __shared__ uint4 lds[kBigUnits];
  const int job = xcd_tile(grid_block(), p.m_tiles * p.n_tiles * p.parts);
  if (job < 0) return;
  int tm, tn;
  tile_at(job % (p.m_tiles * p.n_tiles), p.m_tiles, p.n_tiles, tm, tn);
  big_tile<E, I, true>(p, tm * big_rows(I), tn * kBN, job / (p.m_tiles * p.n_tiles), lds);
}

// ---------------------------------------------------------------- which kernel
// How a product is cut. mt = 0: linear_few; 1: of one row; 16: linear_big, of nt = 2 tiles of I = 2 alone, of 4 tiles of I = 4, but for what
// at most half fills the last round of an undivided K.
struct Cut {
  int mt, nt, parts;
};
int big_full(int tiles, const Cut &c) {
  const int left = tiles % device_cus();
  return c.nt == 2 ? 0 : 2 * left <= device_cus() ? tiles - left : tiles;
}
constexpr int kTileWaves = 4, kTileStage = 128;

// linear_few for up to 16 rows (tiles: 4 x 14336 x 4096 19.5 us for 16.0, 16 rows 20.0 for 18.2, 16 x 4096 x 4096 10.5 for 7.9), NT = 2 where
// that leaves a workgroup for three CUs in four at least (1 x 14336 x 4096 14.5 us, NT = 1 16.3; 1 x 4096 x 14336 19.3 and 12.8; 1 x 8192 x
// 4096 9.5 and 10.0). Otherwise by an estimate from what the tiles measured:
// us that a round of workgroups takes besides its stages, a stage (of 128 bytes of K) of a workgroup that has a CU for itself and of each of
// several on a CU, and what writing, reading and adding the parts' sums takes. Large tiles have a CU each, whole ones and halves in rounds
// of their own. Over M of 17 to 1024 and three N x K the choice was within a tenth of the best of all tiles and parts.
Cut cut(int64_t m, int64_t n, int64_t k) {
  const int64_t cus = device_cus();
  if (m <= 16) return {m == 1 ? 1 : 0, n >= 24 * cus ? 2 : 1, 1};
  constexpr struct { int mt, nt; float round, alone, shared; } kKinds[] = {{4, 2, 5.0f, 0.62f, 0.61f}, {8, 2, 5.0f, 1.0f, 0.85f}};
  constexpr float kFullRound = 9.0f, kFullStage = 1.84f, kHalfRound = 5.0f, kHalfStage = 1.14f, kStart = 5.0f;
  const int64_t stages = (k + kTileStage - 1) / kTileStage, big = (m + big_rows(4) - 1) / big_rows(4) * ((n + kBN - 1) / kBN);
  const int64_t halves = (m + big_rows(2) - 1) / big_rows(2) * ((n + kBN - 1) / kBN);
  Cut best{};
  float least = 0.0f;
  const auto consider = [&](Cut c, float us) {
    if (c.parts > 1) us += 3.0f + static_cast<float>(c.parts) * static_cast<float>(m) * static_cast<float>(n) * 2.1e-6f;
    if (best.parts == 0 || us < least) best = c, least = us;
  };
  for (int parts = 1; parts <= 16 && (parts == 1 || parts * 4 <= stages); ++parts) {
    const float of_part = static_cast<float>((stages + parts - 1) / parts);
    for (const auto &kind : kKinds) {
      const int64_t tiles = (m + 16 * kind.mt - 1) / (16 * kind.mt) * ((n + 16 * kTileWaves * kind.nt - 1) / (16 * kTileWaves * kind.nt));
      const float on_one = static_cast<float>((tiles * parts + cus - 1) / cus), shared = kind.shared * on_one;
      consider({kind.mt, kind.nt, parts}, kind.round + of_part * (kind.alone > shared ? kind.alone : shared));
    }
    const float half = kHalfRound + of_part * kHalfStage, whole = kFullRound + of_part * kFullStage;
    consider({16, 2, parts}, kStart + static_cast<float>((halves * parts + cus - 1) / cus) * half);
    if (parts > 1) {
      consider({16, 4, parts}, kStart + static_cast<float>((big * parts + cus - 1) / cus) * whole);
    } else {
      const bool split = 2 * (big % cus) <= cus;
      consider({16, 4, 1}, kStart + static_cast<float>(split ? big / cus : (big + cus - 1) / cus) * whole + (split && big % cus ? half : 0.0f));
    }
  }
  return best;
}

// f with the kernel of a cut, its name and its waves.
template <typename E, typename F>
int with_kernel(const Cut &c, F f) {
  if (c.mt == 0) return c.nt == 1 ? f(linear_few<E, 1, false>, "linear_few", kFewWaves) : f(linear_few<E, 2, false>, "linear_few", kFewWaves);
  if (c.mt == 1) return c.nt == 1 ? f(linear_few<E, 1, true>, "linear_few", kFewWaves) : f(linear_few<E, 2, true>, "linear_few", kFewWaves);
  if (c.mt == 16 && c.parts == 1) return f(linear_big<E>, "linear_big", kBigThreads / kWave);
  if (c.mt == 16) return f(c.nt == 2 ? linear_big_part<E, 2> : linear_big_part<E, 4>, "linear_big_part", kBigThreads / kWave);
  return c.mt == 4 ? f(linear_tiles<E, 4, 2, 4, kTileWaves, kTileStage>, "linear_tiles", kTileWaves)
                   : f(linear_tiles<E, 8, 2, 4, kTileWaves, kTileStage>, "linear_tiles", kTileWaves);
}

template <typename E>
void launch(Linear p, const Cut &c, hipStream_t s) {
  p.parts = c.parts;
  with_kernel<E>(c, [&](void (*kernel)(Linear), const char *, int waves) {
    dim3 grid;
    if (c.mt <= 1) {
      p.stages = ((p.units + 7) / 8 + waves - 1) / waves;
      grid = tile_grid((p.n + 16 * c.nt - 1) / (16 * c.nt), 1);
    } else if (c.mt == 16) {
      p.stages = ((p.units + 3) / 4 + c.parts - 1) / c.parts;
      const int rows = c.parts == 1 ? big_rows(4) : big_rows(c.nt);
      p.m_tiles = (p.m + rows - 1) / rows, p.n_tiles = (p.n + kBN - 1) / kBN;
      const int tiles = p.m_tiles * p.n_tiles;
      if (c.parts == 1) {
        p.full = big_full(tiles, c);
        grid = tile_grid((p.full + 7) / 8 * 8 + (2 * static_cast<int64_t>(tiles - p.full) + 7) / 8 * 8, 1);
      } else {
        grid = tile_grid(static_cast<int64_t>(tiles) * c.parts, 1);
      }
    } else {
      constexpr int of_stage = kTileStage / kUnit;
      p.stages = ((p.units + of_stage - 1) / of_stage + c.parts - 1) / c.parts;
      p.m_tiles = (p.m + 16 * c.mt - 1) / (16 * c.mt), p.n_tiles = (p.n + 16 * waves * c.nt - 1) / (16 * waves * c.nt);
      grid = tile_grid(static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.parts, 1);
    }
    kernel<<<grid, waves * kWave, 0, s>>>(p);
    return 0;
  });
  if (c.parts == 1) return;
  linear_fold<E><<<tile_grid((static_cast<int64_t>(p.m) * p.pitch / 4 + 255) / 256, 1), 256, 0, s>>>(p);
}

size_t sums_bytes(const Cut &c, int64_t m, int64_t n) {
  return c.parts > 1 ? static_cast<size_t>(c.parts) * m * ((n + 3) / 4 * 4) * sizeof(int32_t) : 0;
}

int check(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (k % kUnit) return fail(INTENT_HIP_ERR_UNSUPPORTED, "linear_i8 takes K in multiples of %d (got %lld)", kUnit, static_cast<long long>(k));
  if (k >= 1 << 17) return fail(INTENT_HIP_ERR_UNSUPPORTED, "linear_i8 sums K below 131072 in 32 bits (got %lld)", static_cast<long long>(k));
  if (m > (1 << 20) || n > (1 << 24) || m * n > (int64_t{1} << 40)) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}

}  // namespace

int linear_i8_resources(int dtype, int64_t m, int64_t n, int64_t k, IntentHipKernelResources *out) {
  if (int rc = check(m, n, k)) return rc;
  const Cut c = cut(m, n, k);
  const auto describe = [&](void (*kernel)(Linear), const char *which, int waves) {
    char name[64];
    snprintf(name, sizeof(name), "linear_i8 %s<%s,%d,%d>", which, dtype == INTENT_HIP_F16 ? "f16" : "bf16", c.mt, c.nt);
    return describe_kernel(reinterpret_cast<const void *>(kernel), name, waves * kWave, out);
  };
  return dtype == INTENT_HIP_F16 ? with_kernel<f16_t>(c, describe) : with_kernel<bf16_t>(c, describe);
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_linear_i8_workspace_bytes(int64_t m, int64_t n, int64_t k, size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (int rc = check(m, n, k)) return rc;
  if (m == 0 || n == 0) return INTENT_HIP_OK;
  *bytes = sums_bytes(cut(m, n, k), m, n);
  return INTENT_HIP_OK;
}

extern "C" int intent_hip_linear_i8(int dtype, const int8_t *x, const int8_t *weight, const float *x_scales, const float *weight_scales,
                                    const float *bias, void *y, int64_t m, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int64_t ldy,
                                    void *workspace, size_t workspace_bytes, void *stream) {
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "linear_i8 dtype must be F16 or BF16, got %d", dtype);
  if (ldx < 0 || ldw < 0 || ldy < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (int rc = check(m, n, k)) return rc;
  if (m == 0 || n == 0) return INTENT_HIP_OK;
  if (y == nullptr || x_scales == nullptr || weight_scales == nullptr || (k > 0 && (x == nullptr || weight == nullptr)))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  if (k > 0 && (ldx % kUnit || !aligned(x, kUnit)))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "rows of x must be 16-byte aligned, their stride a multiple of 16");
  if (k > 0 && (ldw % kUnit || !aligned(weight, kUnit)))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "weight rows must be 16-byte aligned, their stride a multiple of 16");
  if (!aligned(y, 2)) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "y is not aligned to its type");
  Linear p{};
  p.x = x, p.w = weight, p.xs = x_scales, p.ws = weight_scales, p.bias = bias, p.y = static_cast<uint16_t *>(y);
  p.ldx = ldx, p.ldw = ldw, p.ldy = ldy;
  p.m = static_cast<int>(m), p.n = static_cast<int>(n), p.pitch = (p.n + 3) / 4 * 4, p.units = static_cast<int>(k / kUnit);
  p.wide = n % 8 == 0 && ldy % 8 == 0 && aligned(y, 16) ? 8 : n % 4 == 0 && ldy % 4 == 0 && aligned(y, 8) ? 4 : 1;
  const Cut c = cut(m, n, k);
  if (c.parts > 1) {
    const size_t bytes = sums_bytes(c, m, n);
    if (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16))
      return fail(INTENT_HIP_ERR_WORKSPACE, "linear_i8 needs %zu workspace bytes, 16-byte aligned", bytes);
    p.sums = static_cast<int32_t *>(workspace);
  }
  if (dtype == INTENT_HIP_F16)
    launch<f16_t>(p, c, as_stream(stream));
  else
    launch<bf16_t>(p, c, as_stream(stream));
  return hipPeekAtLastError() != hipSuccess ? launch_status("linear_i8") : INTENT_HIP_OK;
}

// Products with 4-bit weights, y = x W^T, for gfx950. No reference counterpart.
//
// W[n, k] = e2m1 element * 2^(exponents[n, k / 32] - 127) in the type of x (one rounding; exact in its normal range), products
// summed in f32, one rounding at the end.
//
// Design. v_mfma_f32_16x16x32 with 16 weight rows as rows and 16 rows of x as columns. The sum over K may run in any order,
// so lane (r, g) takes block g of four of weight row r as it lies in memory (16 bytes, one exponent), converts it in four
// parts, and reads the same 32 values of its row of x. Weights go from memory to registers: no wave needs another's.
//   * linear_few, up to 16 rows of x: a workgroup's 16 waves take a run of K each and add their sums through the LDS. Bound by
//     the weights' bytes and by x, which every workgroup reads (1 x 14336 x 4096: 7.7 us, 4.1 TB/s; 8 rows 10.7, 16
//     rows 12.6; 1 x 4096 x 4096: 3.7, most of it latency: one or two steps a wave; 1 x 128256 x 4096: 59.5, 4.7 TB/s).
//   * linear_tiles: a workgroup's waves share 16 MT rows of x, which pass through the LDS 128 columns at a time (in 16-byte
//     units, unit u of row r at u ^ r % 16, so that the 16 rows of a read are in different banks), and take 16 NT weight
//     rows each. A lane's weight rows are NT apart, so its results are 4 NT consecutive columns of y. Where tiles are few, K
//     is divided over workgroups, whose f32 sums a second kernel adds in order.
//     The small tiles are bound by the latency of a stage and by x's way to the LDS. They keep four stages on their way (32 x
//     4096 x 14336: 22 -> 16.7 us; 256 x 4096 x 4096: 40 -> 24.4), and the smallest shares its rows of x among eight waves
//     (16.7 -> 15.8, 24.4 -> 21.0). Exponents come four stages at a time, a word a lane, and a lane permutation brings them to
//     where they are needed: a byte a lane and stage touches as many cache lines as the weights (21.0 -> 18.2; the tiles of
//     128 x 128 lose up to 4 %). Eight stages on their way instead of four are no faster (32 x 4096 x 14336: 16.0, four 15.2).
//     The large tiles are bound by the matrix pipe and the conversions beside it (1021 x 14336 x 4096: 103 us, 1160
//     TFLOP/s, among other calls, 111 behind others of its kind; the type's own product 90 to 97; three stages, and so one
//     workgroup a CU, 174).
#include <stdio.h>

#include <type_traits>

#include "mx.hpp"
#include "stages.hpp"

namespace intent_hip {
namespace {

constexpr int kFewWaves = 16;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct Linear {
  const uint16_t *x;
  const uint8_t *w, *e;
  uint16_t *y;
  float *sums;                         // [parts][m][n] where K is divided
  int64_t ldx, ldw, lde, ldy;
  int m, n, blocks;                    // blocks: K / 32
  int m_tiles, n_tiles, parts, stages; // linear_tiles: stages of 128 columns of a part
  int wide;                            // y takes stores of so many elements (1, 4 or 8)
};

template <typename E>
__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t c) {
  if constexpr (std::is_same_v<E, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight e2m1 elements (the low four bits first) as 16-bit values.
template <typename E>
__device__ __forceinline__ uint4 eight(uint32_t word, float scale) {
  if constexpr (std::is_same_v<E, f16_t>)
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 3)));
  else
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3)));
}

// kCount consecutive results of one row of y, from column n on.
template <typename E, int kCount>
__device__ __forceinline__ void store(const Linear &p, int m, int n, const float (&v)[kCount]) {
  if (m >= p.m || n >= p.n) return;
  uint16_t *y = p.y + m * p.ldy + n;
  if (p.wide >= 4) {
    uint32_t words[kCount / 2];
#pragma unroll
    for (int i = 0; i < kCount / 2; ++i)
      words[i] = from_f32<E>(v[2 * i]).bits | static_cast<uint32_t>(from_f32<E>(v[2 * i + 1]).bits) << 16;
    if (kCount >= 8 && p.wide == 8) {
#pragma unroll
      for (int i = 0; i + 8 <= kCount; i += 8)
        if (n + i < p.n) *reinterpret_cast<uint4 *>(y + i) = make_uint4(words[i / 2], words[i / 2 + 1], words[i / 2 + 2], words[i / 2 + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < kCount; i += 4)
        if (n + i < p.n) *reinterpret_cast<uint2 *>(y + i) = make_uint2(words[i / 2], words[i / 2 + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kCount; ++i)
      if (n + i < p.n) y[i] = from_f32<E>(v[i]).bits;
  }
}

// Up to 16 rows of x by 16 NT weight rows a workgroup; its 16 waves take a run of K each. The loads of kAhead steps of 128
// columns are on their way at once, the exponents of all weight rows in one, which a lane permutation brings to where they are
// needed (16 x 14336 x 4096: 12.8 us with a load a weight row, 12.2 so). Columns of the product behind the rows of x are never
// stored, so their lanes read any row.
//
// kOne: x is one row. Its 128 columns of a step are a word a lane, and every lane takes the 16 words of its block from the lanes
// of its row of 16: loads of 16 bytes a lane, 16 times each value, hold up the weights' (1 x 4096 x 14336: 10.5 us, so 8.6; 1 x
// 14336 x 4096: 8.9 and 7.8).
template <int kFirst>
__device__ __forceinline__ uint4 words_of_row(uint32_t own) {
  const int v = static_cast<int>(own);
  return make_uint4(__builtin_amdgcn_update_dpp(0, v, 0x150 + kFirst, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, v, 0x151 + kFirst, 0xF, 0xF, false),
                    __builtin_amdgcn_update_dpp(0, v, 0x152 + kFirst, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, v, 0x153 + kFirst, 0xF, 0xF, false));
}

template <typename E, int NT, bool kOne>
__global__ __launch_bounds__(kFewWaves *kWave) void linear_few(Linear p) {
  constexpr int kAhead = 2, kSums = NT * 4;
  __shared__ float sums[kFewWaves][kSums][kWave];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * 16 * NT;
  const uint8_t *w[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j)         // rows behind the last are not stored
    w[j] = p.w + static_cast<int64_t>(min(n0 + r * NT + j, p.n - 1)) * p.ldw + g * 16;
  const uint8_t *const e = p.e + static_cast<int64_t>(min(n0 + r * NT + g % NT, p.n - 1)) * p.lde;
  const uint16_t *x = kOne ? p.x + g * 32 + r * 2 : p.x + min(r, p.m - 1) * p.ldx + g * 32;
  f32x4_t acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4_t{0, 0, 0, 0};
  const int first = min(wave * p.stages * 4, p.blocks), last = min(first + p.stages * 4, p.blocks);
  for (int b0 = first; b0 < last; b0 += kAhead * 4) {
    uint4 raw[kAhead][NT], v[kAhead][4];
    uint32_t one[kAhead];
    uint32_t power[kAhead];            // of step i: word i, of weight row r NT + g in lane (r, g)
    const bool whole = b0 + kAhead * 4 <= last;
    if (b0 + kAhead * 4 <= p.blocks) {
      if (g < NT) __builtin_memcpy(power, e + b0, sizeof(power));
    } else {                           // behind K any
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        uint32_t byte[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) byte[t] = e[min(b0 + i * 4 + t, p.blocks - 1)];
        power[i] = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = b0 + i * 4;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        raw[i][j] = make_uint4(0, 0, 0, 0);
        if (whole || b + g < last) raw[i][j] = *reinterpret_cast<const uint4 *>(w[j] + b * 16);
      }
      if constexpr (kOne) {
        one[i] = 0;
        if (whole || b + g < last) one[i] = *reinterpret_cast<const uint32_t *>(x + b * 32);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v[i][c] = make_uint4(0, 0, 0, 0);
          if (whole || b + g < last) v[i][c] = *reinterpret_cast<const uint4 *>(x + b * 32 + c * 8);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if constexpr (kOne) {
        v[i][0] = words_of_row<0>(one[i]), v[i][1] = words_of_row<4>(one[i]);
        v[i][2] = words_of_row<8>(one[i]), v[i][3] = words_of_row<12>(one[i]);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t words[4] = {raw[i][j].x, raw[i][j].y, raw[i][j].z, raw[i][j].w};
        const uint32_t word = __builtin_amdgcn_ds_bpermute((j * 16 + r) * 4, static_cast<int>(power[i]));
        const float scale = mx_scale(whole || b0 + i * 4 + g < last ? word >> (8 * g) & 0xFF : 127);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[j] = mfma<E>(eight<E>(words[c], scale), v[i][c], acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][i * NT + j][lane] = acc[j][i];
  __syncthreads();
  if (wave >= kSums || r >= p.m) return;
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) total += sums[i][wave][lane];
  const int n = n0 + g * kSums + wave;
  if (n < p.n) p.y[r * p.ldy + n] = from_f32<E>(total).bits;
}

// 16 MT rows of x by 16 NT weight rows for each of W waves; S stages of 128 columns are on their way or in use. Each has an LDS array
// of its own, and the loop is unrolled by S: the compiler then knows which loads into the LDS a read has to wait for.
template <typename E, int MT, int NT, int S, int W>
__global__ __launch_bounds__(W *kWave, 2) void linear_tiles(Linear p) {
  constexpr int kRows = 16 * MT, kUnits = kRows * 16, kLoads = kUnits / (W * kWave);     // 16-byte units of a stage
  constexpr int kRead = MT <= 4 ? 4 : 1;               // quarters of a stage read before their products, as registers allow
  constexpr int kIssued = kLoads + NT;                 // loads of a wave per stage, always as many (the exponents' come on top)
  static_assert(S == 2 || S == 4, "one LDS array per stage, four stages a turn of the loop");
  __shared__ uint4 x_0[kUnits], x_1[kUnits], x_2[S > 2 ? kUnits : 1], x_3[S > 2 ? kUnits : 1];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.m_tiles * p.n_tiles;
  int tile = xcd_tile(grid_block(), tiles * p.parts);
  if (tile < 0) return;
  const int part = tile / tiles;
  tile -= part * tiles;
  const int m0 = tile % p.m_tiles * kRows, n0 = (tile / p.m_tiles * W + wave) * 16 * NT;
  const int first = min(part * p.stages * 4, p.blocks), last = min(p.blocks, first + p.stages * 4);     // blocks of K of this part
  const int stages = (last - first + 3) / 4;
  // Units of x that this thread brings in: row i * 4 W + own_row, its unit `unit` to the place that the thread's load fills.
  const int own_row = wave * 4 + g, unit = r ^ (own_row & 15);
  const uint16_t *from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i)                     // rows behind the last are not stored
    from[i] = p.x + static_cast<int64_t>(min(m0 + i * 4 * W + own_row, p.m - 1)) * p.ldx + unit * 8;
  const uint8_t *w[NT], *e[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t row = min(n0 + r * NT + j, p.n - 1);
    w[j] = p.w + row * p.ldw;
    e[j] = p.e + row * p.lde;
  }
  uint4 raw[S][NT];
  uint32_t powers[NT], later[NT];      // of four stages: lane (r, g) holds those of stage g
  const auto array = [&](int u) -> uint4 * { return u == 0 ? x_0 : u == 1 ? x_1 : u == 2 ? x_2 : x_3; };
  const auto issue = [&](int t, int u) {               // stage t (the last again behind it) into set u
    const int b0 = first + min(t, stages - 1) * 4;
    uint4 *stage = array(u);
    if (b0 + 4 <= last) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint16_t *src = from[i] + static_cast<int64_t>(b0) * 32;
        __builtin_amdgcn_global_load_lds(src, (lds_void_t *)(stage + (i * W + wave) * kWave), 16, 0, 0);
      }
    } else {                                           // K ends inside the stage: zeros behind it
      const uint16_t *zero = reinterpret_cast<const uint16_t *>(&kZeroUnit);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint16_t *src = b0 + unit / 4 < last ? from[i] + static_cast<int64_t>(b0) * 32 : zero;
        __builtin_amdgcn_global_load_lds(src, (lds_void_t *)(stage + (i * W + wave) * kWave), 16, 0, 0);
      }
    }
    const int b = min(b0 + g, last - 1);
#pragma unroll
    for (int j = 0; j < NT; ++j) raw[u][j] = *reinterpret_cast<const uint4 *>(w[j] + static_cast<int64_t>(b) * 16);
  };
  const auto fetch = [&](int t) {                      // the exponents of stages t .. t + 3, behind K any
    const int b = first + (t + g) * 4;
    if (first + t * 4 + 16 <= p.blocks) {
#pragma unroll
      for (int j = 0; j < NT; ++j) __builtin_memcpy(&later[j], e[j] + b, 4);
    } else {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t byte[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) byte[i] = e[j][min(b + i, p.blocks - 1)];
        later[j] = byte[0] | byte[1] << 8 | byte[2] << 16 | byte[3] << 24;
      }
    }
  };
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
  if (stages > 0) {
    fetch(0);
#pragma unroll
    for (int u = 0; u < S - 1; ++u) issue(u, u);
    for (int t0 = 0; t0 < stages; t0 += 4) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (t0 + u >= stages) break;
        INTENT_WAIT_VMCNT((S - 2) * kIssued);          // this wave's loads of the stage have come
        stage_barrier();                               // everybody's have, and nobody reads the set that is filled next
        if (u == 0) {
#pragma unroll
          for (int j = 0; j < NT; ++j) powers[j] = later[j];
        }
        issue(t0 + u + S - 1, (u + S - 1) % S);
        if (u == (S == 4 ? 0 : 3) && t0 + 4 < stages) fetch(t0 + 4);       // (S = 2 has no registers to spare before)
        const bool held = first + (t0 + u) * 4 + g < last;
        uint4 own[NT];
        float scale[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t word = __builtin_amdgcn_ds_bpermute((u * 16 + r) * 4, static_cast<int>(powers[j]));
          own[j] = held ? raw[u % S][j] : make_uint4(0, 0, 0, 0);
          scale[j] = mx_scale(word >> (8 * g) & 0xFF);
        }
#pragma unroll
        for (int c0 = 0; c0 < 4; c0 += kRead) {
          uint4 v[kRead][MT];
#pragma unroll
          for (int c = 0; c < kRead; ++c)
#pragma unroll
            for (int i = 0; i < MT; ++i) v[c][i] = array(u % S)[(i * 16 + r) * 16 + ((g * 4 + c0 + c) ^ r)];
#pragma unroll
          for (int c = c0; c < c0 + kRead; ++c) {
            uint4 a[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) a[j] = eight<E>(c == 0 ? own[j].x : c == 1 ? own[j].y : c == 2 ? own[j].z : own[j].w, scale[j]);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int j = 0; j < NT; ++j) acc[i][j] = mfma<E>(a[j], v[c - c0][i], acc[i][j]);
          }
        }
      }
    }
    INTENT_WAIT_VMCNT(0);                              // nothing is on its way into the LDS of an ended workgroup
  }
  // A lane's results: row m0 + 16 i + r of y, columns n0 + (4 g + k) NT + j.
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    float row[4 * NT];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < NT; ++j) row[k * NT + j] = acc[i][j][k];
    const int m = m0 + i * 16 + r, n = n0 + g * 4 * NT;
    if (p.parts == 1) {
      store<E>(p, m, n, row);
    } else if (m < p.m) {
      float *to = p.sums + (static_cast<int64_t>(part) * p.m + m) * p.n + n;
      if (p.wide > 1) {
#pragma unroll
        for (int k = 0; k < 4 * NT; k += 4)
          if (n + k < p.n) *reinterpret_cast<float4 *>(to + k) = make_float4(row[k], row[k + 1], row[k + 2], row[k + 3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4 * NT; ++k)
          if (n + k < p.n) to[k] = row[k];
      }
    }
  }
}

// y from the parts' sums, in order: kCount columns a thread.
template <typename E, int kCount>
__global__ __launch_bounds__(256) void linear_fold(Linear p) {
  const int64_t all = static_cast<int64_t>(p.m) * p.n, at = (static_cast<int64_t>(grid_block()) * 256 + threadIdx.x) * kCount;
  if (at >= all) return;
  typedef float held_t __attribute__((ext_vector_type(kCount)));
  held_t total = 0.0f;
#pragma unroll 8
  for (int i = 0; i < p.parts; ++i) total += *reinterpret_cast<const held_t *>(p.sums + i * all + at);
  const int64_t m = at / p.n;
  uint16_t *y = p.y + m * p.ldy + (at - m * p.n);
  if constexpr (kCount == 4)
    *reinterpret_cast<uint2 *>(y) = make_uint2(from_f32<E>(total[0]).bits | static_cast<uint32_t>(from_f32<E>(total[1]).bits) << 16,
                                               from_f32<E>(total[2]).bits | static_cast<uint32_t>(from_f32<E>(total[3]).bits) << 16);
  else
    *y = from_f32<E>(total[0]).bits;
}

// How a product is cut.
struct Cut {
  int mt, nt, parts;                   // mt = 0: linear_few; 1: of one row
};
constexpr int tile_waves(int mt) { return mt == 2 ? 8 : 4; }

// linear_few for up to 16 rows, NT by the weight rows there are for the workgroups (16 x 14336 x 4096: NT = 1 23.8 us, 2 16.9,
// 4 12.7; 2 x 4096 x 14336: 11.3, 16.4, 26.7; one row of 14336 x 4096: 8.7, 7.8, 8.7, of 4096 x 4096: 3.6, 4.7, 6.9). Where more than eight rows meet a long K and few weight rows, x read once per
// 16 weight rows costs more than the weights (16 x 4096 x 14336: 19.8 us, in tiles 15.5).
// linear_tiles otherwise, by an estimate from what its tiles measured: us a stage takes a workgroup that has a CU for itself,
// and each of several on a CU, and what writing, reading and adding the parts' sums takes. It is within a fifth of the best of
// all tiles and parts at M of 17 to 1021 and N x K of 1000 x 4096 to 28672 x 8192.
Cut cut(int64_t m, int64_t n, int64_t k) {
  const int cus = device_cus();
  if (m == 1) return {1, n >= 24 * cus ? 2 : 1, 1};
  if (m <= 16 && (m <= 8 || n >= 24 * cus || k < 6144)) return {0, n >= 48 * cus ? 4 : n >= 24 * cus ? 2 : 1, 1};
  constexpr struct { int mt, nt; float alone, shared; } kKinds[] = {{2, 1, 0.53f, 0.5f}, {4, 2, 0.9f, 0.7f}, {8, 2, 1.3f, 0.9f}, {8, 4, 2.1f, 1.67f}};
  const int64_t stages = (k + 127) / 128;
  Cut best{};
  float least = 0.0f;
  for (const auto &kind : kKinds) {
    const int64_t per_tile = 16 * tile_waves(kind.mt) * kind.nt;
    const int64_t tiles = ((m + 16 * kind.mt - 1) / (16 * kind.mt)) * ((n + per_tile - 1) / per_tile);
    for (int parts = 1; parts <= 16 && (parts == 1 || parts * 4 <= stages); ++parts) {
      const float on_one = static_cast<float>((tiles * parts + cus - 1) / cus), shared = kind.shared * on_one;
      float us = static_cast<float>((stages + parts - 1) / parts) * (kind.alone > shared ? kind.alone : shared);
      if (parts > 1) us += 3.0f + static_cast<float>(parts) * static_cast<float>(m) * static_cast<float>(n) * 2.3e-6f;
      if (best.parts == 0 || us < least) best = {kind.mt, kind.nt, parts}, least = us;
    }
  }
  return best;
}

// f with the kernel of a cut, its name and its waves.
template <typename E, typename F>
int with_kernel(const Cut &c, F f) {
  if (c.mt == 0)
    return c.nt == 1   ? f(linear_few<E, 1, false>, "linear_few", kFewWaves)
           : c.nt == 2 ? f(linear_few<E, 2, false>, "linear_few", kFewWaves)
                       : f(linear_few<E, 4, false>, "linear_few", kFewWaves);
  if (c.mt == 1) return c.nt == 1 ? f(linear_few<E, 1, true>, "linear_few", kFewWaves) : f(linear_few<E, 2, true>, "linear_few", kFewWaves);
  return c.mt == 2   ? f(linear_tiles<E, 2, 1, 4, tile_waves(2)>, "linear_tiles", tile_waves(2))
         : c.mt == 4 ? f(linear_tiles<E, 4, 2, 4, tile_waves(4)>, "linear_tiles", tile_waves(4))
         : c.nt == 2 ? f(linear_tiles<E, 8, 2, 2, tile_waves(8)>, "linear_tiles", tile_waves(8))
                     : f(linear_tiles<E, 8, 4, 2, tile_waves(8)>, "linear_tiles", tile_waves(8));
}

template <typename E>
void launch(Linear p, const Cut &c, hipStream_t s) {
  p.parts = c.parts;
  with_kernel<E>(c, [&](void (*kernel)(Linear), const char *, int waves) {
    const int runs = c.mt <= 1 ? waves : c.parts;
    p.stages = ((p.blocks + 3) / 4 + runs - 1) / runs;
    dim3 grid(static_cast<unsigned>((p.n + 16 * c.nt - 1) / (16 * c.nt)));
    if (c.mt > 1) {
      p.m_tiles = (p.m + 16 * c.mt - 1) / (16 * c.mt), p.n_tiles = (p.n + 16 * waves * c.nt - 1) / (16 * waves * c.nt);
      grid = tile_grid(static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.parts, 1);
    }
    kernel<<<grid, waves * kWave, 0, s>>>(p);
    return 0;
  });
  if (c.parts == 1) return;
  const int64_t all = static_cast<int64_t>(p.m) * p.n;
  if (p.wide > 1)
    linear_fold<E, 4><<<tile_grid((all / 4 + 255) / 256, 1), 256, 0, s>>>(p);
  else
    linear_fold<E, 1><<<tile_grid((all + 255) / 256, 1), 256, 0, s>>>(p);
}

int check(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (k % kMxBlock)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "weights are blocks of %d elements (got K = %lld)", kMxBlock, static_cast<long long>(k));
  if (m > (1 << 20) || n > (1 << 24) || k > INT32_MAX / 64) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}
}  // namespace

int linear_mxfp4_resources(int dtype, int64_t m, int64_t n, int64_t k, IntentHipKernelResources *out) {
  if (int rc = check(m, n, k)) return rc;
  const Cut c = cut(m, n, k);
  const auto describe = [&](void (*kernel)(Linear), const char *which, int waves) {
    char name[64];
    snprintf(name, sizeof(name), "%s<%s,%d,%d>", which, dtype == INTENT_HIP_F16 ? "f16" : "bf16", c.mt, c.nt);
    return describe_kernel(reinterpret_cast<const void *>(kernel), name, waves * kWave, out);
  };
  return dtype == INTENT_HIP_F16 ? with_kernel<f16_t>(c, describe) : with_kernel<bf16_t>(c, describe);
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_linear_mxfp4_workspace_bytes(int64_t m, int64_t n, int64_t k, size_t *bytes) {
  if (bytes == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null output");
  *bytes = 0;
  if (int rc = check(m, n, k)) return rc;
  if (m == 0 || n == 0) return INTENT_HIP_OK;
  const Cut c = cut(m, n, k);
  if (c.parts > 1) *bytes = static_cast<size_t>(c.parts) * m * n * sizeof(float);
  return INTENT_HIP_OK;
}

extern "C" int intent_hip_linear_mxfp4(int dtype, const void *x, const uint8_t *weight, const uint8_t *exponents, void *y,
                                       int64_t m, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int64_t lde, int64_t ldy,
                                       void *workspace, size_t workspace_bytes, void *stream) {
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "linear_mxfp4 dtype must be F16 or BF16, got %d", dtype);
  if (ldx < 0 || ldw < 0 || lde < 0 || ldy < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (int rc = check(m, n, k)) return rc;
  if (m == 0 || n == 0) return INTENT_HIP_OK;
  if (y == nullptr || (k > 0 && (x == nullptr || weight == nullptr || exponents == nullptr)))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  if (k > 0 && (ldx % 8 || !aligned(x, 16)))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "rows of x must be 16-byte aligned, their stride a multiple of 8 elements");
  if (k > 0 && (ldw % 16 || !aligned(weight, 16)))
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "weight rows must be 16-byte aligned, their stride a multiple of 16 bytes");
  if (!aligned(y, 2)) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "y is not aligned to its type");
  Linear p{};
  p.x = static_cast<const uint16_t *>(x), p.w = weight, p.e = exponents, p.y = static_cast<uint16_t *>(y);
  p.ldx = ldx, p.ldw = ldw, p.lde = lde, p.ldy = ldy;
  p.m = static_cast<int>(m), p.n = static_cast<int>(n), p.blocks = static_cast<int>(k / kMxBlock);
  p.wide = n % 8 == 0 && ldy % 8 == 0 && aligned(y, 16) ? 8 : n % 4 == 0 && ldy % 4 == 0 && aligned(y, 8) ? 4 : 1;
  const Cut c = cut(m, n, k);
  if (c.parts > 1) {
    const size_t bytes = static_cast<size_t>(c.parts) * m * n * sizeof(float);
    if (workspace == nullptr || workspace_bytes < bytes || !aligned(workspace, 16))
      return fail(INTENT_HIP_ERR_WORKSPACE, "linear_mxfp4 needs %zu workspace bytes, 16-byte aligned", bytes);
    p.sums = static_cast<float *>(workspace);
  }
  if (dtype == INTENT_HIP_F16)
    launch<f16_t>(p, c, as_stream(stream));
  else
    launch<bf16_t>(p, c, as_stream(stream));
  return hipPeekAtLastError() != hipSuccess ? launch_status("linear_mxfp4") : INTENT_HIP_OK;
}

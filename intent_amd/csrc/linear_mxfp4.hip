// Products with 4-bit weights, y = x W^T, for gfx950. No reference counterpart.
//
// W[n, k] = e2m1 element * 2^(exponents[n, k / 32] - 127) in the type of x (one rounding; exact in its normal range), products
// summed in f32, one rounding at the end.
//
// Design. v_mfma_f32_16x16x32 with 16 weight rows as rows and 16 rows of x as columns. The sum over K may run in any order,
// so lane (r, g) takes block g of four of weight row r as it lies in memory (16 bytes, one exponent), converts it in four
// parts, and reads the same 32 values of its row of x. Weights go from memory to registers: no wave needs another's.
//   * linear_few, up to 16 rows of x: a workgroup's waves take 128 columns of K in turn and add their sums through the LDS.
//     Bound by the weights' bytes.
//   * linear_tiles: a workgroup's waves share 16 MT rows of x, which pass through the LDS 128 columns at a time (in 16-byte
//     units, unit u of row r at u ^ r % 16, so that the 16 rows of a read are in different banks), and take 16 NT weight
//     rows each. A lane's weight rows are NT apart, so its results are 4 NT consecutive columns of y. Where tiles are few, K
//     is divided over workgroups, whose f32 sums a second kernel adds in order.
#include <stdio.h>

#include <type_traits>

#include "mx.hpp"

namespace intent_hip {
namespace {

constexpr int kWaves = 4;

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

// Up to 16 rows of x: 16 weight rows a workgroup of W waves.
template <typename E, int W>
__global__ __launch_bounds__(W *kWave) void linear_few(Linear p) {
  constexpr int kAhead = 4;            // steps on their way at once
  __shared__ float sums[W][4][kWave];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * 16;
  const int64_t row = min(n0 + r, p.n - 1);                    // rows behind the last are not stored
  const uint8_t *w = p.w + row * p.ldw, *e = p.e + row * p.lde;
  const bool live = r < p.m;
  const uint16_t *x = p.x + (live ? r : 0) * p.ldx;
  f32x4_t acc = {0, 0, 0, 0};
  for (int b0 = wave * 4; b0 < p.blocks; b0 += W * 4 * kAhead) {
    uint4 raw[kAhead], v[kAhead][4];
    uint8_t power[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int b = b0 + i * W * 4 + g;
      raw[i] = make_uint4(0, 0, 0, 0);
      power[i] = 127;
      if (b < p.blocks) {
        raw[i] = *reinterpret_cast<const uint4 *>(w + b * 16);
        power[i] = e[b];
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[i][c] = make_uint4(0, 0, 0, 0);
        if (live && b < p.blocks) v[i][c] = *reinterpret_cast<const uint4 *>(x + b * 32 + c * 8);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      const float scale = mx_scale(power[i]);
#pragma unroll
      for (int c = 0; c < 4; ++c) acc = mfma<E>(eight<E>(words[c], scale), v[i][c], acc);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave != 0) return;
  float total[4] = {};
#pragma unroll
  for (int j = 0; j < W; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) total[i] += sums[j][i][lane];
  store<E>(p, r, n0 + g * 4, total);
}

typedef __attribute__((address_space(3))) void lds_void_t;

// 16 MT rows of x by 64 NT weight rows a workgroup.
template <typename E, int MT, int NT>
__global__ __launch_bounds__(kWaves *kWave) void linear_tiles(Linear p) {
  constexpr int kRows = 16 * MT, kUnits = kRows * 16, kLoads = kUnits / (kWaves * kWave);     // 16-byte units of a stage
  __shared__ uint4 x_s[2 * kUnits];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles = p.m_tiles * p.n_tiles;
  int tile = xcd_tile(grid_block(), tiles * p.parts);
  if (tile < 0) return;
  const int part = tile / tiles;
  tile -= part * tiles;
  const int m0 = tile % p.m_tiles * kRows, n0 = (tile / p.m_tiles * kWaves + wave) * 16 * NT;
  const int first = part * p.stages * 4, last = min(p.blocks, first + p.stages * 4);     // blocks of K of this part
  // Units of x that this thread brings in: unit u of LDS row (u / 16) comes from unit (u % 16) ^ (row % 16) of x's row.
  const uint16_t *from[kLoads];
  int unit[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int at = (i * kWaves + wave) * kWave + lane, row = at / 16;
    unit[i] = (at ^ row) & 15;
    from[i] = p.x + static_cast<int64_t>(min(m0 + row, p.m - 1)) * p.ldx + unit[i] * 8;       // rows behind the last are not stored
  }
  const auto bring = [&](int b, int to) {
    uint4 *stage = x_s + to * kUnits;
    if (b + 4 <= last) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint16_t *src = from[i] + static_cast<int64_t>(b) * 32;
        __builtin_amdgcn_global_load_lds(src, (lds_void_t *)(stage + (i * kWaves + wave) * kWave), 16, 0, 0);
      }
    } else {                           // K ends inside the stage: zeros behind it
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (b + unit[i] / 4 < last) v = *reinterpret_cast<const uint4 *>(from[i] + static_cast<int64_t>(b) * 32);
        stage[(i * kWaves + wave) * kWave + lane] = v;
      }
    }
  };
  const uint8_t *w[NT], *e[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t row = min(n0 + r * NT + j, p.n - 1);
    w[j] = p.w + row * p.ldw;
    e[j] = p.e + row * p.lde;
  }
  uint4 raw[NT];
  uint8_t power[NT];
  const auto fetch = [&](int b0) {
    const int b = b0 + g;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      raw[j] = make_uint4(0, 0, 0, 0);
      power[j] = 127;
      if (b < last) {
        raw[j] = *reinterpret_cast<const uint4 *>(w[j] + b * 16);
        power[j] = e[j][b];
      }
    }
  };
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
  if (first < last) {
    bring(first, 0);
    fetch(first);
  }
  for (int b0 = first, at = 0; b0 < last; b0 += 4, at ^= 1) {
    uint4 own[NT];
    float scale[NT];
    __syncthreads();                   // this stage has come, and nobody reads the other
#pragma unroll
    for (int j = 0; j < NT; ++j) own[j] = raw[j], scale[j] = mx_scale(power[j]);
    if (b0 + 4 < last) {
      bring(b0 + 4, at ^ 1);
      fetch(b0 + 4);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint4 v[MT], a[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) v[i] = x_s[at * kUnits + (i * 16 + r) * 16 + ((g * 4 + c) ^ r)];
#pragma unroll
      for (int j = 0; j < NT; ++j) a[j] = eight<E>(c == 0 ? own[j].x : c == 1 ? own[j].y : c == 2 ? own[j].z : own[j].w, scale[j]);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mfma<E>(a[j], v[i], acc[i][j]);
    }
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
#pragma unroll
      for (int k = 0; k < 4 * NT; ++k)
        if (n + k < p.n) to[k] = row[k];
    }
  }
}

// y from the parts' sums, in order.
template <typename E>
__global__ __launch_bounds__(256) void linear_fold(Linear p) {
  const int64_t all = static_cast<int64_t>(p.m) * p.n, at = static_cast<int64_t>(grid_block()) * 256 + threadIdx.x;
  if (at >= all) return;
  float total = 0.0f;
#pragma unroll 4
  for (int i = 0; i < p.parts; ++i) total += p.sums[i * all + at];
  const int64_t m = at / p.n;
  p.y[m * p.ldy + (at - m * p.n)] = from_f32<E>(total).bits;
}

// How a product is cut.
struct Cut {
  int mt, nt, waves, parts;            // mt = 0: linear_few with `waves` waves
};
Cut cut(int64_t m, int64_t n, int64_t k) {
  if (m <= 16) return {0, 1, n >= 16 * 16 * device_cus() / 8 ? 4 : n >= 16 * device_cus() ? 8 : 16, 1};
  const auto tiles = [&](int mt, int nt) { return ((m + 16 * mt - 1) / (16 * mt)) * ((n + 64 * nt - 1) / (64 * nt)); };
  Cut c{8, 4, 4, 1};
  if (m <= 32) c.mt = 2, c.nt = 1;
  else if (m <= 64) c.mt = 4, c.nt = 2;
  else if (tiles(8, 4) < 3 * device_cus() / 4) c.nt = 2;
  const int64_t stages = (k + 127) / 128, own = tiles(c.mt, c.nt), wanted = 2 * device_cus() / (own > 0 ? own : 1);
  c.parts = static_cast<int>(wanted < 1 ? 1 : wanted > stages / 4 ? (stages / 4 < 1 ? 1 : stages / 4) : wanted);
  return c;
}

template <typename E>
void launch(Linear p, const Cut &c, hipStream_t s) {
  if (c.mt == 0) {
    const dim3 grid(static_cast<unsigned>((p.n + 15) / 16));
    if (c.waves == 4)
      linear_few<E, 4><<<grid, 4 * kWave, 0, s>>>(p);
    else if (c.waves == 8)
      linear_few<E, 8><<<grid, 8 * kWave, 0, s>>>(p);
    else
      linear_few<E, 16><<<grid, 16 * kWave, 0, s>>>(p);
    return;
  }
  p.m_tiles = (p.m + 16 * c.mt - 1) / (16 * c.mt), p.n_tiles = (p.n + 64 * c.nt - 1) / (64 * c.nt), p.parts = c.parts;
  p.stages = ((p.blocks + 3) / 4 + c.parts - 1) / c.parts;
  const dim3 grid = tile_grid(static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.parts, 1);
  if (c.mt == 2)
    linear_tiles<E, 2, 1><<<grid, kWaves * kWave, 0, s>>>(p);
  else if (c.mt == 4)
    linear_tiles<E, 4, 2><<<grid, kWaves * kWave, 0, s>>>(p);
  else if (c.nt == 2)
    linear_tiles<E, 8, 2><<<grid, kWaves * kWave, 0, s>>>(p);
  else
    linear_tiles<E, 8, 4><<<grid, kWaves * kWave, 0, s>>>(p);
  if (c.parts > 1) linear_fold<E><<<tile_grid((static_cast<int64_t>(p.m) * p.n + 255) / 256, 1), 256, 0, s>>>(p);
}

}  // namespace

int linear_mxfp4_resources(int dtype, int64_t m, int64_t n, int64_t k, IntentHipKernelResources *out) {
  const Cut c = cut(m, n, k);
  char name[64];
  const auto describe = [&](const void *half, const void *brain, int waves) {
    return describe_kernel(dtype == INTENT_HIP_F16 ? half : brain, name, waves * kWave, out);
  };
  const char *const type = dtype == INTENT_HIP_F16 ? "f16" : "bf16";
  if (c.mt == 0) {
    snprintf(name, sizeof(name), "linear_few<%s,%d>", type, c.waves);
    return c.waves == 4   ? describe(reinterpret_cast<const void *>(linear_few<f16_t, 4>), reinterpret_cast<const void *>(linear_few<bf16_t, 4>), 4)
           : c.waves == 8 ? describe(reinterpret_cast<const void *>(linear_few<f16_t, 8>), reinterpret_cast<const void *>(linear_few<bf16_t, 8>), 8)
                          : describe(reinterpret_cast<const void *>(linear_few<f16_t, 16>), reinterpret_cast<const void *>(linear_few<bf16_t, 16>), 16);
  }
  snprintf(name, sizeof(name), "linear_tiles<%s,%d,%d>", type, c.mt, c.nt);
  return c.mt == 2   ? describe(reinterpret_cast<const void *>(linear_tiles<f16_t, 2, 1>), reinterpret_cast<const void *>(linear_tiles<bf16_t, 2, 1>), kWaves)
         : c.mt == 4 ? describe(reinterpret_cast<const void *>(linear_tiles<f16_t, 4, 2>), reinterpret_cast<const void *>(linear_tiles<bf16_t, 4, 2>), kWaves)
         : c.nt == 2 ? describe(reinterpret_cast<const void *>(linear_tiles<f16_t, 8, 2>), reinterpret_cast<const void *>(linear_tiles<bf16_t, 8, 2>), kWaves)
                     : describe(reinterpret_cast<const void *>(linear_tiles<f16_t, 8, 4>), reinterpret_cast<const void *>(linear_tiles<bf16_t, 8, 4>), kWaves);
}

}  // namespace intent_hip

using namespace intent_hip;

namespace {
int check(int64_t m, int64_t n, int64_t k) {
  if (m < 0 || n < 0 || k < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (k % kMxBlock)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "weights are blocks of %d elements (got K = %lld)", kMxBlock, static_cast<long long>(k));
  if (m > (1 << 20) || n > (1 << 24) || k > INT32_MAX / 64) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}
}  // namespace

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

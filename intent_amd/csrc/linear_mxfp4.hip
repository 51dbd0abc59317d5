// Products with 4-bit weights, y = x W^T, for gfx950. No reference counterpart.
//
// W[n, k] = e2m1 element * 2^(exponents[n, k / 32] - 127) in the type of x (one rounding; exact in its normal range), products
// summed in f32, one rounding at the end.
//
// Design. v_mfma_f32_16x16x32 with 16 weight rows as rows and 16 rows of x as columns. The sum over K may run in any order,
// so lane (r, g) takes block g of four of weight row r as it lies in memory (16 bytes, one exponent), converts it in four
// parts, and reads the same 32 values of its row of x. A workgroup's waves take 128 columns of K in turn and add their sums
// through the LDS. Few rows: bound by the weights' bytes.
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
  int64_t ldx, ldw, lde, ldy;
  int m, n, blocks;                    // blocks: K / 32
  bool quads;                          // rows of y take 8-byte stores
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

// Four results of one row of y, columns n .. n + 3.
template <typename E>
__device__ __forceinline__ void store(const Linear &p, int m, int n, f32x4_t v) {
  if (m >= p.m || n >= p.n) return;
  uint16_t *y = p.y + m * p.ldy + n;
  if (p.quads) {
    *reinterpret_cast<uint2 *>(y) = make_uint2(
        from_f32<E>(v[0]).bits | static_cast<uint32_t>(from_f32<E>(v[1]).bits) << 16,
        from_f32<E>(v[2]).bits | static_cast<uint32_t>(from_f32<E>(v[3]).bits) << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.n) y[i] = from_f32<E>(v[i]).bits;
  }
}

// A workgroup: 16 NT weight rows, 16 MT rows of x.
template <typename E, int MT, int NT>
__global__ __launch_bounds__(kWaves *kWave) void linear_few(Linear p) {
  __shared__ float sums[kWaves / 2][MT * NT * 4][kWave];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = static_cast<int>(blockIdx.x) * 16 * NT, m0 = static_cast<int>(blockIdx.y) * 16 * MT;
  const uint8_t *w[NT], *e[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int64_t row = min(n0 + j * 16 + r, p.n - 1);         // rows behind the last are not stored
    w[j] = p.w + row * p.ldw;
    e[j] = p.e + row * p.lde;
  }
  const uint16_t *x[MT];
  bool live[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    live[i] = m0 + i * 16 + r < p.m;
    x[i] = p.x + static_cast<int64_t>(live[i] ? m0 + i * 16 + r : 0) * p.ldx;
  }
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0, 0, 0, 0};
  for (int b0 = wave * 4; b0 < p.blocks; b0 += kWaves * 4) {
    const int b = b0 + g;
    uint4 raw[NT], v[MT][4];
    float scale[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      raw[j] = make_uint4(0, 0, 0, 0);
      scale[j] = 1.0f;
      if (b < p.blocks) {
        raw[j] = *reinterpret_cast<const uint4 *>(w[j] + static_cast<int64_t>(b) * 16);
        scale[j] = mx_scale(e[j][b]);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        v[i][c] = make_uint4(0, 0, 0, 0);
        if (live[i] && b < p.blocks) v[i][c] = *reinterpret_cast<const uint4 *>(x[i] + static_cast<int64_t>(b) * 32 + c * 8);
      }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t words[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint4 a = eight<E>(words[c], scale[j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = mfma<E>(a, v[i][c], acc[i][j]);
      }
    }
  }
#pragma unroll
  for (int half = kWaves / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int t = 0; t < MT * NT * 4; ++t) sums[wave - half][t][lane] = acc[t / 4 / NT][t / 4 % NT][t % 4];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int t = 0; t < MT * NT * 4; ++t) acc[t / 4 / NT][t / 4 % NT][t % 4] += sums[wave][t][lane];
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) store<E>(p, m0 + i * 16 + r, n0 + j * 16 + g * 4, acc[i][j]);
}

template <typename E>
void launch(const Linear &p, hipStream_t s) {
  const auto grid = [&](int mt, int nt) {
    return dim3(static_cast<unsigned>((p.n + 16 * nt - 1) / (16 * nt)), static_cast<unsigned>((p.m + 16 * mt - 1) / (16 * mt)));
  };
  if (p.m <= 16)
    linear_few<E, 1, 1><<<grid(1, 1), kWaves * kWave, 0, s>>>(p);
  else if (p.m <= 32)
    linear_few<E, 2, 2><<<grid(2, 2), kWaves * kWave, 0, s>>>(p);
  else
    linear_few<E, 4, 4><<<grid(4, 4), kWaves * kWave, 0, s>>>(p);
}

}  // namespace

int linear_mxfp4_resources(int dtype, int64_t m, IntentHipKernelResources *out) {
  const bool half = dtype == INTENT_HIP_F16;
  if (m <= 16)
    return half ? describe_kernel(reinterpret_cast<const void *>(linear_few<f16_t, 1, 1>), "linear_few<f16,1,1>", kWaves * kWave, out)
                : describe_kernel(reinterpret_cast<const void *>(linear_few<bf16_t, 1, 1>), "linear_few<bf16,1,1>", kWaves * kWave, out);
  if (m <= 32)
    return half ? describe_kernel(reinterpret_cast<const void *>(linear_few<f16_t, 2, 2>), "linear_few<f16,2,2>", kWaves * kWave, out)
                : describe_kernel(reinterpret_cast<const void *>(linear_few<bf16_t, 2, 2>), "linear_few<bf16,2,2>", kWaves * kWave, out);
  return half ? describe_kernel(reinterpret_cast<const void *>(linear_few<f16_t, 4, 4>), "linear_few<f16,4,4>", kWaves * kWave, out)
              : describe_kernel(reinterpret_cast<const void *>(linear_few<bf16_t, 4, 4>), "linear_few<bf16,4,4>", kWaves * kWave, out);
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_linear_mxfp4(int dtype, const void *x, const uint8_t *weight, const uint8_t *exponents, void *y,
                                       int64_t m, int64_t n, int64_t k, int64_t ldx, int64_t ldw, int64_t lde, int64_t ldy,
                                       void *stream) {
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "linear_mxfp4 dtype must be F16 or BF16, got %d", dtype);
  if (m < 0 || n < 0 || k < 0 || ldx < 0 || ldw < 0 || lde < 0 || ldy < 0)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent or stride");
  if (k % kMxBlock)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "weights are blocks of %d elements (got K = %lld)", kMxBlock, static_cast<long long>(k));
  if (m > (1 << 20) || n > INT32_MAX / 64 || k > INT32_MAX / 64) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
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
  p.quads = n % 4 == 0 && ldy % 4 == 0 && aligned(y, 8);
  if (dtype == INTENT_HIP_F16)
    launch<f16_t>(p, as_stream(stream));
  else
    launch<bf16_t>(p, as_stream(stream));
  return hipPeekAtLastError() != hipSuccess ? launch_status("linear_mxfp4") : INTENT_HIP_OK;
}

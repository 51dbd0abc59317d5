// Blocks of 32 elements that share a power of two (the OCP microscaling formats), for gfx950: e4m3 elements of the paged
// cache, e2m1 elements of the 4-bit weights. A block's exponent byte b stands for 2^(b - 127); 255 stands for NaN. The
// conversions are the chip's own (v_cvt_scalef32_*): one rounding to the target type, subnormals kept.
#pragma once

#include "common.hpp"

namespace intent_hip {

constexpr int kMxBlock = 32;

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bfloat2_t __attribute__((ext_vector_type(2)));
typedef short short2_t __attribute__((ext_vector_type(2)));

// The scale operand of the conversions, whose exponent field alone counts (2^-127 has a field of zero).
__device__ __forceinline__ float mx_scale(int exponent) {
  return __uint_as_float(exponent == 0 ? 0x00400000u : static_cast<uint32_t>(exponent) << 23);
}

// The elements 2 * kHalf and 2 * kHalf + 1 of four e4m3 elements, as two 16-bit values of type E.
template <typename E, bool kHalf>
__device__ __forceinline__ uint32_t mx_pair_e4m3(uint32_t word, float scale) {
  if constexpr (__is_same(E, f16_t))
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, kHalf));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, kHalf));
}

// The exponent byte of a block whose largest finite magnitude is `size`: the smallest e >= -127 with size <= 448 * 2^e.
// size = 1.m * 2^x needs e = x - 8, and one more where 1.m exceeds 1.75.
__device__ __forceinline__ int mx_exponent_e4m3(float size) {
  const uint32_t bits = __float_as_uint(size);
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000);
  return e < 0 ? 0 : e;
}

// Four values as e4m3 elements at a block's scale. |value| <= 448 * scale or not finite; what is not finite is held as NaN
// (the conversion itself would take an infinity to 448).
__device__ __forceinline__ uint32_t mx_quad_e4m3(float a, float b, float c, float d, float scale) {
  const auto settled = [](float v) {
    return (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u ? __uint_as_float(__float_as_uint(v) | 0x7FC00000u) : v;
  };
  short2_t word = {0, 0};
  word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, settled(a), settled(b), scale, false);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, settled(c), settled(d), scale, true);
  return __builtin_bit_cast(uint32_t, word);
}

// The sequence of packed row `row`: the number of sequences among the first `sequences` that end at or before it, found 64
// ends at a time by all lanes of the wave (`row` is the wave's). `sequences` when there is none.
__device__ __forceinline__ int sequence_of(const int32_t *cu, int sequences, int64_t row) {
  const int lane = threadIdx.x & 63;
  int first = 0, count = sequences;            // the answer is first .. first + count
  while (count > 0) {
    const int step = (count + 63) / 64;
    const int at = (lane + 1) * step;          // the end of the at-th of them
    const bool past = at <= count && cu[first + at] <= row;
    const int steps = __popcll(__ballot(past));
    first += steps * step;
    count = step == 1 ? 0 : min(step - 1, count - steps * step);
  }
  return first;
}

// The pages of a sequence's tokens. Tables are read as given; what they name outside their arrays is no page.
struct PageTable {
  const int32_t *offsets, *indices;
  int64_t positions, pages;
  int ps;
  // The page of logical page `at` of sequence s, or -1.
  __device__ __forceinline__ int64_t page(int s, int64_t at) const {
    const int64_t first = offsets[s], last = offsets[s + 1];
    if (at < 0 || at >= last - first || first < 0 || first + at >= positions) return -1;
    const int64_t page = indices[first + at];
    return page < 0 || page >= pages ? -1 : page;
  }
};

}  // namespace intent_hip

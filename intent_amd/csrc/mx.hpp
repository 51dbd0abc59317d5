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
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));

// The scale operand of the conversions: its exponent field alone counts, and a field of 0 is 2^-127 there.
__device__ __forceinline__ float mx_scale(int exponent) { return __uint_as_float(static_cast<uint32_t>(exponent) << 23); }

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

// Four e4m3 elements of two pairs of 16-bit values of type E, at a block's scale: finite magnitudes of at most 448 * scale
// (the conversion itself would take an infinity to 448), or NaN.
template <typename E>
__device__ __forceinline__ uint32_t mx_quad_e4m3(uint32_t low, uint32_t high, float scale) {
  short2_t word = {0, 0};
  if constexpr (__is_same(E, f16_t)) {
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(word, __builtin_bit_cast(half2_t, low), scale, false);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(word, __builtin_bit_cast(half2_t, high), scale, true);
  } else {
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(word, __builtin_bit_cast(bfloat2_t, low), scale, false);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(word, __builtin_bit_cast(bfloat2_t, high), scale, true);
  }
  return __builtin_bit_cast(uint32_t, word);
}

// Two 16-bit values with what is not finite taken out (to 0), or turned into NaN.
template <typename E, bool kNaN>
__device__ __forceinline__ uint32_t mx_settled(uint32_t pair) {
  constexpr uint32_t inf = __is_same(E, f16_t) ? 0x7C00u : 0x7F80u;
  const auto one = [](uint32_t v) { return (v & inf) != inf ? v : kNaN ? v | 0x7FFFu : 0u; };
  return one(pair & 0xFFFFu) | one(pair >> 16) << 16;
}

// The larger (smaller) of each half of two pairs of 16-bit magnitudes (sign bits clear: they order as whole numbers).
__device__ __forceinline__ uint32_t mx_larger(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
}

__device__ __forceinline__ uint32_t mx_smaller(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
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
  // The page of logical page `at` of a sequence that holds `held` of them from offsets entry `first` on, or -1.
  __device__ __forceinline__ int64_t page(int64_t first, int64_t held, int64_t at) const {
    if (at < 0 || at >= held || first < 0 || first + at >= positions) return -1;
    const int64_t page = indices[first + at];
    return page < 0 || page >= pages ? -1 : page;
  }
};

}  // namespace intent_hip

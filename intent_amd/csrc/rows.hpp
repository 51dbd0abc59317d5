// Rows of 16-bit elements held in the registers of a workgroup, and rows of 8-bit integers with a scale each, for gfx950.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace intent_hip {

constexpr int kPiece = 8;              // elements of a thread's piece
constexpr int kMaxRowWaves = 16;

// Pieces as they may lie in rows of any alignment: an access of 16 bytes may begin at any byte here.
typedef uint32_t loose_x4_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t loose_x2_t __attribute__((ext_vector_type(2), aligned(1)));
typedef float loose_f4_t __attribute__((ext_vector_type(4), aligned(4)));

// Where the elements of a row lie in its threads: piece j of thread i is eight elements from 8 (i + threads j) on. kPieces: pieces
// begin at 16 bytes (8, of 8-bit integers) and each is whole or behind the row; otherwise the row's last piece goes by elements.
template <bool kPieces>
struct RowPlace {
  int d, threads, thread;
  __device__ __forceinline__ int column(int j) const { return kPiece * (thread + threads * j); }
  __device__ __forceinline__ bool holds(int j, int i) const { return column(j) + (kPieces ? 0 : i) < d; }
  __device__ __forceinline__ bool whole(int j) const { return column(j) + (kPieces ? 0 : kPiece - 1) < d; }
};

// A piece on its way: of a row's last one that is not whole, the last eight elements of the row, so that every thread loads once and
// none waits; `settled` is the piece itself, 0 behind the row.
template <bool kPieces>
__device__ __forceinline__ uint4 load_piece(const uint16_t *row, const RowPlace<kPieces> &at, int j) {
  if constexpr (kPieces) {
    return at.whole(j) ? *reinterpret_cast<const uint4 *>(row + at.column(j)) : make_uint4(0, 0, 0, 0);
  } else {
    loose_x4_t v = {0, 0, 0, 0};
    if (at.d >= kPiece) {
      if (at.holds(j, 0)) v = *reinterpret_cast<const loose_x4_t *>(row + min(at.column(j), at.d - kPiece));
    } else if (at.column(j) == 0) {
#pragma unroll
      for (int i = 0; i < kPiece - 1; ++i)
        if (i < at.d) v[i / 2] |= static_cast<uint32_t>(row[i]) << (16 * (i & 1));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
}

template <bool kPieces>
__device__ __forceinline__ uint4 settled(uint4 v, const RowPlace<kPieces> &at, int j) {
  if constexpr (!kPieces) {
    const int by = at.column(j) - (at.d - kPiece);
    if (at.d >= kPiece && by > 0 && by < kPiece) {
      if (by & 1)
        v = make_uint4(__builtin_amdgcn_alignbit(v.y, v.x, 16), __builtin_amdgcn_alignbit(v.z, v.y, 16), __builtin_amdgcn_alignbit(v.w, v.z, 16), v.w >> 16);
      if (by & 2) v = make_uint4(v.y, v.z, v.w, 0);
      if (by & 4) v = make_uint4(v.z, v.w, 0, 0);
    }
  }
  return v;
}

template <bool kPieces>
__device__ __forceinline__ void store_piece(uint16_t *row, const RowPlace<kPieces> &at, int j, uint4 v) {
  row += at.column(j);
  if constexpr (kPieces) {
    if (at.whole(j)) *reinterpret_cast<uint4 *>(row) = v;
  } else {
    const loose_x4_t words = {v.x, v.y, v.z, v.w};
    if (at.whole(j)) {
      *reinterpret_cast<loose_x4_t *>(row) = words;
    } else {
#pragma unroll
      for (int i = 0; i < kPiece - 1; ++i)
        if (at.holds(j, i)) row[i] = static_cast<uint16_t>(words[i / 2] >> (16 * (i & 1)));
    }
  }
}

template <bool kPieces>
__device__ __forceinline__ void store_piece(int8_t *row, const RowPlace<kPieces> &at, int j, uint2 v) {
  row += at.column(j);
  if constexpr (kPieces) {
    if (at.whole(j)) *reinterpret_cast<uint2 *>(row) = v;
  } else {
    const loose_x2_t words = {v.x, v.y};
    if (at.whole(j)) {
      *reinterpret_cast<loose_x2_t *>(row) = words;
    } else {
#pragma unroll
      for (int i = 0; i < kPiece - 1; ++i)
        if (at.holds(j, i)) row[i] = static_cast<int8_t>(words[i / 4] >> (8 * (i & 3)));
    }
  }
}

// The f32 weights of a piece; 0 behind the row. (Taken as the rows' pieces are, 16384 x 2049 took 71 us forward for 66.)
template <bool kPieces>
__device__ __forceinline__ void load_weights(const float *w, const RowPlace<kPieces> &at, int j, float (&out)[kPiece]) {
  w += at.column(j);
#pragma unroll
  for (int i = 0; i < kPiece; ++i) out[i] = 0.0f;
  if (at.whole(j)) {
    const loose_f4_t u = *reinterpret_cast<const loose_f4_t *>(w), v = *reinterpret_cast<const loose_f4_t *>(w + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = u[i], out[4 + i] = v[i];
  } else if constexpr (!kPieces) {
#pragma unroll
    for (int i = 0; i < kPiece - 1; ++i)
      if (at.holds(j, i)) out[i] = w[i];
  }
}

template <bool kPieces>
__device__ __forceinline__ void store_weights(float *w, const RowPlace<kPieces> &at, int j, const float (&v)[kPiece]) {
  w += at.column(j);
  if (at.whole(j)) {
    const loose_f4_t a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    *reinterpret_cast<loose_f4_t *>(w) = a, *reinterpret_cast<loose_f4_t *>(w + 4) = b;
  } else if constexpr (!kPieces) {
#pragma unroll
    for (int i = 0; i < kPiece - 1; ++i)
      if (at.holds(j, i)) w[i] = v[i];
  }
}

template <typename E>
__device__ __forceinline__ void widen_piece(uint4 raw, float (&out)[kPiece]) {
  const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < kPiece; ++i) out[i] = to_f32(E{static_cast<uint16_t>(words[i / 2] >> (16 * (i & 1)))});
}

template <typename E>
__device__ __forceinline__ uint4 narrow_piece(const float (&v)[kPiece]) {
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    words[i] = from_f32<E>(v[2 * i]).bits | static_cast<uint32_t>(from_f32<E>(v[2 * i + 1]).bits) << 16;
  return make_uint4(words[0], words[1], words[2], words[3]);
}

// The largest of whole numbers over the wave, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  const auto move = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v = max(v, move(v, std::integral_constant<int, 0xB1>{}));
  v = max(v, move(v, std::integral_constant<int, 0x4E>{}));
  v = max(v, move(v, std::integral_constant<int, 0x141>{}));
  v = max(v, move(v, std::integral_constant<int, 0x140>{}));
  const auto lane = [&](int at) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), at)); };
  return max(max(lane(0), lane(16)), max(lane(32), lane(48)));
}

// Sums (and, as `most`, the largest of whole numbers) over the threads of a row, in each of them: within the wave, then through
// `slots` of the LDS, of which a workgroup uses another set for each reduction until a barrier lies between. Every thread of the
// workgroup comes by. A row of one wave needs no barrier.
template <int N>
struct RowSlots {
  uint32_t v[kMaxRowWaves][N];
};

template <int N, int M>
__device__ __forceinline__ void row_reduce(float (&sums)[N], uint32_t (&most)[M], int waves, RowSlots<N + M> &slots) {
#pragma unroll
  for (int i = 0; i < N; ++i) sums[i] = wave_sum(sums[i]);
#pragma unroll
  for (int i = 0; i < M; ++i) most[i] = wave_max(most[i]);
  if (waves == 1) return;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots.v[wave][i] = __float_as_uint(sums[i]);
#pragma unroll
    for (int i = 0; i < M; ++i) slots.v[wave][N + i] = most[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) sums[i] = 0.0f;
  for (int w = 0; w < waves; ++w) {
#pragma unroll
    for (int i = 0; i < N; ++i) sums[i] += __uint_as_float(slots.v[w][i]);
#pragma unroll
    for (int i = 0; i < M; ++i) most[i] = max(most[i], slots.v[w][N + i]);
  }
}

// first: the row's first wave, where a workgroup holds several rows.
template <int N>
__device__ __forceinline__ void row_reduce(float (&sums)[N], int waves, RowSlots<N> &slots, int first = 0) {
#pragma unroll
  for (int i = 0; i < N; ++i) sums[i] = wave_sum(sums[i]);
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slots.v[threadIdx.x >> 6][i] = __float_as_uint(sums[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) sums[i] = 0.0f;
  for (int w = first; w < first + waves; ++w)
#pragma unroll
    for (int i = 0; i < N; ++i) sums[i] += __uint_as_float(slots.v[w][i]);
}

// The largest alone.
__device__ __forceinline__ void row_largest(uint32_t &most, int waves, RowSlots<1> &slots) {
  most = wave_max(most);
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) slots.v[threadIdx.x >> 6][0] = most;
  __syncthreads();
  for (int w = 0; w < waves; ++w) most = max(most, slots.v[w][0]);
}

// ---------------------------------------------------------------- rows of 8-bit integers
constexpr uint32_t kInfinity = 0x7F800000u;

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// round(127 v / m), halves to even, for the values v of a row of largest magnitude m (given as its bits, whose order takes NaN
// for the largest). Both are scaled by the power of two that brings m to 1 .. 2, so neither 127 v nor 1 / m leaves f32; the
// quotient is corrected by its remainder, and so falls on a border where 127 v / m does: of 16-bit v and m, no other quotient
// is nearer to a border than 2^-19 of itself. A row of zeros has a scale of 0; one that holds an infinity or NaN a scale of NaN
// and elements of 0.
struct RowQuant {
  float times, most, inverse;
  bool finite;
  __device__ __forceinline__ explicit RowQuant(uint32_t bits) {
    finite = bits < kInfinity;
    const int up = min(254 - static_cast<int>(bits >> 23), 247);      // exponent of the power of two: 2^(up - 127), at most 2^120
    const float power = finite ? __uint_as_float(static_cast<uint32_t>(max(up, 1)) << 23) : 0.0f;
    times = 127.0f * power;
    most = finite ? __uint_as_float(bits) * power : 0.0f;
    inverse = most > 0.0f ? 1.0f / most : 0.0f;
  }
  // The integer in the low 8 bits.
  __device__ __forceinline__ uint32_t operator()(float v) const {
    const float wide = v * times;
    float q = wide * inverse;
    q = fmaf(fmaf(-q, most, wide), inverse, q);
    return __float_as_uint(q + 12582912.0f);                           // 1.5 * 2^23: the sum's last bit counts ones
  }
  __device__ __forceinline__ uint2 piece(const float (&v)[kPiece]) const {
    if (!finite) return make_uint2(0, 0);
    uint32_t b[kPiece];
#pragma unroll
    for (int i = 0; i < kPiece; ++i) b[i] = (*this)(v[i]);
    const auto pack = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
      return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
    };
    return make_uint2(pack(b[0], b[1], b[2], b[3]), pack(b[4], b[5], b[6], b[7]));
  }
};

// What an integer counts: m / 127.
__device__ __forceinline__ float row_scale(uint32_t bits) {
  return bits < kInfinity ? __uint_as_float(bits) / 127.0f : __uint_as_float(0x7FC00000u);
}

constexpr int kMaxRow = kPiece * kWave * kMaxRowWaves * 2;      // 16384 elements: two pieces of 16 waves' threads

// Waves of a row of `pieces` pieces a thread.
inline int row_waves(int64_t d, int pieces) {
  const int64_t of_wave = int64_t{kWave} * kPiece * pieces;
  return static_cast<int>((d + of_wave - 1) / of_wave);
}

}  // namespace intent_hip

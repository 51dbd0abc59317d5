// Rows made 8-bit integers with a scale each, plain or of silu(gate) * up, for gfx950. No reference counterpart.
//
//   a = x, or g / (1 + e^-g) * u in f32;  scale = max|a| / 127,  q = round(127 a / max|a|), halves to even (rows.hpp)
// of every row. A row of zeros has a scale of 0; one that holds an infinity or NaN a scale of NaN and elements of 0.
//
// e^-g and the reciprocal are the instructions' own, off by (|g| + 4) 2^-23 of themselves, so an element whose quotient lies within about 2^-16
// of a border may be its neighbour. With both corrected to f32's last bits the gated 16384 x 4096 took 71 us for 61, and as many elements of
// ordinary gates were others than in 64 bits: the roundings of a itself move them as far.
//
// Bound by the rows' bytes, which are read once: a row stays in the registers of its threads, up to four pieces of 16 bytes each,
// 32768 elements in all. Measured: 16384 x 4096 36.0 us (5.6 TB/s), the gated form 61 (5.5), 4096 x 14336 33 (5.3), 8192 x 8191, whose rows
// begin anywhere, 43 (4.6; two bytes at a time 90), 32 x 4096 4.3, a launch.
#include <stdio.h>

#include <algorithm>

#include "rows.hpp"

namespace intent_hip {
namespace {

constexpr int kWaveRows = 4;           // rows of a workgroup where a wave holds a row
constexpr int kMaxQuantRow = 2 * kMaxRow;

struct Quantize {
  const uint16_t *x, *up;              // up: null where x itself is made integers
  int8_t *q;
  float *scales;
  int64_t xs, us, qs;                  // strides of a row
  int64_t rows;
  int d, waves;
};

template <typename E, int P, int W, bool kPieces, bool kGated>
__global__ __launch_bounds__(W *kWave) void quantize_rows(Quantize p) {
  __shared__ RowSlots<1> slots;
  const int wave_rows = p.waves == 1 ? kWaveRows : 1;
  const int64_t row = static_cast<int64_t>(grid_block()) * wave_rows + (p.waves == 1 ? threadIdx.x >> 6 : 0);
  if (row >= p.rows) return;           // of a whole wave; of a row of several waves the whole workgroup
  const RowPlace<kPieces> at{p.d, p.waves * kWave, static_cast<int>(p.waves == 1 ? threadIdx.x & 63 : threadIdx.x)};
  uint4 x[P], up[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    x[j] = load_piece(p.x + row * p.xs, at, j);
    if constexpr (kGated) up[j] = load_piece(p.up + row * p.us, at, j);
  }
  float a[P][kPiece];
  uint32_t most[1] = {0};
#pragma unroll
  for (int j = 0; j < P; ++j) {
    widen_piece<E>(settled(x[j], at, j), a[j]);
    if constexpr (kGated) {
      float u[kPiece];
      widen_piece<E>(settled(up[j], at, j), u);
#pragma unroll
      for (int i = 0; i < kPiece; ++i) a[j][i] = a[j][i] * __builtin_amdgcn_rcpf(1.0f + __expf(-a[j][i])) * u[i];
    }
#pragma unroll
    for (int i = 0; i < kPiece; ++i) most[0] = max(most[0], magnitude(a[j][i]));
  }
  row_largest(most[0], p.waves, slots);
  const RowQuant quant(most[0]);
#pragma unroll
  for (int j = 0; j < P; ++j) store_piece(p.q + row * p.qs, at, j, quant.piece(a[j]));
  if (at.thread == 0) p.scales[row] = row_scale(most[0]);
}

// How a row lies over threads: pieces of a thread, and the waves that its kernel is built for. Two pieces from rows of 1024 on leave fewer
// waves to meet: 16384 x 2048 20.5 us, one piece 22.4; of 16384 x 1024 both take 13.0, and 8192 x 8192 takes 36.5 in two, 37.0 in four.
struct Layout {
  int pieces, most;
};
Layout layout_of(int64_t d) { return row_waves(d, 1) <= 2 ? Layout{1, 4} : row_waves(d, 2) <= 8 ? Layout{2, 8} : Layout{4, 16}; }

bool in_pieces(int64_t d, uint64_t wide, uint64_t narrow) { return d % kPiece == 0 && (wide | 2 * narrow) % 16 == 0; }

template <typename F>
int with_kernel(int dtype, int64_t d, bool whole, bool gated, F f) {
  const auto typed = [&](auto pieces, auto waves, auto in, auto two) {
    return f(dtype == INTENT_HIP_F16 ? quantize_rows<f16_t, pieces.value, waves.value, in.value, two.value>
                                     : quantize_rows<bf16_t, pieces.value, waves.value, in.value, two.value>);
  };
  const auto shaped = [&](auto in, auto two) {
    const int pieces = layout_of(d).pieces;
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> pair;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 8> eight;
    const std::integral_constant<int, 16> sixteen;
    return pieces == 1 ? typed(one, four, in, two) : pieces == 2 ? typed(pair, eight, in, two) : typed(four, sixteen, in, two);
  };
  if (whole) return gated ? shaped(std::true_type{}, std::true_type{}) : shaped(std::true_type{}, std::false_type{});
  return gated ? shaped(std::false_type{}, std::true_type{}) : shaped(std::false_type{}, std::false_type{});
}

unsigned row_threads(int waves) { return static_cast<unsigned>((waves == 1 ? kWaveRows : waves) * kWave); }
int layout_waves(int64_t d) { return std::max(1, row_waves(d, layout_of(d).pieces)); }

}  // namespace

int quantize_rows_resources(int dtype, int gated, int64_t d, uint64_t mix, IntentHipKernelResources *out) {
  if (d < 0 || d > kMaxQuantRow) return fail(INTENT_HIP_ERR_UNSUPPORTED, "quantize_rows takes rows of up to %d elements", kMaxQuantRow);
  const bool whole = in_pieces(d, mix, 0);
  char name[64];
  snprintf(name, sizeof(name), "quantize_rows<%s,%d,%s,%s>", dtype == INTENT_HIP_F16 ? "f16" : "bf16", layout_of(d).pieces,
           whole ? "true" : "false", gated ? "true" : "false");
  return with_kernel(dtype, d, whole, gated != 0, [&](void (*kernel)(Quantize)) {
    return describe_kernel(reinterpret_cast<const void *>(kernel), name, static_cast<int>(row_threads(layout_waves(d))), out);
  });
}

namespace {

int launch(const char *name, bool gated, int dtype, const void *x, const void *up, int8_t *output, float *scales, int64_t rows, int64_t d,
           const int64_t (&strides)[3], void *stream) {
  if (rows < 0 || d < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "%s dtype must be F16 or BF16, got %d", name, dtype);
  for (const int64_t s : strides)
    if (s < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  if (d > kMaxQuantRow)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "%s takes rows of up to %d elements, got %lld", name, kMaxQuantRow, static_cast<long long>(d));
  if (rows > (1 << 30)) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  if (rows == 0) return INTENT_HIP_OK;
  if (scales == nullptr || (d > 0 && (x == nullptr || output == nullptr || (gated && up == nullptr))))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  Quantize p{};
  p.x = static_cast<const uint16_t *>(x), p.up = static_cast<const uint16_t *>(up), p.q = output, p.scales = scales;
  p.xs = strides[0], p.us = strides[1], p.qs = strides[2], p.rows = rows, p.d = static_cast<int>(d), p.waves = layout_waves(d);
  const auto at = [](const void *a) { return static_cast<uint64_t>(reinterpret_cast<uintptr_t>(a)); };
  uint64_t wide = at(x) | (gated ? at(up) : 0), narrow = at(output);
  if (rows > 1) wide |= 2 * static_cast<uint64_t>(p.xs | (gated ? p.us : 0)), narrow |= static_cast<uint64_t>(p.qs);
  const int of_group = p.waves == 1 ? kWaveRows : 1;
  with_kernel(dtype, d, in_pieces(d, wide, narrow), gated, [&](void (*kernel)(Quantize)) {
    kernel<<<tile_grid((rows + of_group - 1) / of_group, 1), row_threads(p.waves), 0, as_stream(stream)>>>(p);
    return 0;
  });
  return hipPeekAtLastError() != hipSuccess ? launch_status(name) : INTENT_HIP_OK;
}

}  // namespace
}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_quantize_rows(int dtype, const void *x, int8_t *output, float *scales, int64_t rows, int64_t d, int64_t ldx,
                                        int64_t ldo, void *stream) {
  return launch("quantize_rows", false, dtype, x, nullptr, output, scales, rows, d, {ldx, 0, ldo}, stream);
}

extern "C" int intent_hip_swiglu_quantize_rows(int dtype, const void *gate, const void *up, int8_t *output, float *scales, int64_t rows,
                                               int64_t d, int64_t ldg, int64_t ldu, int64_t ldo, void *stream) {
  return launch("swiglu_quantize_rows", true, dtype, gate, up, output, scales, rows, d, {ldg, ldu, ldo}, stream);
}

// Rows written into and read back from a paged cache of e4m3 elements with a shared power of two per 32, for gfx950. No
// reference counterpart.
//
//   append  token i of the new tokens of sequence s, row cu[s] + i, is position lengths[s] - (cu[s + 1] - cu[s]) + i; it goes
//           to slot position % PS of the sequence's page position / PS. A block's exponent is the smallest e >= -127 with
//           max |x| <= 448 * 2^e over its finite values, its elements are e4m3(x * 2^-e), NaN and infinities held as NaN.
//   read    row cu[s] + i of the outputs is position i of sequence s: element * 2^e in the storage type; 0 where the tables
//           have no page.
//
// Rows behind cu[sequences], positions before 0 or behind the sequence's pages, and pages outside the cache are left alone.
//
// A wave takes a piece of 512 elements of up to 4 consecutive rows, all on their way at once: where its lanes' elements lie in
// a row is found once, and the tables are asked again only where a sequence or a page ends. Consecutive rows stay on one XCD,
// so the exponents of a page's tokens, which share lines, leave its L2 together. Bound by bytes (8 prompts of up to 8191, 8 key
// heads of 128: appended in 28.5 us, 5.1 TB/s; read in 30.5, 4.8 TB/s); a token for each of 32 sequences by latency, 3.3 us.
#include <stdio.h>

#include "mx.hpp"

namespace intent_hip {
namespace {

constexpr int kWaves = 4;

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

struct Rows {
  uint16_t *rows[2];                 // keys, values
  uint8_t *cache[2], *exponents[2];
  int64_t rs[2][2], cs[2][3], es[2][3];
  int chunks[2];                     // of 8 elements, per row: heads * width / 8
  int width[2];                      // chunks of a head
  const int32_t *cu, *lengths;
  PageTable table;
  int total, sequences;
  int blocks;
  int pieces;                        // of 64 chunks, per row: a wave's
};

// What a lane holds of a row: a chunk of the wave's piece, at the same place of every row.
struct Place {
  bool live, first;                  // first of its block: the lane that holds the exponent
  uint16_t *rows;                    // of the operand, at the chunk's head and place
  uint8_t *cache, *exponents;
  int64_t row_stride, page_stride, slot_stride, page_exponents, slot_exponents;
};
__device__ __forceinline__ Place place_of(const Rows &p, int chunk) {
  Place at{};
  at.live = chunk < p.chunks[0] + p.chunks[1];
  const bool value = chunk >= p.chunks[0];
  const unsigned in = value ? chunk - p.chunks[0] : chunk, width = value ? p.width[1] : p.width[0];
  const unsigned head = in / width, c = in - head * width;
  at.rows = (value ? p.rows[1] : p.rows[0]) + head * (value ? p.rs[1][1] : p.rs[0][1]) + c * 8;
  at.cache = (value ? p.cache[1] : p.cache[0]) + head * (value ? p.cs[1][2] : p.cs[0][2]) + c * 8;
  at.exponents = (value ? p.exponents[1] : p.exponents[0]) + head * (value ? p.es[1][2] : p.es[0][2]) + c / 4;
  at.row_stride = value ? p.rs[1][0] : p.rs[0][0];
  at.page_stride = value ? p.cs[1][0] : p.cs[0][0], at.slot_stride = value ? p.cs[1][1] : p.cs[0][1];
  at.page_exponents = value ? p.es[1][0] : p.es[0][0], at.slot_exponents = value ? p.es[1][1] : p.es[0][1];
  at.first = (c & 3) == 0;
  return at;
}

// Walks the rows of a wave: the sequence, position, page and place of each. Rows of one sequence follow each other, so the
// tables are asked again only where a sequence or a page ends.
struct Walk {
  int s, begin, end;                 // the sequence and its rows
  int shift;                         // position of a row: row + shift
  int first, held;                   // its logical pages
  int64_t page;                      // -1: none
  unsigned slot;
  bool none;                         // no sequence has the row

  __device__ __forceinline__ void sequence(const Rows &p, int row) {
    const int at = sequence_of(p.cu, p.sequences, row);
    none = at >= p.sequences;
    s = none ? p.sequences - 1 : at;
    // All that is known of the sequence is asked for at once.
    const int rows0 = p.cu[s], rows1 = p.cu[s + 1], pages0 = p.table.offsets[s], pages1 = p.table.offsets[s + 1];
    const int length = p.lengths != nullptr ? p.lengths[s] : rows1 - rows0;
    begin = none ? row : rows0, end = none ? INT32_MAX : rows1;
    if (row < begin || row >= end) none = true, end = row + 1;      // offsets that leave rows out, or do not rise
    shift = length - rows1;
    first = pages0, held = pages1 - pages0;
    locate(p, row);
  }
  __device__ __forceinline__ void locate(const Rows &p, int row) {
    const int64_t position = static_cast<int64_t>(row) + shift;
    page = -1;
    slot = 0;
    if (none || position < 0) return;
    const unsigned logical = static_cast<unsigned>(position) / static_cast<unsigned>(p.table.ps);
    slot = static_cast<unsigned>(position) - logical * p.table.ps;
    page = p.table.page(first, held, logical);
  }
  __device__ __forceinline__ void next(const Rows &p, int row) {
    if (row >= end) return sequence(p, row);
    if (page < 0 || ++slot >= static_cast<unsigned>(p.table.ps)) locate(p, row);
  }
};

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, 0xF, 0xF, false);
}

// R: consecutive rows that a wave holds at once. The elements of many rows (R > 1) are more than the L2s hold and pass them by
// (33.6 -> 28.9 us; with a reader of the rows behind it 65.2 -> 60.3). Not the exponents, whose bytes would reach memory one by
// one (35), nor what cache_read writes: alone it would take 23.6 us instead of 34.8, with the reader of its rows, who then finds
// none of them on the chip, 66.0 instead of 62.5.
template <typename E, int R>
__global__ __launch_bounds__(kWaves * kWave) void cache_append(Rows p) {
  constexpr uint32_t kMagnitude = 0x7FFF7FFFu, kInfinity = __is_same(E, f16_t) ? 0x7C00u : 0x7F80u;
  const int block = xcd_tile(grid_block(), p.blocks);
  if (block < 0) return;
  const int job = block * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = job / p.pieces * R, rows = min(R, p.total - first);
  if (rows <= 0) return;
  const Place at = place_of(p, job % p.pieces * kWave + (threadIdx.x & 63));
  uint4 raw[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    raw[i] = make_uint4(0, 0, 0, 0);
    if (i < rows && at.live) raw[i] = *reinterpret_cast<const uint4 *>(at.rows + (first + i) * at.row_stride);
  }
  int64_t page[R], slot[R];
  Walk walk;
  walk.sequence(p, first);
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i > 0 && i < rows) walk.next(p, first + i);
    page[i] = i < rows ? walk.page : -1, slot[i] = walk.slot;
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (page[i] < 0) continue;
    // The block's largest magnitude, two at a time; what is not finite is settled only where there is any.
    uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    uint32_t size = mx_larger(mx_larger(words[0] & kMagnitude, words[1] & kMagnitude),
                              mx_larger(words[2] & kMagnitude, words[3] & kMagnitude));
    if (__any(max(size & 0xFFFFu, size >> 16) >= kInfinity)) {
      size = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        size = mx_larger(size, mx_settled<E, false>(words[j]) & kMagnitude);
        words[j] = mx_settled<E, true>(words[j]);
      }
    }
    size = mx_larger(size, dpp_bits<0xB1>(size));
    size = mx_larger(size, dpp_bits<0x4E>(size));
    const int exponent = mx_exponent_e4m3(to_f32(E{static_cast<uint16_t>(max(size & 0xFFFFu, size >> 16))}));
    const float scale = mx_scale(exponent);
    const uint2 out = make_uint2(mx_quad_e4m3<E>(words[0], words[1], scale), mx_quad_e4m3<E>(words[2], words[3], scale));
    if (!at.live) continue;
    uint8_t *const to = at.cache + page[i] * at.page_stride + slot[i] * at.slot_stride;
    if constexpr (R > 1)
      __builtin_nontemporal_store(u32x2_t{out.x, out.y}, reinterpret_cast<u32x2_t *>(to));
    else
      *reinterpret_cast<uint2 *>(to) = out;
    if (at.first) at.exponents[page[i] * at.page_exponents + slot[i] * at.slot_exponents] = static_cast<uint8_t>(exponent);
  }
}

template <typename E, int R>
__global__ __launch_bounds__(kWaves * kWave) void cache_read(Rows p) {
  const int block = xcd_tile(grid_block(), p.blocks);
  if (block < 0) return;
  const int job = block * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int first = job / p.pieces * R, rows = min(R, p.total - first);
  if (rows <= 0) return;
  Walk walk;
  walk.sequence(p, first);
  const Place at = place_of(p, job % p.pieces * kWave + (threadIdx.x & 63));
  uint2 raw[R];
  uint8_t power[R];
  bool none[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i > 0 && i < rows) walk.next(p, first + i);
    none[i] = i >= rows || walk.none;
    raw[i] = make_uint2(0, 0);
    power[i] = 127;
    if (none[i] || walk.page < 0 || !at.live) continue;
    const int64_t slot = walk.slot;
    raw[i] = *reinterpret_cast<const uint2 *>(at.cache + walk.page * at.page_stride + slot * at.slot_stride);
    power[i] = at.exponents[walk.page * at.page_exponents + slot * at.slot_exponents];
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (none[i] || !at.live) continue;
    const float scale = mx_scale(power[i]);
    *reinterpret_cast<uint4 *>(at.rows + (first + i) * at.row_stride) =
        make_uint4(mx_pair_e4m3<E, false>(raw[i].x, scale), mx_pair_e4m3<E, true>(raw[i].x, scale),
                   mx_pair_e4m3<E, false>(raw[i].y, scale), mx_pair_e4m3<E, true>(raw[i].y, scale));
  }
}

// Rows of a wave: four where that still leaves every CU its 32 waves (23585 rows of 8 + 8 heads of 128: appended in 33.7 us before
// its stores passed the L2s by, one row a wave 43.5; read in 34.9 and 54.3), else one (32 rows: 4.4 us with the launch, four 5.7).
int together(int64_t rows, int64_t pieces) { return rows * pieces < 128 * device_cus() ? 1 : 4; }

// strides: k[3], v[3], then per cache its elements [4] and exponents [4].
int fill(Rows *p, int dtype, const void *k, const void *v, const void *key_cache, const uint8_t *key_exponents,
         const void *value_cache, const uint8_t *value_exponents, const int32_t *cu, const int32_t *page_offsets,
         const int32_t *page_indices, int64_t rows, int64_t sequences, int64_t kv_heads, int64_t d, int64_t dv, int64_t pages,
         int64_t ps, int64_t positions, const int64_t *strides) {
  if (dtype != INTENT_HIP_F16 && dtype != INTENT_HIP_BF16)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "paged cache rows must be F16 or BF16, got %d", dtype);
  if (rows < 0 || sequences < 0 || kv_heads < 0 || d < 0 || dv < 0 || pages < 0 || ps < 0 || positions < 0)
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative extent");
  if (d % kMxBlock || dv % kMxBlock)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "cache rows are blocks of %d elements (got widths %lld, %lld)", kMxBlock,
                static_cast<long long>(d), static_cast<long long>(dv));
  if (kv_heads > INT32_MAX / 64 || d > INT32_MAX / 64 || dv > INT32_MAX / 64 || sequences > INT32_MAX / 64 ||
      kv_heads * (d + dv) > INT32_MAX / 64 || ps > INT32_MAX || rows > INT32_MAX / 64)
    return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  if (rows == 0 || sequences == 0 || kv_heads == 0 || d + dv == 0) return INTENT_HIP_OK;
  if (ps < 1 && pages > 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "pages hold no token");
  if (strides == nullptr || cu == nullptr || page_offsets == nullptr || (positions > 0 && page_indices == nullptr) ||
      (d > 0 && k == nullptr) || (dv > 0 && v == nullptr) ||
      (pages > 0 && ((d > 0 && (key_cache == nullptr || key_exponents == nullptr)) ||
                     (dv > 0 && (value_cache == nullptr || value_exponents == nullptr)))))
    return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  for (int i = 0; i < 22; ++i)
    if (strides[i] < 0) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "negative stride");
  const void *row_pointers[2] = {k, v}, *caches[2] = {key_cache, value_cache};
  const uint8_t *exponents[2] = {key_exponents, value_exponents};
  const int64_t widths[2] = {d, dv};
  for (int i = 0; i < 2; ++i) {
    const int64_t *r = strides + 3 * i, *c = strides + 6 + 8 * i, *e = c + 4;
    if (widths[i] == 0) continue;
    if (r[2] != 1 || c[3] != 1 || (widths[i] > kMxBlock && e[3] != 1))
      return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "rows, elements and exponents need unit inner stride");
    if (r[0] % 8 || r[1] % 8 || !aligned(row_pointers[i], 16))
      return fail(INTENT_HIP_ERR_UNSUPPORTED, "rows must be 16-byte aligned, their strides multiples of 8 elements");
    if (c[0] % 16 || c[1] % 16 || c[2] % 16 || !aligned(caches[i], 16))
      return fail(INTENT_HIP_ERR_UNSUPPORTED, "cache elements must be 16-byte aligned, their strides multiples of 16");
    p->rows[i] = static_cast<uint16_t *>(const_cast<void *>(row_pointers[i]));
    p->cache[i] = static_cast<uint8_t *>(const_cast<void *>(caches[i]));
    p->exponents[i] = const_cast<uint8_t *>(exponents[i]);
    for (int j = 0; j < 2; ++j) p->rs[i][j] = r[j];
    for (int j = 0; j < 3; ++j) p->cs[i][j] = c[j], p->es[i][j] = e[j];
  }
  for (int i = 0; i < 2; ++i) {
    p->width[i] = static_cast<int>(widths[i] / 8 > 0 ? widths[i] / 8 : 1);
    p->chunks[i] = static_cast<int>(kv_heads * widths[i] / 8);
  }
  p->cu = cu;
  p->table = {page_offsets, page_indices, positions, pages, static_cast<int>(ps > 0 ? ps : 1)};
  p->total = static_cast<int>(rows);
  p->sequences = static_cast<int>(sequences);
  p->pieces = (p->chunks[0] + p->chunks[1] + kWave - 1) / kWave;
  if (rows * p->pieces > INT32_MAX / 2) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  p->blocks = static_cast<int>(((rows + together(rows, p->pieces) - 1) / together(rows, p->pieces) * p->pieces + kWaves - 1) / kWaves);
  return INTENT_HIP_OK;
}

}  // namespace

// width: elements of a row, of all key heads' keys and values.
int paged_cache_resources(int dtype, int reading, int64_t rows, int64_t width, IntentHipKernelResources *out) {
  const bool half = dtype == INTENT_HIP_F16;
  const int r = together(rows, (width / 8 + kWave - 1) / kWave);
  char name[64];
  snprintf(name, sizeof(name), "cache_%s<%s,%d>", reading ? "read" : "append", half ? "f16" : "bf16", r);
  const auto describe = [&](const void *one, const void *four) { return describe_kernel(r == 1 ? one : four, name, kWaves * kWave, out); };
  if (reading)
    return half ? describe(reinterpret_cast<const void *>(cache_read<f16_t, 1>), reinterpret_cast<const void *>(cache_read<f16_t, 4>))
                : describe(reinterpret_cast<const void *>(cache_read<bf16_t, 1>), reinterpret_cast<const void *>(cache_read<bf16_t, 4>));
  return half ? describe(reinterpret_cast<const void *>(cache_append<f16_t, 1>), reinterpret_cast<const void *>(cache_append<f16_t, 4>))
              : describe(reinterpret_cast<const void *>(cache_append<bf16_t, 1>), reinterpret_cast<const void *>(cache_append<bf16_t, 4>));
}

}  // namespace intent_hip

using namespace intent_hip;

extern "C" int intent_hip_paged_cache_append(int dtype, const void *k, const void *v, void *key_cache, uint8_t *key_exponents,
                                             void *value_cache, uint8_t *value_exponents, const int32_t *cu_seqlens,
                                             const int32_t *page_offsets, const int32_t *page_indices, const int32_t *lengths,
                                             int64_t rows, int64_t sequences, int64_t kv_heads, int64_t d, int64_t dv,
                                             int64_t pages, int64_t ps, int64_t positions, const int64_t *strides, void *stream) {
  Rows p{};
  if (int rc = fill(&p, dtype, k, v, key_cache, key_exponents, value_cache, value_exponents, cu_seqlens, page_offsets,
                    page_indices, rows, sequences, kv_heads, d, dv, pages, ps, positions, strides))
    return rc;
  if (rows == 0 || sequences == 0 || kv_heads == 0 || d + dv == 0 || pages == 0 || positions == 0) return INTENT_HIP_OK;
  if (lengths == nullptr) return fail(INTENT_HIP_ERR_INVALID_ARGUMENT, "null pointer");
  p.lengths = lengths;
  const dim3 grid = tile_grid(p.blocks, 1);
  const bool half = dtype == INTENT_HIP_F16;
  if (together(p.total, p.pieces) == 1)
    (half ? cache_append<f16_t, 1> : cache_append<bf16_t, 1>)<<<grid, kWaves * kWave, 0, as_stream(stream)>>>(p);
  else
    (half ? cache_append<f16_t, 4> : cache_append<bf16_t, 4>)<<<grid, kWaves * kWave, 0, as_stream(stream)>>>(p);
  return hipPeekAtLastError() != hipSuccess ? launch_status("cache_append") : INTENT_HIP_OK;
}

extern "C" int intent_hip_paged_cache_read(int dtype, const void *key_cache, const uint8_t *key_exponents,
                                           const void *value_cache, const uint8_t *value_exponents, const int32_t *cu_seqlens,
                                           const int32_t *page_offsets, const int32_t *page_indices, void *k, void *v,
                                           int64_t rows, int64_t sequences, int64_t kv_heads, int64_t d, int64_t dv,
                                           int64_t pages, int64_t ps, int64_t positions, const int64_t *strides, void *stream) {
  Rows p{};
  if (int rc = fill(&p, dtype, k, v, key_cache, key_exponents, value_cache, value_exponents, cu_seqlens, page_offsets,
                    page_indices, rows, sequences, kv_heads, d, dv, pages, ps, positions, strides))
    return rc;
  if (rows == 0 || sequences == 0 || kv_heads == 0 || d + dv == 0) return INTENT_HIP_OK;
  const dim3 grid = tile_grid(p.blocks, 1);
  const bool half = dtype == INTENT_HIP_F16;
  if (together(p.total, p.pieces) == 1)
    (half ? cache_read<f16_t, 1> : cache_read<bf16_t, 1>)<<<grid, kWaves * kWave, 0, as_stream(stream)>>>(p);
  else
    (half ? cache_read<f16_t, 4> : cache_read<bf16_t, 4>)<<<grid, kWaves * kWave, 0, as_stream(stream)>>>(p);
  return hipPeekAtLastError() != hipSuccess ? launch_status("cache_read") : INTENT_HIP_OK;
}

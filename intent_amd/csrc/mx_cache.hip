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
#include "mx.hpp"

namespace intent_hip {
namespace {

constexpr int kWaves = 4;

struct Rows {
  uint16_t *rows[2];                 // keys, values
  uint8_t *cache[2], *exponents[2];
  int64_t rs[2][2], cs[2][3], es[2][3];
  int chunks[2];                     // of 8 elements, per row: heads * width / 8
  int width[2];                      // chunks of a head
  const int32_t *cu, *lengths;
  PageTable table;
  int64_t total;
  int sequences, pieces;             // pieces: waves per row
};

// Which operand, head and chunk of it a lane's chunk of a row is.
struct Chunk {
  int which, head, at;
};
__device__ __forceinline__ Chunk chunk_of(const Rows &p, int chunk) {
  const int which = chunk >= p.chunks[0];
  if (which) chunk -= p.chunks[0];
  return {which, chunk / p.width[which], chunk % p.width[which]};
}

// One wave per 64 chunks of a row; a lane holds 8 elements, a quad of lanes a block.
template <typename E>
__global__ __launch_bounds__(kWaves * kWave) void cache_append(Rows p) {
  const int64_t job = static_cast<int64_t>(grid_block()) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = job / p.pieces;
  if (row >= p.total) return;
  const int lane = threadIdx.x & 63;
  const int s = sequence_of(p.cu, p.sequences, row);
  if (s >= p.sequences) return;
  const int64_t begin = p.cu[s], end = p.cu[s + 1];
  if (row < begin) return;
  const int64_t position = static_cast<int64_t>(p.lengths[s]) - (end - begin) + (row - begin);
  if (position < 0) return;
  const int64_t page = p.table.page(s, position / p.table.ps);
  if (page < 0) return;
  const int64_t slot = position % p.table.ps;
  const int chunk = static_cast<int>(job % p.pieces) * kWave + lane;
  const bool live = chunk < p.chunks[0] + p.chunks[1];
  const Chunk c = chunk_of(p, live ? chunk : 0);
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (live)
    raw = *reinterpret_cast<const uint4 *>(p.rows[c.which] + row * p.rs[c.which][0] + c.head * p.rs[c.which][1] + c.at * 8);
  const uint16_t *bits = reinterpret_cast<const uint16_t *>(&raw);
  float v[8], size = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = to_f32(E{bits[i]});
    const float a = fabsf(v[i]);
    size = fmaxf(size, a < INFINITY ? a : 0.0f);
  }
  size = fmaxf(size, dpp_move<0xB1>(size));
  size = fmaxf(size, dpp_move<0x4E>(size));
  const int exponent = mx_exponent_e4m3(size);
  const float scale = mx_scale(exponent);
  const uint2 out = make_uint2(mx_quad_e4m3(v[0], v[1], v[2], v[3], scale), mx_quad_e4m3(v[4], v[5], v[6], v[7], scale));
  if (!live) return;
  const int64_t *cs = p.cs[c.which], *es = p.es[c.which];
  *reinterpret_cast<uint2 *>(p.cache[c.which] + page * cs[0] + slot * cs[1] + c.head * cs[2] + c.at * 8) = out;
  if ((c.at & 3) == 0)
    p.exponents[c.which][page * es[0] + slot * es[1] + c.head * es[2] + c.at / 4] = static_cast<uint8_t>(exponent);
}

template <typename E>
__global__ __launch_bounds__(kWaves * kWave) void cache_read(Rows p) {
  const int64_t job = static_cast<int64_t>(grid_block()) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = job / p.pieces;
  if (row >= p.total) return;
  const int lane = threadIdx.x & 63;
  const int s = sequence_of(p.cu, p.sequences, row);
  if (s >= p.sequences) return;
  const int64_t begin = p.cu[s];
  if (row < begin) return;
  const int64_t position = row - begin;
  const int64_t page = p.table.page(s, position / p.table.ps);
  const int64_t slot = position % p.table.ps;
  const int chunk = static_cast<int>(job % p.pieces) * kWave + lane;
  if (chunk >= p.chunks[0] + p.chunks[1]) return;
  const Chunk c = chunk_of(p, chunk);
  uint4 out = make_uint4(0, 0, 0, 0);
  if (page >= 0) {
    const int64_t *cs = p.cs[c.which], *es = p.es[c.which];
    const uint2 raw =
        *reinterpret_cast<const uint2 *>(p.cache[c.which] + page * cs[0] + slot * cs[1] + c.head * cs[2] + c.at * 8);
    const float scale = mx_scale(p.exponents[c.which][page * es[0] + slot * es[1] + c.head * es[2] + c.at / 4]);
    out = make_uint4(mx_pair_e4m3<E, false>(raw.x, scale), mx_pair_e4m3<E, true>(raw.x, scale),
                     mx_pair_e4m3<E, false>(raw.y, scale), mx_pair_e4m3<E, true>(raw.y, scale));
  }
  *reinterpret_cast<uint4 *>(p.rows[c.which] + row * p.rs[c.which][0] + c.head * p.rs[c.which][1] + c.at * 8) = out;
}

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
      kv_heads * (d + dv) > INT32_MAX / 64 || ps > INT32_MAX || rows > int64_t{1} << 31)
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
  p->total = rows;
  p->sequences = static_cast<int>(sequences);
  p->pieces = (p->chunks[0] + p->chunks[1] + kWave - 1) / kWave;
  if ((rows * p->pieces + kWaves - 1) / kWaves > INT32_MAX) return fail(INTENT_HIP_ERR_UNSUPPORTED, "extents too large");
  return INTENT_HIP_OK;
}

dim3 grid(const Rows &p) { return tile_grid((p.total * p.pieces + kWaves - 1) / kWaves, 1); }

}  // namespace

int paged_cache_resources(int dtype, int reading, IntentHipKernelResources *out) {
  const bool half = dtype == INTENT_HIP_F16;
  if (reading)
    return half ? describe_kernel(reinterpret_cast<const void *>(cache_read<f16_t>), "cache_read<f16>", kWaves * kWave, out)
                : describe_kernel(reinterpret_cast<const void *>(cache_read<bf16_t>), "cache_read<bf16>", kWaves * kWave, out);
  return half ? describe_kernel(reinterpret_cast<const void *>(cache_append<f16_t>), "cache_append<f16>", kWaves * kWave, out)
              : describe_kernel(reinterpret_cast<const void *>(cache_append<bf16_t>), "cache_append<bf16>", kWaves * kWave, out);
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
  if (dtype == INTENT_HIP_F16)
    cache_append<f16_t><<<grid(p), kWaves * kWave, 0, as_stream(stream)>>>(p);
  else
    cache_append<bf16_t><<<grid(p), kWaves * kWave, 0, as_stream(stream)>>>(p);
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
  if (dtype == INTENT_HIP_F16)
    cache_read<f16_t><<<grid(p), kWaves * kWave, 0, as_stream(stream)>>>(p);
  else
    cache_read<bf16_t><<<grid(p), kWaves * kWave, 0, as_stream(stream)>>>(p);
  return hipPeekAtLastError() != hipSuccess ? launch_status("cache_read") : INTENT_HIP_OK;
}

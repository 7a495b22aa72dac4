// The 4-bit key/value cache: where its rows lie, and the launch interface of
// its kernels.
//
// A row (one token's key or value of one head) is hd channels in groups of
// 32, G = ceil(hd / 32).  A group has a scale s and an offset m, both bf16,
// and per channel a 4-bit code c that stands for m + c s:
//
//   m = the largest bf16 at most min(x)
//   s = the smallest bf16 >= 2^-126 with 15 s >= max(x) - m (0 if max(x) = m)
//   c = the number of borders m + (k + 1/2) s, k = 0..14, below x
//
// so |x - (m + c s)| <= s / 2.  Asymmetric codes with a 16-bit scale and
// offset (5 bits per channel in all) halve the squared error that the fp4
// format with its own block scale has on normal values; every step of the
// definition is a comparison of exactly representable numbers, so the codes
// do not depend on how they are computed.
//
//   codes   uint8 [pages, heads, page, 16 G]: the dword of channels
//           32 g + 8 o .. + 7 (nibble j: channel j) is dword 4 g + o of a
//           value row and dword G o + g of a key row.  The key order gives
//           MFMA lane group o the o-th octet of every channel group in
//           4 G consecutive bytes: a wave's operands for 16 keys are one
//           load per lane of one contiguous 1 KB (hd = 128).
//   params  bf16 pairs [pages, heads, page, G]: s in the low half of a
//           dword, m in the high half.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "asa_launch.hpp"

namespace asa {

struct CachePool {
  int pages, heads, page, page_shift, hd, G;
  uint8_t* k_codes;
  uint8_t* v_codes;
  uint32_t* k_params;
  uint32_t* v_params;
};

// The row of position `t` of a sequence with page table row `table` (`cols`
// entries): page * heads * page_size + offset within the page, to which the
// head's h * page_size is added; -1 where no page of the pool holds it.
__device__ __forceinline__ int64_t cache_row(const CachePool& c, const int32_t* table, int cols,
                                             int t, int h) {
  const int pi = t >> c.page_shift;
  if (t < 0 || pi >= cols) return -1;
  const int pg = table[pi];
  if (pg < 0 || pg >= c.pages) return -1;
  return (int64_t(pg) * c.heads + h) * c.page + (t & (c.page - 1));
}

struct CacheRowsParams {
  CachePool c;
  int B, n, cols;
  const int32_t* table;  // [B, cols]
  const int32_t* start;  // [B] position of token 0; nullptr: 0
  const int32_t* limit;  // write: [B] tokens of each sequence; nullptr: n
                         // read: [B] first position without a token
  const void* k;         // write: [B, heads, n, hd] by strides
  const void* v;
  void* ok;              // read: [B, heads, n, hd] contiguous
  void* ov;
  Lay lk, lv;
  bool chunks;           // 16-byte chunks: every row starts on one and hd % 8 == 0
};
hipError_t launch_cache_write(const CacheRowsParams& p, int dtype, hipStream_t s);
hipError_t launch_cache_read(const CacheRowsParams& p, int dtype, hipStream_t s);

struct CacheAttnParams {
  CachePool c;
  int B, H, NQ, cols, maxlen;
  int rep, R;             // query heads per key head; rows per key head: rep * NQ
  const int32_t* table;   // [B, cols]
  const int32_t* lengths; // [B]
  const int32_t* q_idx;   // [B, NQ] or nullptr: lengths - NQ + i
  const void* q;
  Lay lq;
  bool chunks;            // as above, for q
  void* out;              // [B, H, NQ, hd] contiguous
  float alpha, scale;
  float e, zc, zb;        // 1 / (alpha - 1), (alpha - 1) |scale|, 10 (alpha - 1)
  int pc;                 // pow_class_of(e)
  int plan;               // CachePlan
  int span, nsplit;       // split plan: keys per score block, score blocks per row tile
  int tile_rows;          // split plan: query rows that share a score block
  // split plan, rows = min(tile_rows, R), tiles of them per key head, n =
  // span * nsplit: dots [B * c.heads, tiles, n / 64, rows, 64], and each 64
  // keys' maxima [B * c.heads, tiles, rows, n / 64]
  float* scores;
  float* gmax;
};
// How attention runs: one block per 16 rows that holds their scores in LDS,
// or the keys split over score blocks, then one block per row.
enum CachePlan : int { kCacheOneBlock = 0, kCacheSplit = 1 };
// Keys whose maxima are kept together, and the static LDS of a one-block
// kernel beside its dots (an upper bound).
constexpr int kCacheGranule = 64;
constexpr size_t kCacheOneStatic = 45056;
// One-block plan: dynamic LDS bytes, and the keys of a row there.
inline size_t cache_one_lds(const CacheAttnParams& p, int* stride) {
  const int rows = p.R < p.tile_rows ? p.R : p.tile_rows;
  *stride = (p.maxlen + kCacheGranule - 1) / kCacheGranule * kCacheGranule;
  return size_t(rows) * (*stride + *stride / kCacheGranule) * 4 +
         size_t((p.maxlen + p.c.page - 1) / p.c.page + 1) * 4;
}
// Rows of the workspace's tensors (B * c.heads * tiles * rows).
size_t cache_score_rows(const CacheAttnParams& p);
// Fills plan, span, nsplit and tile_rows; returns the workspace bytes.
size_t cache_attn_plan(CacheAttnParams& p, int dtype, size_t max_lds, int cus);
hipError_t launch_cache_attn(const CacheAttnParams& p, int dtype, hipStream_t s);
// By the queries' type (one translation unit each).
hipError_t launch_cache_attn_bf16(const CacheAttnParams& p, hipStream_t s);
hipError_t launch_cache_attn_f16(const CacheAttnParams& p, hipStream_t s);
hipError_t launch_cache_attn_f32(const CacheAttnParams& p, hipStream_t s);

}  // namespace asa

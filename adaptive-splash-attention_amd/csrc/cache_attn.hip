// How attention over the 4-bit cache runs, and its dispatch by type.
#include "asa_cache.hpp"
#include "asa_device.hpp"

namespace asa {

size_t cache_score_rows(const CacheAttnParams& p) {
  const int rows = p.R < p.tile_rows ? p.R : p.tile_rows;
  return size_t(p.B) * p.c.heads * ((p.R + rows - 1) / rows) * rows;
}

size_t cache_attn_plan(CacheAttnParams& p, int dtype, size_t max_lds, int cus) {
  // Rows of a tile: as few as hold the call's, so that as many key tiles as
  // possible share a result; fp32 queries (three operand reads of LDS for
  // each key tile) share two at most.
  p.tile_rows = p.R > 8 ? 16 : p.R > 4 || dtype == kElemF32 ? 8 : 4;
  const long long nrt = (p.R + p.tile_rows - 1) / p.tile_rows, tiles = (long long)p.B * p.c.heads * nrt;
  // One launch or two.  With a tile of rows for nearly every compute unit one
  // block each is faster as long as two fit a unit's LDS (head dimension 128,
  // four rows per key head, us with one launch / two: 256 tiles of 512 keys
  // 13.4 / 17.7, of 4096 29.1 / 33.6; 1024 tiles of 2048 53 / 71).  Fewer
  // tiles leave units idle that split keys would use (8 tiles of 2048 keys
  // 17.1 / 11.7, 64 tiles 17.7 / 14.1), but the second launch is not made up
  // for by few bytes of keys (8 tiles of 512: 11.4 / 11.5) unless a block has
  // more rows than waves (16 rows, 8 tiles of 300: 18.5 / 13.1).
  int stride = 0;
  const size_t lds = cache_one_lds(p, &stride);
  p.span = p.nsplit = 0;
  const bool many = tiles >= cus * 3 / 4 && lds <= 72 * 1024;
  const bool few = (long long)p.maxlen * p.c.G <= 2048 && p.R <= 8;
  if ((many || few) && lds + kCacheOneStatic <= max_lds) {
    p.plan = kCacheOneBlock;
    return 0;
  }
  p.plan = kCacheSplit;
  // Four score blocks per compute unit (what its registers hold), of at least
  // 256 keys (the largest page: a block starts on a page) and at most 2048
  // (1 x 131072: 21.0 us against 22.4 with eight of 512 keys; 16 x 32768: 85
  // against 88 with four of 4096, whose last ones run alone).
  long long span = (p.maxlen * tiles + 4LL * cus - 1) / (4LL * cus);
  span = (span + 255) / 256 * 256;
  if (span > 2048) span = 2048;
  p.span = int(span);
  p.nsplit = int((p.maxlen + span - 1) / span);
  return cache_score_rows(p) * p.nsplit * (size_t(p.span) + p.span / kCacheGranule) * sizeof(float);
}

hipError_t launch_cache_attn(const CacheAttnParams& call, int dtype, hipStream_t s) {
  CacheAttnParams p = call;
  p.e = 1.0f / (p.alpha - 1.0f);
  p.pc = pow_class_of(p.e);
  p.zc = (p.alpha - 1.0f) * (p.scale < 0.0f ? -p.scale : p.scale);
  p.zb = 10.0f * (p.alpha - 1.0f);
  if (dtype == kElemBF16) return launch_cache_attn_bf16(p, s);
  if (dtype == kElemF16) return launch_cache_attn_f16(p, s);
  return launch_cache_attn_f32(p, s);
}

}  // namespace asa

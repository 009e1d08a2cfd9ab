// Parameters of the eviction by accumulated attention weight (evict.cu).
#pragma once
#include "common.cuh"

namespace dab {

constexpr int EVICT_MAX_ROWS = 9;     // the mass among them
constexpr int EVICT_MIN_TILE = 32;
constexpr int EVICT_MAX_BYTES = 4096;  // of an entry's rows together

struct EvictParams {
  float* mass; int64_t mb, mh;           // [B, H, cap], strides in elements
  int32_t* lengths; int64_t lb, lh;      // [B, H]
  // row buffers moved with the mass: base, strides over batch and head in bytes, bytes per row,
  // and the widest unit (4, 8 or 16 bytes) that its base, strides and rows are multiples of
  uint8_t* row[EVICT_MAX_ROWS];
  int64_t rb[EVICT_MAX_ROWS], rh[EVICT_MAX_ROWS];
  int bytes[EVICT_MAX_ROWS], unit[EVICT_MAX_ROWS], shift[EVICT_MAX_ROWS];  // log2(units a row), or -1
  int n_rows;
  int B, H, cap;
  int budget, trigger, first, recent;
  int tile, tile_shift;                  // entries per moved tile, a power of two
  int max_tiles, max_words;              // of a full head: tiles, words of 32 entries
  // workspace: error word; per head (threshold key, ties kept, length or 0 if left alone, ticket);
  // per head and tile (kept, ties before it); per tile of the result whether its rows have been read,
  // and the tile its first entry comes from with (kept, ties before that); per 32 entries (surely
  // kept, ties)
  int* err;
  uint4* cut;
  uint2* before;
  uint32_t* loaded;
  uint4* begins;
  uint2* words;
};

}  // namespace dab

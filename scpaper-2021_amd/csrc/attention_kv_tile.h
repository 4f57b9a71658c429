// Attention over a cache for many rows a key/value head (attention_kv_tile.hip): what its callers need.
#pragma once
#include "attention_kv.hip.h"

namespace et {

struct KvTilePlan {
    int blocks, splits, waves;  // waves: of a block, which has 32 rows for each
    size_t bytes;
};
template <int HD> constexpr int kTilePart = (2 + HD / 2) * 64;  // floats that a wave of a shared-out block leaves: references, sums, values, a lane's side by side with the others'

// Waves of a block for rows that are many enough, and whether there is work enough as well: workgroups times 32 keys.  Against 16 rows a wave (attention_kv.hip.h), us, 4 bits (8 bits):
//   heads of 128, 16 sequences of 2000, 8 heads: 64 rows 63.7 | 60.7 (60.5 | 63.7)   96 rows 64.0 | 83.5 (60.2 | 87.3)   256 rows 84.5 | 167 (86.0 | 176)   400 rows 131 | 266 (132 | 280)
//   of 96, the same: 96 rows 63.9 | 63.6, 128 rows 65.1 | 68.1, 256 rows 82.7 | 123;   of 64, 16 heads: 64 rows 67.4 | 53.6, 96 rows 64.7 | 73.0, 256 rows 92.4 | 171;   of 32: 128 rows 61.1 | 58.2, 160 rows 66.4 | 70.5
//   one sequence of 30000, 4 heads: of 128 96 rows 52.1 | 51.5, 256 rows 60.9 | 85.4;   of 64 128 rows 40.2 | 31.8, 256 rows 48.4 | 47.3, 400 rows 55.3 | 81.1
//   8 heads of 128: 1 x 1000, 400 rows (496 of those units) 25.3 | 19.7;   2 x 4000, 128 rows (2000) 32.2 | 41.8;   4 x 3000, 128 rows (3000) 34.6 | 46.9
//   8 sequences of 512 rows, 8 heads of 64, a window of 1 (1536 units) 25.3 | 17.0, 128 (2048) 27.1 | 23.4, 256 (2560) 30.2 | 28.3, 512 (3584) 35.5 | 37.3;   2 of 2048, 4 heads, 512 (1792) 27.8 | 20.8;   8 of 512, 8 heads of 96, 256 (2560) 38.2 | 37.8,
//   512 (3584) 46.3 | 50.5;   of 128, a window of 1 (1536) 30.6 | 34.0, 512 48.4 | 69.2;   1 of 4096, 2 heads of 128 with four each, a window of 1 (1536) 34.9 | 33.9, 64 (1792) 29.6 | 36.8
//   of 128 and up to 64 rows, two waves a block: 16 x 2000, 40 rows 46.8 | 52.8, 64 rows 48.2 | 60.6 (47.6 | 63.6), with unequal lengths 45.3 | 48.9;   64 x 2000 130 | 171, unequal 116 | 106;   2 x 8000 (4016 units)
//   38.8 | 41.7, 4 x 3000 (3040) 34.4 | 34.7, 8 x 1000 (2048) 26.1 | 21.6, 1 x 30000, 4 heads (3756) 49.3 | 39.6, 8 heads (7512) 57.1 | 54.4
int kv_tile_most_waves(int hd, long long rows);  // 0: none
int kv_tile_waves(const et_kv_cache *c, long long positions, int B, long long rows);
int kv_tile_plan(const char *fn, KvTilePlan &p, const et_kv_cache *c, long long positions, int B, int n, int nh, int waves);
int kv_tile_run(const char *fn, const KvMhaCall &call, long long positions, int waves, size_t need, KvSightArgs &a, et_stream stream);  // need: bytes of workspace; a: the rows' sight

}  // namespace et

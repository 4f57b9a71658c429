// Attention over a cache for many rows a key/value head (attention_kv_tile.hip): what its callers need.
#pragma once
#include "attention_kv.hip.h"

namespace et {

struct KvTilePlan {
    int blocks, splits, waves;  // waves: of a block, which has 32 rows for each
    size_t bytes;
};
template <int HD> constexpr int kTilePart = (2 + HD / 2) * 64;  // floats that a wave of a shared-out block leaves: references, sums, values, a lane's side by side with the others'

// Waves of a block for rows that are many enough, and whether there is work enough as well: workgroups times 32 keys.  Against 16 rows a wave (attention_kv.hip.h), us, 4 bits unless it is said (in
// brackets: starts anywhere in a sequence and counts of any size up to the rows, which a call does not tell and the rule does not follow):
//   16 sequences of 2000, 8 heads of 128: 64 rows, eight waves 65.2 | 64.5, 8 bits 65.4 | 67.3;   96 rows 69.4 | 93.2 (56.1 | 52.9), 8 bits 70.9 | 102;   128 rows 75.3 | 98.7 (58.3 | 49.5);   256 rows 108 | 188
//   (72.5 | 94.9), 8 bits 112 | 200;   400 rows 155 | 264 (107 | 123)
//   the same of 96: 64 rows 56.5 | 52.2 (48.0 | 33.8), 96 rows 60.1 | 70.4 (49.4 | 41.8), 128 rows 63.6 | 77.0 (50.9 | 45.1), 256 rows 93.0 | 143 (64.8 | 73.0)
//   16 heads of 64: 64 rows 78.3 | 56.6, 80 rows 80.5 | 67.7, 96 rows 82.3 | 81.8 (67.3 | 41.6), 8 bits 82.6 | 88.3;   112 rows 84.2 | 93.5 (69.5 | 42.4), 128 rows 84.5 | 103 (71.3 | 46.4), 8 bits 85.6 | 114;   256 rows
//   119 | 195 (86.5 | 78.9)
//   16 heads of 32: 96 rows 59.7 | 50.4, 128 rows 60.8 | 65.2 (53.2 | 39.8), 160 rows 71.4 | 79.9 (55.1 | 40.6), 256 rows 79.8 | 121 (63.5 | 53.8)
//   one sequence of 30000, 4 heads: of 128 96 rows 52.2 | 52.6, 128 rows 53.0 | 56.2, 256 rows 63.9 | 88.5;   of 96 (3752 of those units) 128 rows 47.2 | 45.3, 256 rows 55.9 | 71.0;   of 64 (3752) 128 rows
//   42.6 | 32.0, 256 rows 50.8 | 49.1, 400 rows (7504) 57.8 | 81.1;   of 32 256 rows 38.7 | 36.0, 400 rows 42.1 | 56.8
//   8 heads of 128: 1 x 1000, 400 rows (512) 21.4 | 18.3;   1 x 1500 (768) 23.5 | 23.6;   1 x 2000 (1024) 26.3 | 38.9;   2 x 2000, 128 rows (1024) 23.1 | 24.2;   4 x 1000 (1024) 21.6 | 19.3;   1 x 4000 (1008)
//   27.1 | 25.2;   2 x 4000 (2016) 30.4 | 43.2;   4 x 3000 (3008) 36.1 | 50.6;   windows of 1: 8 of 512 rows (1664) 29.4 | 35.1, 4 (832) 21.9 | 18.9, of 2 heads with four each 4096 rows (896) 18.6 | 35.0
//   8 sequences of 512 rows, 8 heads of 64: a window of 1 (1664) 24.6 | 16.5, 128 (2048) 25.9 | 22.8, 256 (2048) 29.5 | 25.1, 512 (2048) 26.9 | 27.5;   2 of 2048, 4 heads, 512 (1792) 26.9 | 21.6;   4 x 1000, 16 heads,
//   128 rows (2048) 21.1 | 26.2, 8 (4096) 32.7 | 32.1, 16 (8192) 49.5 | 58.2;   8 of 512, 8 heads of 96, 256 (2048) 35.2 | 35.4, 512 (2048) 33.5 | 38.5;   8 x 1000, 16 heads of 32, 160 rows (4096) 27.8 | 26.6, 4 x 2000 (4032)
//   25.5 | 30.2
//   of 128 and up to 64 rows, two waves a block: 16 x 2000, 40 rows 46.7 | 54.7 (37.8 | 33.2), 64 rows 47.4 | 64.5 (35.5 | 39.3), 8 bits 49.3 | 67.3;   64 x 2000 147 | 189 (103 | 89.1);   2 x 8000 (4000 units)
//   37.5 | 41.6, 4 x 3000 (3008) 30.5 | 36.1 (24.0 | 22.4), 8 x 1000 (2048) 23.1 | 19.1, 1 x 30000, 4 heads (3752) 49.1 | 39.5, 8 heads (7504) 57.1 | 59.6
int kv_tile_most_waves(int hd, long long rows);  // 0: none
int kv_tile_waves(const et_kv_cache *c, long long positions, int B, long long rows);
int kv_tile_plan(const char *fn, KvTilePlan &p, const et_kv_cache *c, long long positions, int B, int n, int nh, int waves);
int kv_tile_run(const char *fn, const KvMhaCall &call, long long positions, int waves, size_t need, KvSightArgs &a, et_stream stream);  // need: bytes of workspace; a: the rows' sight

}  // namespace et

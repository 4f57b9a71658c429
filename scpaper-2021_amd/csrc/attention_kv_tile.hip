// Attention over a cache of keys and values in 4 or 8 bits for many rows a key/value head: pieces of prompts and large trees (rows' sight: attention_kv_sight.hip).
//
// The other kernels multiply the codes themselves and apply a group's scale to every score and every weight, five vector instructions a score and group: with many rows that is what bounds
// them.  Here a workgroup turns 32 keys and values at a time into binary16 numbers in LDS, each in two, high and low (rounded to one, results were off by 1.7 times their own rounding), and
// its waves, 32 rows each, multiply those: the codes are taken apart once for all rows, and the rest is matrix products and the softmax.
//
//   S^T = K Q^T: rows of the product are keys, columns the wave's rows, so a lane ends with 16 of the 32 scores of one row, and the other half of the row is in the lane 32 away.
//   Z^T = V^T P^T: rows are channels, columns the same rows again: what a lane scored are the very keys that it weighs, and a row's factors are a number of its lane.
//
// v = high + low, high cut off to binary16, low, less than a step of it, rounded: off by 2^-21 of v at most.  S = high q + low q; Z = high w + low w + high rest, w a weight in binary16, rest what
// that leaves; low times rest, 2^-21, is left out.  With low, q, w and rest of the corrections in 8 bits, whose products take half the time, 4096 rows of 32 heads over 8 of 128, two sequences of 6000,
// took 327 us where this takes 369 (16 nodes of 32 heads over 8, 8 bits, 8 sequences that see 4112 tokens: 46.4 and 44.7), but a score's terms were off by up to 1.3e-4 of themselves, and a result
// by up to 3.3e-4 of the sum of its probabilities times |values|.
//
// One product a pair would be 104 us of those 369 at the 1352 TFLOP/s that a large binary16 product reaches; with the corrections, 2.5 of them, it is 260.  The rest is vector work (some 360
// instructions a wave and 32 keys, a third of them to take codes apart) that the products do not hide: registers allow two waves a SIMD, and while one multiplies the other issues an instruction every
// eight clocks, where two take one every four.  Eight waves share a stage, since with four each stage served half as many rows; with 16 rows a wave LDS was read twice as often.
//
// Up to 64 rows of heads of 128 two waves share a stage, and a workgroup is two such pairs, each with every other tile of its keys (16 nodes of 32 heads over 8, 8 bits, 8 sequences that see 4112
// tokens, with what the nodes see: 44.8 us; eight waves 65.5, blocks of 16 rows 60.4).  With corrections in 8 bits the same for heads of 64 took 272 us where blocks of 16 rows took 371, 64 sequences of
// 4096 and 16 heads, but 209 where those took 180 with sequences and trees of unequal size; four waves for up to 128 rows were within a tenth of eight, on either side.
#include "attention_kv.hip.h"
#include "attention_kv_tile.h"

namespace et {

namespace {

// LDS of a stage, in pieces of 16 bytes, for each 32 keys.  Keys: high parts [channel / 8, the even ones first][33 places of 32 keys], and low parts as well.  Values: high parts [keys / 8 of
// them][channel], and low parts as well.
constexpr int kWaves = 8;
template <int HD> struct TileShape {
    static constexpr int kSets = HD <= 64 ? 2 : 1;  // of 32 keys
    static constexpr int kTokens = 32 * kSets, kPieces = 2 * kSets;
    static constexpr int kRow = 33;                 // 32 keys, and one on to other banks
    static constexpr int kKeyLow = HD / 8 * kRow, kValue = 2 * kKeyLow, kValueLow = kValue + 4 * HD, kSet = kValueLow + 4 * HD;
    static constexpr int kStage = kSets * kSet;
    static constexpr int kShares = kTokens * HD / 16;  // of 16 numbers: of the keys, and as many of the values
};
// W waves share a stage, each with 32 rows; GROUPS of them are a workgroup, each with its own keys.  A group of eight has two stages, others one.  At the end half of the groups' sums, then a
// wave's rows, lie there.
template <int HD, int W, int GROUPS> constexpr int tile_lds() {
    constexpr int stages = (W == kWaves ? 2 : GROUPS) * TileShape<HD>::kStage, rows = (W * 32 * (HD + 2) * 2 + 15) / 16;
    constexpr int sums = GROUPS == 1 ? 0 : GROUPS / 2 * W * kTilePart<HD> / 4;
    return stages > rows ? (stages > sums ? stages : sums) : (rows > sums ? rows : sums);
}

// The channel that place p of the values' channels holds: so that lanes with neighbouring units of 16 bits store neighbouring pieces.
template <int BITS, int HD> __device__ __forceinline__ int place_channel(int p) {
    constexpr int C = 16 / BITS, N = HD / C;
    return p % N * C + p / N;
}

// Two codes, in the low bits of a word's halves: 1024 + code has the code in its lowest bits.  (mask, base: in registers, so that both are put to use in one instruction.)
__device__ __forceinline__ h2 codes_of(unsigned word, unsigned mask, unsigned base) { return __builtin_bit_cast(h2, (word & mask) | base) - h2{1024, 1024}; }
// code * scale + low as two binary16 numbers.  The first is cut off: rounding the scale up may carry a group's last steps beyond binary16's range, which then are its largest number and what is left.
// (minus: -1 that the compiler does not know, with which widening and subtracting are one instruction.)
__device__ __forceinline__ void parted(h2 &high, h2 &low, h2 code, h2 scale, h2 lowest, float minus) {
    float v[2], rest[2];
#pragma unroll
    for (int e = 0; e < 2; e++) v[e] = __builtin_fmaf((float)code[e], (float)scale[e], (float)lowest[e]);
    high = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(v[0], v[1]));
#pragma unroll
    for (int e = 0; e < 2; e++) rest[e] = __builtin_fmaf((float)high[e], minus, v[e]);
    low = h2{(_Float16)rest[0], (_Float16)rest[1]};
}
// Of two tokens' words of a scale and a lowest value: both scales, and both lowest values.
__device__ __forceinline__ h2 scales_of(unsigned a, unsigned b) { return __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x05040100u)); }
__device__ __forceinline__ h2 lows_of(unsigned a, unsigned b) { return __builtin_bit_cast(h2, __builtin_amdgcn_perm(b, a, 0x07060302u)); }

__device__ __forceinline__ unsigned word_of(h2 x) { return __builtin_bit_cast(unsigned, x); }

// Every wave's LDS accesses are done.  (__syncthreads would wait for loads from memory, too, which are on their way for the next turn.)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ float across_max(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float across_sum(float v) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}

// A wave's results [32 rows][HD], of lane l row l % 32, through LDS (rows of HD + 2 numbers) to Z.
template <int BITS, int HD, int BLOCKS>
__device__ __forceinline__ void rows_to_lds(_Float16 *lds, const f16v *acc, int first_block, float factor, bool none, int lane) {
    _Float16 *row = lds + (lane & 31) * (HD + 2);
#pragma unroll
    for (int k = 0; k < BLOCKS; k++)
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const float v = none ? 0.0f : acc[k][r] * factor;
            row[place_channel<BITS, HD>(32 * (first_block + k) + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3))] = (_Float16)(v > 65504.0f ? 65504.0f : v);  // (as result_value)
        }
}
template <int HD> __device__ __forceinline__ void rows_to_memory(const _Float16 *lds, const KvSightArgs &a, int b, int kv, int row0, int rows, int first, int step) {
    for (int e = first; e < rows * (HD / 2); e += step) {
        const int h = e / (HD / 2), w = e - h * (HD / 2), row = row0 + h, i = a.n == 1 ? 0 : row / a.per, r = row - i * a.per;
        *reinterpret_cast<unsigned *>(a.Z + ((size_t)b * a.n + i) * a.ldz + (size_t)(kv * a.per + r) * HD + 2 * w) = *reinterpret_cast<const unsigned *>(lds + h * (HD + 2) + 2 * w);
    }
}

// GROUPS times W waves of 32 rows each.
template <int BITS, int HD, int W, int GROUPS> __global__ __launch_bounds__(W * GROUPS * 64, 2) void mha_kv_tile_kernel(KV_LEADING, const KvSightArgs a) {
    using T = TileShape<HD>;
    constexpr int TB = HD * BITS / 8, G = HD / 32, CHUNKS = HD / 16, BLOCKS = HD / 32, SETS = T::kSets, PIECES = T::kPieces, SHARES = T::kShares;
    constexpr int SLOTS = W == kWaves ? 3 : 2;
    // What a thread takes apart of a stage.  Of eight waves some take a share of the keys, 16 channels of one, and as many a share of the values, two channels of eight tokens.  Of two each
    // takes two shares of the keys, and a wide one of the values, four channels.
    constexpr bool WIDE = W == 2;
    static_assert(W == kWaves || (WIDE && HD == 128), "two waves have 2 * 128 and 128 shares");
    constexpr int KEY_TURNS = WIDE ? 2 : 1, KEY_WORDS = BITS / 2 + 1, PAIRS = WIDE ? 2 : 1, VALUE_CODES = WIDE ? BITS : 4, UNITS = HD / 2 / PAIRS;
    constexpr int KEYS_AT = WIDE ? VALUE_CODES + 8 : 0, WORDS = WIDE ? KEYS_AT + KEY_TURNS * KEY_WORDS : VALUE_CODES + 8;
    constexpr int AHEAD = WIDE ? 4 : HD == 128 ? 6 : 8;  // pieces of a stage that are asked for ahead of the products that they are for, as far as there are registers
    constexpr bool ALIKE = HD == 64 || HD == 128, VALUES_ALIKE = WIDE || ALIKE;  // a wave's shares are of one piece of 16 keys
    __shared__ uint4 lds[tile_lds<HD, W, GROUPS>()];
    __shared__ unsigned all_marks[GROUPS == 1 ? 1 : W * GROUPS][64];
    __shared__ unsigned all_bad[GROUPS][SLOTS][SETS][G + 1];  // keys whose values are no numbers, of each group of channels and of any; of this tile, the next, and one to clear
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, half = lane >> 5, team = wave / W, member = wave % W;
    auto &bad = all_bad[team];
    const int kv = blockIdx.x, nkv = gridDim.x;
    int b = blockIdx.y;
    if (WIDE && starts_at && nkv * gridDim.y > 256 && gridDim.y <= 64) {
        // the longest sequences first: of 64 of 0 to 2000 tokens and 8 heads, 64 rows, 104 us rather than 117 (of 2000 each 137 either way)
        const int B = gridDim.y, key = lane < B ? (int)((unsigned)starts_at[lane] + (counts_at ? (unsigned)counts_at[lane] : 0u)) : 0;
        int rank = 0;
        for (int j = 0; j < B; j++) {
            const int other = __builtin_amdgcn_readlane(key, j);
            rank += other > key || (other == key && j < lane) ? 1 : 0;
        }
        b = __builtin_ctzll(__ballot(lane < B && rank == b));
    }
    const int block = splits == 1 ? blockIdx.z : blockIdx.z / splits, split = blockIdx.z - block * splits;

    const int32_t *table = table_at + (size_t)b * max_pages;
    // the rows of this block and of this wave, and what they see
    const int start = starts_at ? ET_KV_CONST(int32_t, starts_at)[b] : 0;
    const int count = counts_at ? min(max(ET_KV_CONST(int32_t, counts_at)[b], 0), n) : n;
    const int first_row = block * (32 * W), rows = min(32 * W, count * per - first_row);
    if (rows <= 0) return;
    const long long most = (long long)max_pages * a.page;
    const int end = (int)min(max((long long)start + count, 0LL), most);
    auto row_of = [&](int row) { return n == 1 ? 0 : row / per; };  // of the call's rows
    auto limit = [&](int i) { return a.causal ? (int)min((long long)end, max((long long)start + i + 1, 0LL)) : end; };
    KvTiles<true, T::kTokens> tiles;
    const int last_i = row_of(first_row + rows - 1);
    tiles.around(a, start, count, row_of(first_row), last_i, limit(last_i));
    const int v_end = tiles.end(limit(last_i));
    const int row0 = first_row + 32 * member, mine = min(32, rows - 32 * member);  // (of the last block's waves some may have none: they fill the stages only)
    const int wave_first = row_of(row0), wave_last = row_of(row0 + max(mine, 1) - 1);
    const int lim_least = limit(wave_first), lim_most = mine > 0 ? limit(wave_last) : 0;
    // positions of tiles that this wave's rows see some of, and all of
    KvTiles<true, T::kTokens> near;
    near.around(a, start, count, wave_first, wave_last, lim_most);
    const int sees_first = near.head * T::kTokens, sees_from = (near.head + near.gap) * T::kTokens, sees_to = lim_most, whole_from = near.whole_from, whole_to = min(lim_least, near.whole_to);

    // tiles of this group: from `own` on, `step` apart
    const int own = split * GROUPS + team, step = splits * GROUPS;

    // Pages of the pieces of the next tiles, a lane each, asked for 64 at a time: where they lie and which of them have one.  (Asked for tile by tile through the scalar cache, every wait for
    // LDS in between waited for them as well.)
    constexpr int TURNS_ASKED = 64 / PIECES;
    int pages, offs, next_pages, next_offs;
    auto ask = [&](int v) {
        const int piece = PIECES * tiles.tile(v + lane / PIECES * step) + lane % PIECES;
        const int pidx = (int)(((unsigned long long)(unsigned)piece * magic) >> shift);
        next_offs = (piece - pidx * page_pieces) << 4;
        next_pages = pidx < max_pages ? table[pidx] : -1;
    };
    ask(own);

    h8 q[CHUNKS];
    const int row = min(row0 + min(c, max(mine, 1) - 1), first_row + rows - 1), i_row = row_of(row), r_row = row - i_row * per;
    const int lim = limit(i_row);
    KvSight<true> sight;
    sight.of(a, b, n, i_row, start, count);
    const _Float16 *qrow = a.Q + ((size_t)b * n + i_row) * a.ldq + (size_t)(kv * per + r_row) * HD + half * 8;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
        q[i] = *reinterpret_cast<const h8 *>(qrow + 16 * i);
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf((float)q[i][e]));
    }
    top = across_max(top);
    const int up = top > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
    const float grow = query_growth(top, up, a.scale_log2e);
    const float key_scale = __builtin_ldexpf(fabsf(a.scale_log2e), -up);
#pragma unroll
    for (int i = 0; i < CHUNKS; i++) {
        // in the order that the keys' codes come out of their words
        constexpr int order[2][8] = {{0, 4, 1, 5, 2, 6, 3, 7}, {0, 2, 1, 3, 4, 6, 5, 7}};
        const h8 x = q[i];
#pragma unroll
        for (int e = 0; e < 8; e++) q[i][e] = (_Float16)((float)x[order[BITS == 8][e]] * grow);
    }

    const char *k_codes = a.k_codes + (size_t)kv * a.page * TB, *v_codes = a.v_codes + (size_t)kv * a.page * TB;
    const unsigned *k_scales = a.k_scales + (size_t)kv * (G * a.page), *v_scales = a.v_scales + (size_t)kv * (G * a.page);
    const unsigned page_bytes = (unsigned)nkv * a.page * TB, page_scales = (unsigned)nkv * G * a.page;

    float minus = -1.0f;
    unsigned mask = BITS == 4 ? 0x000f000fu : 0x00ff00ffu, base = 0x64006400u;
    asm("" : "+s"(minus));
    asm("" : "+v"(mask));
    asm("" : "+v"(base));
    // a tile's codes and scales, on their way: of values, then of keys
    const bool takes_keys = WIDE || 64 * member < SHARES, takes_values = WIDE || (!takes_keys && 64 * member < 2 * SHARES);
    const int key_share0 = 64 * member, value_share0 = WIDE ? key_share0 : 64 * member - SHARES;
    unsigned words[WORDS];
    // (a wide share of 8-bit values is two units of 16 bits a token side by side; of 4-bit values one, whose upper half narrow shares leave to another thread)
    struct ValueShare {
        int of, unit, pair, group;
    };
    auto value_share = [&](int lane) {
        const int of = (value_share0 + lane) / UNITS, rest = value_share0 + lane - of * UNITS;
        const int unit = WIDE ? BITS / 4 * rest : BITS == 4 ? rest % (HD / 4) : rest;
        return ValueShare{of, unit, WIDE || BITS == 8 ? 0 : rest / (HD / 4), BITS == 4 ? unit >> 3 : unit >> 4};
    };
    unsigned long long have = 0;  // pieces asked for that have pages
    int turn = TURNS_ASKED;       // of those asked for, the next to fetch
    unsigned ok = 0;              // of the tile that was fetched last: its pieces that have pages
    auto fetch = [&](int v) {     // tile v of those counted without the gap
        if (turn == TURNS_ASKED) {
            const bool is = next_pages >= 0 && next_pages < a.npages;
            have = __ballot(is);
            pages = is ? next_pages : 0, offs = is ? next_offs : 0;
            turn = 0;
            ask(v + TURNS_ASKED * step);
        }
        int lane_now = lane;
        if (WIDE) asm("" : "+v"(lane_now));  // (what follows from it is worked out anew each time: kept, it takes registers that there are not)
        const int first = PIECES * turn++;
        ok = (unsigned)(have >> first) & ((1u << PIECES) - 1);
        auto pick = [&](int of, int piece, bool alike) { return (unsigned)(alike ? __builtin_amdgcn_readlane(of, first + piece) : __shfl(of, first + piece)); };
        if (takes_keys) {
#pragma unroll
            for (int k = 0; k < KEY_TURNS; k++) {
                const int s0 = key_share0 + 128 * k;
                const int s = s0 + lane_now, key = s / (HD / 16), u = s - key * (HD / 16), piece = (ALIKE ? s0 : s) / (HD / 16) >> 4;
                const unsigned of_page = pick(pages, piece, ALIKE), at = pick(offs, piece, ALIKE);
                unsigned w[BITS / 2];
                load_words<BITS / 2>(w, k_codes + ((size_t)of_page * page_bytes + at * TB) + (unsigned)((key & 15) * TB + u * (2 * BITS)));
#pragma unroll
                for (int i = 0; i < BITS / 2; i++) words[KEYS_AT + KEY_WORDS * k + i] = w[i];
                words[KEYS_AT + KEY_WORDS * k + BITS / 2] = (k_scales + ((size_t)of_page * page_scales + at))[(unsigned)((u >> 1) * a.page + (key & 15))];
            }
        }
        if (takes_values) {  // of the values of eight keys: 4 half .. and 8 + 4 half .. of a piece
            const ValueShare from = value_share(lane_now);
            const int piece = (VALUES_ALIKE ? value_share0 / UNITS : from.of) >> 1;
            const unsigned of_page = pick(pages, piece, VALUES_ALIKE), at = pick(offs, piece, VALUES_ALIKE);
            const char *p = v_codes + ((size_t)of_page * page_bytes + at * TB) + (unsigned)((from.of & 1) * 4 * TB + from.unit * 8);
#pragma unroll
            for (int i = 0; i < VALUE_CODES / 4; i++) {
                const u2 x = *reinterpret_cast<const u2 *>(p + 8 * i), y = *reinterpret_cast<const u2 *>(p + 8 * TB + 8 * i);
                words[4 * i] = x[0], words[4 * i + 1] = x[1], words[4 * i + 2] = y[0], words[4 * i + 3] = y[1];
            }
            const unsigned *sc = v_scales + ((size_t)of_page * page_scales + at) + (unsigned)(from.group * a.page + (from.of & 1) * 4);
            const u4 m = *reinterpret_cast<const u4 *>(sc), o = *reinterpret_cast<const u4 *>(sc + 8);
#pragma unroll
            for (int i = 0; i < 4; i++) words[VALUE_CODES + i] = m[i], words[VALUE_CODES + 4 + i] = o[i];
        }
    };
    // .. as numbers, in a stage
    auto fill = [&](uint4 *stage, unsigned (*flags)[G + 1]) {
        int lane_now = lane;
        if (WIDE) asm("" : "+v"(lane_now));  // (as above)
        if (takes_keys) {
#pragma unroll
            for (int k = 0; k < KEY_TURNS; k++) {
                __builtin_amdgcn_sched_barrier(0);  // (one after the other: two at once take more registers than there are)
                const int s0 = key_share0 + 128 * k, s = s0 + lane_now;
                const int key = s / (HD / 16), u = s - key * (HD / 16);
                const unsigned *codes = words + KEYS_AT + KEY_WORDS * k, scale = codes[BITS / 2];
                const h2 sc = scales_of(scale, scale), lo = lows_of(scale, scale);
                uint4 *set = stage + (key >> 5) * T::kSet + (key & 31);
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    h2 high[4], low[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const unsigned word = BITS == 4 ? codes[p] >> (4 * e) : codes[2 * p + (e >> 1)] >> (8 * (e & 1));
                        parted(high[e], low[e], codes_of(word, mask, base), sc, lo, minus);
                    }
                    uint4 *to = set + (p * (HD / 16) + u) * T::kRow;
                    to[0] = uint4{word_of(high[0]), word_of(high[1]), word_of(high[2]), word_of(high[3])};
                    to[T::kKeyLow] = uint4{word_of(low[0]), word_of(low[1]), word_of(low[2]), word_of(low[3])};
                }
            }
        }
        if (takes_values) {
            const unsigned *scales = words + VALUE_CODES;
            const ValueShare to = value_share(lane_now);
#pragma unroll
            for (int p = 0; p < PAIRS; p++) {
                __builtin_amdgcn_sched_barrier(0);
                const int of = to.of, unit = to.unit + (BITS == 8 ? p : 0), pair = BITS == 4 ? to.pair + p : 0;
                h2 high[2][4], low[2][4], sum = {0, 0};
#pragma unroll
                for (int x = 0; x < 4; x++) {  // tokens 2 x and the next
                    const h2 sc = scales_of(scales[2 * x], scales[2 * x + 1]), lo = lows_of(scales[2 * x], scales[2 * x + 1]);
                    const unsigned w = BITS == 4 ? words[x] >> (8 * pair) : words[4 * p + x];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        parted(high[i][x], low[i][x], codes_of(w >> (BITS * i), mask, base), sc, lo, minus);
                        sum = __builtin_elementwise_fma(low[i][x], h2{0, 0}, sum);
                    }
                }
                // What is not a number, or infinite, must not meet the zero weight of a row that does not see it: it leaves the stage, and the rows that do see it are marked.  (The low part of such a value is no number either.)
                if (word_of(sum) != 0) {
                    unsigned keys = 0;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const bool is = (word_of(low[0][e >> 1]) >> (16 * (e & 1)) & 0x7c00u) == 0x7c00u || (word_of(low[1][e >> 1]) >> (16 * (e & 1)) & 0x7c00u) == 0x7c00u;
                        if (is) {
                            keys |= 1u << (16 * (of >> 1 & 1) + 4 * (of & 1) + (e & 3) + (e >> 2) * 8);
#pragma unroll
                            for (int i = 0; i < 2; i++) high[i][e >> 1][e & 1] = low[i][e >> 1][e & 1] = (_Float16)0.0f;
                        }
                    }
                    atomicOr(&flags[of >> 2][to.group], keys);
                    atomicOr(&flags[of >> 2][G], keys);
                }
                uint4 *set = stage + (of >> 2) * T::kSet;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int place = (BITS == 4 ? 2 * pair + i : i) * (HD / (16 / BITS)) + unit;
                    uint4 *at = set + T::kValue + (of & 3) * HD + place;
                    at[0] = uint4{word_of(high[i][0]), word_of(high[i][1]), word_of(high[i][2]), word_of(high[i][3])};
                    at[T::kValueLow - T::kValue] = uint4{word_of(low[i][0]), word_of(low[i][1]), word_of(low[i][2]), word_of(low[i][3])};
                }
            }
        }
    };

    float ref = kNothing, l = 0.0f;
    unsigned not_numbers = 0;  // groups of whose values this row sees some
    f16v acc[BLOCKS];
#pragma unroll
    for (int k = 0; k < BLOCKS; k++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[k][r] = 0.0f;

    if (threadIdx.x < GROUPS * SLOTS * SETS * (G + 1)) (&all_bad[0][0][0][0])[threadIdx.x] = 0;
    // a tile in a stage, with its marks and its pieces that have pages
    auto compute = [&](const int tile, const uint4 *stage, const unsigned (*marks)[G + 1], const unsigned now) {
        if (tile < sees_to && (tile < sees_first || tile >= sees_from)) {
            // (products go first: one takes one of eight turns to issue, and leaves the others to vector work of the SIMD's other wave, which would leave it none)
            __builtin_amdgcn_s_setprio(1);
            unsigned marked[SETS];
            f16v s[SETS];
#pragma unroll
            for (int x = 0; x < SETS; x++) {
                marked[x] = marks[x][G];
                s[x] = f16v{};
                const uint4 *keys = stage + x * T::kSet + c;
#pragma unroll
                for (int part = 0; part < 2; part++)
#pragma unroll
                    for (int i = 0; i < CHUNKS; i++)
                        s[x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, keys[part * T::kKeyLow + (half * CHUNKS + i) * T::kRow]), q[i], s[x], 0, 0, 0);
            }
            constexpr int READS = 2 * CHUNKS * SETS, EARLY = READS < AHEAD ? READS : AHEAD;
            __builtin_amdgcn_sched_group_barrier(0x100, EARLY, 0);
#pragma unroll
            for (int i = 0; i < READS - EARLY; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, EARLY, 0);
            __builtin_amdgcn_s_setprio(0);
            const bool whole = tile + T::kTokens <= whole_to && (tile >= whole_from || tile + T::kTokens <= a.sinks) && now == (1u << PIECES) - 1;
            unsigned seen[SETS];
#pragma unroll
            for (int x = 0; x < SETS; x++) seen[x] = ~0u;
            if (!whole) {
#pragma unroll
                for (int x = 0; x < SETS; x++) {
                    // (from the lane's first key on: what a register is compared with or shifted by is a constant then, and needs none itself)
                    const int at = tile + 32 * x, first = at + 4 * half, to = lim - first, low = sight.low - first, sinks = a.sinks - first;
                    const unsigned tree = sight.tree(a, at) >> (4 * half);
                    unsigned keep = 0;
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const int key = 8 * (r >> 2) + (r & 3);
                        const bool is = (now >> (2 * x + (r >> 3)) & 1u) && key < to && (key >= low || key < sinks) && (tree & 1u << key);
                        keep |= is ? 1u << key : 0u;
                        s[x][r] = is ? s[x][r] : kNothing;
                    }
                    seen[x] = keep;
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int e = 1; e < 16 * SETS; e++) top = fmaxf(top, s[e >> 4][e & 15]);
            const float reach = across_max(top) * key_scale;
            // a weight is at most 2^15; a row's reference moves by its own scores alone, so that its bits do not depend on the rows beside it
            const bool moves = reach > ref + 15.0f;
            if (__any(moves)) {
                const float next = moves ? reach - 11.0f : ref, f = __builtin_amdgcn_exp2f(ref - next);
                ref = next;
                l *= f;
#pragma unroll
                for (int k = 0; k < BLOCKS; k++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[k][r] *= f;
            }
#pragma unroll
            for (int x = 0; x < SETS; x++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[x][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r], key_scale, -ref));
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16 * SETS; e++) s[e >> 4][e & 15] = seen[e >> 4] & 1u << (8 * (e >> 2 & 3) + (e & 3)) ? s[e >> 4][e & 15] : 0.0f;
            }
#pragma unroll
            for (int x = 0; x < SETS; x++)
                if (__builtin_amdgcn_readfirstlane(marked[x]) != 0) {
#pragma unroll
                    for (int g = 0; g < G; g++) not_numbers |= (marks[x][g] >> (4 * half) & seen[x] & 0x0f0f0f0fu) != 0 ? 1u << g : 0u;
                }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int x = 0; x < SETS; x++) {
                h8 weights[2], rests[2];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float p0 = s[x][2 * e], p1 = s[x][2 * e + 1];
                    unsigned w = word_of(h2{(_Float16)p0, (_Float16)p1});
                    asm("" : "+v"(w));  // (or each half is rounded once more, on its own)
                    const h2 wide = __builtin_bit_cast(h2, w);
                    weights[e >> 2][2 * (e & 3)] = wide[0], weights[e >> 2][2 * (e & 3) + 1] = wide[1];
                    rests[e >> 2][2 * (e & 3)] = (_Float16)__builtin_fmaf((float)wide[0], minus, p0), rests[e >> 2][2 * (e & 3) + 1] = (_Float16)__builtin_fmaf((float)wide[1], minus, p1);
                    l += p0;
                    l += p1;
                }
                const uint4 *values = stage + x * T::kSet + T::kValue + half * HD + c;
#pragma unroll
                for (int m = 0; m < BLOCKS; m++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const h8 high = __builtin_bit_cast(h8, values[2 * k * HD + 32 * m]), low = __builtin_bit_cast(h8, values[T::kValueLow - T::kValue + 2 * k * HD + 32 * m]);
                        acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(high, weights[k], acc[m], 0, 0, 0);
                        acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(high, rests[k], acc[m], 0, 0, 0);
                        acc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(low, weights[k], acc[m], 0, 0, 0);
                    }
            }
            constexpr int VALUES = 4 * BLOCKS * SETS;
            __builtin_amdgcn_sched_group_barrier(0x100, AHEAD < VALUES ? AHEAD : VALUES, 0);
#pragma unroll
            for (int i = 0; i < (VALUES - AHEAD) / 4; i++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };

    if (own < v_end) fetch(own);
    if (W == kWaves) {
        // Each turn computes a tile and fills in the next one, into the other stage; the first only fills in.  Half of the waves, one of every SIMD, fill in before they compute, the others behind,
        // so that a SIMD has vector work beside matrix products.
        const bool early = wave < kWaves / 2;
        int slot = 2, buffer = 1;
        unsigned now = 0;
        for (int v = own - step; v < v_end; v += step) {
            lds_barrier();
            const int next_slot = slot == 2 ? 0 : slot + 1, clear_slot = next_slot == 2 ? 0 : next_slot + 1;
            const bool more = v + step < v_end;
            const unsigned then = ok;
            if (threadIdx.x < SETS * (G + 1)) (&bad[clear_slot][0][0])[threadIdx.x] = 0;
            auto go_on = [&]() {
                fill(lds + (buffer ^ 1) * T::kStage, bad[next_slot]);
                if (v + 2 * step < v_end) fetch(v + 2 * step);
            };
            if (early && more) go_on();
            if (v >= own) compute(tiles.tile(v) * T::kTokens, lds + buffer * T::kStage, bad[slot], now);
            if (!early && more) go_on();
            now = then;
            slot = next_slot;
            buffer ^= 1;
        }
    } else {
        // Each turn fills in a tile and computes it: a second workgroup of the compute unit has vector work beside the products.
        const int first = split * GROUPS;
        uint4 *stage = lds + team * T::kStage;
        int slot = 0, v = own;
        for (int u = first; u < v_end; u += step) {
            lds_barrier();
            const unsigned now = ok;
            if (v < v_end) {
                fill(stage, bad[slot]);
                if (v + step < v_end) fetch(v + step);
            }
            lds_barrier();
            if (v < v_end) {
                const int by = threadIdx.x - team * (W * 64);
                if (by < SETS * (G + 1)) (&bad[slot ^ 1][0][0])[by] = 0;
                compute(tiles.tile(v) * T::kTokens, stage, bad[slot], now);
            }
            slot ^= 1;
            v += step;
        }
        // the groups' sums to the first
        float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
        for (int some = GROUPS / 2; some > 0; some /= 2) {
            __syncthreads();
            if (team >= some && team < 2 * some) {
                float *to = sums + (wave - some * W) * kTilePart<HD> + lane;
                to[0] = ref, to[64] = l;
#pragma unroll
                for (int k = 0; k < BLOCKS; k++)
#pragma unroll
                    for (int r = 0; r < 16; r++) to[(2 + 16 * k + r) * 64] = acc[k][r];
                all_marks[wave][lane] = not_numbers;
            }
            __syncthreads();
            if (team < some) {
                const float *from = sums + wave * kTilePart<HD> + lane;
                const float other = from[0], most = fmaxf(ref, other), f = __builtin_amdgcn_exp2f(ref - most), fo = __builtin_amdgcn_exp2f(other - most);
                ref = most;
                l = l * f + from[64] * fo;
#pragma unroll
                for (int k = 0; k < BLOCKS; k++)
#pragma unroll
                    for (int r = 0; r < 16; r++) acc[k][r] = acc[k][r] * f + from[(2 + 16 * k + r) * 64] * fo;
                not_numbers |= all_marks[wave + some * W][lane];
            }
        }
        if (team > 0) return;
    }

    const float sum = across_sum(l);
    not_numbers |= (unsigned)__shfl_xor((int)not_numbers, 32);
    if (__any(not_numbers != 0)) {
#pragma unroll
        for (int m = 0; m < BLOCKS; m++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (not_numbers >> (place_channel<BITS, HD>(32 * m + 8 * (r >> 2) + 4 * half + (r & 3)) >> 5) & 1u) acc[m][r] = __builtin_nanf("");
    }
    if (splits > 1) {
        if (mine <= 0) return;
        float *part = a.parts + (((size_t)blockIdx.z * units + (unsigned)(b * nkv + kv)) * W + member) * kTilePart<HD> + lane;
        part[0] = ref;
        part[64] = sum;
#pragma unroll
        for (int m = 0; m < BLOCKS; m++)
#pragma unroll
            for (int r = 0; r < 16; r++) part[(2 + 16 * m + r) * 64] = acc[m][r];
        return;
    }
    if (GROUPS == 1) __syncthreads();  // the stages are read
    if (mine <= 0) return;
    // (where groups' sums were, a wave has read its own alone)
    constexpr int APART = GROUPS == 1 ? 32 * (HD + 2) : 2 * kTilePart<HD>;
    static_assert(W * APART * 2 <= sizeof(lds), "a wave's rows");
    _Float16 *mem = reinterpret_cast<_Float16 *>(lds) + member * APART;
    rows_to_lds<BITS, HD, BLOCKS>(mem, acc, 0, 1.0f / sum, sum == 0.0f, lane);
    wave_lds_order();
    rows_to_memory<HD>(mem, a, b, kv, row0, mine, lane, 64);
}

// The parts of 32 rows: a wave for each 32 channels.
template <int BITS, int HD> __global__ __launch_bounds__(HD * 2) void mha_kv_tile_join_kernel(const KvSightArgs a) {
    __shared__ _Float16 lds[32 * (HD + 2)];
    const int lane = threadIdx.x & 63, m = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x, block = blockIdx.y, wave = blockIdx.z, waves = gridDim.z;
    const int b = unit / a.nkv, kv = unit - b * a.nkv;
    const int row0 = (block * waves + wave) * 32, rows = min(32, (a.counts ? min(max(a.counts[b], 0), a.n) : a.n) * a.per - row0);
    if (rows <= 0) return;
    const float *part = a.parts + (((size_t)block * a.splits * a.units + unit) * waves + wave) * kTilePart<HD> + lane;
    const size_t next = (size_t)a.units * waves * kTilePart<HD>;
    float ref = kNothing, l = 0.0f;
    f16v acc = {};
    for (int s0 = 0; s0 < a.splits; s0 += 4) {  // four parts asked for at once
        float r[4], ls[4];
        f16v vs[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float *p = part + (s0 + k < a.splits ? s0 + k : s0) * next;
            r[k] = s0 + k < a.splits ? p[0] : kNothing;
            ls[k] = p[64];
#pragma unroll
            for (int e = 0; e < 16; e++) vs[k][e] = p[(2 + 16 * m + e) * 64];
        }
        const float most = fmaxf(fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3])), ref), was = __builtin_amdgcn_exp2f(ref - most);
        ref = most;
        l *= was;
        acc *= was;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = s0 + k < a.splits ? __builtin_amdgcn_exp2f(r[k] - most) : 0.0f;
            l = __builtin_fmaf(ls[k], f, l);
#pragma unroll
            for (int e = 0; e < 16; e++) acc[e] = __builtin_fmaf(f, vs[k][e], acc[e]);
        }
    }
    rows_to_lds<BITS, HD, 1>(lds, &acc, m, 1.0f / l, l == 0.0f, lane);
    __syncthreads();
    rows_to_memory<HD>(lds, a, b, kv, row0, rows, threadIdx.x, HD * 2);
}

struct TileForm {
    void (*kernel)(KV_LEADING, const KvSightArgs);
    void (*join)(const KvSightArgs);
};
template <int BITS, int HD> TileForm tile_form(int waves) {
    if constexpr (HD == 128) {
        if (waves == 2) return {mha_kv_tile_kernel<BITS, HD, 2, 2>, mha_kv_tile_join_kernel<BITS, HD>};
    }
    return {mha_kv_tile_kernel<BITS, HD, kWaves, 1>, mha_kv_tile_join_kernel<BITS, HD>};
}
template <int BITS> TileForm tile_form(int hd, int waves) {
    switch (hd) {
        case 32: return tile_form<BITS, 32>(waves);
        case 64: return tile_form<BITS, 64>(waves);
        case 96: return tile_form<BITS, 96>(waves);
        default: return tile_form<BITS, 128>(waves);
    }
}

}  // namespace

int kv_tile_most_waves(int hd, long long rows) { return hd > 128 ? 0 : rows > (hd == 128 ? 64 : hd == 32 ? 128 : 96) ? kWaves : hd == 128 && rows > 32 ? 2 : 0; }
int kv_tile_waves(const et_kv_cache *c, long long positions, int B, long long rows) {
    const int waves = kv_tile_most_waves(c->hd, rows);
    const long long work = (long long)B * c->nkv * ((rows + 32 * kWaves - 1) / (32 * kWaves)) * ((positions + 31) / 32);
    return work >= (waves == 2 ? 4000 : c->hd == 128 ? 1024 : 3000) ? waves : 0;
}

int kv_tile_plan(const char *fn, KvTilePlan &p, const et_kv_cache *c, long long positions, int B, int n, int nh, int waves) {
    ET_REQUIRE(nh > 0 && nh % c->nkv == 0, ET_ERR_INVALID_ARG, "%s: nh=%d must be a multiple of nkv=%d", fn, nh, c->nkv);
    const long long rows = (long long)n * (nh / c->nkv), units = (long long)B * c->nkv;
    const long long blocks = (rows + 32 * waves - 1) / (32 * waves), groups = units * blocks;
    ET_REQUIRE(rows <= 0x7fffffffLL && B <= 65535 && blocks <= 65535 && groups <= (1LL << 24), ET_ERR_UNSUPPORTED, "%s: B=%d n=%d nh=%d", fn, B, n, nh);
    p.blocks = (int)blocks;
    p.waves = waves;
    const int tokens = c->hd <= 64 ? 64 : 32;
    const long long tiles = (positions + tokens - 1) / tokens, at_once = waves == 2 ? 512 : 256;
    p.splits = groups == 0 ? 1 : (int)std::max(1LL, std::min({at_once / groups, tiles / (waves == 2 ? 8 : 4), waves == 2 ? 64LL : 256LL}));
    p.splits = std::min(p.splits, (int)(65535 / std::max(1LL, blocks)));
    p.bytes = p.splits > 1 ? (size_t)(groups * p.splits * waves) * (2 + c->hd / 2) * 64 * sizeof(float) : 0;
    return ET_OK;
}

int kv_tile_run(const char *fn, const KvMhaCall &call, long long positions, int waves, size_t need, KvSightArgs &a, et_stream stream) {
    KvTilePlan p;
    int st = kv_tile_plan(fn, p, call.cache, positions, call.B, call.n, call.nh, waves);
    if (st == ET_OK) st = kv_check_call(fn, call, need);
    if (st != ET_OK || call.B == 0 || call.n == 0) return st;
    const KvPieces pieces = kv_fill(call, a);
    a.cols = 1;
    a.block_rows = 32 * p.waves;
    a.splits = p.splits;
    const TileForm f = call.cache->bits == 4 ? tile_form<4>(a.hd, p.waves) : tile_form<8>(a.hd, p.waves);
    st = launch_kernel("mha_kv_tile_kernel", f.kernel, dim3((unsigned)a.nkv, (unsigned)call.B, (unsigned)(p.blocks * p.splits)), (unsigned)(p.waves == 2 ? 4 : p.waves) * 64, 0, as_stream(stream), call.table,
                       call.starts, call.counts, call.max_pages, a.units, a.splits, a.per, pieces.magic, pieces.shift, pieces.of_page, call.n, a);
    if (st != ET_OK || p.splits == 1) return st;
    return launch_kernel("mha_kv_tile_join_kernel", f.join, dim3((unsigned)a.units, (unsigned)p.blocks, (unsigned)p.waves), (unsigned)a.hd * 2, 0, as_stream(stream), a);
}

}  // namespace et

// Block tables and slot maps of a paged cache, built from what each sequence holds (et_abi.h): pages that a sequence's tokens no longer need go to the end of a ring of free pages, those that
// they need and do not have come from its front, both in the order of (sequence, page), so that the result depends on nothing but the arguments.
//
// A wave takes a stretch of entries; what it gives and takes is placed by counting those of the waves before it.  Small tables are one workgroup's, in one launch; larger ones take two, since
// no workgroup waits for another: the first counts, the second places.  Slots of many rows are written by a launch of their own (kv_tables_forms.h).  Bound by a launch and dependent accesses (8 sequences of 64 pages: 4.4 us), and by the table's bytes where it is large:
// 512 sequences of 8192 pages are read in 6.0 us (2.8 TB/s) and read and written in 12.5 (2.7 TB/s).  Sixteen entries at once for a lane rather than four changed neither.  With thousands of
// sequences bound by adding up the counts of all workgroups before one's own, which grows with the square: 4096 sequences of 8 pages 59 us, 65535 7400.
#include "common.hip.h"
#include "kv_tables_forms.h"

namespace et {
namespace {

struct TablesArgs {
    const int32_t *before;
    int32_t *table;
    const int32_t *starts, *counts, *shared;
    int32_t *ring;
    const int32_t *state;
    int32_t *next_state;
    long long *slots;
    int2 *sums;       // of every wave of the first launch: pages needed and given; behind them the ring's head and count
    int max_pages, page, npages, B, n, window, sinks;
};

constexpr int kOneWaves = 16, kManyWaves = 8;

// The pages that a sequence needs: i < end, and i < first or i >= near.  Those before `own` are not its own to give or take.
struct Needs {
    int end, near, own;
};
__device__ __forceinline__ Needs needs_of(const TablesArgs &a, int b) {
    const long long start = a.starts ? a.starts[b] : 0, count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
    const long long tokens = max(start + count, 0LL), low = a.window ? start - a.window + 1 : 0;
    Needs s;
    s.end = (int)min((tokens + a.page - 1) / a.page, (long long)a.max_pages);
    s.near = low > 0 ? (int)min(low / a.page, (long long)a.max_pages) : 0;
    s.own = a.shared ? min(max(a.shared[b], 0), a.max_pages) : 0;
    return s;
}

// Head and count of the ring, brought into its bounds.
__device__ __forceinline__ int2 ring_state(const TablesArgs &a) {
    const int head = a.state[0] % a.npages;
    return int2{head < 0 ? head + a.npages : head, min(max(a.state[1], 0), a.npages)};
}

// What entry i of a sequence is to become.
enum Fate { kStays, kNone, kTaken, kGiven };
__device__ __forceinline__ Fate fate_of(const TablesArgs &a, const Needs &s, int i, int page, int first_pages) {
    if (i < s.own) return kStays;
    const bool held = page >= 0 && page < a.npages, wanted = i < s.end && (i < first_pages || i >= s.near);
    return held ? (wanted ? kStays : kGiven) : (wanted ? kTaken : kNone);
}

// Pages.
struct Counted {
    int needed, given;
};

// A wave's entries [from, to): of all tables, counted through (ONE), or of the workgroup's sequence.
template <bool ONE> __device__ __forceinline__ void stretch(const TablesArgs &a, int wave, int &from, int &to) {
    constexpr int W = ONE ? kOneWaves : kManyWaves;
    const int entries = ONE ? a.B * a.max_pages : a.max_pages;
    const int some = (entries + W * 64 - 1) / (W * 64) * 64;
    from = (int)min((long long)wave * some, (long long)entries);
    to = (int)min((long long)from + some, (long long)entries);
}

template <bool ONE> __device__ __forceinline__ Counted count_stretch(const TablesArgs &a, const Needs *needs, int from, int to, int first_pages) {
    const int lane = threadIdx.x & 63;
    Counted c = {0, 0};
    const int32_t *before = a.before + (ONE ? 0 : (size_t)blockIdx.x * a.max_pages);
    for (int e0 = from; e0 < to; e0 += 4 * 64) {
        int page[4];
#pragma unroll
        for (int k = 0; k < 4; k++) page[k] = before[min(e0 + 64 * k + lane, to - 1)];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = e0 + 64 * k + lane, b = ONE ? min(e, to - 1) / a.max_pages : 0;
            const Fate f = e < to ? fate_of(a, needs[b], e - b * a.max_pages, page[k], first_pages) : kStays;
            c.needed += __builtin_popcountll(__ballot(f == kTaken));
            c.given += __builtin_popcountll(__ballot(f == kGiven));
        }
    }
    return c;
}

// base: what the waves before this one need and give.
template <bool ONE> __device__ __forceinline__ void place_stretch(const TablesArgs &a, const Needs *needs, int from, int to, int first_pages, Counted base, int2 ring) {
    const int lane = threadIdx.x & 63;
    const unsigned long long below = (1ull << lane) - 1;
    const size_t at = ONE ? 0 : (size_t)blockIdx.x * a.max_pages;
    for (int e0 = from; e0 < to; e0 += 4 * 64) {
        int page[4];
#pragma unroll
        for (int k = 0; k < 4; k++) page[k] = a.before[at + min(e0 + 64 * k + lane, to - 1)];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = e0 + 64 * k + lane, b = ONE ? min(e, to - 1) / a.max_pages : 0;
            const Fate f = e < to ? fate_of(a, needs[b], e - b * a.max_pages, page[k], first_pages) : kStays;
            const unsigned long long takes = __ballot(f == kTaken), gives = __ballot(f == kGiven);
            int now = f == kStays ? page[k] : -1;
            if (f == kTaken) {
                const int rank = base.needed + __builtin_popcountll(takes & below);
                if (rank < ring.y) now = a.ring[(int)(((long long)ring.x + rank) % a.npages)];
            }
            if (f == kGiven) {
                const long long rank = (long long)ring.y + base.given + __builtin_popcountll(gives & below);
                if (rank < a.npages) a.ring[(int)((ring.x + rank) % a.npages)] = page[k];
            }
            base.needed += __builtin_popcountll(takes);
            base.given += __builtin_popcountll(gives);
            if (e < to) a.table[at + e] = now;
        }
    }
}

__device__ __forceinline__ void store_state(const TablesArgs &a, Counted total, int2 ring) {
    const int taken = min(total.needed, ring.y);
    a.next_state[0] = (int)(((long long)ring.x + taken) % a.npages);
    a.next_state[1] = (int)min((long long)ring.y + total.given, (long long)a.npages) - taken;  // (what was dropped has no place: places of pages that were taken are not free ones)
    a.next_state[2] = total.needed - taken;
}

// Where row i of sequence b lies in a table that is written: page number * page + place, or -1.
__device__ __forceinline__ long long slot_of(const TablesArgs &a, int b, int i) {
    const int count = a.counts ? min(max(a.counts[b], 0), a.n) : a.n;
    const long long pos = (long long)(a.starts ? a.starts[b] : 0) + i;
    if (i >= count || pos < 0 || pos >= (long long)a.max_pages * a.page) return -1;
    const int at = (int)pos / a.page, page = a.table[(size_t)b * a.max_pages + at];
    return page >= 0 && page < a.npages ? (long long)page * a.page + ((int)pos - at * a.page) : -1;
}

// Slots of the rows of sequences from b0 on, whose tables the workgroup has written.
__device__ __forceinline__ void store_slots(const TablesArgs &a, int b0, int sequences, int threads) {
    if (!a.slots) return;
    const unsigned rows = (unsigned)sequences * (unsigned)a.n;
    for (unsigned r = threadIdx.x; r < rows; r += threads) {
        const unsigned of = r / (unsigned)a.n;
        a.slots[(size_t)b0 * a.n + r] = slot_of(a, b0 + (int)of, (int)(r - of * (unsigned)a.n));
    }
}

__global__ __launch_bounds__(kOneWaves * 64) void kv_tables_one_kernel(const TablesArgs a) {
    __shared__ Needs needs[kOneSequences];
    __shared__ Counted counted[kOneWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first_pages = (int)(((long long)a.sinks + a.page - 1) / a.page);
    for (int b = threadIdx.x; b < a.B; b += kOneWaves * 64) needs[b] = needs_of(a, b);
    const int2 ring = ring_state(a);
    __syncthreads();
    int from, to;
    stretch<true>(a, wave, from, to);
    const Counted c = count_stretch<true>(a, needs, from, to, first_pages);
    if ((threadIdx.x & 63) == 0) counted[wave] = c;
    __syncthreads();  // (and every thread has the ring's state)
    Counted base = {0, 0}, total = {0, 0};
#pragma unroll
    for (int w = 0; w < kOneWaves; w++) {
        if (w < wave) base.needed += counted[w].needed, base.given += counted[w].given;
        total.needed += counted[w].needed, total.given += counted[w].given;
    }
    place_stretch<true>(a, needs, from, to, first_pages, base, ring);
    if (threadIdx.x == 0) store_state(a, total, ring);
    __syncthreads();
    store_slots(a, 0, a.B, kOneWaves * 64);
}

__global__ __launch_bounds__(kManyWaves * 64) void kv_tables_count_kernel(const TablesArgs a) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first_pages = (int)(((long long)a.sinks + a.page - 1) / a.page);
    const Needs needs = needs_of(a, blockIdx.x);
    int from, to;
    stretch<false>(a, wave, from, to);
    const Counted c = count_stretch<false>(a, &needs, from, to, first_pages);
    if ((threadIdx.x & 63) == 0) a.sums[(size_t)blockIdx.x * kManyWaves + wave] = int2{c.needed, c.given};
    if (blockIdx.x == 0 && threadIdx.x == 0) a.sums[(size_t)a.B * kManyWaves] = ring_state(a);  // (the second launch may write over it)
}

__global__ __launch_bounds__(kManyWaves * 64) void kv_tables_place_kernel(const TablesArgs a) {
    __shared__ Counted part[kManyWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first_pages = (int)(((long long)a.sinks + a.page - 1) / a.page);
    const Needs needs = needs_of(a, blockIdx.x);
    const int2 ring = a.sums[(size_t)a.B * kManyWaves];
    Counted c = {0, 0};
    for (size_t w = threadIdx.x; w < (size_t)blockIdx.x * kManyWaves; w += kManyWaves * 64) {
        const int2 s = a.sums[w];
        c.needed += s.x, c.given += s.y;
    }
#pragma unroll
    for (int step = 1; step < 64; step *= 2) c.needed += __shfl_xor(c.needed, step), c.given += __shfl_xor(c.given, step);
    if (lane == 0) part[wave] = c;
    __syncthreads();
    Counted base = {0, 0};
#pragma unroll
    for (int w = 0; w < kManyWaves; w++) base.needed += part[w].needed, base.given += part[w].given;
    Counted total = base;
#pragma unroll
    for (int w = 0; w < kManyWaves; w++) {
        const int2 s = a.sums[(size_t)blockIdx.x * kManyWaves + w];
        if (w < wave) base.needed += s.x, base.given += s.y;
        total.needed += s.x, total.given += s.y;
    }
    int from, to;
    stretch<false>(a, wave, from, to);
    place_stretch<false>(a, &needs, from, to, first_pages, base, ring);
    if ((int)blockIdx.x == a.B - 1 && threadIdx.x == 0) store_state(a, total, ring);
    __syncthreads();
    store_slots(a, blockIdx.x, 1, kManyWaves * 64);
}

// Slots of many rows, behind the launch that writes the tables.
__global__ __launch_bounds__(256) void kv_slots_kernel(const TablesArgs a) {
    const int i = (int)(blockIdx.x * 256 + threadIdx.x);
    if (i < a.n) a.slots[(size_t)blockIdx.y * a.n + i] = slot_of(a, blockIdx.y, i);
}

int check_sizes(const char *fn, int max_pages, int B) {
    ET_REQUIRE(max_pages > 0 && B >= 0, ET_ERR_INVALID_ARG, "%s: max_pages=%d B=%d", fn, max_pages, B);
    // (max_pages: entries rounded up to those of all waves, and the last step behind them, stay below 2^31)
    ET_REQUIRE(B <= 65535 && max_pages <= 0x7ffffe00 && (long long)B * max_pages <= 0x7fffffffLL, ET_ERR_UNSUPPORTED, "%s: B=%d max_pages=%d", fn, B, max_pages);
    return ET_OK;
}

size_t tables_bytes(int max_pages, int B) { return tables_of_one_workgroup(max_pages, B) ? 0 : ((size_t)B * kManyWaves + 1) * sizeof(int2); }

}  // namespace
}  // namespace et

using namespace et;

extern "C" {

int et_kv_tables_workspace(int max_pages, int B, size_t *bytes) {
    ET_REQUIRE(bytes, ET_ERR_INVALID_ARG, "et_kv_tables_workspace: NULL pointer");
    const int st = check_sizes("et_kv_tables_workspace", max_pages, B);
    if (st == ET_OK) *bytes = tables_bytes(max_pages, B);
    return st;
}

int et_kv_tables(const int32_t *before, int32_t *table, int max_pages, int page, int npages, const int32_t *starts, const int32_t *counts, const int32_t *shared, int B, int n,
                 int window, int sinks, int32_t *free_pages, const int32_t *free_state, int32_t *next_state, int64_t *slots, void *workspace, size_t workspace_bytes,
                 et_stream stream) {
    static const char *fn = "et_kv_tables";
    ET_REQUIRE(before && table && free_pages && free_state && next_state, ET_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const int st = check_sizes(fn, max_pages, B);
    if (st != ET_OK) return st;
    ET_REQUIRE(page > 0 && npages > 0 && n >= 0 && window >= 0 && sinks >= 0, ET_ERR_INVALID_ARG, "%s: page=%d npages=%d n=%d window=%d sinks=%d", fn, page, npages, n, window, sinks);
    ET_REQUIRE((long long)max_pages * page <= 0x7fffff80LL, ET_ERR_UNSUPPORTED, "%s: max_pages * page = %lld positions", fn, (long long)max_pages * page);
    ET_REQUIRE((reinterpret_cast<uintptr_t>(slots) & 7) == 0 && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0, ET_ERR_UNSUPPORTED, "%s: slots and the workspace must be 8-byte aligned", fn);
    const size_t need = tables_bytes(max_pages, B);
    ET_REQUIRE(workspace_bytes >= need && (workspace || need == 0), ET_ERR_INVALID_ARG, "%s: a workspace of %zu bytes, %zu are needed", fn, workspace ? workspace_bytes : 0, need);
    TablesArgs a;
    a.before = before;
    a.table = table;
    a.starts = starts;
    a.counts = counts;
    a.shared = shared;
    a.ring = free_pages;
    a.state = free_state;
    a.next_state = next_state;
    a.slots = reinterpret_cast<long long *>(slots);
    a.sums = static_cast<int2 *>(workspace);
    a.max_pages = max_pages;
    a.page = page;
    a.npages = npages;
    a.B = B;
    a.n = n;
    a.window = window;
    a.sinks = sinks;
    const bool one = tables_of_one_workgroup(max_pages, B), apart = slots && slots_apart(max_pages, B, n);
    if (apart) a.slots = nullptr;
    int sl;
    if (one) {
        sl = launch_kernel("kv_tables_one_kernel", kv_tables_one_kernel, dim3(1), kOneWaves * 64, 0, as_stream(stream), a);
    } else {
        sl = launch_kernel("kv_tables_count_kernel", kv_tables_count_kernel, dim3((unsigned)B), kManyWaves * 64, 0, as_stream(stream), a);
        if (sl == ET_OK) sl = launch_kernel("kv_tables_place_kernel", kv_tables_place_kernel, dim3((unsigned)B), kManyWaves * 64, 0, as_stream(stream), a);
    }
    if (sl != ET_OK || !apart) return sl;
    a.slots = reinterpret_cast<long long *>(slots);
    return launch_kernel("kv_slots_kernel", kv_slots_kernel, dim3((unsigned)((n + 255LL) / 256), (unsigned)B), 256, 0, as_stream(stream), a);
}

}  // extern "C"

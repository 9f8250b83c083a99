// Pages of a cache: copied, shared by rows that go on from other rows, counted, moved to the front of the pool.
//
//   copy     the first tokens[i] slots of page src[i] -> page dst[i], in every plane
//   fork     table[child, j] = table[parent, j] for whole pages of the first len positions; the len mod page tokens behind them are copied to a
//            new page, whose slots the row names from there on
//   count    refs[g] = how many (row, page of the row's length) pairs name page g; free = the pages with refs 0, ascending
//   compact  U = the number of pages with refs > 0; the i-th of them at U or behind moves to the i-th free page below U; the rows' slots
//            follow: a page's new number is itself below U, otherwise dst[rank among the late ones]
//
// Copies are bound by memory: 2 bytes of traffic per byte at 0.97 to 0.98 of the measured copy bandwidth where hundreds of pages move.  Everything
// else is a few thousand integers: launches, trips to memory in a chain and barriers.  So a copy of few pages is one launch, counting a
// small pool one CTA, and the kernels of a longer chain start ahead of the end of the one before.
// Nothing depends on the order of atomics: counts are sums, and lists are made by ranks.
#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kMaxFork = 1024;        // entries of a fork call
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kUnit = 512;            // bytes that a warp moves with one vector per lane; four of them at a time
constexpr int kFewPairs = 32;         // pairs of a copy call that every CTA looks through by itself
constexpr int kSmallPool = 24000;     // pages, and five quarters of those held, that one CTA counts in its shared memory
// Counters of int go on by up to a grid's threads behind the last page or number; the rows' pages are multiplied in 64 bits.
constexpr int kMaxPages = 1 << 30, kMaxRows = 1 << 20;
constexpr int kWords = 8;             // of 32 pages that a warp ranks where many CTAs do (32: 7 us to mark a million pages, 8: 3)
constexpr int kChunk = kWarps * kWords * 32;

// x / d for x < 2^31 by a multiplication.
struct Divisor {
    uint32_t d, m;
    int shift;
    __device__ __forceinline__ uint32_t of(uint32_t x) const { return d == 1 ? x : __umulhi(x, m) >> shift; }
};
Divisor divisor(uint32_t d) {
    // m = ceil(2^(32 + shift) / d) with 2^shift < d <= 2^(shift + 1): below 2^32, and x m / 2^(32 + shift) is too large by less than x / 2^(32 + shift) < 1 / d
    Divisor x{d, 0, 0};
    if (d <= 1) return x;
    while ((2u << x.shift) < d && x.shift < 31) ++x.shift;
    x.m = static_cast<uint32_t>(((uint64_t(1) << (32 + x.shift)) + d - 1) / d);
    return x;
}

struct Pool {
    uint8_t* planes;
    int64_t plane_stride;
    int num_planes, slot_bytes, page_size, num_pages;
};

struct Table {
    const int32_t* slots;
    int64_t rows, stride, cols;
};

__device__ __forceinline__ void report(int* status, int index) { atomicExch(&status[kStatusBadIndex], bad_index_word(index)); }

// How pages are cut into units.  A run is a page of one plane.
struct Units {
    int per_run;          // units of a run of kUnit bytes and more
    int group_log;        // smaller ones: 2^group_log lanes have one
    Divisor per_run_div, planes_div;
};

// Runs [0, pairs * planes): run r is the first slots_of(pair) slots of page src[pair] in its plane.  Warps all over the device take neighbouring
// units.
template <class SlotsOf>
__device__ __forceinline__ void move_pages(const Pool& pool, const Units& units, const int32_t* src, const int32_t* dst, int pairs, SlotsOf&& slots_of) {
    const int lane = threadIdx.x & 31;
    const int64_t page_bytes = static_cast<int64_t>(pool.page_size) * pool.slot_bytes;
    const int64_t runs = static_cast<int64_t>(pairs) * pool.num_planes;
    const int runs_log = 5 - units.group_log;                                 // of a unit, where runs are small
    const int64_t all = runs_log > 0 ? (runs + (1 << runs_log) - 1) >> runs_log : runs * units.per_run;
    const int within = lane & ((1 << units.group_log) - 1);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps * 4;
    for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * 4; at < all; at += step) {
        // the first unit's run by a division, the others' by steps
        int64_t run = at, piece = 0;
        if (runs_log == 0) {
            run = at < 0x7fffffff ? units.per_run_div.of(static_cast<uint32_t>(at)) : at / units.per_run;
            piece = at - run * units.per_run;
        }
        uint4 v[4];
        uint8_t* to[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            to[k] = nullptr;
            const int64_t r = runs_log > 0 ? (run << runs_log) + (lane >> units.group_log) : run;
            const int64_t offset = runs_log > 0 ? within * 16 : piece * kUnit + lane * 16;
            if (runs_log > 0 || ++piece == units.per_run) {
                ++run;
                piece = 0;
            }
            if (r >= runs) continue;
            const uint32_t pair = units.planes_div.of(static_cast<uint32_t>(r)), plane = static_cast<uint32_t>(r) - pair * pool.num_planes;
            if (offset >= static_cast<int64_t>(slots_of(pair)) * pool.slot_bytes) continue;
            uint8_t* base = pool.planes + plane * pool.plane_stride + offset;
            v[k] = __ldcs(reinterpret_cast<const uint4*>(base + src[pair] * page_bytes));
            to[k] = base + dst[pair] * page_bytes;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (to[k] != nullptr) __stcs(reinterpret_cast<uint4*>(to[k]), v[k]);
    }
}

// ---- copy ----------------------------------------------------------------------------------------------------------

// How many slots of each pair are copied: none of a pair whose destination another pair names too, or reads from.  One CTA.
__global__ void __launch_bounds__(1024, 1)
copy_check_kernel(const int32_t* src, const int32_t* dst, const int32_t* tokens, int count, int page_size, int num_pages, int words,
                  uint32_t* named, uint32_t* clash, int32_t* slots, int* status) {
    const int tid = threadIdx.x;
    pdl_launch_dependents();
    for (int w = tid; w < words; w += 1024) named[w] = clash[w] = 0;
    __syncthreads();
    auto there = [&](int i) {
        const int a = src[i], b = dst[i];
        return a >= 0 && b >= 0 && a != b && a < num_pages && b < num_pages && (tokens == nullptr || tokens[i] > 0);
    };
    for (int i = tid; i < count; i += 1024) {
        if (!there(i)) continue;
        const uint32_t bit = 1u << (dst[i] & 31);
        if (atomicOr(&named[dst[i] >> 5], bit) & bit) atomicOr(&clash[dst[i] >> 5], bit);
    }
    __syncthreads();
    for (int i = tid; i < count; i += 1024) {
        if (!there(i)) continue;
        const uint32_t bit = 1u << (src[i] & 31);
        if (__ldcg(&named[src[i] >> 5]) & bit) atomicOr(&clash[src[i] >> 5], bit);
    }
    __syncthreads();
    for (int i = tid; i < count; i += 1024) {
        int n = 0;
        if (there(i)) {
            if (__ldcg(&clash[dst[i] >> 5]) >> (dst[i] & 31) & 1) report(status, dst[i]);
            else n = tokens == nullptr ? page_size : min(tokens[i], page_size);
        } else if (src[i] >= 0 && dst[i] >= 0 && src[i] != dst[i] && (tokens == nullptr || tokens[i] > 0)) {
            report(status, src[i] >= num_pages ? src[i] : dst[i]);
        }
        slots[i] = n;
    }
}

// slots NULL: the pairs are few, and each CTA finds by itself which of its own clash with others.
__global__ void __launch_bounds__(kThreads)
copy_pages_kernel(const Pool pool, const Units units, const int32_t* src, const int32_t* dst, const int32_t* tokens, const int32_t* slots, int count,
                  int* status) {
    __shared__ int s_src[kFewPairs], s_dst[kFewPairs], s_slots[kFewPairs];
    pdl_wait_prior();
    if (slots != nullptr) {
        move_pages(pool, units, src, dst, count, [&](uint32_t pair) { return slots[pair]; });
        return;
    }
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const int a = src[i], b = dst[i], n = tokens == nullptr ? pool.page_size : min(max(tokens[i], 0), pool.page_size);
        const bool inside = a < pool.num_pages && b < pool.num_pages, wanted = a >= 0 && b >= 0 && a != b && n > 0;
        s_src[i] = wanted && inside ? a : -1;
        s_dst[i] = wanted && inside ? b : -2;
        s_slots[i] = wanted && inside ? n : 0;
        if (wanted && !inside && blockIdx.x == 0) report(status, a >= pool.num_pages ? a : b);
    }
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < count; i += kWarps) {
        const int b = s_dst[i];
        if (b < 0) continue;
        bool clash = false;
        for (int k = threadIdx.x & 31; k < count; k += 32) clash = clash || s_src[k] == b || (s_dst[k] == b && k != i);
        if (__any_sync(0xffffffffu, clash) && (threadIdx.x & 31) == 0) {
            s_slots[i] = 0;
            if (blockIdx.x == 0) report(status, b);
        }
    }
    __syncthreads();
    move_pages(pool, units, src, dst, count, [&](uint32_t pair) { return s_slots[pair]; });
}

// ---- fork ----------------------------------------------------------------------------------------------------------

struct ForkParams {
    Pool pool;
    int32_t* table;
    int64_t rows, stride, cols;
    const int32_t *parents, *children, *lens, *new_pages;
    int count;
    int* status;
};

__global__ void __launch_bounds__(kThreads)
fork_rows_kernel(const ForkParams p) {
    const int i = blockIdx.y, tid = threadIdx.x, P = p.pool.page_size;
    const int parent = p.parents[i], child = p.children[i], len = p.lens[i];
    auto row_there = [&](int r) { return r >= 0 && r < p.rows; };
    // the page that entry j copies from, -1: it copies nothing
    auto source = [&](int j, int* slot_out) {
        const int n = p.lens[j], r = p.parents[j];
        if (n <= 0 || n > p.cols || !row_there(r) || n % P == 0) return -1;
        const int slot = p.table[r * p.stride + n / P * P];
        if (slot_out != nullptr) *slot_out = slot;
        return slot >= 0 && slot / P < p.pool.num_pages && slot % P == 0 ? slot / P : -1;
    };
    const bool first = blockIdx.x == 0 && tid == 0;
    if (!row_there(parent) || !row_there(child) || len < 0 || len > p.cols || parent == child) {
        if (first) report(p.status, !row_there(parent) ? parent : !row_there(child) || parent == child ? child : len);
        return;
    }
    const int part = len % P, full = len - part;
    int from = -1, to = -1, slot = 0;
    if (part > 0) {
        from = source(i, &slot);
        to = p.new_pages[i];
        if (from < 0 || to < 0 || to >= p.pool.num_pages) {
            if (first) report(p.status, from < 0 ? slot : to);
            return;
        }
    }
    // 2 KB of a run per warp; its first ones are under way while the entries are compared
    const int64_t page_bytes = static_cast<int64_t>(P) * p.pool.slot_bytes, bytes = static_cast<int64_t>(part) * p.pool.slot_bytes;
    const int lane = tid & 31;
    const uint32_t pieces = static_cast<uint32_t>((bytes + 4 * kUnit - 1) / (4 * kUnit)), items = pieces * p.pool.num_planes, step = gridDim.x * kWarps;
    uint32_t it = blockIdx.x * kWarps + (tid >> 5);
    uint4 v[4];
    uint8_t* base = nullptr;
    int left = 0;
    auto load = [&]() {
        const uint32_t plane = it / pieces;
        const int64_t at = static_cast<int64_t>(it - plane * pieces) * (4 * kUnit);
        base = p.pool.planes + plane * p.pool.plane_stride + at + lane * 16;
        left = static_cast<int>(min(bytes - at, int64_t(4 * kUnit))) - lane * 16;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k * kUnit < left) v[k] = *reinterpret_cast<const uint4*>(base + from * page_bytes + k * kUnit);
    };
    if (it < items) load();
    bool bad_row = false, bad_page = false;
    for (int j = tid; j < p.count; j += kThreads) {
        if (j != i && (p.children[j] == child || p.parents[j] == child)) bad_row = true;
        if (part > 0) {
            const int n = p.lens[j];
            if (j != i && n > 0 && n % P != 0 && p.new_pages[j] == to) bad_page = true;
            if (source(j, nullptr) == to) bad_page = true;
        }
    }
    bad_row = __syncthreads_or(bad_row);
    bad_page = __syncthreads_or(bad_page);
    if (bad_row || bad_page) {
        if (first) report(p.status, bad_row ? child : to);
        return;
    }
    const int32_t* old = p.table + parent * p.stride;
    int32_t* row = p.table + child * p.stride;
    const int64_t end = part > 0 ? min(static_cast<int64_t>(full) + P, p.cols) : full;
    for (int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + tid; at < end; at += static_cast<int64_t>(gridDim.x) * kThreads)
        row[at] = at < full ? old[at] : to * P + static_cast<int>(at - full);
    for (; it < items; it += step) {
        if (it >= step) load();
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k * kUnit < left) __stcs(reinterpret_cast<uint4*>(base + to * page_bytes + k * kUnit), v[k]);
    }
}

// ---- count ---------------------------------------------------------------------------------------------------------

struct HeldParams {
    Table table;
    const int32_t *rows, *lens, *held;
    int count, held_count, page_size, num_pages;
    int* status;
};

// The pages that entry i of the rows holds (i = count: those named outside the table), every step-th of them from the first-th on.
template <class Each>
__device__ __forceinline__ void each_page(const HeldParams& p, int i, int first, int step, Each&& each) {
    if (i == p.count) {
        for (int k = first; k < p.held_count; k += step) {
            const int g = p.held[k];
            if (g >= 0 && g < p.num_pages) each(g, 1);
            else report(p.status, g);
        }
        return;
    }
    const int r = p.rows[i];
    if (r < 0 || r >= p.table.rows) {
        if (first == 0) report(p.status, r);
        return;
    }
    const int64_t len = min(static_cast<int64_t>(max(p.lens[i], 0)), p.table.cols);
    const int32_t* row = p.table.slots + r * p.table.stride;
    const uint32_t P = static_cast<uint32_t>(p.page_size);
    const int64_t stride = static_cast<int64_t>(step) * P;
    for (int64_t at = static_cast<int64_t>(first) * P; at < len; at += 4 * stride) {
        int slot[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) slot[k] = at + k * stride < len ? row[at + k * stride] : 0;
        const bool alike = at + 3 * stride < len && slot[0] == slot[1] && slot[0] == slot[2] && slot[0] == slot[3];   // (zeros behind a row's pages)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (at + k * stride >= len || (alike && k > 0)) break;
            const uint32_t g = static_cast<uint32_t>(slot[k]) / P;
            if (slot[k] >= 0 && g < static_cast<uint32_t>(p.num_pages) && static_cast<uint32_t>(slot[k]) == g * P) each(static_cast<int>(g), alike ? 4 : 1);
            else report(p.status, slot[k]);
        }
    }
}

__global__ void __launch_bounds__(kThreads)
count_held_kernel(const HeldParams p, int32_t* refs) {
    pdl_launch_dependents();
    pdl_wait_prior();
    // Rows whose lengths reach past their pages name page 0 from there on, where tables begin as zeros: one addition per warp and four places
    // of it.  (Half a million additions to one page one by one: 300 us; by warps 17.  The framework's own requests have no such lengths.)
    each_page(p, blockIdx.x, blockIdx.y * kThreads + threadIdx.x, gridDim.y * kThreads, [&](int g, int n) {
        const uint32_t with = __activemask();
        int same;
        __match_all_sync(with, g, &same);
        const int all = same ? static_cast<int>(__reduce_add_sync(with, n)) : n;
        if (!same || (threadIdx.x & 31) == __ffs(with) - 1) atomicAdd(&refs[g], all);
    });
}

// Which pages are held, a bit each, and how many of the CTA's kChunk.
__global__ void __launch_bounds__(kThreads)
mark_held_kernel(const int32_t* refs, int num_pages, uint32_t* bits, int32_t* counts) {
    __shared__ int s_sum[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait_prior();
    uint32_t mine = 0;
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
        const int64_t page = static_cast<int64_t>(blockIdx.x) * kChunk + (warp * kWords + k) * 32 + lane;
        const uint32_t word = __ballot_sync(0xffffffffu, page < num_pages && refs[page] != 0);
        if (lane == k) mine = word;
    }
    if (lane < kWords) bits[(blockIdx.x * kWarps + warp) * kWords + lane] = mine;
    const int sum = __reduce_add_sync(0xffffffffu, __popc(mine));
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        int all = 0;
        for (int w = 0; w < kWarps; ++w) all += s_sum[w];
        counts[blockIdx.x] = all;
    }
}

// Where each page of the CTA's kChunk stands: each(page, held, pages held before it, all of them, those of them below that number).
template <class Each>
__device__ __forceinline__ void ranked_pages(const uint32_t* bits, const int32_t* counts, int chunks, int num_pages, Each&& each) {
    __shared__ int s_sum[3][kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = blockIdx.x;
    auto all = [&](int v, int which) {
        v = __reduce_add_sync(0xffffffffu, v);
        __syncthreads();
        if (lane == 0) s_sum[which][warp] = v;
        __syncthreads();
        int sum = 0;
        for (int w = 0; w < kWarps; ++w) sum += s_sum[which][w];
        return sum;
    };
    const uint32_t mine = lane < kWords ? bits[(me * kWarps + warp) * kWords + lane] : 0u;
    int before = 0, total = 0;
    for (int c = tid; c < chunks; c += kThreads) {
        total += counts[c];
        if (c < me) before += counts[c];
    }
    before = all(before, 0);
    total = all(total, 1);
    int below = 0;
    const int edge = total / kChunk, rest = total - edge * kChunk - tid * 32;   // the chunk that the number lies in; pages below it from this word on
    for (int c = tid; c < edge; c += kThreads) below += counts[c];
    if (edge < chunks && tid < kChunk / 32 && rest > 0) below += __popc(bits[edge * (kChunk / 32) + tid] & (rest >= 32 ? ~0u : (1u << rest) - 1u));
    below = all(below, 2);
    int scan = __popc(mine);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += up;
    }
    __syncthreads();
    if (lane == 31) s_sum[0][warp] = scan;
    __syncthreads();
    scan += before - __popc(mine);
    for (int w = 0; w < warp; ++w) scan += s_sum[0][w];
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
        const uint32_t word = __shfl_sync(0xffffffffu, mine, k);
        const int base = __shfl_sync(0xffffffffu, scan, k);
        const int64_t page = static_cast<int64_t>(me) * kChunk + (warp * kWords + k) * 32 + lane;
        if (page < num_pages) each(static_cast<int>(page), (word >> lane & 1) != 0, base + __popc(word & ((1u << lane) - 1u)), total, below);
    }
}

// All of that by one CTA of 1024 threads, the counts in its shared memory.
template <class Each>
__device__ __forceinline__ void count_and_rank(const HeldParams& p, int* refs, Each&& each) {
    __shared__ int s_sum[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int g = tid; g < p.num_pages; g += 1024) refs[g] = 0;
    __syncthreads();
    for (int i = warp; i < p.count; i += 32) each_page(p, i, lane, 32, [&](int g, int n) { atomicAdd(&refs[g], n); });
    each_page(p, p.count, tid, 1024, [&](int g, int n) { atomicAdd(&refs[g], n); });
    __syncthreads();
    const int share = (p.num_pages + 1023) / 1024 * 32, first = warp * share, end = min(first + share, p.num_pages);   // of a warp
    int held = 0;
    for (int g = first + lane; g < end; g += 32) held += refs[g] != 0;
    held = __reduce_add_sync(0xffffffffu, held);
    if (lane == 0) s_sum[0][warp] = held;
    __syncthreads();
    const int others = s_sum[0][lane];
    const int total = __reduce_add_sync(0xffffffffu, others), before0 = __reduce_add_sync(0xffffffffu, lane < warp ? others : 0);
    int below = 0;
    for (int g = first + lane; g < min(end, total); g += 32) below += refs[g] != 0;
    below = __reduce_add_sync(0xffffffffu, below);
    if (lane == 0) s_sum[1][warp] = below;
    __syncthreads();
    below = __reduce_add_sync(0xffffffffu, s_sum[1][lane]);
    int before = before0;
    for (int base = first; base < end; base += 32) {
        const int g = base + lane, n = g < end ? refs[g] : 0;
        const uint32_t word = __ballot_sync(0xffffffffu, n != 0);
        if (g < end) each(g, n, before + __popc(word & ((1u << lane) - 1u)), total, below);
        before += __popc(word);
    }
}

__device__ __forceinline__ void list_page(int page, bool held, int before, int total, int num_pages, int32_t* free_pages, int32_t* free_count) {
    if (held) free_pages[num_pages - total + before] = -1;
    else free_pages[page - before] = page;
    if (page == 0) free_count[0] = num_pages - total;
}
__global__ void __launch_bounds__(kThreads)
list_free_kernel(const uint32_t* bits, const int32_t* counts, int chunks, int num_pages, int32_t* free_pages, int32_t* free_count) {
    pdl_wait_prior();
    ranked_pages(bits, counts, chunks, num_pages, [&](int page, bool held, int before, int total, int) {
        list_page(page, held, before, total, num_pages, free_pages, free_count);
    });
}
__global__ void __launch_bounds__(1024, 1)
count_small_kernel(const HeldParams p, int32_t* refs, int32_t* free_pages, int32_t* free_count) {
    extern __shared__ int s_refs[];
    count_and_rank(p, s_refs, [&](int page, int n, int before, int total, int) {
        refs[page] = n;
        list_page(page, n != 0, before, total, p.num_pages, free_pages, free_count);
    });
}

// ---- compact -------------------------------------------------------------------------------------------------------

struct CompactParams {
    Pool pool;
    Units units;
    HeldParams held;
    int32_t *out, *map, *used;
    int64_t out_stride;
    int32_t *src, *dst, *rank, *moves;   // pages that move, where to, the number of a page among them; how many
};

__device__ __forceinline__ void plan_page(const CompactParams& p, int page, bool held, int before, int total, int below) {
    if (page < total) {
        p.map[page] = held ? page : -1;
        if (!held) p.dst[page - before] = page;
    } else if (held) {
        p.src[before - below] = page;
        p.rank[page] = before - below;
    } else {
        p.map[page] = -1;
    }
    if (page == 0) {
        p.used[0] = total;
        p.moves[0] = total - below;
    }
}
__global__ void __launch_bounds__(kThreads)
plan_moves_kernel(const uint32_t* bits, const int32_t* counts, int chunks, const CompactParams p) {
    pdl_launch_dependents();
    pdl_wait_prior();
    ranked_pages(bits, counts, chunks, p.pool.num_pages, [&](int page, bool held, int before, int total, int below) {
        plan_page(p, page, held, before, total, below);
    });
}
__global__ void __launch_bounds__(1024, 1)
plan_small_kernel(const CompactParams p) {
    extern __shared__ int s_refs[];
    pdl_launch_dependents();
    count_and_rank(p.held, s_refs, [&](int page, int n, int before, int total, int below) { plan_page(p, page, n != 0, before, total, below); });
}

__global__ void __launch_bounds__(kThreads)
compact_kernel(const CompactParams p) {
    const int P = p.pool.page_size, lane = threadIdx.x & 31;
    const Table& t = p.held.table;
    int group = 1;                            // lanes per page of the table: they read its first slot before they write any
    while (group < 32 && group * 2 <= P) group *= 2;
    const int sub = lane / group, in = lane % group, per_cta = kWarps * 32 / group;
    pdl_wait_prior();
    const int pairs = p.moves[0], total = p.used[0];
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < pairs; i += gridDim.x * kThreads) p.map[p.src[i]] = p.dst[i];
    // A row's table by the CTAs whose number leaves its own when divided by the number of rows.
    const int rows = p.held.count;
    for (int i = rows > 0 ? static_cast<int>(blockIdx.x) % rows : 0; i < rows; i += gridDim.x) {
        const int r = p.held.rows[i];
        if (r < 0 || r >= t.rows) continue;
        const int64_t len = min(static_cast<int64_t>(max(p.held.lens[i], 0)), t.cols);
        const int64_t pages = (len + P - 1) / P;
        const int sharing = (static_cast<int>(gridDim.x) - i + rows - 1) / rows;   // CTAs of this row (0: one, in its turn)
        const int64_t step = static_cast<int64_t>(max(sharing, 1)) * per_cta;
        for (int64_t base = static_cast<int64_t>(blockIdx.x / rows) * per_cta + (threadIdx.x >> 5) * (32 / group); base < pages; base += step) {
            const int64_t j = base + sub, at = j * P;
            const int slot = j < pages ? t.slots[r * t.stride + at] : -1;
            __syncwarp();
            const int g = slot / P;
            if (slot < 0 || g >= p.pool.num_pages || slot % P != 0) continue;
            const int to = g < total ? g : p.dst[p.rank[g]];
            for (int k = in; k < P && at + k < t.cols; k += group) p.out[r * p.out_stride + at + k] = to * P + k;
        }
    }
    move_pages(p.pool, p.units, p.src, p.dst, pairs, [&](uint32_t) { return p.pool.page_size; });
}

// The launches behind another one of the same call start early and wait where they need it.
struct FollowOn {
    const bool was = pdl_launches_enabled();
    explicit FollowOn(bool on = true) { set_pdl_launches(on); }
    ~FollowOn() { set_pdl_launches(was); }
};

// ---- workspace and checks ------------------------------------------------------------------------------------------

struct Layout {
    int chunks;                               // of kChunk pages
    int64_t bits, counts, ints, bytes;        // two arrays of a bit per page, a count per chunk, three arrays of an int per page, a counter
};
Layout layout_of(int num_pages) {
    Layout x;
    auto padded = [](int64_t n) { return div_ceil64(n, 256) * 256; };
    x.chunks = div_ceil(num_pages, kChunk);
    x.bits = padded(static_cast<int64_t>(x.chunks) * (kChunk / 8));
    x.counts = padded(static_cast<int64_t>(x.chunks) * 4);
    x.ints = padded(static_cast<int64_t>(num_pages) * 4);
    x.bytes = 2 * x.bits + x.counts + 3 * x.ints + 256 + 256;
    return x;
}
struct Scratch {
    uint32_t *bits, *bits2;
    int32_t *counts, *ints[3], *one;
};
Scratch scratch_in(void* workspace, const Layout& x) {
    uint8_t* at = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
    Scratch s;
    s.bits = reinterpret_cast<uint32_t*>(at);
    s.bits2 = reinterpret_cast<uint32_t*>(at + x.bits);
    s.counts = reinterpret_cast<int32_t*>(at + 2 * x.bits);
    for (int i = 0; i < 3; ++i) s.ints[i] = reinterpret_cast<int32_t*>(at + 2 * x.bits + x.counts + i * x.ints);
    s.one = reinterpret_cast<int32_t*>(at + 2 * x.bits + x.counts + 3 * x.ints);
    return s;
}
Units units_of(const Pool& pool) {
    Units u;
    const int64_t page_bytes = static_cast<int64_t>(pool.page_size) * pool.slot_bytes;
    u.per_run = static_cast<int>(div_ceil64(page_bytes, kUnit));
    u.group_log = 0;
    while (u.group_log < 5 && (16ll << u.group_log) < page_bytes) ++u.group_log;
    u.per_run_div = divisor(static_cast<uint32_t>(u.per_run));
    u.planes_div = divisor(static_cast<uint32_t>(pool.num_planes));
    return u;
}
// CTAs for `pairs` pages: one for every 16 KB.  As long as they are known to be there, up to sixteen waves of them (a wave: eight CTAs per SM): those
// that run at a time then work on neighbouring pages (700 pages of 1.8 MB: 421 us with one wave, 407 with four, 398 with sixteen, 396 with all).  Where
// `pairs` is what there may be at most, four waves, or half a one if even that is little (800 of 1600 such pages in use 170 us with one wave, 164
// with four; 6 short requests in a pool of 64 pages 11.7, 13, 17 us with half a wave, one, four).
int move_grid(const Pool& pool, const Units& u, int64_t pairs, bool known) {
    const int64_t runs = pairs * pool.num_planes, units = u.group_log < 5 ? (runs >> (5 - u.group_log)) + 1 : runs * u.per_run;
    const int64_t wave = static_cast<int64_t>(sm_count()) * 8;
    return static_cast<int>(min(div_ceil64(units, kWarps * 4), known ? 16 * wave : units * kUnit > (256 << 20) ? 4 * wave : wave / 2));
}

int check_pool(const b200_page_pool* pool, const char* name, Pool* out) {
    B200_CHECK_ARG(pool != nullptr, "%s: NULL pool", name);
    B200_CHECK_ARG(pool->page_size >= 1 && pool->num_pages >= 1 && static_cast<int64_t>(pool->page_size) * pool->num_pages <= 0x7fffffff,
                   "%s: page_size and num_pages must be positive, of fewer than 2^31 slots", name);
    B200_CHECK_ARG(pool->num_pages <= kMaxPages, "%s: num_pages must be at most 2^30", name);
    B200_CHECK_ARG(pool->num_planes >= 1 && static_cast<int64_t>(pool->num_planes) * pool->num_pages <= 0x7fffffff,
                   "%s: num_planes must be positive, with fewer than 2^31 pages in all planes", name);
    B200_CHECK_ARG(pool->slot_bytes >= 16 && pool->slot_bytes % 16 == 0, "%s: slot_bytes must be a positive multiple of 16", name);
    B200_CHECK_ARG(pool->num_planes == 1 || (pool->plane_stride % 16 == 0 && pool->plane_stride >= static_cast<int64_t>(pool->slot_bytes) *
                                                                               pool->page_size * pool->num_pages),
                   "%s: plane_stride must be a multiple of 16 and planes must not overlap", name);
    B200_CHECK_ARG(pool->planes != nullptr && reinterpret_cast<uintptr_t>(pool->planes) % 16 == 0, "%s: planes must not be NULL and be 16-byte aligned", name);
    *out = Pool{static_cast<uint8_t*>(pool->planes), pool->plane_stride, pool->num_planes, pool->slot_bytes, pool->page_size, pool->num_pages};
    return B200_OK;
}
int check_table(const char* name, int64_t rows, int64_t stride, int64_t cols) {
    B200_CHECK_ARG(rows >= 0 && rows <= 0x7fffffff && cols >= 0 && cols <= 0x7fffffff, "%s: table rows and columns must be in [0, 2^31)", name);
    B200_CHECK_ARG(stride >= cols || rows <= 1, "%s: rows of the page table must not overlap", name);
    return B200_OK;
}
int check_workspace(const char* name, const void* workspace, int64_t bytes, const Layout& x) {
    B200_CHECK_ARG(workspace != nullptr && bytes >= x.bytes, "%s: workspace of %lld bytes is too small (need %lld)", name,
                   static_cast<long long>(workspace != nullptr ? bytes : 0), static_cast<long long>(x.bytes));
    return B200_OK;
}

int check_held(const char* name, const HeldParams& p) {
    int err = check_table(name, p.table.rows, p.table.stride, p.table.cols);
    if (err != B200_OK) return err;
    B200_CHECK_ARG(p.count >= 0 && p.count <= kMaxRows && p.held_count >= 0 && p.held_count <= kMaxPages,
                   "%s: count must be in [0, 2^20] and held_count in [0, 2^30]", name);
    B200_CHECK_ARG(p.count == 0 || (p.rows && p.lens && (p.table.slots || p.table.rows * p.table.cols == 0)), "%s: NULL tensor", name);
    B200_CHECK_ARG(p.held_count == 0 || p.held, "%s: NULL tensor", name);
    return B200_OK;
}

// Does one CTA count them sooner than many, in four launches?  (Lengths are on the device: rows may be as long as the table's.)  us by one, by many:
// 1000 pages of which 800 are held 3.3, 8.5, 9600 times held 6.6, 8.4, 64000 times 18, 13; 9000 pages 5.2, 6.8 and 8.7, 6.7 and 20, 8.0; 20000
// pages 8.0, 6.7.  Three launches less are 5 us of the caller's time besides (64 rows of up to 2000 tokens, 9000 pages of 16: a call that nothing
// captures 13.8 by one, 19.2 by many), so that one CTA may take 2 us longer.
bool small(const HeldParams& p) {
    const int64_t held = div_ceil64(p.table.cols, p.page_size) * p.count + p.held_count;
    return p.num_pages + held * 5 / 4 <= kSmallPool;
}
// The pages held, counted and as bits, by many CTAs.
int launch_held(const HeldParams& p, int32_t* refs, uint32_t* bits, int32_t* counts, int chunks, cudaStream_t stream) {
    B200_CHECK_CUDA(cudaMemsetAsync(refs, 0, static_cast<size_t>(p.num_pages) * 4, stream));
    if (p.count > 0 || p.held_count > 0) {
        const int64_t most = max(div_ceil64(p.table.cols, p.page_size), static_cast<int64_t>(p.held_count));
        const int y = static_cast<int>(min(max(div_ceil64(most, 4 * kThreads), int64_t(1)), int64_t(64)));
        B200_CHECK_CUDA(launch_kernel(count_held_kernel, dim3(p.count + 1, y), dim3(kThreads), 0, stream, dim3(1, 1, 1), p, refs));
    }
    FollowOn follow(p.count > 0 || p.held_count > 0);
    B200_CHECK_CUDA(launch_kernel(mark_held_kernel, dim3(chunks), dim3(kThreads), 0, stream, dim3(1, 1, 1), refs, p.num_pages, bits, counts));
    return B200_OK;
}
template <class Kernel, class... Args>
int launch_small(Kernel kernel, const HeldParams& p, cudaStream_t stream, Args... args) {
    const int smem = p.num_pages * 4;
    static std::atomic<uint64_t> asked{0};   // (one per kernel: their types differ)
    B200_CHECK_CUDA(allow_smem(asked, reinterpret_cast<const void*>(kernel), kSmallPool * 4));
    B200_CHECK_CUDA(launch_kernel(kernel, dim3(1), dim3(1024), smem, stream, dim3(1, 1, 1), args...));
    return B200_OK;
}

}  // namespace
}  // namespace b200

extern "C" {

int64_t b200_pages_workspace_bytes(int num_pages) {
    if (num_pages < 1 || num_pages > b200::kMaxPages) return -1;
    return b200::layout_of(num_pages).bytes;
}

int b200_copy_pages(const b200_page_pool* pool, const int32_t* src, const int32_t* dst, const int32_t* tokens, int count,
                    void* workspace, int64_t workspace_bytes, b200_stream_t stream) {
    using namespace b200;
    Pool p;
    int err = check_pool(pool, "copy_pages", &p);
    if (err != B200_OK) return err;
    B200_CHECK_ARG(count >= 0 && count <= p.num_pages, "copy_pages: count must be in [0, num_pages]");
    if (count == 0) return B200_OK;
    B200_CHECK_ARG(src && dst, "copy_pages: NULL tensor");
    const Layout x = layout_of(p.num_pages);
    err = check_workspace("copy_pages", workspace, workspace_bytes, x);
    if (err != B200_OK) return err;
    int* status = device_status_words(&err);
    if (err != B200_OK) return err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const Units units = units_of(p);
    const int grid = move_grid(p, units, count, true);
    // Few pairs that all SMs move at once: every CTA compares all of them.  Others: one CTA does, with a bit per page, ahead of the copies.  (us
    // with that kernel, without: 1 page of 1.8 MB 5.6, 3.7; 16 12.4, 13.5; 128 78, 228; 16 pages of 115 KB 5.7, 4.1; 64 7.1, 7.8; 64 of 1 KB 5.3, 5.5.)
    int32_t* slots = nullptr;
    const bool ahead = count > kFewPairs || grid > sm_count() * 8;
    if (ahead) {
        const Scratch w = scratch_in(workspace, x);
        slots = w.ints[0];
        B200_CHECK_CUDA(launch_kernel(copy_check_kernel, dim3(1), dim3(1024), 0, s, dim3(1, 1, 1), src, dst, tokens, count, p.page_size, p.num_pages,
                                      div_ceil(p.num_pages, 32), w.bits, w.bits2, slots, status));
    }
    FollowOn follow(ahead);
    B200_CHECK_CUDA(launch_kernel(copy_pages_kernel, dim3(grid), dim3(kThreads), 0, s, dim3(1, 1, 1), p, units, src, dst, tokens, slots, count, status));
    return B200_OK;
}

int b200_fork_rows(const b200_page_pool* pool, int32_t* page_table, int64_t table_rows, int64_t page_table_stride, int64_t table_cols,
                   const int32_t* parents, const int32_t* children, const int32_t* lens, const int32_t* new_pages, int count,
                   b200_stream_t stream) {
    using namespace b200;
    ForkParams p;
    int err = check_pool(pool, "fork_rows", &p.pool);
    if (err != B200_OK) return err;
    err = check_table("fork_rows", table_rows, page_table_stride, table_cols);
    if (err != B200_OK) return err;
    B200_CHECK_ARG(count >= 0 && count <= kMaxFork, "fork_rows: count must be in [0, %d]", kMaxFork);
    if (count == 0) return B200_OK;
    B200_CHECK_ARG(page_table && parents && children && lens && new_pages, "fork_rows: NULL tensor");
    p.status = device_status_words(&err);
    if (err != B200_OK) return err;
    p.table = page_table;
    p.rows = table_rows;
    p.stride = page_table_stride;
    p.cols = table_cols;
    p.parents = parents;
    p.children = children;
    p.lens = lens;
    p.new_pages = new_pages;
    p.count = count;
    // (96 rows with half a page of 8.4 MB each: 32.5 us with CTAs for eight per SM, 31.1 with sixteen, 32.2, 34.5, 37.6 with 24, 32, 48: each compares
    // the entries.)
    const int parts = max(1, min(div_ceil(sm_count() * 16, count), 64));
    B200_CHECK_CUDA(launch_kernel(fork_rows_kernel, dim3(parts, count), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), dim3(1, 1, 1), p));
    return B200_OK;
}

int b200_count_pages(int32_t* refs, int32_t* free_pages, int32_t* free_count, const int32_t* page_table, int64_t table_rows,
                     int64_t page_table_stride, int64_t table_cols, const int32_t* rows, const int32_t* lens, int count,
                     const int32_t* held, int held_count, int page_size, int num_pages, void* workspace, int64_t workspace_bytes,
                     b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(page_size >= 1 && num_pages >= 1 && static_cast<int64_t>(page_size) * num_pages <= 0x7fffffff,
                   "count_pages: page_size and num_pages must be positive, of fewer than 2^31 slots");
    B200_CHECK_ARG(num_pages <= kMaxPages, "count_pages: num_pages must be at most 2^30");
    B200_CHECK_ARG(refs && free_pages && free_count, "count_pages: NULL tensor");
    HeldParams p{Table{page_table, table_rows, page_table_stride, table_cols}, rows, lens, held, count, held_count, page_size, num_pages, nullptr};
    int err = check_held("count_pages", p);
    if (err != B200_OK) return err;
    const Layout x = layout_of(num_pages);
    err = check_workspace("count_pages", workspace, workspace_bytes, x);
    if (err != B200_OK) return err;
    p.status = device_status_words(&err);
    if (err != B200_OK) return err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (small(p)) return launch_small(count_small_kernel, p, s, p, refs, free_pages, free_count);
    const Scratch w = scratch_in(workspace, x);
    err = launch_held(p, refs, w.bits, w.counts, x.chunks, s);
    if (err != B200_OK) return err;
    FollowOn follow;
    B200_CHECK_CUDA(launch_kernel(list_free_kernel, dim3(x.chunks), dim3(kThreads), 0, s, dim3(1, 1, 1), w.bits, w.counts, x.chunks, num_pages, free_pages,
                                  free_count));
    return B200_OK;
}

int b200_compact_pages(const b200_page_pool* pool, int32_t* table_out, int64_t table_out_stride, int32_t* map, int32_t* used,
                       const int32_t* page_table, int64_t table_rows, int64_t page_table_stride, int64_t table_cols,
                       const int32_t* rows, const int32_t* lens, int count, const int32_t* held, int held_count, void* workspace,
                       int64_t workspace_bytes, b200_stream_t stream) {
    using namespace b200;
    CompactParams p;
    int err = check_pool(pool, "compact_pages", &p.pool);
    if (err != B200_OK) return err;
    B200_CHECK_ARG(map && used, "compact_pages: NULL tensor");
    p.held = HeldParams{Table{page_table, table_rows, page_table_stride, table_cols}, rows, lens, held, count, held_count, p.pool.page_size,
                        p.pool.num_pages, nullptr};
    err = check_held("compact_pages", p.held);
    if (err != B200_OK) return err;
    B200_CHECK_ARG(count == 0 || table_out || table_rows * table_cols == 0, "compact_pages: NULL tensor");
    B200_CHECK_ARG(table_out_stride >= table_cols || table_rows <= 1, "compact_pages: rows of table_out must not overlap");
    const Layout x = layout_of(p.pool.num_pages);
    err = check_workspace("compact_pages", workspace, workspace_bytes, x);
    if (err != B200_OK) return err;
    p.held.status = device_status_words(&err);
    if (err != B200_OK) return err;
    const Scratch w = scratch_in(workspace, x);
    p.units = units_of(p.pool);
    p.out = table_out;
    p.out_stride = table_out_stride;
    p.map = map;
    p.used = used;
    p.rank = w.ints[0];            // (the counts of holders are not needed any more where ranks are written)
    p.src = w.ints[1];
    p.dst = w.ints[2];
    p.moves = w.one;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (small(p.held)) {
        err = launch_small(plan_small_kernel, p.held, s, p);
        if (err != B200_OK) return err;
    } else {
        err = launch_held(p.held, w.ints[0], w.bits, w.counts, x.chunks, s);
        if (err != B200_OK) return err;
        FollowOn follow;
        B200_CHECK_CUDA(launch_kernel(plan_moves_kernel, dim3(x.chunks), dim3(kThreads), 0, s, dim3(1, 1, 1), w.bits, w.counts, x.chunks, p));
    }
    FollowOn follow;
    const int grid = max(move_grid(p.pool, p.units, p.pool.num_pages / 2 + 1, false), min(count, sm_count() * 8));
    B200_CHECK_CUDA(launch_kernel(compact_kernel, dim3(grid), dim3(kThreads), 0, s, dim3(1, 1, 1), p));
    return B200_OK;
}

}  // extern "C"

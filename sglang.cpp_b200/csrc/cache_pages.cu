// Pages of a cache: copied, shared by rows that go on from other rows, counted, moved to the front of the pool.
#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kMaxFork = 1024;        // entries of a fork call
constexpr int kThreads = 256;
constexpr int kPiece = 2048;          // bytes that a warp moves at a time: four 16-byte vectors per lane

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

// `bytes` (a multiple of 16) from one place to another by a warp.
__device__ __forceinline__ void move_piece(uint8_t* to, const uint8_t* from, int bytes, int lane) {
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = (k * 32 + lane) * 16;
        if (at < bytes) v[k] = *reinterpret_cast<const uint4*>(from + at);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int at = (k * 32 + lane) * 16;
        if (at < bytes) *reinterpret_cast<uint4*>(to + at) = v[k];
    }
}

// ---- copy ----------------------------------------------------------------------------------------------------------

// How many slots of each pair are copied: none of a pair whose destination another pair names too, or reads from.  One CTA.
__global__ void __launch_bounds__(1024, 1)
copy_check_kernel(const int32_t* src, const int32_t* dst, const int32_t* tokens, int count, int page_size, int num_pages, int words,
                  uint32_t* named, uint32_t* clash, int32_t* slots, int* status) {
    const int tid = threadIdx.x;
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
        } else if (src[i] >= 0 && dst[i] >= 0) {
            if (src[i] >= num_pages) report(status, src[i]);
            if (dst[i] >= num_pages) report(status, dst[i]);
        }
        slots[i] = n;
    }
}

__device__ __forceinline__ void move_pages(const Pool& pool, const int32_t* src, const int32_t* dst, const int32_t* slots, int pairs) {
    const int lane = threadIdx.x & 31;
    const int64_t page_bytes = static_cast<int64_t>(pool.page_size) * pool.slot_bytes;
    const int64_t pieces = (page_bytes + kPiece - 1) / kPiece;
    const int64_t items = static_cast<int64_t>(pairs) * pool.num_planes * pieces;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    for (int64_t it = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); it < items; it += warps) {
        const int64_t run = it / pieces, at = (it - run * pieces) * kPiece;
        const int pair = static_cast<int>(run / pool.num_planes), plane = static_cast<int>(run - static_cast<int64_t>(pair) * pool.num_planes);
        const int64_t bytes = static_cast<int64_t>(slots != nullptr ? slots[pair] : pool.page_size) * pool.slot_bytes;
        if (at >= bytes) continue;
        uint8_t* base = pool.planes + plane * pool.plane_stride + at;
        move_piece(base + dst[pair] * page_bytes, base + src[pair] * page_bytes, static_cast<int>(min(bytes - at, static_cast<int64_t>(kPiece))), lane);
    }
}

__global__ void __launch_bounds__(kThreads)
copy_pages_kernel(const Pool pool, const int32_t* src, const int32_t* dst, const int32_t* slots, int count) {
    move_pages(pool, src, dst, slots, count);
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
    if (part == 0) return;
    const int64_t page_bytes = static_cast<int64_t>(P) * p.pool.slot_bytes, bytes = static_cast<int64_t>(part) * p.pool.slot_bytes;
    const int64_t pieces = (bytes + kPiece - 1) / kPiece, items = pieces * p.pool.num_planes;
    for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (tid >> 5); it < items; it += static_cast<int64_t>(gridDim.x) * (kThreads / 32)) {
        const int64_t plane = it / pieces, at = (it - plane * pieces) * kPiece;
        uint8_t* base = p.pool.planes + plane * p.pool.plane_stride + at;
        move_piece(base + to * page_bytes, base + from * page_bytes, static_cast<int>(min(bytes - at, static_cast<int64_t>(kPiece))), tid & 31);
    }
}

// ---- count ---------------------------------------------------------------------------------------------------------

struct HeldParams {
    Table table;
    const int32_t *rows, *lens, *held;
    int count, held_count, page_size, num_pages;
    int* status;
};

// The pages that entry i of the rows holds (blockIdx.x = count: those named outside the table), each once per holder.
template <class Each>
__device__ __forceinline__ void each_page(const HeldParams& p, int i, Each&& each) {
    const int first = blockIdx.y * blockDim.x + threadIdx.x, step = gridDim.y * blockDim.x;
    if (i == p.count) {
        for (int k = first; k < p.held_count; k += step) {
            const int g = p.held[k];
            if (g >= 0 && g < p.num_pages) each(g);
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
    for (int64_t at = static_cast<int64_t>(first) * p.page_size; at < len; at += static_cast<int64_t>(step) * p.page_size) {
        const int slot = row[at];
        if (slot >= 0 && slot / p.page_size < p.num_pages && slot % p.page_size == 0) each(slot / p.page_size);
        else report(p.status, slot);
    }
}

__global__ void __launch_bounds__(kThreads)
mark_pages_kernel(const HeldParams p, uint32_t* bits, int32_t* refs) {
    each_page(p, blockIdx.x, [&](int g) {
        if (refs == nullptr || atomicAdd(&refs[g], 1) == 0) atomicOr(&bits[g >> 5], 1u << (g & 31));
    });
}

// Where each page stands: `each(page, used, pages used before it, total, used below the total)` for the 8192 pages of this CTA.
// Every CTA adds up all of the bits by itself (128 KB for a million pages).
template <class Each>
__device__ __forceinline__ void ranked_pages(const uint32_t* bits, int words, int num_pages, Each&& each) {
    __shared__ int s_sum[3][kThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first = blockIdx.x * kThreads;
    auto all = [&](int v, int which) {
        v = __reduce_add_sync(0xffffffffu, v);
        __syncthreads();
        if (lane == 0) s_sum[which][warp] = v;
        __syncthreads();
        int sum = 0;
        for (int w = 0; w < kThreads / 32; ++w) sum += s_sum[which][w];
        return sum;
    };
    int before = 0, total = 0;
    for (int w = tid; w < words; w += kThreads) {
        const int c = __popc(bits[w]);
        total += c;
        if (w < first) before += c;
    }
    before = all(before, 0);
    total = all(total, 1);
    int below = 0;
    for (int w = tid; w * 32 < total; w += kThreads) below += __popc(total - w * 32 >= 32 ? bits[w] : bits[w] & ((1u << (total - w * 32)) - 1u));
    below = all(below, 2);
    const uint32_t mine = first + tid < words ? bits[first + tid] : 0u;
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
    for (int k = 0; k < 32; ++k) {
        const uint32_t word = __shfl_sync(0xffffffffu, mine, k);
        const int base = __shfl_sync(0xffffffffu, scan, k);
        const int64_t page = (static_cast<int64_t>(first) + warp * 32 + k) * 32 + lane;
        if (page < num_pages) each(static_cast<int>(page), (word >> lane & 1) != 0, base + __popc(word & ((1u << lane) - 1u)), total, below);
    }
}

__global__ void __launch_bounds__(kThreads)
list_free_kernel(const uint32_t* bits, int words, int num_pages, int32_t* free_pages, int32_t* free_count) {
    ranked_pages(bits, words, num_pages, [&](int page, bool used, int before, int total, int) {
        if (used) free_pages[num_pages - total + before] = -1;
        else free_pages[page - before] = page;
        if (page == 0) free_count[0] = num_pages - total;
    });
}

// ---- compact -------------------------------------------------------------------------------------------------------

struct CompactParams {
    Pool pool;
    HeldParams held;
    int32_t *out, *map, *used;
    int64_t out_stride;
    int32_t *src, *dst, *rank, *moves;   // pages that move, where to, the number of a page among them; how many
};

__global__ void __launch_bounds__(kThreads)
plan_moves_kernel(const uint32_t* bits, int words, const CompactParams p) {
    ranked_pages(bits, words, p.pool.num_pages, [&](int page, bool used, int before, int total, int below) {
        if (page < total) {
            p.map[page] = used ? page : -1;
            if (!used) p.dst[page - before] = page;
        } else if (used) {
            p.src[before - below] = page;
            p.rank[page] = before - below;
        } else {
            p.map[page] = -1;
        }
        if (page == 0) {
            p.used[0] = total;
            p.moves[0] = total - below;
        }
    });
}

__global__ void __launch_bounds__(kThreads)
compact_kernel(const CompactParams p) {
    const int pairs = p.moves[0], total = p.used[0], P = p.pool.page_size;
    for (int i = blockIdx.x * kThreads + threadIdx.x; i < pairs; i += gridDim.x * kThreads) p.map[p.src[i]] = p.dst[i];
    // the table: a group of lanes per page, which read its first slot before they write any
    int group = 1;
    while (group < 32 && group * 2 <= P) group *= 2;
    const int lane = threadIdx.x & 31, sub = lane / group, in = lane % group, per_warp = 32 / group;
    const Table& t = p.held.table;
    for (int i = 0; i < p.held.count; ++i) {
        const int r = p.held.rows[i];
        if (r < 0 || r >= t.rows) continue;
        const int64_t len = min(static_cast<int64_t>(max(p.held.lens[i], 0)), t.cols);
        const int pages = static_cast<int>((len + P - 1) / P);
        const int warps = gridDim.x * (kThreads / 32);
        for (int base = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * per_warp; base < pages; base += warps * per_warp) {
            const int j = base + sub;
            const int64_t at = static_cast<int64_t>(j) * P;
            const int slot = j < pages ? t.slots[r * t.stride + at] : -1;
            __syncwarp();
            const int g = slot / P;
            if (slot < 0 || g >= p.pool.num_pages || slot % P != 0) continue;
            const int to = g < total ? g : p.dst[p.rank[g]];
            for (int k = in; k < P && at + k < t.cols; k += group) p.out[r * p.out_stride + at + k] = to * P + k;
        }
    }
    move_pages(p.pool, p.src, p.dst, nullptr, pairs);
}

// ---- workspace and checks ------------------------------------------------------------------------------------------

struct Layout {
    int words;                       // of a bit per page
    int64_t bits, ints, bytes;       // two arrays of bits, then three of an int per page, then a counter
};
Layout layout_of(int num_pages) {
    Layout x;
    x.words = div_ceil(num_pages, 32);
    x.bits = div_ceil64(static_cast<int64_t>(x.words) * 4, 256) * 256;
    x.ints = div_ceil64(static_cast<int64_t>(num_pages) * 4, 256) * 256;
    x.bytes = 2 * x.bits + 3 * x.ints + 256 + 256;
    return x;
}
uint8_t* aligned(void* workspace) {
    return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255));
}

int check_pool(const b200_page_pool* pool, const char* name, Pool* out) {
    B200_CHECK_ARG(pool != nullptr, "%s: NULL pool", name);
    B200_CHECK_ARG(pool->page_size >= 1 && pool->num_pages >= 1 && static_cast<int64_t>(pool->page_size) * pool->num_pages <= 0x7fffffff,
                   "%s: page_size and num_pages must be positive, of fewer than 2^31 slots", name);
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
    B200_CHECK_ARG(p.count >= 0 && p.held_count >= 0, "%s: count and held_count must not be negative", name);
    B200_CHECK_ARG(p.count == 0 || (p.rows && p.lens && (p.table.slots || p.table.rows * p.table.cols == 0)), "%s: NULL tensor", name);
    B200_CHECK_ARG(p.held_count == 0 || p.held, "%s: NULL tensor", name);
    return B200_OK;
}

// The pages held, as bits (and counted).
int launch_mark(const HeldParams& p, uint32_t* bits, int64_t bits_bytes, int32_t* refs, cudaStream_t stream) {
    B200_CHECK_CUDA(cudaMemsetAsync(bits, 0, bits_bytes, stream));
    if (refs != nullptr) B200_CHECK_CUDA(cudaMemsetAsync(refs, 0, static_cast<size_t>(p.num_pages) * 4, stream));
    if (p.count == 0 && p.held_count == 0) return B200_OK;
    const int64_t most = max(div_ceil64(p.table.cols, p.page_size), static_cast<int64_t>(p.held_count));
    const int chunks = static_cast<int>(min(max(div_ceil64(most, kThreads), int64_t(1)), int64_t(64)));
    B200_CHECK_CUDA(launch_kernel(mark_pages_kernel, dim3(p.count + 1, chunks), dim3(kThreads), 0, stream, dim3(1, 1, 1), p, bits, refs));
    return B200_OK;
}

}  // namespace
}  // namespace b200

extern "C" {

int64_t b200_pages_workspace_bytes(int num_pages) {
    if (num_pages < 1) return -1;
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
    uint8_t* ws = aligned(workspace);
    int32_t* slots = reinterpret_cast<int32_t*>(ws + 2 * x.bits);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    B200_CHECK_CUDA(launch_kernel(copy_check_kernel, dim3(1), dim3(1024), 0, s, dim3(1, 1, 1), src, dst, tokens, count, p.page_size, p.num_pages,
                                  x.words, reinterpret_cast<uint32_t*>(ws), reinterpret_cast<uint32_t*>(ws + x.bits), slots, status));
    const int64_t pieces = div_ceil64(static_cast<int64_t>(p.page_size) * p.slot_bytes, kPiece);
    const int64_t blocks = div_ceil64(static_cast<int64_t>(count) * p.num_planes * pieces, kThreads / 32);
    const int grid = static_cast<int>(min(blocks, static_cast<int64_t>(sm_count()) * 8));
    B200_CHECK_CUDA(launch_kernel(copy_pages_kernel, dim3(grid), dim3(kThreads), 0, s, dim3(1, 1, 1), p, src, dst, slots, count));
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
    const int parts = max(1, min(div_ceil(sm_count() * 8, count), 64));
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
    B200_CHECK_ARG(refs && free_pages && free_count, "count_pages: NULL tensor");
    HeldParams p{Table{page_table, table_rows, page_table_stride, table_cols}, rows, lens, held, count, held_count, page_size, num_pages, nullptr};
    int err = check_held("count_pages", p);
    if (err != B200_OK) return err;
    const Layout x = layout_of(num_pages);
    err = check_workspace("count_pages", workspace, workspace_bytes, x);
    if (err != B200_OK) return err;
    p.status = device_status_words(&err);
    if (err != B200_OK) return err;
    uint32_t* bits = reinterpret_cast<uint32_t*>(aligned(workspace));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    err = launch_mark(p, bits, x.bits, refs, s);
    if (err != B200_OK) return err;
    B200_CHECK_CUDA(launch_kernel(list_free_kernel, dim3(div_ceil(x.words, kThreads)), dim3(kThreads), 0, s, dim3(1, 1, 1), bits, x.words, num_pages,
                                  free_pages, free_count));
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
    uint8_t* ws = aligned(workspace);
    uint32_t* bits = reinterpret_cast<uint32_t*>(ws);
    p.out = table_out;
    p.out_stride = table_out_stride;
    p.map = map;
    p.used = used;
    p.src = reinterpret_cast<int32_t*>(ws + 2 * x.bits);
    p.dst = reinterpret_cast<int32_t*>(ws + 2 * x.bits + x.ints);
    p.rank = reinterpret_cast<int32_t*>(ws + 2 * x.bits + 2 * x.ints);
    p.moves = reinterpret_cast<int32_t*>(ws + 2 * x.bits + 3 * x.ints);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    err = launch_mark(p.held, bits, x.bits, nullptr, s);
    if (err != B200_OK) return err;
    B200_CHECK_CUDA(launch_kernel(plan_moves_kernel, dim3(div_ceil(x.words, kThreads)), dim3(kThreads), 0, s, dim3(1, 1, 1), bits, x.words, p));
    B200_CHECK_CUDA(launch_kernel(compact_kernel, dim3(sm_count() * 8), dim3(kThreads), 0, s, dim3(1, 1, 1), p));
    return B200_OK;
}

}  // extern "C"

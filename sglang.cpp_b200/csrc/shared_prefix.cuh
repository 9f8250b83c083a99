// Attention over a shared prefix: what its kernels have in common.
//
// Four launches: a plan (one CTA) that cuts the work into items; the tensor-core kernel over the prefixes of groups with many query
// rows; the rows kernel over everything else; and the kernel that joins a row's parts.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace b200 {

constexpr int kSharedMaxBatch = 1024;
constexpr int kSharedPieces = 4;       // items of the rows kernel per CTA, about
constexpr int kSharedTcTile = 128;     // keys of a tile of the tensor-core kernel, and query rows of one of its chains

constexpr int kSharedMany = 32;        // parts of a row that are too many for one warp, among rows of a few
constexpr int kSharedMinStages = 2;    // of an item of the rows kernel
constexpr int kSharedLongPiece = 6;    // stages of an item that covers the fetching of the next

// Stages of the rows kernel, and tiles of the tensor-core kernel, of one unit: row tiles (or blocks of rows) times what each goes over.
// 64 bits: 32768 row tiles behind 2^20 keys of 8 heads are 2^31 stages.
__host__ __device__ inline int64_t shared_unit_work(int tiles, int each) { return static_cast<int64_t>(tiles) * each; }

// Stages per item: about an item per CTA where that makes short ones (every item costs a microsecond of queries and results, and its
// parts have to be joined: 64 requests of up to 512 keys of their own 34.8 us with 2 stages, 31.4 with 6), several where they
// would be long, and no more of them than there is room for: kSharedPieces per CTA and one per row tile.  (Counts beyond 32-bit division
// are shifted: up to twice as many stages.  A row tile has no more than 2^26.)
__host__ __device__ inline int shared_stages_per_item(int64_t stages, int ctas) {
    const int many = kSharedPieces * ctas;
    if (stages > 0x40000000) {
        int shift = 0;
        while (2 << shift <= many) ++shift;
        const int64_t n = (stages >> shift) + 1;
        return n < (1 << 26) ? static_cast<int>(n) : 1 << 26;
    }
    const int all = static_cast<int>(stages), least = (all + many - 1) / many, one = (all + ctas - 1) / ctas;
    const int n = one < kSharedLongPiece ? one : kSharedLongPiece;
    const int piece = least > n ? least : n;
    return piece > kSharedMinStages ? piece : kSharedMinStages;
}

// Units are the groups' prefixes (0 .. groups) and the requests' own keys (groups .. groups + batch).

// What a CTA of the rows kernel does in one go: stages [s_begin, s_end) of a unit's keys for a tile of its rows.
struct __align__(16) RowsItem {
    int tok0, ntok;    // query tokens of the unit
    int lo, hi;        // its keys [lo, hi) ...
    int start;         // ... read from here: where lo's page copy begins
    int limit0;        // token i sees keys up to limit0 + i
    int table;         // page-table row
    int tile;          // row tile
    int s_begin, s_end;
    int reread;        // other row tiles read the same keys
    int slot;          // of its partial results; -1: there are no more items
};

// ... and of the tensor-core kernel: tiles [t0, t1) of a prefix for a block of rows.
struct __align__(16) TcItem {
    int h;             // KV head
    int tok0, ntok;    // query tokens of the block
    int keys;          // of the prefix
    int t0, t1;
    int table;
    int pad;
};

// Where the parts of a token's rows are.  A row tile has `pieces` parts one behind the other in the rows kernel's slots; in the
// tensor-core kernel's a unit's parts lie at unit + CTA.
struct __align__(16) JoinItem {
    int owned;                                        // 0: by no request, nothing is written
    int own_t, own_first, own_pieces;                 // its place among the request's tokens, the request's own keys
    int pre_t;                                        // its place among the group's tokens
    int pre_first, pre_pieces;                        // the group's prefix in the rows kernel, or ...
    int tc_unit, tc_blocks, tc_first, tc_tiles, tc_cta;   // ... in the tensor-core kernel: units before, blocks per KV head, tiles before,
                                                          // tiles per unit, first CTA
    int many;                                         // 1: more than kSharedMany parts in all
    int pad[3];
};

struct __align__(16) PlanHead {
    int fits;                     // 0: the index arrays are no such arrays; nothing is written
    int rows_items;
    int tc_per, tc_chunked;       // tensor-core kernel: tiles per CTA, in chunks of one unit or in runs
    int next;                     // rows kernel: the first item that nobody has taken yet
    int rows_lead;                // ... and how many a CTA takes ahead of the one it copies
    int rows_first;               // ... and the CTAs that begin with the item of their own number
    int many;                     // tokens whose rows have more than kSharedMany parts
};

struct SharedPlan {
    PlanHead* head;
    int2* tc_of;         // [CTAs] items of a CTA of the tensor-core kernel
    RowsItem* rows;      // [max_slots]
    TcItem* tc;          // [tc_slots], item = slot of its partial results
    JoinItem* join;      // [tokens]
    int* many;           // [tokens] those of many parts
};

struct SharedPrefixParams {
    __nv_bfloat16* out;
    const __nv_bfloat16* q;
    int64_t q_st, q_sh;
    const int32_t* page_table;
    int64_t pt_stride;
    const int32_t *table_idx, *seq_lens, *qo_indptr, *group_indptr, *prefix_lens;
    int tokens, batch, groups;
    int q_heads, kv_heads, group;   // group: query heads per KV head
    int stage_keys, kpc;            // rows kernel: keys per stage, and those that lie together in it (a copy's, with its pages)
    int small, align;               // ... whether pages are too small for copies of them; keys are read from a multiple of this
    int tile_rows, row_tokens;      // ... rows of a row tile, and the query tokens whose heads fill it: tile_rows / group
    const __nv_bfloat16 *k_cache, *v_cache;
    int64_t num_slots;
    float scale_log2;
    float *ws_ml, *ws_o;            // partial rows, (maximum, sum) and x 128: the rows kernel's [max_slots, key groups, kv_heads, row tile],
    int64_t tc_base;                // from here on the tensor-core kernel's [tc_slots, 2 chains, 128]
    int max_slots, tc_slots;
    int tc_rows;                    // groups of more query rows (tokens x group) than this: their prefixes by the tensor-core kernel
    int with_tc;                    // is that kernel launched at all?
    int ctas;                       // of either kernel
    int parts;                      // of a stage in the rows kernel: warps that share the keys of a KV head
    SharedPlan plan;
    int* status;
};

// Half rows (64 elements) of the queries [tokens][heads][128]: `heads` heads of `tokens` tokens per copy.
int make_shared_query_tmap(CUtensorMap* out, const SharedPrefixParams& p, int heads, int tokens);
int launch_shared_prefix_plan(const SharedPrefixParams& p, cudaStream_t stream);
int launch_shared_prefix_tc(const SharedPrefixParams& p, const void* k_cache, const void* v_cache, int page_size, cudaStream_t stream);

}  // namespace b200

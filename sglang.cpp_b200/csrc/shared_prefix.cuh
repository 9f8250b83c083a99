// Attention over a shared prefix: what its kernels have in common.
//
// Four launches: a plan (one CTA) that cuts the work into items; the tensor-core kernel over the prefixes of groups with many query
// rows; the rows kernel over everything else; and the kernel that joins a row's parts.
#pragma once

#include "common.cuh"

namespace b200 {

constexpr int kSharedMaxBatch = 1024;
constexpr int kSharedRowTile = 16;     // query rows of a tile of the rows kernel
constexpr int kSharedTcTile = 128;     // keys of a tile of the tensor-core kernel, and query rows of one of its chains

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
    int pad;
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

// Where the parts of a request's rows are.  A row tile's stages (a unit's key tiles) are spread over neighbouring CTAs, and parts lie
// at tile + CTA (unit + CTA).
struct __align__(16) JoinItem {
    int row0, row1;                      // query rows
    int own_tile, own_tiles, own_first, own_stages;   // tiles before, tiles, stages before, stages per tile
    int pre_row0;                        // first query row of the group
    int pre_tile, pre_tiles, pre_first, pre_stages;   // the group's prefix in the rows kernel, or ...
    int tc_unit, tc_blocks, tc_first, tc_tiles, tc_cta;   // ... in the tensor-core kernel: units before, blocks per KV head, tiles before,
                                                          // tiles per unit, first CTA
};

struct __align__(16) PlanHead {
    int fits;                     // 0: index arrays ask for more room than the host has counted; nothing is written
    int early, early_stages, late_stages;   // rows kernel: stages of each of the first `early` CTAs, and of each of the others
    int tc_per, tc_chunked;       // tensor-core kernel: tiles per CTA, in chunks of one unit or in runs
    int pad[2];
};

struct SharedPlan {
    PlanHead* head;
    int2* rows_of;       // [CTAs] items of a CTA of the rows kernel
    int2* tc_of;         // [CTAs] ... of the tensor-core kernel
    RowsItem* rows;      // [max_slots], item = slot of its partial results
    TcItem* tc;          // [tc_slots]
    JoinItem* join;      // [batch]
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
    int stage_keys, kpc;            // rows kernel: keys per stage and per copy
    int64_t num_slots;
    float scale_log2;
    float *ws_ml, *ws_o;            // partial rows, (maximum, sum) and x 128: the rows kernel's [max_slots, key groups, kv_heads, row tile],
    int64_t tc_base;                // from here on the tensor-core kernel's [tc_slots, 2 chains, 128]
    int max_slots, tc_slots;
    int tc_rows;                    // groups of more query rows (tokens x group) than this: their prefixes by the tensor-core kernel
    int with_tc;                    // is that kernel launched at all?
    int ctas;                       // of either kernel
    SharedPlan plan;
    int* status;
};

int launch_shared_prefix_plan(const SharedPrefixParams& p, cudaStream_t stream);
int launch_shared_prefix_tc(const SharedPrefixParams& p, const void* k_cache, const void* v_cache, int page_size, cudaStream_t stream);

}  // namespace b200

// Attention over a shared prefix: what its kernels have in common (parameters, and how the work is laid out on the device).
#pragma once

#include "common.cuh"

namespace b200 {

constexpr int kSharedMaxBatch = 1024;

// What a call leaves in the workspace for the kernel that joins the parts.  Units are the groups' prefixes (0 .. groups), then
// the requests' own keys; `stage` and `tile` count the stages and row tiles of the units before.
struct SharedPlan {
    int* per;        // stages per CTA of the rows kernel; tiles per CTA of the tensor-core kernel, and whether in chunks
    int* stage;      // [groups + batch + 1]
    int* tile;       // [groups + batch + 1]
    int* prefix;     // [groups] keys that are read once for the group
    int* group_of;   // [batch], -1: none
    int *tc_first, *tc_unit;   // [groups + 1] tiles and units of the groups before, in the tensor-core kernel
    int* tc_cta;     // [groups] the CTA of a group's first chunk there
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
    float *ws_ml, *ws_o;            // rows kernel: [max_slots, key groups, kv_heads, row tile] (maximum, sum), and x 128
    int max_slots;
    int tc_rows;                    // groups of more rows (tokens x group) than this: their prefixes by the tensor-core kernel
    int tc_slots;
    int64_t tc_base;                // its partial rows in ws_ml and ws_o: [tc_slots, 256] from here
    bool after_tc;                  // the rows kernel follows the tensor-core kernel
    SharedPlan plan;
    int* status;
};

#ifdef __CUDACC__
// Query rows of the requests before b; bounds hold whatever the array says.
__device__ __forceinline__ int shared_row(const SharedPrefixParams& p, int b) { return min(max(p.qo_indptr[b], 0), p.tokens); }
__device__ __forceinline__ int shared_len(const SharedPrefixParams& p, int b) {
    return static_cast<int>(min(static_cast<int64_t>(max(p.seq_lens[b], 0)), p.pt_stride));
}
__device__ __forceinline__ int shared_bound(const SharedPrefixParams& p, int g) { return min(max(p.group_indptr[g], 0), p.batch); }

// The group that request b belongs to, -1 for none (s_bound: shared_bound of 0 .. groups).
__device__ __forceinline__ int shared_group_of(const int* s_bound, int groups, int b) {
    if (groups == 0 || b < s_bound[0] || b >= s_bound[groups]) return -1;
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_bound[mid] <= b) lo = mid; else hi = mid;
    }
    return lo;
}

// The keys that are read once for a group: those that its caller names, as far as they lie before every query row of its requests;
// none for a request that shares with nobody.  All threads of a block; ends with a barrier.
__device__ __forceinline__ void shared_prefixes(const SharedPrefixParams& p, int* s_bound, int* s_prefix) {
    const int nt = static_cast<int>(blockDim.x);
    for (int g = threadIdx.x; g <= p.groups; g += nt) s_bound[g] = p.groups > 0 ? shared_bound(p, g) : 0;
    for (int g = threadIdx.x; g < p.groups; g += nt)
        s_prefix[g] = shared_bound(p, g + 1) - shared_bound(p, g) > 1 ? max(p.prefix_lens[g], 0) : 0;
    __syncthreads();
    for (int b = threadIdx.x; b < p.batch; b += nt) {
        const int rows = shared_row(p, b + 1) - shared_row(p, b);
        const int g = shared_group_of(s_bound, p.groups, b);
        if (g >= 0 && rows > 0) atomicMin(&s_prefix[g], max(shared_len(p, b) - rows, 0));
    }
    __syncthreads();
}
#endif

int launch_shared_prefix_tc(const SharedPrefixParams& p, const void* k_cache, const void* v_cache, int page_size, cudaStream_t stream);

}  // namespace b200

// Causal attention over whole prompts that lie behind one another, without a cache.
//
// For row i of a sequence, head h and its key / value head g = h / (q_heads / kv_heads):
//   s_j = scale q_i . k_j  (j <= i),  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum_j exp(s_j - m).
#include "common.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int kMaxDim = 128, kMaxBatch = 1024, kMaxGroup = 128;

struct PromptParams {
    __nv_bfloat16* out;
    float* lse;
    const __nv_bfloat16 *q, *k, *v;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
    const int32_t* indptr;
    int tokens, batch, q_heads, kv_heads, dim;
    float scale_log2;
    int* status;
};

// One warp per row and head; a lane holds four elements of the head dimension.
__global__ void __launch_bounds__(256)
prompt_attention_kernel(const PromptParams p) {
    bool odd = false;
    for (int i = threadIdx.x; i < p.batch; i += 256)
        odd = odd || p.indptr[i] < 0 || p.indptr[i + 1] < p.indptr[i] || p.indptr[i + 1] > p.tokens;
    if (__syncthreads_or(odd)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicExch(&p.status[kStatusBadIndex], bad_index_word(p.tokens));
        return;
    }
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int row = static_cast<int>(item / p.q_heads), h = static_cast<int>(item % p.q_heads), g = h / (p.q_heads / p.kv_heads);
    if (row >= p.indptr[p.batch] || row < p.indptr[0]) return;
    int lo = 0, hi = p.batch;                     // the sequence: indptr[lo] <= row < indptr[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.indptr[mid] <= row) lo = mid; else hi = mid;
    }
    const int first = p.indptr[lo], at = lane * 4;
    const bool in = at < p.dim;
    auto load = [&](const __nv_bfloat16* base, float (&x)[4]) {
        const uint2 u = in ? *reinterpret_cast<const uint2*>(base + at) : make_uint2(0, 0);
        x[0] = bf16_lo(u.x);
        x[1] = bf16_hi(u.x);
        x[2] = bf16_lo(u.y);
        x[3] = bf16_hi(u.y);
    };
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, sum = 0.f;
    load(p.q + row * p.q_st + h * p.q_sh, q);
    for (int j = first; j <= row; ++j) {
        float k[4], v[4];
        load(p.k + j * p.k_st + g * p.k_sh, k);
        load(p.v + j * p.v_st + g * p.v_sh, v);
        const float s = warp_sum(q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3]) * p.scale_log2;
        const float now = fmaxf(m, s), old = exp2f(m - now), w = exp2f(s - now);
        sum = sum * old + w;
        for (int i = 0; i < 4; ++i) o[i] = o[i] * old + w * v[i];
        m = now;
    }
    if (in) {
        uint2 u;
        u.x = pack_bf16(o[0] / sum, o[1] / sum);
        u.y = pack_bf16(o[2] / sum, o[3] / sum);
        *reinterpret_cast<uint2*>(p.out + (static_cast<int64_t>(row) * p.q_heads + h) * p.dim + at) = u;
    }
    if (lane == 0 && p.lse != nullptr) p.lse[static_cast<int64_t>(row) * p.q_heads + h] = m * 0.6931471805599453f + logf(sum);
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_attention_prompt(const b200_prompt_attention_args* a, b200_stream_t stream) {
    using namespace b200;
    B200_CHECK_ARG(a != nullptr, "attention_prompt: NULL arguments");
    B200_CHECK_ARG(a->tokens >= 0 && a->batch >= 0 && a->batch <= kMaxBatch, "attention_prompt: batch must be in [0, %d], tokens not negative", kMaxBatch);
    B200_CHECK_ARG(a->head_dim >= 8 && a->head_dim <= kMaxDim && a->head_dim % 8 == 0, "attention_prompt: head_dim must be a multiple of 8 up to %d", kMaxDim);
    B200_CHECK_ARG(a->kv_heads >= 1 && a->q_heads >= 1 && a->q_heads % a->kv_heads == 0 && a->q_heads / a->kv_heads <= kMaxGroup,
                   "attention_prompt: q_heads must be a multiple of kv_heads with group size <= %d", kMaxGroup);
    const int64_t strides[6] = {a->q_stride_token, a->q_stride_head, a->k_stride_token, a->k_stride_head, a->v_stride_token, a->v_stride_head};
    for (int64_t s : strides)
        B200_CHECK_ARG(s > 0 && s % 8 == 0 && s < (1ll << 38), "attention_prompt: strides must be positive multiples of 8");
    B200_CHECK_ARG(a->sm_scale > 0.f && a->sm_scale <= 1e30f, "attention_prompt: sm_scale must be a positive number");
    B200_CHECK_ARG(static_cast<int64_t>(a->tokens) * a->q_heads <= (1 << 28), "attention_prompt: too many query rows");
    if (a->batch == 0 || a->tokens == 0) return B200_OK;
    B200_CHECK_ARG(a->out && a->q && a->k && a->v && a->indptr, "attention_prompt: NULL tensor");
    for (const void* t : {static_cast<const void*>(a->out), a->q, a->k, a->v})
        B200_CHECK_ARG(reinterpret_cast<uintptr_t>(t) % 16 == 0, "attention_prompt: out, q, k and v must be 16-byte aligned");
    int err = B200_OK;
    PromptParams p;
    p.status = device_status_words(&err);
    if (err != B200_OK) return err;
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.lse = a->lse;
    p.q = static_cast<const __nv_bfloat16*>(a->q);
    p.k = static_cast<const __nv_bfloat16*>(a->k);
    p.v = static_cast<const __nv_bfloat16*>(a->v);
    p.q_st = a->q_stride_token;
    p.q_sh = a->q_stride_head;
    p.k_st = a->k_stride_token;
    p.k_sh = a->k_stride_head;
    p.v_st = a->v_stride_token;
    p.v_sh = a->v_stride_head;
    p.indptr = a->indptr;
    p.tokens = a->tokens;
    p.batch = a->batch;
    p.q_heads = a->q_heads;
    p.kv_heads = a->kv_heads;
    p.dim = a->head_dim;
    p.scale_log2 = a->sm_scale * 1.4426950408889634f;
    const int64_t items = static_cast<int64_t>(a->tokens) * a->q_heads;
    B200_CHECK_CUDA(launch_kernel(prompt_attention_kernel, dim3(static_cast<unsigned>((items + 7) / 8)), dim3(256), 0,
                                  static_cast<cudaStream_t>(stream), dim3(1, 1, 1), p));
    return B200_OK;
}

}  // extern "C"

// C-ABI entry points of the ragged operators: argument validation and launch.
#include <math.h>

#include "rkv_common.cuh"
#include "rkv_kernels.h"
#include "rkv_ragged.h"

using namespace rkv;

namespace {

inline cudaStream_t S(void* s) { return static_cast<cudaStream_t>(s); }

inline int status_of(cudaError_t e) { return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA; }

// Pool storage [num_slots, Hkv, P, D] shared by every request.
int check_pool(const rkv_kv_layout* kv) {
    if (!kv || !kv->k || !kv->v) return RKV_ERR_INVALID_ARGUMENT;
    if (kv->dtype != RKV_F32 && kv->dtype != RKV_F16 && kv->dtype != RKV_BF16) return RKV_ERR_UNSUPPORTED;
    if (kv->head_dim < 1 || kv->head_dim > kMaxHeadDim) return RKV_ERR_UNSUPPORTED;
    if (kv->num_kv_heads < 1 || kv->num_kv_heads > 65535 || kv->page_size < 1 || kv->num_slots < 1)
        return RKV_ERR_INVALID_ARGUMENT;
    if (kv->row_map) return RKV_ERR_UNSUPPORTED;
    return RKV_OK;
}

}  // namespace

extern "C" {

int rkv_ragged_page_tables(const int64_t* lengths, const int64_t* new_lengths, int64_t requests,
                           int64_t page_size, int64_t* page_table, int64_t pt_stride,
                           int64_t pt_width, int64_t* ring, int64_t ring_size, int64_t* state,
                           int64_t* out_lengths, int64_t* out_state, int64_t* slot_map,
                           int64_t* positions, int64_t max_new_tokens, int64_t* token_starts,
                           void* stream) {
    if (requests < 0 || page_size < 1 || pt_width < 0 || pt_stride < pt_width || ring_size < 1 ||
        max_new_tokens < 0)
        return RKV_ERR_INVALID_ARGUMENT;
    // page_size * pt_width is a token count, page_size * ring_size a slot id
    if (pt_width > INT64_MAX / page_size || ring_size > INT64_MAX / page_size)
        return RKV_ERR_INVALID_ARGUMENT;
    // and so is the sum of it over all requests
    if (requests > 0 && pt_width * page_size > INT64_MAX / requests) return RKV_ERR_INVALID_ARGUMENT;
    if (!ring || !state || !out_state || !token_starts) return RKV_ERR_INVALID_ARGUMENT;
    if (requests > 0 && (!lengths || !new_lengths || !out_lengths)) return RKV_ERR_INVALID_ARGUMENT;
    if (requests > 0 && pt_width > 0 && !page_table) return RKV_ERR_INVALID_ARGUMENT;
    if (max_new_tokens > 0 && (!slot_map || !positions)) return RKV_ERR_INVALID_ARGUMENT;
    ragged::TableParams p{lengths, new_lengths, requests, page_size, page_table, pt_stride, pt_width,
                          ring, ring_size, state, out_lengths, out_state, slot_map, positions,
                          max_new_tokens, token_starts, 0, 0, ragged::FastDiv()};
    p.in_place = out_lengths == lengths || out_lengths == new_lengths || out_state == state;
    p.narrow = pt_width * page_size < (1ll << 31);
    if (p.narrow) p.div_p = ragged::FastDiv((uint32_t)(page_size < (1ll << 31) ? page_size : 1));
    return status_of(ragged::launch_tables(p, S(stream)));
}

int rkv_ragged_append(const rkv_kv_layout* pool, const void* k_new, const void* v_new,
                      int64_t new_stride_t, int64_t new_stride_h, int64_t n_new,
                      const int64_t* slot_map, void* stream) {
    const int st = check_pool(pool);
    if (st) return st;
    if (n_new < 0) return RKV_ERR_INVALID_ARGUMENT;
    if (n_new == 0) return RKV_OK;
    if (!k_new || !v_new || !slot_map) return RKV_ERR_INVALID_ARGUMENT;
    ragged::AppendParams p{const_cast<void*>(pool->k), const_cast<void*>(pool->v), pool->stride_h,
                           pool->stride_p, pool->stride_t, pool->page_size, pool->num_slots,
                           k_new, v_new, new_stride_t, new_stride_h, n_new, slot_map,
                           (int)pool->num_kv_heads, pool->head_dim, pool->dtype,
                           pool->page_size < (1ll << 31), ragged::FastDiv()};
    if (p.narrow) p.div_p = ragged::FastDiv((uint32_t)pool->page_size);
    return status_of(ragged::launch_append(p, S(stream)));
}

size_t rkv_ragged_decode_attention_workspace_size(const rkv_query* q, const rkv_kv_layout* pool) {
    if (!q || !pool || pool->num_kv_heads < 1 || pool->batch < 0 || pool->head_dim < 1 ||
        pool->head_dim > kMaxHeadDim || q->num_heads < 1 || q->num_heads % pool->num_kv_heads)
        return 0;
    return RKV_WORKSPACE_HEADER_BYTES +
           ragged::decode_workspace_bytes(q->num_heads, pool->num_kv_heads, pool->head_dim);
}

int rkv_ragged_decode_attention(const rkv_query* q, const rkv_kv_layout* pool,
                                const int64_t* lengths, const int64_t* starts, float scale,
                                const rkv_output* out, float* lse, void* workspace,
                                size_t workspace_bytes, void* stream) {
    const int st = check_pool(pool);
    if (st) return st;
    if (!q || !q->q || !out || !out->out) return RKV_ERR_INVALID_ARGUMENT;
    if (q->q_len != 1 || q->dtype != pool->dtype || out->dtype != pool->dtype) return RKV_ERR_UNSUPPORTED;
    if (q->num_heads < 1 || q->num_heads % pool->num_kv_heads) return RKV_ERR_INVALID_ARGUMENT;
    if (pool->batch < 0 || pool->num_tokens < 0 || pool->num_tokens % pool->page_size)
        return RKV_ERR_INVALID_ARGUMENT;
    if (!(scale >= 0.f) || isinf(scale * 1.44269504f)) return RKV_ERR_INVALID_ARGUMENT;    // (log2 e)
    if (pool->batch == 0) return RKV_OK;
    if (!lengths || (pool->num_tokens > 0 && !pool->page_table)) return RKV_ERR_INVALID_ARGUMENT;
    if (pool->batch * q->num_heads > 0x7fffffff) return RKV_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < rkv_ragged_decode_attention_workspace_size(q, pool))
        return RKV_ERR_WORKSPACE_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return RKV_ERR_ALIGNMENT;
    ragged::DecodeParams p{};
    p.q = q->q; p.q_stride_b = q->stride_b; p.q_stride_h = q->stride_h;
    p.k = pool->k; p.v = pool->v;
    p.stride_h = pool->stride_h; p.stride_p = pool->stride_p; p.stride_t = pool->stride_t;
    p.P = pool->page_size; p.num_slots = pool->num_slots;
    p.table = pool->page_table; p.table_stride = pool->pt_stride_b;
    p.W = pool->num_tokens / pool->page_size;
    p.lengths = lengths; p.starts = starts;
    p.B = (int)pool->batch; p.Hq = q->num_heads; p.Hkv = (int)pool->num_kv_heads;
    p.D = pool->head_dim; p.dtype = pool->dtype;
    p.scale = scale > 0.f ? scale : (float)(1.0 / sqrt((double)pool->head_dim));
    p.out = out->out; p.o_stride_b = out->stride_b; p.o_stride_h = out->stride_h; p.lse = lse;
    // (the header is not used, and left as it is: other calls may share the workspace)
    p.ws = static_cast<char*>(workspace) + RKV_WORKSPACE_HEADER_BYTES;
    if (p.P < (1ll << 31)) p.div_p = ragged::FastDiv((uint32_t)p.P);
    return status_of(ragged::launch_decode(p, S(stream)));
}

int rkv_ragged_stream_error(int clear, int* code, void* stream) {
    if (!code) return RKV_ERR_INVALID_ARGUMENT;
    *code = 0;
    int a = 0, b = 0;
    if (ragged::read_table_error(clear, &a, S(stream)) != cudaSuccess ||
        ragged::read_decode_error(clear, &b, S(stream)) != cudaSuccess)
        return RKV_ERR_CUDA;
    *code = a > b ? a : b;
    return RKV_OK;
}

int rkv_ragged_error(int clear, int* code) {
    if (!code) return RKV_ERR_INVALID_ARGUMENT;
    *code = 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return RKV_ERR_CUDA;
    return rkv_ragged_stream_error(clear, code, nullptr);
}

}  // extern "C"

// Host-side interface of paged.hip / paged_attn.hip (internal): the operators over a caller's paged KV cache.
#pragma once
#include "ptts_common.h"

// the text behind ptts_last_error(); returns `code` (engine.hip)
int ptts_set_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// bits of the caller's status word (PTTS_PAGED_* of the C ABI)
enum { PAGED_BAD_POSITION = 1, PAGED_BAD_PAGE = 2, PAGED_BAD_LENGTH = 4, PAGED_BAD_STARTS = 8 };

struct PagedBatchArgs {
    const int* table;        // [n_seqs][table_stride] page ids
    int64_t table_stride;
    const int* past;         // [n_seqs] tokens cached before the call
    const int* starts;       // [n_seqs + 1] first token of every sequence, or null: token t belongs to sequence t
    int max_pages, n_pages, page_shift, n_seqs, tokens;
};

#if defined(__HIPCC__)
// starts must ascend within [0, tokens]; one workgroup of a launch looks at all of them
__device__ inline void check_starts(const int* starts, int n_seqs, int tokens, int* status) {
    for (int i = threadIdx.x; i < n_seqs; i += blockDim.x)
        if (starts[i] < 0 || starts[i] > starts[i + 1] || starts[i + 1] > tokens) atomicOr(status, PAGED_BAD_STARTS);
}
#endif

struct RotaryArgs {
    const float *cos_t, *sin_t;   // [positions][dims / 2]
    int positions, dims, interleaved;
};

struct RotaryEmbedArgs {
    const void* x;
    void* out;
    int64_t xs[2], os[2];    // token, head strides (elements)
    const int* pos;          // [tokens]
    RotaryArgs rot;
    int* status;
    int tokens, heads, head_dim;
};

struct AppendArgs {
    const void *q, *k, *v;                   // v null: it is in the cache already
    void *q_out, *k_cache, *v_cache;
    int64_t qs[2], qos[2], ks[2], vs[2];     // token, head
    int64_t kc[3], vc[3];                    // page, head, slot
    PagedBatchArgs b;
    RotaryArgs rot;                          // cos_t null: no rotation
    const int* pos;                          // [tokens] or null: the position is the slot
    int* status;
    int q_heads, kv_heads, head_dim;         // q_heads 0: no q
};

// x / d for 0 <= x < 2^31: the high half of 2 x times m = ceil(2^(31 + s) / d), s = ceil(log2 d), shifted by s
struct IntDiv { uint32_t m, s; };
inline IntDiv make_int_div(uint32_t d) {
    IntDiv r = {0, 0};
    while (((uint64_t)1 << r.s) < d) ++r.s;
    r.m = (uint32_t)((((uint64_t)1 << (31 + r.s)) + d - 1) / d);
    return r;
}
#if defined(__HIPCC__)
__device__ __forceinline__ int int_div(int x, IntDiv d) { return (int)(__umulhi(2u * (uint32_t)x, d.m) >> d.s); }
#endif

struct PagedAttnArgs {
    const void *q, *k, *v;
    void* out;
    const int* table;
    const int* past;
    const int* starts;
    const uint8_t* mask;     // [n_seqs][mask_stride], keys < mask_width with 0 are no keys; null: none
    int* status;
    float* part;             // partial results of a split launch: [split][row][D + 2]
    int* sched;              // what a launch in front left of many sequences, or null
    int64_t qs[2], os[2], kc[3], vc[3];
    int64_t table_stride, mask_stride;
    float scale_log2;        // softmax scale * log2(e)
    int max_pages, n_pages, page_shift, n_seqs, tokens, mask_width, causal;
    int q_heads, kv_heads, group;
    int splits, min_share;   // most shares of a tile's keys; least keys of one
    IntDiv by_group, by_kv_heads;
};

hipError_t rotary_embed_launch(const RotaryEmbedArgs& a, int dtype, hipStream_t s);
hipError_t kv_append_launch(const AppendArgs& a, int in_dtype, int cache_dtype, hipStream_t s);
// rows of one sequence never exceed max_new * group; the choice of kernel and split follows from it and from max_pages
int64_t paged_attn_workspace(const PagedAttnArgs& a, int max_new, int head_dim, int dtype);
hipError_t paged_attn_launch(const PagedAttnArgs& a, int max_new, int head_dim, int dtype, hipStream_t s);

// the engine's own long prefill through these operators (long_prefill.hip): npos positions from pos0 on of B utterances
struct LongPrefillArgs {
    float* q;                // [B * npos][ldq] fp32, scaled; rotary variant: q | k, unturned
    KVPool pool;
    const float* bias;       // additive mask [B][ld_bias] (0 / finfo.min) or null
    void* ofrag;             // B fragments, feature count D
    const float *cos_t, *sin_t;   // rotary variant: [positions][32]; null: k is in the cache
    int ldq, layer, ld_bias, D, H, B, npos, pos0, positions;
};
int64_t long_prefill_workspace(const LongPrefillArgs& a, int dtype);
hipError_t long_prefill_launch(const LongPrefillArgs& a, int dtype, void* workspace, int64_t workspace_bytes, hipStream_t s);

// Causal self-attention of a prefill chunk whose context is longer than attn_causal_kernel's score rows (5120 positions), through the
// operators over a paged cache: the engine's pool is one of their caches (64-token pages, page / head / slot strides), its utterances are
// the sequences of a batch of equal chunks.  Also the only route on which a chunk's keys pass matrix instructions once per 128 queries
// instead of once per query.
//   * rotary variant: kv_append turns q and k in one launch and stores k (v is in the cache already, from the projection's epilogue)
//   * queries leave the projection as fp32 rows, scaled by hd^-0.5.  A bf16 cache takes them rounded to bf16 (2^-8 of a score, as the
//     keys they meet are rounded); an fp32 cache takes them as they are.
//   * the additive mask (0 or finfo.min per key) becomes a key mask; a row of padding that sees no key comes out as zeros
//   * rows leave as MFMA fragments for the out_proj GEMM
// The status word is the operators', and nobody reads it: page ids are checked where a table is set, lengths and starts are made here, and
// prompt and generated positions together never exceed the rotary table's, so that no bit of it can be set.
#include "attn.h"
#include "paged.h"

namespace {

struct Layout {                 // byte offsets into the workspace
    int64_t table, past, starts, mask, q, out, part, bytes;
    int pages;                  // of an utterance's context
};

Layout layout_of(const LongPrefillArgs& a, int dtype) {
    Layout l;
    const int64_t rows = (int64_t)a.B * a.npos, esz = dtype == PTTS_BF16 ? 2 : 4;
    int64_t at = 256;           // the status word
    auto take = [&](int64_t bytes) { const int64_t p = at; at += (bytes + 255) / 256 * 256; return p; };
    l.pages = (a.pos0 + a.npos + PTTS_PAGE_TOKENS - 1) / PTTS_PAGE_TOKENS;
    l.table = take((int64_t)a.B * l.pages * 4);
    l.past = take((int64_t)a.B * 4);
    l.starts = take(((int64_t)a.B + 1) * 4);
    l.mask = take((int64_t)a.B * l.pages * PTTS_PAGE_TOKENS);
    l.q = take(dtype == PTTS_BF16 ? rows * a.H * PTTS_HEAD_DIM * 2 : 0);
    l.out = take(rows * a.H * PTTS_HEAD_DIM * esz);
    l.part = at;
    l.bytes = at;
    return l;
}

// one block per utterance: its row of the page table, its lengths, its mask
__global__ __launch_bounds__(256) void long_prefill_batch_kernel(LongPrefillArgs a, int pages, int* status, int* table, int* past, int* starts,
                                                                 uint8_t* mask) {
    const int b = blockIdx.x;
    if (threadIdx.x == 0) {
        past[b] = a.pos0;
        starts[b] = b * a.npos;
        if (b == a.B - 1) starts[a.B] = a.B * a.npos;
        if (b == 0) *status = 0;
    }
    for (int i = threadIdx.x; i < pages; i += 256)
        table[b * pages + i] = a.pool.block_table ? a.pool.block_table[(size_t)b * a.pool.max_blocks + i] : b * a.pool.max_blocks + i;
    if (a.bias)
        for (int i = threadIdx.x; i < a.pos0 + a.npos; i += 256) mask[(size_t)b * pages * PTTS_PAGE_TOKENS + i] = a.bias[(size_t)b * a.ld_bias + i] > -1.f;
}

// four features a thread
__global__ __launch_bounds__(256) void long_prefill_round_kernel(const float* q, int ldq, int D, int rows, uint16_t* out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / (D / 4), c = i % (D / 4) * 4;
    if (row >= rows) return;
    const float4 x = *reinterpret_cast<const float4*>(q + row * ldq + c);
    uint2 y;
    y.x = (uint32_t)to_elem<PBF16>(x.x) | (uint32_t)to_elem<PBF16>(x.y) << 16;
    y.y = (uint32_t)to_elem<PBF16>(x.z) | (uint32_t)to_elem<PBF16>(x.w) << 16;
    *reinterpret_cast<uint2*>(out + row * D + c) = y;
}

// eight features a thread: a 16-byte piece of a bf16 fragment, eight words of fp32 ones
template <typename P>
__global__ __launch_bounds__(256) void long_prefill_frag_kernel(const typename P::elem_t* rows, int D, int n, typename P::elem_t* frag) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / (D / 8);
    const int c = (int)(i % (D / 8)) * 8;
    if (row >= n) return;
    typename P::elem_t* to = frag + (row >> 5) * 32 * D;
#pragma unroll
    for (int j = 0; j < 8; ++j) to[frag_off<P>((int)row & 31, c + j)] = rows[row * D + c + j];
}

PagedAttnArgs attention_args(const LongPrefillArgs& a, const Layout& l, char* ws, int dtype) {
    PagedAttnArgs g = {};
    const int64_t esz = dtype == PTTS_BF16 ? 2 : 4, rows = (int64_t)a.B * a.npos;
    char* layer = reinterpret_cast<char*>(a.pool.base) + (int64_t)a.layer * 2 * a.pool.kv_elems() * esz;
    g.k = layer;
    g.v = layer + (int64_t)a.pool.kv_elems() * esz;
    g.kc[0] = g.vc[0] = a.pool.page_elems();
    g.kc[1] = g.vc[1] = a.pool.head_elems();
    g.kc[2] = g.vc[2] = PTTS_HEAD_DIM;
    g.q = dtype == PTTS_BF16 ? static_cast<const void*>(ws + l.q) : a.q;
    g.qs[0] = dtype == PTTS_BF16 ? a.D : a.ldq;
    g.os[0] = a.D;
    g.qs[1] = g.os[1] = PTTS_HEAD_DIM;
    g.out = ws + l.out;
    g.status = reinterpret_cast<int*>(ws);
    g.table = reinterpret_cast<int*>(ws + l.table);
    g.past = reinterpret_cast<int*>(ws + l.past);
    g.starts = reinterpret_cast<int*>(ws + l.starts);
    g.table_stride = g.max_pages = l.pages;
    g.mask_stride = (int64_t)l.pages * PTTS_PAGE_TOKENS;
    if (a.bias) { g.mask = reinterpret_cast<uint8_t*>(ws + l.mask); g.mask_width = a.pos0 + a.npos; }
    g.part = reinterpret_cast<float*>(ws + l.part);
    g.scale_log2 = 1.44269504088896340736f;              // the queries are scaled already
    g.n_pages = a.pool.n_pages; g.page_shift = 6; g.n_seqs = a.B; g.tokens = (int)rows; g.causal = 1;
    g.q_heads = g.kv_heads = a.H; g.group = 1;
    return g;
}

}  // namespace

int64_t long_prefill_workspace(const LongPrefillArgs& a, int dtype) {
    const Layout l = layout_of(a, dtype);
    return l.bytes + paged_attn_workspace(attention_args(a, l, nullptr, dtype), a.npos, PTTS_HEAD_DIM, dtype);
}

hipError_t long_prefill_launch(const LongPrefillArgs& a, int dtype, void* workspace, int64_t workspace_bytes, hipStream_t s) {
    if (a.npos <= 0 || a.B <= 0 || a.D != a.H * PTTS_HEAD_DIM || workspace_bytes < long_prefill_workspace(a, dtype)) return hipErrorInvalidValue;
    const Layout l = layout_of(a, dtype);
    char* ws = static_cast<char*>(workspace);
    const PagedAttnArgs g = attention_args(a, l, ws, dtype);
    const int rows = g.tokens;
    hipLaunchKernelGGL(long_prefill_batch_kernel, dim3(a.B), dim3(256), 0, s, a, l.pages, g.status, const_cast<int*>(g.table), const_cast<int*>(g.past),
                       const_cast<int*>(g.starts), reinterpret_cast<uint8_t*>(ws + l.mask));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.cos_t) {
        AppendArgs p = {};
        p.q = p.q_out = a.q;
        p.k = a.q + a.D;
        p.k_cache = const_cast<void*>(g.k); p.v_cache = const_cast<void*>(g.v);
        p.qs[0] = p.qos[0] = p.ks[0] = a.ldq;
        p.qs[1] = p.qos[1] = p.ks[1] = PTTS_HEAD_DIM;
        for (int i = 0; i < 3; ++i) p.kc[i] = p.vc[i] = g.kc[i];
        p.b = PagedBatchArgs{g.table, g.table_stride, g.past, g.starts, g.max_pages, g.n_pages, g.page_shift, g.n_seqs, g.tokens};
        p.rot = RotaryArgs{a.cos_t, a.sin_t, a.positions, PTTS_HEAD_DIM, 0};
        p.status = g.status;
        p.q_heads = p.kv_heads = a.H; p.head_dim = PTTS_HEAD_DIM;
        e = kv_append_launch(p, PTTS_F32, dtype, s);
        if (e != hipSuccess) return e;
    }
    if (dtype == PTTS_BF16) {
        const int64_t n = (int64_t)rows * (a.D / 4);
        hipLaunchKernelGGL(long_prefill_round_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, a.q, a.ldq, a.D, rows, reinterpret_cast<uint16_t*>(ws + l.q));
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    e = paged_attn_launch(g, a.npos, PTTS_HEAD_DIM, dtype, s);
    if (e != hipSuccess) return e;
    const int64_t n = (int64_t)rows * (a.D / 8);
    const dim3 grid((unsigned)((n + 255) / 256)), block(256);
    if (dtype == PTTS_BF16) hipLaunchKernelGGL(long_prefill_frag_kernel<PBF16>, grid, block, 0, s, reinterpret_cast<uint16_t*>(ws + l.out), a.D, rows, reinterpret_cast<uint16_t*>(a.ofrag));
    else hipLaunchKernelGGL(long_prefill_frag_kernel<PF32>, grid, block, 0, s, reinterpret_cast<float*>(ws + l.out), a.D, rows, reinterpret_cast<float*>(a.ofrag));
    return hipGetLastError();
}

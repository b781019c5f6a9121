// Rotary positions and the append of keys and values to a caller's paged cache, and the C entries of the paged operators.
//
// Rotation: the pair (a, b) of a head becomes (a cos t - b sin t, b cos t + a sin t); pairs are (i, i + r / 2) (half layout) or
// (2 i, 2 i + 1) (interleaved) of the first r features, the features behind them are copied.  cos t / sin t come from the caller's
// fp32 tables, built from 64-bit angles: an angle formed in 32 bits is off by half a unit of position * 2^-24, 4e-3 at position 131072.
// Products and sum are rounded one by one (no fma contraction), so that a row has the same bits whichever kernel or layout turns it.
#include "../../include/parler_tts_hip.h"
#include "ptts_common.h"
#include "gemm.h"
#include "paged.h"
#include <climits>
#include <cmath>
#include <initializer_list>

namespace {

template <typename T, int N> struct alignas(sizeof(T) * N) Pack { T e[N]; };

template <typename T> __device__ inline float widen(T v);
template <> __device__ inline float widen<uint16_t>(uint16_t v) { return bf16_bits_to_float(v); }
template <> __device__ inline float widen<float>(float v) { return v; }
template <typename T> __device__ inline T narrow(float v);
template <> __device__ inline uint16_t narrow<uint16_t>(float v) { return float_to_bf16_bits(v); }     // half a bf16 step: the caller's type
template <> __device__ inline float narrow<float>(float v) { return v; }

// i / d for i < 65536, 1 <= d <= 65536: m = ceil(2^32 / d) (d = 1: m = 0, the quotient is i)
struct SmallDiv { uint32_t m; };
__device__ inline int small_div(int i, SmallDiv d) { return d.m ? (int)__umulhi((uint32_t)i, d.m) : i; }

// One unit of work: N pairs of a rotated head (two runs of N elements), or 2 N elements that are copied.
template <typename T, int N> struct Unit { Pack<T, N> a, b; };

template <typename T, int N> __device__ inline void turn(Unit<T, N>& u, const float* cos_t, const float* sin_t, int interleaved) {
#pragma clang fp contract(off)
    const Pack<float, N> c = *reinterpret_cast<const Pack<float, N>*>(cos_t), s = *reinterpret_cast<const Pack<float, N>*>(sin_t);
    float x[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) { x[i] = widen<T>(u.a.e[i]); x[N + i] = widen<T>(u.b.e[i]); }
    float y[2 * N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : N + i;
        y[ia] = x[ia] * c.e[i] - x[ib] * s.e[i];
        y[ib] = x[ib] * c.e[i] + x[ia] * s.e[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) { u.a.e[i] = narrow<T>(y[i]); u.b.e[i] = narrow<T>(y[N + i]); }
}

struct UnitMap {            // where the units of one token lie
    SmallDiv per_token, per_head;
    int upt, uph, rotated;  // units per token and head; the first `rotated` units of a head turn
    int tokens_per_block;
};

template <int N> __device__ inline void unit_offsets(const RotaryArgs& r, int rotated, int c, int* oa, int* ob) {
    if (c >= rotated) { *oa = rotated * 2 * N + (c - rotated) * 2 * N; *ob = *oa + N; }
    else if (r.interleaved) { *oa = c * 2 * N; *ob = *oa + N; }
    else { *oa = c * N; *ob = r.dims / 2 + c * N; }
}

// Bound by the stream of rows (a product and a sum a feature): a thread moves two 16-byte pieces, the two runs of its pairs, in the widest
// loads that strides, alignment and the rotated width allow (else element by element: a width that is no multiple of 8 features in f32, 16 in
// bf16, makes a rotation of 41283 tokens x 24 heads of 64 take 120 us instead of 87 in f32, 99 instead of 46 in bf16, and an append of 21
// thousand 235 instead of 151, 205 instead of 88).  A workgroup takes whole tokens, so that a token's position is one address for many
// lanes and the table rows stay in the cache.  Measured: 41283 tokens x 24 heads of 64 in f32, 507 MB:
// 91 - 94 us, 5400 - 5560 GB/s (a copy of 1 GiB reaches 5060, of 256 MiB 5400); 32 tokens x 16 heads in bf16: 3.1 us on the device, 7.8 with the call.
template <typename T, int N, bool IL>
__global__ __launch_bounds__(256) void rotary_embed_kernel(RotaryEmbedArgs a, UnitMap m) {
    const int t0 = blockIdx.x * m.tokens_per_block;
    const int n = min(m.tokens_per_block, a.tokens - t0) * m.upt;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int tl = small_div(i, m.per_token), r = i - tl * m.upt, h = small_div(r, m.per_head), c = r - h * m.uph;
        const int64_t t = t0 + tl;
        const int pos = a.pos[t];
        const bool ok = (unsigned)pos < (unsigned)a.rot.positions;
        int oa, ob;
        unit_offsets<N>(a.rot, m.rotated, c, &oa, &ob);
        const T* x = reinterpret_cast<const T*>(a.x) + t * a.xs[0] + h * a.xs[1];
        T* o = reinterpret_cast<T*>(a.out) + t * a.os[0] + h * a.os[1];
        Unit<T, N> u;
        u.a = *reinterpret_cast<const Pack<T, N>*>(x + oa);
        u.b = *reinterpret_cast<const Pack<T, N>*>(x + ob);
        if (!ok) {
            u = Unit<T, N>{};
            if (r == 0) atomicOr(a.status, PAGED_BAD_POSITION);
        } else if (c < m.rotated) {
            const int64_t row = (int64_t)pos * (a.rot.dims / 2) + c * N;
            turn<T, N>(u, a.rot.cos_t + row, a.rot.sin_t + row, IL);
        }
        *reinterpret_cast<Pack<T, N>*>(o + oa) = u.a;
        *reinterpret_cast<Pack<T, N>*>(o + ob) = u.b;
    }
}

// Sequence of a token and its first token; false: the token lies behind the last sequence (or in front of the first).
__device__ inline bool find_sequence(const PagedBatchArgs& b, int t, int* seq, int* first, int* end) {
    if (!b.starts) { *seq = t; *first = t; *end = t + 1; return true; }
    int lo = 0, hi = b.n_seqs;                        // largest s with starts[s] <= t: never an empty sequence
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.starts[mid] <= t) lo = mid; else hi = mid;
    }
    *seq = lo; *first = b.starts[lo]; *end = b.starts[lo + 1];
    return t >= *first && t < *end;
}

constexpr int APPEND_TOKENS = 64;      // most tokens of one workgroup

// The rows of a block's tokens are looked up once (sequence, page, slot, position), then every thread moves units of q, k and v, as above.
// Bound by the stream of rows, behind the look-up's dependent trips (starts, length, page id: a chain of 3 us): 24 prompts of 257 to 1500
// tokens x 24 heads, 389 MB: 86 us, 4530 GB/s; a step of 32 tokens 3.3 us on the device, 11.7 with the call; a ragged batch of 24 chunks of up
// to 401 tokens x 16/8 heads of 64 10.2 us (8 of them its bytes; 11.7 profiled beside an attention).  Loads or stores past the caches: 1.3 times as long for the small batches.
template <typename T, typename TC, int N, bool IL>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, UnitMap m) {
    __shared__ int page_of[APPEND_TOKENS], slot_of[APPEND_TOKENS], pos_of[APPEND_TOKENS];   // page -1: nothing to do, -2: refused
    if (blockIdx.x == 0 && a.b.starts) check_starts(a.b.starts, a.b.n_seqs, a.b.tokens, a.status);
    const int t0 = blockIdx.x * m.tokens_per_block, nt = min(m.tokens_per_block, a.b.tokens - t0);
    if ((int)threadIdx.x < nt) {
        const int t = t0 + threadIdx.x;
        int s, first, end, page = -1, slot = 0, pos = 0;
        if (find_sequence(a.b, t, &s, &first, &end)) {
            const int past = a.b.past[s];
            const int64_t at = (int64_t)past + (t - first);
            int bad = 0;
            if (first < 0 || end > a.b.tokens) bad = PAGED_BAD_STARTS;
            else if (past < 0 || at >= ((int64_t)a.b.max_pages << a.b.page_shift)) bad = PAGED_BAD_LENGTH;
            else {
                page = a.b.table[s * a.b.table_stride + (at >> a.b.page_shift)];
                slot = (int)at & ((1 << a.b.page_shift) - 1);
                pos = a.pos ? a.pos[t] : (int)at;
                if ((unsigned)page >= (unsigned)a.b.n_pages) bad = PAGED_BAD_PAGE;
                else if (a.rot.cos_t && (unsigned)pos >= (unsigned)a.rot.positions) bad = PAGED_BAD_POSITION;
            }
            if (bad) { page = -2; atomicOr(a.status, bad); }
        }
        page_of[threadIdx.x] = page; slot_of[threadIdx.x] = slot; pos_of[threadIdx.x] = pos;
    }
    __syncthreads();
    const int n = nt * m.upt;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int tl = small_div(i, m.per_token), r = i - tl * m.upt, h = small_div(r, m.per_head), c = r - h * m.uph;
        const int64_t t = t0 + tl;
        const int page = page_of[tl];
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
        if (page == -1 || (page < 0 && !is_q)) continue;
        const int hk = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
        int oa, ob;
        unit_offsets<N>(a.rot, m.rotated, c, &oa, &ob);
        const T* x = is_q ? reinterpret_cast<const T*>(a.q) + t * a.qs[0] + h * a.qs[1]
                          : (is_v ? reinterpret_cast<const T*>(a.v) + t * a.vs[0] + hk * a.vs[1]
                                  : reinterpret_cast<const T*>(a.k) + t * a.ks[0] + hk * a.ks[1]);
        Unit<T, N> u;
        u.a = *reinterpret_cast<const Pack<T, N>*>(x + oa);
        u.b = *reinterpret_cast<const Pack<T, N>*>(x + ob);
        if (page < 0) u = Unit<T, N>{};
        if (is_q) {
            if (c < m.rotated && page >= 0) {
                const int64_t row = (int64_t)pos_of[tl] * (a.rot.dims / 2) + c * N;
                turn<T, N>(u, a.rot.cos_t + row, a.rot.sin_t + row, IL);
            }
            T* o = reinterpret_cast<T*>(a.q_out) + t * a.qos[0] + h * a.qos[1];
            *reinterpret_cast<Pack<T, N>*>(o + oa) = u.a;
            *reinterpret_cast<Pack<T, N>*>(o + ob) = u.b;
        } else {
            if (c < m.rotated && !is_v) {
                const int64_t row = (int64_t)pos_of[tl] * (a.rot.dims / 2) + c * N;
                turn<T, N>(u, a.rot.cos_t + row, a.rot.sin_t + row, IL);
            }
            const int64_t* cs = is_v ? a.vc : a.kc;
            TC* o = reinterpret_cast<TC*>(is_v ? a.v_cache : a.k_cache) + page * cs[0] + hk * cs[1] + slot_of[tl] * cs[2];
            Pack<TC, N> ya, yb;
#pragma unroll
            for (int j = 0; j < N; ++j) { ya.e[j] = narrow<TC>(widen<T>(u.a.e[j])); yb.e[j] = narrow<TC>(widen<T>(u.b.e[j])); }
            *reinterpret_cast<Pack<TC, N>*>(o + oa) = ya;
            *reinterpret_cast<Pack<TC, N>*>(o + ob) = yb;
        }
    }
}

SmallDiv make_div(int d) { return SmallDiv{d == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d)}; }

UnitMap make_map(int heads, int head_dim, int rot_dims, int n, int tokens, bool looks_up) {
    UnitMap m;
    m.uph = head_dim / (2 * n);
    m.upt = heads * m.uph;
    m.rotated = rot_dims / (2 * n);
    m.per_token = make_div(m.upt);
    m.per_head = make_div(m.uph);
    // One unit a thread; two (the nearest number of tokens) where a launch is large and a block's look-ups have to pay.  Measured, one, two and
    // four units in us: rotation of 41283 tokens x 24 heads of 64 in f32 94, 98.7, 106.5; appends of 24 prompts, 16 heads of 64: 64.4, 56.0, 59.0,
    // and of 24 chunks, 16/8 heads: 11.5, 10.2, 11.3.
    const bool two = looks_up && (int64_t)tokens * m.upt > 256 * 256;
    m.tokens_per_block = two ? (512 + m.upt / 2) / m.upt : 256 / m.upt;
    if (m.tokens_per_block < 1) m.tokens_per_block = 1;
    if (looks_up && m.tokens_per_block > APPEND_TOKENS) m.tokens_per_block = APPEND_TOKENS;
    return m;
}

// all rows of a tensor of these extents at multiples of `bytes` (the stride of a single entry addresses nothing and may be anything)
bool aligned(const void* p, const int64_t* strides, std::initializer_list<int64_t> extents, int64_t bytes, int64_t esz) {
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
    for (const int64_t n : extents) {
        if (n > 1 && *strides * esz % bytes) return false;
        ++strides;
    }
    return true;
}

}  // namespace

hipError_t rotary_embed_launch(const RotaryEmbedArgs& a, int dtype, hipStream_t s) {
    const int esz = dtype == PTTS_BF16 ? 2 : 4, full = 16 / esz;
    const bool wide = a.rot.dims % (2 * full) == 0 && a.head_dim % (2 * full) == 0 && aligned(a.x, a.xs, {a.tokens, a.heads}, 16, esz) &&
                      aligned(a.out, a.os, {a.tokens, a.heads}, 16, esz) && aligned(a.rot.cos_t, nullptr, {}, 16, 4) &&
                      aligned(a.rot.sin_t, nullptr, {}, 16, 4);
    const UnitMap m = make_map(a.heads, a.head_dim, a.rot.dims, wide ? full : 1, a.tokens, false);
    const dim3 grid((a.tokens + m.tokens_per_block - 1) / m.tokens_per_block), block(256);
#define LAUNCH(T, N)                                                                                        \
    do {                                                                                                    \
        if (a.rot.interleaved) hipLaunchKernelGGL((rotary_embed_kernel<T, N, true>), grid, block, 0, s, a, m); \
        else hipLaunchKernelGGL((rotary_embed_kernel<T, N, false>), grid, block, 0, s, a, m);               \
    } while (0)
    if (dtype == PTTS_BF16) { if (wide) LAUNCH(uint16_t, 8); else LAUNCH(uint16_t, 1); }
    else { if (wide) LAUNCH(float, 4); else LAUNCH(float, 1); }
#undef LAUNCH
    return hipGetLastError();
}

hipError_t kv_append_launch(const AppendArgs& a, int in_dtype, int cache_dtype, hipStream_t s) {
    const int esz = in_dtype == PTTS_BF16 ? 2 : 4, full = 16 / esz;
    const int csz = cache_dtype == PTTS_BF16 ? 2 : 4;
    bool wide = a.rot.dims % (2 * full) == 0 && a.head_dim % (2 * full) == 0 && aligned(a.k, a.ks, {a.b.tokens, a.kv_heads}, 16, esz) &&
                (!a.v || aligned(a.v, a.vs, {a.b.tokens, a.kv_heads}, 16, esz)) &&
                aligned(a.k_cache, a.kc, {a.b.n_pages, a.kv_heads, 1 << a.b.page_shift}, full * csz, csz) &&
                aligned(a.v_cache, a.vc, {a.b.n_pages, a.kv_heads, 1 << a.b.page_shift}, full * csz, csz);
    if (a.q_heads) wide = wide && aligned(a.q, a.qs, {a.b.tokens, a.q_heads}, 16, esz) && aligned(a.q_out, a.qos, {a.b.tokens, a.q_heads}, 16, esz);
    if (a.rot.cos_t) wide = wide && aligned(a.rot.cos_t, nullptr, {}, 16, 4) && aligned(a.rot.sin_t, nullptr, {}, 16, 4);
    const UnitMap m = make_map(a.q_heads + (a.v ? 2 : 1) * a.kv_heads, a.head_dim, a.rot.dims, wide ? full : 1, a.b.tokens, true);
    const dim3 grid((a.b.tokens + m.tokens_per_block - 1) / m.tokens_per_block), block(256);
#define LAUNCH(T, TC, N)                                                                                      \
    do {                                                                                                      \
        if (a.rot.interleaved) hipLaunchKernelGGL((kv_append_kernel<T, TC, N, true>), grid, block, 0, s, a, m); \
        else hipLaunchKernelGGL((kv_append_kernel<T, TC, N, false>), grid, block, 0, s, a, m);                \
    } while (0)
    if (in_dtype == PTTS_BF16) { if (wide) LAUNCH(uint16_t, uint16_t, 8); else LAUNCH(uint16_t, uint16_t, 1); }
    else if (cache_dtype == PTTS_BF16) { if (wide) LAUNCH(float, uint16_t, 4); else LAUNCH(float, uint16_t, 1); }
    else { if (wide) LAUNCH(float, float, 4); else LAUNCH(float, float, 1); }
#undef LAUNCH
    return hipGetLastError();
}

// ---- C entries ----------------------------------------------------------------------------------------------------------
namespace {

#define REFUSE(code, ...) return ptts_set_error(code, __VA_ARGS__)

// rows of a written tensor may not share elements: the smaller stride holds the row inside it, the larger one all rows of the smaller
bool overlaps_itself(const int64_t* st, const int64_t* n, int dims, int64_t inner) {
    bool used[3] = {false, false, false};
    int64_t span = inner;                      // elements from the first to behind the last of what has been nested so far
    for (int k = 0; k < dims; ++k) {
        int best = -1;
        for (int i = 0; i < dims; ++i)
            if (!used[i] && (best < 0 || st[i] < st[best])) best = i;
        used[best] = true;
        if (n[best] <= 1) continue;
        if (st[best] < span) return true;
        span += (n[best] - 1) * st[best];
    }
    return false;
}

bool fits(const int64_t* st, const int64_t* n, int dims) {     // offsets are formed in 64 bits; keep them far from the end
    int64_t span = 0;
    for (int i = 0; i < dims; ++i) {
        if (n[i] <= 1) continue;
        if (st[i] < 0 || st[i] > ((int64_t)1 << 44)) return false;
        span += st[i] * (n[i] - 1) / 4;
        if (span > ((int64_t)1 << 56)) return false;
    }
    return true;
}

int check_rotary(const ptts_rotary* r, int head_dim) {
    if (!r->cos_t || !r->sin_t) REFUSE(PTTS_E_INVALID, "rotary: null table");
    if (r->positions <= 0) REFUSE(PTTS_E_INVALID, "rotary: %d positions", r->positions);
    if (r->dims <= 0 || r->dims % 2 || r->dims > head_dim) REFUSE(PTTS_E_INVALID, "rotary: %d features of a head of %d", r->dims, head_dim);
    return PTTS_OK;
}

int check_kv(const ptts_paged_kv* c) {
    if (!c) REFUSE(PTTS_E_INVALID, "null cache");
    if (c->dtype != PTTS_DTYPE_F32 && c->dtype != PTTS_DTYPE_BF16) REFUSE(PTTS_E_INVALID, "cache dtype must be 0 (f32) or 1 (bf16)");
    if (!c->k || !c->v) REFUSE(PTTS_E_INVALID, "null cache tensor");
    if (c->n_pages <= 0 || c->kv_heads <= 0) REFUSE(PTTS_E_INVALID, "cache of %d pages, %d heads", c->n_pages, c->kv_heads);
    if (c->page_tokens < 16 || c->page_tokens > 4096 || (c->page_tokens & (c->page_tokens - 1)))
        REFUSE(PTTS_E_UNSUPPORTED, "pages of %d tokens: a power of two from 16 to 4096 is served", c->page_tokens);
    if (c->head_dim != 64 && c->head_dim != 128) REFUSE(PTTS_E_UNSUPPORTED, "head_dim %d: 64 and 128 are served", c->head_dim);
    const int64_t n[3] = {c->n_pages, c->kv_heads, c->page_tokens};
    if (!fits(c->k_strides, n, 3) || !fits(c->v_strides, n, 3)) REFUSE(PTTS_E_INVALID, "cache strides out of range");
    if (overlaps_itself(c->k_strides, n, 3, c->head_dim) || overlaps_itself(c->v_strides, n, 3, c->head_dim))
        REFUSE(PTTS_E_INVALID, "rows of the cache share elements");
    const int esz = c->dtype == PTTS_DTYPE_BF16 ? 2 : 4;
    if (c->k_strides[2] * esz >= ((int64_t)1 << 27) || c->v_strides[2] * esz >= ((int64_t)1 << 27))
        REFUSE(PTTS_E_UNSUPPORTED, "slots of a page 128 MiB or more apart");
    if (!aligned(c->k, c->k_strides, {n[0], n[1], n[2]}, 16, esz) || !aligned(c->v, c->v_strides, {n[0], n[1], n[2]}, 16, esz))
        REFUSE(PTTS_E_INVALID, "cache rows must start at multiples of 16 bytes");
    return PTTS_OK;
}

int check_batch(const ptts_paged_batch* b, bool written) {
    if (!b) REFUSE(PTTS_E_INVALID, "null batch");
    if (b->n_seqs < 0 || b->tokens < 0 || b->max_pages < 0) REFUSE(PTTS_E_INVALID, "negative batch sizes");
    if (b->n_seqs > 0 && (!b->past || (!b->table && b->max_pages > 0))) REFUSE(PTTS_E_INVALID, "null page table or lengths");
    if (!b->starts && b->tokens != b->n_seqs) REFUSE(PTTS_E_INVALID, "%d tokens of %d sequences need starts", b->tokens, b->n_seqs);
    // sequences may read the same row of pages; where they write, no two of them own a slot
    if (b->n_seqs <= 1) return PTTS_OK;
    if (b->table_stride < b->max_pages && (written || b->table_stride != 0)) REFUSE(PTTS_E_INVALID, "page table rows overlap");
    if ((int64_t)b->table_stride > INT_MAX) REFUSE(PTTS_E_INVALID, "page table stride out of range");
    return PTTS_OK;
}

int check_rows(const char* name, const void* p, const int64_t* st, int64_t tokens, int64_t heads, int64_t d, bool written) {
    if (!p) REFUSE(PTTS_E_INVALID, "null %s", name);
    const int64_t n[2] = {tokens, heads};
    if (!fits(st, n, 2)) REFUSE(PTTS_E_INVALID, "%s: strides out of range", name);
    if (written && overlaps_itself(st, n, 2, d)) REFUSE(PTTS_E_INVALID, "%s: rows share elements", name);
    return PTTS_OK;
}

// a tensor of rows of `inner` contiguous elements
struct Strided { const void* p; const int64_t *st, *n; int dims, esz; int64_t inner; };

// Whether two of them have a byte in common: whether the distance of their first bytes plus indices times strides plus places within the rows
// can be 0.  Indices of equal strides count as one (their difference), as slices of one buffer's rows have them.  Places that reach
// everything between two ends are an interval; a stride no longer than it extends it, the longer ones are tried, longest first (few of a
// stride can fit, where the shorter ones reach less far than it).  Exact, up to 4096 trials; what would take more counts as shared.
struct Meeting {
    int64_t st[6], lo[6], hi[6];     // bytes, least and largest index; ascending
    int64_t low, high;               // the interval
    int dims = 0, trials = 0;
    void add(int64_t s, int64_t l, int64_t h) {
        int i = dims++;
        for (; i > 0 && st[i - 1] > s; --i) { st[i] = st[i - 1]; lo[i] = lo[i - 1]; hi[i] = hi[i - 1]; }
        st[i] = s; lo[i] = l; hi[i] = h;
    }
    static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }       // b > 0
    bool reaches(int64_t x, int left) {        // 0 from x, by the first `left` strides and the interval
        if (++trials > 4096) return true;
        if (left == 0) return x + low <= 0 && x + high >= 0;
        int64_t l = low, h = high;
        for (int i = 0; i < left - 1; ++i) { l += lo[i] * st[i]; h += hi[i] * st[i]; }
        const int64_t s = st[left - 1];
        const int64_t from = -floor_div(x + h, s), to = floor_div(-x - l, s);
        for (int64_t d = from > lo[left - 1] ? from : lo[left - 1]; d <= to && d <= hi[left - 1]; ++d)
            if (reaches(x + d * s, left - 1)) return true;
        return false;
    }
};

int64_t bytes_spanned(const Strided& t) {
    int64_t e = t.inner;
    for (int i = 0; i < t.dims; ++i) e += (t.n[i] - 1) * t.st[i];
    return e * t.esz;
}

bool share_memory(const Strided& a, const Strided& b) {
    const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    if (pb >= pa ? (int64_t)(pb - pa) >= bytes_spanned(a) : (int64_t)(pa - pb) >= bytes_spanned(b)) return false;
    Meeting m;
    bool taken[3] = {false, false, false};
    for (int i = 0; i < a.dims; ++i) {
        if (a.n[i] <= 1 || a.st[i] == 0) continue;
        int64_t hi = 0;
        for (int j = 0; j < b.dims; ++j)
            if (!taken[j] && b.n[j] > 1 && b.st[j] * b.esz == a.st[i] * a.esz) { taken[j] = true; hi = b.n[j] - 1; break; }
        m.add(a.st[i] * a.esz, 1 - a.n[i], hi);
    }
    for (int j = 0; j < b.dims; ++j)
        if (!taken[j] && b.n[j] > 1 && b.st[j] != 0) m.add(b.st[j] * b.esz, 0, b.n[j] - 1);
    m.low = 1 - a.inner * a.esz;
    m.high = b.inner * b.esz - 1;
    int k = 0;
    for (; k < m.dims && m.st[k] <= m.high - m.low + 1; ++k) { m.low += m.lo[k] * m.st[k]; m.high += m.hi[k] * m.st[k]; }
    for (int i = k; i < m.dims; ++i) { m.st[i - k] = m.st[i]; m.lo[i - k] = m.lo[i]; m.hi[i - k] = m.hi[i]; }
    return m.reaches((int64_t)(pb - pa), m.dims - k);
}

// the same rows at the same places
bool in_place(const Strided& a, const Strided& b) {
    if (a.p != b.p) return false;
    for (int i = 0; i < a.dims; ++i)
        if (a.n[i] > 1 && a.st[i] != b.st[i]) return false;
    return true;
}

// whether a tensor and the cache's keys or values share memory
bool in_cache(const ptts_paged_kv* c, const Strided& t) {
    const int esz = c->dtype == PTTS_DTYPE_BF16 ? 2 : 4;
    const int64_t n[3] = {c->n_pages, c->kv_heads, c->page_tokens};
    return share_memory(Strided{c->k, c->k_strides, n, 3, esz, c->head_dim}, t) || share_memory(Strided{c->v, c->v_strides, n, 3, esz, c->head_dim}, t);
}

PagedBatchArgs batch_args(const ptts_paged_kv* c, const ptts_paged_batch* b) {
    PagedBatchArgs r;
    r.table = b->table; r.table_stride = b->table_stride; r.past = b->past; r.starts = b->starts;
    r.max_pages = b->max_pages; r.n_pages = c->n_pages; r.n_seqs = b->n_seqs; r.tokens = b->tokens;
    r.page_shift = __builtin_ctz((unsigned)c->page_tokens);
    return r;
}

RotaryArgs rotary_args(const ptts_rotary* r) {
    RotaryArgs a = {nullptr, nullptr, 0, 0, 0};
    if (r) { a.cos_t = r->cos_t; a.sin_t = r->sin_t; a.positions = r->positions; a.dims = r->dims; a.interleaved = r->interleaved ? 1 : 0; }
    return a;
}

#define TRY(expr)                       \
    do {                                \
        const int rc_ = (expr);         \
        if (rc_ != PTTS_OK) return rc_; \
    } while (0)

int launched(const char* what, hipError_t e) {
    if (e != hipSuccess) REFUSE(PTTS_E_HIP, "%s failed: %s", what, hipGetErrorString(e));
    return PTTS_OK;
}

constexpr int MAX_UNITS = 32768;      // units of work of a token (SmallDiv)

}  // namespace

extern "C" {

int ptts_rotary_embed(const ptts_rotary* rot, int32_t dtype, int32_t tokens, int32_t heads, int32_t head_dim, const void* x,
                      int64_t x_token_stride, int64_t x_head_stride, const int32_t* positions, void* out, int64_t out_token_stride,
                      int64_t out_head_stride, int32_t* status, void* stream) {
    if (!rot || !status) REFUSE(PTTS_E_INVALID, "null argument");
    if (dtype != PTTS_DTYPE_F32 && dtype != PTTS_DTYPE_BF16) REFUSE(PTTS_E_INVALID, "dtype must be 0 (f32) or 1 (bf16)");
    if (tokens < 0 || heads <= 0 || head_dim <= 0 || head_dim % 2) REFUSE(PTTS_E_INVALID, "%d tokens of %d heads of %d", tokens, heads, head_dim);
    if ((int64_t)heads * head_dim / 2 > MAX_UNITS) REFUSE(PTTS_E_UNSUPPORTED, "%d heads of %d: at most 65536 features a token", heads, head_dim);
    TRY(check_rotary(rot, head_dim));
    if (tokens == 0) return PTTS_OK;
    if (!positions) REFUSE(PTTS_E_INVALID, "null positions");
    RotaryEmbedArgs a;
    a.x = x; a.out = out; a.xs[0] = x_token_stride; a.xs[1] = x_head_stride; a.os[0] = out_token_stride; a.os[1] = out_head_stride;
    TRY(check_rows("x", x, a.xs, tokens, heads, head_dim, false));
    TRY(check_rows("out", out, a.os, tokens, heads, head_dim, true));
    const int esz = dtype == PTTS_DTYPE_BF16 ? 2 : 4;
    const int64_t n[2] = {tokens, heads};
    const Strided xs = {x, a.xs, n, 2, esz, head_dim}, os = {out, a.os, n, 2, esz, head_dim};
    if (!in_place(xs, os) && share_memory(xs, os))
        REFUSE(PTTS_E_INVALID, "x and out share memory in another layout than in place");
    a.pos = positions; a.rot = rotary_args(rot); a.status = status; a.tokens = tokens; a.heads = heads; a.head_dim = head_dim;
    return launched("ptts_rotary_embed", rotary_embed_launch(a, dtype, (hipStream_t)stream));
}

int ptts_kv_append(const ptts_paged_kv* cache, const ptts_paged_batch* batch, int32_t dtype, const void* k, int64_t k_token_stride,
                   int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride, const ptts_rotary* rot,
                   const int32_t* positions, int32_t q_heads, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                   int64_t q_out_token_stride, int64_t q_out_head_stride, int32_t* status, void* stream) {
    TRY(check_kv(cache));
    TRY(check_batch(batch, true));
    if (!status) REFUSE(PTTS_E_INVALID, "null status");
    if (dtype != PTTS_DTYPE_F32 && dtype != PTTS_DTYPE_BF16) REFUSE(PTTS_E_INVALID, "dtype must be 0 (f32) or 1 (bf16)");
    if (dtype == PTTS_DTYPE_BF16 && cache->dtype != PTTS_DTYPE_BF16) REFUSE(PTTS_E_UNSUPPORTED, "bf16 rows into an f32 cache");
    if (rot) TRY(check_rotary(rot, cache->head_dim));
    if (q_heads < 0 || (q_heads == 0) != (q == nullptr) || (q_heads == 0) != (q_out == nullptr)) REFUSE(PTTS_E_INVALID, "q: %d heads", q_heads);
    const int64_t T = batch->tokens, D = cache->head_dim;
    if (((int64_t)q_heads + 2 * (int64_t)cache->kv_heads) * D / 2 > MAX_UNITS)
        REFUSE(PTTS_E_UNSUPPORTED, "%d query and %d key heads of %d: at most 65536 features a token", q_heads, cache->kv_heads, cache->head_dim);
    if (T == 0 || batch->n_seqs == 0) return PTTS_OK;
    AppendArgs a;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.k_cache = cache->k; a.v_cache = cache->v;
    a.qs[0] = q_token_stride; a.qs[1] = q_head_stride; a.qos[0] = q_out_token_stride; a.qos[1] = q_out_head_stride;
    a.ks[0] = k_token_stride; a.ks[1] = k_head_stride; a.vs[0] = v_token_stride; a.vs[1] = v_head_stride;
    TRY(check_rows("k", k, a.ks, T, cache->kv_heads, D, false));
    TRY(check_rows("v", v, a.vs, T, cache->kv_heads, D, false));
    const int esz = dtype == PTTS_DTYPE_BF16 ? 2 : 4;
    const int64_t n[2] = {T, cache->kv_heads}, nq[2] = {T, q_heads};
    const Strided ks = {k, a.ks, n, 2, esz, D}, vs = {v, a.vs, n, 2, esz, D};
    if (q_heads) {
        TRY(check_rows("q", q, a.qs, T, q_heads, D, false));
        TRY(check_rows("q_out", q_out, a.qos, T, q_heads, D, true));
        const Strided qs = {q, a.qs, nq, 2, esz, D}, qos = {q_out, a.qos, nq, 2, esz, D};
        if (!in_place(qs, qos) && share_memory(qs, qos))
            REFUSE(PTTS_E_INVALID, "q and q_out share memory in another layout than in place");
        if (share_memory(ks, qos) || share_memory(vs, qos)) REFUSE(PTTS_E_INVALID, "q_out shares memory with k or v");
        if (in_cache(cache, qs) || in_cache(cache, qos)) REFUSE(PTTS_E_INVALID, "q or q_out share memory with the cache");
    }
    // rows may be stored over while another workgroup still reads them, and which slots are stored to is known on the device only
    if (in_cache(cache, ks) || in_cache(cache, vs)) REFUSE(PTTS_E_INVALID, "k or v share memory with the cache");
    const int64_t nc[3] = {cache->n_pages, cache->kv_heads, cache->page_tokens};
    const int csz = cache->dtype == PTTS_DTYPE_BF16 ? 2 : 4;
    if (share_memory(Strided{cache->k, cache->k_strides, nc, 3, csz, D}, Strided{cache->v, cache->v_strides, nc, 3, csz, D}))
        REFUSE(PTTS_E_INVALID, "keys and values of the cache share memory");
    for (int i = 0; i < 3; ++i) { a.kc[i] = cache->k_strides[i]; a.vc[i] = cache->v_strides[i]; }
    a.b = batch_args(cache, batch); a.rot = rotary_args(rot); a.pos = rot ? positions : nullptr; a.status = status;
    a.q_heads = q_heads; a.kv_heads = cache->kv_heads; a.head_dim = cache->head_dim;
    return launched("ptts_kv_append", kv_append_launch(a, dtype, cache->dtype, (hipStream_t)stream));
}

}  // extern "C"

namespace {
int attn_args(const ptts_paged_kv* cache, const ptts_paged_batch* batch, int32_t q_heads, int32_t max_new, PagedAttnArgs* a) {
    TRY(check_kv(cache));
    TRY(check_batch(batch, false));
    if (q_heads <= 0 || q_heads % cache->kv_heads) REFUSE(PTTS_E_INVALID, "%d query heads over %d key heads", q_heads, cache->kv_heads);
    if (q_heads > 65535) REFUSE(PTTS_E_UNSUPPORTED, "%d query heads", q_heads);
    if (max_new < 0) REFUSE(PTTS_E_INVALID, "max_new %d", max_new);
    if ((int64_t)batch->max_pages * cache->page_tokens > INT_MAX - 4095) REFUSE(PTTS_E_UNSUPPORTED, "a page table row reaches past 2^31 - 4096 tokens");
    if ((int64_t)batch->tokens * (q_heads / cache->kv_heads) > INT_MAX - 65536) REFUSE(PTTS_E_UNSUPPORTED, "too many query rows");
    *a = PagedAttnArgs();
    a->k = cache->k; a->v = cache->v;
    for (int i = 0; i < 3; ++i) { a->kc[i] = cache->k_strides[i]; a->vc[i] = cache->v_strides[i]; }
    const PagedBatchArgs b = batch_args(cache, batch);
    a->table = b.table; a->table_stride = b.table_stride; a->past = b.past; a->starts = b.starts;
    a->max_pages = b.max_pages; a->n_pages = b.n_pages; a->page_shift = b.page_shift; a->n_seqs = b.n_seqs; a->tokens = b.tokens;
    a->q_heads = q_heads; a->kv_heads = cache->kv_heads; a->group = q_heads / cache->kv_heads;
    return PTTS_OK;
}
}  // namespace

extern "C" {

int64_t ptts_paged_attention_workspace(const ptts_paged_kv* cache, const ptts_paged_batch* batch, int32_t q_heads, int32_t max_new) {
    PagedAttnArgs a;
    TRY(attn_args(cache, batch, q_heads, max_new, &a));
    if (a.tokens == 0 || a.n_seqs == 0) return 0;
    return paged_attn_workspace(a, max_new, cache->head_dim, cache->dtype);
}

int ptts_paged_attention(const ptts_paged_kv* cache, const ptts_paged_batch* batch, int32_t q_heads, const void* q, int64_t q_token_stride,
                         int64_t q_head_stride, void* out, int64_t out_token_stride, int64_t out_head_stride, float scale, int32_t causal,
                         const uint8_t* key_mask, int64_t mask_stride, int32_t mask_width, int32_t max_new, void* workspace,
                         int64_t workspace_bytes, int32_t* status, void* stream) {
    PagedAttnArgs a;
    TRY(attn_args(cache, batch, q_heads, max_new, &a));
    if (!status) REFUSE(PTTS_E_INVALID, "null status");
    if (!(scale > 0.f) || !std::isfinite(scale)) REFUSE(PTTS_E_INVALID, "softmax scale must be positive and finite");
    if (key_mask && (mask_width < 0 || (mask_stride < mask_width && batch->n_seqs > 1))) REFUSE(PTTS_E_INVALID, "key mask of %d columns", mask_width);
    const int64_t T = batch->tokens, D = cache->head_dim;
    if (T == 0 || batch->n_seqs == 0) return PTTS_OK;
    a.q = q; a.out = out;
    a.qs[0] = q_token_stride; a.qs[1] = q_head_stride; a.os[0] = out_token_stride; a.os[1] = out_head_stride;
    TRY(check_rows("q", q, a.qs, T, q_heads, D, false));
    TRY(check_rows("out", out, a.os, T, q_heads, D, true));
    const int esz = cache->dtype == PTTS_DTYPE_BF16 ? 2 : 4;
    if (!aligned(q, a.qs, {T, q_heads}, 16, esz) || !aligned(out, a.os, {T, q_heads}, 16, esz)) REFUSE(PTTS_E_INVALID, "rows of q and out must start at multiples of 16 bytes");
    const int64_t n[2] = {T, q_heads};
    const Strided os = {out, a.os, n, 2, esz, D};
    if (share_memory(Strided{q, a.qs, n, 2, esz, D}, os)) REFUSE(PTTS_E_INVALID, "q and out share memory");
    if (in_cache(cache, os)) REFUSE(PTTS_E_INVALID, "out shares memory with the cache");
    a.mask = key_mask && mask_width > 0 ? key_mask : nullptr; a.mask_stride = mask_stride; a.mask_width = a.mask ? mask_width : 0;
    a.scale_log2 = scale * 1.4426950408889634f; a.causal = causal ? 1 : 0; a.status = status;
    const int64_t need = paged_attn_workspace(a, max_new, cache->head_dim, cache->dtype);
    if (need > 0 && (!workspace || workspace_bytes < need)) REFUSE(PTTS_E_INVALID, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    if ((uintptr_t)workspace % 16) REFUSE(PTTS_E_INVALID, "workspace must start at a multiple of 16 bytes");
    a.part = (float*)workspace;
    return launched("ptts_paged_attention", paged_attn_launch(a, max_new, cache->head_dim, cache->dtype, (hipStream_t)stream));
}

}  // extern "C"

// Attention of new tokens over a paged KV cache: o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j a query may see.
//
// Both kernels make ONE pass over the keys with the running maximum and sum of the softmax, and both hold the scores TRANSPOSED:
// S^T = K Q^T puts a query into a column, so that a lane owns one query and a few of its scores; the maximum is a register maximum
// plus one or two lane swaps, the running state is one register per lane, and the probabilities are already the B operand of
// O^T = V^T P^T when the keys of a matrix step are numbered as the accumulator left them (key 8 (j / 4) + 4 h + j % 4 in slot j of
// half h: any numbering serves as long as V^T uses the same one).  V^T comes out of LDS by transposing reads (bf16) or plain
// dword reads (f32: a lane reads its feature of the slot's key).
//   * "rows" of a (sequence, key head) are its new tokens times the query heads of the group: a page is read once for all of them;
//   * K and V travel to LDS by LDS-DMA, 16 bytes a lane, 16-byte chunks XOR-swizzled by the row so that neither the row-wise reads
//     of K nor the transposing reads of V meet in a bank;
//   * scores, maxima, sums and outputs are 32 bits; in bf16 the probabilities are rounded once (half a bf16 step of each, the type
//     of V and of the result) to enter the matrix unit.
//
// A value that is not finite in a row that some queries may not see would reach them as 0 * inf in the matrix unit.  Nothing in the
// loops guards against it: a query whose result is not finite is computed again, alone, over the keys it sees (row_alone).
#include "ptts_common.h"
#include "gemm.h"
#include "paged.h"
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

template <int N> __device__ inline void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ inline void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename P> __device__ inline void load16(const typename P::elem_t* p, float* f);
template <> __device__ inline void load16<PBF16>(const uint16_t* p, float* f) {
    const u32x4 r = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = r[i];
        f[2 * i] = __builtin_bit_cast(float, w << 16);
        f[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
    }
}
template <> __device__ inline void load16<PF32>(const float* p, float* f) {
    const f32x4 r = *reinterpret_cast<const f32x4*>(p);
    f[0] = r[0]; f[1] = r[1]; f[2] = r[2]; f[3] = r[3];
}

__device__ inline float swap_max32(float x) {      // maximum over lanes l and l ^ 32
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
#else
    return x;
#endif
}
__device__ inline float swap_max16(float x) {      // maximum over lanes l and l ^ 16
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
#else
    return x;
#endif
}
__device__ inline float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}
// Transposing reads of V: 16 lanes take a block of 4 keys x 16 features (each lane 4 features of one key), lane i ends with feature i of
// the 4 keys.  A and B are the two blocks of a matrix step.  Written out, because hipcc drains the LDS-DMA in flight in front of the
// builtin; the wait stands in the same statement as the reads.
template <int OFF_A, int OFF_B> __device__ inline void read_v4(unsigned a0, unsigned a1, unsigned a2, unsigned a3, s16x8 (&v)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
    s16x4 r[8];
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                 : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(OFF_A), "n"(OFF_B) : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_shufflevector(r[2 * i], r[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#endif
}
// the same for two feature blocks a0, a1 of two steps
template <int A, int B, int C, int D> __device__ inline void read_v2(unsigned a0, unsigned a1, s16x8 (&v)[4]) {
#if defined(__HIP_DEVICE_COMPILE__)
    s16x4 r[8];
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %1, %8 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%10\n\tds_read_b64_tr_b16 %3, %9 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:%12\n\tds_read_b64_tr_b16 %5, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %9 offset:%12\n\tds_read_b64_tr_b16 %7, %9 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
                 : "v"(a0), "v"(a1), "n"(A), "n"(B), "n"(C), "n"(D) : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_shufflevector(r[2 * i], r[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
#endif
}
__device__ inline unsigned lds_address(const void* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
#else
    return 0;
#endif
}
template <int I, int N, typename F> __device__ inline void unrolled(F&& f) {      // f(integral constant I), f(I + 1), ...
    if constexpr (I < N) { f(std::integral_constant<int, I>()); unrolled<I + 1, N>(f); }
}
__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- where a workgroup's rows lie ------------------------------------------------------------------------------------------
struct Span {          // one sequence's new tokens
    int seq, first, n, past;
    bool bad;          // its length leads behind its row of the page table: every row becomes NaN
};

// The sequence and its tile that tile t of a launch is, where tiles hold M rows: a prefix sum over the sequences' tiles, 64 sequences at
// a time, by every wave for itself (lengths and cache lengths come in one round trip).  Tiles of no sequence are the launch's last ones:
// with holes between the sequences (a numbering that needs no sum) the dispatcher put all work of equal chunks on half of the CUs.
__device__ inline bool find_tile(const PagedAttnArgs& a, int t, int M, Span* sp, int* tile) {
    if (!a.starts) {
        const int per = (a.group + M - 1) / M, s = t / per;
        sp->seq = sp->first = s;
        sp->n = 1;
        sp->past = uniform(a.past[s]);
        *tile = t - s * per;
    } else {
        const int lane = threadIdx.x & 63;
        int rest = t, i0 = 0, sel, first = 0, n = 0, past = 0, sum;
        for (;; i0 += 64) {
            if (i0 >= a.n_seqs) return false;
            const int i = min(i0 + lane, a.n_seqs - 1);
            first = a.starts[i];
            const int end = a.starts[i + 1];
            past = a.past[i];
            n = i0 + lane < a.n_seqs && first >= 0 && end <= a.tokens ? max(end - first, 0) : 0;       // starts that are wrong own no rows
            const int own = (n * a.group + M - 1) / M;
            sum = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) { const int x = __shfl_up(sum, d); sum += lane >= d ? x : 0; }
            sel = __popcll(__ballot(sum <= rest));
            if (sel < 64) { sum -= own; break; }
            rest -= __builtin_amdgcn_readlane(sum, 63);
        }
        sel = uniform(sel);
        sp->seq = i0 + sel;
        sp->first = __builtin_amdgcn_readlane(first, sel);
        sp->n = __builtin_amdgcn_readlane(n, sel);
        sp->past = __builtin_amdgcn_readlane(past, sel);
        *tile = rest - __builtin_amdgcn_readlane(sum, sel);
        if (sp->n == 0) return false;
    }
    const int64_t reach = (int64_t)a.max_pages << a.page_shift;
    sp->bad = sp->past < 0 || (int64_t)sp->past + (a.causal ? sp->n : 0) > reach;
    if (sp->bad) {
        if (threadIdx.x == 0) atomicOr(a.status, PAGED_BAD_LENGTH);
        sp->past = 0;
    }
    return true;
}

// ---- page ids of the keys ahead, one per lane ---------------------------------------------------------------------------------
struct Pages {
    const int* row;
    int base, ids, n_pages;     // lane l holds the id of page base + l
    bool bad;
    __device__ inline void load(int first, int last) {       // pages first .. (at most 64), none behind `last`
        base = first;
        const int i = first + (int)(threadIdx.x & 63);
        ids = row[min(i, last)];
        const bool wrong = (unsigned)ids >= (unsigned)n_pages;
        bad = bad || __any(wrong);
        if (wrong) ids = 0;
    }
    __device__ inline int get(int page) const { return __builtin_amdgcn_readlane(ids, page - base); }
};

// ---- a tile of KT rows of K or V on its way to LDS: one wave moves ROWS of them -------------------------------------------------
// chunk c (16 bytes) of row r stands at chunk c ^ (r & 7) of the row's LDS image.  Rows at or behind `end` are read from the last row
// in front of it: what lies there is seen by nobody, and may be anything.
template <typename P, int D, int ROWS>
__device__ inline void dma_rows(const char* base, int64_t page_bytes, int64_t slot_bytes, const Pages& pg, int page_shift, int key0, int row0,
                                int end, char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) void lds_void;
    constexpr int RB = D * (int)sizeof(typename P::elem_t), RPI = 1024 / RB, CPR = RB / 16;
    const int lane = threadIdx.x & 63, rl = lane / CPR, c = lane % CPR;
    const int mask = (1 << page_shift) - 1;
#pragma unroll
    for (int i = 0; i < ROWS / RPI; ++i) {
        const int r = row0 + i * RPI;                                   // first row of this instruction: its rows share a page
        const int page = pg.get(min(key0 + r, end - 1) >> page_shift);
        const int slot = min(key0 + r + rl, end - 1) & mask;
        const char* src = base + page * page_bytes + slot * slot_bytes + ((c ^ ((r + rl) & 7)) << 4);
        __builtin_amdgcn_global_load_lds(reinterpret_cast<const void*>(src), (lds_void*)(lds + r * RB), 16, 0, 0);
    }
#endif
}

// keys that may be looked at at all, as bits: the key mask's bytes of the tile (lane i: key key0 + i), ones behind its last column
__device__ inline uint64_t tile_mask(const PagedAttnArgs& a, int seq, int key0) {
    if (!a.mask || key0 >= a.mask_width) return ~0ull;
    const int j = key0 + (int)(threadIdx.x & 63);
    bool live = true;
    if (j < a.mask_width) live = a.mask[seq * a.mask_stride + j] != 0;
    return __ballot(live);
}

// ---- one query over the keys [k0, k1) it sees, by one wave (see the head of the file) ------------------------------------------
template <typename P, int D>
__device__ inline void row_alone(const PagedAttnArgs& a, int seq, int kvh, const typename P::elem_t* q, int k0, int k1, float* m_out, float* l_out,
                                 float (&acc)[D / 64]) {
    typedef typename P::elem_t elem_t;
    constexpr int V = 16 / sizeof(elem_t), R = D / 64;
    const int lane = threadIdx.x & 63, mask = (1 << a.page_shift) - 1;
    const elem_t* kb = reinterpret_cast<const elem_t*>(a.k) + kvh * a.kc[1];
    const elem_t* vb = reinterpret_cast<const elem_t*>(a.v) + kvh * a.vc[1];
    const int* table = a.table + seq * a.table_stride;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.f;
    for (int j0 = k0; j0 < k1; j0 += 64) {
        const int j = j0 + lane;
        float sc = -INFINITY;
        int page = -1;
        if (j < k1 && (!a.mask || j >= a.mask_width || a.mask[seq * a.mask_stride + j])) {
            page = table[j >> a.page_shift];
            if ((unsigned)page >= (unsigned)a.n_pages) page = 0;        // the caller of this has found it already
            const elem_t* kp = kb + page * a.kc[0] + (j & mask) * a.kc[2];
            float d = 0.f;
            for (int c = 0; c < D; c += V) {
                float x[V], y[V];
                load16<P>(q + c, x);
                load16<P>(kp + c, y);
#pragma unroll
                for (int i = 0; i < V; ++i) d = fmaf(x[i], y[i], d);
            }
            sc = d * a.scale_log2;
        }
        const float mn = fmaxf(m, wave_max(sc)), mu = mn == -INFINITY ? 0.f : mn;
        const float p = page >= 0 ? exp2_hw(sc - mu) : 0.f, al = exp2_hw(m - mu);
        l = l * al + wave_sum(p);
        m = mn;
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] *= al;
        for (int i = 0; i < 64 && j0 + i < k1; ++i) {
            const int pg = __shfl(page, i);
            const float pi = __shfl(p, i);
            if (pg < 0) continue;
            const elem_t* vp = vb + pg * a.vc[0] + ((j0 + i) & mask) * a.vc[2];
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] = fmaf(pi, from_elem<P>(vp[r * 64 + lane]), acc[r]);
        }
    }
    *m_out = m; *l_out = l;
}

// where the partial results of a split launch lie: outputs [split][token * q_heads + head][D], behind them (maximum, sum) pairs
template <int D> __device__ inline float* part_out(const PagedAttnArgs& a, int split, int64_t row) {
    return a.part + ((int64_t)split * a.tokens * a.q_heads + row) * D;
}
template <int D> __device__ inline float* part_ml(const PagedAttnArgs& a, int split, int64_t row) {
    const int64_t rows = (int64_t)a.tokens * a.q_heads;
    return a.part + (int64_t)a.splits * rows * D + (split * rows + row) * 2;
}

template <typename P, int D>
__device__ inline void store_row_alone(const PagedAttnArgs& a, int seq, int kvh, int64_t token, int head, int split, int k0, int k1) {
    typedef typename P::elem_t elem_t;
    const int lane = threadIdx.x & 63;
    float m, l, acc[D / 64];
    row_alone<P, D>(a, seq, kvh, reinterpret_cast<const elem_t*>(a.q) + token * a.qs[0] + head * a.qs[1], k0, k1, &m, &l, acc);
    const int64_t row = token * a.q_heads + head;
#pragma unroll
    for (int r = 0; r < D / 64; ++r) {
        if (a.splits > 1) part_out<D>(a, split, row)[r * 64 + lane] = acc[r];
        else (reinterpret_cast<elem_t*>(a.out) + token * a.os[0] + head * a.os[1])[r * 64 + lane] = to_elem<P>(l == 0.f ? 0.f : acc[r] / l);
    }
    if (a.splits > 1 && lane == 0) { float* ml = part_ml<D>(a, split, row); ml[0] = m; ml[1] = l; }
}

// keys of split `split`: equal shares of whole tiles
__device__ inline void split_range(const PagedAttnArgs& a, int split, int end, int KT, int* k0, int* k1) {
    if (a.splits == 1) { *k0 = 0; *k1 = end; return; }
    const int tiles = (end + KT - 1) / KT, share = (tiles + a.splits - 1) / a.splits;
    *k0 = min(split * share * KT, end);
    *k1 = min(*k0 + share * KT, end);
}

template <typename P> __device__ inline void store4(typename P::elem_t* p, float a, float b, float c, float d);
template <> __device__ inline void store4<PBF16>(uint16_t* p, float a, float b, float c, float d) {
    typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
    const bf16x4 v = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
    *reinterpret_cast<bf16x4*>(p) = v;
}
template <> __device__ inline void store4<PF32>(float* p, float a, float b, float c, float d) {
    const f32x4 v = {a, b, c, d};
    *reinterpret_cast<f32x4*>(p) = v;
}

// =================================================================================================================================
// Chunks: a workgroup owns 128 rows (32 per wave), the keys pass in tiles of KT through a ring of LDS buffers.
// =================================================================================================================================
template <typename P, int D> struct TileCfg {
    static constexpr int M = 128, NW = 4;
    static constexpr int RB = D * (int)sizeof(typename P::elem_t);
    static constexpr int KT = RB <= 256 ? 64 : 32;
    static constexpr int TILE = KT * RB;                       // bytes of K or V of a tile
    static constexpr int NBUF = 65536 / (2 * TILE);            // ring of tiles: 64 KiB, two workgroups on a CU
    static constexpr int LDS = NBUF * 2 * TILE;                // [buffer][K, V]
    static constexpr int DMA = 2 * TILE / NW / 1024;           // LDS-DMA instructions per wave and tile
};

template <typename P, int D>
__global__ __launch_bounds__(256, 2) void paged_attn_tile_kernel(PagedAttnArgs a) {
    typedef typename P::elem_t elem_t;
    typedef TileCfg<P, D> C;
    constexpr int KT = C::KT, RB = C::RB, EPL = P::EPL, NKS = D / (2 * EPL), NKB = KT / 32, NDB = D / 32;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), l31 = lane & 31, h = lane >> 5;

    if (blockIdx.x == 0 && a.starts) check_starts(a.starts, a.n_seqs, a.tokens, a.status);
    // consecutive workgroups go to consecutive XCDs: with the key head innermost, an XCD's L2 holds few heads' pages
    const int kvh = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads, split = rest % a.splits;
    Span sp;
    int tile;
    if (!find_tile(a, rest / a.splits, C::M, &sp, &tile)) return;
    const int rows = sp.n * a.group;
    tile = (rows + C::M - 1) / C::M - 1 - tile;                // the rows that see most first
    const int r0 = tile * C::M, r_end = min(r0 + C::M, rows);
    const int row = r0 + w * 32 + l31;                         // this lane's query
    const bool live = row < r_end;
    const int tok = live ? row / a.group : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
    const int64_t token = sp.first + tok;
    int lim = live && !sp.bad ? sp.past + (a.causal ? tok + 1 : 0) : 0;       // keys 0 .. lim - 1 are seen
    const int tile_end = sp.bad ? 0 : sp.past + (a.causal ? (r_end - 1) / a.group + 1 : 0);
    int k0, k1;
    split_range(a, split, tile_end, KT, &k0, &k1);
    const int wr0 = r0 + w * 32, wr1 = min(wr0 + 32, r_end);                  // rows of this wave: [wr0, wr1)
    const int w_end = wr0 < wr1 && !sp.bad ? (a.causal ? sp.past + (wr1 - 1) / a.group + 1 : sp.past) : 0;   // keys any of them sees
    const int w_all = wr0 < wr1 && !sp.bad ? (a.causal ? sp.past + wr0 / a.group + 1 : sp.past) : 0;         // keys all of them see

    Pages pg;
    pg.row = a.table + sp.seq * a.table_stride; pg.n_pages = a.n_pages; pg.bad = false; pg.base = 0; pg.ids = 0;
    const int64_t kp = a.kc[0] * (int)sizeof(elem_t), ks = a.kc[2] * (int)sizeof(elem_t);
    const int64_t vp = a.vc[0] * (int)sizeof(elem_t), vs = a.vc[2] * (int)sizeof(elem_t);
    const char* kbase = reinterpret_cast<const char*>(a.k) + kvh * a.kc[1] * (int)sizeof(elem_t);
    const char* vbase = reinterpret_cast<const char*>(a.v) + kvh * a.vc[1] * (int)sizeof(elem_t);
    auto fetch = [&](int key0, int buf) {
        const int last = (k1 - 1) >> a.page_shift;
        if (((min(key0 + KT, k1) - 1) >> a.page_shift) >= pg.base + 64) pg.load(key0 >> a.page_shift, last);
        char* lds = smem + buf * 2 * C::TILE;
        dma_rows<P, D, KT / C::NW>(kbase, kp, ks, pg, a.page_shift, key0, w * (KT / C::NW), k1, lds);
        dma_rows<P, D, KT / C::NW>(vbase, vp, vs, pg, a.page_shift, key0, w * (KT / C::NW), k1, lds + C::TILE);
    };

    // B operand of S^T = K Q^T: 16-byte chunk 2 s + h of the lane's query row at step s (and of the lane's key row for A)
    u32x4 qf[NKS];
    {
        const elem_t* qp = reinterpret_cast<const elem_t*>(a.q) + token * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int s = 0; s < NKS; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + (2 * s + h) * EPL);
    }
    f32x16 o[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;       // maximum of the query's scores (log2 units), sum of the weights of this half's keys

    // the query rows arrive before the first tile is sent for: a wait for them inside the loop would be one for the tiles in flight too
    if (k0 < k1) pg.load(k0 >> a.page_shift, (k1 - 1) >> a.page_shift);
#pragma unroll
    for (int t = 0; t < NKS; ++t) asm volatile("" : "+v"(qf[t]));
#pragma unroll
    for (int i = 0; i < C::NBUF - 1; ++i)
        if (k0 + i * KT < k1) fetch(k0 + i * KT, i);
    int buf = 0;
    for (int key0 = k0; key0 < k1; key0 += KT, buf = buf + 1 == C::NBUF ? 0 : buf + 1) {
        const int ahead = min(C::NBUF - 2, (k1 - key0 - 1) / KT);           // younger tiles that stay in flight
        if (C::NBUF > 3 && ahead >= 2) wait_vm<2 * C::DMA>();
        else if (C::NBUF > 2 && ahead >= 1) wait_vm<C::DMA>();
        else wait_vm<0>();
        wait_lds();
        __builtin_amdgcn_s_barrier();        // the tile has landed, and every wave has left the buffer of the tile before it
        if (key0 + (C::NBUF - 1) * KT < k1) fetch(key0 + (C::NBUF - 1) * KT, buf == 0 ? C::NBUF - 1 : buf - 1);
        if (key0 >= w_end) continue;         // nothing here for this wave's rows (it keeps moving its share of the tiles)
        const char* kt = smem + buf * 2 * C::TILE;
        const char* vt = kt + C::TILE;

        f32x16 s[NKB];
#pragma unroll
        for (int b = 0; b < NKB; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.f;
            const int kr = b * 32 + l31;
#pragma unroll
            for (int t = 0; t < NKS; ++t) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + kr * RB + (((2 * t + h) ^ (kr & 7)) << 4));
                if constexpr (P::IS_BF16) {
                    s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[t]), s[b], 0, 0, 0);
                } else {
                    const f32x4 kx = __builtin_bit_cast(f32x4, kf), qx = __builtin_bit_cast(f32x4, qf[t]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(kx[j], qx[j], s[b], 0, 0, 0);
                }
            }
        }
        const uint64_t alive = tile_mask(a, sp.seq, key0);
        if (key0 + KT > w_all || alive != ~0ull) {             // some key of the tile is not for some query
            const int left = lim - key0;
            const uint64_t see = (left >= 64 ? ~0ull : (left <= 0 ? 0ull : (1ull << left) - 1)) & alive;
            const uint32_t half[2] = {(uint32_t)(see >> (4 * h)), (uint32_t)(see >> 32 >> (4 * h))};
#pragma unroll
            for (int b = 0; b < NKB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[b][r] = (half[b] >> ((r & 3) + 8 * (r >> 2))) & 1 ? s[b][r] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        mx = swap_max32(mx) * a.scale_log2;
        // weights are kept relative to a maximum that may lag behind by 2^8 (their type holds that range as well as any): the sums
        // are rescaled only when a query's maximum has risen further
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx), al = mn == -INFINITY ? 1.f : exp2_hw(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= al;
        }
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int b = 0; b < NKB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = exp2_hw(fmaf(s[b][r], a.scale_log2, -mu));
                l += s[b][r];
            }
        if constexpr (P::IS_BF16) {
#if defined(__HIP_DEVICE_COMPILE__)
            // key 16 kk + 4 h + 0 .. 3 in slots 0 .. 3, 8 further on in slots 4 .. 7; the chunk swizzle of a row depends on 4 h + i16 / 4 only
            // and moves feature block d by 64 bytes for odd d, two blocks by 128
            const int i16 = lane & 15, vrow = 4 * h + (i16 >> 2), c0 = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);
            const unsigned va = lds_address(vt) + vrow * RB + ((c0 ^ (vrow & 7)) << 4) + (i16 & 1) * 8, vb = va ^ 64;
            unrolled<0, KT / 16>([&](auto KK) {
                constexpr int kk = decltype(KK)::value;
                if constexpr (NDB == 2 && (kk & 1)) return;           // done with the step in front
                s16x8 vf[4];
                if constexpr (NDB == 2) read_v2<16 * kk * RB, (16 * kk + 8) * RB, (16 * kk + 16) * RB, (16 * kk + 24) * RB>(va, vb, vf);
                else read_v4<16 * kk * RB, (16 * kk + 8) * RB>(va, vb, va + 128, vb + 128, vf);
#pragma unroll
                for (int u = 0; u < 4 / NDB; ++u) {
                    bf16x8 pf;
#pragma unroll
                    for (int j = 0; j < 8; ++j) pf[j] = (__bf16)s[(kk + u) >> 1][8 * ((kk + u) & 1) + j];
#pragma unroll
                    for (int d = 0; d < NDB; ++d)
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf[u * NDB + d]), pf, o[d], 0, 0, 0);
                }
            });
#endif
        } else {
#pragma unroll
            for (int b = 0; b < NKB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int vr = b * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
#pragma unroll
                    for (int d = 0; d < NDB; ++d) {
                        const int f = d * 32 + l31;
                        const float vx = *reinterpret_cast<const float*>(vt + vr * RB + (((f >> 2) ^ (vr & 7)) << 4) + (f & 3) * 4);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vx, s[b][r], o[d], 0, 0, 0);
                    }
                }
        }
    }
    wait_vm<0>();
    if (pg.bad && threadIdx.x == 0) atomicOr(a.status, PAGED_BAD_PAGE);
    const bool bad = pg.bad || sp.bad;
    l += __shfl_xor(l, 32);
    float inv = l == 0.f ? 0.f : 1.f / l;
    if (bad) { l = NAN; inv = NAN; }
    // a result that is not finite: of this query's own making, or a key that it does not see
    bool odd = false;
    if (!bad) {
        float z = l * 0.f;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = fmaf(o[d][r], 0.f, z);
        odd = live && !(z == 0.f);
    }
    const uint64_t odds = __ballot(odd);
    if (live) {
        const int64_t orow = token * a.q_heads + head;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int f = d * 32 + 2 * r + 4 * h;
                if (a.splits > 1) store4<PF32>(part_out<D>(a, split, orow) + f, o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
                else store4<P>(reinterpret_cast<elem_t*>(a.out) + token * a.os[0] + head * a.os[1] + f, o[d][r] * inv, o[d][r + 1] * inv,
                               o[d][r + 2] * inv, o[d][r + 3] * inv);
            }
        if (a.splits > 1 && h == 0) { float* ml = part_ml<D>(a, split, orow); ml[0] = m; ml[1] = l; }
    }
    uint32_t again = (uint32_t)odds | (uint32_t)(odds >> 32);
    while (again) {
        const int i = __builtin_ctz(again);
        again &= again - 1;
        const int rr = wr0 + i, tk = rr / a.group;
        store_row_alone<P, D>(a, sp.seq, kvh, sp.first + tk, kvh * a.group + rr - tk * a.group, split, k0,
                              min(k1, sp.past + (a.causal ? tk + 1 : 0)));
    }
}

// =================================================================================================================================
// Few rows (at most 16 per sequence and key head: single tokens, their groups, short drafts): bound by the stream of the cache.  A wave
// owns every NW-th tile of 32 keys and two LDS buffers of its own, so that nothing in the loop waits for another wave; the waves'
// states are joined once at the end.
// =================================================================================================================================
template <typename P, int D> struct StepCfg {
    static constexpr int M = 16, KT = 32;
    static constexpr int RB = D * (int)sizeof(typename P::elem_t);
    static constexpr int TILE = KT * RB, STAGE = 2 * TILE;
    static constexpr int NW = 65536 / (2 * STAGE);             // 4, 2, 2, 1 waves: 64 KiB of LDS, two workgroups on a CU
    static constexpr int DMA = STAGE / 1024;
    static_assert(NW * 16 * (D + 2) * 4 <= NW * 2 * STAGE, "the waves' states fit where their tiles were");
};

template <typename P, int D>
__global__ __launch_bounds__((StepCfg<P, D>::NW * 64)) void paged_attn_step_kernel(PagedAttnArgs a) {
    typedef typename P::elem_t elem_t;
    typedef StepCfg<P, D> C;
    constexpr int KT = C::KT, RB = C::RB, EPL = P::EPL, NKS = D / (4 * EPL), NDB = D / 16, NW = C::NW;
    __shared__ __attribute__((aligned(1024))) char smem[NW * 2 * C::STAGE];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;

    if (blockIdx.x == 0 && a.starts) check_starts(a.starts, a.n_seqs, a.tokens, a.status);
    const int kvh = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads, split = rest % a.splits;
    Span sp;
    int tile;
    if (!find_tile(a, rest / a.splits, C::M, &sp, &tile)) return;
    const int rows = sp.n * a.group, r0 = tile * C::M, r_end = min(r0 + C::M, rows);
    const int row = r0 + l15;
    const bool live = row < r_end;
    const int tok = live ? row / a.group : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
    const int64_t token = sp.first + tok;
    const int lim = live && !sp.bad ? sp.past + (a.causal ? tok + 1 : 0) : 0;
    const int tile_end = sp.bad ? 0 : sp.past + (a.causal ? (r_end - 1) / a.group + 1 : 0);
    const int all = r_end - r0 == C::M && !sp.bad ? sp.past + (a.causal ? r0 / a.group + 1 : 0) : 0;      // keys every column sees
    int k0, k1;
    split_range(a, split, tile_end, KT, &k0, &k1);

    Pages pg;
    pg.row = a.table + sp.seq * a.table_stride; pg.n_pages = a.n_pages; pg.bad = false; pg.base = 0; pg.ids = 0;
    const int64_t kp = a.kc[0] * (int)sizeof(elem_t), ks = a.kc[2] * (int)sizeof(elem_t);
    const int64_t vp = a.vc[0] * (int)sizeof(elem_t), vs = a.vc[2] * (int)sizeof(elem_t);
    const char* kbase = reinterpret_cast<const char*>(a.k) + kvh * a.kc[1] * (int)sizeof(elem_t);
    const char* vbase = reinterpret_cast<const char*>(a.v) + kvh * a.vc[1] * (int)sizeof(elem_t);
    char* ring = smem + w * 2 * C::STAGE;
    const int first = k0 + w * KT;
    auto fetch = [&](int key0, int buf) {
        if (((min(key0 + KT, k1) - 1) >> a.page_shift) >= pg.base + 64) pg.load(key0 >> a.page_shift, (k1 - 1) >> a.page_shift);
        char* lds = ring + buf * C::STAGE;
        dma_rows<P, D, KT>(kbase, kp, ks, pg, a.page_shift, key0, 0, k1, lds);
        dma_rows<P, D, KT>(vbase, vp, vs, pg, a.page_shift, key0, 0, k1, lds + C::TILE);
    };

    u32x4 qf[NKS];
    {
        const elem_t* qp = reinterpret_cast<const elem_t*>(a.q) + token * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int t = 0; t < NKS; ++t) qf[t] = *reinterpret_cast<const u32x4*>(qp + (4 * t + g) * EPL);
    }
    f32x4 o[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d) o[d] = {0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;
    if (first < k1) pg.load(first >> a.page_shift, (k1 - 1) >> a.page_shift);
#pragma unroll
    for (int t = 0; t < NKS; ++t) asm volatile("" : "+v"(qf[t]));

    if (first < k1) fetch(first, 0);
    int buf = 0;
    for (int key0 = first; key0 < k1; key0 += NW * KT, buf ^= 1) {
        wait_lds();                          // the other buffer's reads are over
        if (key0 + NW * KT < k1) { fetch(key0 + NW * KT, buf ^ 1); wait_vm<C::DMA>(); }
        else wait_vm<0>();
        const char* kt = ring + buf * C::STAGE;
        const char* vt = kt + C::TILE;
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[b] = {0, 0, 0, 0};
            const int kr = b * 16 + l15;
#pragma unroll
            for (int t = 0; t < NKS; ++t) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + kr * RB + (((4 * t + g) ^ (kr & 7)) << 4));
                if constexpr (P::IS_BF16) {
                    s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[t]), s[b], 0, 0, 0);
                } else {
                    const f32x4 kx = __builtin_bit_cast(f32x4, kf), qx = __builtin_bit_cast(f32x4, qf[t]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[j], qx[j], s[b], 0, 0, 0);
                }
            }
        }
        const uint64_t alive = tile_mask(a, sp.seq, key0);
        if (key0 + KT > all || (uint32_t)alive != ~0u) {
            const int left = lim - key0;
            const uint32_t see = (left >= 32 ? ~0u : (left <= 0 ? 0u : (1u << left) - 1)) & (uint32_t)alive;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[b][r] = (see >> (16 * b + 4 * g + r)) & 1 ? s[b][r] : -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = swap_max32(swap_max16(mx)) * a.scale_log2;
        if (__any(mx > m + 8.f)) {           // as in the tile kernel
            const float mn = fmaxf(m, mx), al = mn == -INFINITY ? 1.f : exp2_hw(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < NDB; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[d][r] *= al;
        }
        const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[b][r] = exp2_hw(fmaf(s[b][r], a.scale_log2, -mu));
                l += s[b][r];
            }
        if constexpr (P::IS_BF16) {
#if defined(__HIP_DEVICE_COMPILE__)
            // slots 0 .. 3 of group g: keys 4 g .. of the lower 16, slots 4 .. 7: of the upper 16
            bf16x8 pf;
#pragma unroll
            for (int j = 0; j < 8; ++j) pf[j] = (__bf16)s[j >> 2][j & 3];
            const int vrow = 4 * g + (l15 >> 2);
            const unsigned va = lds_address(vt) + vrow * RB + ((((l15 >> 1) & 1) ^ (vrow & 7)) << 4) + (l15 & 1) * 8;
            unrolled<0, NDB / 4>([&](auto Q) {
                constexpr int q4 = decltype(Q)::value;               // feature blocks 4 q4 .. (32 bytes each, swizzled within 128)
                s16x8 vf[4];
                read_v4<q4 * 128, q4 * 128 + 16 * RB>(va, va ^ 32, va ^ 64, va ^ 96, vf);
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    o[4 * q4 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vf[d]), pf, o[4 * q4 + d], 0, 0, 0);
            });
#endif
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int vr = 16 * b + 4 * g + r;
#pragma unroll
                    for (int d = 0; d < NDB; ++d) {
                        const int f = d * 16 + l15;
                        const float vx = *reinterpret_cast<const float*>(vt + vr * RB + (((f >> 2) ^ (vr & 7)) << 4) + (f & 3) * 4);
                        o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx, s[b][r], o[d], 0, 0, 0);
                    }
                }
        }
    }
    wait_vm<0>();
    if (pg.bad && lane == 0) atomicOr(a.status, PAGED_BAD_PAGE);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (pg.bad || sp.bad) l = NAN;

    // join the waves: outputs [NW][16][D] (16-byte pieces XOR-swizzled by the row) and maxima, sums [NW][16] in the place of the tiles
    __syncthreads();
    float* sm = reinterpret_cast<float*>(smem) + NW * 16 * D;
#pragma unroll
    for (int d = 0; d < NDB; ++d)
        *reinterpret_cast<f32x4*>(smem + ((w * 16 + l15) * D + (((d * 4 + g) ^ (l15 & 7)) << 2)) * 4) = o[d];
    if (g == 0) { sm[w * 16 + l15] = m; sm[(NW + w) * 16 + l15] = l; }
    __syncthreads();
    constexpr int PPR = D / 4;               // pieces per row
    for (int i = threadIdx.x; i < 16 * PPR; i += NW * 64) {
        const int q = i / PPR, piece = i % PPR, rr = r0 + q;
        const bool on = rr < r_end;
        float top = sm[q], f[NW], sum = 0.f;
#pragma unroll
        for (int v = 1; v < NW; ++v) top = fmaxf(top, sm[v * 16 + q]);
        const float mu = top == -INFINITY ? 0.f : top;
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < NW; ++v) {
            f[v] = exp2_hw(sm[v * 16 + q] - mu);
            sum = fmaf(sm[(NW + v) * 16 + q], f[v], sum);
            const f32x4 x = *reinterpret_cast<const f32x4*>(smem + ((v * 16 + q) * D + ((piece ^ (q & 7)) << 2)) * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = fmaf(x[j], f[v], acc[j]);
        }
        const bool ruined = sum != sum && (pg.bad || sp.bad);
        const float z = fmaf(acc[0], 0.f, fmaf(acc[1], 0.f, fmaf(acc[2], 0.f, fmaf(acc[3], 0.f, sum * 0.f))));
        const int tk = on ? rr / a.group : 0, hd = kvh * a.group + (on ? rr - tk * a.group : 0);
        const int64_t t64 = sp.first + tk;
        if (on) {
            if (a.splits > 1) {
                const int64_t orow = t64 * a.q_heads + hd;
                *reinterpret_cast<f32x4*>(part_out<D>(a, split, orow) + piece * 4) = acc;
                if (piece == 0) { float* ml = part_ml<D>(a, split, orow); ml[0] = top; ml[1] = sum; }
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                store4<P>(reinterpret_cast<elem_t*>(a.out) + t64 * a.os[0] + hd * a.os[1] + piece * 4, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
            }
        }
        // rows of this wave's pieces whose result is not finite (64 lanes hold 64 / PPR rows), again and alone
        uint64_t odds = __ballot(on && !ruined && !(z == 0.f));
        while (odds) {
            const int src = __builtin_ctzll(odds), rw = (i - lane + src) / PPR;
            const uint64_t same = PPR == 64 ? ~0ull : (((1ull << PPR) - 1) << (src / PPR * PPR));
            odds &= ~same;
            const int ar = r0 + uniform(rw), at = ar / a.group;
            store_row_alone<P, D>(a, sp.seq, kvh, sp.first + at, kvh * a.group + ar - at * a.group, split, k0,
                                  min(k1, sp.past + (a.causal ? at + 1 : 0)));
        }
    }
}

// =================================================================================================================================
// Joins the partial results of a split launch: W waves per (token, query head).  The (maximum, sum) pairs of all splits (at most 64) sit
// one per lane; 16-byte pieces of the partial outputs are then read by 64 / (D / 4) splits at a time and wave.
// =================================================================================================================================
template <typename P, int D, int W>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnArgs a) {
    typedef typename P::elem_t elem_t;
    constexpr int LPR = D / 4, SPW = 64 / LPR;          // lanes per row, splits per wave
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, piece = lane % LPR, sub = lane / LPR;
    const int64_t row = (int64_t)blockIdx.x * (4 / W) + (W == 1 ? w : 0);
    if (row >= (int64_t)a.tokens * a.q_heads) return;
    const int64_t token = row / a.q_heads;
    const int head = (int)(row - token * a.q_heads);
    if (a.starts) {          // rows of no sequence (padding, bad starts) have no partial results
        int lo = 0, hi = a.n_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.starts[mid] <= token) lo = mid; else hi = mid;
        }
        if (a.starts[lo] < 0 || a.starts[lo + 1] > a.tokens || token < a.starts[lo] || token >= a.starts[lo + 1]) return;
    }
    float m = -INFINITY, l = 0.f;
    if (lane < a.splits) { const float2 ml = *reinterpret_cast<const float2*>(part_ml<D>(a, lane, row)); m = ml.x; l = ml.y; }
    const float top = wave_max(m), f = l == 0.f ? 0.f : exp2_hw(m - (top == -INFINITY ? 0.f : top));
    const float sum = wave_sum(l * f);
    f32x4 acc = {0, 0, 0, 0};
    for (int s0 = W == 1 ? 0 : w * SPW; s0 < a.splits; s0 += W * SPW) {
        const int s = s0 + sub;
        const float fs = __shfl(f, s & 63);
        if (s < a.splits && fs != 0.f) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(part_out<D>(a, s, row) + piece * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(x[i], fs, acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (SPW >= 4) acc[i] += __shfl_xor(acc[i], 16);
        acc[i] += __shfl_xor(acc[i], 32);
    }
    if constexpr (W > 1) {
        __shared__ f32x4 other[W][LPR];
        if (sub == 0) other[w][piece] = acc;
        __syncthreads();
        if (w != 0) return;
#pragma unroll
        for (int i = 1; i < W; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += other[i][piece][j];
    }
    if (sub == 0) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        store4<P>(reinterpret_cast<elem_t*>(a.out) + token * a.os[0] + head * a.os[1] + piece * 4, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
}

struct Plan { bool step; int tiles, splits; };

// max_new tokens a sequence at most (0: not known) make at most max_new * group rows per key head: up to 16 take the step kernel.
// Workgroups are few where rows are few: the keys are then shared out over `splits` workgroups.  Two workgroups fit a CU; a share has
// at least 256 keys (its partial result costs a row of f32 outputs twice).
Plan make_plan(const PagedAttnArgs& a, int max_new) {
    Plan p;
    const int64_t most = (a.starts ? max_new : 1) * (int64_t)a.group;       // 0: not known
    p.step = most > 0 && most <= 16;
    const int M = p.step ? 16 : 128;
    const int64_t ub = a.starts ? (int64_t)a.tokens * a.group / M + a.n_seqs : (int64_t)a.n_seqs * ((a.group + M - 1) / M);
    p.tiles = (int)ub;
    int64_t est = most > 0 ? (int64_t)a.n_seqs * ((most + M - 1) / M) : ub;
    if (est > ub) est = ub;
    const int64_t groups = est * a.kv_heads, keys = (int64_t)a.max_pages << a.page_shift;
    int64_t s = 512 / (groups > 0 ? groups : 1);
    if (s > keys / 256) s = keys / 256;
    if (s > 64) s = 64;
    p.splits = s < 1 ? 1 : (int)s;
    return p;
}

template <typename P, int D>
hipError_t launch(PagedAttnArgs a, int max_new, hipStream_t s) {
    const Plan p = make_plan(a, max_new);
    a.splits = p.splits;
    const int64_t rows = (int64_t)a.tokens * a.q_heads, groups = (int64_t)p.tiles * p.splits * a.kv_heads;
    if (groups > 0x7fffffff || rows > 0x7fffffff) return hipErrorInvalidValue;
    if (p.step) hipLaunchKernelGGL((paged_attn_step_kernel<P, D>), dim3((unsigned)groups), dim3(StepCfg<P, D>::NW * 64), 0, s, a);
    else hipLaunchKernelGGL((paged_attn_tile_kernel<P, D>), dim3((unsigned)groups), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    if (p.splits > 8) hipLaunchKernelGGL((paged_attn_join_kernel<P, D, 4>), dim3((unsigned)rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((paged_attn_join_kernel<P, D, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

int64_t paged_attn_workspace(const PagedAttnArgs& a, int max_new, int head_dim, int) {
    const Plan p = make_plan(a, max_new);
    return p.splits == 1 ? 0 : (int64_t)p.splits * a.tokens * a.q_heads * (head_dim + 2) * (int64_t)sizeof(float);
}

hipError_t paged_attn_launch(const PagedAttnArgs& a, int max_new, int head_dim, int dtype, hipStream_t s) {
    if (dtype == PTTS_BF16) return head_dim == 64 ? launch<PBF16, 64>(a, max_new, s) : launch<PBF16, 128>(a, max_new, s);
    return head_dim == 64 ? launch<PF32, 64>(a, max_new, s) : launch<PF32, 128>(a, max_new, s);
}

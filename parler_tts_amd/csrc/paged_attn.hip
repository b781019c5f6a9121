// Attention of new tokens over a paged KV cache: o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j a query may see.
//
// Three kernels (chunks in bf16, chunks in f32, few rows) make ONE pass over the keys with the running maximum and sum of the softmax, and
// all hold the scores TRANSPOSED:
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

template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename P> __device__ __forceinline__ void load16(const typename P::elem_t* p, float* f);
template <> __device__ __forceinline__ void load16<PBF16>(const uint16_t* p, float* f) {
    const u32x4 r = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = r[i];
        f[2 * i] = __builtin_bit_cast(float, w << 16);
        f[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
    }
}
template <> __device__ __forceinline__ void load16<PF32>(const float* p, float* f) {
    const f32x4 r = *reinterpret_cast<const f32x4*>(p);
    f[0] = r[0]; f[1] = r[1]; f[2] = r[2]; f[3] = r[3];
}

__device__ __forceinline__ float swap_max32(float x) {      // maximum over lanes l and l ^ 32
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
#else
    return x;
#endif
}
__device__ __forceinline__ float swap_max16(float x) {      // maximum over lanes l and l ^ 16
#if defined(__HIP_DEVICE_COMPILE__)
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    return fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
#else
    return x;
#endif
}
__device__ __forceinline__ float exp2_hw(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_exp2f(x);
#else
    return x;
#endif
}
// Transposing read of V: 16 lanes take a block of 4 keys x 16 features (each lane 4 features of one key), lane i ends with feature i of
// the 4 keys.  The two halves of a matrix step's operand.
__device__ __forceinline__ bf16x8 read_v(unsigned lo, unsigned hi) {
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)lo);
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)hi);
    v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
#endif
    return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ u32x4 read_lds(unsigned p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
    return *(lds_u32x4*)(uintptr_t)p;
#else
    return {0, 0, 0, 0};
#endif
}
__device__ __forceinline__ float read_lds_f32(unsigned p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) const float lds_f32;
    return *(lds_f32*)(uintptr_t)p;
#else
    return 0.f;
#endif
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
#else
    return 0;
#endif
}
// Chunk c (16 bytes) of row r stands at chunk c ^ swizzle(r) of the row's LDS image.  16 lanes that read one chunk of 16 rows (K), and 32
// lanes that read 4 x 64 or 8 x 32 bytes of neighbouring rows (V), then meet in no bank: 64 banks hold 16 chunks, and the low bits of the
// row move the high bits of the chunk (bf16) or, for f32 (V: 4 rows 4 apart, 64 bytes each), bits 2 and 3 do.
template <int RB, bool BF16> __device__ __forceinline__ unsigned swizzle(unsigned r) {
    if (RB == 128) return ((r >> 1 & 1) << 2) | ((r >> 2 & 1) << 1) | (r >> 3 & 1);
    return BF16 ? ((r & 3) << 2) | ((r >> 2 & 1) << 1) | (r >> 3 & 1) : r & 15;
}
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_add(int x) {      // x plus the moved x, where there is one
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ unsigned wave_max_u32(unsigned x) {
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xf, 0xf, true));
    x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xf, 0xf, true));
    const unsigned a = max((unsigned)__builtin_amdgcn_readlane((int)x, 0), (unsigned)__builtin_amdgcn_readlane((int)x, 16));
    const unsigned b = max((unsigned)__builtin_amdgcn_readlane((int)x, 32), (unsigned)__builtin_amdgcn_readlane((int)x, 48));
    return max(a, b);
}
__device__ __forceinline__ int scan_add(int x) {        // sum over the lanes up to this one
    x = dpp_add<0x111, 0xf>(x); x = dpp_add<0x112, 0xf>(x); x = dpp_add<0x114, 0xf>(x); x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);                         // lane 15 of a row of 16 into the next row
    return dpp_add<0x143, 0xc>(x);                      // lane 31 into the upper half
}
template <int I, int N, typename F> __device__ __forceinline__ void each(F&& f) {      // f(0), f(1), ... with the number as a type
    if constexpr (I < N) { f(std::integral_constant<int, I>()); each<I + 1, N>(f); }
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ---- which rows and keys a workgroup takes -------------------------------------------------------------------------------------
// A launch's items are (tile of M rows of a sequence, share of its keys, key head).  Their numbers come from the lengths on the device:
// every wave sums the sequences' tiles up for itself, 64 sequences at a time, all lengths in one round trip.  Behind MANY_SEQS sequences one
// workgroup does that once, in a launch in front (4 us), and leaves its groups of 64 and their first items in the workspace for a search; one
// token each without shares needs neither.  Items are numbered without
// holes (with holes between the sequences the dispatcher put all work of equal chunks on half of the CUs).
// Keys are shared out only where that evens the load: a tile whose keys exceed what one of SLOTS workgroups would get of everything (by the
// factor LAG) is cut into shares of that size, at least min_share keys each (a share costs its rows' f32 partial results, written and read
// once more).  SLOTS are two workgroups on each of 256 CUs.  Counting the third that head dim 64 has room for made finer shares and lost
// more at their ends than it won: prompts of up to 7770 over 2324 keys, 2 heads of 64: 68 us, with two 58; a batch of 24 chunks 81, 76.
constexpr int SLOTS = 512, MAX_SPLITS = 256;
constexpr int MANY_SEQS = 128;
constexpr float TILE_LAG = 2.f, STEP_LAG = 2.f;

// The schedule of a launch in front, in ints: first item of every group of 64 sequences and their number behind them, the same of tiles, and the
// sequences of the groups in the order of their items: index, first token, new tokens, cached ones.
__host__ __device__ inline int sched_groups(int n_seqs) { return (n_seqs + 63) / 64; }
__host__ __device__ inline int64_t sched_ints(int n_seqs) { return 2 * ((int64_t)sched_groups(n_seqs) + 1) + 256 * (int64_t)sched_groups(n_seqs); }

struct Item {
    int seq, first, n, past;    // the sequence, its first token, its new tokens, its cached ones
    int tile, split, splits;    // of the sequence's tiles; share of the keys; shares of this tile
    int end, k0, k1;            // keys any of the tile's rows sees; this item's keys
    bool bad;                   // the length leads behind the row of the page table: every row becomes NaN
};

// SORTED (and by_length): of every 64 sequences the longest first, so that what starts last is short.
template <int M, int KT, bool SORTED> struct Schedule {
    int seq, first, n, past;    // this lane's sequence of the current 64
    int base;                   // number of the first of these
    int sum, own;               // (tile, share) pairs of the lane's sequence, and of all up to it
    int share;                  // tiles of KT keys of a share (of all keys: not cut)
    int items;                  // pairs of the batch
    bool by_length = true;      // sort at all (few items have a CU each, in any order)

    // Starts that descend can give the same rows to any number of sequences: sums over groups stay at the largest number instead of wrapping,
    // so that they ascend whatever starts say.  (64 sequences cannot wrap: each has 2^25 - 1024 tiles at most, see make_plan.)
    static __host__ __device__ __forceinline__ int add_items(int x, int y) { return x > 0x7fffffff - y ? 0x7fffffff : x + y; }
    __device__ __forceinline__ int launch_items(const PagedAttnArgs& a) const { return (int)min((int64_t)items * a.kv_heads, (int64_t)0x7fffffff); }

    __device__ __forceinline__ void load(const PagedAttnArgs& a, int i0) {
        const int lane = threadIdx.x & 63, i = min(i0 + lane, a.n_seqs - 1);
        base = i0;
        seq = i;
        if (a.starts) {
            first = a.starts[i];
            const int end = a.starts[i + 1];
            n = first >= 0 && end > first && end <= a.tokens ? end - first : 0;      // starts that are wrong own no rows
        } else { first = i; n = 1; }
        past = a.past[i];
        if (i0 + lane >= a.n_seqs) n = 0;
    }
    __device__ __forceinline__ void load_group(const PagedAttnArgs& a, int g) {      // of the launch in front
        const int lane = threadIdx.x & 63, groups = sched_groups(a.n_seqs);
        const int* e = a.sched + 2 * (groups + 1) + (int64_t)g * 256 + lane;
        base = g * 64;
        seq = e[0]; first = e[64]; n = e[128]; past = e[192];
    }
    // group of item (or tile) t among the first items `from`; t becomes its number within the group
    static __device__ __forceinline__ int find_group(const int* from, int groups, int* t) {
        const int lane = threadIdx.x & 63;
        int lo = 0, len = groups;
        for (;;) {
            const int step = (len + 63) / 64, i = min(lane * step, len - 1), v = from[lo + i];
            const int k = uniform((int)__popcll(__ballot(lane * step < len && v <= *t)) - 1);
            lo += k * step;
            if (step == 1) { *t -= __builtin_amdgcn_readlane(v, k); return lo; }
            len = min(step, len - k * step);
        }
    }
    static __device__ __forceinline__ bool bad_length(const PagedAttnArgs& a, int np, int pp) {
        return pp < 0 || (int64_t)pp + (a.causal ? np : 0) > ((int64_t)a.max_pages << a.page_shift);
    }
    __device__ __forceinline__ int row_tiles(const PagedAttnArgs& a) const { return (n * a.group + M - 1) / M; }
    __device__ __forceinline__ int key_tiles(const PagedAttnArgs& a) const {
        return bad_length(a, n, past) ? 1 : (past + (a.causal ? n : 0) + KT - 1) / KT;
    }
    __device__ __forceinline__ int shares(int kt) const { return kt <= share ? 1 : (kt + share - 1) / share; }
    __device__ __forceinline__ void count(const PagedAttnArgs& a) {
        own = row_tiles(a);
        if (a.splits > 1) own *= shares(key_tiles(a));
        sum = scan_add(own);
    }
    __device__ __forceinline__ void sort(const PagedAttnArgs& a) {
        const int lane = threadIdx.x & 63, here = min(a.n_seqs - base, 64), key = n > 0 ? key_tiles(a) : 0;
        if (here <= 1) return;
        // eight classes of length, longest first, in order within a class
        const float top = (float)wave_max_u32((unsigned)key);
        const int cls = 7 - min((int)((float)key * (8.f / (top + 1.f))), 7);
        int rank = 0, before = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const uint64_t m = __ballot(lane < here && cls == c);
            const int mine = before + (int)__popcll(m & ((1ull << lane) - 1));
            rank = cls == c ? mine : rank;
            before += (int)__popcll(m);
        }
        if (lane >= here) rank = lane;
        seq = __builtin_amdgcn_ds_permute(rank << 2, seq);
        first = __builtin_amdgcn_ds_permute(rank << 2, first);
        n = __builtin_amdgcn_ds_permute(rank << 2, n);
        past = __builtin_amdgcn_ds_permute(rank << 2, past);
    }
    // what the lane's sequence adds to the work of the batch (tiles of rows times the tiles of keys they see on average), and its keys
    __device__ __forceinline__ void weigh(const PagedAttnArgs& a, float* work, int* most) const {
        const int rt = row_tiles(a), kt = key_tiles(a);
        *work += (float)rt * (float)(a.causal ? max(kt - n / (2 * KT), 1) : kt);
        *most = max(*most, rt > 0 ? kt : 0);
    }
    // share for the whole batch: a slot's part of everything; a little more where the shares' ends would need a second round of a few workgroups
    __device__ __forceinline__ void choose_share(const PagedAttnArgs& a, float mean, int most, float lag, bool one_group) {
        share = 0x3fffffff;
        if ((float)most <= lag * mean) return;
        const int least = max(a.min_share / KT, (most + a.splits - 1) / a.splits);
        const int front = a.causal ? min((past + KT) / KT, key_tiles(a)) : key_tiles(a);       // tiles the first row sees
        for (int step = 4; step <= 8; ++step) {
            share = max((int)ceilf(mean * 0.25f * (float)step), least);
            if (!one_group || step == 8) break;
            const int all = uniform(__builtin_amdgcn_readlane(scan_add(row_tiles(a) * (shares(key_tiles(a)) + shares(front))), 63));
            if (all * a.kv_heads <= 2 * SLOTS) break;
        }
        share = uniform(share);
    }
    // share for the whole batch, the number of items
    __device__ __forceinline__ void plan(const PagedAttnArgs& a, float lag) {
        share = 0x3fffffff;
        load(a, 0);
        if (a.splits > 1) {
            float work = 0.f;
            int most = 0;
            for (int i0 = 0;;) {
                weigh(a, &work, &most);
                i0 += 64;
                if (i0 >= a.n_seqs) break;
                load(a, i0);
            }
            choose_share(a, wave_sum(work) * (float)a.kv_heads / SLOTS, (int)wave_max_u32((unsigned)most), lag, a.n_seqs <= 64);
            if (a.n_seqs > 64) load(a, 0);
        }
        number(a);
    }
    __device__ __forceinline__ void number(const PagedAttnArgs& a) {
        items = 0;
        for (int i0 = 0;;) {
            if (SORTED && by_length) sort(a);
            count(a);
            items = add_items(items, __builtin_amdgcn_readlane(sum, 63));
            i0 += 64;
            if (i0 >= a.n_seqs) break;
            load(a, i0);
        }
    }
    // item t < items
    __device__ __forceinline__ void find(const PagedAttnArgs& a, int t, Item* it, const int* from) {
        if (a.sched) {
            const int groups = sched_groups(a.n_seqs);
            load_group(a, find_group(from, groups, &t));
            count(a);
        } else if (a.n_seqs > 64) {
            load(a, 0);
            for (;;) {
                if (SORTED && by_length) sort(a);
                count(a);
                const int here = __builtin_amdgcn_readlane(sum, 63);
                if (t < here || base + 64 >= a.n_seqs) break;
                t -= here;
                load(a, base + 64);
            }
        }
        const int sel = uniform(min((int)__popcll(__ballot(sum <= t)), 63));
        it->seq = __builtin_amdgcn_readlane(seq, sel);
        it->first = __builtin_amdgcn_readlane(first, sel);
        it->n = __builtin_amdgcn_readlane(n, sel);
        it->past = __builtin_amdgcn_readlane(past, sel);
        t -= __builtin_amdgcn_readlane(sum - own, sel);
        place(a, t, it);
    }
    // tile and share of the sequence's pair t
    __device__ __forceinline__ void place(const PagedAttnArgs& a, int t, Item* it) const {
        const int tiles = (it->n * a.group + M - 1) / M;
        it->bad = bad_length(a, it->n, it->past);
        if (it->bad) it->past = 0;
        it->split = 0;
        if (a.splits > 1) {
            const int cuts = it->bad ? 1 : shares((it->past + (a.causal ? it->n : 0) + KT - 1) / KT);
            if (cuts > 1) { const int q = t / cuts; it->split = t - q * cuts; t = q; }
        }
        it->tile = tiles - 1 - t;                      // the rows that see most first
        it->end = it->bad ? 0 : it->past;
        if (a.causal && !it->bad) it->end += int_div(min((it->tile + 1) * M, it->n * a.group) - 1, a.by_group) + 1;
        const int kt = (it->end + KT - 1) / KT;
        it->splits = a.splits > 1 ? shares(kt) : 1;
        it->k0 = 0;
        it->k1 = it->end;
        // a share is shorter than the keys it is cut from; the end of the last one may lie past 2^31
        if (it->splits > 1) { it->k0 = min(it->split * share * KT, it->end); it->k1 = it->k0 + min(share * KT, it->end - it->k0); }
    }
};

// The arguments once more, for what stands behind a main loop: read there, instead of kept in scalar registers through it.
__device__ __forceinline__ PagedAttnArgs arguments_again() {
    PagedAttnArgs z = {};
#if defined(__HIP_DEVICE_COMPILE__)
    uintptr_t p = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    typedef const __attribute__((address_space(4))) PagedAttnArgs kernarg;
    __builtin_memcpy(&z, (kernarg*)p, sizeof(z));
#endif
    return z;
}

template <typename S> __device__ __forceinline__ void begin(const PagedAttnArgs& a, S& sched, float lag) {
    if (blockIdx.x == 0 && a.starts) check_starts(a.starts, a.n_seqs, a.tokens, a.status);
    if (a.sched) {
        sched.share = a.splits > 1 ? __builtin_bit_cast(int, a.part[0]) : 0x3fffffff;
        sched.items = a.sched[sched_groups(a.n_seqs)];
        return;
    }
    sched.plan(a, lag);
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.splits > 1) a.part[0] = __builtin_bit_cast(float, sched.share);
}

template <int M, int KT, bool SORTED>
__global__ __launch_bounds__(1024) void paged_attn_schedule_kernel(PagedAttnArgs a, float lag) {
    __shared__ float works[16];
    __shared__ int mosts[16], items[16], tiles[16];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), groups = sched_groups(a.n_seqs);
    int *item0 = a.sched, *tile0 = a.sched + groups + 1, *entry = a.sched + 2 * (groups + 1);
    Schedule<M, KT, SORTED> sc;
    sc.share = 0x3fffffff;
    if (a.splits > 1) {
        float work = 0.f;
        int most = 0;
        for (int g = w; g < groups; g += 16) {
            sc.load(a, g * 64);
            sc.weigh(a, &work, &most);
        }
        work = wave_sum(work);
        most = (int)wave_max_u32((unsigned)most);
        if (lane == 0) { works[w] = work; mosts[w] = most; }
        __syncthreads();
        work = 0.f;
        for (int i = 0; i < 16; ++i) { work += works[i]; most = max(most, mosts[i]); }
        sc.load(a, 0);
        sc.choose_share(a, work * (float)a.kv_heads / SLOTS, most, lag, false);
        if (threadIdx.x == 0) a.part[0] = __builtin_bit_cast(float, sc.share);
    }
    int item_at = 0, tile_at = 0;
    for (int g0 = 0; g0 < groups; g0 += 16) {
        const int g = g0 + w;
        int mine = 0, rows = 0;
        if (g < groups) {
            sc.load(a, g * 64);
            if (SORTED) sc.sort(a);
            sc.count(a);
            mine = __builtin_amdgcn_readlane(sc.sum, 63);
            rows = __builtin_amdgcn_readlane(scan_add(sc.row_tiles(a)), 63);
            int* e = entry + (int64_t)g * 256 + lane;
            e[0] = sc.seq; e[64] = sc.first; e[128] = sc.n; e[192] = sc.past;
        }
        if (lane == 0) { items[w] = mine; tiles[w] = rows; }
        __syncthreads();
        int before = item_at, tiles_before = tile_at;
        for (int i = 0; i < 16; ++i) {
            if (i == w && g < groups && lane == 0) { item0[g] = before; tile0[g] = tiles_before; }
            before = sc.add_items(before, items[i]);
            tiles_before = sc.add_items(tiles_before, tiles[i]);
        }
        item_at = before;
        tile_at = tiles_before;
        __syncthreads();
    }
    if (threadIdx.x == 0) { item0[groups] = item_at; tile0[groups] = tile_at; }
}

// ---- page ids of the keys ahead, one per lane ---------------------------------------------------------------------------------
struct Pages {
    const int* row;
    int base, ids, n_pages;     // lane l holds the id of page base + l
    bool bad;
    __device__ __forceinline__ void load(int first, int last) {       // pages first .. (at most 64), none behind `last`
        base = first;
        const int i = first + (int)(threadIdx.x & 63);
        ids = row[min(i, last)];
        const bool wrong = (unsigned)ids >= (unsigned)n_pages;
        bad = bad || __any(wrong);
        if (wrong) ids = 0;
    }
    __device__ __forceinline__ int get(int page) const { return __builtin_amdgcn_readlane(ids, page - base); }
};

// ---- ROWS rows of K or V on their way to LDS, by one wave ------------------------------------------------------------------------
// Rows at or behind `end` are read from the last row in front of it: what lies there is seen by nobody, and may be anything.  A wave
// instruction moves RPI rows, which share a page (pages hold 16 tokens or more); its address is a scalar base and a 32-bit lane offset
// (slot strides are below 2^27 bytes).  The LDS-DMA is written out: behind its builtin hipcc drains every transfer in flight in front of
// the next transposing read, wherever that reads.  It has no register results; the kernels wait for it by counted vmcnt.  ONCE: rows that one
// workgroup reads, as a rule, are not kept by the caches (32 x 2000 keys, 16 heads of 64: 45.9 us, kept 51.9; where all sequences share their
// pages 29.4, 28.8; chunks, whose tiles share their keys, lose by it: 4 prompts of 1024 over 2 heads of 128 38, 35).
template <typename P, int D, bool ONCE = false> struct Rows {
    static constexpr int RB = D * (int)sizeof(typename P::elem_t), RPI = 1024 / RB, CPR = RB / 16;
    const char* base;
    int64_t page_bytes;
    int slot_bytes;
    __device__ __forceinline__ Rows(const void* cache, const int64_t* strides, int kvh) {
        constexpr int E = sizeof(typename P::elem_t);
        base = reinterpret_cast<const char*>(cache) + kvh * strides[1] * E;
        page_bytes = strides[0] * E;
        slot_bytes = (int)(strides[2] * E);
    }
    template <int ROWS> __device__ __forceinline__ void fetch(const Pages& pg, int page_shift, int key0, int row0, int end, unsigned lds) const {
        const int lane = threadIdx.x & 63, rl = lane / CPR, c = lane % CPR, mask = (1 << page_shift) - 1;
#pragma unroll
        for (int i = 0; i < ROWS / RPI; ++i) {
            const int r = row0 + i * RPI;
            const unsigned chunk = (c ^ swizzle<RB, P::IS_BF16>((r + rl) & 15)) << 4;
            if (key0 + r + RPI <= end) {
                send(base + pg.get((key0 + r) >> page_shift) * page_bytes + (int64_t)((key0 + r) & mask) * slot_bytes, rl * slot_bytes + chunk, lds + r * RB);
            } else {                                            // some of the rows, or all, are behind the end
                const int last = min(key0 + r, end - 1);
                send(base + pg.get(last >> page_shift) * page_bytes + (int64_t)(last & mask) * slot_bytes,
                     (min(key0 + r + rl, end - 1) - last) * slot_bytes + chunk, lds + r * RB);
            }
        }
    }
    static __device__ __forceinline__ void send(const char* src, unsigned off, unsigned lds) {
#if defined(__HIP_DEVICE_COMPILE__)
        const int to = __builtin_amdgcn_readfirstlane(lds);
        if constexpr (ONCE) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(to), "v"(off), "s"(src) : "memory");
        else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(src) : "memory");
#endif
    }
    // 16 rows that are all there (key a multiple of 16: they share a page), one instruction a time
    __device__ __forceinline__ const char* slice(const Pages& pg, int page_shift, int key) const {
        return base + pg.get(key >> page_shift) * page_bytes + (int64_t)(key & ((1 << page_shift) - 1)) * slot_bytes;
    }
    template <int I> __device__ __forceinline__ void fetch_one(const char*& src, unsigned lds, unsigned lane) const {
        const unsigned rl = lane / CPR, c = lane % CPR;
        send(src, rl * (unsigned)slot_bytes + ((c ^ swizzle<RB, P::IS_BF16>(I * RPI + rl)) << 4), lds + I * RPI * RB);
        src += RPI * slot_bytes;
    }
};

// keys that may be looked at at all, as bits: the key mask's bytes of the tile (lane i: key key0 + i), ones behind its last column
__device__ __forceinline__ uint64_t tile_mask(const PagedAttnArgs& a, int seq, int key0) {
    if (!a.mask || key0 >= a.mask_width) return ~0ull;
    const int j = key0 + (int)(threadIdx.x & 63);
    bool live = true;
    if (j < a.mask_width) live = a.mask[seq * a.mask_stride + j] != 0;
    return __ballot(live);
}

// ---- one query over the keys [k0, k1) it sees, by one wave (see the head of the file) ------------------------------------------
template <typename P, int D>
__device__ __forceinline__ void row_alone(const PagedAttnArgs& a, int seq, int kvh, const typename P::elem_t* q, int k0, int k1, float* m_out, float* l_out,
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
            if ((unsigned)page >= (unsigned)a.n_pages) page = 0;        // rows that meet a bad page are NaN and do not come here
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

// where the partial results of cut tiles lie: the share (for the join), outputs [split][token * q_heads + head][D], (maximum, sum) pairs
constexpr int PART_HEAD = 4;
template <int D> __device__ __forceinline__ float* part_out(const PagedAttnArgs& a, int split, int64_t row) {
    return a.part + PART_HEAD + ((int64_t)split * a.tokens * a.q_heads + row) * D;
}
template <int D> __device__ __forceinline__ float* part_ml(const PagedAttnArgs& a, int split, int64_t row) {
    const int64_t rows = (int64_t)a.tokens * a.q_heads;
    return a.part + PART_HEAD + (int64_t)a.splits * rows * D + (split * rows + row) * 2;
}

template <typename P, int D>
__device__ __forceinline__ void store_row_alone(const PagedAttnArgs& a, const Item& it, int kvh, int row) {
    typedef typename P::elem_t elem_t;
    const int lane = threadIdx.x & 63, tok = int_div(row, a.by_group), head = kvh * a.group + row - tok * a.group;
    const int64_t token = it.first + tok;
    float m, l, acc[D / 64];
    row_alone<P, D>(a, it.seq, kvh, reinterpret_cast<const elem_t*>(a.q) + token * a.qs[0] + head * a.qs[1], it.k0,
                    min(it.k1, it.past + (a.causal ? tok + 1 : 0)), &m, &l, acc);
    const int64_t orow = token * a.q_heads + head;
#pragma unroll
    for (int r = 0; r < D / 64; ++r) {
        if (it.splits > 1) part_out<D>(a, it.split, orow)[r * 64 + lane] = acc[r];
        else (reinterpret_cast<elem_t*>(a.out) + token * a.os[0] + head * a.os[1])[r * 64 + lane] = to_elem<P>(l == 0.f ? 0.f : acc[r] / l);
    }
    if (it.splits > 1 && lane == 0) { float* ml = part_ml<D>(a, it.split, orow); ml[0] = m; ml[1] = l; }
}

template <typename P> __device__ __forceinline__ void store4(typename P::elem_t* p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<PBF16>(uint16_t* p, float a, float b, float c, float d) {
    typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
    const bf16x4 v = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
    *reinterpret_cast<bf16x4*>(p) = v;
}
template <> __device__ __forceinline__ void store4<PF32>(float* p, float a, float b, float c, float d) {
    const f32x4 v = {a, b, c, d};
    *reinterpret_cast<f32x4*>(p) = v;
}

// =================================================================================================================================
// Chunks in bf16: a workgroup owns 128 rows (32 per wave), the keys pass in tiles of 64.
// One wave alone keeps the matrix unit busy: the products of the NEXT tile's scores go out between the exponentials of this one, the
// products with V between the additions of its weights and the maximum of the next scores.  (With a tile's steps one after the other, two
// waves per SIMD spent 2300 cycles on 1024 of matrix work at D = 128; they overlap their phases only by chance.)  K runs one tile ahead of
// V, so each has a ring of its own: iteration i sends for K(i + NB) and V(i + NB - 1) into the buffers that iteration i - 1 left, one
// instruction between two products.  Iterations with less in front of the end are written out apart: they wait for all in flight.
// =================================================================================================================================
// Three workgroups on a CU at head dim 64 (48 KiB, 168 registers: four fragments read ahead), two at 128 (64 KiB, 248 registers).
// Bound: at head dim 128 the matrix unit, under a power limit (prompt of 8191 tokens, 16 heads over 4: 279 - 294 us a call in a stream of
// calls, 935 - 985 TFLOP/s; profiled, by the run's median, 305 - 331 us, 830 - 900, its shortest launches 292 - 299; the library's product of 8192^3
// reaches 1162 - 1202); at 64 the vector unit beside it (per tile and wave 32 exponentials, 130 other
// operations, 16 products: 8191 tokens, 16 heads: 182 us, 755 TFLOP/s; with two workgroups on a CU 199).  Short chunks: a workgroup's start
// (lengths, page ids and first tiles are three dependent trips to memory, 5.6 us) and the unequal lengths.
// Tried and left: the sum of the weights by the matrix unit or by two-element dot products (no change); 64 rows a wave (registers).
template <int D> struct ChunkCfg {
    static constexpr int M = 128, NW = 4, KT = 64, RB = D * 2;
    static constexpr int TILE = KT * RB;
    static constexpr int NB = D == 64 ? 3 : 2;
    static constexpr int LDS = 2 * NB * TILE;                  // [K ring][V ring]
    static constexpr int DMA = TILE / NW / 1024;               // LDS-DMA instructions per wave and tile of K or of V
};

template <int D>
__global__ __launch_bounds__(256, (D == 64 ? 3 : 2)) void paged_attn_chunk_kernel(PagedAttnArgs a) {
    typedef PBF16 P;
    typedef uint16_t elem_t;
    typedef ChunkCfg<D> C;
    constexpr int KT = C::KT, RB = C::RB, NB = C::NB, NKS = D / 16, NDB = D / 32, NQ = 2 * NKS, NP = 4 * NDB;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), l31 = lane & 31, h = lane >> 5;

    Schedule<C::M, KT, true> sched;
    begin(a, sched, TILE_LAG);
    const int all = sched.launch_items(a);
    int item = blockIdx.x;
    if (item >= all) return;
    // up to two on a CU: the longest item beside the shortest (4 prompts of 1024, 16 heads of 128 over 2: 34 us, in order 41)
    if (all > SLOTS / 2 && all <= SLOTS && item >= SLOTS / 2) item = all - 1 - (item - SLOTS / 2);
    // consecutive workgroups go to consecutive XCDs: with the key head innermost, an XCD's L2 holds few heads' pages
    const int at = int_div(item, a.by_kv_heads), kvh = item - at * a.kv_heads;
    Item it;
    sched.find(a, at, &it, a.sched);
    if (it.split >= it.splits) return;
    const int k0 = it.k0, k1 = it.k1, r0 = it.tile * C::M, r_end = min(r0 + C::M, it.n * a.group);
    int row = r0 + w * 32 + l31;                               // this lane's query
    int lim;                                                   // keys 0 .. lim - 1 are seen
    const int wr0 = r0 + w * 32, wr1 = min(wr0 + 32, r_end);                            // rows of this wave: [wr0, wr1)
    const bool some = wr0 < wr1 && !it.bad;
    const int w_end = some ? it.past + (a.causal ? int_div(wr1 - 1, a.by_group) + 1 : 0) : 0;    // keys any of them sees
    const int w_all = some ? it.past + (a.causal ? int_div(wr0, a.by_group) + 1 : 0) : 0;          // keys all of them see

    Pages pg;
    pg.row = a.table + it.seq * a.table_stride; pg.n_pages = a.n_pages; pg.bad = false; pg.base = 0; pg.ids = 0;
    const Rows<P, D> krows(a.k, a.kc, kvh), vrows(a.v, a.vc, kvh);
    const unsigned kring = lds_address(smem), vring = kring + NB * C::TILE;
    const int last_page = (k1 - 1) >> a.page_shift;
    // K of the tile at key0, V of the tile in front of it
    auto fetch_k = [&](int key0, int buf) { krows.template fetch<KT / C::NW>(pg, a.page_shift, key0, w * (KT / C::NW), k1, kring + buf * C::TILE); };
    auto fetch_v = [&](int key0, int buf) { vrows.template fetch<KT / C::NW>(pg, a.page_shift, key0, w * (KT / C::NW), k1, vring + buf * C::TILE); };
    auto pages_for = [&](int vkey, int kkey) {
        if (((min(kkey + KT, k1) - 1) >> a.page_shift) >= pg.base + 64) pg.load(min(vkey, k1 - 1) >> a.page_shift, last_page);
    };
    // lane parts of the LDS addresses: row l31 of K (chunk 2 t + h at step t), the two blocks of read_v
    const unsigned ka = l31 * RB + ((h ^ swizzle<RB, true>(l31 & 15)) << 4);
    const int i16 = lane & 15, vr = 4 * h + (i16 >> 2), vc = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);
    const unsigned va = vr * RB + ((vc ^ swizzle<RB, true>(vr)) << 4) + (i16 & 1) * 8;
    const unsigned vb = (vr + 8) * RB + ((vc ^ swizzle<RB, true>(vr + 8)) << 4) + (i16 & 1) * 8;

    bf16x8 qf[NKS];
    {
        const bool live = row < r_end;
        const int tok = live ? int_div(row, a.by_group) : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
        lim = live && !it.bad ? it.past + (a.causal ? tok + 1 : 0) : 0;
        const elem_t* qp = reinterpret_cast<const elem_t*>(a.q) + (int64_t)(it.first + tok) * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int t = 0; t < NKS; ++t) qf[t] = *reinterpret_cast<const bf16x8*>(qp + (2 * t + h) * 8);
    }
    f32x16 o[NDB], sa[2], sb[2];      // the scores of a tile and of the next take turns
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;       // maximum of the query's scores (log2 units), sum of the weights of this half's keys

    if (k0 < k1) pg.load(k0 >> a.page_shift, last_page);
    // the query rows arrive before the first tile is sent for: a wait for them further on would be one for the tiles in flight too
#pragma unroll
    for (int t = 0; t < NKS; ++t) asm volatile("" : "+v"(qf[t]));
    if (k0 < k1) {
        fetch_k(k0, 0);
#pragma unroll
        for (int j = 1; j < NB; ++j) {                         // rows behind the end are its last row: as many transfers for a short range
            pages_for(k0 + (j - 1) * KT, k0 + j * KT);
            fetch_k(k0 + j * KT, j);
            fetch_v(k0 + (j - 1) * KT, j - 1);
        }
        wait_vm<(NB - 1) * 2 * C::DMA>();
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sa[b][r] = 0.f;
#pragma unroll
            for (int t = 0; t < NKS; ++t)
                sa[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, read_lds(kring + b * 32 * RB + (ka ^ (t << 5)))), qf[t], sa[b], 0, 0, 0);
        }
    }
    float mx = -INFINITY;               // maximum of a tile's scores, unmasked
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sa[b][r]);
    int buf = 0;                        // of V(i), and of the K(i) that is in `s`
    // one tile; FULL: the tiles it sends for lie in front of the end
    auto iteration = [&](int key0, f32x16 (&s)[2], f32x16 (&sn)[2], auto full) {
        constexpr bool FULL = decltype(full)::value;
        const int knext = buf + 1 == NB ? 0 : buf + 1, free_v = buf == 0 ? NB - 1 : buf - 1;
        if constexpr (FULL) wait_vm<(NB - 2) * 2 * C::DMA>();
        else wait_vm<0>();
        wait_lds();
        __builtin_amdgcn_s_barrier();        // K(i + 1) and V(i) have landed, every wave has left K(i) and V(i - 1)
        const unsigned kt = kring + knext * C::TILE, vt = vring + buf * C::TILE;
        const unsigned ksend = kring + buf * C::TILE + w * (KT / C::NW) * RB, vsend = vring + free_v * C::TILE + w * (KT / C::NW) * RB;
        pages_for(key0 + (NB - 1) * KT, key0 + NB * KT);
        const char *ksrc = nullptr, *vsrc = nullptr;
        if constexpr (FULL) {
            ksrc = krows.slice(pg, a.page_shift, key0 + NB * KT + w * (KT / C::NW));
            vsrc = vrows.slice(pg, a.page_shift, key0 + (NB - 1) * KT + w * (KT / C::NW));
        } else {
            if (key0 + NB * KT < k1) fetch_k(key0 + NB * KT, buf);
            if (key0 + (NB - 1) * KT < k1) fetch_v(key0 + (NB - 1) * KT, free_v);
        }
        buf = knext;
        unsigned dma_lane = lane;
        if constexpr (D == 128) asm volatile("" : "+v"(dma_lane));   // the lane offsets of the transfers are computed anew (8 registers)
        if (key0 >= w_end) {                 // nothing here for this wave's rows (it keeps moving its share of the tiles)
            if constexpr (FULL) {
                each<0, C::DMA>([&](auto I) { krows.template fetch_one<decltype(I)::value>(ksrc, ksend, dma_lane); });
                each<0, C::DMA>([&](auto I) { vrows.template fetch_one<decltype(I)::value>(vsrc, vsend, dma_lane); });
            }
            return;
        }
        // operand fragments from LDS, AHEAD steps ahead: K of the next tile (steps 0 .. NQ - 1), then V of this one.  (The step is xor-ed into
        // the whole address, not into its lane part: that would be 16 registers kept.)
        constexpr int RING = D == 64 ? 4 : 6, AHEAD = RING - 1;
        bf16x8 fr[RING];
        const unsigned kat = kt + ka, vat = vt + va, vbt = vt + vb;
        auto fragment = [&](int u) {
            if (u < NQ) fr[u % RING] = __builtin_bit_cast(bf16x8, read_lds((kat ^ (u % NKS << 5)) + (u / NKS) * 32 * RB));
            else {
                const int v = u - NQ;
                fr[u % RING] = read_v((vat ^ (v % NDB << 6)) + 16 * (v / NDB) * RB, (vbt ^ (v % NDB << 6)) + 16 * (v / NDB) * RB);
            }
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) fragment(u);
        const uint64_t alive = tile_mask(a, it.seq, key0);
        if (key0 + KT > w_all || alive != ~0ull) {             // some key of the tile is not for some query
            const int left = lim - key0;
            const uint64_t see = (left >= 64 ? ~0ull : (left <= 0 ? 0ull : (1ull << left) - 1)) & alive;
            const uint32_t half[2] = {(uint32_t)(see >> (4 * h)), (uint32_t)(see >> 32 >> (4 * h))};
            mx = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[b][r] = (half[b] >> ((r & 3) + 8 * (r >> 2))) & 1 ? s[b][r] : -INFINITY;
                    mx = fmaxf(mx, s[b][r]);
                }
        }
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

        // scores of the next tile (behind the last: of whatever the buffer holds, unused) beside the weights of this one
        bf16x8 pf[4];
        constexpr int SQ = 32 / NQ, SP = 32 / NP, EVERY = NQ / (2 * C::DMA);
#pragma unroll
        for (int r = 0; r < 16; ++r) sn[0][r] = sn[1][r] = 0.f;
        __builtin_amdgcn_sched_barrier(0);
        each<0, NQ>([&](auto U) {
            constexpr int u = decltype(U)::value;
            if (u + AHEAD < NQ + NP) fragment(u + AHEAD);
            sn[u / NKS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[u % RING], qf[u % NKS], sn[u / NKS], 0, 0, 0);
            if constexpr (FULL && u % EVERY == 0) {
                constexpr int i = u / EVERY;
                if constexpr (i < C::DMA) krows.template fetch_one<i>(ksrc, ksend, dma_lane);
                else vrows.template fetch_one<i - C::DMA>(vsrc, vsend, dma_lane);
            }
#pragma unroll
            for (int j = 0; j < SQ; ++j) {
                const int e = u * SQ + j;
                s[e >> 4][e & 15] = exp2_hw(fmaf(s[e >> 4][e & 15], a.scale_log2, -mu));
            }
#pragma unroll
            for (int j = 0; j < SQ; ++j) {
                const int e = u * SQ + j;
                l += s[e >> 4][e & 15];
                pf[e >> 3][e & 7] = (__bf16)s[e >> 4][e & 15];
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        mx = sn[0][0];
        each<0, NP>([&](auto V) {
            constexpr int v = decltype(V)::value;
            if (v + AHEAD < NP) fragment(NQ + v + AHEAD);
            o[v % NDB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr[(NQ + v) % RING], pf[v / NDB], o[v % NDB], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < SP; ++j) mx = fmaxf(mx, sn[(v * SP + j) >> 4][(v * SP + j) & 15]);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    int key0 = k0;
    for (; key0 + (NB + 2) * KT <= k1; key0 += 2 * KT) {
        iteration(key0, sa, sb, std::true_type());
        iteration(key0 + KT, sb, sa, std::true_type());
    }
    for (; key0 < k1; key0 += KT) {
        iteration(key0, sa, sb, std::false_type());
        sa[0] = sb[0];
        sa[1] = sb[1];
    }
    wait_vm<0>();
    const PagedAttnArgs z = arguments_again();
    asm volatile("" : "+v"(row));            // recomputed here, not kept through the loop
    const bool live = row < r_end;
    const int tok = live ? int_div(row, z.by_group) : 0, head = kvh * z.group + (live ? row - tok * z.group : 0);
    const int64_t token = it.first + tok;
    if ((pg.bad || it.bad) && threadIdx.x == 0) atomicOr(z.status, (pg.bad ? PAGED_BAD_PAGE : 0) | (it.bad ? PAGED_BAD_LENGTH : 0));
    const bool bad = pg.bad || it.bad;
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
        const int64_t orow = token * z.q_heads + head;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int f = d * 32 + 2 * r + 4 * h;
                if (it.splits > 1) store4<PF32>(part_out<D>(z, it.split, orow) + f, o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]);
                else store4<P>(reinterpret_cast<elem_t*>(z.out) + token * z.os[0] + head * z.os[1] + f, o[d][r] * inv, o[d][r + 1] * inv,
                               o[d][r + 2] * inv, o[d][r + 3] * inv);
            }
        if (it.splits > 1 && h == 0) { float* ml = part_ml<D>(z, it.split, orow); ml[0] = m; ml[1] = l; }
    }
    uint32_t again = (uint32_t)odds | (uint32_t)(odds >> 32);
    while (again) {
        const int i = __builtin_ctz(again);
        again &= again - 1;
        store_row_alone<P, D>(z, it, kvh, wr0 + i);
    }
}

// =================================================================================================================================
// Chunks in f32: a workgroup owns 64 rows, 16 per wave (the f32 matrix rate is a sixteenth of bf16's and the same for 16 x 16 x 4 as for
// 32 x 32 x 2: the smaller shape wastes fewer rows of a ragged batch), the keys pass in tiles of 32 through a ring of LDS buffers.
// Bound: the f32 matrix unit in long chunks (128 tokens over 30000 keys, 16 heads of 128 over 4: 302 us, 104 TFLOP/s; the library's product
// of 4096^3 reaches 144), starts, joins and unequal lengths in short ones (5 chunks of up to 257 over up to 1290 keys, 16 heads of 64: 43 us
// and 6 of the join, 13 of them matrix work).
// =================================================================================================================================
template <int D> struct TileCfg {
    static constexpr int M = 64, NW = 4, KT = 32, RB = D * 4;
    static constexpr int TILE = KT * RB;                       // bytes of K or V of a tile
    static constexpr int NBUF = D == 64 ? 3 : 2;               // 48 / 64 KiB: three / two workgroups on a CU
    static constexpr int LDS = NBUF * 2 * TILE;                // [buffer][K, V]
    static constexpr int DMA = 2 * TILE / NW / 1024;           // LDS-DMA instructions per wave and tile
};

template <int D>
__global__ __launch_bounds__(256, 2) void paged_attn_tile_kernel(PagedAttnArgs a) {
    typedef PF32 P;
    typedef float elem_t;
    typedef TileCfg<D> C;
    constexpr int KT = C::KT, RB = C::RB, NKS = D / 16, NDB = D / 16;
    __shared__ __attribute__((aligned(1024))) char smem[C::LDS];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;

    Schedule<C::M, KT, true> sched;
    begin(a, sched, TILE_LAG);
    const int item = blockIdx.x;
    if (item >= sched.launch_items(a)) return;
    const int at = int_div(item, a.by_kv_heads), kvh = item - at * a.kv_heads;
    Item it;
    sched.find(a, at, &it, a.sched);
    if (it.split >= it.splits) return;
    const int k0 = it.k0, k1 = it.k1, r0 = it.tile * C::M, r_end = min(r0 + C::M, it.n * a.group);
    const int row = r0 + w * 16 + l15;                                                  // this lane's query
    const bool live = row < r_end;
    const int tok = live ? int_div(row, a.by_group) : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
    const int64_t token = it.first + tok;
    const int lim = live && !it.bad ? it.past + (a.causal ? tok + 1 : 0) : 0;           // keys 0 .. lim - 1 are seen
    const int wr0 = r0 + w * 16, wr1 = min(wr0 + 16, r_end);                            // rows of this wave: [wr0, wr1)
    const bool some = wr0 < wr1 && !it.bad;
    const int w_end = some ? it.past + (a.causal ? int_div(wr1 - 1, a.by_group) + 1 : 0) : 0;    // keys any of them sees
    const int w_all = some ? it.past + (a.causal ? int_div(wr0, a.by_group) + 1 : 0) : 0;        // keys all of them see

    Pages pg;
    pg.row = a.table + it.seq * a.table_stride; pg.n_pages = a.n_pages; pg.bad = false; pg.base = 0; pg.ids = 0;
    const Rows<P, D> krows(a.k, a.kc, kvh), vrows(a.v, a.vc, kvh);
    const unsigned lds = lds_address(smem);
    auto fetch = [&](int key0, int buf) {
        if (((min(key0 + KT, k1) - 1) >> a.page_shift) >= pg.base + 64) pg.load(key0 >> a.page_shift, (k1 - 1) >> a.page_shift);
        const unsigned to = lds + buf * 2 * C::TILE;
        krows.template fetch<KT / C::NW>(pg, a.page_shift, key0, w * (KT / C::NW), k1, to);
        vrows.template fetch<KT / C::NW>(pg, a.page_shift, key0, w * (KT / C::NW), k1, to + C::TILE);
    };
    const unsigned ka = l15 * RB + ((g ^ swizzle<RB, false>(l15)) << 4);                // row l15 of K, chunk 4 t + g at step t

    f32x4 qf[NKS];
    {
        const elem_t* qp = reinterpret_cast<const elem_t*>(a.q) + token * a.qs[0] + head * a.qs[1];
#pragma unroll
        for (int t = 0; t < NKS; ++t) qf[t] = *reinterpret_cast<const f32x4*>(qp + (4 * t + g) * 4);
    }
    f32x4 o[NDB];
#pragma unroll
    for (int d = 0; d < NDB; ++d) o[d] = {0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;       // maximum of the query's scores (log2 units), sum of the weights of this lane's keys
    if (k0 < k1) pg.load(k0 >> a.page_shift, (k1 - 1) >> a.page_shift);
    // the query rows arrive before the first tile is sent for: a wait for them inside the loop would be one for the tiles in flight too
#pragma unroll
    for (int t = 0; t < NKS; ++t) asm volatile("" : "+v"(qf[t]));
#pragma unroll
    for (int i = 0; i < C::NBUF - 1; ++i)
        if (k0 + i * KT < k1) fetch(k0 + i * KT, i);
    int buf = 0;
    for (int key0 = k0; key0 < k1; key0 += KT, buf = buf + 1 == C::NBUF ? 0 : buf + 1) {
        if (C::NBUF > 2 && key0 + KT < k1) wait_vm<C::DMA>();                           // the younger tile stays in flight
        else wait_vm<0>();
        wait_lds();
        __builtin_amdgcn_s_barrier();        // the tile has landed, and every wave has left the buffer of the tile before it
        if (key0 + (C::NBUF - 1) * KT < k1) fetch(key0 + (C::NBUF - 1) * KT, buf == 0 ? C::NBUF - 1 : buf - 1);
        if (key0 >= w_end) continue;         // nothing here for this wave's rows (it keeps moving its share of the tiles)
        const unsigned kt = lds + buf * 2 * C::TILE, vt = kt + C::TILE;
        // operands are read two steps (of four products each) ahead; left to itself, hipcc reads, waits and multiplies in turn
        f32x4 s[2], kf[3];
        const unsigned kat = kt + ka;
        auto key_fragment = [&](int u) { kf[u % 3] = __builtin_bit_cast(f32x4, read_lds((kat ^ (u % NKS << 6)) + (u / NKS) * 16 * RB)); };
        key_fragment(0);
        key_fragment(1);
#pragma unroll
        for (int u = 0; u < 2 * NKS; ++u) {
            if (u + 2 < 2 * NKS) key_fragment(u + 2);
            if (u % NKS == 0) s[u / NKS] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) s[u / NKS] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[u % 3][j], qf[u % NKS][j], s[u / NKS], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        // step e: feature 16 d + l15 of key 16 (e / 4) + 4 g + e % 4
        float vx[3][NDB];
        const unsigned vat = vt + 4 * g * RB + (l15 & 3) * 4;
        auto value_fragment = [&](int e) {
            const int r = (e >> 2) * 16 + (e & 3);
            const unsigned sw = swizzle<RB, false>((r + 4 * g) & 15);
#pragma unroll
            for (int d = 0; d < NDB; ++d) vx[e % 3][d] = read_lds_f32(vat + r * RB + (((d * 4 + (l15 >> 2)) ^ sw) << 4));
        };
        value_fragment(0);
        value_fragment(1);
        __builtin_amdgcn_sched_barrier(0);
        const uint64_t alive = tile_mask(a, it.seq, key0);
        if (key0 + KT > w_all || (uint32_t)alive != ~0u) {             // some key of the tile is not for some query
            const int left = lim - key0;
            const uint32_t see = (left >= 32 ? ~0u : (left <= 0 ? 0u : (1u << left) - 1)) & (uint32_t)alive;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[b][r] = (see >> (16 * b + 4 * g + r)) & 1 ? s[b][r] : -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = swap_max32(swap_max16(mx)) * a.scale_log2;
        if (__any(mx > m + 8.f)) {           // as in the chunk kernel
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
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e + 2 < 8) value_fragment(e + 2);
#pragma unroll
            for (int d = 0; d < NDB; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[e % 3][d], s[e >> 2][e & 3], o[d], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    wait_vm<0>();
    if ((pg.bad || it.bad) && threadIdx.x == 0) atomicOr(a.status, (pg.bad ? PAGED_BAD_PAGE : 0) | (it.bad ? PAGED_BAD_LENGTH : 0));
    const bool bad = pg.bad || it.bad;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float inv = l == 0.f ? 0.f : 1.f / l;
    if (bad) { l = NAN; inv = NAN; }
    bool odd = false;                        // as in the chunk kernel
    if (!bad) {
        float z = l * 0.f;
#pragma unroll
        for (int d = 0; d < NDB; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) z = fmaf(o[d][r], 0.f, z);
        odd = live && !(z == 0.f);
    }
    const uint64_t odds = __ballot(odd);
    if (live) {
        const int64_t orow = token * a.q_heads + head;
#pragma unroll
        for (int d = 0; d < NDB; ++d) {
            const int f = d * 16 + 4 * g;
            if (it.splits > 1) store4<P>(part_out<D>(a, it.split, orow) + f, o[d][0], o[d][1], o[d][2], o[d][3]);
            else store4<P>(reinterpret_cast<elem_t*>(a.out) + token * a.os[0] + head * a.os[1] + f, o[d][0] * inv, o[d][1] * inv, o[d][2] * inv, o[d][3] * inv);
        }
        if (it.splits > 1 && g == 0) { float* ml = part_ml<D>(a, it.split, orow); ml[0] = m; ml[1] = l; }
    }
    uint32_t again = (uint32_t)(odds | odds >> 16 | odds >> 32 | odds >> 48) & 0xffffu;
    while (again) {
        const int i = __builtin_ctz(again);
        again &= again - 1;
        store_row_alone<P, D>(a, it, kvh, wr0 + i);
    }
}

// =================================================================================================================================
// Few rows (at most 16 per sequence and key head: single tokens, their groups, short drafts): bound by the stream of the cache.  A wave
// owns every NW-th tile of 32 (f32: 16) keys and two LDS buffers of its own, so that nothing in the loop waits for another wave; the waves'
// states are joined once at the end.
// Lengths in order, long beside short on a CU: 32 sequences of 100 - 2500 keys, 16 heads of 64 33 us, as they come 40; up to 8 tokens each 33, 37.
// Measured: 32 sequences of 700 - 2579 keys, 16 heads of 64 in bf16: 37.5 us, 5800 GB/s; two of 120001 - 131070 keys, 32 heads of 128 over 4:
// 86.8 us with 5 of the join, 5760 GB/s; a copy of 1 GiB reaches 5060.  One sequence of up to 700 keys is a chain of dependent trips: 7 us.
// =================================================================================================================================
template <typename P, int D> struct StepCfg {
    static constexpr int M = 16, KT = P::IS_BF16 ? 32 : 16;
    static constexpr int RB = D * (int)sizeof(typename P::elem_t);
    static constexpr int TILE = KT * RB, STAGE = 2 * TILE;
    static constexpr int DMA = STAGE / 1024;
    static_assert(16 * (D + 2) * 4 + 4 <= 2 * STAGE, "the waves' states fit where their tiles were");
};

template <typename P, int D, int NW>
__global__ __launch_bounds__(NW * 64) void paged_attn_step_kernel(PagedAttnArgs a) {
    typedef typename P::elem_t elem_t;
    typedef StepCfg<P, D> C;
    constexpr int KT = C::KT, KB = KT / 16, RB = C::RB, EPL = P::EPL, NKS = D / (4 * EPL), NDB = D / 16;
    __shared__ __attribute__((aligned(1024))) char smem[NW * 2 * C::STAGE];
    const int lane = threadIdx.x & 63, w = uniform(threadIdx.x >> 6), l15 = lane & 15, g = lane >> 4;

    Schedule<C::M, KT, true> sched;
    // up to 512 keys the order saves less than it takes (32 x 201 keys, 16 heads: 6.9 us, in order 7.5)
    const bool unequal = a.n_seqs <= 64 && (a.max_pages << a.page_shift) > 512;
    sched.by_length = unequal && a.n_seqs * a.kv_heads > SLOTS / 2;
    Item it;
    int kvh;
    const int item = blockIdx.x;
    if (!a.starts && a.splits == 1) {        // one token each, whole: items follow from their numbers
        const int tiles = (a.group + C::M - 1) / C::M, all = a.n_seqs * tiles * a.kv_heads;
        const bool order = unequal && all > SLOTS / 2;          // long ones first, up to two on a CU beside short ones, as in chunks
        const int number = order && all <= SLOTS && item >= SLOTS / 2 ? all - 1 - (item - SLOTS / 2) : item;
        const int at = int_div(number, a.by_kv_heads), q = tiles == 1 ? at : at / tiles;
        kvh = number - at * a.kv_heads;
        it.n = 1;
        if (order) {
            sched.load(a, 0);
            sched.sort(a);
            it.seq = __builtin_amdgcn_readlane(sched.seq, q);
            it.past = __builtin_amdgcn_readlane(sched.past, q);
        } else {
            it.seq = q;
            it.past = a.past[q];
        }
        it.first = it.seq;
        sched.place(a, at - q * tiles, &it);
    } else {
        begin(a, sched, STEP_LAG);
        const int all = sched.launch_items(a);
        if (item >= all) return;
        const int number = sched.by_length && all > SLOTS / 2 && all <= SLOTS && item >= SLOTS / 2 ? all - 1 - (item - SLOTS / 2) : item;
        const int at = int_div(number, a.by_kv_heads);
        kvh = number - at * a.kv_heads;
        sched.find(a, at, &it, a.sched);
    }
    if (it.split >= it.splits) return;
    const int k0 = it.k0, k1 = it.k1, r0 = it.tile * C::M, r_end = min(r0 + C::M, it.n * a.group);
    const int row = r0 + l15;
    const bool live = row < r_end;
    const int tok = live ? int_div(row, a.by_group) : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
    const int64_t token = it.first + tok;
    const int lim = live && !it.bad ? it.past + (a.causal ? tok + 1 : 0) : 0;
    const int all = r_end - r0 == C::M && !it.bad ? it.past + (a.causal ? int_div(r0, a.by_group) + 1 : 0) : 0;      // keys every column sees

    Pages pg;
    pg.row = a.table + it.seq * a.table_stride; pg.n_pages = a.n_pages; pg.bad = false; pg.base = 0; pg.ids = 0;
    const Rows<P, D, true> krows(a.k, a.kc, kvh), vrows(a.v, a.vc, kvh);
    const unsigned ring = lds_address(smem) + w * 2 * C::STAGE;
    const int first = k0 + w * KT;
    auto fetch = [&](int key0, int buf) {
        if (((min(key0 + KT, k1) - 1) >> a.page_shift) >= pg.base + 64) pg.load(key0 >> a.page_shift, (k1 - 1) >> a.page_shift);
        const unsigned to = ring + buf * C::STAGE;
        krows.template fetch<KT>(pg, a.page_shift, key0, 0, k1, to);
        vrows.template fetch<KT>(pg, a.page_shift, key0, 0, k1, to + C::TILE);
    };
    const unsigned ka = l15 * RB + ((g ^ swizzle<RB, P::IS_BF16>(l15)) << 4);
    const int vr = 4 * g + (l15 >> 2), vc = (l15 >> 1) & 1;
    const unsigned va = vr * RB + ((vc ^ swizzle<RB, P::IS_BF16>(vr)) << 4) + (l15 & 1) * 8;       // and 16 rows further on

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
        const unsigned kt = ring + buf * C::STAGE, vt = kt + C::TILE;
        f32x4 s[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            s[b] = {0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < NKS; ++t) {
                const u32x4 kf = read_lds(kt + b * 16 * RB + (ka ^ (t << 6)));
                if constexpr (P::IS_BF16) {
                    s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, qf[t]), s[b], 0, 0, 0);
                } else {
                    const f32x4 kx = __builtin_bit_cast(f32x4, kf), qx = __builtin_bit_cast(f32x4, qf[t]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[j], qx[j], s[b], 0, 0, 0);
                }
            }
        }
        const uint64_t alive = tile_mask(a, it.seq, key0);
        constexpr uint32_t seen = KT == 32 ? ~0u : (1u << KT % 32) - 1;
        if (key0 + KT > all || ((uint32_t)alive & seen) != seen) {
            const int left = lim - key0;
            const uint32_t see = (left >= KT ? seen : (left <= 0 ? 0u : (1u << left) - 1)) & (uint32_t)alive;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[b][r] = (see >> (16 * b + 4 * g + r)) & 1 ? s[b][r] : -INFINITY;
        }
        float mx = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
        if constexpr (KB == 2) mx = fmaxf(mx, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
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
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[b][r] = exp2_hw(fmaf(s[b][r], a.scale_log2, -mu));
                l += s[b][r];
            }
        if constexpr (P::IS_BF16) {
            // slots 0 .. 3 of group g: keys 4 g .. of the lower 16, slots 4 .. 7: of the upper 16
            bf16x8 pf;
#pragma unroll
            for (int j = 0; j < 8; ++j) pf[j] = (__bf16)s[j >> 2][j & 3];
#pragma unroll
            for (int d = 0; d < NDB; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(read_v(vt + (va ^ (d << 5)), vt + 16 * RB + (va ^ (d << 5))), pf, o[d], 0, 0, 0);
        } else {
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * b + 4 * g + r;
                    const unsigned at = vt + row * RB + (l15 & 3) * 4, sw = swizzle<RB, P::IS_BF16>(row & 15);
#pragma unroll
                    for (int d = 0; d < NDB; ++d)
                        o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(read_lds_f32(at + (((d * 4 + (l15 >> 2)) ^ sw) << 4)), s[b][r], o[d], 0, 0, 0);
                }
        }
    }
    wait_vm<0>();
    if ((pg.bad || it.bad) && lane == 0) atomicOr(a.status, (pg.bad ? PAGED_BAD_PAGE : 0) | (it.bad ? PAGED_BAD_LENGTH : 0));
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (pg.bad || it.bad) l = NAN;

    // join the waves: outputs [NW][16][D] (16-byte pieces XOR-swizzled by the row), maxima, sums [NW][16] and whether the wave met a bad page
    // [NW] in the place of the tiles
    __syncthreads();
    float* sm = reinterpret_cast<float*>(smem) + NW * 16 * D;
    int* met_bad = reinterpret_cast<int*>(sm + 2 * NW * 16);
#pragma unroll
    for (int d = 0; d < NDB; ++d)
        *reinterpret_cast<f32x4*>(smem + ((w * 16 + l15) * D + (((d * 4 + g) ^ (l15 & 7)) << 2)) * 4) = o[d];
    if (g == 0) { sm[w * 16 + l15] = m; sm[(NW + w) * 16 + l15] = l; }
    if (lane == 0) met_bad[w] = pg.bad;
    __syncthreads();
    bool bad = it.bad;                       // every wave looks at the pages of its own tiles, and finishes rows of all
#pragma unroll
    for (int v = 0; v < NW; ++v) bad = bad || met_bad[v] != 0;
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
        const float z = fmaf(acc[0], 0.f, fmaf(acc[1], 0.f, fmaf(acc[2], 0.f, fmaf(acc[3], 0.f, sum * 0.f))));
        const int tk = on ? int_div(rr, a.by_group) : 0, hd = kvh * a.group + (on ? rr - tk * a.group : 0);
        const int64_t t64 = it.first + tk;
        if (on) {
            if (it.splits > 1) {
                const int64_t orow = t64 * a.q_heads + hd;
                *reinterpret_cast<f32x4*>(part_out<D>(a, it.split, orow) + piece * 4) = acc;
                if (piece == 0) { float* ml = part_ml<D>(a, it.split, orow); ml[0] = top; ml[1] = sum; }
            } else {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                store4<P>(reinterpret_cast<elem_t*>(a.out) + t64 * a.os[0] + hd * a.os[1] + piece * 4, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
            }
        }
        // rows of this wave's pieces whose result is not finite (64 lanes hold 64 / PPR rows), again and alone
        uint64_t odds = __ballot(on && !bad && !(z == 0.f));
        while (odds) {
            const int src = __builtin_ctzll(odds), rw = (i - lane + src) / PPR;
            const uint64_t same = PPR == 64 ? ~0ull : (((1ull << PPR) - 1) << (src / PPR * PPR));
            odds &= ~same;
            store_row_alone<P, D>(a, it, kvh, r0 + uniform(rw));
        }
    }
}

// =================================================================================================================================
// Joins the partial results of cut tiles.  A workgroup takes RPB rows of a tile: 256 / (D / 4) of them, one 16-byte piece of a row per
// thread, or (few rows, many shares) a single one, the shares dealt out over its threads.  Bound by its launch and two trips to memory: 4 to
// 6 us (one share after the other: 128 rows of 116 shares took 30).
// =================================================================================================================================
template <typename P, int D, int M, int KT, int RPB>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttnArgs a) {
    typedef typename P::elem_t elem_t;
    constexpr int LPR = D / 4, SP = 256 / (RPB * LPR), PARTS = M / RPB;
    static_assert(SP * RPB * LPR == 256, "one piece per thread");
    __shared__ float weight[RPB == 1 ? MAX_SPLITS : 1], red[8];
    __shared__ f32x4 pieces[RPB == 1 ? 256 : 1];
    const int share = __builtin_bit_cast(int, a.part[0]);
    Schedule<M, KT, false> sched;
    sched.share = 0x3fffffff;
    const int t = blockIdx.x / PARTS, groups = sched_groups(a.n_seqs);
    if (a.sched) sched.items = a.sched[2 * groups + 1];
    else {
        sched.load(a, 0);
        sched.number(a);
    }
    if (t >= sched.launch_items(a)) return;
    const int at = int_div(t, a.by_kv_heads), kvh = t - at * a.kv_heads;
    Item it;
    sched.find(a, at, &it, a.sched + groups + 1);
    const int kt = (it.end + KT - 1) / KT, splits = min(kt <= share ? 1 : (kt + share - 1) / share, a.splits);
    if (splits == 1) return;                 // written already
    const int tid = threadIdx.x, piece = tid % LPR, sub = tid / LPR % SP;
    const int row = it.tile * M + (blockIdx.x % PARTS) * RPB + (RPB == 1 ? 0 : tid / LPR);
    const bool live = row < it.n * a.group;
    if (RPB == 1 && !live) return;
    const int tok = live ? int_div(row, a.by_group) : 0, head = kvh * a.group + (live ? row - tok * a.group : 0);
    const int64_t token = it.first + tok, orow = token * a.q_heads + head;
    f32x4 acc = {0, 0, 0, 0};
    float sum = 0.f;
    if constexpr (RPB > 1) {
        float top = -INFINITY;
        for (int s0 = 0; s0 < splits; s0 += 8) {       // eight shares in one round trip
            float m[8], l[8];
            f32x4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int s = min(s0 + u, splits - 1);
                const float* ml = part_ml<D>(a, s, orow);
                m[u] = ml[0];
                l[u] = s0 + u < splits ? ml[1] : 0.f;
                x[u] = *reinterpret_cast<const f32x4*>(part_out<D>(a, s, orow) + piece * 4);
            }
            float next = top;
#pragma unroll
            for (int u = 0; u < 8; ++u) next = fmaxf(next, m[u]);
            const float mu = next == -INFINITY ? 0.f : next, keep = exp2_hw(top - mu);
            top = next;
            sum *= keep;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] *= keep;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float f = l[u] == 0.f ? 0.f : exp2_hw(m[u] - mu);
                sum = fmaf(l[u], f, sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = l[u] == 0.f ? acc[i] : fmaf(x[u][i], f, acc[i]);
            }
        }
    } else {
        float m = -INFINITY, l = 0.f;
        if (tid < splits) { const float* ml = part_ml<D>(a, tid, orow); m = ml[0]; l = ml[1]; }
        float top = wave_max(m);
        if ((tid & 63) == 0) red[tid >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float f = exp2_hw(m - (top == -INFINITY ? 0.f : top));      // no key: e^-inf
        weight[tid] = f;
        const float part = wave_sum(l * f);
        if ((tid & 63) == 0) red[4 + (tid >> 6)] = part;
        __syncthreads();
        sum = (red[4] + red[5]) + (red[6] + red[7]);
#pragma unroll 4
        for (int s = sub; s < splits; s += SP) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(part_out<D>(a, s, orow) + piece * 4);
            const float fs = weight[s];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(x[i], fs, acc[i]);
        }
        pieces[tid] = acc;
        __syncthreads();
        if (sub != 0) return;
        for (int s = 1; s < SP; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += pieces[s * LPR + piece][i];
    }
    if (live) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        store4<P>(reinterpret_cast<elem_t*>(a.out) + token * a.os[0] + head * a.os[1] + piece * 4, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
}

struct Plan { bool step, scheduled; int tiles, splits, min_share; };
// floats of the share and the partial results in the workspace; the schedule lies behind them
int64_t part_floats(const PagedAttnArgs& a, const Plan& p, int head_dim) {
    return PART_HEAD + (p.splits == 1 ? 0 : (int64_t)p.splits * a.tokens * a.q_heads * (head_dim + 2));
}

// max_new tokens a sequence at most (0: not known) make at most max_new * group rows per key head.  Up to 16 take the step kernel; up to 128
// where its tiles of 16 are no more than the CUs and the keys are few (128 KiB of them): four waves then share a tile's keys, where the
// chunk kernel leaves them to one wave a row (bf16, 8 x 32 rows over 500 keys, 8 heads of 64: 9.6 us, 13.3; 4 x 60 rows over 200, 16 heads: 7.2,
// 9.9; f32: 12.9, 20.6; over more keys it loses: 1 x 120 rows over 6000, head dim 128: 27.9, 22.8).
Plan make_plan(const PagedAttnArgs& a, int max_new, int head_dim, int dtype) {
    const int row_of_cache = head_dim * (dtype == PTTS_BF16 ? 2 : 4);
    Plan p;
    const int64_t most = (a.starts ? max_new : 1) * (int64_t)a.group;       // 0: not known
    const int64_t keys = (int64_t)a.max_pages << a.page_shift;
    const bool more_rows = most > 16 && most <= 128 && keys * row_of_cache <= 131072 && a.n_seqs * a.kv_heads * ((most + 15) / 16) <= 256;
    p.step = (most > 0 && most <= 16) || more_rows;
    // the tiles of 64 sequences are summed in 32 bits, and starts may give all rows to each of them
    if (a.starts && (int64_t)a.tokens * a.group > ((int64_t)1 << 29) - 65536) p.step = false;
    const int M = p.step ? 16 : (dtype == PTTS_BF16 ? 128 : 64);
    const int64_t ub = a.starts ? (int64_t)a.tokens * a.group / M + a.n_seqs : (int64_t)a.n_seqs * ((a.group + M - 1) / M);
    p.tiles = (int)ub;
    int64_t est = most > 0 ? (int64_t)a.n_seqs * ((most + M - 1) / M) : ub;
    if (est > ub) est = ub;
    // Most shares of a tile: none where the launch covers most CUs (`idle`: those it leaves over; from 160 items on cutting gains nothing but
    // evenness) and the keys that a workgroup could be left with alone take less time than the join: 512 keys of chunks in bf16, 64 KiB of
    // K for few rows, two least shares in f32.  Measured, whole and cut, in us: 12 chunks of 128 over 1900 keys, 16 heads of 64 in bf16
    // (192 items) 37, 47; 15 x 74 rows over 372, 10/5 heads of 128 16.5, 24; 4 x 259 over 779, 4/2 heads of 64 (40 items) 16.2, 13.8; single
    // tokens over 1900 keys, 16 x 16 heads of 64 26, 31; over 900, 16 heads of 128 (16 items) 22, 12; over 500 (64 items) 13.5, 12.
    // Never more than 128 MiB of partial results.
    const int64_t row_bytes = (int64_t)a.tokens * a.q_heads * (head_dim + 2) * 4;
    p.min_share = 32768 / row_of_cache < 32 ? 32 : 32768 / row_of_cache;    // 32 KiB of keys: 256 rows of 64 in bf16, 64 of 128 in f32
    int64_t s = keys / p.min_share;
    const int64_t items = est * a.kv_heads, idle = items < 160 ? 256 - items : 0;
    const int64_t alone = p.step ? 65536 / row_of_cache : dtype == PTTS_BF16 ? 512 : p.min_share * 2;
    const int64_t limit = p.step ? 4096 : dtype == PTTS_BF16 ? 2048 : p.min_share * 8;
    if (keys <= limit && keys * idle <= alone * 256) s = 1;
    if (s > MAX_SPLITS) s = MAX_SPLITS;
    if (s > ((int64_t)128 << 20) / row_bytes) s = ((int64_t)128 << 20) / row_bytes;
    p.splits = s < 2 ? 1 : (int)s;
    p.scheduled = a.n_seqs > MANY_SEQS && !(p.step && !a.starts && p.splits == 1);
    return p;
}

// Four waves with stages of 16 KiB have a CU to themselves, two share it with another workgroup: four where the launch gives a CU no
// second workgroup anyway (bf16, head dim 128: 64 tokens over 100 keys, 16/4 heads 6.8 us, 9.1; 30000 keys, 16/4 heads 25.3, 21.1).
template <typename P, int D>
void launch_step(const PagedAttnArgs& a, unsigned items, hipStream_t s) {
    if constexpr (StepCfg<P, D>::STAGE > 8192) {
        if (items > 256) {
            hipLaunchKernelGGL((paged_attn_step_kernel<P, D, 2>), dim3(items), dim3(128), 0, s, a);
            return;
        }
    }
    hipLaunchKernelGGL((paged_attn_step_kernel<P, D, 4>), dim3(items), dim3(256), 0, s, a);
}

template <typename P, int D>
hipError_t launch(PagedAttnArgs a, int max_new, hipStream_t s) {
    const Plan p = make_plan(a, max_new, D, P::IS_BF16 ? PTTS_BF16 : PTTS_F32);
    a.splits = p.splits;
    a.min_share = p.min_share;
    a.by_group = make_int_div((uint32_t)a.group);
    a.by_kv_heads = make_int_div((uint32_t)a.kv_heads);
    // cutting adds at most 2 SLOTS items: a share is no less than a slot's part of a work that counts at least half of every tile's keys
    // (64 more for the roundings of that sum)
    const int64_t groups = (int64_t)p.tiles * a.kv_heads;
    const int64_t cut = groups * p.splits < groups + 2 * SLOTS + 64 ? groups * p.splits : groups + 2 * SLOTS + 64;
    if (cut > 0x7fffffff / 16) return hipErrorInvalidValue;
    a.sched = p.scheduled ? reinterpret_cast<int*>(a.part) + part_floats(a, p, D) : nullptr;
    if (p.scheduled) {
        if (p.step) hipLaunchKernelGGL((paged_attn_schedule_kernel<16, StepCfg<P, D>::KT, false>), dim3(1), dim3(1024), 0, s, a, STEP_LAG);
        else if constexpr (P::IS_BF16) hipLaunchKernelGGL((paged_attn_schedule_kernel<128, 64, true>), dim3(1), dim3(1024), 0, s, a, TILE_LAG);
        else hipLaunchKernelGGL((paged_attn_schedule_kernel<64, 32, true>), dim3(1), dim3(1024), 0, s, a, TILE_LAG);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.step) launch_step<P, D>(a, (unsigned)cut, s);
    else if constexpr (P::IS_BF16) hipLaunchKernelGGL(paged_attn_chunk_kernel<D>, dim3((unsigned)cut), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(paged_attn_tile_kernel<D>, dim3((unsigned)cut), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    constexpr int RPB = 1024 / D;
    if (p.step) hipLaunchKernelGGL((paged_attn_join_kernel<P, D, 16, StepCfg<P, D>::KT, 1>), dim3((unsigned)groups * 16), dim3(256), 0, s, a);
    else if constexpr (P::IS_BF16) hipLaunchKernelGGL((paged_attn_join_kernel<P, D, 128, 64, RPB>), dim3((unsigned)groups * (128 / RPB)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((paged_attn_join_kernel<P, D, 64, 32, RPB>), dim3((unsigned)groups * (64 / RPB)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

int64_t paged_attn_workspace(const PagedAttnArgs& a, int max_new, int head_dim, int dtype) {
    const Plan p = make_plan(a, max_new, head_dim, dtype);
    if (p.splits == 1 && !p.scheduled) return 0;
    return (part_floats(a, p, head_dim) + (p.scheduled ? sched_ints(a.n_seqs) : 0)) * (int64_t)sizeof(float);
}

hipError_t paged_attn_launch(const PagedAttnArgs& a, int max_new, int head_dim, int dtype, hipStream_t s) {
    if (dtype == PTTS_BF16) return head_dim == 64 ? launch<PBF16, 64>(a, max_new, s) : launch<PBF16, 128>(a, max_new, s);
    return head_dim == 64 ? launch<PF32, 64>(a, max_new, s) : launch<PF32, 128>(a, max_new, s);
}

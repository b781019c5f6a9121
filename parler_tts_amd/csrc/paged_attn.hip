// Attention of new tokens over a paged KV cache: o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j a query may see.
#include "ptts_common.h"
#include "gemm.h"
#include "paged.h"

namespace {

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

// One wave per (token, query head), 64 keys a time: a lane takes one key's score, then the lanes are the features of the output.
template <typename P, int D>
__global__ __launch_bounds__(64) void paged_attn_simple_kernel(PagedAttnArgs a) {
    typedef typename P::elem_t elem_t;
    constexpr int V = 16 / sizeof(elem_t), R = D / 64;
    __shared__ float qs[D];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    if (t == 0 && h == 0 && a.starts) check_starts(a.starts, a.n_seqs, a.tokens, a.status);
    int s = t, first = t, end = t + 1;
    if (a.starts) {
        int lo = 0, hi = a.n_seqs;                    // largest s with starts[s] <= t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.starts[mid] <= t) lo = mid; else hi = mid;
        }
        s = lo; first = a.starts[s]; end = a.starts[s + 1];
        if (t < first || t >= end) return;            // behind the last sequence
    }
    const int past = a.past[s], reach = a.max_pages << a.page_shift;
    bool bad = past < 0 || first < 0 || end > a.tokens;
    const int64_t see = (int64_t)past + (a.causal ? t - first + 1 : 0);
    int lim = see > reach ? 0 : (int)see;
    if (bad || see > reach) { if (lane == 0) atomicOr(a.status, first < 0 || end > a.tokens ? PAGED_BAD_STARTS : PAGED_BAD_LENGTH); bad = true; lim = 0; }
    const elem_t* qp = reinterpret_cast<const elem_t*>(a.q) + t * a.qs[0] + h * a.qs[1];
    for (int d = lane; d < D; d += 64) qs[d] = from_elem<P>(qp[d]);
    __syncthreads();
    const int kvh = h / a.group;
    const elem_t* kb = reinterpret_cast<const elem_t*>(a.k) + kvh * a.kc[1];
    const elem_t* vb = reinterpret_cast<const elem_t*>(a.v) + kvh * a.vc[1];
    const int* table = a.table + s * a.table_stride;
    float m = -INFINITY, l = 0.f, acc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] = 0.f;
    for (int j0 = 0; j0 < lim; j0 += 64) {
        const int j = j0 + lane;
        float sc = -INFINITY;
        int page = -1;
        if (j < lim) {
            page = table[j >> a.page_shift];
            const bool ok = (unsigned)page < (unsigned)a.n_pages;
            if (!ok) { atomicOr(a.status, PAGED_BAD_PAGE); bad = true; }
            const bool live = ok && (!a.mask || j >= a.mask_width || a.mask[s * a.mask_stride + j]);
            if (live) {
                const elem_t* kp = kb + page * a.kc[0] + (j & ((1 << a.page_shift) - 1)) * a.kc[2];
                float d = 0.f;
                for (int c = 0; c < D; c += V) {
                    float f[V];
                    load16<P>(kp + c, f);
#pragma unroll
                    for (int i = 0; i < V; ++i) d = fmaf(qs[c + i], f[i], d);
                }
                sc = d * a.scale_log2;
            } else page = -1;
        }
        const float mn = fmaxf(m, wave_max(sc));
        const float mu = mn == -INFINITY ? 0.f : mn;
        const float p = page >= 0 ? exp2f(sc - mu) : 0.f, al = exp2f(m - mu);
        l = l * al + wave_sum(p);
        m = mn;
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] *= al;
        for (int i = 0; i < 64 && j0 + i < lim; ++i) {
            const int pg = __shfl(page, i);
            const float pi = __shfl(p, i);
            if (pg < 0) continue;
            const elem_t* vp = vb + pg * a.vc[0] + ((j0 + i) & ((1 << a.page_shift) - 1)) * a.vc[2];
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] = fmaf(pi, from_elem<P>(vp[r * 64 + lane]), acc[r]);
        }
    }
    bad = __any(bad);
    elem_t* op = reinterpret_cast<elem_t*>(a.out) + t * a.os[0] + h * a.os[1];
#pragma unroll
    for (int r = 0; r < R; ++r) op[r * 64 + lane] = to_elem<P>(bad ? NAN : (l == 0.f ? 0.f : acc[r] / l));
}

}  // namespace

int64_t paged_attn_workspace(const PagedAttnArgs&, int, int, int) { return 0; }

hipError_t paged_attn_launch(const PagedAttnArgs& a, int max_new, int head_dim, int dtype, hipStream_t s) {
    dim3 grid(a.tokens, a.q_heads), block(64);
    if (dtype == PTTS_BF16) {
        if (head_dim == 64) hipLaunchKernelGGL((paged_attn_simple_kernel<PBF16, 64>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_attn_simple_kernel<PBF16, 128>), grid, block, 0, s, a);
    } else {
        if (head_dim == 64) hipLaunchKernelGGL((paged_attn_simple_kernel<PF32, 64>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((paged_attn_simple_kernel<PF32, 128>), grid, block, 0, s, a);
    }
    return hipGetLastError();
}

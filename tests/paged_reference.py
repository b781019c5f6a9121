"""Plain statements, in 64 bits on the CPU, of the paged-cache operators, and the bounds their results are held to."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # a rounding's largest relative error


def turn(x, cos, sin, rotary_dim, layout):
    """x [tokens, heads, dim], cos / sin [tokens, rotary_dim / 2], all float64; also the sum of the products' magnitudes"""
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = slice(0, rotary_dim // 2), slice(rotary_dim // 2, rotary_dim)
    else:
        a, b = slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)
    out, size = x.clone(), torch.zeros_like(x)
    out[..., a], out[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., b] * cos + x[..., a] * sin
    size[..., a] = (x[..., a] * cos).abs() + (x[..., b] * sin).abs()
    size[..., b] = (x[..., b] * cos).abs() + (x[..., a] * sin).abs()
    return out, size


def turn_bound(out, size, dtype):
    """table rounded (2^-24), product rounded, difference rounded: 3 x 2^-24 of the products' magnitudes, then the result's own rounding
    (relative to what is rounded, which is off by the first part already)"""
    h = HALF_STEP[dtype]
    inner = 3.1 * 2.0 ** -24 * size
    return inner + (0 if dtype == torch.float32 else h) * (out.abs() + inner) + 1e-37


def gather(cache, pages, keys):
    """the first `keys` rows of a sequence out of [pages, heads, page_tokens, dim] -> [heads, keys, dim] float64"""
    t = cache[pages].double().permute(1, 0, 2, 3)
    return t.reshape(t.shape[0], -1, t.shape[3])[:, :keys]


def attend(q, k_cache, v_cache, table, past, starts, scale, causal=True, key_mask=None):
    """-> (out, bound) float64 [tokens, heads, dim] over the rows of the batch's sequences (others NaN).

    The bound, term by term: a score is off by a float32 dot product of D terms (D + 2 roundings of 2^-24 of sum |q k|, doubled for the
    matrix unit's own order) times the scale, and by the rounding of its argument of exp2 and exp2 itself (8 x 2^-24 of 1 + |score|, the
    subtraction of the maximum included).  A weight is off by that much relatively; in bfloat16 it is rounded once more (2^-8).  The sums over
    n keys add n x 2^-24 of sum p |v|.  The output is rounded at the end."""
    dtype = q.dtype
    half = HALF_STEP[dtype]
    tokens, heads, dim = q.shape
    kv_heads = k_cache.shape[1]
    group = heads // kv_heads
    out = torch.full((tokens, heads, dim), math.nan, dtype=torch.float64)
    bound = torch.full((tokens, heads, dim), math.nan, dtype=torch.float64)
    for s in range(len(past)):
        a, b = starts[s], starts[s + 1]
        n, p = b - a, past[s]
        keys = p + n if causal else p
        if n == 0:
            continue
        if keys == 0:
            out[a:b], bound[a:b] = 0, 0
            continue
        pages = table[s, : -(-keys // k_cache.shape[2])].long()
        k, v = gather(k_cache, pages, keys), gather(v_cache, pages, keys)
        seen = torch.ones(n, keys, dtype=torch.bool)
        if causal:
            seen = torch.arange(keys)[None] <= torch.arange(n)[:, None] + p
        if key_mask is not None:
            w = min(keys, key_mask.shape[1])
            live = torch.ones(keys, dtype=torch.bool)
            live[:w] = key_mask[s, :w].bool()
            seen = seen & live
        for h in range(heads):
            x, kk, vv = q[a:b, h].double(), k[h // group], v[h // group]
            used = seen.any(0)                       # keys nobody sees may hold anything
            kk, vv = torch.where(used[:, None], kk, 0), torch.where(used[:, None], vv, 0)
            sc = torch.where(seen, x @ kk.T * scale, -math.inf)
            m = sc.amax(-1, keepdim=True)
            m = torch.where(m == -math.inf, 0, m)
            e = torch.exp(sc - m)
            tot = e.sum(-1, keepdim=True)
            w = e / torch.where(tot == 0, 1, tot)
            # a value that is not finite may only reach the rows that see its key
            o = torch.stack([(w[i][:, None] * torch.where(seen[i][:, None], vv, 0)).sum(0) for i in range(n)]) if not vv.isfinite().all() else w @ vv
            size = w @ vv.abs() if vv.isfinite().all() else o.abs()
            err = (2 * (dim + 2) * 2.0 ** -24 * (x.abs() @ kk.abs().T) * scale + 8 * 2.0 ** -24 * (1 + torch.where(seen, sc, 0).abs()))
            err = torch.where(seen, err, 0).amax(-1, keepdim=True)
            rel = 2 * err + (half if dtype == torch.bfloat16 else 0) + (keys + 16) * 2.0 ** -24
            out[a:b, h] = o
            bound[a:b, h] = rel * size + half * (o.abs() + rel * size) + 1e-30
    return out, bound


def make_batch(lengths, page, extra_pages=2, seed=0, width=None):
    """[(new, past), ...] -> starts (list), past (list), table [n, width] int32 of pages in no order, number of pages"""
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + p) // page) for n, p in lengths]
    ids = torch.randperm(sum(need) + extra_pages, generator=g).int()
    table = torch.full((len(lengths), width or max(max(need), 1)), 0, dtype=torch.int32)
    at, starts = 0, [0]
    for s, m in enumerate(need):
        table[s, :m] = ids[at:at + m]
        at += m
        starts.append(starts[-1] + lengths[s][0])
    return starts, [p for _, p in lengths], table, ids.numel()

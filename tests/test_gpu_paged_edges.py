"""Paged-cache operators at their edges: rows that a bad page concerns, contexts near the largest, starts that wrap, calls across streams.
References and bounds: tests/paged_reference.py."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import BF, F32, close, ints, paged, rnd  # noqa: F401  (paged: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("heads,kv_heads", [(8, 1), (16, 1), (16, 2)])
@pytest.mark.parametrize("page", [16, 64])
def test_every_head_of_a_row_that_meets_a_bad_page_is_nan(paged, page, heads, kv_heads, dtype, dim):
    """Few rows, many of them per key head, so that every wave of a workgroup finishes some: a bad id at the first, a middle and the last page
    of the context (whole, and in shares) may not be taken for page 0, which holds another sequence's keys."""
    from parler_tts_amd._hip import PttsError

    for keys in (20, 300, 6000):
        starts, past, table, pages = ref.make_batch([(1, keys - 1), (1, 30)], page, seed=keys)
        own = -(-keys // page)
        table[table == 0], table[1, 0] = int(table[1, 0]), 0                  # page 0 is the other sequence's
        kc, vc = rnd(2, pages, kv_heads, page, dim, dtype=dtype), rnd(3, pages, kv_heads, page, dim, dtype=dtype)
        q = rnd(1, 2, heads, dim, dtype=dtype)
        want, bound = ref.attend(q, kc, vc, table, past, starts, dim ** -0.5)
        cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
        for at in sorted({0, 1, own // 3, own // 2, own - 2, own - 1} & set(range(own))):
            bad = table.clone()
            bad[0, at] = pages if at % 2 else -1
            for begins in (None, ints(starts)):
                got = paged.paged_attention(q.cuda(), cache, bad.cuda(), ints(past), begins, max_new=1)
                assert got[0].isnan().all(), (keys, at, got[0].isnan().all(-1).tolist())
                close(got[1:], want[1:], bound[1:], "the other sequence")
                with pytest.raises(PttsError, match="page id"):
                    cache.check()


@pytest.mark.parametrize("kv_heads,keys", [(3, 2143000000), (3, 2 ** 31 - 4096), (1, 2 ** 31 - 8192)])
def test_contexts_near_the_largest(paged, kv_heads, keys):
    """Two pages of 4096 tokens under a context of two thousand million keys: zeros everywhere but on the last page, whose keys score 13 and
    hold ones.  The weights' sum counts whole numbers in float32 (less than 2^24 per lane), the last page's share of it is exact but
    for the exponential (argument 13 log2(e) = 18.8, off by 2 roundings, exp2 by one more: 2^-18 relative) and 257 additions of shares; then
    the output's rounding."""
    page, dim = 4096, 64
    pages = -(-keys // page)
    k = torch.zeros(2, kv_heads, page, dim, dtype=BF)
    k[1] = 1.625                                                          # 64 x 1.625 / 8 = 13
    v = torch.zeros_like(k)
    v[1] = 1.0
    table = torch.zeros(1, pages, dtype=torch.int32)
    table[0, -1] = 1
    cache = paged.PagedKVCache.from_tensors(k.cuda(), v.cuda())
    got = paged.paged_attention(torch.ones(1, kv_heads, dim, dtype=BF, device="cuda"), cache, table.cuda(), ints([keys - 1]))
    last = keys - (pages - 1) * page
    want = last * math.exp(13.0) / (last * math.exp(13.0) + (keys - last))
    assert want > 0.2
    assert (got.double() - want).abs().max() <= want * (2.0 ** -8 + 2.0 ** -17 + 260 * 2.0 ** -24)
    cache.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("seqs", [3, 100, 300])
@pytest.mark.parametrize("max_new", [0, 1])
def test_starts_at_the_ends_of_their_type_own_no_rows(paged, max_new, seqs, dtype):
    """an end of -2^31 behind a first token of 5 would be 2^31 - 5 tokens in 32-bit arithmetic"""
    from parler_tts_amd._hip import PttsError

    low, high = -2 ** 31, 2 ** 31 - 1
    page, heads, dim, total = 16, 4, 64, 20
    kc, vc, q = rnd(2, 2, 2, page, dim, dtype=dtype), rnd(3, 2, 2, page, dim, dtype=dtype), rnd(1, total, heads, dim, dtype=dtype)
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    table = torch.tensor([[0, 1]], dtype=torch.int32).expand(seqs, -1).contiguous()
    past = [3] * seqs
    want, bound = ref.attend(q, kc, vc, table, past[:1], [0, 5], dim ** -0.5)
    for tail in ([low, total], [low, high], [high, low], [low + 1, high], [high, total]):
        starts = [0] + [5] * (seqs - 2) + tail
        out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
        paged.paged_attention(q.cuda(), cache, table.cuda(), ints(past), ints(starts), max_new=max_new, out=out)
        close(out[:5], want[:5], bound[:5], tail)
        assert (out[5:] == 5.0).all(), tail
        with pytest.raises(PttsError, match="starts"):
            cache.check()


@pytest.mark.parametrize("max_new,seqs", [(0, 1 << 21), (1, 1 << 18)], ids=["chunks", "few rows"])
def test_descending_starts_that_give_all_rows_to_every_other_sequence(paged, max_new, seqs):
    """2^31 tiles by number: counts stay at the largest number and ascend.  All sequences read the same keys, so that every row has one result."""
    from parler_tts_amd._hip import PttsError

    tokens, heads, dim, page = 1 << 15, 8, 64, 16
    kc, vc, q = rnd(2, 1, 1, page, dim, dtype=BF), rnd(3, 1, 1, page, dim, dtype=BF), rnd(1, tokens, heads, dim, dtype=BF).cuda()
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
    starts[1::2] = tokens
    past = torch.full((seqs,), page, dtype=torch.int32, device="cuda")
    got = paged.paged_attention(q, cache, table.expand(seqs, -1), past, starts, causal=False, max_new=max_new)
    with pytest.raises(PttsError, match="starts"):
        cache.check()
    want = paged.paged_attention(q, cache, table, past[:1], ints([0, tokens]), causal=False, max_new=max_new)
    assert torch.equal(got, want)
    one, bound = ref.attend(q[:64].cpu(), kc, vc, table.cpu(), [page], [0, 64], dim ** -0.5, causal=False)
    close(got[:64], one, bound)
    cache.check()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_of_a_single_entry_are_not_looked_at(paged, dtype):
    """one token, one head, one page, one key head, one column of a table, each with an odd stride there: the bits of the contiguous call"""
    page, dim = 16, 64

    def odd(t, dim_of_one, stride):
        st = list(t.stride())
        st[dim_of_one] = stride
        return torch.as_strided(t, t.shape, st)

    for heads, tokens, pages in ((4, 1, 3), (1, 5, 3), (2, 3, 1)):
        kv_heads = 1
        kc, vc = rnd(2, pages, kv_heads, page, dim, dtype=dtype).cuda(), rnd(3, pages, kv_heads, page, dim, dtype=dtype).cuda()
        q, k, v = (rnd(i, tokens, h, dim, dtype=dtype).cuda() for i, h in ((4, heads), (5, kv_heads), (6, kv_heads)))
        table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
        rotary = paged.RotaryTable(dim, 64)
        at = [table, ints([page * (pages - 1) + 3]), ints([0, tokens])]
        pos = torch.arange(tokens, dtype=torch.int32, device="cuda")

        def calls(kc, vc, q, k, v, out, table):
            cache = paged.PagedKVCache.from_tensors(kc, vc)
            x = paged.kv_append(cache, k, v, table, *at[1:], rotary=rotary, q=q)
            o = paged.paged_attention(x, cache, table, *at[1:], out=out)
            cache.check()
            return x, o, paged.rotary_embed(q, pos, rotary), kc, vc

        want = calls(kc.clone(), vc.clone(), q, k, v, torch.empty_like(q), table)
        ones = [i for i, m in enumerate((tokens, heads)) if m == 1]
        q2, out = q.clone(), torch.empty_like(q)
        for i in ones:
            q2, out = odd(q2, i, 3), odd(out, i, 5)
        rows = [odd(t, 1, 7) if tokens > 1 else odd(odd(t, 1, 7), 0, 9) for t in (k, v)]
        pools = [odd(t.clone(), 1, 11) if pages > 1 else odd(odd(t.clone(), 1, 11), 0, 13) for t in (kc, vc)]
        wide = torch.zeros(1, 2 * pages, dtype=torch.int32, device="cuda")
        wide[:, ::2] = table
        got = calls(*pools, q2, *rows, out, wide[:, ::2] if pages == 1 else table)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (heads, tokens, pages)


def busy():
    """some 20 ms of work on the current stream (float32 products, 144 TFLOP/s at most)"""
    a = torch.ones(8192, 8192, device="cuda")
    for _ in range(3):
        a = a @ a * 0
    return a


def test_a_check_sees_calls_of_every_stream(paged):
    """a call behind other work on another stream, and a cache made behind it: neither is ready when the host goes on"""
    from parler_tts_amd._hip import PttsError

    k = rnd(1, 4, 2, 16, 64).cuda()
    q, table, past = rnd(2, 1, 2, 64).cuda(), ints([[9, 1]]), ints([3])
    cache, rotary = paged.PagedKVCache.from_tensors(k, k.clone()), paged.RotaryTable(64, 10)
    busy()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        keep = busy()
        paged.paged_attention(q, cache, table, past)
        paged.rotary_embed(q, past + 9, rotary)
    with pytest.raises(PttsError, match="page id"):
        cache.check()
    with torch.cuda.stream(side):
        paged.rotary_embed(q, past, rotary)
        keep = busy()
        late = paged.PagedKVCache.from_tensors(k, k.clone())
    paged.paged_attention(q, late, table, past)
    torch.cuda.synchronize()
    with pytest.raises(PttsError, match="page id"):
        late.check()
    with pytest.raises(PttsError, match="position"):
        rotary.check()
    for x in (cache, late, rotary):
        x.check()
    assert (keep == 0).all()


def test_a_cache_made_while_a_graph_is_captured(paged):
    k, v, q, table, past = rnd(1, 4, 2, 16, 64).cuda(), rnd(2, 4, 2, 16, 64).cuda(), rnd(3, 1, 2, 64).cuda(), ints([[0, 1]]), ints([3])
    want = paged.paged_attention(q, paged.PagedKVCache.from_tensors(k, v), table, past)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = paged.paged_attention(q, paged.PagedKVCache.from_tensors(k, v), table, past)
    for _ in range(3):
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_gradients_of_a_cache_are_refused(paged):
    k, q, table, past = rnd(1, 4, 2, 16, 64).cuda(), rnd(3, 1, 2, 64).cuda(), ints([[0, 1]]), ints([3])
    leaf = k.clone().requires_grad_()
    with pytest.raises(ValueError, match="requires a gradient"):
        paged.PagedKVCache.from_tensors(k, leaf)
    with torch.no_grad():
        kept = paged.PagedKVCache.from_tensors(leaf, k)
        paged.paged_attention(q, kept, table, past)
    with pytest.raises(ValueError, match="cache.k requires a gradient"):
        paged.paged_attention(q, kept, table, past)
    with pytest.raises(ValueError, match="cache.k requires a gradient"):
        paged.kv_append(kept, q, q, table, past)


def test_what_a_call_writes_counts_as_changed_in_place(paged):
    """autograd notices that what it saved is no longer there"""
    k, q, table, past = rnd(1, 4, 2, 16, 64).cuda(), rnd(3, 1, 2, 64).cuda(), ints([[0, 1]]), ints([3])
    pool = torch.stack([k, k])
    cache, rotary = paged.PagedKVCache.from_tensors(pool[0], pool[1]), paged.RotaryTable(64, 10)
    w = torch.ones((), device="cuda", requires_grad=True)
    out = torch.empty_like(q)
    for write, tensor in ((lambda: paged.kv_append(cache, q, q, table, past), cache.k), (lambda: paged.kv_append(cache, q, q, table, past), pool),
                          (lambda: paged.kv_append(cache, q, q, table, past, rotary=rotary, q=q, q_out=out), out),
                          (lambda: paged.paged_attention(q, cache, table, past, out=out), out),
                          (lambda: paged.rotary_embed(q, past, rotary, out=out), out)):
        loss = (w * tensor).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    for read in (cache.k, q):                               # what a call only reads keeps its version
        loss = (w * read).sum()
        paged.paged_attention(q, cache, table, past, out=out)
        paged.rotary_embed(q, past, rotary, out=out)
        loss.backward()
    with torch.inference_mode():
        paged.kv_append(cache, q, q, table, past, q=q, q_out=torch.empty_like(q))


def test_the_tensors_of_a_cache_stay_those_the_kernels_know(paged):
    cache, table, past = paged.PagedKVCache(4, 16, 2, 64, dtype=F32), ints([[0, 1]]), ints([3])
    q = rnd(1, 1, 2, 64).cuda()
    for name in ("k", "v", "status", "kv_heads", "device"):
        with pytest.raises(AttributeError, match=f"PagedKVCache.{name} is fixed"):
            setattr(cache, name, getattr(cache, name))
    cache.layer = 7
    cache.k[:] = 1.0                                        # their contents are the caller's
    paged.paged_attention(q, cache, table, past)
    rotary = paged.RotaryTable(64, 16)
    rotary.sin.data = rotary.sin.data.clone()
    with pytest.raises(ValueError, match="sin has other memory"):
        paged.kv_append(cache, q, q, table, past, rotary=rotary)
    cache.v.data = cache.v.data.clone()
    for call in (lambda: paged.paged_attention(q, cache, table, past), lambda: paged.kv_append(cache, q, q, table, past)):
        with pytest.raises(ValueError, match="v has other memory"):
            call()


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("n", [5, 100, 200])
def test_each_kind_of_bad_entry_sets_its_own_bit(paged, n, single):
    """lengths of -3 and 2^31 - 1, and a bad page, each alone and together: the bits of the status word, and NaN in the rows concerned alone"""
    dim = 64
    starts, past, table, pages = ref.make_batch([(1 if single else 1 + i % 4, 30 + i % 50) for i in range(n)], 16)
    kc, vc, q = rnd(2, pages, 1, 16, dim), rnd(3, pages, 1, 16, dim), rnd(1, starts[-1], 1, dim)
    want, bound = ref.attend(q, kc, vc, table, past, starts, 0.125)
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    for spoiled, bits in (([("page", 1)], 2), ([("past", 2, -3)], 4), ([("past", 3, 2 ** 31 - 1)], 4), ([("page", 0), ("past", n - 1, -3)], 6)):
        t, p, keep = table.clone(), list(past), torch.ones(starts[-1], dtype=torch.bool)
        for what in spoiled:
            if what[0] == "page":
                t[what[1], 1] = -5
            else:
                p[what[1]] = what[2]
            keep[starts[what[1]]:starts[what[1] + 1]] = False
        got = paged.paged_attention(q.cuda(), cache, t.cuda(), ints(p), None if single else ints(starts))
        assert int(cache.status) == bits
        assert got[~keep.cuda()].isnan().all()
        close(got[keep.cuda()], want[keep], bound[keep])
        cache.status.zero_()


def test_inference_mode_and_its_tensors(paged):
    """they have no version to raise: caches and outputs made inside are served, inside and outside"""
    k, q, table, past = rnd(1, 4, 2, 16, 64).cuda(), rnd(3, 1, 2, 64).cuda(), ints([[0, 1]]), ints([3])
    base = paged.PagedKVCache.from_tensors(k.clone(), k.clone())
    want = paged.paged_attention(paged.kv_append(base, q, q, table, past, q=q), base, table, past)
    with torch.inference_mode():
        cache, out, turned = paged.PagedKVCache(4, 16, 2, 64, dtype=F32), torch.empty_like(q), torch.empty_like(q)
    for inside in (True, False):
        with torch.inference_mode(inside):
            if inside:
                cache.k.copy_(k)
                cache.v.copy_(k)
            paged.kv_append(cache, q, q, table, past, q=q, q_out=turned)
            assert paged.paged_attention(turned, cache, table, past, out=out) is out
            assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (F32, 64), (BF, 128), (F32, 128)])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("top,spoiled", [(5990, 100), (10, 5000), (3000, 3001)], ids=["behind", "in front", "beside"])
def test_values_that_are_not_finite_count_however_small_their_weight(paged, top, spoiled, new, dtype, dim):
    """one key scores 120 more than the rest, whose weights of e^-120 are 0 in float32: 0 times NaN or infinity is still no number, whichever share
    the value lies in; all else is the top key's value"""
    starts, past, table, pages = ref.make_batch([(new, 6000)], 64)
    kc, vc = torch.zeros(pages, 1, 64, dim, dtype=dtype), rnd(3, pages, 1, 64, dim, dtype=dtype)
    at = lambda key: (int(table[0, key // 64]), 0, key % 64)
    kc[at(top)] = 120.0 / dim ** 0.5
    for feature, value in ((3, math.nan), (5, math.inf), (dim - 1, -math.inf)):
        vc[at(spoiled)][feature] = value
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    got = paged.paged_attention(torch.ones(new, 2, dim, dtype=dtype, device="cuda"), cache, table.cuda(), ints(past), ints(starts), max_new=new)
    lost = [3, 5, dim - 1]
    rest = [i for i in range(dim) if i not in lost]
    assert not got[..., lost].isfinite().any()
    want = vc[at(top)].double()[rest].expand(new, 2, -1)
    # 6000 weights of e^-119 beside one: nothing; the output's rounding of its one value, and a weight of exp2(0) = 1
    close(got[..., rest], want, want.abs() * 2.0 ** -20)

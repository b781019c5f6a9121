"""Paged-cache operators on the GPU against plain statements in 64 bits (tests/paged_reference.py, which also derives the bounds)."""
import math

import pytest
import torch

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def paged():
    from parler_tts_amd import paged

    return paged


def rnd(seed, *shape, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def close(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max()
    assert over <= 0, (what, float(over), float((got - want).abs().max()))


# ---------------------------------------------------------------------------------------------------------------- rotary

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 48), (64, 50), (128, 128), (128, 2), (72, 70), (256, 32)])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (5, 3), (700, 16)])
def test_rotary_embed(paged, dtype, layout, dim, rot, tokens, heads):
    scaling = {"type": "yarn", "factor": 8.0, "original_positions": 512} if rot > 2 else None
    table = paged.RotaryTable(dim, 4001, rotary_dim=rot, layout=layout, scaling=scaling)
    x = rnd(1, tokens, heads, dim, dtype=dtype)
    pos = torch.randint(0, 4001, (tokens,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    pos[0] = 4000
    freq, gain = paged.rotary_frequencies(rot, scaling=scaling)
    ang = pos.double()[:, None] * freq
    want, size = ref.turn(x.double(), torch.cos(ang) * gain, torch.sin(ang) * gain, rot, layout)
    got = paged.rotary_embed(x.cuda(), pos.cuda(), table)
    close(got, want, ref.turn_bound(want, size, dtype))
    assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
    table.check()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides_alignment_and_in_place_agree_to_the_bit(paged, layout):
    table = paged.RotaryTable(64, 100, layout=layout)
    x = rnd(3, 33, 6, 64, dtype=BF).cuda()
    pos = ints([i * 3 for i in range(33)])
    want = paged.rotary_embed(x, pos, table)
    wide = torch.zeros(33, 6, 2, 96, dtype=BF, device="cuda")
    for view in (wide[:, :, 0, :64], wide[:, :, 1, 1:65], wide.permute(1, 0, 2, 3)[:, :, 0, 32:].permute(1, 0, 2)):
        view.copy_(x)
        assert torch.equal(paged.rotary_embed(view, pos, table), want)
        other = torch.full_like(wide, 7.0)
        out = other[:, :, 1, 3:67]
        assert paged.rotary_embed(view, pos, table, out=out) is out and torch.equal(out, want)
        other[:, :, 1, 3:67] = 7.0
        assert (other == 7.0).all()
        assert paged.rotary_embed(view, pos, table, out=view) is view and torch.equal(view, want)
        wide.zero_()
    flat = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(paged.rotary_embed(flat, pos, table), want)
    one = x[:, :1].expand(-1, 6, -1)                        # a broadcast input
    assert torch.equal(paged.rotary_embed(one, pos, table), want[:, :1].expand(-1, 6, -1))
    with pytest.raises(Exception, match="share"):
        paged.rotary_embed(x, pos, table, out=one)


def test_rotary_positions_outside_the_table_give_zeros_and_an_error(paged):
    from parler_tts_amd._hip import PttsError

    table = paged.RotaryTable(64, 100)
    x = rnd(4, 6, 2, 64).cuda()
    got = paged.rotary_embed(x, ints([0, 99, 100, -1, 2 ** 31 - 1, 5]), table)
    assert (got[2:5] == 0).all() and (got[[0, 1, 5]] != 0).any(-1).all()
    with pytest.raises(PttsError, match="position outside"):
        table.check()
    table.check()


def test_rotary_embed_of_nothing(paged):
    table = paged.RotaryTable(64, 100)
    assert paged.rotary_embed(torch.empty(0, 4, 64, device="cuda"), ints([]), table).shape == (0, 4, 64)


# ---------------------------------------------------------------------------------------------------------------- append

APPENDS = [  # lengths (new, past), page, heads, kv heads, dim, rotary dim, layout
    ([(1, 0)], 16, 1, 1, 64, 64, "half"),
    ([(1, 5), (1, 63), (1, 64), (1, 200)], 64, 16, 16, 64, 64, "half"),
    ([(3, 0), (0, 7), (70, 60), (0, 0), (1, 129)], 64, 8, 2, 128, 96, "interleaved"),
    ([(33, 15), (130, 1)], 16, 7, 7, 64, 50, "half"),
    ([(257, 0), (5, 1000)], 128, 4, 1, 128, 128, "interleaved"),
]


def append_inputs(lengths, page, heads, kv_heads, dim, dtype, seed, padding=3):
    starts, past, table, pages = ref.make_batch(lengths, page, seed=seed)
    total = starts[-1] + padding
    q, k, v = (rnd(seed + i, total, h, dim, dtype=dtype) for i, h in ((1, heads), (2, kv_heads), (3, kv_heads)))
    return starts, past, table, pages, q, k, v


def append_reference(lengths, starts, table, k, v, q, kc, vc, freq, rot, layout, dtype):
    """expected caches and q (64 bits) with their bounds; everything else as it was"""
    wk, wv, wq = kc.double(), vc.double(), torch.full(q.shape, 5.0, dtype=torch.float64)
    bk, bv, bq = torch.zeros_like(wk), torch.zeros_like(wv), torch.zeros_like(wq)
    page = kc.shape[2]
    for s, (n, past) in enumerate(lengths):
        for i in range(n):
            t, slot = starts[s] + i, past + i
            ang = torch.tensor([float(slot)], dtype=torch.float64)[:, None] * freq
            p, r = int(table[s, slot // page]), slot % page
            o, size = ref.turn(k[t:t + 1].double(), torch.cos(ang), torch.sin(ang), rot, layout)
            wk[p, :, r], bk[p, :, r] = o[0], ref.turn_bound(o, size, kc.dtype)[0]
            wv[p, :, r] = v[t].to(kc.dtype).double()
            o, size = ref.turn(q[t:t + 1].double(), torch.cos(ang), torch.sin(ang), rot, layout)
            wq[t], bq[t] = o[0], ref.turn_bound(o, size, dtype)[0]
    return wk, bk, wv, bv, wq, bq


@pytest.mark.parametrize("dtype,cache_dtype", [(BF, BF), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{len(c[0])}seq-p{c[1]}-{c[2]}/{c[3]}x{c[4]}-{c[6]}{c[5]}")
def test_kv_append(paged, case, dtype, cache_dtype):
    lengths, page, heads, kv_heads, dim, rot, layout = case
    starts, past, table, pages, q, k, v = append_inputs(lengths, page, heads, kv_heads, dim, dtype, 10)
    kc, vc = rnd(20, pages, kv_heads, page, dim, dtype=cache_dtype), rnd(21, pages, kv_heads, page, dim, dtype=cache_dtype)
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    rotary = paged.RotaryTable(dim, 2000, rotary_dim=rot, layout=layout)
    freq, _ = paged.rotary_frequencies(rot)
    wk, bk, wv, bv, wq, bq = append_reference(lengths, starts, table, k, v, q, kc, vc, freq, rot, layout, dtype)
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    got = paged.kv_append(cache, k.cuda(), v.cuda(), table.cuda(), ints(past), ints(starts), rotary=rotary, q=q.cuda(), q_out=out)
    assert got is out
    close(got, wq, bq, "q")                     # rows behind the last sequence kept their 5.0
    close(cache.k, wk, bk, "k")
    assert torch.equal(cache.v.double().cpu(), wv)
    cache.check()
    if all(n == 1 for n, _ in lengths):         # one token each: the same call without starts
        again = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
        n = len(lengths)
        paged.kv_append(again, k[:n].cuda(), v[:n].cuda(), table.cuda(), ints(past), rotary=rotary)
        assert torch.equal(again.k, cache.k) and torch.equal(again.v, cache.v)


def test_append_layouts_of_rows_and_cache_agree_to_the_bit(paged):
    """slices of one projection's rows, an unaligned slice, a cache whose pages hold [slot][head]; q turned in place"""
    lengths, page, heads, kv_heads, dim = [(5, 3), (0, 0), (66, 61)], 32, 6, 2, 64
    starts, past, table, pages, q, k, v = append_inputs(lengths, page, heads, kv_heads, dim, BF, 30)
    rotary = paged.RotaryTable(dim, 500, rotary_dim=32)
    args = (table.cuda(), ints(past), ints(starts))
    base = paged.PagedKVCache(pages, page, kv_heads, dim)
    want = paged.kv_append(base, k.cuda(), v.cuda(), *args, rotary=rotary, q=q.cuda(), q_out=torch.zeros_like(q).cuda())
    total = q.shape[0]
    for lead in (0, 1):                         # lead 1: rows at odd addresses
        rows = torch.zeros(total, (heads + 2 * kv_heads) * dim + 8, dtype=BF, device="cuda")[:, lead:lead + (heads + 2 * kv_heads) * dim]
        rows = rows.view(total, heads + 2 * kv_heads, dim) if lead == 0 else rows.unflatten(1, (heads + 2 * kv_heads, dim))
        rows.copy_(torch.cat([q, k, v], 1))
        pool = torch.zeros(pages, page, 2, kv_heads, dim, dtype=BF, device="cuda")
        cache = paged.PagedKVCache.from_tensors(pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2))
        qv = rows[:, :heads]
        got = paged.kv_append(cache, rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:], *args, rotary=rotary, q=qv, q_out=qv)
        assert torch.equal(got[:starts[-1]], want[:starts[-1]]) and torch.equal(got[starts[-1]:].cpu(), q[starts[-1]:])
        assert torch.equal(cache.k, base.k) and torch.equal(cache.v, base.v)


def test_append_without_rotation_and_with_given_positions(paged):
    lengths, page = [(4, 2), (3, 17)], 16
    starts, past, table, pages, q, k, v = append_inputs(lengths, page, 2, 2, 64, F32, 40, padding=0)
    args = (table.cuda(), ints(past), ints(starts))
    plain = paged.PagedKVCache(pages, page, 2, 64, dtype=F32)
    assert paged.kv_append(plain, k.cuda(), v.cuda(), *args) is None
    for s, (n, p) in enumerate(lengths):
        for i in range(n):
            assert torch.equal(plain.k[table[s, (p + i) // page], :, (p + i) % page].cpu(), k[starts[s] + i])
    rotary = paged.RotaryTable(64, 50)
    pos = ints([9, 0, 49, 1, 2, 3, 3])
    moved = paged.PagedKVCache(pages, page, 2, 64, dtype=F32)
    got = paged.kv_append(moved, k.cuda(), v.cuda(), *args, rotary=rotary, positions=pos, q=q.cuda())
    assert torch.equal(got, paged.rotary_embed(q.cuda(), pos, rotary))
    turned = paged.PagedKVCache(pages, page, 2, 64, dtype=F32)
    paged.kv_append(turned, paged.rotary_embed(k.cuda(), pos, rotary), v.cuda(), *args)
    assert torch.equal(moved.k, turned.k) and torch.equal(moved.v, plain.v)


def test_append_leaves_out_what_cannot_be_placed(paged):
    from parler_tts_amd._hip import PttsError

    page, width = 16, 2
    k = rnd(50, 8, 2, 64).cuda()
    rotary = paged.RotaryTable(64, 30)
    for table, past, starts, bad_tokens, match in (
            ([[0, 1], [2, 9]], [15, 15], [0, 4, 8], [5, 6, 7], "page id"),
            ([[0, 1], [-1, 2]], [0, 15], [0, 4, 8], [4], "page id"),
            ([[0, 1], [2, 3]], [30, 0], [0, 4, 8], [0, 1, 2, 3], "position|longer"),
            ([[0, 1], [2, 3]], [0, -2], [0, 4, 8], [4, 5, 6, 7], "negative"),
            ([[0, 1], [2, 3]], [0, 0], [0, 4, 11], [4, 5, 6, 7], "starts")):
        cache = paged.PagedKVCache(4, page, 2, 64, dtype=F32)
        q = paged.kv_append(cache, k, k, ints(table), ints(past), ints(starts), rotary=rotary, q=k)
        assert (q[bad_tokens] == 0).all() and (q.flatten(1) != 0).any(1).sum() == 8 - len(bad_tokens)
        assert int((cache.v != 0).any(-1).all(1).sum()) == 8 - len(bad_tokens)
        with pytest.raises(PttsError, match=match):
            cache.check()
        cache.check()


# ---------------------------------------------------------------------------------------------------------------- attention

def attend(paged, lengths, page, heads, kv_heads, dim, dtype, seed=0, causal=True, mask=None, scale=None, max_new=0, single=False, padding=0,
           spread=1.0, k_edit=None):
    starts, past, table, pages = ref.make_batch(lengths, page, seed=seed)
    total = starts[-1] + padding
    q = rnd(seed + 1, total, heads, dim, dtype=dtype)
    kc, vc = rnd(seed + 2, pages, kv_heads, page, dim, dtype=dtype) * spread, rnd(seed + 3, pages, kv_heads, page, dim, dtype=dtype)
    kc = kc.to(dtype)
    if k_edit:
        k_edit(kc, vc, table, past, starts)
    s = dim ** -0.5 if scale is None else scale
    want, bound = ref.attend(q, kc, vc, table, past, starts, s, causal, mask)
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    out = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    got = paged.paged_attention(q.cuda(), cache, table.cuda(), ints(past), None if single else ints(starts), scale=scale, causal=causal,
                                key_mask=None if mask is None else mask.cuda(), max_new=max_new, out=out)
    assert got is out
    n = starts[-1]
    close(got[:n], want[:n], bound[:n], (lengths, page, heads, kv_heads, dim, dtype))
    assert (got[n:] == 5.0).all()
    cache.check()
    return got


SINGLES = [[(1, 0)], [(1, 1)], [(1, 14), (1, 15), (1, 16), (1, 31)], [(1, 62), (1, 63), (1, 64), (1, 65), (1, 127), (1, 128)],
           [(1, 300), (1, 0), (1, 2579), (1, 1000)], [(1, 9000)]]
CHUNKS = [[(2, 0)], [(5, 11), (16, 0), (17, 47)], [(31, 1), (32, 0), (33, 64)], [(127, 0), (128, 3), (129, 200)],
          [(1, 100), (0, 50), (200, 0), (0, 0), (64, 64), (1, 0)], [(700, 130)]]
SHAPES = [(4, 4, 64), (8, 2, 128), (5, 1, 64), (3, 3, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("lengths", SINGLES, ids=lambda l: "+".join(str(p) for _, p in l))
def test_single_tokens(paged, lengths, heads, kv_heads, dim, dtype):
    one = attend(paged, lengths, 64, heads, kv_heads, dim, dtype, single=True)
    two = attend(paged, lengths, 64, heads, kv_heads, dim, dtype, max_new=1)
    assert torch.equal(one, two)
    attend(paged, lengths, 16, heads, kv_heads, dim, dtype, seed=5)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("lengths", CHUNKS, ids=lambda l: "+".join(f"{n}@{p}" for n, p in l))
def test_chunks(paged, lengths, heads, kv_heads, dim, dtype):
    attend(paged, lengths, 64, heads, kv_heads, dim, dtype, padding=3)
    attend(paged, lengths, 32, heads, kv_heads, dim, dtype, seed=7, max_new=max(n for n, _ in lengths))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[(1, 40), (1, 0)], [(3, 70), (40, 0), (20, 200)]], ids=["single", "chunk"])
def test_not_causal(paged, lengths, dtype):
    """states that were cached once: every token sees the same keys, none at all where past is 0"""
    attend(paged, lengths, 16, 4, 2, 64, dtype, causal=False, padding=1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("group", [1, 2, 3, 6, 16, 20, 33])
def test_groups_of_heads(paged, group, dtype):
    attend(paged, [(1, 77), (1, 500)], 64, group * 2, 2, 64, dtype, single=True)
    attend(paged, [(3, 77), (9, 130)], 64, group, 1, 128, dtype, max_new=9)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_pages(paged, page, dtype):
    attend(paged, [(40, page - 1), (1, page), (17, 2 * page + 5)], page, 2, 2, 64, dtype)
    attend(paged, [(1, page - 1), (1, page), (1, 3 * page)], page, 2, 1, 128, dtype, single=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths,single", [([(1, 99), (1, 200), (1, 5), (1, 0)], True), ([(70, 30), (1, 200), (6, 0), (40, 100)], False)], ids=["single", "chunk"])
def test_key_masks(paged, lengths, single, dtype):
    """padding in front, holes, a mask that leaves rows (or everything) empty, narrower and wider than the keys, one row for all"""
    g = torch.Generator().manual_seed(3)
    for width in (1, 7, 64, 150, 400):
        mask = torch.rand(4, width, generator=g) < 0.5
        mask[0, :3] = False
        mask[2] = False                                     # nothing left where the mask covers every key
        attend(paged, lengths, 16, 4, 2, 64, dtype, mask=mask, single=single)
    attend(paged, lengths, 64, 4, 4, 128, dtype, mask=torch.zeros(4, 400, dtype=torch.bool), single=single)
    attend(paged, lengths, 64, 4, 4, 64, dtype, mask=torch.tensor([[False] * 5 + [True]]).expand(4, 6), single=single)
    attend(paged, lengths, 64, 4, 4, 64, dtype, mask=torch.zeros(4, 0, dtype=torch.bool), single=single)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lengths,single", [([(1, 20), (1, 140)], True), ([(70, 30), (5, 0), (40, 100)], False)], ids=["single", "chunk"])
def test_what_masked_and_unused_places_hold_does_not_matter(paged, lengths, single, dtype, poison):
    def edit(kc, vc, table, past, starts):
        page = kc.shape[2]
        used = torch.zeros(kc.shape[0], page, dtype=torch.bool)
        for s in range(len(past)):
            for j in range(past[s] + starts[s + 1] - starts[s]):
                used[table[s, j // page], j % page] = not (2 <= j < 5)     # keys 2 .. 4 are masked
        for c in (kc, vc):
            c.permute(0, 2, 1, 3)[~used] = poison

    mask = torch.ones(len(lengths), 9, dtype=torch.bool)
    mask[:, 2:5] = False
    for heads, kv_heads, dim, page in ((4, 4, 64, 64), (4, 1, 128, 16)):
        attend(paged, lengths, page, heads, kv_heads, dim, dtype, mask=mask, k_edit=edit, single=single)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_a_value_that_is_not_finite_reaches_only_the_rows_that_see_it(paged, dtype, poison):
    """token 37's key and value are not finite: the tokens in front of it do not notice"""
    page, n = 64, 90
    starts, past, table, pages = ref.make_batch([(n, 10)], page)
    for where in ("k", "v", "both"):
        kc, vc = rnd(2, pages, 2, page, 64, dtype=dtype), rnd(3, pages, 2, page, 64, dtype=dtype)
        clean_k, clean_v = kc.clone(), vc.clone()
        p, r = int(table[0, 47 // page]), 47 % page
        if where != "v":
            kc[p, :, r] = math.nan
        if where != "k":
            vc[p, :, r, 5:40] = poison
        q = rnd(1, n, 4, 64, dtype=dtype)
        want, bound = ref.attend(q, clean_k, clean_v, table, past, starts, 0.125)
        cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
        got = paged.paged_attention(q.cuda(), cache, table.cuda(), ints(past), ints(starts))
        close(got[:37], want[:37], bound[:37], where)
        if where != "v":
            assert got[37:].isnan().all()
        else:
            assert not got[37:, :, 5:40].isfinite().any()
            close(got[37:, :, :5], want[37:, :, :5], bound[37:, :, :5], where)
            close(got[37:, :, 40:], want[37:, :, 40:], bound[37:, :, 40:], where)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scores_of_every_size(paged, dtype):
    """nearly one-hot rows, flat rows, a scale of one, running maxima that rise with every tile"""
    attend(paged, [(60, 200), (1, 300)], 64, 2, 2, 64, dtype, spread=12.0)
    attend(paged, [(60, 200), (1, 300)], 64, 2, 2, 64, dtype, spread=1e-3)
    attend(paged, [(60, 200), (1, 300)], 64, 2, 2, 128, dtype, scale=1.0)
    attend(paged, [(1, 600)], 64, 2, 2, 64, dtype, single=True, spread=12.0)

    def rising(kc, vc, table, past, starts):
        page = kc.shape[2]
        for j in range(past[0] + starts[1]):
            kc[table[0, j // page], :, j % page] = (kc[table[0, j // page], :, j % page].float() * 0.05 * (1 + j / 16)).to(kc.dtype)

    attend(paged, [(70, 500)], 64, 2, 2, 64, dtype, k_edit=rising)
    attend(paged, [(1, 570)], 64, 2, 2, 64, dtype, k_edit=rising, single=True)


def test_strides_of_q_out_and_cache_agree_to_the_bit(paged):
    lengths, page, heads, kv_heads, dim = [(20, 30), (1, 100), (7, 0)], 32, 4, 2, 64
    for single in (False, True):
        lengths = [(1, p) for _, p in lengths] if single else lengths
        starts, past, table, pages = ref.make_batch(lengths, page)
        q, kc, vc = rnd(1, starts[-1], heads, dim, dtype=BF).cuda(), rnd(2, pages, kv_heads, page, dim, dtype=BF).cuda(), rnd(3, pages, kv_heads, page, dim, dtype=BF).cuda()
        args = (table.cuda(), ints(past), None if single else ints(starts))
        want = paged.paged_attention(q, paged.PagedKVCache.from_tensors(kc, vc), *args)
        pool = torch.zeros(pages, page, 2, kv_heads, dim, dtype=BF, device="cuda")
        pool[:, :, 0], pool[:, :, 1] = kc.transpose(1, 2), vc.transpose(1, 2)
        cache = paged.PagedKVCache.from_tensors(pool[:, :, 0].transpose(1, 2), pool[:, :, 1].transpose(1, 2))
        rows = torch.zeros(starts[-1], heads + 3, dim + 8, dtype=BF, device="cuda")
        rows[:, 1:1 + heads, :dim] = q
        out = torch.full((heads, starts[-1], dim + 16), 5.0, dtype=BF, device="cuda")
        got = paged.paged_attention(rows[:, 1:1 + heads, :dim], cache, *args, out=out[..., 8:8 + dim].transpose(0, 1))
        assert torch.equal(got, want) and (out[..., :8] == 5.0).all() and (out[..., 8 + dim:] == 5.0).all()
        wide = torch.zeros(table.shape[0], table.shape[1] + 9, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table.cuda()
        assert torch.equal(paged.paged_attention(q, cache, wide[:, :table.shape[1]], *args[1:]), want)
        close(paged.paged_attention(q, cache, wide, *args[1:]), want.double().cpu(), 2 ** -7 * want.double().abs().cpu() + 2 ** -7, "wider table")
        with pytest.raises(Exception, match="share"):
            paged.paged_attention(q, cache, *args, out=q)
        both = torch.full((starts[-1], 2 * heads + 1, dim), 5.0, dtype=BF, device="cuda")     # q and out beside each other in one buffer's rows
        for at, to in ((0, heads + 1), (heads + 1, 1)):
            both.fill_(5.0)
            both[:, at:at + heads] = q
            got = paged.paged_attention(both[:, at:at + heads], cache, *args, out=both[:, to:to + heads])
            rest = [i for i in range(2 * heads + 1) if not (at <= i < at + heads or to <= i < to + heads)]
            assert torch.equal(got, want) and torch.equal(both[:, at:at + heads], q) and (both[:, rest] == 5.0).all()
        with pytest.raises(Exception, match="share"):
            paged.paged_attention(both[:, :heads], cache, *args, out=both[:, heads - 1:2 * heads - 1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("single", [True, False])
def test_bad_pages_and_lengths_give_nan_rows_and_an_error(paged, single, dtype):
    from parler_tts_amd._hip import PttsError

    page, heads, dim = 16, 2, 64
    new = 1 if single else 20
    for table, past, bad, match in (([[0, 1, 2, 3], [4, 5, 99, 6]], [20, 20], None, "page id"), ([[0, 1, 2, 3], [4, -1, 6, 7]], [20, 20], 1, "page id"),
                                    ([[0, 1, 2, 3], [4, 5, 6, 7]], [20, 64], 1, "longer"), ([[0, 1, 2, 3], [4, 5, 6, 7]], [20, -1], 1, "negative"),
                                    ([[0, 1, 2, 3], [4, 5, 6, 7]], [20, 2 ** 31 - 1], 1, "longer")):
        starts = [0, new, 2 * new]
        kc, vc, q = rnd(2, 8, heads, page, dim, dtype=dtype), rnd(3, 8, heads, page, dim, dtype=dtype), rnd(1, 2 * new, heads, dim, dtype=dtype)
        cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
        got = paged.paged_attention(q.cuda(), cache, ints(table), ints(past), None if single else ints(starts))
        want, bound = ref.attend(q[:new], kc, vc, torch.tensor(table)[:1], past[:1], [0, new], dim ** -0.5)
        close(got[:new], want, bound, "the other sequence")
        if bad is not None:
            rows = got[new:]
            if match == "longer" and past[1] == 64 and not single:
                assert rows.isnan().all()
            if match == "page id":
                rows = rows[-1:]
            assert rows.isnan().all()
            with pytest.raises(PttsError, match=match):
                cache.check()
        elif not single:                      # page 99 is reached by the tokens from slot 32 on
            assert got[-8:].isnan().all()
            with pytest.raises(PttsError, match=match):
                cache.check()
        else:                                 # ... and by no token of the shorter batch
            cache.check()
            want, bound = ref.attend(q[1:], kc, vc, torch.tensor(table)[1:], past[1:], [0, 1], dim ** -0.5)
            close(got[1:], want, bound)


def test_bad_starts_are_not_followed(paged):
    from parler_tts_amd._hip import PttsError

    kc = rnd(2, 8, 2, 16, 64).cuda()
    for starts in ([0, 10, 400], [0, 300, 20], [-7, 5, 20], [5, 2, 1]):
        cache = paged.PagedKVCache.from_tensors(kc, kc.clone())
        out = torch.zeros(20, 2, 64, device="cuda")
        paged.paged_attention(rnd(1, 20, 2, 64).cuda(), cache, ints([[0, 1, 2, 3], [4, 5, 6, 7]]), ints([3, 3]), ints(starts), out=out)
        with pytest.raises(PttsError, match="starts"):
            cache.check()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_offsets_past_32_bits(paged, dtype):
    """pages whose elements lie past 2^32 of the cache's first, for reads and for writes"""
    heads, page, dim, gap = 2, 64, 128, 1 << 20
    n_pages = (1 << 32) // gap + 6
    buf = torch.empty(n_pages * gap, dtype=dtype, device="cuda")
    k = torch.as_strided(buf, (n_pages, heads, page, dim), (gap, page * dim, dim, 1))
    v = torch.as_strided(buf, (n_pages, heads, page, dim), (gap, page * dim, dim, 1), heads * page * dim)
    ids = torch.tensor([[n_pages - 1, 0, n_pages - 3], [1, n_pages - 2, 2]], dtype=torch.int32)
    cache = paged.PagedKVCache.from_tensors(k, v)
    small = paged.PagedKVCache(6, page, heads, dim, dtype=dtype)
    few = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    rotary = paged.RotaryTable(dim, 200)
    kk, vv, q = rnd(1, 300, heads, dim, dtype=dtype).cuda(), rnd(2, 300, heads, dim, dtype=dtype).cuda(), rnd(3, 300, 4, dim, dtype=dtype).cuda()
    outs = []
    for c, t in ((cache, ids), (small, few)):
        at = (t.cuda(), ints([0, 0]), ints([0, 150, 300]))
        x = paged.kv_append(c, kk, vv, *at, rotary=rotary, q=q)
        o = paged.paged_attention(x, c, *at)
        one = paged.paged_attention(x[:2], c, t.cuda(), ints([149, 120]))
        outs.append((x, o, one))
        c.check()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    for s in range(2):
        for j in range(3):
            rows = min(page, 150 - 64 * j)
            assert torch.equal(cache.k[ids[s, j], :, :rows], small.k[few[s, j], :, :rows])
            assert torch.equal(cache.v[ids[s, j], :, :rows], small.v[few[s, j], :, :rows])


# ---------------------------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_serving_in_chunks_equals_one_attention_over_everything(paged, dtype, layout):
    """three sequences arrive in chunks of unlike size, then grow token by token: every output against causal attention over the whole
    sequence, from the rows that went in (rotation included)"""
    heads, kv_heads, dim, page = 6, 2, 64, 16
    total = [75, 40, 130]
    g = torch.Generator().manual_seed(0)
    q, k, v = ([rnd(10 * i + s, n, h, dim, dtype=dtype) for s, n in enumerate(total)] for i, h in ((1, heads), (2, kv_heads), (3, kv_heads)))
    _, _, table, pages = ref.make_batch([(n, 0) for n in total], page)
    rotary = paged.RotaryTable(dim, 256, layout=layout, rotary_dim=48)
    cache = paged.PagedKVCache(pages, page, kv_heads, dim, dtype=dtype)
    done, outs = [0, 0, 0], [[], [], []]
    rounds = [[30, 0, 64], [1, 33, 1], [40, 1, 60]]
    while any(d < n for d, n in zip(done, total)):
        want = rounds.pop(0) if rounds else [1, 1, 1]
        step = [min(w, n - d) for w, n, d in zip(want, total, done)]
        starts = [0, step[0], step[0] + step[1], sum(step)]
        take = lambda rows: torch.cat([r[d:d + n] for r, d, n in zip(rows, done, step)]).cuda()
        at = (table.cuda(), ints(done), ints(starts))
        x = paged.kv_append(cache, take(k), take(v), *at, rotary=rotary, q=take(q))
        o = paged.paged_attention(x, cache, *at)
        for s in range(3):
            outs[s].append(o[starts[s]:starts[s + 1]].cpu())
            done[s] += step[s]
    cache.check()
    for s, n in enumerate(total):
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        xq = paged.rotary_embed(q[s].cuda(), pos, rotary).cpu()
        keys = paged.rotary_embed(k[s].cuda(), pos, rotary).cpu()
        pad = -(-n // page) * page - n
        blocks = lambda t: torch.cat([t, torch.zeros(pad, kv_heads, dim, dtype=dtype)]).reshape(-1, page, kv_heads, dim).transpose(1, 2)
        ids = torch.arange((n + pad) // page, dtype=torch.int32)[None]
        want, bound = ref.attend(xq, blocks(keys), blocks(v[s]), ids, [0], [0, n], dim ** -0.5)
        close(torch.cat(outs[s]), want, bound, s)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_steps_replay_with_other_lengths_beside_eager_work(paged, dtype):
    """one decode step captured twice (two graphs), replayed with lengths that grow in place, eager calls between the replays"""
    heads, kv_heads, dim, page, n = 4, 2, 64, 16, 3
    pages = n * 8
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().reshape(n, 8).cuda()
    rotary = paged.RotaryTable(dim, 128)
    filled = (rnd(2, pages, kv_heads, page, dim, dtype=dtype).cuda(), rnd(3, pages, kv_heads, page, dim, dtype=dtype).cuda())
    cache = paged.PagedKVCache.from_tensors(filled[0].clone(), filled[1].clone())
    eager = paged.PagedKVCache.from_tensors(filled[0].clone(), filled[1].clone())
    past = ints([0, 17, 100])
    q, k, v = (torch.empty(n, h, dim, dtype=dtype, device="cuda") for h in (heads, kv_heads, kv_heads))

    def step(c, at):
        x = paged.kv_append(c, k, v, table, at, rotary=rotary, q=q)
        return paged.paged_attention(x, c, table, at)

    for t in (q, k, v):
        t.copy_(rnd(9, *t.shape, dtype=dtype))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, past)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(cache, past)
        graphs.append((g, o))
    cache.k.copy_(filled[0]); cache.v.copy_(filled[1])
    at = past.clone()
    for i in range(12):
        for j, t in enumerate((q, k, v)):
            t.copy_(rnd(100 + 3 * i + j, *t.shape, dtype=dtype))
        want = step(eager, at)
        g, o = graphs[i % 2]
        g.replay()
        junk = step(eager, at)                # the same rows again, beside the replay
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(junk, want), i
        past.add_(1)
        at.add_(1)
    assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)
    cache.check()


def test_other_streams_and_two_calls_at_once(paged):
    """two streams work on two batches of one cache at the same time; results equal those of the calls alone, bit for bit"""
    heads, kv_heads, dim, page = 8, 8, 64, 64
    starts, past, table, pages = ref.make_batch([(1, 2000 + 37 * s) for s in range(12)], page)
    cache = paged.PagedKVCache.from_tensors(rnd(2, pages, kv_heads, page, dim, dtype=BF).cuda(), rnd(3, pages, kv_heads, page, dim, dtype=BF).cuda())
    q = rnd(1, 12, heads, dim, dtype=BF).cuda()
    halves = [(q[:6], table[:6].cuda(), ints(past[:6])), (q[6:], table[6:].cuda(), ints(past[6:]))]
    want = [paged.paged_attention(a, cache, t, p) for a, t, p in halves]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, (a, t, p) in zip(streams, halves):
            with torch.cuda.stream(s):
                got.append(paged.paged_attention(a, cache, t, p))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_results_do_not_change_from_call_to_call(paged):
    starts, past, table, pages = ref.make_batch([(300, 900), (1, 2000), (40, 0)], 64)
    for dtype in (BF, F32):
        cache = paged.PagedKVCache.from_tensors(rnd(2, pages, 2, 64, 128, dtype=dtype).cuda(), rnd(3, pages, 2, 64, 128, dtype=dtype).cuda())
        q = rnd(1, starts[-1], 8, 128, dtype=dtype).cuda()
        first = paged.paged_attention(q, cache, table.cuda(), ints(past), ints(starts))
        for _ in range(4):
            assert torch.equal(paged.paged_attention(q, cache, table.cuda(), ints(past), ints(starts)), first)


def test_wrapper_refusals(paged):
    cache = paged.PagedKVCache(4, 16, 2, 64)
    table, past, starts = ints([[0, 1], [2, 3]]), ints([3, 3]), ints([0, 1, 2])
    q = torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    k = torch.zeros(2, 2, 64, dtype=BF, device="cuda")
    good = lambda **kw: paged.paged_attention(**{**dict(q=q, cache=cache, table=table, past=past, starts=starts), **kw})
    good()
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q.cpu()), dict(q=q[..., :32]), dict(q=q[0]), dict(table=table.long()), dict(table=table[:1]),
                dict(past=past.cpu()), dict(past=past.float()), dict(starts=starts[:2]), dict(starts=None, q=q[:1]), dict(scale=0.0), dict(scale=math.nan),
                dict(key_mask=torch.ones(2, 5, device="cuda")), dict(key_mask=torch.ones(3, 5, dtype=torch.bool, device="cuda")), dict(out=q.float()),
                dict(out=torch.zeros(2, 2, 64, dtype=BF, device="cuda")), dict(max_new=-1), dict(out=q), dict(q=q.clone().requires_grad_())):
        with pytest.raises((ValueError, RuntimeError)):
            good(**bad)
    put = lambda **kw: paged.kv_append(**{**dict(cache=cache, k=k, v=k, table=table, past=past, starts=starts), **kw})
    put()
    rotary = paged.RotaryTable(64, 32)
    for bad in (dict(k=k[:1]), dict(v=k.float()), dict(k=k[:, :1]), dict(q=q.float()), dict(q_out=q), dict(positions=past), dict(rotary=paged.RotaryTable(128, 32)),
                dict(rotary=rotary, positions=past.long()), dict(rotary=rotary, positions=past[:1]), dict(q=q, q_out=q[:, :2]), dict(k=k.double(), v=k.double())):
        with pytest.raises((ValueError, RuntimeError)):
            put(**bad)
    full = paged.PagedKVCache(4, 16, 2, 64, dtype=F32)
    with pytest.raises((ValueError, RuntimeError)):
        put(cache=full)                          # bfloat16 rows into a float32 cache


def test_empty_batches(paged):
    cache = paged.PagedKVCache(4, 16, 2, 64)
    none = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    table, past = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), ints([])
    assert paged.paged_attention(none, cache, table, past).shape == (0, 2, 64)
    assert paged.kv_append(cache, none, none, table, past) is None
    pad = torch.ones(3, 2, 64, dtype=BF, device="cuda")                   # three padding rows of no sequence
    out = paged.paged_attention(pad, cache, ints([[0, 1]]), ints([0]), ints([0, 0]), out=pad * 5)
    assert (out == 5).all()
    paged.kv_append(cache, pad, pad, ints([[0, 1]]), ints([0]), ints([0, 0]))
    assert (cache.k == 0).all() and (cache.v == 0).all()
    cache.check()

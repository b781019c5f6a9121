"""Paged-cache operators without a GPU, at their edges: memory that tensors share, strides that address nothing, the wrapper's promises."""
import ctypes as C
import math
import random

import pytest
import torch

from parler_tts_amd import _hip, paged
from tests.test_paged_cpu import P, append, attend, batch, kv, lib, rotary, strides  # noqa: F401  (lib: the fixture)

# a call that is not refused reaches the launch, which fails where there is no device (and must not happen on made-up addresses where there is one)
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: for machines without a GPU")
LAUNCHED = -3


def places(at, st, n, esz, inner=64):
    """bytes that rows at `at` take"""
    t = torch.tensor([0])
    for s, m in zip(st, n):
        t = (t[:, None] + torch.arange(m)[None] * s).reshape(-1)
    t = (t[:, None] + torch.arange(inner)[None]).reshape(-1)
    return set(((at + t[:, None] * esz) + torch.arange(esz)[None]).reshape(-1).tolist())


def layout(rng, n, inner=64):
    """strides of rows that do not meet themselves: extents nested in a random order, with gaps"""
    order, st, span = list(range(len(n))), [0] * len(n), inner
    rng.shuffle(order)
    for i in order:
        st[i] = span + rng.choice([0, 0, 1, 17, 64, 3 * 64])
        span += (n[i] - 1) * st[i]
    return st


def is_refused(lib, rc, words):
    assert rc in (-1, LAUNCHED), (rc, lib.ptts_last_error())
    if rc == -1:
        assert words in lib.ptts_last_error(), lib.ptts_last_error()
    return rc == -1


@no_gpu
@pytest.mark.parametrize("seed", range(4))
def test_rows_that_share_memory_are_told_from_rows_beside_each_other(lib, seed):
    """x and out of a rotation, q and out of an attention, q and q_out, q_out and k of an append: against the sets of their bytes"""
    rng = random.Random(seed)
    shared = 0
    for _ in range(300):
        tokens, heads = rng.randint(1, 5), rng.randint(1, 4)
        n = [tokens, heads]
        a, b = layout(rng, n), layout(rng, n)
        if rng.random() < 0.6:
            b = list(a)                                   # slices of one buffer's rows
        bf16 = rng.random() < 0.5
        esz = 2 if bf16 else 4
        off = rng.randint(-(tokens * heads * 100), tokens * heads * 100) * esz
        at = 4 * P + off
        meets = bool(places(4 * P, a, n, esz) & places(at, b, n, esz))
        shared += meets
        same = off == 0 and a == b
        r = rotary()
        rc = lib.ptts_rotary_embed(C.byref(r), int(bf16), tokens, heads, 64, 4 * P, *a, P, at, *b, P, None)
        assert is_refused(lib, rc, b"share memory") == (meets and not same)
        far = kv(dtype=int(bf16), k=64 * P, v=128 * P)
        one = batch(starts=None, tokens=tokens, n_seqs=tokens)
        rc = append(lib, far, one, int(bf16), 256 * P, (128, 64), 512 * P, (128, 64), None, heads, 4 * P, a, at, b)
        assert is_refused(lib, rc, b"share memory") == (meets and not same)
        if all(x % (16 // esz) == 0 for x in a + b) and off % 16 == 0:
            c = kv(dtype=int(bf16), k=64 * P, v=128 * P, kv_heads=1)
            rc = attend(lib, c, one, heads, 4 * P, a, at, b, ws=1024 * P)
            assert is_refused(lib, rc, b"share memory") == meets
        # two key heads beside the query heads
        nk, sk = [tokens, 2], layout(rng, [tokens, 2])
        if rng.random() < 0.6:
            sk[0] = max(a[0], sk[1] + 64)
        over = bool(places(4 * P, sk, nk, esz) & places(at, b, n, esz))
        for first in (True, False):
            rows = (4 * P, sk, 512 * P, (128, 64)) if first else (512 * P, (128, 64), 4 * P, sk)
            rc = append(lib, far, one, int(bf16), *rows, None, heads, 256 * P, (1 << 12, 64), at, b)
            assert is_refused(lib, rc, b"q_out shares memory with k or v") == over
    assert 50 < shared < 250


@no_gpu
@pytest.mark.parametrize("seed", range(2))
def test_rows_within_the_cache_are_told_from_rows_beside_it(lib, seed):
    """out of an attention and all rows of an append against the sets of the cache's bytes: gaps of a cache may hold rows, its slots may not"""
    rng = random.Random(100 + seed)
    refused = 0
    for _ in range(60):
        tokens, pages, dim = rng.randint(1, 20), rng.randint(1, 3), 64
        bf16 = rng.random() < 0.5
        esz = 2 if bf16 else 4
        nc, n = [pages, 2, 16], [tokens, 2]
        st = [8 * x for x in layout(rng, nc, dim // 8)]
        rows = rng.choice([[8 * x for x in layout(rng, n, dim // 8)], [st[2], st[1]]])
        inner, outer = sorted(zip(rows, n))
        if outer[1] > 1 and outer[0] < dim + (inner[1] - 1) * inner[0] or inner[1] > 1 and inner[0] < dim:
            rows = [2 * dim, dim]                         # extents that are not nested count as rows that meet themselves
        span = sum((m - 1) * x for m, x in zip(nc, st)) + dim
        at = 64 * P + 16 * rng.randint(-tokens * 20, span * esz // 16)
        cached = places(64 * P, st, nc, esz)
        meets = bool(cached & places(at, rows, n, esz))
        refused += meets
        one = batch(starts=None, tokens=tokens, n_seqs=tokens)
        for which in ("k", "v"):
            pools = dict(k=64 * P, v=512 * P) if which == "k" else dict(k=512 * P, v=64 * P)
            c = kv(dtype=int(bf16), k_strides=strides(*st), v_strides=strides(*st), n_pages=pages, page_tokens=16, **pools)
            rc = attend(lib, c, one, 2, 128 * P, (128, 64), at, rows, ws=1024 * P)
            assert is_refused(lib, rc, b"out shares memory with the cache") == meets
            clear = [(128 * P, (128, 64)), (136 * P, (128, 64)), (144 * P, (128, 64)), (152 * P, (128, 64))]
            for i in range(4):                            # k, v, q, q_out
                k, v, q, qo = clear[:i] + [(at, rows)] + clear[i + 1:]
                rc = append(lib, c, one, int(bf16), *k, *v, None, 2, *q, *qo)
                assert is_refused(lib, rc, b"share memory with the cache") == meets
        c = kv(dtype=int(bf16), k=64 * P, v=at, k_strides=strides(*st), v_strides=strides(*st), n_pages=pages, page_tokens=16)
        rc = append(lib, c, one, int(bf16), 512 * P, (128, 64), 520 * P, (128, 64))
        assert is_refused(lib, rc, b"keys and values of the cache share memory") == bool(cached & places(at, st, nc, esz))
    assert 5 < refused < 55, refused


def test_keys_that_are_the_values_too_can_be_read_but_not_appended_to(lib):
    c = kv(k=64 * P, v=64 * P)
    assert append(lib, c) == -1 and b"keys and values" in lib.ptts_last_error()
    if not torch.cuda.is_available():
        assert attend(lib, c, ws=1024 * P) == LAUNCHED


@no_gpu
def test_strides_of_a_single_entry_are_not_looked_at(lib):
    """they address nothing and may be anything; of two entries they count"""
    odd = 3
    c1 = kv(k_strides=strides(odd, 4096, 64), v_strides=strides(-odd, 4096, 64), n_pages=1, k=64 * P, v=128 * P)
    h1 = kv(k_strides=strides(8192, odd, 64), v_strides=strides(8192, 1 << 50, 64), kv_heads=1, k=64 * P, v=128 * P)
    far = kv(k=64 * P, v=128 * P)
    one, two = batch(starts=None, tokens=1, n_seqs=1, table_stride=-odd), batch(starts=None, tokens=2, n_seqs=2)
    for c, b, heads, qs, os in ((far, one, 4, (odd, 64), (odd, 64)), (far, one, 4, (-odd, 64), (1 << 50, 64)), (h1, two, 1, (128, odd), (64, -odd)),
                                (c1, two, 2, (128, 64), (128, 64)), (h1, two, 2, (128, 64), (128, 64))):
        assert attend(lib, c, b, heads, qs=qs, os=os, ws=1024 * P, mask=256 * P, mstride=4, mwidth=4) == LAUNCHED, lib.ptts_last_error()
        row = (64, odd) if c.kv_heads == 1 else ((odd, 64) if b is one else (128, 64))
        assert append(lib, c, b, 1, 256 * P, row, 512 * P, row, None, heads, P, qs, 2 * P, os) == LAUNCHED, lib.ptts_last_error()
    assert attend(lib, far, one, 4, ws=1024 * P, mask=256 * P, mstride=0, mwidth=4) == LAUNCHED
    assert attend(lib, far, two, 4, qs=(260, 64), ws=1024 * P) == attend(lib, far, two, 4, os=(260, 64), ws=1024 * P) == -1
    assert attend(lib, far, two, 4, ws=1024 * P, mask=256 * P, mstride=0, mwidth=4) == -1
    assert attend(lib, kv(k=64 * P, v=128 * P, k_strides=strides(8196, 4096, 64)), two, 4, ws=1024 * P) == -1
    assert append(lib, far, batch(starts=None, tokens=2, n_seqs=2, table_stride=3)) == -1


def test_a_check_waits_for_every_stream_before_it_reads_and_after_it_clears(monkeypatch):
    done = []

    class Status:
        is_cuda, device = True, torch.device("cuda", 3)

        def item(self):
            done.append("read")
            return 2

        def zero_(self):
            done.append("clear")

    monkeypatch.setattr(torch.cuda, "synchronize", lambda device: done.append(f"wait {device.index}"))
    with pytest.raises(_hip.PttsError, match="page id"):
        paged._read_status(Status(), "paged cache")
    assert done == ["wait 3", "read", "clear", "wait 3"]
    paged.RotaryTable(64, 4, device="cpu").check()        # nothing to wait for


class StubCache:
    """what the argument checks of the wrapper look at, on the host"""
    _index = -1

    def __init__(self, k, v):
        self.k, self.v = k, v

    def _check_held(self):
        pass


def test_gradients_and_tangents_that_would_be_lost_are_refused():
    import torch.autograd.forward_ad as fwad

    table, pos = RotaryTableOnHost(), torch.zeros(3, dtype=torch.int32)
    x, page = torch.randn(3, 2, 64), torch.randn(2, 1, 16, 64)
    with fwad.dual_level():
        for t in (fwad.make_dual(x, torch.ones_like(x)), fwad.make_dual(x.clone(), torch.zeros_like(x))):
            with pytest.raises(ValueError, match="tangent"):
                paged.rotary_embed(t, pos, table)
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                paged.rotary_embed(t, pos, table)
        with pytest.raises(ValueError, match="ROCm device"):
            paged.rotary_embed(x, pos, table)
    cached = lambda k, v: paged._batch(StubCache(k, v), 3, pos[None].expand(3, -1).contiguous(), pos, None)
    cached(page, page)
    leaf = page.clone().requires_grad_()
    for k, v, name in ((leaf, page, "cache.k"), (page, leaf * 2, "cache.v")):
        with pytest.raises(ValueError, match=f"{name} requires a gradient"):
            cached(k, v)
        with torch.no_grad():
            cached(k, v)
    with fwad.dual_level(), pytest.raises(ValueError, match="cache.v has a tangent"):
        cached(page, fwad.make_dual(page, page))


def RotaryTableOnHost():
    return paged.RotaryTable(64, 16, device="cpu")


def test_the_tensors_of_a_table_stay_those_the_kernels_know():
    table = RotaryTableOnHost()
    for name in ("cos", "sin", "status", "positions", "rotary_dim", "_c"):
        with pytest.raises(AttributeError, match=f"RotaryTable.{name} is fixed"):
            setattr(table, name, getattr(table, name))
    table.note = "mine"                                    # a user's own attributes are theirs
    table.note = "still"
    pos, x = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64)
    with pytest.raises(ValueError, match="ROCm device"):
        paged.rotary_embed(x, pos, table)
    table.cos.data = table.cos.data.clone()
    with pytest.raises(ValueError, match="cos has other memory"):
        paged.rotary_embed(x, pos, table)


def test_sizes_that_do_not_fit_32_bits_are_refused_not_cut():
    """(expanded tensors: the sizes without the memory)"""
    table, big = RotaryTableOnHost(), 2 ** 32
    pages, pos = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    starts = torch.zeros(3, dtype=torch.int32)
    cache = StubCache(torch.zeros(1), torch.zeros(1))
    paged._batch(cache, 2 ** 31 - 1, pages, pos, starts)
    for tokens in (2 ** 31, big, big + 2):
        with pytest.raises(ValueError, match="less than 2\\^31"):
            paged._batch(cache, tokens, pages, pos, starts)
    x = torch.zeros(1, 1, 64).expand(1, big + 2, 64)
    with pytest.raises(ValueError, match="less than 2\\^31"):
        paged.rotary_embed(x, pos[:1], table)
    cache.__dict__.update(kv_heads=2, head_dim=64, dtype=torch.float32)
    for max_new in (-1, 2 ** 31, big, big + 1):
        with pytest.raises(ValueError, match="max_new"):
            paged.paged_attention(torch.zeros(2, 2, 64), cache, pages, pos, max_new=max_new)
    for rows in (lambda: paged.paged_attention(x, cache, pages, pos[:1]),
                 lambda: paged.kv_append(cache, torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), pages[:1], pos[:1], q=x)):
        with pytest.raises(ValueError, match="heads"):
            rows()


def test_single_tokens_over_long_tables_need_a_workspace_and_ask_for_all_of_it(lib):
    b, c = batch(starts=None, tokens=2, max_pages=4096, table_stride=4096), kv(k=64 * P, v=128 * P)
    need = lib.ptts_paged_attention_workspace(C.byref(c), C.byref(b), 4, 1)
    assert need > 0
    for refused in (dict(wsb=need - 1), dict(ws=4 * P + 4), dict(wsb=0)):
        assert attend(lib, c, b, max_new=1, **refused) == -1 and b"workspace" in lib.ptts_last_error()
    if not torch.cuda.is_available():
        assert attend(lib, c, b, max_new=1, ws=1024 * P, wsb=need) == LAUNCHED


def test_calls_run_on_the_device_of_their_cache_and_leave_the_current_one(monkeypatch):
    """host tensors that say they are on device 1 while device 0 is current, a library that notes what is current when it is called"""
    current, seen = [0], []

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class library:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, current[0], args[-1]))
                return 32 if name == "ptts_paged_attention_workspace" else 0

            return call

    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(paged, "_current_device", lambda: current[0])
    monkeypatch.setattr(paged, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(paged._hip, "load_library", lambda: library())
    table = RotaryTableOnHost()
    cache = StubCache(torch.zeros(2, 1, 16, 64), torch.zeros(2, 1, 16, 64))
    cache.__dict__.update(_index=1, kv_heads=1, head_dim=64, dtype=torch.float32, device=torch.device("cpu"), _ref=0, _status=0, _workspace={})
    x, pages, pos = torch.zeros(2, 1, 64), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    paged.rotary_embed(x, pos, table)
    paged.kv_append(cache, x, x, pages, pos, rotary=table, q=x)
    paged.paged_attention(x, cache, pages, pos)
    assert [s for s in seen if s[0] != "ptts_paged_attention_workspace"] == [
        (name, 1, 1001) for name in ("ptts_rotary_embed", "ptts_kv_append", "ptts_paged_attention")] and current == [0]


def test_yarn_is_linear_in_turns_as_the_paper_has_it():
    """not in the pair's index, as others have it: the part of a frequency that is kept, between 1 and 32 turns within the original positions"""
    base, _ = paged.rotary_frequencies(128)
    yarn, _ = paged.rotary_frequencies(128, scaling={"type": "yarn", "factor": 16, "original_positions": 4096})
    turns = 4096 * base / (2 * math.pi)
    kept = (yarn / base - 1 / 16) / (1 - 1 / 16)
    between = (turns > 1) & (turns < 32)
    assert between.sum() > 10
    # 64-bit roundings: a few of yarn / base (2^-53 of at most 1), over 15 / 16
    assert (kept - (turns - 1) / 31)[between].abs().max() < 16 * 2.0 ** -53
    assert "TURNS" in paged.rotary_frequencies.__doc__ and "INDEX" in paged.rotary_frequencies.__doc__


@no_gpu
def test_rows_in_place_may_differ_in_strides_of_a_single_entry(lib):
    """one token, or one head: the stride that differs addresses nothing"""
    r, far = rotary(), kv(k=64 * P, v=128 * P)
    one = batch(starts=None, tokens=1, n_seqs=1)
    for tokens, heads, a, b, ok in ((1, 4, (256, 64), (999, 64), True), (3, 1, (64, 64), (64, 7), True), (2, 4, (256, 64), (300, 64), False)):
        rc = lib.ptts_rotary_embed(C.byref(r), 1, tokens, heads, 64, P, *a, P, P, *b, P, None)
        assert rc == (LAUNCHED if ok else -1)
    assert append(lib, far, one, 1, 256 * P, (128, 64), 512 * P, (128, 64), None, 4, P, (256, 64), P, (999, 64)) == LAUNCHED
    assert append(lib, far, one, 1, 256 * P, (128, 64), 512 * P, (128, 64), None, 4, P, (256, 64), P, (256, 65)) == -1

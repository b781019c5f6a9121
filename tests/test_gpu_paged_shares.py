"""Paged attention where the keys of a tile are shared out over workgroups, where sequences come in more than one group of 64, and what
such calls do beside each other.  References and bounds: tests/paged_reference.py (a joined result adds one rescaling per share to the sums:
part of the 16 roundings that the bound adds to the number of keys)."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import BF, F32, attend, close, ints, paged, rnd  # noqa: F401  (paged: the fixture)

pytestmark = pytest.mark.gpu


def spread_lengths(n, seed, new=1, top=90, long_ones=(), long_past=0):
    g = torch.Generator().manual_seed(seed)
    lengths = [(int(torch.randint(0 if new > 1 else 1, new + 1, (1,), generator=g)), int(torch.randint(0, top, (1,), generator=g))) for _ in range(n)]
    for i in long_ones:
        lengths[i] = (lengths[i][0] or 1, long_past + i)
    return lengths


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("n", [64, 65, 130, 200])
def test_more_than_64_sequences(paged, n, dtype, dim):
    """single tokens and ragged chunks, whole and (two sequences are far longer than the rest) in shares"""
    attend(paged, spread_lengths(n, n), 16, 2, 1, dim, dtype, single=True)
    attend(paged, spread_lengths(n, n, long_ones=(3, n - 1), long_past=4500), 64, 2, 1, dim, dtype, single=True)
    attend(paged, spread_lengths(n, n, new=24), 16, 2, 1, dim, dtype, padding=2)
    attend(paged, spread_lengths(n, n, new=24, long_ones=(0, n - 2), long_past=2500), 64, 2, 1, dim, dtype, padding=2)


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("lengths", [[(100, 6000)], [(1, 5000), (130, 0), (3, 2700)], [(40, 4095), (1, 4096), (17, 4097)]],
                         ids=lambda l: "+".join(f"{n}@{p}" for n, p in l))
def test_chunks_in_shares(paged, lengths, dtype, dim):
    attend(paged, lengths, 64, 4, 2, dim, dtype)
    attend(paged, lengths, 16, 4, 2, dim, dtype, causal=False, seed=3)
    g = torch.Generator().manual_seed(4)
    mask = torch.rand(len(lengths), 6200, generator=g) < 0.3
    mask[-1, :2600] = False                         # whole shares without a key
    attend(paged, lengths, 64, 4, 2, dim, dtype, mask=mask)


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
def test_single_tokens_in_shares(paged, dtype, dim):
    for lengths, heads, kv_heads in (([(1, 9000)], 16, 1), ([(1, 7000), (1, 0), (1, 300), (1, 4096)], 6, 3), ([(1, 5000 + 64 * i) for i in range(9)], 16, 16)):
        attend(paged, lengths, 64, heads, kv_heads, dim, dtype, single=True)
    mask = torch.ones(2, 7001, dtype=torch.bool)
    mask[0, :5000] = False
    mask[1] = False
    attend(paged, [(1, 7000), (1, 6000)], 64, 4, 2, dim, dtype, mask=mask, single=True)
    attend(paged, [(1, 7000), (1, 0)], 64, 4, 2, dim, dtype, causal=False, single=True)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_longest_sequence_told_wrongly_changes_nothing_but_the_kernel(paged, dtype):
    lengths = [(40, 100), (1, 3000), (150, 7), (0, 9)]
    for max_new in (0, 1, 3, 150, 100000):
        attend(paged, lengths, 32, 4, 2, 64, dtype, max_new=max_new, padding=1)
        attend(paged, lengths, 64, 6, 1, 128, dtype, max_new=max_new)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("seqs,heads", [(5, 60), (9, 33), (20, 15), (33, 16)])
def test_launches_of_half_a_card_to_two_rounds(paged, seqs, heads, dtype):
    """256 to 530 tiles: the second half of a launch of up to 512 is dealt out from its end"""
    attend(paged, [(100 if s % 3 else 7, 40 * (s % 5)) for s in range(seqs)], 32, heads, heads, 64, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 30])
def test_values_that_are_not_finite_within_shares(paged, new, dtype):
    """a NaN value under one key of a share ruins the features it stands at, a masked one nothing"""
    starts, past, table, pages = ref.make_batch([(new, 6000)], 64)
    kc, vc = rnd(2, pages, 1, 64, 64, dtype=dtype), rnd(3, pages, 1, 64, 64, dtype=dtype)
    q = rnd(1, new, 2, 64, dtype=dtype)
    want, bound = ref.attend(q, kc, vc, table, past, starts, 0.125)
    mask = torch.ones(1, 6000 + new, dtype=torch.bool)
    mask[0, 3333] = False
    hidden, hbound = ref.attend(q, kc, vc, table, past, starts, 0.125, key_mask=mask)
    vc[int(table[0, 3333 // 64]), :, 3333 % 64, 7:9] = math.nan
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    at = (table.cuda(), ints(past), ints(starts))
    got = paged.paged_attention(q.cuda(), cache, *at)
    assert got[..., 7:9].isnan().all()
    rest = [i for i in range(64) if i not in (7, 8)]
    close(got[..., rest], want[..., rest], bound[..., rest])
    close(paged.paged_attention(q.cuda(), cache, *at, key_mask=mask.cuda()), hidden, hbound)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 30])
def test_bad_pages_within_shares(paged, new, dtype):
    from parler_tts_amd._hip import PttsError

    starts, past, table, pages = ref.make_batch([(new, 6000), (new, 5000)], 64)
    kc, vc = rnd(2, pages, 1, 64, 64, dtype=dtype), rnd(3, pages, 1, 64, 64, dtype=dtype)
    q = rnd(1, 2 * new, 2, 64, dtype=dtype)
    want, bound = ref.attend(q, kc, vc, table, past, starts, 0.125)
    table[0, 50] = pages
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    got = paged.paged_attention(q.cuda(), cache, table.cuda(), ints(past), ints(starts))
    assert got[:new].isnan().all()
    close(got[new:], want[new:], bound[new:])
    with pytest.raises(PttsError, match="page id"):
        cache.check()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_sequences_that_share_pages(paged, new, dtype):
    """one prompt's pages under every sequence (the same rows of the table, expanded, and a table that lists a page twice)"""
    starts, past, table, pages = ref.make_batch([(new, 300)], 32)
    n = 5
    kc, vc = rnd(2, pages, 2, 32, 64, dtype=dtype), rnd(3, pages, 2, 32, 64, dtype=dtype)
    table[0, 2] = table[0, 1]
    q = rnd(1, n * new, 4, 64, dtype=dtype)
    starts, past = [new * i for i in range(n + 1)], [300 - i for i in range(n)]
    tables = table.expand(n, -1)
    want, bound = ref.attend(q, kc, vc, tables, past, starts, 0.125)
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    one = table.cuda()
    got = paged.paged_attention(q.cuda(), cache, one.expand(n, -1), ints(past), ints(starts))
    close(got, want, bound)
    assert torch.equal(paged.paged_attention(q.cuda(), cache, one.expand(n, -1).contiguous(), ints(past), ints(starts)), got)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_captured_calls_in_shares_replay_beside_each_other(paged, dtype):
    """two graphs of calls with partial results, replayed on two streams at once with eager calls between, lengths changed in place"""
    heads, kv_heads, dim, page = 8, 2, 64, 64
    starts, past, table, pages = ref.make_batch([(1, 6000), (1, 300), (1, 5000)], page)
    cache = paged.PagedKVCache.from_tensors(rnd(2, pages, kv_heads, page, dim, dtype=dtype).cuda(), rnd(3, pages, kv_heads, page, dim, dtype=dtype).cuda())
    table = table.cuda()
    lengths = [ints([6000, 300, 5000]), ints([100, 299, 4990])]
    chunk = ints([0, 30, 30, 70])
    q = [rnd(5, 3, heads, dim, dtype=dtype).cuda(), rnd(6, 70, heads, dim, dtype=dtype).cuda()]
    calls = [lambda: paged.paged_attention(q[0], cache, table, lengths[0]),
             lambda: paged.paged_attention(q[1], cache, table, lengths[1], chunk, max_new=40)]
    for c in calls:
        c()
    torch.cuda.synchronize()
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = c()
        graphs.append((g, o))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(6):
        for t in (*q, ):
            t.copy_(rnd(50 + i, *t.shape, dtype=dtype))
        lengths[0].sub_(37)
        lengths[1].add_(1)
        lengths[1][1] = 270 if i % 2 else 0
        want = [c() for c in calls]
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        junk = [c() for c in calls]
        torch.cuda.synchronize()
        for (_, o), w, j in zip(graphs, want, junk):
            assert torch.equal(o, w) and torch.equal(j, w), i
    cache.check()


def test_another_current_device_is_left_as_it_was(paged):
    """a call takes the device of its cache and the current stream there"""
    cache = paged.PagedKVCache(4, 16, 2, 64)
    q = torch.zeros(1, 2, 64, dtype=BF, device="cuda")
    before = torch.cuda.current_device()
    with torch.cuda.stream(torch.cuda.Stream()):
        out = paged.paged_attention(q, cache, ints([[0]]), ints([3]))
    torch.cuda.synchronize()
    assert torch.cuda.current_device() == before and (out == 0).all()


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (BF, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("rows", [17, 33, 127, 128, 129])
def test_some_rows_over_few_keys(paged, rows, dtype, dim):
    """between the kernel for few rows and the one for chunks, either side of the rule, ragged; keys around the rule's 128 KiB"""
    edge = 131072 // (dim * (2 if dtype == BF else 4))
    attend(paged, [(rows, 30), (1, 0), (rows // 2, edge - rows // 2 - 64)], 32, 2, 2, dim, dtype, max_new=rows, padding=1)
    attend(paged, [(rows, edge - rows), (3, 5)], 64, 2, 2, dim, dtype, max_new=rows)
    attend(paged, [(max(rows // 4, 1), 40), (rows // 8, 70)], 16, 8, 2, dim, dtype, max_new=rows // 4, causal=False)
    mask = torch.rand(2, 90, generator=torch.Generator().manual_seed(1)) < 0.5
    attend(paged, [(rows, 40), (9, 60)], 16, 2, 1, dim, dtype, max_new=rows, mask=mask)


@pytest.mark.parametrize("dtype,dim", [(BF, 64), (F32, 128)])
@pytest.mark.parametrize("n", [128, 129, 700, 4200])
def test_hundreds_of_sequences(paged, n, dtype, dim):
    """the schedule of a launch in front: groups of 64 searched once and (beyond 64 groups) twice; whole, in shares, ragged with empty ones"""
    attend(paged, spread_lengths(n, n, top=40), 16, 1, 1, dim, dtype, single=True)
    attend(paged, spread_lengths(n, n, top=40, long_ones=(3, n // 2, n - 1), long_past=4500), 64, 1, 1, dim, dtype, single=True)
    attend(paged, spread_lengths(n, n, new=5, top=40), 16, 2, 1, dim, dtype, padding=2, max_new=5)
    attend(paged, spread_lengths(n, n, new=5, top=40, long_ones=(0, n - 2), long_past=2500), 64, 2, 1, dim, dtype, padding=2)
    empty = [(0, 3)] * n
    for i in (0, n // 2, n // 2 + 1, n - 1):
        empty[i] = (70 + i % 7, 100 + i)
    attend(paged, empty, 64, 2, 2, dim, dtype, padding=1)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_captured_call_over_hundreds_of_sequences(paged, dtype):
    n, dim = 300, 64
    starts, past, table, pages = ref.make_batch([(i % 3, 30 + i) for i in range(n)], 32)
    cache = paged.PagedKVCache.from_tensors(rnd(2, pages, 1, 32, dim, dtype=dtype).cuda(), rnd(3, pages, 1, 32, dim, dtype=dtype).cuda())
    q = rnd(1, starts[-1], 2, dim, dtype=dtype).cuda()
    at, table, begins = ints(past), table.cuda(), ints(starts)
    call = lambda: paged.paged_attention(q, cache, table, at, begins)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = call()
    for i in range(4):
        at.sub_(7)
        want = call()
        g.replay()
        junk = call()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(junk, want), i
    cache.check()


@pytest.mark.parametrize("single", [True, False])
def test_bad_entries_among_hundreds_of_sequences(paged, single):
    from parler_tts_amd._hip import PttsError

    n, dim = 200, 64
    starts, past, table, pages = ref.make_batch([(1 if single else 1 + i % 4, 30 + i % 50) for i in range(n)], 16)
    kc, vc, q = rnd(2, pages, 1, 16, dim), rnd(3, pages, 1, 16, dim), rnd(1, starts[-1], 1, dim)
    want, bound = ref.attend(q, kc, vc, table, past, starts, 0.125)
    cache = paged.PagedKVCache.from_tensors(kc.cuda(), vc.cuda())
    table[50, 1] = -5
    past[120], past[130] = -3, 2 ** 31 - 1
    got = paged.paged_attention(q.cuda(), cache, table.cuda(), ints(past), None if single else ints(starts))
    keep = torch.ones(starts[-1], dtype=torch.bool)
    for s in (50, 120, 130):
        keep[starts[s]:starts[s + 1]] = False
        assert got[starts[s]:starts[s + 1]].isnan().all()
    close(got[keep.cuda()], want[keep], bound[keep])
    with pytest.raises(PttsError, match="page id.*longer|longer.*page id|page id"):
        cache.check()

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

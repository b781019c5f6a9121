"""Paged-cache operators without a GPU, at their edges: memory that tensors share, strides that address nothing, the wrapper's promises."""
import ctypes as C
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


def verdict(lib, rc, words):
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
        assert verdict(lib, rc, b"share memory") == (meets and not same)
        far = kv(dtype=int(bf16), k=64 * P, v=128 * P)
        one = batch(starts=None, tokens=tokens, n_seqs=tokens)
        rc = append(lib, far, one, int(bf16), 256 * P, (128, 64), 512 * P, (128, 64), None, heads, 4 * P, a, at, b)
        assert verdict(lib, rc, b"share memory") == (meets and not same)
        if all(x % (16 // esz) == 0 for x in a + b) and off % 16 == 0:
            c = kv(dtype=int(bf16), k=64 * P, v=128 * P, kv_heads=1)
            rc = attend(lib, c, one, heads, 4 * P, a, at, b, ws=1024 * P)
            assert verdict(lib, rc, b"share memory") == meets
        # two key heads beside the query heads
        nk, sk = [tokens, 2], layout(rng, [tokens, 2])
        if rng.random() < 0.6:
            sk[0] = max(a[0], sk[1] + 64)
        over = bool(places(4 * P, sk, nk, esz) & places(at, b, n, esz))
        for first in (True, False):
            rows = (4 * P, sk, 512 * P, (128, 64)) if first else (512 * P, (128, 64), 4 * P, sk)
            rc = append(lib, far, one, int(bf16), *rows, None, heads, 256 * P, (1 << 12, 64), at, b)
            assert verdict(lib, rc, b"q_out shares memory with k or v") == over
    assert 50 < shared < 250

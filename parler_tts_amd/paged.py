"""Operators over a paged KV cache of the caller's: rotary positions, the append of new keys and values, the attention over them.

The engine behind ``generate()`` keeps its cache to itself.  These are the same steps for a cache, a page table and a ragged batch that
the caller owns (grouped heads, head dim 64 or 128, float32 or bfloat16), as calls on PyTorch tensors:

    cache  = PagedKVCache(num_pages, page_tokens, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda")
    rotary = RotaryTable(head_dim, max_positions)
    q = kv_append(cache, k, v, table, past, starts, rotary=rotary, q=q)      # store k (turned) and v, turn q
    o = paged_attention(q, cache, table, past, starts, max_new=longest)

``table`` [sequences, pages] int32 lists every sequence's pages, ``past`` [sequences] int32 how many of its tokens the cache held before
this call, ``starts`` [sequences + 1] int32 where its new tokens begin in q / k / v (None: one new token each).  They are read on the
device when the work runs, so a captured graph serves other lengths after an in-place update.  What they say wrongly is never followed
out of a buffer: it sets ``cache.status`` / ``rotary.status``, which ``check()`` turns into an error, and the rows concerned come out as
zeros (``kv_append``, ``rotary_embed``) or NaN (``paged_attention``; rows of the same sequence that are computed with them may be NaN too).
Where ``starts`` are wrong, rows are as ``out`` held them or of one of the sequences that claim them.

Work goes to the current stream of the tensors' device and nothing is synchronised.  No gradients: forward only (tensors that ask for one are
refused, those of the cache too); what a call writes counts as changed in place.
"""
from __future__ import annotations

import ctypes as C
import math
from types import SimpleNamespace
from typing import Any, Dict, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _hip

_DTYPES = {torch.float32: _hip.DTYPE_F32, torch.bfloat16: _hip.DTYPE_BF16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


# the current stream's handle without the object around it (2.6 us of a call that launches in 3); the device likewise
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_changed = getattr(torch._C, "_increment_version", None) or increment_version      # of a tuple of tensors


# the level of forward-mode gradients, below 0 where there is none (looking for a tangent there takes 0.3 us a tensor)
_forward = forward_ad if hasattr(forward_ad, "_current_level") else SimpleNamespace(_current_level=0)


def _no_gradient(name: str, t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient; this operator has none (torch.no_grad(), or detach it)")
    if _forward._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a tangent; this operator has no forward-mode gradient")


def _new_status(device: torch.device) -> torch.Tensor:
    status = torch.zeros(1, dtype=torch.int32, device=device)
    if status.is_cuda:                  # calls on other streams find it cleared (and a rotary table made)
        with torch.cuda.device(device):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
    return status


def _read_status(status: torch.Tensor, who: str) -> None:
    wait = torch.cuda.synchronize if status.is_cuda else lambda device: None
    wait(status.device)                 # calls on any stream
    bits = int(status.item())
    if bits:
        status.zero_()
        wait(status.device)             # what follows on another stream sets its bits behind the clearing
        raise _hip.PttsError(-1, f"{who}: " + "; ".join(t for b, t in _hip.PAGED_STATUS.items() if bits & b))


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, scaling: Optional[Dict[str, Any]] = None):
    """(angle per position of every pair, float64 [rotary_dim / 2]; factor on cos and sin) of rotary positions.

    ``scaling`` stretches them to contexts longer than the model was trained on (factor s > 0):
      None                                       f_i = theta^(-2 i / rotary_dim)
      {"type": "linear", "factor": s}            f_i / s: positions interpolated
      {"type": "ntk", "factor": s}               theta * s^(r / (r - 2)) in theta's place: the slowest pair interpolated, the fastest kept
      {"type": "yarn", "factor": s, "original_positions": L [, "beta_fast": 32, "beta_slow": 1, "attention_factor": a]}
          pairs that turn more than beta_fast times within L positions kept, those below beta_slow interpolated, linear in the number
          of TURNS between; cos and sin times a = 0.1 ln s + 1 (Peng et al., "YaRN: Efficient Context Window Extension", 2023)

    There are two ramps by the name of yarn.  This is the paper's.  Checkpoints are also trained with one that is linear in the pair's INDEX
    between the (rounded) indices where a pair turns beta_fast and beta_slow times: it shares the ends, and differs between them (head dim
    128, s = 16, L = 4096: the paper's frequencies are up to 67 % lower).  Rows of such a checkpoint are not to be turned by these frequencies.
    """
    _need(isinstance(rotary_dim, int) and rotary_dim > 0 and rotary_dim % 2 == 0, f"rotary_dim {rotary_dim}: a positive even number")
    _need(theta > 0 and math.isfinite(theta), f"theta {theta}")
    given = dict(scaling or {"type": "none"})
    kind = given.pop("type", None)
    known = {"none": (), "linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_positions", "beta_fast", "beta_slow", "attention_factor")}
    _need(kind in known, f"rotary scaling type {kind!r}: one of {sorted(known)}")
    _need(set(given) <= set(known[kind]), f"rotary scaling {kind!r} takes {known[kind]}, got {sorted(given)}")
    _need(kind == "none" or "factor" in given, f"rotary scaling {kind!r} needs a factor")
    s = float(given.get("factor", 1.0))
    _need(s > 0 and math.isfinite(s), f"rotary scaling factor {s}")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if kind == "ntk":
        _need(rotary_dim > 2, "ntk scaling needs more than one pair")
        theta = theta * s ** (rotary_dim / (rotary_dim - 2))
    freq, gain = theta ** (-2.0 * i / rotary_dim), 1.0
    if kind == "linear":
        freq = freq / s
    elif kind == "yarn":
        fast, slow = float(given.get("beta_fast", 32.0)), float(given.get("beta_slow", 1.0))
        _need("original_positions" in given and given["original_positions"] > 0, "yarn scaling needs original_positions")
        _need(fast > slow, "yarn scaling needs beta_fast > beta_slow")
        keep = ((given["original_positions"] * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        freq = keep * freq + (1.0 - keep) * freq / s
        gain = given.get("attention_factor")
        gain = 0.1 * math.log(s) + 1.0 if gain is None else float(gain)
    return freq, gain


class _Held:
    """Tensors whose addresses, strides and sizes the kernels are told of once: the attributes stay as they were made (others may be added),
    and a tensor that was given other memory since is noticed by the next call."""

    def _hold(self, one: str, two: str) -> None:
        self._names, self._one, self._two = (one, two), getattr(self, one), getattr(self, two)
        self._at_one, self._at_two = self._one.data_ptr(), self._two.data_ptr()
        self._made = frozenset(self.__dict__) | {"_made"}

    def __setattr__(self, name, value):
        if name in self.__dict__.get("_made", ()):
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: make another {type(self).__name__}")
        object.__setattr__(self, name, value)

    def _check_held(self) -> None:
        if self._one.data_ptr() != self._at_one or self._two.data_ptr() != self._at_two:
            raise ValueError(f"{self._names[self._one.data_ptr() == self._at_one]} has other memory than when the {type(self).__name__} was made: "
                             "make another around it")


class RotaryTable(_Held):
    """cos and sin of every position's angles, float32 on the device from float64 angles; made once, kept with the model.

    ``layout``: "half" turns the pairs (i, i + rotary_dim / 2), "interleaved" the pairs (2 i, 2 i + 1) of the first ``rotary_dim`` (default:
    all) features of a head; the rest pass as they are."""

    def __init__(self, head_dim: int, positions: int, *, theta: float = 10000.0, rotary_dim: Optional[int] = None, layout: str = "half",
                 scaling: Optional[Dict[str, Any]] = None, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        _need(layout in ("half", "interleaved"), f"layout {layout!r}: 'half' or 'interleaved'")
        _need(0 < positions < 2 ** 31, f"positions {positions}")
        _need(head_dim > 0 and head_dim % 2 == 0 and rotary_dim <= head_dim, f"rotary_dim {rotary_dim} of a head of {head_dim}")
        freq, gain = rotary_frequencies(rotary_dim, theta, scaling)
        angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
        self.cos, self.sin = (torch.cos(angle) * gain).float(), (torch.sin(angle) * gain).float()
        self.head_dim, self.positions, self.rotary_dim, self.layout = head_dim, positions, rotary_dim, layout
        self.device, self._index = self.cos.device, self.cos.get_device()
        self.status = _new_status(self.device)
        self._status = self.status.data_ptr()
        self._c = _hip.PttsRotary(self.cos.data_ptr(), self.sin.data_ptr(), positions, rotary_dim, 1 if layout == "interleaved" else 0)
        self._ref = C.addressof(self._c)
        self._hold("cos", "sin")

    def check(self) -> None:
        """waits for the device (every stream); raises if a call since the last check met a position outside the table.  Not to be called while
        another thread makes calls."""
        _read_status(self.status, "rotary_embed")


class PagedKVCache(_Held):
    """One layer's keys and values in pages: ``k``, ``v`` [pages, kv_heads, page_tokens, head_dim]."""

    def __init__(self, num_pages: int, page_tokens: int, kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        shape = (num_pages, kv_heads, page_tokens, head_dim)
        self._adopt(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedKVCache":
        """around tensors (or views: any strides of the first three dimensions) the caller already has"""
        self = cls.__new__(cls)
        self._adopt(k, v)
        return self

    def _adopt(self, k: torch.Tensor, v: torch.Tensor) -> None:
        _need(k.dim() == 4 and k.shape == v.shape, f"k {tuple(k.shape)} and v {tuple(v.shape)}: [pages, kv_heads, page_tokens, head_dim] each")
        _need(k.dtype in _DTYPES and k.dtype == v.dtype, f"a cache of {k.dtype} / {v.dtype}: float32 or bfloat16")
        _need(k.device.type == "cuda" and k.device == v.device, "the cache has to be on one ROCm device")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "the features of a cache row have to be contiguous")
        _no_gradient("k", k)
        _no_gradient("v", v)
        pages, heads, tokens, dim = k.shape
        _need(0 < pages < 2 ** 31 and 0 < heads < 2 ** 31, f"a cache of {pages} pages and {heads} heads")
        _need(16 <= tokens <= 4096 and tokens & (tokens - 1) == 0, f"pages of {tokens} tokens: a power of two from 16 to 4096 is served")
        _need(dim in (64, 128), f"head_dim {dim}: 64 and 128 are served")
        self.k, self.v = k, v
        self.num_pages, self.kv_heads, self.page_tokens, self.head_dim = pages, heads, tokens, dim
        self.dtype, self.device, self._index = k.dtype, k.device, k.get_device()
        self.status = _new_status(self.device)
        self._status = self.status.data_ptr()
        self._c = _hip.PttsPagedKV(k.data_ptr(), v.data_ptr(), (C.c_int64 * 3)(*k.stride()[:3]), (C.c_int64 * 3)(*v.stride()[:3]),
                                   _DTYPES[k.dtype], pages, heads, tokens, dim)
        self._ref = C.addressof(self._c)
        self._workspace: Dict[tuple, int] = {}      # bytes by sizes
        self._hold("k", "v")

    def check(self) -> None:
        """waits for the device (every stream); raises if a call since the last check met a page, length, position or start it could not follow.
        Not to be called while another thread makes calls."""
        _read_status(self.status, "paged cache")


# (device numbers instead of devices, -1 for the host's: a tenth of a microsecond a comparison)
def _rows(name: str, t: torch.Tensor, tokens: Optional[int], heads: Optional[int], dim: int, index: int) -> None:
    shape = t.shape
    if len(shape) != 3 or shape[2] != dim or (tokens is not None and shape[0] != tokens) or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} {tuple(shape)}: [{'tokens' if tokens is None else tokens}, {'heads' if heads is None else heads}, {dim}] expected")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on device {index}")
    if t.stride(2) != 1:
        raise ValueError(f"the features of a row of {name} have to be contiguous")
    if t.requires_grad or _forward._current_level >= 0:
        _no_gradient(name, t)


def _ints(name: str, t: torch.Tensor, dims: int, index: int) -> None:
    if t.dtype is not torch.int32 or t.dim() != dims or t.get_device() != index or (t.stride(-1) != 1 and t.shape[-1] > 1):
        raise ValueError(f"{name} has to be a contiguous int32 tensor of {dims} dimension(s) on device {index}")


def _batch(cache: PagedKVCache, tokens: int, table: torch.Tensor, past: torch.Tensor, starts: Optional[torch.Tensor]):
    index = cache._index
    cache._check_held()
    if cache.k.requires_grad or cache.v.requires_grad or _forward._current_level >= 0:
        _no_gradient("cache.k", cache.k)
        _no_gradient("cache.v", cache.v)
    _ints("table", table, 2, index)
    _ints("past", past, 1, index)
    n = past.shape[0]
    rows, width = table.shape
    if (tokens | n | width) >> 31:      # sizes travel in 32 bits, and ctypes would cut them
        raise ValueError(f"{tokens} tokens of {n} sequences over {width} pages: less than 2^31 of each")
    if rows != n:
        raise ValueError(f"a page table of {rows} rows for {n} sequences")
    at = None
    if starts is not None:
        _ints("starts", starts, 1, index)
        if starts.shape[0] != n + 1:
            raise ValueError(f"starts of {starts.shape[0]} entries for {n} sequences: one more than sequences")
        at = starts.data_ptr()
    elif tokens != n:
        raise ValueError(f"{tokens} tokens of {n} sequences: starts says whose they are")
    stride = table.stride(0) if rows > 1 else width
    return _hip.PttsPagedBatch(table.data_ptr(), stride, past.data_ptr(), at, width, n, tokens)


def rotary_embed(x: torch.Tensor, positions: torch.Tensor, rotary: RotaryTable, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x`` [tokens, heads, head_dim] (float32 or bfloat16) turned by ``positions`` [tokens] int32 -> ``out`` (may be ``x``).
    A row whose position is outside the table becomes zero, and ``rotary.check()`` raises."""
    tokens, heads, given = x.shape[0], x.shape[1] if x.dim() == 3 else None, out is not None
    index = rotary._index
    _rows("x", x, None, None, rotary.head_dim, index)
    if x.dtype not in _DTYPES:
        raise ValueError(f"x of {x.dtype}: float32 or bfloat16")
    _ints("positions", positions, 1, index)
    if positions.shape[0] != tokens:
        raise ValueError(f"{positions.shape[0]} positions for {tokens} tokens")
    if (tokens | heads) >> 31:
        raise ValueError(f"{tokens} tokens of {heads} heads: less than 2^31 of each")
    rotary._check_held()
    if index < 0:
        raise ValueError(f"the rotary table is on {rotary.device}: a ROCm device is needed to turn rows")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    else:
        _rows("out", out, tokens, heads, rotary.head_dim, index)
        if out.dtype != x.dtype:
            raise ValueError(f"out of {out.dtype} for x of {x.dtype}")
    if heads == 0 or tokens == 0:
        return out
    if index != _current_device():
        with torch.cuda.device(index):
            return rotary_embed(x, positions, rotary, out)
    xs, os = x.stride(), out.stride()
    rc = _hip.load_library().ptts_rotary_embed(rotary._ref, _DTYPES[x.dtype], tokens, heads, rotary.head_dim, x.data_ptr(), xs[0], xs[1],
                                               positions.data_ptr(), out.data_ptr(), os[0], os[1], rotary._status, _raw_stream(index))
    if rc:
        _hip.check(rc)
    if given:
        _changed((out,))                # what autograd saved of it is no longer there
    return out


def kv_append(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, past: torch.Tensor,
              starts: Optional[torch.Tensor] = None, *, rotary: Optional[RotaryTable] = None, positions: Optional[torch.Tensor] = None,
              q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Stores ``k``, ``v`` [tokens, kv_heads, head_dim]: token i of sequence s at slot ``past[s] + i``, k turned by ``rotary`` at that
    position (or at ``positions`` [tokens] int32).  ``q`` [tokens, heads, head_dim] is turned in the same launch into ``q_out`` (may be ``q``,
    and shares no memory with ``k`` or ``v``), which is returned.  float32 rows may be stored in a bfloat16 cache.  Rows behind the last
    sequence are left alone, in ``q_out`` too.  None of the rows may lie in the cache (copy what is to move within it), and ``cache.k`` and
    ``cache.v`` share no memory."""
    index, written = cache._index, q_out
    tokens = k.shape[0]
    _rows("k", k, tokens, cache.kv_heads, cache.head_dim, index)
    _rows("v", v, tokens, cache.kv_heads, cache.head_dim, index)
    if k.dtype not in _DTYPES or v.dtype != k.dtype or (k.dtype != cache.dtype and k.dtype != torch.float32):
        raise ValueError(f"k of {k.dtype} and v of {v.dtype} for a cache of {cache.dtype}")
    batch = _batch(cache, tokens, table, past, starts)
    rot = at = None
    if rotary is not None:
        if rotary._index != index or rotary.head_dim != cache.head_dim:
            raise ValueError(f"a rotary table for heads of {rotary.head_dim} on {rotary.device}; the cache has {cache.head_dim} on {cache.device}")
        rotary._check_held()
        rot = rotary._ref
    if positions is not None:
        if rotary is None:
            raise ValueError("positions without a rotary table")
        _ints("positions", positions, 1, index)
        if positions.shape[0] != tokens:
            raise ValueError(f"{positions.shape[0]} positions for {tokens} tokens")
        at = positions.data_ptr()
    ks, vs = k.stride(), v.stride()
    heads, qp, qop, qs, qos = 0, None, None, (0, 0), (0, 0)
    if q is not None:
        _rows("q", q, tokens, None, cache.head_dim, index)
        heads = q.shape[1]
        if q.dtype != k.dtype or heads == 0 or heads >> 31:
            raise ValueError(f"q {tuple(q.shape)} of {q.dtype} beside k of {k.dtype}: 1 to 2^31 - 1 heads of k's type")
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        else:
            _rows("q_out", q_out, tokens, heads, cache.head_dim, index)
            if q_out.dtype != q.dtype:
                raise ValueError(f"q_out of {q_out.dtype} for q of {q.dtype}")
        qp, qop, qs, qos = q.data_ptr(), q_out.data_ptr(), q.stride(), q_out.stride()
    elif q_out is not None:
        raise ValueError("q_out without q")
    if tokens == 0:
        return q_out
    if index != _current_device():
        with torch.cuda.device(index):
            return kv_append(cache, k, v, table, past, starts, rotary=rotary, positions=positions, q=q, q_out=q_out)
    rc = _hip.load_library().ptts_kv_append(cache._ref, C.addressof(batch), _DTYPES[k.dtype], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                            rot, at, heads, qp, qs[0], qs[1], qop, qos[0], qos[1], cache._status, _raw_stream(index))
    if rc:
        _hip.check(rc)
    _changed((cache.k, cache.v) if written is None else (cache.k, cache.v, written))      # what autograd saved of them is no longer there
    return q_out


def paged_attention(q: torch.Tensor, cache: PagedKVCache, table: torch.Tensor, past: torch.Tensor, starts: Optional[torch.Tensor] = None, *,
                    scale: Optional[float] = None, causal: bool = True, key_mask: Optional[torch.Tensor] = None, max_new: int = 0,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q k^T) v over the cache -> [tokens, heads, head_dim], ``scale`` by default head_dim^-0.5.

    causal: token i of sequence s sees the keys 0 .. past[s] + i (its own among them: append first); otherwise every token sees the keys
    0 .. past[s] - 1 (states that were cached once, as a cross-attention reads them).  ``scale`` is positive.  ``key_mask`` [sequences, columns] bool: a False
    column is no key, whatever the cache holds there; keys behind its last column are seen.  A token without keys
    (or with every score -infinity) gets zeros.
    ``q``'s heads are a multiple of the cache's, in groups: head h reads key head h // (heads / kv_heads).
    ``max_new``: the longest sequence's number of new tokens if the caller knows it (0: unknown).  Kernel and workspace are picked by it and
    by the table's WIDTH, before any length is known: rows of unknown number take the kernel for chunks, and a table much wider than the
    contexts brings room and a launch to join shares that nobody may need.  Results hold either way; a tight table and bound are faster.
    bfloat16: scores, sums and the output's sum are float32, the softmax weights are rounded to bfloat16 before they meet the values (half
    a step, 2^-8 of each; the error against 64 bits is 1.3 to 1.4 times that of float32 weights).  float32 rounds nothing more.
    Rows of ``q`` and ``out`` start at multiples of 16 bytes; ``out`` shares no memory with ``q`` or the cache.
    Sequences may share pages, or (an expanded ``table``) all of them.  Rows of no sequence (behind the last, or where ``starts`` are wrong)
    are left as they are in ``out``; rows that descending ``starts`` give to several hold the result of one of these."""
    index, dim, given = cache._index, cache.head_dim, out is not None
    tokens = q.shape[0]
    _rows("q", q, None, None, dim, index)
    heads = q.shape[1]
    if q.dtype != cache.dtype:
        raise ValueError(f"q of {q.dtype} over a cache of {cache.dtype}")
    if heads == 0 or heads % cache.kv_heads or heads >> 31:
        raise ValueError(f"{heads} query heads over {cache.kv_heads} key heads")
    if not 0 <= max_new < 2 ** 31:
        raise ValueError(f"max_new {max_new}")
    batch = _batch(cache, tokens, table, past, starts)
    mask, mask_stride, mask_width = None, 0, 0
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or key_mask.dim() != 2 or key_mask.shape[0] != past.shape[0] or \
                key_mask.get_device() != index or (key_mask.shape[1] > 1 and key_mask.stride(1) != 1):
            raise ValueError(f"key_mask has to be a bool tensor [{past.shape[0]}, columns] on {cache.device}")
        mask_width = min(key_mask.shape[1], 2 ** 31 - 1)      # no context reaches the columns behind
        mask, mask_stride = key_mask.data_ptr() if mask_width else None, max(key_mask.stride(0), mask_width)
        if key_mask.shape[0] > 1 and key_mask.stride(0) < mask_width:
            key_mask = key_mask.contiguous()          # one row for every sequence, expanded
            mask = key_mask.data_ptr()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _rows("out", out, tokens, heads, dim, index)
        if out.dtype != q.dtype:
            raise ValueError(f"out of {out.dtype} for q of {q.dtype}")
    if tokens == 0:
        return out
    if index != _current_device():
        with torch.cuda.device(index):
            return paged_attention(q, cache, table, past, starts, scale=scale, causal=causal, key_mask=key_mask, max_new=max_new, out=out)
    lib = _hip.load_library()
    bref = C.addressof(batch)
    key = (tokens, batch.n_seqs, batch.max_pages, heads, max_new, starts is None)
    need = cache._workspace.get(key)
    if need is None:
        need = lib.ptts_paged_attention_workspace(cache._ref, bref, heads, max_new)
        if need < 0:
            _hip.check(int(need))
        if len(cache._workspace) > 4096:
            cache._workspace.clear()
        cache._workspace[key] = need
    workspace = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    qs, os = q.stride(), out.stride()
    rc = lib.ptts_paged_attention(cache._ref, bref, heads, q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1],
                                  dim ** -0.5 if scale is None else scale, 1 if causal else 0, mask, mask_stride, mask_width, max_new,
                                  workspace.data_ptr() if need else None, need, cache._status, _raw_stream(index))
    if rc:
        _hip.check(rc)
    if given:
        _changed((out,))
    return out

"""What is measured of the paged-cache operators: rotary positions, the append of keys and values to a paged cache, and the
attention of new tokens over it (parler_tts_amd.paged).

``run`` computes an operator either in its plain form - elementary torch operations in 32 bits, rounded once at the end - or, with
``own`` set, through the calls a user makes of the framework.  ``exact`` states the same results in 64 bits, apart from both.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------------

def listed():
    cases = []

    def add(name, **kw):
        cases.append(dict(name=name, **kw))

    # one decode step of the batch the benchmark serves: 32 single tokens, 16 heads of 64 (latency)
    add("rotate_step", op="rotate", dtype="bf16", tokens=32, heads=16, dim=64, rot=64, layout="half", scaling="none", reach=4096)
    # all positions of 32 long clips at the scaled decoder's width, far positions, a quarter of the head left alone
    add("rotate_prompt_fp32", op="rotate", dtype="fp32", tokens=41283, heads=24, dim=64, rot=48, layout="interleaved",
        scaling="yarn", reach=131072)
    # the append of one decode step: one token each for 32 clips of unlike length
    add("append_step", op="append", dtype="bf16", seqs=32, new_min=1, new_max=1, past_min=3, past_max=2579, heads=16, kv_heads=16,
        dim=64, page=64, rot=64, layout="half", scaling="none", packed=False)
    # prompts of 24 requests arriving together, q / k / v slices of one projection's rows
    add("append_prompts", op="append", dtype="bf16", seqs=24, new_min=257, new_max=1500, past_min=0, past_max=0, heads=24,
        kv_heads=24, dim=64, page=64, rot=64, layout="half", scaling="linear", packed=True)
    # ragged chunks in 32 bits (the parity mode's type), grouped heads, small pages
    add("append_chunk_fp32", op="append", dtype="fp32", seqs=7, new_min=1, new_max=259, past_min=0, past_max=1201, heads=16,
        kv_heads=4, dim=128, page=16, rot=128, layout="interleaved", scaling="ntk", packed=False)
    # the smallest call: one clip, one token, a short context (latency)
    add("attend_step_one", op="attend", dtype="bf16", seqs=1, new_min=1, new_max=1, past_min=300, past_max=300, heads=16,
        kv_heads=16, dim=64, page=64, causal=True, masked=0)
    # the decode step of the benchmark's batch at unlike lengths
    add("attend_step_batch", op="attend", dtype="bf16", seqs=32, new_min=1, new_max=1, past_min=700, past_max=2579, heads=16,
        kv_heads=16, dim=64, page=64, causal=True, masked=0)
    # two long contexts, grouped heads: one token each over a cache of 131 thousand
    add("attend_step_far", op="attend", dtype="bf16", seqs=2, new_min=1, new_max=1, past_min=120001, past_max=131070, heads=32,
        kv_heads=4, dim=128, page=64, causal=True, masked=0)
    # a chunk of the batched prefill: padded prompts (masked keys in front) and what is cached before the chunk
    add("attend_chunk_masked", op="attend", dtype="bf16", seqs=32, new_min=128, new_max=128, past_min=0, past_max=1300, heads=16,
        kv_heads=16, dim=64, page=64, causal=True, masked=60)
    # one long prompt at once, grouped heads of 128
    add("attend_prompt", op="attend", dtype="bf16", seqs=1, new_min=8191, new_max=8191, past_min=0, past_max=0, heads=16,
        kv_heads=4, dim=128, page=64, causal=True, masked=0)
    # ragged chunks in 32 bits over small pages
    add("attend_chunk_fp32", op="attend", dtype="fp32", seqs=5, new_min=1, new_max=257, past_min=61, past_max=1290, heads=16,
        kv_heads=16, dim=64, page=16, causal=True, masked=0)
    # one round of a server: prompts' chunks and single tokens in one batch, append and attention as they are called together
    add("serve_mixed", op="serve", dtype="bf16", seqs=24, new_min=1, new_max=401, past_min=0, past_max=2500, heads=16, kv_heads=8,
        dim=64, page=64, rot=64, layout="half", scaling="none", packed=False, causal=True, masked=0)
    return cases


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        for k in w:
            limits[k] = max(limits.get(k, 0), w[k])
    while True:
        op = rng.choice(["rotate", "append", "attend", "attend", "attend", "serve"])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        dim = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 24])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 7, 8])
        if heads > 32:
            continue
        rot = rng.choice([dim, dim, dim // 2, dim - 16, 2 * rng.randint(8, dim // 2)])
        c = dict(op=op, dtype=dtype, heads=heads, dim=dim)
        if op == "rotate":
            c.update(tokens=_log_int(rng, 1, 42000), rot=rot, layout=rng.choice(["half", "interleaved"]),
                     scaling=rng.choice(["none", "linear", "ntk", "yarn"]), reach=rng.choice([4096, 32768, 131072]))
        else:
            seqs = _log_int(rng, 1, 48)
            kind = rng.choice(["single", "chunk", "ragged", "long"])
            if kind == "single":
                lo = hi = 1
            elif kind == "chunk":
                lo = hi = _log_int(rng, 2, 600)
            else:
                lo, hi = 1, _log_int(rng, 2, 8191 if kind == "long" else 1500)
            past = _log_int(rng, 1, 131000 if lo == hi == 1 and seqs <= 4 else 2579)
            c.update(seqs=seqs, new_min=lo, new_max=hi, past_min=rng.choice([0, past // 3, past]), past_max=past, kv_heads=kv_heads,
                     page=rng.choice([16, 32, 64, 64, 128]))
            if op in ("append", "serve"):
                c.update(rot=rot, layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                         packed=rng.random() < 0.4)
            if op in ("attend", "serve"):
                c.update(causal=op == "serve" or rng.random() < 0.85, masked=rng.choice([0, 0, 0, 1, 60]))
        w = work(c)
        if w["bytes"] <= limits["bytes"] and w["flops"] <= limits["flops"] and _plain_scores(c) <= 4e9:
            return c


def _lengths(case):
    """(new tokens, cached tokens) of every sequence: the case's alone, spread over its two ranges in no order"""
    n = case["seqs"]

    def spread(lo, hi, step):
        if n == 1:
            return [hi]
        return [lo + int(round((hi - lo) * ((i * step + 0.31) % 1.0))) for i in range(n)]

    return spread(case["new_min"], case["new_max"], 0.6180339887), spread(case["past_min"], case["past_max"], 0.7548776662)


def _visible(case, new, past):
    """pairs of a query and a key it may see (the padding in front counts as seen: it has to be looked at)"""
    return new * past + new * (new + 1) // 2 if case["causal"] else new * past


def _plain_scores(case):
    """the largest score matrix the plain form holds, in elements"""
    if case["op"] not in ("attend", "serve"):
        return 0
    return max(n * (p + n) for n, p in zip(*_lengths(case))) * case["heads"]


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    d, h = case["dim"], case["heads"]
    if case["op"] == "rotate":
        n = case["tokens"] * h * d
        return {"bytes": 2 * n * size + case["tokens"] * 4, "flops": 3 * case["tokens"] * h * case["rot"]}
    new, past = _lengths(case)
    total, hk = sum(new), case["kv_heads"]
    nbytes, flops = 0, 0
    if case["op"] in ("append", "serve"):
        nbytes += 2 * total * (h + 2 * hk) * d * size
        flops += 3 * total * (h + hk) * case["rot"]
    if case["op"] in ("attend", "serve"):
        keys = [p + (n if case["causal"] else 0) for n, p in zip(new, past)]
        nbytes += 2 * total * h * d * size + 2 * sum(keys) * hk * d * size
        flops += sum(4 * _visible(case, n, p) * h * d for n, p in zip(new, past))
        if case["op"] == "serve":      # q and the new rows of the cache stay on the chip between the two at best
            nbytes -= total * (h + 2 * hk) * d * size
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------------

SCALING = {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 8.0},
           "yarn": {"type": "yarn", "factor": 16.0, "original_positions": 4096}}


def _normal(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def _tables(case, reach):
    """cos and sin of every position's angles, in 32 bits from 64"""
    r, theta = case["rot"], 10000.0
    s = SCALING[case["scaling"]]
    i = torch.arange(r // 2, device=DEVICE, dtype=torch.float64)
    gain = 1.0
    if s and s["type"] == "ntk":
        theta *= s["factor"] ** (r / (r - 2))
    freq = theta ** (-2.0 * i / r)
    if s and s["type"] == "linear":
        freq = freq / s["factor"]
    if s and s["type"] == "yarn":
        keep = ((s["original_positions"] * freq / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        freq = keep * freq + (1 - keep) * freq / s["factor"]
        gain = 0.1 * math.log(s["factor"]) + 1.0
    angle = torch.arange(reach, device=DEVICE, dtype=torch.float64)[:, None] * freq
    return (torch.cos(angle) * gain).float(), (torch.sin(angle) * gain).float()


def _rotary(case, reach):
    if own:
        from parler_tts_amd.paged import RotaryTable

        return RotaryTable(case["dim"], reach, rotary_dim=case["rot"], layout=case["layout"], scaling=SCALING[case["scaling"]],
                           device=DEVICE)
    return _tables(case, reach)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, d, h = DTYPES[case["dtype"]], case["dim"], case["heads"]
    st = {"case": case}
    if case["op"] == "rotate":
        st["x"] = _normal(gen, case["tokens"], h, d, dtype=dtype)
        st["positions"] = torch.randint(0, case["reach"], (case["tokens"],), generator=gen, device=DEVICE, dtype=torch.int32)
        st["rotary"] = _rotary(case, case["reach"])
        return st
    new, past = _lengths(case)
    total, hk, page = sum(new), case["kv_heads"], case["page"]
    pages = [(n + p + page - 1) // page for n, p in zip(new, past)]
    # pages are handed out in no order, as a server's pool does after a while; three of them belong to nobody
    ids = torch.randperm(sum(pages) + 3, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.zeros(len(new), max(pages), dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = ids[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st.update(new=new, past_list=past, starts_list=starts, table=table,
              past=torch.tensor(past, dtype=torch.int32, device=DEVICE), starts=torch.tensor(starts, dtype=torch.int32, device=DEVICE))
    shape = (ids.numel(), hk, page, d)
    st["k_cache"] = _normal(gen, *shape, dtype=dtype)
    st["v_cache"] = _normal(gen, *shape, dtype=dtype)
    if case.get("packed"):
        rows = _normal(gen, total, h + 2 * hk, d, dtype=dtype)
        st["q"], st["k"], st["v"] = rows[:, :h], rows[:, h:h + hk], rows[:, h + hk:]
    else:
        st["q"] = _normal(gen, total, h, d, dtype=dtype)
        if case["op"] != "attend":
            st["k"], st["v"] = _normal(gen, total, hk, d, dtype=dtype), _normal(gen, total, hk, d, dtype=dtype)
    if case["op"] != "attend":
        st["rotary"] = _rotary(case, max(n + p for n, p in zip(new, past)))
    if case.get("masked"):
        # prompts padded in front: up to `masked` keys of every sequence are no keys at all
        width = case["masked"] + 4
        pad = torch.randint(0, case["masked"] + 1, (len(new),), generator=gen, device=DEVICE)
        st["key_mask"] = torch.arange(width, device=DEVICE)[None] >= pad[:, None]
    else:
        st["key_mask"] = None
    if own:
        from parler_tts_amd.paged import PagedKVCache

        st["cache"] = PagedKVCache.from_tensors(st["k_cache"], st["v_cache"])
    return st


# ---------------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------------

def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    from parler_tts_amd import paged

    case = st["case"]
    op = case["op"]
    if op == "rotate":
        return paged.rotary_embed(st["x"], st["positions"], st["rotary"])
    starts = None if case["new_max"] == 1 else st["starts"]
    q, out = st["q"], {}
    if op != "attend":
        q = paged.kv_append(st["cache"], st["k"], st["v"], st["table"], st["past"], starts, rotary=st["rotary"], q=q)
        out.update(q=q, k=st["k_cache"], v=st["v_cache"])
    if op != "append":
        out["o"] = paged.paged_attention(q, st["cache"], st["table"], st["past"], starts, causal=case["causal"],
                                         key_mask=st["key_mask"], max_new=case["new_max"])
    return out


def _turn(x, cos, sin, rot, layout):
    """x [tokens, heads, dim] in 32 bits, cos / sin [tokens, rot / 2]"""
    cos, sin = cos[:, None], sin[:, None]
    out = x.clone()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return out


def _run_plain(st):
    case = st["case"]
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "rotate":
        cos, sin = st["rotary"]
        at = st["positions"].long()
        return _turn(st["x"].float(), cos[at], sin[at], case["rot"], case["layout"]).to(dtype)
    out, q = {}, st["q"]
    if case["op"] != "attend":
        cos, sin = st["rotary"]
        seq = torch.repeat_interleave(torch.arange(case["seqs"], device=DEVICE), (st["starts"][1:] - st["starts"][:-1]).long(),
                                      output_size=q.shape[0])
        slot = torch.arange(q.shape[0], device=DEVICE) - st["starts"][seq].long() + st["past"][seq].long()
        page = st["table"][seq, slot // case["page"]].long()
        q = _turn(q.float(), cos[slot], sin[slot], case["rot"], case["layout"]).to(dtype)
        st["k_cache"][page, :, slot % case["page"]] = _turn(st["k"].float(), cos[slot], sin[slot], case["rot"], case["layout"]).to(dtype)
        st["v_cache"][page, :, slot % case["page"]] = st["v"]
        out.update(q=q, k=st["k_cache"], v=st["v_cache"])
    if case["op"] != "append":
        out["o"] = _attend_plain(st, q).to(dtype)
    return out


def _attend_plain(st, q):
    case = st["case"]
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.empty(q.shape, dtype=torch.float32, device=DEVICE)
    for s, (n, past) in enumerate(zip(st["new"], st["past_list"])):
        a, b = st["starts_list"][s], st["starts_list"][s + 1]
        keys = past + (n if case["causal"] else 0)
        if keys == 0:
            out[a:b] = 0
            continue
        ids = st["table"][s, :(keys + page - 1) // page].long()
        k = st["k_cache"][ids].float().permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :keys]
        v = st["v_cache"][ids].float().permute(1, 0, 2, 3).reshape(hk, -1, d)[:, :keys]
        x = q[a:b].float().reshape(n, hk, h // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
        scores = torch.matmul(x, k.transpose(1, 2)).mul_(d ** -0.5).view(hk, h // hk, n, keys)
        if case["causal"]:
            ahead = torch.arange(keys, device=DEVICE)[None] > torch.arange(n, device=DEVICE)[:, None] + past
            scores.masked_fill_(ahead, -math.inf)
        if st["key_mask"] is not None:
            width = min(keys, st["key_mask"].shape[1])
            scores[..., :width].masked_fill_(~st["key_mask"][s, :width], -math.inf)
        top = scores.amax(-1, keepdim=True)
        scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
        total = scores.sum(-1, keepdim=True)
        scores.div_(torch.where(total == 0, torch.ones_like(total), total))
        o = torch.matmul(scores.view(hk, -1, keys), v)
        out[a:b] = o.view(hk, h // hk, n, d).permute(2, 0, 1, 3).reshape(n, h, d)
    return out


# ---------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------------

def _turned_exactly(x, positions, case):
    """a complex product: the pair (a, b) as a + ib times gain * exp(i * position * frequency)"""
    r = case["rot"]
    n = torch.arange(0, r, 2, device=DEVICE, dtype=torch.float64)
    scaling = SCALING[case["scaling"]] or {"type": "none"}
    f = scaling.get("factor", 1.0)
    log_theta = math.log(10000.0) + (math.log(f) * r / (r - 2) if scaling["type"] == "ntk" else 0.0)
    freq, gain = torch.exp(-n / r * log_theta), 1.0
    if scaling["type"] == "linear":
        freq = freq / f
    elif scaling["type"] == "yarn":
        turns = scaling["original_positions"] * freq / (2 * math.pi)
        blend = torch.where(turns >= 32, torch.ones_like(turns), torch.where(turns <= 1, torch.zeros_like(turns), (turns - 1) / 31))
        freq, gain = freq * (blend + (1 - blend) / f), 1.0 + 0.1 * math.log(f)
    turn = torch.polar(torch.full_like(freq, gain).expand(positions.numel(), -1).contiguous(), positions.double()[:, None] * freq)
    x = x.double()
    if case["layout"] == "half":
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., r:]], -1)
    z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn[:, None]
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], -1)


def exact(case, seed):
    st = _plain_inputs(case, seed)
    if case["op"] == "rotate":
        return _turned_exactly(st["x"], st["positions"], case)
    dtype, out = DTYPES[case["dtype"]], {}
    q, k_cache, v_cache = st["q"], st["k_cache"].double(), st["v_cache"].double()
    if case["op"] != "attend":
        at = torch.cat([torch.arange(p, p + n, device=DEVICE) for n, p in zip(st["new"], st["past_list"])])
        q, k = _turned_exactly(q, at, case), _turned_exactly(st["k"], at, case)
        for s, (n, past) in enumerate(zip(st["new"], st["past_list"])):
            row = st["starts_list"][s]
            for slot in range(past, past + n):
                if slot % case["page"] and slot != past:
                    continue
                room = min(case["page"] - slot % case["page"], past + n - slot)
                page, first = int(st["table"][s, slot // case["page"]]), slot % case["page"]
                k_cache[page, :, first:first + room] = k[row:row + room].transpose(0, 1)
                v_cache[page, :, first:first + room] = st["v"][row:row + room].double().transpose(0, 1)
                row += room
        out.update(q=q, k=k_cache, v=v_cache)
        if case["op"] == "serve":      # the attention reads what the cache and q hold: values of the stored type
            q, k_cache, v_cache = q.to(dtype), k_cache.to(dtype).double(), v_cache.to(dtype).double()
    if case["op"] != "append":
        out["o"] = _attended_exactly(st, q.double(), k_cache, v_cache)
    return out


def _attended_exactly(st, q, k_cache, v_cache):
    case = st["case"]
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros_like(q)
    for s, (n, past) in enumerate(zip(st["new"], st["past_list"])):
        first = st["starts_list"][s]
        last = past + n if case["causal"] else past
        if last == 0:
            continue
        used = st["table"][s, :-(-last // page)].long()
        live = torch.ones(last, dtype=torch.bool, device=DEVICE)
        if st["key_mask"] is not None:
            m = st["key_mask"][s, :last]
            live[:m.numel()] = m
        for head in range(case["heads"]):
            k = k_cache[used, head // group].reshape(-1, case["dim"])[:last]
            v = v_cache[used, head // group].reshape(-1, case["dim"])[:last]
            for i in range(0, n, 1024):
                rows = q[first + i:first + min(i + 1024, n), head]
                sees = live.expand(rows.shape[0], -1)
                if case["causal"]:
                    reach = past + i + torch.arange(rows.shape[0], device=DEVICE)
                    sees = sees & (torch.arange(last, device=DEVICE)[None] <= reach[:, None])
                w = torch.where(sees, rows @ k.t() / math.sqrt(case["dim"]), -math.inf)
                w = torch.softmax(w, -1)
                out[first + i:first + i + rows.shape[0], head] = torch.where(sees.any(-1, keepdim=True), w, torch.zeros_like(w)) @ v
    return out


def _plain_inputs(case, seed):
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept

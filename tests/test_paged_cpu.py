"""Paged-cache operators without a GPU: what the C entries refuse before anything is launched, the rotary frequencies, the wrapper's checks."""
import ctypes as C
import math
import os

import pytest
import torch

from parler_tts_amd import _hip
from parler_tts_amd.paged import PagedKVCache, RotaryTable, rotary_embed, rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_hip.LIB_PATH):
        import __graft_entry__ as g

        g.build()
    return _hip.load_library()


P = 1 << 20       # an aligned address nobody follows: every call below is refused first


def kv(**kw):
    d = dict(k=P, v=P, k_strides=(C.c_int64 * 3)(2 * 64 * 64, 64 * 64, 64), v_strides=(C.c_int64 * 3)(2 * 64 * 64, 64 * 64, 64), dtype=1,
             n_pages=8, kv_heads=2, page_tokens=64, head_dim=64)
    d.update(kw)
    c = _hip.PttsPagedKV()
    for k, v in d.items():
        setattr(c, k, v)
    return c


def batch(**kw):
    d = dict(table=P, table_stride=4, past=P, starts=P, max_pages=4, n_seqs=2, tokens=5)
    d.update(kw)
    b = _hip.PttsPagedBatch()
    for k, v in d.items():
        setattr(b, k, v)
    return b


def rotary(**kw):
    d = dict(cos_t=P, sin_t=P, positions=128, dims=64, interleaved=0)
    d.update(kw)
    r = _hip.PttsRotary()
    for k, v in d.items():
        setattr(r, k, v)
    return r


def strides(*s):
    return (C.c_int64 * 3)(*s)


def attend(lib, c=None, b=None, heads=4, q=P, qs=(256, 64), out=2 * P, os=(256, 64), scale=0.125, mask=None, mstride=0, mwidth=0, max_new=0,
           ws=None, wsb=1 << 40, status=P):
    return lib.ptts_paged_attention(C.byref(c or kv()), C.byref(b or batch()), heads, q, *qs, out, *os, scale, 1, mask, mstride, mwidth,
                                    max_new, 4 * P if ws is None else ws, wsb, status, None)


def append(lib, c=None, b=None, dtype=1, k=P, ks=(128, 64), v=2 * P, vs=(128, 64), r=None, heads=0, q=None, qs=(0, 0), qo=None, qos=(0, 0),
           status=P):
    return lib.ptts_kv_append(C.byref(c or kv()), C.byref(b or batch()), dtype, k, *ks, v, *vs, C.byref(r) if r else None, None,
                              heads, q, *qs, qo, *qos, status, None)


BAD_CACHES = [dict(k=None), dict(v=None), dict(dtype=2), dict(n_pages=0), dict(kv_heads=0), dict(page_tokens=48), dict(page_tokens=8),
              dict(page_tokens=8192), dict(head_dim=96), dict(head_dim=0), dict(k=P + 2), dict(k_strides=strides(8192, 4096, 60)),
              dict(v_strides=strides(8192, 4096, 32)), dict(v_strides=strides(4096, 4096, 64)), dict(k_strides=strides(-8192, 4096, 64)),
              dict(k_strides=strides(1 << 50, 4096, 64))]
BAD_BATCHES = [dict(n_seqs=-1), dict(tokens=-1), dict(max_pages=-1), dict(past=None), dict(table=None), dict(starts=None), dict(table_stride=3)]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_bad_caches_are_refused_before_a_launch(lib, bad):
    assert attend(lib, kv(**bad)) in (-1, -5) and lib.ptts_last_error()
    assert append(lib, kv(**bad)) in (-1, -5)
    assert lib.ptts_paged_attention_workspace(C.byref(kv(**bad)), C.byref(batch()), 4, 0) in (-1, -5)


@pytest.mark.parametrize("bad", BAD_BATCHES, ids=str)
def test_bad_batches_are_refused_before_a_launch(lib, bad):
    assert attend(lib, b=batch(**bad)) == -1 and append(lib, b=batch(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(heads=3), dict(heads=0), dict(q=None), dict(q=P + 8), dict(qs=(256, 60)), dict(out=None), dict(out=2 * P + 4),
                                 dict(os=(64, 64)), dict(os=(256, 0)), dict(out=P), dict(out=P + 512), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=math.inf), dict(scale=math.nan), dict(mask=P, mstride=3, mwidth=4), dict(mask=P, mwidth=-1, mstride=4),
                                 dict(max_new=-1), dict(status=None), dict(qs=(-256, 64))], ids=str)
def test_bad_attention_calls_are_refused_before_a_launch(lib, bad):
    assert attend(lib, **bad) in (-1, -5) and lib.ptts_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(k=None), dict(v=None), dict(r=rotary(dims=66)), dict(r=rotary(dims=7)), dict(r=rotary(dims=0)),
                                 dict(r=rotary(cos_t=None)), dict(r=rotary(positions=0)), dict(heads=2), dict(heads=2, q=P, qs=(128, 64)),
                                 dict(heads=2, q=P, qs=(128, 64), qo=P + 64, qos=(128, 64)), dict(heads=2, q=P, qs=(128, 64), qo=3 * P, qos=(64, 64)),
                                 dict(heads=-1), dict(status=None), dict(c=kv(dtype=0, k_strides=strides(8192, 4096, 64)))], ids=str)
def test_bad_appends_are_refused_before_a_launch(lib, bad):
    assert append(lib, **bad) in (-1, -5) and lib.ptts_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(heads=0), dict(dim=63), dict(tokens=-1), dict(x=None), dict(out=None), dict(pos=None),
                                 dict(os=(32, 64)), dict(out=P + 64), dict(status=None), dict(r=rotary(dims=80))], ids=str)
def test_bad_rotations_are_refused_before_a_launch(lib, bad):
    d = dict(dtype=1, tokens=3, heads=2, dim=64, x=P, xs=(128, 64), pos=P, out=2 * P, os=(128, 64), status=P, r=rotary())
    d.update(bad)
    rc = lib.ptts_rotary_embed(C.byref(d["r"]), d["dtype"], d["tokens"], d["heads"], d["dim"], d["x"], *d["xs"], d["pos"], d["out"], *d["os"],
                               d["status"], None)
    assert rc in (-1, -5) and lib.ptts_last_error()


def test_a_workspace_that_is_too_small_is_refused(lib):
    """one token of two sequences over long tables: split over the keys, so partial results need room"""
    b = batch(starts=None, tokens=2, max_pages=4096, table_stride=4096)
    need = lib.ptts_paged_attention_workspace(C.byref(kv()), C.byref(b), 4, 1)
    assert need >= 0
    if need > 0:
        assert attend(lib, b=b, max_new=1, wsb=need - 1) == -1 and b"workspace" in lib.ptts_last_error()
        assert attend(lib, b=b, max_new=1, ws=4 * P + 4, wsb=1 << 40) == -1


def test_an_empty_batch_launches_nothing(lib):
    b = batch(n_seqs=0, tokens=0, starts=None)
    assert attend(lib, b=b) == 0 and append(lib, b=b) == 0
    assert lib.ptts_paged_attention_workspace(C.byref(kv()), C.byref(b), 4, 0) == 0


def test_the_cache_has_to_be_on_a_gpu_and_of_a_served_shape():
    with pytest.raises(ValueError, match="ROCm device"):
        PagedKVCache.from_tensors(torch.zeros(2, 2, 64, 64), torch.zeros(2, 2, 64, 64))
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        PagedKVCache.from_tensors(torch.zeros(2, 2, 64, 64).half(), torch.zeros(2, 2, 64, 64).half())
    with pytest.raises(ValueError, match="pages, kv_heads"):
        PagedKVCache.from_tensors(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64))


@pytest.mark.parametrize("bad", [dict(rotary_dim=7), dict(rotary_dim=66), dict(layout="other"), dict(positions=0), dict(scaling={"type": "cubic"}),
                                 dict(scaling={"type": "linear"}), dict(scaling={"type": "linear", "factor": 0}), dict(theta=-1.0),
                                 dict(scaling={"type": "linear", "factor": 2, "beta_fast": 3}), dict(scaling={"type": "yarn", "factor": 4}),
                                 dict(scaling={"type": "ntk", "factor": 2}, rotary_dim=2)], ids=str)
def test_bad_rotary_tables_are_refused(bad):
    d = dict(head_dim=64, positions=16, device="cpu")
    d.update(bad)
    with pytest.raises(ValueError):
        RotaryTable(**d)


def test_rotary_tables_are_64_bit_angles_rounded_once():
    """far positions: an angle of 131071 radians formed in 32 bits would be off by 4e-3"""
    t = RotaryTable(64, 131072, device="cpu")
    for pos in (0, 1, 4095, 131071):
        for i in (0, 1, 17, 31):
            angle = pos * 10000.0 ** (-2 * i / 64)
            # the angle's own 64-bit roundings: 4 x 2^-53 of it
            tol = 2.0 ** -24 + 4 * 2.0 ** -53 * (angle + 1)
            assert abs(float(t.cos[pos, i]) - math.cos(angle)) <= tol and abs(float(t.sin[pos, i]) - math.sin(angle)) <= tol


def test_rotary_scalings_keep_fast_pairs_and_stretch_slow_ones():
    base, one = rotary_frequencies(128)
    assert one == 1.0 and base[0] == 1.0
    lin, _ = rotary_frequencies(128, scaling={"type": "linear", "factor": 4})
    assert torch.allclose(lin * 4, base, rtol=1e-15, atol=0)
    ntk, _ = rotary_frequencies(128, scaling={"type": "ntk", "factor": 4})
    assert ntk[0] == 1.0 and abs(float(ntk[-1] * 4 / base[-1]) - 1) < 1e-12          # the slowest pair exactly interpolated
    yarn, gain = rotary_frequencies(128, scaling={"type": "yarn", "factor": 16, "original_positions": 4096})
    turns = 4096 * base / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], base[turns >= 32]) and torch.allclose(yarn[turns <= 1] * 16, base[turns <= 1], rtol=1e-15, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((yarn[mid] < base[mid]) & (yarn[mid] > base[mid] / 16)).all()
    assert abs(gain - (0.1 * math.log(16) + 1)) < 1e-15
    assert rotary_frequencies(128, scaling={"type": "yarn", "factor": 16, "original_positions": 4096, "attention_factor": 1.5})[1] == 1.5


def test_the_wrapper_refuses_what_does_not_fit_the_table():
    t = RotaryTable(64, 16, device="cpu")
    pos = torch.zeros(3, dtype=torch.int32)
    for x, p in ((torch.zeros(3, 2, 32), pos), (torch.zeros(3, 2, 64).half(), pos), (torch.zeros(3, 2, 64), pos.long()),
                 (torch.zeros(4, 2, 64), pos), (torch.zeros(3, 2, 128)[..., ::2], pos), (torch.zeros(3, 2, 64, requires_grad=True), pos),
                 (torch.zeros(3, 64), pos)):
        with pytest.raises(ValueError):
            rotary_embed(x, p, t)


def test_tensors_in_host_memory_are_refused_not_launched_on():
    t = RotaryTable(64, 16, device="cpu")
    with pytest.raises(ValueError, match="ROCm device"):
        rotary_embed(torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), t)
    with pytest.raises(ValueError, match="ROCm device"):
        PagedKVCache(4, 16, 2, 64, device="cpu")


def test_public_names():
    import parler_tts_amd as p

    for name in ("PagedKVCache", "RotaryTable", "rotary_embed", "kv_append", "paged_attention"):
        assert hasattr(p, name)


def test_the_matrix_instructions_of_the_attention_kernels_are_guarded_and_waited_for():
    """on the assembly that hipcc makes of them: no product under EXEC masking alone, no result read by inline assembly too early"""
    import importlib.util

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for name in ("check_mfma_guards", "check_mfma_asm_hazard"):
        spec = importlib.util.spec_from_file_location(name, os.path.join(root, "tools", name + ".py"))
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        assert mod.main([os.path.join(root, "parler_tts_amd", "csrc", "paged_attn.hip")]) == 0


def test_a_decoder_configuration_carries_its_rotary_scaling():
    from parler_tts_amd.configuration import ParlerTTSDecoderConfig, tiny_config
    from parler_tts_amd.weights import rope_tables

    scaling = {"type": "linear", "factor": 4.0}
    cfg = tiny_config(position_embedding="rope", rope_scaling=scaling).decoder
    assert ParlerTTSDecoderConfig.from_dict(cfg.to_dict()) == cfg and cfg.rope_scaling == scaling
    cos, sin = rope_tables(cfg, 9)
    freq, gain = rotary_frequencies(64, 10000.0, scaling=scaling)
    angle = torch.arange(9, dtype=torch.float64)[:, None] * freq
    assert torch.equal(cos, (torch.cos(angle) * gain).float()) and torch.equal(sin, (torch.sin(angle) * gain).float())
    plain = tiny_config(position_embedding="rope").decoder
    assert "rope_scaling" not in plain.to_dict()
    inv = torch.pow(torch.tensor(10000.0), -torch.arange(0, 64, 2, dtype=torch.float32) / 64)
    assert torch.equal(rope_tables(plain, 9)[0], torch.cos(torch.arange(9, dtype=torch.float32)[:, None] * inv))
    with pytest.raises(ValueError, match="type"):
        tiny_config(position_embedding="rope", rope_scaling={"type": "dynamic", "factor": 2.0})
    assert tiny_config(rope_scaling=scaling).decoder.rope_scaling is None      # no rotary positions: kept as an unknown entry, as before


def test_scalar_addresses_of_the_asynchronous_loads_are_written_in_time(tmp_path):
    """A vector instruction's write of a scalar register has to be five wait states old when a memory instruction reads it; hipcc sees to
    that for instructions it models, and the loads into LDS are inline assembly.  (Scalar instructions' writes need none.)"""
    import re
    import subprocess

    csrc = os.path.join(ROOT, "parler_tts_amd", "csrc")
    out = tmp_path / "paged_attn.s"
    subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "--cuda-device-only", "-S", os.path.join(csrc, "paged_attn.hip"), "-o", str(out)], check=True, capture_output=True)

    def early(lines):
        loads, found = 0, []
        for i, line in enumerate(lines):
            m = re.match(r"global_load_lds_dwordx4 v\d+, s\[(\d+):(\d+)\]", line)
            if not m:
                continue
            loads += 1
            waited = 0
            for x in reversed(lines[max(i - 40, 0):i]):
                if x.endswith(":"):
                    continue
                w = re.match(r"v_(?:readlane|readfirstlane)_b32 s(\d+)", x)
                if w and int(m[1]) <= int(w[1]) <= int(m[2]):
                    found.append((x, line))
                    break
                s = re.match(r"s_nop (\d+)", x)
                waited += 1 + (int(s[1]) if s else 0)
                if waited >= 5:
                    break
        return loads, found

    text = [t.split(";")[0].strip() for t in out.read_text().split("\n")]
    loads, found = early([t for t in text if t and (not t.startswith(".") or t.startswith(".LBB"))])
    assert loads > 100 and not found, found[:3]
    assert early(["v_readlane_b32 s5, v1, 3", "s_mov_b32 m0, s9", "s_nop 0", "global_load_lds_dwordx4 v2, s[4:5]"])[1]

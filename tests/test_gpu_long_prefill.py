"""Prefill behind position 5120 (score rows longer than the LDS holds): the engine's chunks go through the operators over a paged cache."""
import pytest
import torch

from tests.test_gpu_parity import _models, _oracle_vs_engine, hip  # noqa: F401  (hip: the fixture)

pytestmark = pytest.mark.gpu

YARN = {"type": "yarn", "factor": 4.0, "original_positions": 2048}


def model(**variant):
    from parler_tts_amd.configuration import tiny_config
    from parler_tts_amd.weights import synthetic_state_dict

    cfg = tiny_config(max_positions=6000, **variant)
    return cfg, synthetic_state_dict(cfg, seed=11, never_eos=True, ln_jitter=0.1, parts=("text_encoder", "decoder"))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("variant", [dict(), dict(position_embedding="rope"), dict(position_embedding="rope", rope_scaling=YARN)],
                         ids=["sinusoidal", "rope", "rope-yarn"])
def test_prompts_longer_than_the_score_rows(hip, dtype, variant):  # noqa: F811
    """5250 prompt positions (41 chunks, the last two behind the limit) of three ragged utterances against the plain PyTorch decoder,
    teacher-forced, held to what the same comparison is held to at 60 positions (tests/test_gpu_parity.py, decoder variants)"""
    cfg, sd = model(**variant)
    got, want, _, _ = _oracle_vs_engine(cfg, sd, dtype, B=3, T=10, P=5250, L=9, seed=12, steps=8, ragged=True)
    assert (got - want).abs().max() < (2e-4 if dtype == "fp32" else 0.08), (got - want).abs().max()
    _models.clear()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("variant", [dict(), dict(position_embedding="rope")], ids=["sinusoidal", "rope"])
def test_page_tables_masks_and_chunks_change_nothing(hip, dtype, variant, monkeypatch):  # noqa: F811
    """the same call with a page table read from memory: equal bit for bit; in chunks of 40: within the bound above"""
    cfg, sd = model(**variant)
    run = lambda reuse: _oracle_vs_engine(cfg, sd, dtype, B=2, T=10, P=5200, L=5, seed=3, steps=4, ragged=True, reuse_ref=reuse)[0]
    base = run(False)
    again = run(True)
    assert torch.equal(base, again)
    monkeypatch.setenv("PTTS_FORCE_PAGE_TABLE", "1")
    assert torch.equal(run(True), base)
    monkeypatch.setenv("PTTS_PREFILL_CHUNK", "40")
    assert (run(True) - base).abs().max() < (2e-4 if dtype == "fp32" else 0.08)
    _models.clear()


def test_a_second_call_with_a_longer_prompt_grows_the_workspace(hip):  # noqa: F811
    from parler_tts_amd.modeling import ParlerTTSForConditionalGeneration

    cfg, sd = model()
    m = ParlerTTSForConditionalGeneration(cfg, sd, dtype="bf16", device="cuda:0")
    g = torch.Generator().manual_seed(1)
    enc = torch.randn(2, 8, cfg.text_encoder.d_model, generator=g).cuda()
    prompt = torch.randint(2, cfg.vocab_size, (2, 5800), generator=g).cuda()
    ids = []
    for n in (5800, 100, 5300, 5800, 5130, 5800):
        m.generate(encoder_outputs=(enc,), prompt_input_ids=prompt[:, :n], do_sample=False, max_length=12, return_raw_ids=True)
        ids.append((n, m.last_raw_ids.clone()))
    same = [x for n, x in ids if n == 5800]
    assert all(torch.equal(x, same[0]) for x in same)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_short_prompts_on_the_long_route(hip, dtype):  # noqa: F811
    """PTTS_PREFILL_PAGED_FROM: every chunk, and (in chunks of 3) those behind position 4 only, against the default, on the cases and within the bounds of
    the batched prefill's own equivalence test (tests/test_gpu_parity.py); bf16 rounds the queries once more"""
    from tests.test_gpu_parity import _fresh_engine_logits

    tol = 2e-5 if dtype == "fp32" else 0.04
    for name in ("tiny_greedy", "tiny_greedy_ragged", "tiny_cfg"):
        a = _fresh_engine_logits(name, dtype, {"PTTS_PREFILL_PAGED_FROM": None})
        for env in ({"PTTS_PREFILL_PAGED_FROM": "0"}, {"PTTS_PREFILL_PAGED_FROM": "4", "PTTS_PREFILL_CHUNK": "3"}):
            b = _fresh_engine_logits(name, dtype, env)
            assert (a - b).abs().max().item() < tol, (name, env, (a - b).abs().max().item())

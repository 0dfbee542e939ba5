"""Beam search on the HIP engine: the engine's calls against the CPU oracle's, and the GPT session's search against the
oracle's and a float64 one (tests/test_beam_search.py, tests/beam_reference.py)."""
import numpy as np
import pytest

import nnengine
import test_beam_search as cpu_tests
from helpers import nrm_err

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [0, 1])
def test_calls_match_oracle(hip, cpu, seed):
    _, h = cpu_tests.run_ops(hip, seed)
    _, c = cpu_tests.run_ops(cpu, seed)
    for n in ("beam", "token", "table2", "lens2"):
        assert np.array_equal(h[n], c[n]), n
    for n in ("qr", "O", "score", "K", "V"):
        assert nrm_err(h[n], c[n]) <= 1e-5, n


def test_refusals(hip):
    for call, msg in cpu_tests.refusals(hip):
        with pytest.raises(nnengine.EngineError, match=msg):
            call()


@pytest.mark.parametrize("variant", cpu_tests.VARIANTS, ids=lambda v: v["pos_enc"])
@pytest.mark.parametrize("beams,n_prompt,max_new", [(1, 3, 5), (4, 5, 6), (7, 1, 20), (3, 14, 4), (23, 2, 3)])
def test_session_beam_search(hip, variant, beams, n_prompt, max_new):
    cfg = dict(cpu_tests.SMALL, **variant)
    params = cpu_tests.params_of(cfg, 3)
    g = hip.gpt(**cfg)
    g.set_params(params)
    prompt = np.random.default_rng(beams + n_prompt).integers(0, 23, n_prompt).tolist()
    for eos in (5, 23):
        print(f"[beam] {variant['pos_enc']} beams {beams} prompt {n_prompt} eos {eos}", flush=True)
        cpu_tests.check_beams(g.beam_search(prompt, beams, max_new, eos), params, prompt, beams, max_new, eos, cfg)


def test_long_prompt_and_training_between(hip):
    """A prompt of several chunks; a training step and a step of incremental inference in between change nothing."""
    cfg = dict(cpu_tests.SMALL, seq_len=160, pos_enc="alibi")
    params = cpu_tests.params_of(cfg, 4)
    g = hip.gpt(**cfg)
    g.set_params(params)
    prompt = np.random.default_rng(1).integers(0, 23, 150).tolist()
    first = g.beam_search(prompt, 4, 5, 5)
    cpu_tests.check_beams(first, params, prompt, 4, 5, 5, cfg)
    toks = np.random.default_rng(2).integers(0, 23, (161, 1))
    step0 = [g.forward_step(int(t), i, i) for i, t in enumerate(toks[:6, 0])]
    g.load_batch(toks[:160].astype(np.float32), toks[1:].T.reshape(-1))
    g.forward_loss()
    assert g.beam_search(prompt, 4, 5, 5) == first
    with pytest.raises(nnengine.EngineError, match="forward pass"):
        g.backward()
    g.forward_loss()
    g.backward()
    g.zero_grad()
    assert g.beam_search(prompt, 4, 5, 5) == first
    g.reset_cache()
    step1 = [g.forward_step(int(t), i, i) for i, t in enumerate(toks[:6, 0])]
    assert all(np.array_equal(a, b) for a, b in zip(step0, step1))


def test_one_beam_is_greedy(hip):
    """A 768-wide model with 12 heads: one beam follows generate at temperature 0, unless two logits are closer than
    float32 sums tell apart (totals then agree)."""
    cfg = dict(vocab_size=1024, d_model=768, seq_len=64, num_heads=12, d_ff=512, num_layers=2, pos_enc="rope")
    g = hip.gpt(**cfg)
    g.set_params(cpu_tests.params_of(cfg, 6, 0.05))
    prompt = list(range(40))
    one = g.beam_search(prompt, 1, 12)
    assert one[0][0] == g.generate(prompt, 12)
    best = g.beam_search(prompt, 8, 12)
    assert best[0][1] >= one[0][1] - 1e-3 and [s for _, s in best] == sorted((s for _, s in best), reverse=True)


@pytest.mark.parametrize("beams", [2, 6, 40, 70])
def test_group_whose_first_sequence_has_no_parent(hip, beams):
    cpu_tests.orphan_first(hip, beams)


def test_slices_are_copies(hip, cpu):
    h, c = cpu_tests.through_views(hip), cpu_tests.through_views(cpu)
    for n in ("table2", "lens2", "k", "v", "before", "both", "tables"):
        assert np.array_equal(h[n], c[n]), n
    for n in ("q", "O", "K", "V", "after"):
        assert nrm_err(h[n], c[n]) <= 1e-6, n

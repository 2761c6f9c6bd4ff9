"""Generation by sampling on the device (DecoderTransformerGpu.generate_sampled) against the same tokens drawn on the
host, by the definition in float64, from the logits that the model's single steps give."""
import numpy as np
import pytest

from oracle import model as OM
from tests.e4m3_ref import sample
from tests.test_model_gpu import _gpu_model

pytestmark = pytest.mark.gpu


def _model(ctx, vocab, batch, seq=48):
    cfg = OM.Config(vocab=vocab, d_model=64, n_layer=2, n_head=2, d_ff=128, seq_len_max=seq)
    P = OM.init_params(cfg, 5)
    P["w_tok"] = P["w_tok"] * np.float32(8)  # logits that differ
    return cfg, _gpu_model(ctx, cfg, batch, P)


@pytest.mark.parametrize("vocab,b", [(256, 3), (1024, 5), (8192, 2), (40000, 2), (256, 70)])
@pytest.mark.parametrize("kw", [{}, dict(temperature=0.7, top_k=20), dict(top_p=0.9, min_p=0.02), dict(temperature=1.3, top_k=100, top_p=0.8)])
def test_tokens_are_those_drawn_from_the_steps_logits(ctx, vocab, b, kw):
    cfg, m = _model(ctx, vocab, b)
    rng = np.random.default_rng(vocab)
    prompts = rng.integers(0, vocab, (b, 9)).astype(np.uint32)
    steps = 6
    u = rng.random((steps, b)).astype(np.float32)
    cache, other = m.kv_cache(b, 32), m.kv_cache(b, 32)
    logits = m.prefill_kv(cache, prompts)
    m.prefill_kv(other, prompts)
    tokens, logprob = m.generate_sampled(other, u, **kw)
    assert other.current_len == 9 + steps
    args = {n: (np.float32(x) if n != "top_k" else x) for n, x in kw.items()}
    for s in range(steps):
        for i in range(b):
            want, lp, near = sample(logits[i], u[s, i], **{n: float(x) if n != "top_k" else x for n, x in args.items()})
            assert tokens[s, i] == want or near < 1e-9
            if tokens[s, i] == want:
                assert abs(logprob[s, i] - lp) <= 2.0**-24 * abs(lp) + 1e-9
        logits, _ = m.generate_step_kv(cache, tokens[s])
    # the last token was fed as well: both caches go on alike
    a, _ = m.generate_step_kv(cache, tokens[-1])
    c, _ = m.generate_step_kv(other, tokens[-1])
    assert np.array_equal(a, c)
    for x in (cache, other, m):
        x.destroy()


def test_without_temperature_it_is_greedy(ctx):
    cfg, m = _model(ctx, 512, 4)
    prompts = np.random.default_rng(1).integers(0, 512, (4, 5)).astype(np.uint32)
    cache = m.kv_cache(4, 40)
    first = m.prefill_kv(cache, prompts).argmax(1)
    greedy = m.generate_greedy(cache, 10)
    m.prefill_kv(cache, prompts)
    tokens, logprob = m.generate_sampled(cache, np.zeros((11, 4)), temperature=0.0)
    assert np.array_equal(tokens[0], first) and np.array_equal(tokens[1:], greedy) and np.all(logprob == 0)
    # filters of each sequence's own, and a second run with more steps than the first
    m.prefill_kv(cache, prompts)
    again, _ = m.generate_sampled(cache, np.full((20, 4), 0.99), temperature=[0.0, 1.0, 0.0, 1.0], top_k=[0, 1, 5, 0],
                                  top_p=[1.0, 1.0, 0.5, 1e-6])
    assert np.array_equal(again[:11], tokens)
    cache.destroy(), m.destroy()


def test_refusals(ctx):
    from aurora_amd.gpu import AuroraError

    cfg, m = _model(ctx, 256, 2)
    cache = m.kv_cache(2, 16)
    with pytest.raises(AuroraError, match="prefill"):
        m.generate_sampled(cache, np.zeros((1, 2)))
    prompts = np.ones((2, 10), np.uint32)
    m.prefill_kv(cache, prompts)
    with pytest.raises(AuroraError, match="full"):
        m.generate_sampled(cache, np.zeros((7, 2)))
    assert cache.current_len == 10
    with pytest.raises(ValueError, match="shape"):
        m.generate_sampled(cache, np.zeros((2, 3)))
    tokens, _ = m.generate_sampled(cache, np.zeros((0, 2)))
    assert tokens.shape == (0, 2) and cache.current_len == 10
    m.generate_sampled(cache, np.zeros((6, 2)))
    assert cache.current_len == 16
    cache.destroy(), m.destroy()

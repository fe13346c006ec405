"""The decoder runner's sampling: each token drawn from the logits of the step before it."""
import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
dec = importlib.import_module("onnxruntime-mlx_amd.decoder")

CFG = dict(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, inter=512, vocab=1000)
SETTINGS = dict(temperature=1.3, top_k=40, top_p=0.9, min_p=0.01)
PROMPT = np.random.default_rng(3).integers(0, CFG["vocab"], size=9)


def drawn(logits, u, temperature, top_k, top_p, min_p):
    """The definition of sample_rows for one row, in 64 bits."""
    x = logits.astype(np.float64)
    order = np.argsort(-x, kind="stable")
    w = np.exp((x - x.max()) / np.float64(np.float32(temperature)))
    keep = np.zeros(len(x), bool)
    total, before = w[order[:top_k]].sum(), 0.0
    for i in order[:top_k]:
        keep[i] = before < np.float64(np.float32(top_p)) * total
        before += w[i]
    keep &= w >= np.float64(np.float32(min_p))
    cum = np.cumsum(np.where(keep, w, 0.0))
    return cum / cum[-1], int(np.argmax((cum > u * cum[-1]) & keep))


def test_each_token_is_drawn_from_its_logits():
    import torch

    cfg = dec.DecoderConfig(**CFG)
    r = dec.DecoderRunner(cfg, dec.make_weights(cfg, seed=5), cap=64, max_prompt=16,
                          sampling=dict(seed=11, **SETTINGS))
    random = torch.Generator(device="cuda").manual_seed(11)
    r.reset()
    r.prefill(PROMPT)
    S = len(PROMPT)
    for _ in range(12):
        torch.cuda.synchronize()
        u = float(torch.empty(1, device="cuda").uniform_(generator=random))
        cdf, want = drawn(r.logits[0, S - 1].float().cpu().numpy(), u, **SETTINGS)
        assert np.abs(cdf - u).min() > 1e-6  # no draw at a border
        assert int(r.next_id) == want
        r.decode_step()
        S = 1


def test_same_seed_same_tokens():
    cfg = dec.DecoderConfig(**CFG)
    w = dec.make_weights(cfg, seed=5)
    r = dec.DecoderRunner(cfg, w, cap=64, max_prompt=16, sampling=dict(seed=1, **SETTINGS))
    first = r.generate(PROMPT, steps=20)[0]
    assert r.generate(PROMPT, steps=20)[0] == first
    other = dec.DecoderRunner(cfg, w, cap=64, max_prompt=16, sampling=dict(seed=2, **SETTINGS))
    assert other.generate(PROMPT, steps=20)[0] != first


def test_temperature_zero_is_greedy():
    cfg = dec.DecoderConfig(**CFG)
    w = dec.make_weights(cfg, seed=5)
    r = dec.DecoderRunner(cfg, w, cap=64, max_prompt=16, sampling=dict(temperature=0.0))
    greedy = dec.DecoderRunner(cfg, w, cap=64, max_prompt=16)
    assert r.generate(PROMPT, steps=15)[0] == greedy.generate(PROMPT, steps=15)[0]


def test_refusals():
    cfg = dec.DecoderConfig(**CFG)
    w = dec.make_weights(cfg, seed=5)
    with pytest.raises(ValueError, match="argmax_node"):
        dec.DecoderRunner(cfg, w, cap=64, max_prompt=16, argmax_node=True, sampling={})
    with pytest.raises(ValueError, match="top_n"):
        dec.DecoderRunner(cfg, w, cap=64, max_prompt=16, sampling=dict(top_n=3))

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


def test_paged_cache_and_sampling_in_turn(ortmi):
    """Tokens of two sequences: attention over quantised pages, logits, a drawn token, whose
    query, key and value are the next step's. Every step against 64 bits."""
    import torch
    from kvq_ref import Attention, random_scales, rotary

    H, KV, hd, blk, V, dt = 4, 2, 64, 16, 500, torch.float16
    g = torch.Generator().manual_seed(8)
    ks, vs = (random_scales(g, KV, hd, "int4", False) for _ in range(2))
    cos, sin = rotary(g, 64, hd // 2, dt)
    ref = Attention(dt, "int4", H, KV, hd, ks, vs, 0.0, cos, sin)
    table = [torch.randn((V, n * hd), generator=g).to(dt) for n in (H, KV, KV)]
    head = torch.randn((H * hd, V), generator=g) * 0.3
    pages = [torch.zeros((8, blk, KV, hd // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    bt = torch.tensor([[5, 2, 7], [1, 6, 0]], dtype=torch.int32).cuda()
    kb = [torch.zeros((64, KV, hd // 2), dtype=torch.uint8) for _ in range(2)]
    vb = [x.clone() for x in kb]
    news, past = [list(range(20)), [3, 400, 17]], [0, 0]
    for _ in range(8):
        n = [len(x) for x in news]
        q, k, v = (t[torch.tensor(news[0] + news[1])] for t in table)
        out = ortmi.paged_attention_quantized(
            q.cuda(), k.cuda(), v.cuda(), *pages, ks.cuda(), vs.cuda(),
            torch.tensor([0, n[0], n[0] + n[1]], dtype=torch.int32).cuda(),
            torch.tensor(past, dtype=torch.int32).cuda(), bt, cos.cuda(), sin.cuda(),
            num_heads=H, kv_num_heads=KV, do_rotary=1)
        torch.cuda.synchronize()
        got, start = out.double().cpu(), 0
        for b in range(2):
            rows = slice(start, start + n[b])
            pos = torch.arange(past[b], past[b] + n[b])
            kb[b][pos], vb[b][pos] = ref.new_codes(k[rows], v[rows], pos)
            end = past[b] + n[b]
            o, tol = ref.rows(q[rows], pos, kb[b][:end], vb[b][:end],
                              torch.ones(end, dtype=torch.bool))
            assert ((got[rows] - o).abs() <= tol).all(), (b, past)
            start += n[b]
        last = torch.tensor([n[0] - 1, n[0] + n[1] - 1])
        logits = (got[last].float() @ head).to(dt)
        u = torch.rand(2, generator=g)
        ids, _ = ortmi.sample_rows(logits.cuda(), u.cuda(), **SETTINGS)
        for b in range(2):
            cdf, want = drawn(logits[b].float().numpy(), float(u[b]), **SETTINGS)
            assert np.abs(cdf - float(u[b])).min() > 1e-6
            assert int(ids[b]) == want
            past[b] += n[b]
            news[b] = [want]

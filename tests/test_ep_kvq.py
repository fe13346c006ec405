"""GroupQueryAttention with a quantised cache through the execution provider: what it claims
(CPU), and its steps against the kernel library's own entry point (GPU)."""
import importlib

import numpy as np
import pytest

PKG = "onnxruntime-mlx_amd"
hx = importlib.import_module(PKG + ".harness")
F16, F32, I32, I8, U8, F8 = hx.FLOAT16, hx.FLOAT, hx.INT32, hx.INT8, hx.UINT8, 17
H, KV, HD, CAP = 4, 2, 64, 40


def graph(cache=I8, scales=(1, 1), types=("PER_TENSOR", "PER_TENSOR"), batch=1, cap=CAP,
          width=None, extra=None, at=None, past=True, sdtype=F32, pv=None):
    g = hx.Graph()
    width = width or (HD // 2 if cache == U8 else HD)
    ins = ["q", "k", "v", "pk" if past else "", "pv" if past else "", "sl", "tot", "cos", "sin",
           "", "", "", "ks", "vs"]
    for n, heads in (("q", H), ("k", KV), ("v", KV)):
        g.value(n, F16, [batch, -1, heads * HD])
    if past:
        g.value("pk", cache, [batch, KV, cap, width])
        g.value("pv", cache if pv is None else pv, [batch, KV, cap, width])
    g.value("sl", I32, [batch])
    g.value("tot", I32, [1])
    g.value("o", F16, [batch, -1, H * HD])
    for n in ("ok", "ov"):
        g.value(n, cache, [batch, KV, -1, width])
    rows = np.arange(64, dtype=np.float64)[:, None] * 1e4 ** (-np.arange(HD // 2) / (HD / 2))
    g.initializer("cos", np.cos(rows).astype(np.float16))
    g.initializer("sin", np.sin(rows).astype(np.float16))
    for n, s in zip(("ks", "vs"), scales):
        if s is None:
            ins[12 if n == "ks" else 13] = ""
        else:
            g.value(n, sdtype, [s] if isinstance(s, int) else list(s))
    for i, (name, dtype, dims) in (at or {}).items():
        ins += [""] * (i + 1 - len(ins))
        ins[i] = name
        g.value(name, dtype, dims)
    while not ins[-1]:
        ins.pop()
    attrs = dict(num_heads=H, kv_num_heads=KV, do_rotary=1)
    for name, t in zip(("k_quant_type", "v_quant_type"), types):
        if t is not None:
            attrs[name] = t
    attrs.update(extra or {})
    g.node("GroupQueryAttention", ins, ["o", "ok", "ov"], domain="com.microsoft", **attrs)
    g.io([n for n in ins if n and n not in ("cos", "sin")], ["o", "ok", "ov"])
    return g


CHANNEL = ("PER_CHANNEL", "PER_CHANNEL")


@pytest.mark.parametrize("kw,claimed", [
    (dict(), True),
    (dict(cache=U8), True),
    (dict(cache=F8), True),
    (dict(scales=((KV, HD), (KV, HD)), types=CHANNEL), True),
    (dict(scales=(1, (KV, HD)), types=("PER_TENSOR", "PER_CHANNEL")), True),
    (dict(extra=dict(kv_cache_bit_width=8)), True),
    (dict(cache=U8, extra=dict(kv_cache_bit_width=4)), True),
    (dict(at={14: ("qn", F16, [HD]), 15: ("kn", F16, [HD])}), True),
    (dict(cache=U8, extra=dict(kv_cache_bit_width=8)), False),     # 4 bits
    (dict(extra=dict(kv_cache_bit_width=4)), False),               # 8 bits
    (dict(cache=U8, width=HD), False),                             # two codes a byte
    (dict(cache=F16), False),                                      # not codes
    (dict(pv=U8), False),                                          # two types
    (dict(scales=(1, None)), False),
    (dict(scales=(None, None)), False),
    (dict(scales=(2, 2)), False),
    (dict(types=CHANNEL), False),                                  # scales of one
    (dict(types=("PER_TENSOR", None)), False),
    (dict(types=("PER_TOKEN", "PER_TOKEN")), False),
    (dict(sdtype=F16), False),
    (dict(past=False), False),
    (dict(extra=dict(local_window_size=8)), False),
    (dict(extra=dict(sliding_window_cache=1, local_window_size=8)), False),
    (dict(at={10: ("bias", F16, [1, 1, 1, CAP])}), False),
    (dict(at={11: ("sink", F16, [H])}), False),
])
def test_claim(kw, claimed):
    assert hx.Session(graph(**kw), compile=False, force_device=True).claimed(0) is claimed


TORCH = {I8: "int8", U8: "uint8", F8: "float8_e4m3fn"}


@pytest.mark.gpu
@pytest.mark.parametrize("host", [False, True], ids=["device", "host"])
@pytest.mark.parametrize("channel", [False, True], ids=["tensor", "channel"])
@pytest.mark.parametrize("cache", [I8, U8, F8], ids=["int8", "int4", "fp8"])
def test_steps(ortmi, monkeypatch, cache, channel, host):
    """A prompt piece, single tokens and another piece of two sequences of different lengths,
    present over past: what the kernel library gives for the same calls, bit by bit."""
    import torch

    monkeypatch.setenv("ORTMI_EP_MEMORY", "cpu" if host else "hbm")
    B, dev = 2, "cpu" if host else "cuda"
    rng = np.random.default_rng(5)
    shape = (KV, HD) if channel else (1,)
    types = CHANNEL if channel else ("PER_TENSOR", "PER_TENSOR")
    sess = hx.Session(graph(cache, (shape, shape), types, batch=B))
    assert sess.partitions() == [[0]]
    step = {I8: 0.03, U8: 0.4, F8: 0.01}[cache]
    ks, vs = (torch.from_numpy((step * rng.uniform(0.5, 1.0, shape)).astype(np.float32))
              for _ in range(2))
    width = HD // 2 if cache == U8 else HD
    raw = [torch.zeros((B, KV, CAP, width), dtype=torch.uint8) for _ in range(4)]
    dtype = getattr(torch, TORCH[cache])
    kc, vc = (x.to(dev).view(dtype) for x in raw[:2])
    rk, rv = (x.cuda().view(dtype) for x in raw[2:])
    rows = np.arange(64, dtype=np.float64)[:, None] * 1e4 ** (-np.arange(HD // 2) / (HD / 2))
    cos, sin = (torch.from_numpy(f(rows).astype(np.float16)).cuda() for f in (np.cos, np.sin))
    sess.bind_output("ok", kc)
    sess.bind_output("ov", vc)
    total = 0
    for S, behind in ((7, 3), (1, 3), (1, 3), (12, 3), (1, 0)):
        total += S
        lens = torch.tensor([total - 1, total - 1 - behind], dtype=torch.int32)
        q, k, v = (torch.from_numpy(rng.standard_normal((B, S, n * HD)).astype(np.float16))
                   for n in (H, KV, KV))
        o = torch.empty((B, S, H * HD), dtype=torch.float16, device=dev)
        sess.bind_output("o", o)
        tot = torch.tensor([total], dtype=torch.int32)
        feeds = dict(q=(q, F16), k=(k, F16), v=(v, F16), pk=(kc, cache), pv=(vc, cache),
                     sl=(lens, I32), tot=(tot, I32), ks=(ks, F32), vs=(vs, F32))
        feeds = {n: (t.to(dev) if n not in ("sl", "tot") else t, d) for n, (t, d) in feeds.items()}
        torch.cuda.synchronize()
        sess.run(feeds)
        torch.cuda.synchronize()
        want = ortmi.group_query_attention_quantized(
            q.cuda(), k.cuda(), v.cuda(), rk, rv, ks.cuda(), vs.cuda(), lens.cuda(), total, cos,
            sin, num_heads=H, kv_num_heads=KV, do_rotary=1, k_quant_type=types[0],
            v_quant_type=types[1], present_key=rk, present_value=rv)[0]
        assert torch.equal(o.cpu(), want.cpu())
        for a, b in ((kc, rk), (vc, rv)):
            assert torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))
    sess.close()


@pytest.mark.gpu
def test_growing_cache(ortmi):
    """A full past: present is a longer buffer of its own."""
    import torch

    rng = np.random.default_rng(9)
    sess = hx.Session(graph(I8, cap=9))
    past = [torch.from_numpy(rng.integers(-128, 128, (1, KV, 9, HD), dtype=np.int8)).cuda()
            for _ in range(2)]
    q, k, v = (torch.from_numpy(rng.standard_normal((1, 2, n * HD)).astype(np.float16)).cuda()
               for n in (H, KV, KV))
    ks, vs = (torch.tensor([0.02], device="cuda") for _ in range(2))
    present = [torch.zeros((1, KV, 11, HD), dtype=torch.int8, device="cuda") for _ in range(2)]
    o = torch.empty((1, 2, H * HD), dtype=torch.float16, device="cuda")
    for n, t in (("o", o), ("ok", present[0]), ("ov", present[1])):
        sess.bind_output(n, t)
    torch.cuda.synchronize()
    sess.run(dict(q=(q, F16), k=(k, F16), v=(v, F16), pk=(past[0], I8), pv=(past[1], I8),
                  sl=(torch.tensor([10], dtype=torch.int32), I32),
                  tot=(torch.tensor([11], dtype=torch.int32), I32), ks=(ks, F32), vs=(vs, F32)))
    torch.cuda.synchronize()
    rows = np.arange(64, dtype=np.float64)[:, None] * 1e4 ** (-np.arange(HD // 2) / (HD / 2))
    cos, sin = (torch.from_numpy(f(rows).astype(np.float16)).cuda() for f in (np.cos, np.sin))
    want = ortmi.group_query_attention_quantized(
        q, k, v, past[0], past[1], ks, vs, torch.tensor([10], dtype=torch.int32, device="cuda"),
        11, cos, sin, num_heads=H, kv_num_heads=KV, do_rotary=1, k_quant_type="PER_TENSOR",
        v_quant_type="PER_TENSOR")
    for a, b in zip((o, *present), want):
        assert torch.equal(a, b)
    sess.close()

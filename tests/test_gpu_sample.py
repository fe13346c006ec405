"""Sampling on the GPU against numpy in 64 bits: tokens are equal, log-probabilities within
the steps of fp32 that a value of theirs has (the weights are 2e-12 exact).

A token can differ from the reference's where the uniform number, or a border of the kept
entries, falls within the weights' error of a border between entries: about 1e-9 of the
cases here."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def reference(x, u, temperature, top_k, top_p, min_p):
    """x [V] float64: (token, log-probability)."""
    ok = ~np.isnan(x) & (x > -np.inf)
    if not ok.any():
        return -1, -math.inf
    x = np.where(ok, x, -np.inf)
    order = np.lexsort((np.arange(len(x)), -x))[:int(ok.sum())]
    best = order[0]
    if not temperature > 0 or min_p > 1 or top_k == 1:
        return best, 0.0
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == x[best], 1.0, np.exp((x[order] - x[best]) / temperature))
    if top_p < 1:
        before = np.cumsum(w) - w
        n = max(1, int(np.sum(before < top_p * w.sum())))
        order, w = order[:n], w[:n]
    if min_p > 0:
        n = max(1, int(np.sum(w >= min_p)))
        order, w = order[:n], w[:n]
    back = np.argsort(order)
    cum = np.cumsum(w[back])
    some = np.flatnonzero(w[back] > 0)
    i = int(np.searchsorted(cum, u * cum[-1], side="right"))
    i = int(some[-1]) if i >= len(cum) else i
    return order[back[i]], math.log(w[back[i]] / cum[-1])


def run(ortmi, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x [rows, V] in its type; settings numbers or lists of one per row."""
    def arg(v, dtype):
        return torch.tensor(v, dtype=dtype).cuda() if isinstance(v, (list, tuple)) else v

    def row(v, r, dtype):
        return dtype(v[r]) if isinstance(v, (list, tuple)) else dtype(v)

    ids, lp = ortmi.sample_rows(x.cuda(), torch.tensor(u, dtype=torch.float32).cuda(),
                                temperature=arg(temperature, torch.float32),
                                top_k=arg(top_k, torch.int32), top_p=arg(top_p, torch.float32),
                                min_p=arg(min_p, torch.float32))
    torch.cuda.synchronize()
    ids, lp = ids.cpu().numpy(), lp.cpu().numpy()
    x64 = x.double().numpy()
    f = lambda v: float(np.float32(v))  # noqa: E731  (settings are 32-bit numbers)
    for r in range(x.shape[0]):
        want, p = reference(x64[r], f(u[r]), row(temperature, r, f), row(top_k, r, int),
                            row(top_p, r, f), row(min_p, r, f))
        assert ids[r] == want, (r, ids[r], want)
        if math.isinf(p):
            assert lp[r] == p
        else:
            # fp32 rounding, and weights 2e-12 exact above units of 2^-44.
            assert abs(lp[r] - p) <= 2.0 ** -23 * abs(p) + 1e-9, (r, lp[r], p)
    return ids


def logits(rows, V, dtype, seed, sd=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, V), generator=g) * sd).to(DT[dtype])


def numbers(rows, seed):
    return np.random.default_rng(seed).random(rows, np.float32).tolist()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 8191, 8192, 8193, 32064, 50257, 151936])
def test_sizes(ortmi, dtype, V):
    rows = 5
    x, u = logits(rows, V, dtype, V), numbers(rows, V)
    run(ortmi, x, u)
    run(ortmi, x, u, temperature=0.7, top_k=40, top_p=0.9)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kw", [
    dict(top_k=1), dict(top_k=2), dict(top_k=50), dict(top_k=1500), dict(top_k=5000),
    dict(top_k=10 ** 6), dict(top_p=0.0), dict(top_p=1e-6), dict(top_p=0.5), dict(top_p=0.99),
    dict(top_p=0.999999), dict(min_p=0.1), dict(min_p=1.0), dict(min_p=1.5), dict(min_p=1e-4),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=0.01),
    dict(temperature=30.0), dict(temperature=1e-30), dict(temperature=math.inf),
    dict(top_k=100, top_p=0.8, min_p=0.05, temperature=1.3),
    dict(top_k=-3, top_p=1.5, min_p=-0.5), dict(top_k=700, top_p=0.95, temperature=3.0),
])
def test_settings(ortmi, dtype, kw):
    rows = 6
    run(ortmi, logits(rows, 5000, dtype, 11), numbers(rows, 12), **kw)


def test_a_setting_for_each_row(ortmi):
    rows = 40
    r = np.random.default_rng(5)
    run(ortmi, logits(rows, 3001, "bf16", 6), numbers(rows, 7),
        temperature=[float(t) for t in r.choice([0.0, 0.5, 1.0, 2.0], rows)],
        top_k=[int(k) for k in r.choice([0, 1, 3, 50, 4000], rows)],
        top_p=[float(p) for p in r.choice([0.1, 0.9, 1.0], rows)],
        min_p=[float(p) for p in r.choice([0.0, 0.02, 0.5], rows)])


def test_ties(ortmi):
    """Equal logits: the lower index first; a border inside a group of equals."""
    rows = 4
    for V, dtype in ((1, "f16"), (4096, "bf16"), (20000, "f32")):
        run(ortmi, torch.zeros((rows, V), dtype=DT[dtype]), numbers(rows, V))
        run(ortmi, torch.zeros((rows, V), dtype=DT[dtype]), numbers(rows, V), top_k=17)
        run(ortmi, torch.zeros((rows, V), dtype=DT[dtype]), numbers(rows, V), top_p=0.5)
        run(ortmi, torch.zeros((rows, V), dtype=DT[dtype]), numbers(rows, V), top_k=1000,
            top_p=0.25)
    x = (logits(8, 6000, "f32", 3) * 2).round() / 2  # a few dozen different logits
    x[0, ::2] = -0.0
    for kw in (dict(top_k=100), dict(top_p=0.6), dict(top_k=300, top_p=0.7), dict(min_p=0.3)):
        run(ortmi, x, numbers(8, 4), **kw)
        run(ortmi, x.half(), numbers(8, 4), **kw)


def test_masked_rows(ortmi):
    """-inf, the type's lowest value, NaN and +inf among the logits."""
    inf, nan = math.inf, math.nan
    for dtype in ("f16", "bf16", "f32"):
        x = logits(7, 2000, dtype, 9)
        x[0, :] = -inf
        x[1, :] = nan
        x[2, 10:] = -inf
        x[3, ::3] = nan
        x[4, :1999] = torch.finfo(x.dtype).min
        x[5, [7, 900]] = inf
        x[6, 5:] = torch.finfo(x.dtype).min
        for kw in ({}, dict(top_k=20), dict(top_p=0.9), dict(temperature=0.0), dict(min_p=0.1)):
            ids = run(ortmi, x, numbers(7, 3), **kw)
            assert ids[0] == ids[1] == -1 and ids[2] < 10 and ids[4] == 1999
            assert ids[5] in (7, 900) and ids[6] < 5


def test_extreme_uniform_numbers(ortmi):
    x = logits(4, 1000, "f16", 1)
    u = [0.0, float(np.nextafter(np.float32(1), np.float32(0))), 1e-30, 0.5]
    for kw in ({}, dict(top_k=30), dict(top_p=0.7)):
        run(ortmi, x, u, **kw)
    # 1 and beyond take the last kept entry.
    ids = ortmi.sample_rows(x.cuda(), torch.tensor([1.0, 2.0, -1.0, float("nan")]).cuda())[0]
    assert ids[0].item() <= 999 and ids[1].item() >= 0 and ids[2].item() == 0
    assert 0 <= ids[3].item() < 1000


def test_wide_and_narrow_rows(ortmi):
    """Logits far apart, and so close that only low bits differ."""
    x = logits(4, 9000, "f32", 2)
    run(ortmi, x * 1e4, numbers(4, 1), top_p=0.9)
    run(ortmi, x * 1e-4 + 100, numbers(4, 2), top_k=77, top_p=0.9)
    run(ortmi, x * 1e30, numbers(4, 3), top_k=10)
    run(ortmi, x * 1e-38, numbers(4, 4), top_k=10, top_p=0.5)


def test_shares(ortmi):
    """Many uniform numbers over one row: each token as often as its weight says."""
    x = logits(1, 12, "f32", 8)
    n = 4096
    u = ((torch.arange(n) + 0.5) / n).cuda()
    ids = ortmi.sample_rows(x.expand(n, 12).contiguous().cuda(), u, top_k=5)[0].cpu()
    w = torch.softmax(x[0].double(), 0)
    keep = torch.topk(w, 5).indices
    share = torch.zeros(12, dtype=torch.float64)
    share[keep] = w[keep] / w[keep].sum()
    count = torch.bincount(ids, minlength=12).double() / n
    assert (count - share).abs().max() <= 1.0 / n  # an interval's length, rounded


def test_same_every_time_and_on_another_stream(ortmi):
    x, u = logits(64, 32064, "bf16", 4).cuda(), torch.tensor(numbers(64, 9)).cuda()
    a = ortmi.sample_rows(x, u, top_p=0.95)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ortmi.sample_rows(x, u, top_p=0.95)
    side.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_captured_and_replayed(ortmi):
    x, u = logits(3, 32064, "f16", 4).cuda(), torch.tensor(numbers(3, 9)).cuda()
    V = x.shape[1]
    need = ortmi.load_kernels().ortmi_sample_rows_workspace_size(3, V)
    ws = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ortmi.sample_rows(x, u, top_k=50, top_p=0.9, workspace=ws)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, lp = ortmi.sample_rows(x, u, top_k=50, top_p=0.9, workspace=ws)
    for step in range(4):
        x.add_(torch.randn(x.shape, device="cuda") * 0.3)
        u.copy_(torch.rand(3))
        want = ortmi.sample_rows(x, u, top_k=50, top_p=0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, want[0]) and torch.equal(lp, want[1])


def test_shapes_and_refusals(ortmi):
    x = logits(6, 100, "f32", 4).cuda()
    u = torch.rand(6).cuda()
    ids, lp = ortmi.sample_rows(x.view(2, 3, 100), u)
    assert ids.shape == lp.shape == (2, 3)
    assert ortmi.sample_rows(x[:0], u[:0])[0].numel() == 0
    for bad in (dict(uniform=u[:5]), dict(uniform=u.double()), dict(logits=x.t()),
                dict(logits=x.double()), dict(logits=x.cpu()), dict(top_k=torch.ones(6).cuda()),
                dict(top_p=torch.ones(5).cuda()),
                dict(logits=torch.zeros((1, (1 << 18) + 1)).cuda(), uniform=u[:1]),
                dict(logits=torch.zeros((6, 0)).cuda())):
        with pytest.raises((TypeError, ValueError, ortmi.KernelError)):
            ortmi.sample_rows(**{**dict(logits=x, uniform=u), **bad})

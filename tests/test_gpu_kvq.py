"""Attention over quantised key-value caches on the GPU against 64-bit arithmetic
(kvq_ref.py, where the bound on an output is derived). Codes are compared exactly."""

from __future__ import annotations

import pytest
import torch
from kvq_ref import CDT, DT, Attention, random_codes, random_scales, rotary

pytestmark = pytest.mark.gpu


def close(out, ref, tol, what=""):
    out = out.double().cpu().reshape(ref.shape)
    bad = ~((out - ref).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outputs off, first at {i}: "
                             f"{out[i]} against {ref[i]} +- {tol[i]}")


def put(t, shift=0):
    """On the GPU, `shift` elements behind an aligned address."""
    raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    buf = torch.zeros(raw.numel() + shift, dtype=raw.dtype, device="cuda")
    buf[shift:] = raw.flatten().cuda()
    return buf[shift:].view(t.dtype).view(t.shape)


def stored(t):
    return t.view(torch.uint8).cpu()


def make_gqa(code="int8", dtype="f16", B=1, S=1, past=40, H=4, KV=2, hd=64, channel=True,
             half=None, interleaved=False, packed=False, mode="inplace", lens=None, room=3,
             normed=False, scale=0.0, seed=0, shift=0):
    """(arguments of the call, reference, new rows): lens = tokens of each sequence."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed * 7919 + S * 131 + past + H + hd)
    half = hd // 2 if half is None else half
    n = [past + S] * B if lens is None else list(lens)

    def rnd(*shape, sd=1.0):
        return (torch.randn(shape, generator=g) * sd).to(dt)

    q, k, v = rnd(B, S, H * hd), rnd(B, S, KV * hd), rnd(B, S, KV * hd)
    cap = past if mode == "grow" else past + S + room
    kb, vb = (random_codes(g, (B, KV, cap, hd), code) for _ in range(2))
    ks, vs = (random_scales(g, KV, hd, code, channel) for _ in range(2))
    cos, sin = rotary(g, past + S + 2, half, dt) if half else (None, None)
    qw, kw = (rnd(hd, sd=0.1) + 1 for _ in range(2)) if normed else (None, None)
    ref = Attention(dt, code, H, KV, hd, ks, vs, scale, cos, sin, interleaved, qw, kw)
    dev = lambda t: None if t is None else put(t, shift)  # noqa: E731
    pk, pv = (put(t.view(CDT[code]), shift) for t in (kb, vb))
    args = dict(query=dev(torch.cat([q, k, v], -1)) if packed else dev(q),
                key=None if packed else dev(k), value=None if packed else dev(v), past_key=pk,
                past_value=pv, k_scale=ks.cuda(), v_scale=vs.cuda(),
                seqlens_k=None if lens is None else
                torch.tensor([x - 1 for x in n], dtype=torch.int32).cuda(),
                total_sequence_length=past + S, cos_cache=dev(cos), sin_cache=dev(sin),
                num_heads=H, kv_num_heads=KV, scale=scale, do_rotary=int(half > 0),
                rotary_interleaved=int(interleaved), q_norm_weight=dev(qw),
                k_norm_weight=dev(kw), k_quant_type="PER_CHANNEL" if channel else "PER_TENSOR",
                v_quant_type="PER_CHANNEL" if channel else "PER_TENSOR")
    if mode == "inplace":
        args.update(present_key=pk, present_value=pv)
    return args, dict(ref=ref, q=q, k=k, v=v, kb=kb, vb=vb, n=n, S=S, mode=mode, past=past)


def check_gqa(ortmi, got, t):
    out, pk, pv = got
    ref, S = t["ref"], t["S"]
    grow = t["mode"] == "grow"
    pk, pv = stored(pk), stored(pv)
    for b, n in enumerate(t["n"]):
        p0 = max(n - S, 0)
        real = min(n, S)
        pos = torch.arange(p0, p0 + real)
        kc, vc = ref.new_codes(t["k"][b, :real], t["v"][b, :real], pos)
        kb, vb = t["kb"][b].transpose(0, 1).clone(), t["vb"][b].transpose(0, 1).clone()
        if grow:
            pad = kb.new_zeros((S, *kb.shape[1:]))
            kb, vb = torch.cat([kb[:t["past"]], pad]), torch.cat([vb[:t["past"]], pad])
        kb[p0:p0 + real], vb[p0:p0 + real] = kc, vc
        # Rows of a grown buffer past the sequence's end hold anything.
        keep = n if grow else kb.shape[0]
        assert torch.equal(pk[b].transpose(0, 1)[:keep], kb[:keep]), f"keys of sequence {b}"
        assert torch.equal(pv[b].transpose(0, 1)[:keep], vb[:keep]), f"values of sequence {b}"
        o, tol = ref.rows(t["q"][b, :real], pos, kb[:n], vb[:n], torch.ones(n, dtype=torch.bool))
        close(out[b, :real], o, tol, f"sequence {b}")
        assert (out[b, real:] == 0).all(), "padded rows are zero"


def run_gqa(ortmi, **kw):
    args, t = make_gqa(**kw)
    got = ortmi.group_query_attention_quantized(**args)
    torch.cuda.synchronize()
    check_gqa(ortmi, got, t)


@pytest.mark.parametrize("code", ["int8", "int4", "fp8"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_token(ortmi, code, dtype, hd):
    run_gqa(ortmi, code=code, dtype=dtype, hd=hd, B=2, past=77, H=6, KV=2)


@pytest.mark.parametrize("past", [0, 1, 14, 15, 30, 31, 32, 63, 126, 127, 128, 255, 640])
def test_token_lengths(ortmi, past):
    run_gqa(ortmi, past=past, H=8, KV=2, hd=128)


@pytest.mark.parametrize("H,KV", [(1, 1), (3, 3), (7, 1), (14, 2), (16, 1), (17, 1), (40, 1),
                                  (64, 1)])
def test_groups(ortmi, H, KV):
    run_gqa(ortmi, H=H, KV=KV, past=70, B=2, code="int4")


@pytest.mark.parametrize("code", ["int8", "int4", "fp8"])
@pytest.mark.parametrize("S,past", [(2, 0), (5, 33), (16, 100), (17, 0), (33, 64), (64, 1),
                                    (100, 29), (130, 0)])
def test_rows(ortmi, code, S, past):
    run_gqa(ortmi, code=code, S=S, past=past, H=4, KV=2, hd=64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("S,past,hd", [(9, 200, 128), (40, 40, 96), (75, 0, 128)])
def test_rows_types(ortmi, dtype, S, past, hd):
    run_gqa(ortmi, dtype=dtype, S=S, past=past, hd=hd, H=6, KV=2, B=2)


@pytest.mark.parametrize("hd", [16, 48, 80, 192, 256])
def test_other_heads(ortmi, hd):
    run_gqa(ortmi, hd=hd, S=3, past=20, code="int4")
    run_gqa(ortmi, hd=hd, S=1, past=20, code="fp8", dtype="f32")


def test_options(ortmi):
    run_gqa(ortmi, interleaved=True, S=4)
    run_gqa(ortmi, half=12, S=4)
    run_gqa(ortmi, half=7, S=3, code="int4")
    run_gqa(ortmi, half=0, S=4)
    run_gqa(ortmi, packed=True, S=4, B=2)
    run_gqa(ortmi, channel=False, S=4)
    run_gqa(ortmi, normed=True, S=4, B=2)
    run_gqa(ortmi, normed=True, S=70, hd=128, interleaved=True)
    run_gqa(ortmi, scale=0.3, S=2)
    run_gqa(ortmi, scale=-0.2, S=40)


@pytest.mark.parametrize("shift", [1, 3, 8])
def test_unaligned(ortmi, shift):
    run_gqa(ortmi, shift=shift, S=1, past=50, hd=128)
    run_gqa(ortmi, shift=shift, S=70, past=5, code="fp8")


@pytest.mark.parametrize("mode", ["copy", "grow"])
@pytest.mark.parametrize("S,past", [(1, 0), (1, 60), (20, 33), (70, 130)])
def test_present_of_its_own(ortmi, mode, S, past):
    run_gqa(ortmi, mode=mode, S=S, past=past, B=2, code="int4")


def test_lengths_on_the_device(ortmi):
    run_gqa(ortmi, B=4, S=1, past=200, lens=[201, 1, 64, 130])
    run_gqa(ortmi, B=3, S=6, past=100, lens=[106, 6, 33], H=8)
    # A padded prompt: sequences shorter than S, one of them empty.
    run_gqa(ortmi, B=4, S=40, past=0, lens=[40, 1, 0, 17])
    run_gqa(ortmi, B=3, S=100, past=0, lens=[100, 65, 3], H=8, hd=128)


def test_long_split(ortmi):
    run_gqa(ortmi, S=1, past=6000, H=4, KV=1, hd=128, B=2, lens=[6001, 2500])
    run_gqa(ortmi, S=50, past=3000, H=4, KV=1, hd=64, code="int4")


def test_values_that_are_not_finite(ortmi):
    """New rows: NaN is stored as 0, infinities as the largest code. Codes behind a
    sequence's end and rows of other heads do not reach an output."""
    args, t = make_gqa(code="fp8", S=3, past=20, B=2, lens=[23, 10], room=40)
    for x, d in ((t["k"], args["key"]), (t["v"], args["value"])):
        x[0, 0, 5], x[0, 1, 6], x[0, 2, 7] = float("nan"), float("inf"), -float("inf")
        d.copy_(x)
    for name, b in (("past_key", "kb"), ("past_value", "vb")):
        t[b][0, :, 23:], t[b][1, :, 10:] = 0x7F, 0xFF
        args[name].view(torch.uint8).copy_(t[b])
    # A rotation mixes a NaN into the channel that it turns with: no rotation here.
    args["do_rotary"], t["ref"].cos = 0, None
    got = ortmi.group_query_attention_quantized(**args)
    torch.cuda.synchronize()
    assert torch.isfinite(got[0].float()).all()
    check_gqa(ortmi, got, t)
    # A query row that is not finite stays in its own output row.
    args, t = make_gqa(S=4, past=20)
    args["query"][0, 1] = float("nan")
    out = ortmi.group_query_attention_quantized(**args)[0]
    assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, [0, 2, 3]].float()).all()


def test_large_and_small_values(ortmi):
    """Scores far beyond an fp16 product's range, and scales near its smallest values."""
    for S in (1, 40):
        args, t = make_gqa(S=S, past=90, dtype="bf16", channel=False)
        t["ref"].s_k = t["ref"].s_k * 2.0 ** -20
        args["k_scale"] *= 2.0 ** -20
        t["q"] *= 2.0 ** 20
        t["k"] *= 2.0 ** -20
        args["query"].copy_(t["q"])
        args["key"].copy_(t["k"])
        got = ortmi.group_query_attention_quantized(**args)
        torch.cuda.synchronize()
        check_gqa(ortmi, got, t)


def test_captured_and_replayed(ortmi):
    """One captured step, replayed as the sequences grow, against eager calls."""
    args, t = make_gqa(B=2, S=1, past=300, lens=[20, 250], room=3)
    eager = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    eager["present_key"], eager["present_value"] = eager["past_key"], eager["past_value"]
    need = ortmi.load_kernels().ortmi_group_query_attention_quantized_workspace_size(
        2, 1, 4, 2, 64, 301)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    before = args["past_key"].clone(), args["past_value"].clone()
    with torch.cuda.stream(side):
        ortmi.group_query_attention_quantized(**args, workspace=ws)
    side.synchronize()
    with torch.cuda.graph(graph):
        out = ortmi.group_query_attention_quantized(**args, workspace=ws)[0]
    args["past_key"].copy_(before[0])
    args["past_value"].copy_(before[1])
    for step in range(4):
        want = ortmi.group_query_attention_quantized(**eager)[0]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(args["past_key"], eager["past_key"])
        for a in (args, eager):
            a["seqlens_k"] += 13
            a["query"].mul_(0.9)
            a["key"].add_(0.1)


def test_on_another_stream(ortmi):
    args, t = make_gqa(B=2, S=1, past=500, H=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ortmi.group_query_attention_quantized(**args)
    side.synchronize()
    check_gqa(ortmi, got, t)


def test_offsets_past_32_bits(ortmi):
    """Slabs that begin behind 2^32 bytes."""
    cap, B, hd = 1 << 20, 36, 128
    args, t = make_gqa(B=1, S=1, past=50, H=4, KV=1, hd=hd, room=0)
    big = {}
    for name in ("past_key", "past_value"):
        big[name] = torch.empty((B, 1, cap, hd), dtype=torch.int8, device="cuda")
        big[name][B - 1, :, :51] = args[name][0]
    assert (B - 1) * cap * hd > 1 << 32
    rep = lambda x: x.expand(B, *x.shape[1:]).contiguous()  # noqa: E731
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens[B - 1] = 50
    args.update(query=rep(args["query"]), key=rep(args["key"]), value=rep(args["value"]),
                past_key=big["past_key"], past_value=big["past_value"],
                present_key=big["past_key"], present_value=big["past_value"], seqlens_k=lens)
    out, pk, pv = ortmi.group_query_attention_quantized(**args)
    torch.cuda.synchronize()
    check_gqa(ortmi, (out[B - 1:], pk[B - 1:, :, :51].clone(), pv[B - 1:, :, :51].clone()), t)


# ------------------------------------------------------------------------- pages --
def make_paged(code="int8", dtype="f16", past=(40, 3), new=(1, 5), H=4, KV=2, hd=64, blk=16,
               channel=True, half=None, interleaved=False, normed=False, sink=False, spare=2,
               extra=0, seed=0, limit=None):
    """`extra` tokens behind the last sequence."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed * 7919 + sum(past) + 31 * sum(new) + H + hd + blk)
    half = hd // 2 if half is None else half
    T, end = sum(new) + extra, [p + n for p, n in zip(past, new)]
    nb = [-(-max(e, 1) // blk) for e in end]
    total = sum(nb) + spare
    perm = torch.randperm(total, generator=g)
    bt = torch.zeros((len(nb), max(nb)), dtype=torch.int32)
    o = 0
    for b, x in enumerate(nb):
        bt[b, :x] = perm[o:o + x].int()
        o += x

    def rnd(*shape, sd=1.0):
        return (torch.randn(shape, generator=g) * sd).to(dt)

    q, k, v = rnd(T, H * hd), rnd(T, KV * hd), rnd(T, KV * hd)
    kb, vb = (random_codes(g, (total, blk, KV, hd), code) for _ in range(2))
    ks, vs = (random_scales(g, KV, hd, code, channel) for _ in range(2))
    cos, sin = rotary(g, max(end) + 2, half, dt) if half else (None, None)
    qw, kw = (rnd(hd, sd=0.1) + 1 for _ in range(2)) if normed else (None, None)
    sk = rnd(H, sd=2.0) if sink else None
    ref = Attention(dt, code, H, KV, hd, ks, vs, 0.0, cos, sin, interleaved, qw, kw, sink=sk)
    cum = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    kind = "PER_CHANNEL" if channel else "PER_TENSOR"
    args = dict(query=dev(q), key=dev(k), value=dev(v),
                key_cache=kb.view(CDT[code]).cuda(), value_cache=vb.view(CDT[code]).cuda(),
                k_scale=ks.cuda(), v_scale=vs.cuda(), cumulative_sequence_length=cum.cuda(),
                past_seqlens=torch.tensor(past, dtype=torch.int32).cuda(), block_table=bt.cuda(),
                cos_cache=dev(cos), sin_cache=dev(sin), head_sink=dev(sk), q_norm_weight=dev(qw),
                k_norm_weight=dev(kw), num_heads=H, kv_num_heads=KV, do_rotary=int(half > 0),
                rotary_interleaved=int(interleaved), k_quant_type=kind, v_quant_type=kind,
                max_context=limit)
    return args, dict(ref=ref, q=q, k=k, v=v, kb=kb, vb=vb, bt=bt, past=past, new=new, blk=blk,
                      total=total, limit=limit)


def check_paged(got, args, t):
    ref, blk = t["ref"], t["blk"]
    kb, vb = t["kb"].flatten(0, 1).clone(), t["vb"].flatten(0, 1).clone()
    at, jobs = 0, []
    for b, (p, n) in enumerate(zip(t["past"], t["new"])):
        j = torch.arange(p + n)
        ids = t["bt"][b].long()[j // blk]
        ok = (ids >= 0) & (ids < t["total"])
        slots = torch.where(ok, ids, 0) * blk + j % blk
        pos = j[p:]
        kc, vc = ref.new_codes(t["k"][at:at + n], t["v"][at:at + n], pos)
        w = ok[p:]
        kb[slots[p:][w]], vb[slots[p:][w]] = kc[w], vc[w]
        jobs.append((at, n, pos, slots, ok))
        at += n
    assert torch.equal(stored(args["key_cache"]).flatten(0, 1), kb), "key pages"
    assert torch.equal(stored(args["value_cache"]).flatten(0, 1), vb), "value pages"
    for at, n, pos, slots, ok in jobs:
        if n == 0:
            continue
        if t["limit"]:
            slots, ok = slots[:t["limit"]], ok[:t["limit"]]
        o, tol = ref.rows(t["q"][at:at + n], pos, kb[slots], vb[slots], ok)
        close(got[at:at + n], o, tol, f"tokens from {at}")


def run_paged(ortmi, **kw):
    args, t = make_paged(**kw)
    got = ortmi.paged_attention_quantized(**args)
    torch.cuda.synchronize()
    check_paged(got, args, t)


@pytest.mark.parametrize("code", ["int8", "int4", "fp8"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_pages(ortmi, code, dtype, hd):
    run_paged(ortmi, code=code, dtype=dtype, hd=hd, past=(40, 3, 0, 200, 127),
              new=(1, 5, 33, 1, 70))


@pytest.mark.parametrize("blk", [1, 5, 8, 16, 24, 32, 48, 100, 256])
def test_page_sizes(ortmi, blk):
    run_paged(ortmi, blk=blk, past=(100, 31, 15), new=(1, 2, 40))
    run_paged(ortmi, blk=blk, past=(130,), new=(1,), code="int4", hd=128)


@pytest.mark.parametrize("H,KV", [(3, 3), (14, 2), (16, 1), (20, 1), (64, 1)])
def test_page_groups(ortmi, H, KV):
    run_paged(ortmi, H=H, KV=KV, past=(100, 31, 0), new=(1, 2, 21))


def test_page_options(ortmi):
    run_paged(ortmi, interleaved=True, half=16)
    run_paged(ortmi, half=0, channel=False)
    run_paged(ortmi, normed=True, sink=True)
    run_paged(ortmi, sink=True, past=(1500, 0, 700), new=(1, 80, 30), H=8, KV=1)
    run_paged(ortmi, hd=80, past=(20, 5), new=(1, 4))


def test_many_sequences(ortmi):
    past = tuple((37 * i) % 90 for i in range(150))
    run_paged(ortmi, past=past, new=tuple(1 if i % 3 else i % 4 for i in range(150)), hd=64)
    run_paged(ortmi, past=past, new=(1,) * 150, hd=64, H=2, KV=2, code="int4")


def test_long_pages(ortmi):
    run_paged(ortmi, past=(5000, 100, 2047), new=(1, 1, 1), H=4, KV=1, hd=128)
    run_paged(ortmi, past=(3000, 2), new=(40, 150), H=4, KV=1, hd=128, code="int4")


def test_rows_behind_the_last_sequence(ortmi):
    args, t = make_paged(extra=4, past=(20, 7), new=(1, 30))
    got = ortmi.paged_attention_quantized(**args)
    torch.cuda.synchronize()
    check_paged(got, args, t)
    lib, p = ortmi.load_kernels(), lambda x: x.data_ptr()
    T = args["query"].shape[0]
    out = torch.full((T, 256), 7.0, dtype=torch.float16, device="cuda")
    bt = args["block_table"]
    need = lib.ortmi_paged_attention_quantized_workspace_size(T, 2, 4, 2, 64, bt.shape[1] * 16)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    ortmi.check(lib.ortmi_paged_attention_quantized(
        p(args["query"]), p(args["key"]), p(args["value"]), p(args["key_cache"]),
        p(args["value_cache"]), t["total"], 16, p(args["cumulative_sequence_length"]),
        p(args["past_seqlens"]), p(bt), 2, bt.shape[1], T, bt.shape[1] * 16,
        p(args["cos_cache"]), p(args["sin_cache"]), 32, args["cos_cache"].shape[0], 0, None, None,
        None, 1e-6, p(args["k_scale"]), p(args["v_scale"]), 1, 1, ortmi.ORTMI_INT8, p(out), 4, 2,
        64, 0.0, 10, p(ws), need, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    check_paged(out, args, t)
    assert (out[T - 4:] == 7).all()


def test_bad_blocks(ortmi):
    """Positions whose block is not of the cache are neither written nor attended; pages that
    a sequence does not hold may hold NaN."""
    args, t = make_paged(code="fp8", past=(70, 40), new=(2, 30), spare=4)
    for bad in ((0, 1, -1), (0, 2, t["total"]), (1, 3, 1 << 30)):
        t["bt"][bad[0], bad[1]] = bad[2]
    args["block_table"].copy_(t["bt"])
    free = [i for i in range(t["total"]) if not (t["bt"] == i).any()]
    for name, b in (("key_cache", "kb"), ("value_cache", "vb")):
        t[b][free] = 0x7F
        args[name].view(torch.uint8).copy_(t[b])
    got = ortmi.paged_attention_quantized(**args)
    torch.cuda.synchronize()
    check_paged(got, args, t)


def test_no_block_at_all(ortmi):
    """A row that attends nothing is zero, or all its weight is the sink's."""
    for sink in (False, True):
        args, t = make_paged(past=(20,), new=(1,), sink=sink)
        t["bt"][:] = -1
        args["block_table"].fill_(-1)
        got = ortmi.paged_attention_quantized(**args)
        torch.cuda.synchronize()
        assert (got == 0).all()


def test_context_limit(ortmi):
    run_paged(ortmi, past=(100, 10), new=(1, 40), limit=64)
    run_paged(ortmi, past=(300, 10), new=(1, 300), limit=200)


def test_malformed_lengths(ortmi):
    """Lengths that contradict each other give some output, and no access outside."""
    args, t = make_paged(past=(40, 3, 9), new=(1, 5, 3))
    for cum in ([0, 500, 2, 9], [-5, 1, 6, 9], [3, 3, 3, 3], [9, 9, 9, 9]):
        for past in ([1 << 30, 5, 9], [-7, 3, 2 ** 31 - 1]):
            args["cumulative_sequence_length"].copy_(torch.tensor(cum))
            args["past_seqlens"].copy_(torch.tensor(past))
            ortmi.paged_attention_quantized(**args)
            torch.cuda.synchronize()


def test_pages_past_32_bits(ortmi):
    """Pages behind 2^32 bytes of the cache."""
    args, t = make_paged(past=(100, 31), new=(1, 40), hd=128, KV=2, spare=0)
    blk, used = t["blk"], t["total"]
    total = (1 << 32) // (blk * 2 * 128) + used + 8
    far = total - used
    for name, b in (("key_cache", "kb"), ("value_cache", "vb")):
        big = torch.empty((total, blk, 2, 128), dtype=torch.int8, device="cuda")
        big[far:] = args[name]
        args[name] = big
    args["block_table"] += far
    got = ortmi.paged_attention_quantized(**args)
    torch.cuda.synchronize()
    args["key_cache"], args["value_cache"] = (args[n][far:].clone()
                                              for n in ("key_cache", "value_cache"))
    check_paged(got, args, t)


def test_pages_captured_and_replayed(ortmi):
    args, t = make_paged(past=(500, 31, 4), new=(1, 1, 1), hd=128, H=8)
    eager = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in args.items()}
    bt = args["block_table"]
    need = ortmi.load_kernels().ortmi_paged_attention_quantized_workspace_size(
        3, 3, 8, 2, 128, bt.shape[1] * 16)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ortmi.paged_attention_quantized(**args, workspace=ws)
    side.synchronize()
    with torch.cuda.graph(graph):
        out = ortmi.paged_attention_quantized(**args, workspace=ws)
    for step in range(4):
        want = ortmi.paged_attention_quantized(**eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(args["key_cache"], eager["key_cache"])
        for a in (args, eager):
            a["past_seqlens"].add_(torch.tensor([0, 1, 3], device="cuda", dtype=torch.int32))
            a["query"].mul_(0.9)
            a["value"].add_(0.1)


def test_a_run_of_steps(ortmi):
    """A prompt, drafted tokens and single tokens in turn over one slab cache and over pages
    that hold the same sequence: codes equal, outputs within twice the bound."""
    H, KV, hd, blk, total = 8, 2, 128, 16, 150
    g = torch.Generator().manual_seed(5)
    dt = torch.bfloat16
    ks, vs = (random_scales(g, KV, hd, "int8", True) for _ in range(2))
    cos, sin = rotary(g, total, hd // 2, dt)
    ref = Attention(dt, "int8", H, KV, hd, ks, vs, 0.0, cos, sin)
    slab = [torch.zeros((1, KV, total, hd), dtype=torch.int8, device="cuda") for _ in range(2)]
    pages = [torch.zeros((total // blk + 1, blk, KV, hd), dtype=torch.int8, device="cuda")
             for _ in range(2)]
    bt = torch.arange(total // blk + 1, dtype=torch.int32).flip(0)[None].contiguous().cuda()
    kb = torch.zeros((total, KV, hd), dtype=torch.uint8)
    vb = kb.clone()
    at = 0
    kw = dict(num_heads=H, kv_num_heads=KV, do_rotary=1, k_quant_type="PER_CHANNEL",
              v_quant_type="PER_CHANNEL")
    for S in (90, 1, 1, 5, 1, 17, 1):
        q, k, v = (torch.randn((S, n * hd), generator=g).to(dt) for n in (H, KV, KV))
        pos = torch.arange(at, at + S)
        kb[at:at + S], vb[at:at + S] = ref.new_codes(k, v, pos)
        o, tol = ref.rows(q, pos, kb[:at + S], vb[:at + S],
                          torch.ones(at + S, dtype=torch.bool))
        a = ortmi.group_query_attention_quantized(
            q[None].cuda(), k[None].cuda(), v[None].cuda(), *slab, ks.cuda(), vs.cuda(), None,
            at + S, cos.cuda(), sin.cuda(), present_key=slab[0], present_value=slab[1], **kw)[0]
        b = ortmi.paged_attention_quantized(
            q.cuda(), k.cuda(), v.cuda(), *pages, ks.cuda(), vs.cuda(),
            torch.tensor([0, S], dtype=torch.int32).cuda(),
            torch.tensor([at], dtype=torch.int32).cuda(), bt, cos.cuda(), sin.cuda(), **kw)
        torch.cuda.synchronize()
        close(a[0], o, tol, f"slab, {S} tokens at {at}")
        close(b, o, tol, f"pages, {S} tokens at {at}")
        at += S
    assert torch.equal(stored(slab[0])[0].transpose(0, 1)[:at], kb[:at])
    assert torch.equal(stored(slab[1])[0].transpose(0, 1)[:at], vb[:at])

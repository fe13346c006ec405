"""Timed cases of attention over quantised key-value caches and of token sampling.

Kinds of case ("kind" of the case dict):

  gqa     one GroupQueryAttention call whose past and present hold codes (int8, packed
          int4 or fp8 e4m3) with static scales: new rows are rotated, quantised and
          written into the shared buffer, and every key and value is read as the
          buffer holds it. One token, a few drafted tokens, or a prompt.
  paged   the same over a block-paged cache, sequences that decode beside sequences
          that bring a chunk of a prompt.
  sample  one token per row of logits, from temperature, top-k, top-p, min-p and one
          given uniform number per row.

Head layouts and lengths are those of this repository's benchmark, decoder layouts and
tests. Inputs are made on the GPU from the seed alone. `own` selects the framework's
operators; without it `run` computes the same from elementary torch operations: in 32
bits, and in 64 where a value is rounded to a code or compared with a border.
"""

from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

PKG = "onnxruntime-mlx_amd"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
# Bytes per cached element, and the largest code.
CODE_BYTES = {"int8": 1.0, "int4": 0.5, "fp8": 1.0}
CODE_MAX = {"int8": 127.0, "int4": 7.0, "fp8": 448.0}


def listed():
    return [
        # A small decoder's single request, early in its answer: the smallest call.
        dict(name="gqa_int8_token", kind="gqa", dtype="f16", code="int8", channel=False, B=1, S=1,
             past=511, H=12, KV=2, hd=128, ragged=False),
        # One decode step of eight sequences at a 4096-token context.
        dict(name="gqa_int8_batch8_4k", kind="gqa", dtype="f16", code="int8", channel=True, B=8,
             S=1, past=4096, H=32, KV=8, hd=128, ragged=False),
        # Sixteen long documents, of different lengths, in the smallest cache.
        dict(name="gqa_int4_batch16_32k", kind="gqa", dtype="bf16", code="int4", channel=True,
             B=16, S=1, past=32767, H=32, KV=8, hd=128, ragged=True),
        # Eight drafted tokens verified at once by an fp32-activation export.
        dict(name="gqa_int8_f32_draft8", kind="gqa", dtype="f32", code="int8", channel=True, B=1,
             S=8, past=1003, H=14, KV=2, hd=64, ragged=False),
        # A 2048-token prompt.
        dict(name="gqa_int8_prompt_2k", kind="gqa", dtype="f16", code="int8", channel=True, B=1,
             S=2048, past=0, H=32, KV=8, hd=128, ragged=False),
        # A second turn of two conversations: ragged prompt pieces behind cached ones.
        dict(name="gqa_fp8_turn", kind="gqa", dtype="bf16", code="fp8", channel=False, B=2, S=333,
             past=1500, H=14, KV=2, hd=64, ragged=True),
        # Continuous batching, all sequences decoding.
        dict(name="paged_int8_decode", kind="paged", dtype="f16", code="int8", channel=True,
             nseq=32, prefill=0, chunk=1, lo=256, hi=8192, H=32, KV=8, hd=128, blk=16),
        # Continuous batching: four prompt chunks beside 28 decoding sequences.
        dict(name="paged_int4_mixed", kind="paged", dtype="bf16", code="int4", channel=True,
             nseq=32, prefill=4, chunk=256, lo=256, hi=8192, H=32, KV=8, hd=128, blk=16),
        # A few short sequences of a small model, prompt chunks of odd length among them.
        dict(name="paged_fp8_small", kind="paged", dtype="f16", code="fp8", channel=False, nseq=5,
             prefill=2, chunk=77, lo=100, hi=700, H=14, KV=2, hd=64, blk=32),
        # One request's next token with common settings: latency counts.
        dict(name="sample_one", kind="sample", dtype="f16", rows=1, V=151936, temperature=0.8,
             top_k=50, top_p=0.9, min_p=0.0, mixed=False),
        # A batch that samples from the nucleus alone, fp32 logits.
        dict(name="sample_nucleus32", kind="sample", dtype="f32", rows=32, V=128256,
             temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, mixed=False),
        # A large serving batch, every request with settings of its own.
        dict(name="sample_mixed256", kind="sample", dtype="bf16", rows=256, V=151936,
             temperature=0.9, top_k=64, top_p=0.92, min_p=0.02, mixed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["gqa", "paged", "sample"], [5, 3, 3])[0]
    if kind == "sample":
        V = rng.choice([32064, 128256, 151936, _log_int(rng, 1000, 151936)])
        return dict(kind=kind, dtype=rng.choice(["f16", "bf16", "f32"]),
                    rows=_log_int(rng, 1, 128), V=V,
                    temperature=round(rng.uniform(0.3, 1.5), 2),
                    top_k=rng.choice([0, 0, 1, 20, 50, _log_int(rng, 2, 1000)]),
                    top_p=rng.choice([1.0, 1.0, 0.9, round(rng.uniform(0.1, 0.999), 3)]),
                    min_p=rng.choice([0.0, 0.0, 0.05, round(rng.uniform(0.0, 0.3), 3)]),
                    mixed=rng.random() < 0.3)
    code = rng.choices(["int8", "int4", "fp8"], [4, 3, 2])[0]
    channel = rng.random() < 0.6
    H, KV = rng.choice([(14, 2), (12, 2), (32, 8), (24, 8), (32, 32), (16, 4)])
    if kind == "gqa":
        dtype = rng.choices(["f16", "bf16", "f32"], [5, 4, 2])[0]
        hd = rng.choice([64, 96, 128, 128])
        form = rng.choices(["token", "draft", "prompt"], [5, 2, 4])[0]
        S = {"token": 1, "draft": rng.randint(2, 16), "prompt": _log_int(rng, 17, 2048)}[form]
        B = _log_int(rng, 1, 16) if S <= 16 else _log_int(rng, 1, 4)
        past = _log_int(rng, 1, 32767) if S <= 16 or rng.random() < 0.4 else 0
        while (B * KV * (past + S) * hd > 2 ** 27 or B * H * S * (past + S / 2) * hd > 2 ** 32):
            past, S, B = past * 2 // 3, max(1, S * 2 // 3), max(1, B * 2 // 3)
        return dict(kind=kind, dtype=dtype, code=code, channel=channel, B=B, S=S, past=past, H=H,
                    KV=KV, hd=hd, ragged=rng.random() < 0.5)
    return dict(kind=kind, dtype=rng.choice(["f16", "bf16"]), code=code, channel=channel,
                nseq=_log_int(rng, 2, 32), prefill=rng.randint(0, 4),
                chunk=_log_int(rng, 2, 256), lo=256, hi=_log_int(rng, 300, 8192), H=min(H, 32),
                KV=min(KV, 8), hd=rng.choice([64, 128]), blk=rng.choice([16, 32, 48]))


# ----------------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, shape, dtype, sd=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * sd).to(dtype)


def _rotary(max_pos, hd, dtype, base=10000.0):
    half = hd // 2
    inv = 1.0 / base ** (torch.arange(half, dtype=torch.float64, device="cuda") / half)
    ang = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return ang.cos().to(dtype), ang.sin().to(dtype)


def _scales(g, c, KV, hd):
    """Scale of 3.5 standard deviations at the largest code (calibrated on such rows),
    per tensor [1] or per channel [KV, hd] with channels of different sizes."""
    n = (KV, hd) if c["channel"] else (1,)
    spread = 0.75 + 0.5 * torch.rand(n, generator=g, device="cuda")
    return spread * (3.5 / CODE_MAX[c["code"]])


def _random_codes(g, shape, code):
    """Codes of standard normal rows under _scales: [..., hd] -> the stored form."""
    x = torch.randn(shape, generator=g, device="cuda") * (CODE_MAX[code] / 3.5)
    if code == "int8":
        return x.round_().clamp_(-128, 127).to(torch.int8)
    if code == "fp8":
        return x.clamp_(-448, 448).to(torch.float8_e4m3fn)
    u = x.round_().clamp_(-8, 7).add_(8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _lengths(c):
    """Tokens of each sequence, the new ones included: the same for all seeds."""
    rng = np.random.default_rng(c["B"] * 7919 + c["past"] * 31 + c["S"])
    full = c["past"] + c["S"]
    if not c["ragged"]:
        return np.full(c["B"], full)
    # Behind a cache every sequence brings S tokens; a first prompt is padded to S.
    low = c["S"] + c["past"] // 2 if c["past"] else max(1, c["S"] // 2)
    n = rng.integers(low, full + 1, size=c["B"])
    n[0] = full
    return n


def _page_lengths(c):
    """(tokens of each sequence, new tokens of each): the same for all seeds."""
    rng = np.random.default_rng(c["nseq"] * 7919 + c["hi"])
    ctx = rng.integers(c["lo"], max(c["lo"], c["hi"]) + 1, size=c["nseq"])
    new = np.ones(c["nseq"], np.int64)
    k = min(c["prefill"], c["nseq"])
    # Chunks of different lengths, the first a whole one.
    new[:k] = rng.integers(max(1, c["chunk"] * 3 // 4), c["chunk"] + 1, size=k)
    new[:min(k, 1)] = c["chunk"]
    return np.maximum(ctx, new), new


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["kind"] == "sample":
        rows, V = c["rows"], c["V"]
        # A peaked row: a normal body of logits and some candidates above it.
        x = torch.randn((rows, V), generator=g, device="cuda") * 1.8
        top = torch.randint(0, V, (rows, 40), generator=g, device="cuda")
        high = 8 + 3 * torch.randn((rows, 40), generator=g, device="cuda")
        x.scatter_reduce_(1, top, high, "amax")
        st = dict(case=c, logits=x.to(DTYPES[c["dtype"]]),
                  uniform=torch.rand(rows, generator=g, device="cuda"),
                  temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"],
                  min_p=c["min_p"])
        if c["mixed"]:  # one setting for each row, greedy and unrestricted rows among them
            kind = torch.randint(0, 8, (rows,), generator=g, device="cuda")
            t = c["temperature"] * (0.7 + 0.6 * torch.rand(rows, generator=g, device="cuda"))
            st["temperature"] = torch.where(kind == 0, 0.0, t)
            st["top_k"] = torch.where(kind < 4, c["top_k"], 0).to(torch.int32)
            st["top_p"] = torch.where(kind % 2 == 0, c["top_p"], 1.0).float()
            st["min_p"] = torch.where(kind % 3 == 0, c["min_p"], 0.0).float()
        return st
    dt, H, KV, hd = DTYPES[c["dtype"]], c["H"], c["KV"], c["hd"]
    ks, vs = _scales(g, c, KV, hd), _scales(g, c, KV, hd)
    if c["kind"] == "gqa":
        B, S = c["B"], c["S"]
        n = _lengths(c)
        cap = c["past"] + S
        d = dict(q=_normal(g, (B, S, H * hd), dt), k=_normal(g, (B, S, KV * hd), dt),
                 v=_normal(g, (B, S, KV * hd), dt),
                 kc=_random_codes(g, (B, KV, cap, hd), c["code"]),
                 vc=_random_codes(g, (B, KV, cap, hd), c["code"]), total=cap)
        d["seqlens_k"] = torch.from_numpy((n - 1).astype(np.int32)).cuda()
    else:
        ctx, new = _page_lengths(c)
        blk, nseq, T = c["blk"], c["nseq"], int(new.sum())
        nblocks = -(-ctx // blk)
        total, maxb = int(nblocks.sum()), int(nblocks.max())
        perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
        first = torch.from_numpy(np.concatenate([[0], np.cumsum(nblocks)[:-1]])).cuda()
        at = first[:, None] + torch.arange(maxb, device="cuda")[None, :]
        used = torch.arange(maxb, device="cuda")[None, :] < torch.from_numpy(nblocks).cuda()[:, None]
        bt = torch.where(used, perm[at.clamp_max(total - 1)], 0).to(torch.int32).contiguous()
        d = dict(q=_normal(g, (T, H * hd), dt), k=_normal(g, (T, KV * hd), dt),
                 v=_normal(g, (T, KV * hd), dt),
                 kc=_random_codes(g, (total, blk, KV, hd), c["code"]),
                 vc=_random_codes(g, (total, blk, KV, hd), c["code"]), bt=bt,
                 context=int(ctx.max()), longest=int(new.max()))
        d["cum"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        d["past"] = torch.from_numpy((ctx - new).astype(np.int32)).cuda()
        cap = int(ctx.max())
    d["cos"], d["sin"] = _rotary(cap, hd, dt)
    return dict(d, case=c, ks=ks, vs=vs)


# -------------------------------------------------------------- plain arithmetic --

def _rope(x, cos, sin, pos):
    """Half-split rotation of x [..., heads, hd] at pos [...]; both 64-bit."""
    cos, sin = cos.double()[pos].unsqueeze(-2), sin.double()[pos].unsqueeze(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _encode(x, scale, code):
    """The stored form of 64-bit rows x [..., KV, hd]: a code is the nearest to x / scale,
    ties to even. Bytes."""
    r = x / (scale.double() if scale.numel() > 1 else scale.double().reshape(()))
    if code == "int8":
        return r.round().clamp(-128, 127).to(torch.int8).view(torch.uint8)
    if code == "int4":
        u = r.round().clamp(-8, 7).add(8).to(torch.uint8)
        return u[..., 0::2] | (u[..., 1::2] << 4)
    _, e = torch.frexp(r)
    step = torch.ldexp(torch.ones_like(r), e.clamp(min=-5) - 4)  # 3 bits behind the first
    return ((r / step).round() * step).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(
        torch.uint8)


def _decode(u, scale, code):
    """32-bit values of stored bytes u [..., KV, n]."""
    if code == "int8":
        x = u.view(torch.int8).float()
    elif code == "fp8":
        x = u.view(torch.float8_e4m3fn).float()
    else:
        x = torch.stack([u & 15, u >> 4], -1).flatten(-2).float() - 8
    return x * scale


def _softmax_rows(q, k, v, see):
    """softmax(q k^T) v over the keys that `see` allows (at least none): 32 bits."""
    s = (q @ k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    s = torch.where(see, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    return (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _gqa_plain(st):
    c = st["case"]
    B, S, H, KV, hd, code = c["B"], c["S"], c["H"], c["KV"], c["hd"], c["code"]
    G = H // KV
    n = st["seqlens_k"].long() + 1
    pos = (n - S).clamp(min=0)[:, None] + torch.arange(S, device="cuda")  # [B, S]
    real = pos < n[:, None]
    q = _rope(st["q"].double().view(B, S, H, hd), st["cos"], st["sin"], pos)
    k = _rope(st["k"].double().view(B, S, KV, hd), st["cos"], st["sin"], pos)
    for cache, x, scale in ((st["kc"], k, st["ks"]),
                            (st["vc"], st["v"].double().view(B, S, KV, hd), st["vs"])):
        u = cache.view(torch.uint8)
        new = _encode(x, scale, code).transpose(1, 2)  # [B, KV, S, bytes]
        at = pos[:, None, :, None].expand_as(new)
        old = u.gather(2, at)
        u.scatter_(2, at, torch.where(real[:, None, :, None], new, old))
    keys = _decode(st["kc"].view(torch.uint8).transpose(1, 2), st["ks"], code).transpose(1, 2)
    vals = _decode(st["vc"].view(torch.uint8).transpose(1, 2), st["vs"], code).transpose(1, 2)
    see = torch.arange(keys.shape[2], device="cuda") <= pos[:, None, None, :, None]
    see = see & real[:, None, None, :, None]
    # Heads of a group as further rows of their key head.
    rows = q.float().view(B, S, KV, G, hd).permute(0, 2, 3, 1, 4).reshape(B, KV, G * S, hd)
    see = see.expand(B, 1, G, S, -1).reshape(B, 1, G * S, -1)
    o = _softmax_rows(rows, keys, vals, see)
    o = o.view(B, KV, G, S, hd).permute(0, 3, 1, 2, 4).reshape(B, S, H * hd)
    return o.to(st["q"].dtype), st["kc"], st["vc"]


def _paged_plain(st):
    c = st["case"]
    H, KV, hd, blk, code = c["H"], c["KV"], c["hd"], c["blk"], c["code"]
    G, T, nseq = H // KV, st["q"].shape[0], c["nseq"]
    cum, past, table = st["cum"].long(), st["past"].long(), st["bt"].long()
    tok = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cum[1:].contiguous(), tok, right=True)
    row = tok - cum[seq]  # the token's place among its sequence's new ones
    pos = past[seq] + row
    slot = table[seq, pos // blk] * blk + pos % blk
    q = _rope(st["q"].double().view(T, H, hd), st["cos"], st["sin"], pos)
    k = _rope(st["k"].double().view(T, KV, hd), st["cos"], st["sin"], pos)
    for cache, x, scale in ((st["kc"], k, st["ks"]),
                            (st["vc"], st["v"].double().view(T, KV, hd), st["vs"])):
        u = cache.view(torch.uint8)
        u.view(-1, *u.shape[2:])[slot] = _encode(x, scale, code)
    # Every sequence's rows side by side, padded to the longest.
    n, longest = st["context"], st["longest"]
    j = torch.arange(n, device="cuda")
    slots = table[:, j // blk] * blk + j % blk  # [nseq, n]; past a sequence's end: hidden
    rows = torch.zeros((nseq, longest, H, hd), device="cuda")
    rows[seq, row] = q.float()
    rows = rows.view(nseq, longest, KV, G, hd).permute(0, 2, 3, 1, 4)
    rows = rows.reshape(nseq, KV, G * longest, hd)
    see = j <= past[:, None, None] + torch.arange(longest, device="cuda")[None, :, None]
    see = see[:, None, None].expand(nseq, 1, G, longest, n).reshape(nseq, 1, G * longest, n)
    kc, vc = (st[x].view(torch.uint8).flatten(0, 1)[slots] for x in ("kc", "vc"))
    o = _softmax_rows(rows, _decode(kc, st["ks"], code).transpose(1, 2),
                      _decode(vc, st["vs"], code).transpose(1, 2), see)
    o = o.view(nseq, KV, G, longest, hd).permute(0, 3, 1, 2, 4)[seq, row]
    return o.reshape(T, H * hd).to(st["q"].dtype), st["kc"], st["vc"]


def _sample_plain(st):
    """Borders (a nucleus' end, the uniform number's place) decide: 64 bits throughout."""
    x = st["logits"].double()
    rows, V = x.shape

    def column(name, dtype):
        return torch.as_tensor(st[name], device="cuda").to(dtype).expand(rows)[:, None]

    t, top_k = column("temperature", torch.float64), column("top_k", torch.int64)
    # Settings are 32-bit numbers, however they are given.
    t = t.float().double()
    top_p, min_p = (column(p, torch.float32).double() for p in ("top_p", "min_p"))
    val, order = torch.sort(x, dim=-1, descending=True, stable=True)
    rank = torch.arange(V, device="cuda")[None, :]
    w = torch.exp((val - val[:, :1]) / torch.where(t > 0, t, 1.0))
    greedy = t <= 0
    keep = (rank < torch.where((top_k > 0) & ~greedy, top_k, V)) & (~greedy | (rank == 0))
    w = torch.where(keep, w, 0.0)
    cum = torch.cumsum(w, -1)
    keep &= (cum - w < top_p * cum[:, -1:]) | (top_p >= 1) | (rank == 0)
    keep &= (w >= min_p) | (min_p <= 0) | (rank == 0)
    w = torch.where(keep, w, 0.0)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    cum = torch.cumsum(by_index, -1)
    u = st["uniform"].double()[:, None]
    hit = (cum > u * cum[:, -1:]) & (by_index > 0)
    ids = torch.argmax(hit.to(torch.uint8), -1)
    p = by_index.gather(1, ids[:, None])[:, 0] / cum[:, -1]
    return ids, torch.log(p).float()


def run(state):
    c = state["case"]
    if own:
        ops = importlib.import_module(PKG + ".ops")
        if c["kind"] == "sample":
            ids, logprobs = ops.sample_rows(
                state["logits"], state["uniform"], temperature=state["temperature"],
                top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
            return dict(ids=ids, logprobs=logprobs)
        kind = "PER_CHANNEL" if c["channel"] else "PER_TENSOR"
        if c["kind"] == "gqa":
            out, k, v = ops.group_query_attention_quantized(
                state["q"], state["k"], state["v"], state["kc"], state["vc"], state["ks"],
                state["vs"], state["seqlens_k"], state["total"], state["cos"], state["sin"],
                num_heads=c["H"], kv_num_heads=c["KV"], do_rotary=1, k_quant_type=kind,
                v_quant_type=kind, present_key=state["kc"], present_value=state["vc"])
            return dict(out=out, present_key=k, present_value=v)
        out = ops.paged_attention_quantized(
            state["q"], state["k"], state["v"], state["kc"], state["vc"], state["ks"],
            state["vs"], state["cum"], state["past"], state["bt"], state["cos"], state["sin"],
            num_heads=c["H"], kv_num_heads=c["KV"], do_rotary=1, k_quant_type=kind,
            v_quant_type=kind, max_context=state["context"])
        return dict(out=out, key_cache=state["kc"], value_cache=state["vc"])
    if c["kind"] == "sample":
        ids, logprobs = _sample_plain(state)
        return dict(ids=ids, logprobs=logprobs)
    if c["kind"] == "gqa":
        out, k, v = _gqa_plain(state)
        return dict(out=out, present_key=k, present_value=v)
    out, k, v = _paged_plain(state)
    return dict(out=out, key_cache=k, value_cache=v)


# --------------------------------------------------------------------------- work --

def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["V"]
        return dict(bytes=n * SIZE[c["dtype"]] + c["rows"] * 16, flops=4 * n)
    H, KV, hd, sz = c["H"], c["KV"], c["hd"], SIZE[c["dtype"]]
    if c["kind"] == "gqa":
        ends, rows = _lengths(c), c["B"] * c["S"]
        news = np.minimum(ends, c["S"])
    else:
        ends, news = _page_lengths(c)
        rows = int(news.sum())
    # Cached rows read, new rows written, activations in and out.
    cached = 2 * KV * hd * CODE_BYTES[c["code"]] * float(ends.sum())
    moved = rows * (2 * H + 2 * KV) * hd * sz
    pairs = sum(float(n) * (e - n) + n * (n + 1) / 2 for e, n in zip(ends, news))
    return dict(bytes=cached + moved, flops=4 * H * hd * pairs)


# -------------------------------------------------------------- 64-bit arithmetic --

def _values64(u, scale, code, hd):
    """[rows, hd] float64 of one key head's stored bytes, scale [] or [hd]."""
    if code == "int8":
        x = u.to(torch.int16)
        x = torch.where(x > 127, x - 256, x).double()
    elif code == "fp8":
        b = u.to(torch.int32)
        e, f = (b >> 3) & 15, (b & 7).double()
        mag = torch.where(e > 0, (1 + f / 8) * torch.pow(2.0, (e - 7).double()), f / 512)
        x = torch.where(b > 127, -mag, mag)
    else:
        x = torch.empty(u.shape[0], hd, dtype=torch.float64, device=u.device)
        x[:, 0::2] = (u % 16).double() - 8
        x[:, 1::2] = (u // 16).double() - 8
    return x * scale


def _turn64(x, cos, sin, p0):
    """x [n, hd] at positions p0, p0 + 1, ..., halves as the parts of a complex number."""
    n, hd = x.shape
    z = torch.complex(x[:, :hd // 2], x[:, hd // 2:])
    r = z * torch.complex(cos[p0:p0 + n].double(), sin[p0:p0 + n].double())
    return torch.cat([r.real, r.imag], 1)


def _nearest64(x, scale, code):
    """The stored bytes [n, ...] of rows x [n, hd]."""
    r = x / scale
    if code == "fp8":
        grid = _values64(torch.arange(127, device=x.device, dtype=torch.uint8),
                         torch.ones((), dtype=torch.float64, device=x.device), "fp8", 0)
        a = r.abs().clamp(max=448.0)
        hi = torch.searchsorted(grid, a.contiguous()).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        below, above = a - grid[lo], grid[hi] - a
        pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
        return (pick + torch.where(torch.signbit(r), 128, 0)).to(torch.uint8)
    low, high = (-128, 127) if code == "int8" else (-8, 7)
    f = torch.floor(r)
    part = r - f
    up = (part > 0.5) | ((part == 0.5) & (torch.remainder(f, 2) == 1))
    i = torch.clamp(f + up.double(), low, high).to(torch.int64)
    if code == "int8":
        return (i % 256).to(torch.uint8)
    return ((i[:, 0::2] + 8) + 16 * (i[:, 1::2] + 8)).to(torch.uint8)


def _attend64(q, keys, vals, p0):
    """q [G, n, hd] at positions p0.., one key head: [G, n, hd]."""
    G, n, hd = q.shape
    out = torch.empty_like(q)
    step = max(1, (1 << 24) // keys.shape[0])
    for s0 in range(0, n, step):
        s1 = min(n, s0 + step)
        end = p0 + s1
        hide = torch.arange(end, device=q.device)[None, :] > \
            torch.arange(p0 + s0, p0 + s1, device=q.device)[:, None]
        for h in range(G):
            sc = (q[h, s0:s1] @ keys[:end].t()) * hd ** -0.5
            out[h, s0:s1] = torch.softmax(sc.masked_fill(hide, -math.inf), -1) @ vals[:end]
    return out


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "sample":
        return _sample64(st)
    H, KV, hd, code = c["H"], c["KV"], c["hd"], c["code"]
    G = H // KV
    if c["kind"] == "gqa":
        ends = _lengths(c)
        news = np.minimum(ends, c["S"])
        q, k, v = (st[x].double().reshape(c["B"], c["S"], -1, hd) for x in ("q", "k", "v"))
        nseq = c["B"]
    else:
        ends, news = _page_lengths(c)
        cuts = np.concatenate([[0], np.cumsum(news)]).astype(int)
        q, k, v = ([st[x][a:b].double().reshape(b - a, -1, hd) for a, b in
                    zip(cuts[:-1], cuts[1:])] for x in ("q", "k", "v"))
        nseq = c["nseq"]
    kc, vc = st["kc"].view(torch.uint8), st["vc"].view(torch.uint8)
    outs = []
    for b in range(nseq):
        e, n = int(ends[b]), int(news[b])
        p0 = e - n
        o = torch.zeros(q[b].shape, dtype=torch.float64, device="cuda")
        where = torch.arange(e, device="cuda")
        if c["kind"] == "paged":
            where = st["bt"][b].long()[where // c["blk"]] * c["blk"] + where % c["blk"]
        for h in range(KV):
            if c["kind"] == "gqa":
                kp, vp = kc[b, h], vc[b, h]
            else:
                kp, vp = (t.flatten(0, 1)[:, h] for t in (kc, vc))
            sk, sv = (s.double()[h] if c["channel"] else s.double()[0]
                      for s in (st["ks"], st["vs"]))
            kp[where[p0:]] = _nearest64(_turn64(k[b][:n, h], st["cos"], st["sin"], p0), sk, code)
            vp[where[p0:]] = _nearest64(v[b][:n, h], sv, code)
            keys = _values64(kp[where], sk, code, hd)
            vals = _values64(vp[where], sv, code, hd)
            rows = torch.stack([_turn64(q[b][:n, h * G + i], st["cos"], st["sin"], p0)
                                for i in range(G)])
            o[:n, h * G:(h + 1) * G] = _attend64(rows, keys, vals, p0).transpose(0, 1)
        outs.append(o.reshape(o.shape[0], H * hd))
    if c["kind"] == "gqa":
        return dict(out=torch.stack(outs), present_key=st["kc"], present_value=st["vc"])
    return dict(out=torch.cat(outs), key_cache=st["kc"], value_cache=st["vc"])


def _sample64(st):
    """Row by row on the host, numpy float64."""
    logits = st["logits"].float().cpu().numpy().astype(np.float64)
    uniform = st["uniform"].cpu().numpy().astype(np.float64)
    rows, V = logits.shape

    def setting(name, dtype):
        x = st[name]
        x = x.cpu().numpy() if isinstance(x, torch.Tensor) else np.full(rows, x)
        return x.astype(dtype)

    temp, top_k = setting("temperature", np.float32), setting("top_k", np.int64)
    top_p, min_p = setting("top_p", np.float32), setting("min_p", np.float32)
    ids, logprobs = np.empty(rows, np.int64), np.empty(rows)
    for r in range(rows):
        x = logits[r]
        best = int(np.argmax(x))
        if temp[r] <= 0:
            ids[r], logprobs[r] = best, 0.0
            continue
        order = np.lexsort((np.arange(V), -x))
        if 0 < top_k[r] < V:
            order = order[:top_k[r]]
        w = np.exp((x[order] - x[best]) / np.float64(temp[r]))
        if top_p[r] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            count = max(1, int(np.sum(before < np.float64(top_p[r]) * w.sum())))
            order, w = order[:count], w[:count]
        if min_p[r] > 0:
            count = max(1, int(np.sum(w >= np.float64(min_p[r]))))
            order, w = order[:count], w[:count]
        back = np.argsort(order)
        cum = np.cumsum(w[back])
        i = min(int(np.searchsorted(cum, uniform[r] * cum[-1], side="right")), len(cum) - 1)
        ids[r], logprobs[r] = order[back[i]], math.log(w[back[i]] / cum[-1])
    return dict(ids=torch.from_numpy(ids), logprobs=torch.from_numpy(logprobs))

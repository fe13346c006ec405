"""Refusals of the operators over quantised caches: on the host, before anything is
launched (no GPU needed)."""

from __future__ import annotations

import ctypes

import pytest
from conftest import load_package

P = ctypes.c_void_p(4096)
INT8, F8, INT4 = 3, 17, 22


@pytest.fixture(scope="module")
def lib():
    return load_package().load_kernels()


def gqa(lib, q=P, k=P, v=P, pk=P, pv=P, cap=64, total=10, lens=None, cos=P, sin=P, half=32,
        max_pos=64, qw=None, kw=None, ks=P, vs=P, cache=INT8, out=P, prk=P, prv=P, B=1, S=1, H=4,
        KV=2, hd=64, dtype=10, ws=P, ws_bytes=1 << 40):
    rc = lib.ortmi_group_query_attention_quantized(
        q, k, v, pk, pv, cap, total, lens, cos, sin, half, max_pos, qw, kw, 1e-6, ks, vs, 0, 0,
        cache, out, prk, prv, B, S, H, KV, hd, 0.0, 0, dtype, ws, ws_bytes, None)
    return rc, lib.ortmi_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(H=3), "num_heads"), (dict(KV=0), "num_heads"), (dict(hd=40), "head_size"),
    (dict(hd=272), "head_size"), (dict(hd=0), "head_size"), (dict(dtype=7), "dtype"),
    (dict(cache=2), "int8"), (dict(cache=10), "int8"), (dict(ks=None), "k_scale"),
    (dict(vs=None), "k_scale"), (dict(sin=None), "cos_cache"), (dict(half=33), "rotary"),
    (dict(half=0), "rotary"), (dict(max_pos=0), "rotary"), (dict(qw=P), "norm"),
    (dict(k=None), "key and value"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(prk=None), "null"), (dict(pk=None), "null past"), (dict(B=-1), "negative"),
    (dict(S=70, total=70), "capacity"), (dict(total=100, S=99), "capacity"),
    (dict(cap=1000, total=65), "cos/sin"), (dict(cap=9, total=10), "present buffers"),
    (dict(B=1 << 20, S=1 << 12, total=1 << 12, cap=1 << 13), "too many rows"),
])
def test_gqa_refusals(lib, kw, word):
    rc, msg = gqa(lib, **kw)
    assert rc == 1 and word in msg, msg


def test_gqa_empty_calls(lib):
    assert gqa(lib, B=0)[0] == 0 and gqa(lib, S=0, total=3)[0] == 0


def paged(lib, q=P, k=P, kc=P, nblk=10, blk=16, cum=P, batch=2, maxb=4, T=3, ctx=64, cos=P,
          sin=P, half=32, max_pos=64, sink=None, qw=None, kw=None, ks=P, vs=P, cache=INT8, H=4,
          KV=2, hd=64, dtype=10, ws=P, ws_bytes=1 << 40):
    rc = lib.ortmi_paged_attention_quantized(
        q, k, P, kc, P, nblk, blk, cum, P, P, batch, maxb, T, ctx, cos, sin, half, max_pos, 0,
        sink, qw, kw, 1e-6, ks, vs, 0, 0, cache, P, H, KV, hd, 0.0, dtype, ws, ws_bytes, None)
    return rc, lib.ortmi_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(H=5), "num_heads"), (dict(hd=72), "head_size"), (dict(dtype=3), "dtype"),
    (dict(cache=1), "int8"), (dict(vs=None), "k_scale"), (dict(cos=None), "cos_cache"),
    (dict(half=40), "rotary"), (dict(kw=P), "norm"), (dict(q=None), "null"),
    (dict(kc=None), "null"), (dict(cum=None), "null"), (dict(nblk=0), "batch shape"),
    (dict(blk=0), "batch shape"), (dict(batch=0), "batch shape"), (dict(maxb=0), "batch shape"),
    (dict(ctx=0), "max_context"), (dict(T=-1), "token count"), (dict(T=1 << 31), "token count"),
])
def test_paged_refusals(lib, kw, word):
    rc, msg = paged(lib, **kw)
    assert rc == 1 and word in msg, msg


def test_paged_empty_call(lib):
    assert paged(lib, T=0)[0] == 0


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "row count"), (dict(cols=0), "columns"),
    (dict(cols=(1 << 18) + 1), "columns"), (dict(x=None), "null"), (dict(u=None), "null"),
    (dict(ids=None), "null"),
])
def test_sample_refusals(lib, kw, word):
    a = dict(x=P, u=P, ids=P, rows=2, cols=100, dtype=10)
    a.update(kw)
    rc = lib.ortmi_sample_rows(a["x"], a["u"], None, None, None, None, 1.0, 0, 1.0, 0.0, a["ids"],
                               None, a["rows"], a["cols"], a["dtype"], None, 0, None)
    assert rc == 1 and word in lib.ortmi_last_error().decode()


def test_sample_empty_call(lib):
    assert lib.ortmi_sample_rows(None, None, None, None, None, None, 1.0, 0, 1.0, 0.0, None, None,
                                 0, 100, 10, None, 0, None) == 0


def test_workspace_refusals(lib):
    need = lib.ortmi_group_query_attention_quantized_workspace_size(1, 1, 4, 2, 64, 4096)
    assert need > 0
    kw = dict(cap=4096, total=4096, max_pos=4096)
    for ws, n in ((P, need - 1), (None, need)):
        rc, msg = gqa(lib, ws=ws, ws_bytes=n, **kw)
        assert rc == 3 and "workspace" in msg
    rc, msg = gqa(lib, ws=ctypes.c_void_p(4104), ws_bytes=need, **kw)
    assert rc == 1 and "aligned" in msg
    need = lib.ortmi_paged_attention_quantized_workspace_size(3, 2, 4, 2, 64, 64)
    assert need > 0
    rc, msg = paged(lib, ws_bytes=need - 1)
    assert rc == 3 and "workspace" in msg

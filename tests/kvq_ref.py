"""64-bit reference of attention over quantised key-value caches, on the CPU.

Codes: the nearest to x / scale, ties to even, clamped to the range, NaN as 0. A code c
stands for c * scale. Rows are rotated (and normalised) in 64 bits before they are
quantised; attention reads every row as the cache holds it."""

from __future__ import annotations

import math

import numpy as np
import torch

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CDT = {"int8": torch.int8, "int4": torch.uint8, "fp8": torch.float8_e4m3fn}
MAX = {"int8": 127.0, "int4": 7.0, "fp8": 448.0}
# Every finite magnitude of fp8 e4m3 by its code.
E4M3 = np.array([(m / 512 if e == 0 else (8 + m) / 8 * 2.0 ** (e - 7))
                 for e in range(16) for m in range(8)][:127])


def encode(r: torch.Tensor, code: str) -> torch.Tensor:
    """Stored bytes of r = x / scale (float64, [..., hd])."""
    a = r.numpy()
    if code == "fp8":
        mag = np.minimum(np.where(np.isnan(a), 0.0, np.abs(a)), 448.0)
        hi = np.minimum(np.searchsorted(E4M3, mag), 126)
        lo = np.maximum(hi - 1, 0)
        dl, dh = mag - E4M3[lo], E4M3[hi] - mag
        pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        sign = np.where(np.signbit(a) & ~np.isnan(a), 128, 0)
        return torch.from_numpy((pick + sign).astype(np.uint8))
    low, high = (-128, 127) if code == "int8" else (-8, 7)
    i = np.clip(np.rint(np.where(np.isnan(a), 0.0, a)), low, high).astype(np.int64)
    if code == "int8":
        return torch.from_numpy((i & 255).astype(np.uint8))
    return torch.from_numpy(((i[..., 0::2] + 8) | ((i[..., 1::2] + 8) << 4)).astype(np.uint8))


def values(u: torch.Tensor, code: str) -> torch.Tensor:
    """float64 code values of stored bytes [..., n]."""
    a = u.numpy()
    if code == "int8":
        return torch.from_numpy(a.astype(np.int8).astype(np.float64))
    if code == "int4":
        x = np.stack([a & 15, a >> 4], -1).reshape(*a.shape[:-1], -1)
        return torch.from_numpy(x.astype(np.float64) - 8)
    mag = np.concatenate([E4M3, [np.nan]])[a & 127]
    return torch.from_numpy(np.where(a & 128, -mag, mag))


def rope(x, cos, sin, pos, interleaved=False):
    """x [n, heads, hd] float64 at positions pos [n]; cos/sin [positions, half]."""
    half = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else \
        (slice(0, half), slice(half, 2 * half))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def norm(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


class Attention:
    """One call. `bound` gives how far an output may be: with Q' (the query row times the
    key scales) and P rounded to `unit` relative, and fp32 sums, a score is off by at most
    d = (unit + hd 2^-24) |scale| sum_c |q_c k_c|, so that P is off by a factor within
    1 +- 2.1 max d, and

        |out - exact| <= (2.1 max d + unit + (keys + 8) 2^-23) sum_j P_j |v_j| + u |exact|

    with u half a step of the output's type."""

    def __init__(self, dtype, code, H, KV, hd, ks, vs, scale=0.0, cos=None, sin=None,
                 interleaved=False, qw=None, kw=None, eps=1e-6, sink=None):
        self.__dict__.update(locals())
        self.sc = scale or hd ** -0.5
        self.s_k = ks.double().expand(KV, hd) if ks.numel() == 1 else ks.double().reshape(KV, hd)
        self.s_v = vs.double().expand(KV, hd) if vs.numel() == 1 else vs.double().reshape(KV, hd)
        # Half a step of the 16-bit products' type; two halves (22 bits) carry fp32.
        self.unit = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
        self.u = torch.finfo(dtype).eps / 2

    def new_codes(self, k, v, pos):
        """Stored rows [n, KV, bytes] of new rows k, v [n, KV * hd] at pos."""
        k = norm(k.double().reshape(-1, self.KV, self.hd), self.kw, self.eps)
        if self.cos is not None:
            k = rope(k, self.cos, self.sin, pos, self.interleaved)
        v = v.double().reshape(-1, self.KV, self.hd)
        return encode(k / self.s_k, self.code), encode(v / self.s_v, self.code)

    def rows(self, q, pos, kb, vb, seen):
        """q [n, H * hd] at positions pos over stored rows kb, vb [keys, KV, bytes], of which
        `seen` [keys] may be attended: (out, bound) [n, H * hd]."""
        q = norm(q.double().reshape(-1, self.H, self.hd), self.qw, self.eps)
        if self.cos is not None:
            q = rope(q, self.cos, self.sin, pos, self.interleaved)
        n, m = q.shape[0], kb.shape[0]
        K, V = values(kb, self.code) * self.s_k, values(vb, self.code) * self.s_v
        out, tol = torch.zeros_like(q), torch.zeros_like(q)
        if n == 0 or m == 0:
            return out.reshape(n, self.H * self.hd), tol.reshape(n, self.H * self.hd)
        see = (torch.arange(m)[None] <= pos[:, None]) & seen[None]
        for h in range(self.H):
            g = h * self.KV // self.H
            s = (q[:, h] @ K[:, g].t()) * self.sc
            s = torch.where(see, s, -math.inf)
            d = (q[:, h].abs() @ torch.nan_to_num(K[:, g]).abs().t()) * abs(self.sc)
            d = torch.where(see, d, 0.0).amax(1) * (self.unit + self.hd * 2.0 ** -24)
            top = s.amax(1)
            if self.sink is not None:
                top = torch.maximum(top, self.sink.double()[h])
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top)[:, None])
            p = torch.where(see, p, 0.0)
            l = p.sum(1)
            if self.sink is not None:
                l = l + torch.exp(self.sink.double()[h] - top)
            p = p / torch.where(l == 0, 1.0, l)[:, None]
            Vg = torch.where(seen[:, None], V[:, g], 0.0)
            out[:, h] = p @ Vg
            tol[:, h] = (2.1 * d + self.unit + (m + 8) * 2.0 ** -23)[:, None] * (p @ Vg.abs()) + \
                self.u * out[:, h].abs() + 1e-30
            if self.dtype == torch.float16:
                tol[:, h] += 2.0 ** -25  # half a step of its subnormals
        return out.reshape(n, -1), tol.reshape(n, -1)


def random_codes(g, shape, code):
    """Stored bytes [..., hd or hd / 2] of normal rows at 3.5 deviations' scale."""
    x = torch.randn(shape, generator=g, dtype=torch.float64) * (MAX[code] / 3.5)
    return encode(x, code)


def random_scales(g, KV, hd, code, channel):
    n = (KV, hd) if channel else (1,)
    return (0.75 + 0.5 * torch.rand(n, generator=g)) * (3.5 / MAX[code])


def rotary(g, rows, half, dtype):
    a = torch.rand((rows, half), generator=g) * 6.3
    return a.cos().to(dtype), a.sin().to(dtype)

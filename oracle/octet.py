"""The 8-bit cache, restated for the tests: quantisation, bytes, scaled rotary positions and the
attention over it, in 64 bits with plain loops and address arithmetic. Independent of the package.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

TILE, GROUP = 16, 32
LIMIT = 1.75 * 2.0 ** 127


def _power(e):
    return torch.pow(torch.tensor(2.0).double(), e.double())


def quantise(x):
    """(codes as bytes [..., d], exponent bytes [..., d / 32]) of rows x [..., d] (CPU)."""
    g = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    bad = ~torch.isfinite(g).all(-1)
    g = torch.where(bad.unsqueeze(-1), torch.zeros_like(g), g).clamp(-LIMIT, LIMIT)
    top = g.abs().amax(-1)
    m, e = torch.frexp(top)                                  # 448 = 0.875 * 2^9
    e = torch.where(m == 0, -117, e - 9 + (m > 0.875).int()).clamp(min=-117)
    y = g.abs() / _power(e).unsqueeze(-1)
    ex = (torch.frexp(y)[1] - 1).clamp(min=-6)               # the code's exponent
    n = torch.round(y / _power(ex - 3)).long()               # 0 .. 16 steps of it
    ex = torch.where(n == 16, ex + 1, ex).long()
    n = torch.where(n == 16, torch.full_like(n, 8), n)
    code = torch.where(n < 8, n, (ex + 7) * 8 + n - 8) + 128 * torch.signbit(g).long()
    code = torch.where(bad.unsqueeze(-1), torch.full_like(code, 0x7F), code)
    byte = torch.where(bad, torch.full_like(e, 127), e + 127)
    return code.reshape(x.shape).to(torch.uint8), byte.to(torch.uint8)


def code_values(c):
    """e4m3 bytes as float64."""
    c = c.long()
    s, e, m = 1 - 2 * (c // 128).double(), c % 128 // 8, (c % 8).double()
    v = s * torch.where(e == 0, m / 512, (1 + m / 8) * _power(e - 7))
    return torch.where(c % 128 == 127, torch.full_like(v, math.nan), v)


def combine(code, byte):
    v = code_values(code).reshape(*byte.shape, GROUP) * _power(byte.long() - 127).unsqueeze(-1)
    return v.reshape(code.shape)


def values(x):
    """What rows x [..., d] stand for once they are stored (float64)."""
    return combine(*quantise(x))


def key_place(d, u, x):
    q, p = x // (d // 4), x % (d // 4) // 16
    return ((p * 4 + q) * 16 + u) * 16 + x % 16


def value_place(d, u, x):
    n, e, N = x // (d // 16), x % (d // 16), d // 16
    b = N * (u % 4) + e
    return 16 * d + (b // 16 * 64 + 16 * (u // 4) + n) * 16 + b % 16


def key_byte(d, u, g):
    P = max(1, d // 128)
    return 32 * d + (g // P * 16 + u) * P + g % P


def value_byte(d, u, g):
    return 32 * d + d // 2 + g * 16 + u


def _base(slot, h, stride, d):
    return slot // TILE * TILE * stride + h * 33 * d


def put(page, stride, slots, kq, vq):
    """Store (codes, bytes) of keys and values [N, H, d] into the flat uint8 page (CPU, in place)."""
    N, H, d = kq[0].shape
    for i, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        u = slot % TILE
        for h in range(H):
            base = _base(slot, h, stride, d)
            for (c, p), place, at in ((kq, key_place, key_byte), (vq, value_place, value_byte)):
                for x in range(d):
                    page[base + place(d, u, x)] = c[i, h, x]
                for g in range(d // GROUP):
                    page[base + at(d, u, g)] = p[i, h, g]


def write(page, stride, slots, key, value):
    put(page, stride, slots, quantise(key), quantise(value))


_PLACES = {}


def places(d):
    """[16, d] bytes of keys', values' codes and [16, d / 32] of their exponents in a record."""
    if d not in _PLACES:
        _PLACES[d] = [torch.tensor([[f(d, u, x) for x in range(m)] for u in range(TILE)])
                      for f, m in ((key_place, d), (key_byte, d // GROUP), (value_place, d),
                                   (value_byte, d // GROUP))]
    return _PLACES[d]


def fields(page, stride, slots, H, d):
    """((codes, bytes) of keys, of values) [n, H, ...] of slots of the uint8 page."""
    page, slots = page.cpu().reshape(-1), slots.long().cpu()
    base = (slots // TILE * TILE * stride)[:, None] + torch.arange(H) * 33 * d
    got = [page[base[..., None] + t[slots % TILE][:, None]] for t in places(d)]
    return (got[0], got[1]), (got[2], got[3])


def read(page, stride, slots, H, d):
    """K and V [n, H, d] float64 of slots of the uint8 page."""
    k, v = fields(page, stride, slots, H, d)
    return combine(*k), combine(*v)


def turn(x, positions, turns, amplitude=1.0, adjacent=False):
    """x [N, heads, d] rotated, each angle reduced in exact arithmetic, the rest in 64 bits."""
    half = len(turns)
    rev = [Fraction(float(t)) for t in turns]
    y = x.double().clone()
    for i, p in enumerate(positions.tolist()):
        for j in range(half):
            a = 2 * math.pi * float((p * rev[j]) % 1)
            c, s = amplitude * math.cos(a), amplitude * math.sin(a)
            u, v = (2 * j, 2 * j + 1) if adjacent else (j, j + half)
            xu, xv = x[i, :, u].double(), x[i, :, v].double()
            y[i, :, u], y[i, :, v] = xu * c - xv * s, xv * c + xu * s
    return y


def attend(q, K, V, scale, window=0, sinks=None):
    """Causal attention of q [Q, HQ, d] at the end of K, V [n, H, d], in 64 bits: (out, lse, spread,
    score): spread = sum p |v|, what a relative error of every softmax weight can move an output by;
    score = the largest sum |q k| * scale of a row, what products in 32 bits round."""
    q = q.double().cpu()
    Q, HQ, d = q.shape
    n, H, _ = K.shape
    G = HQ // H
    out, spread = torch.zeros(2, Q, HQ, d).double()
    lse, score = torch.full((Q, HQ), -math.inf).double(), torch.zeros(Q, HQ, 1).double()
    t = torch.arange(n)
    for p in range(HQ):
        for j in range(Q):
            at = n - Q + j
            seen = (t <= at) & (t > at - window if window else t >= 0)
            k, v = K[seen, p // G], V[seen, p // G]
            s = k @ q[j, p] * scale
            if sinks is not None:
                s = torch.cat([s, sinks[p].double().cpu().reshape(1)])
            if s.numel() == 0:
                continue
            lse[j, p] = torch.logsumexp(s, 0)
            w = torch.exp(s - lse[j, p])[:k.shape[0]]
            out[j, p], spread[j, p] = w @ v, w @ v.abs()
            if k.shape[0]:
                score[j, p] = (k.abs() @ q[j, p].abs()).amax() * abs(scale)
    return out, lse, spread, score

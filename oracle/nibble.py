"""The 4-bit cache, restated for the tests: quantisation, bytes, a step's plan, rotary axes and the
attention over it, in 64 bits with plain loops and address arithmetic. Independent of the package.
"""
from __future__ import annotations

import torch

TILE, GROUP, D = 16, 32, 128
RECORD, VCODES, KPAR, VPAR = 2304, 1024, 2048, 2176
LIMIT, MIN_SCALE = 32640.0, 2.0 ** -14


def quantise(x):
    """(codes, zero codes, scales, parameters) of rows x [..., 128]: codes [..., 4, 32] int64, the
    rest [..., 4]. A group with a value that is not finite has scale NaN and parameter 0x7e00."""
    x = x.double().reshape(*x.shape[:-1], D // GROUP, GROUP)
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad.unsqueeze(-1), torch.zeros_like(x), x).clamp(-LIMIT, LIMIT)
    lo, hi = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
    m, e = torch.frexp(((hi - lo) / 15).cpu())
    s = (torch.ceil(m * 128) * torch.pow(torch.tensor(2.0).double(), (e - 7).double())).to(x.device)
    s = s.clamp(min=MIN_SCALE)
    z = torch.round(-lo / s).clamp(0, 15)
    c = (torch.round(x / s.unsqueeze(-1)) + z.unsqueeze(-1)).clamp(0, 15)
    par = s.half().view(torch.int16).long() + z.long()
    par = torch.where(bad, torch.full_like(par, 0x7E00), par)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    return c.long(), z.long(), s, par


def values(x):
    """What rows x [..., 128] stand for once they are stored (float64)."""
    c, z, s, _ = quantise(x)
    return ((c - z.unsqueeze(-1)) * s.unsqueeze(-1)).reshape(x.shape)


def key_place(u, x):
    """(byte, shift) of token u's key code of dim x within a record."""
    g, qd, j = x // 32, (x % 32) // 8, x % 8
    bit = 32 * ((qd * 16 + u) * 4 + g) + 4 * (j // 2) + 16 * (j % 2)
    return bit // 8, bit % 8


def value_place(u, x):
    g, n, b = x // 32, (x % 32) // 2, x % 2
    dword = ((u // 4 * 16 + n) * 2 + u % 4 // 2) * 2 + g // 2
    bit = 32 * dword + 16 * (u % 2) + 4 * (2 * (g % 2) + b)
    return VCODES + bit // 8, bit % 8


def key_par(u, g):
    return KPAR + 2 * (u * 4 + g)


def value_par(u, g):
    return VPAR + 2 * ((u // 4 * 4 + g) * 4 + u % 4)


def _base(slot, h, stride):
    return slot // TILE * TILE * stride + h * RECORD


def write(page, stride, slots, key, value):
    """Store rows key / value [N, H, 128] into the flat uint8 page (CPU, in place)."""
    kq, vq = quantise(key), quantise(value)
    for i, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        u = slot % TILE
        for h in range(key.shape[1]):
            base = _base(slot, h, stride)
            for (c, _, _, par), place, at in ((kq, key_place, key_par),
                                              (vq, value_place, value_par)):
                row, pr = c[i, h].reshape(-1).tolist(), par[i, h].tolist()
                for x in range(D):
                    byte, shift = place(u, x)
                    old = int(page[base + byte])
                    page[base + byte] = (old & ~(15 << shift) & 255) | (row[x] << shift)
                for g in range(4):
                    page[base + at(u, g)] = pr[g] & 255
                    page[base + at(u, g) + 1] = pr[g] >> 8


_PLACES = {}


def _places():
    if not _PLACES:
        for name, place, par in (("k", key_place, key_par), ("v", value_place, value_par)):
            b = torch.tensor([[place(u, x) for x in range(D)] for u in range(TILE)])
            p = torch.tensor([[par(u, x // 32) for x in range(D)] for u in range(TILE)])
            _PLACES[name] = (b[..., 0], b[..., 1], p)
    return _PLACES


def read(page, stride, slots, H):
    """K and V [n, H, 128] float64 of slots of the flat uint8 page."""
    slots = slots.long().cpu()
    base = slots // TILE * TILE * stride
    out = []
    for name in ("k", "v"):
        byte, shift, par = (t[slots % TILE] for t in _places()[name])       # [n, 128]
        rows = []
        for h in range(H):
            at = (base + h * RECORD).unsqueeze(1)
            b = page[(at + byte).to(page.device)].cpu().long()
            p = (page[(at + par).to(page.device)].cpu().long()
                 + 256 * page[(at + par + 1).to(page.device)].cpu().long())
            code, zero = (b >> shift) & 15, p & 15
            s = (p - zero).to(torch.int16).view(torch.float16).double()
            rows.append((code - zero) * s)
        out.append(torch.stack(rows, 1))
    return out


def table_slots(row, n, block_size):
    t = torch.arange(n)
    return row.cpu().long()[t // block_size] * block_size + t % block_size


def attend(q, K, V, scale):
    """Causal attention of q [Q, HQ, 128] at the end of K, V [n, H, 128], in 64 bits:
    (out, spread, score): spread = sum p |v|, what a relative error of every softmax weight can move
    an output by; score = the largest sum |q k| * scale of a row, what products in 32 bits round."""
    q = q.double().cpu()
    Q, HQ, _ = q.shape
    n, H, _ = K.shape
    G = HQ // H
    out, spread = torch.zeros(Q, HQ, D).double(), torch.zeros(Q, HQ, D).double()
    score = torch.zeros(Q, HQ, 1).double()
    if n == 0:
        return out, spread, score
    for p in range(HQ):
        k, v = K[:, p // G], V[:, p // G]
        s = q[:, p] @ k.t() * scale
        seen = torch.arange(n)[None, :] <= n - Q + torch.arange(Q)[:, None]
        w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        out[:, p], spread[:, p] = w @ v, w @ v.abs()
        score[:, p, 0] = (q[:, p].abs() @ k.abs().t() * abs(scale)).amax(-1)
    return out, spread, score


def rotary(x, positions, cos_sin, sections, interleaved):
    """x [N, heads, d] rotated, in 64 bits; positions [axes, N]."""
    half = sum(sections)
    y = x.double().clone()
    ends = [sum(sections[:i + 1]) for i in range(len(sections))]
    for j in range(half):
        if interleaved:
            a = j % len(sections)
            a = a if j < len(sections) * sections[a] else 0
        else:
            a = next(i for i, e in enumerate(ends) if j < e)
        c = cos_sin[positions[a], j].double().unsqueeze(1)
        s = cos_sin[positions[a], j + half].double().unsqueeze(1)
        u, v = x[:, :, j].double(), x[:, :, j + half].double()
        y[:, :, j], y[:, :, j + half] = u * c - v * s, v * c + u * s
    return y


def plan(computed, counts, table, free, block_size, num_blocks, num_tokens):
    """A step's plan by plain loops: (query_start_loc, seq_lens, slots, positions, used, table)."""
    table, free = [list(r) for r in table], list(free)
    width = len(table[0]) if table else 0
    qsl, seq, slots, pos, taken = [0], [], [], [], 0
    for r, (c, n) in enumerate(zip(computed, counts)):
        for b in range(-(-c // block_size), min(-(-(c + n) // block_size), width)):
            table[r][b] = free[taken] if taken < len(free) else -1
            taken += 1
        qsl.append(min(qsl[-1] + n, num_tokens))
        seq.append(c + n)
        for p in range(c, c + n):
            b = p // block_size
            blk = table[r][b] if b < width else -1
            pos.append(p)
            slots.append(blk * block_size + p % block_size if 0 <= blk < num_blocks else -1)
    slots, pos = slots[:num_tokens], pos[:num_tokens]
    fill = num_tokens - len(slots)
    return qsl, seq, slots + [-1] * fill, pos + [0] * fill, min(taken, len(free)), table

"""Performance cases of the 8-bit cache: rotary positions scaled for long contexts, the cache's
write, its read back and the attention of new tokens over it, one attention layer per pass.

  rotary  `kernels.rotary_scaled`: queries and keys rotated, pairs by halves or adjacent, the angles
          formed from frequencies in 64 bits
  write   `kernels.octet_write_paged`: new keys and values quantised into their slots, the keys
          (and queries) rotated on the way where the case has rotary dims
  read    `kernels.octet_read_paged`: stored keys and values back as 16-bit rows
  decode  `kernels.octet_decode_paged`: one query per running request, or a few drafts, over its
          store, all of it or a window, with attention sinks

`listed()` gives the fixed cases, `draw(rng)` more of the same ranges. A case is a dict of plain
values; `prepare` makes its inputs on the GPU from a seed, `run` is one pass: the package's own
operators where `own` is true, else the same results in plain torch. `exact` gives them in 64 bits,
written apart from both.

The cache holds e4m3 codes with one power of two per group of 32 dims. Of a group x:
  2^e the smallest power of two with max |x| <= 448 * 2^e, e >= -117;  code = e4m3(x / 2^e)
stored as the byte e + 127. Sixteen slots of a block make a tile; a tile holds one record of 33 d
bytes per KV head, with P = max(1, d / 128) and N = d / 16:
  0       key codes, token u, dim x at ((p * 4 + q) * 16 + u) * 16 + x % 16, where
          q = x / (d / 4), p = x % (d / 4) / 16
  16 d    value codes, token u = 4 q + i, dim x = N n + e: with b = N i + e,
          (b / 16 * 64 + q * 16 + n) * 16 + b % 16
  32 d    key exponents, group g of token u at (g / P * 16 + u) * P + g % P
  32.5 d  value exponents, g * 16 + u
"""
import math
import random
import sys
from types import SimpleNamespace

import torch

own = False

POOL_TILES = 96             # distinct tiles a store is filled from
WORKSPACE = 64 << 20        # the buffer a server keeps for its reads
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step's queries and keys, all latency
        dict(name="rotary 8", kind="rotary", tokens=8, heads=32, kv=8, d=128, rot=128,
             adjacent=False, scaled="llama3", far=16000, dtype="fp16", lens=1),
        # a long prompt in a far context, adjacent pairs in half of each head
        dict(name="rotary 8192 adjacent", kind="rotary", tokens=8192, heads=32, kv=8, d=128,
             rot=64, adjacent=True, scaled="yarn", far=1000000, dtype="bf16", lens=2),
        # one new token of each of eight requests, rotated on the way with its queries
        dict(name="write 8x1 rotated", kind="write", heads=32, kv=8, d=128, rot=128,
             adjacent=False, scaled="llama3", dtype="bf16", block=16, batch=8, lo=1, hi=1,
             keep=False, lens=3),
        # a chunk of a long prompt whose keys come rotated; the prompt attends to what is stored
        dict(name="write 1x2048", kind="write", heads=0, kv=8, d=128, rot=0, adjacent=False,
             scaled="none", dtype="bf16", block=16, batch=1, lo=2048, hi=2048, keep=True, lens=4),
        # several prompts of wide heads, ragged and off the tiles' borders, rotated on the way
        dict(name="write 5 wide", kind="write", heads=16, kv=4, d=256, rot=64, adjacent=True,
             scaled="linear", dtype="fp16", block=32, batch=5, lo=150, hi=1100, keep=False,
             lens=5),
        # a short prefix handed to another worker
        dict(name="read 1x700", kind="read", kv=8, d=128, dtype="bf16", block=16, batch=1,
             lo=700, hi=700, lens=6),
        # the stored part of four prompts, for the dense attention of their next chunks
        dict(name="read 4x7656", kind="read", kv=8, d=128, dtype="fp16", block=16, batch=4,
             lo=7656, hi=7656, lens=7),
        # one user, a short context: the smallest attention, all latency
        dict(name="decode 1x1082", kind="decode", heads=32, kv=8, d=128, dtype="bf16", block=16,
             batch=1, lo=1082, hi=1082, queries=1, window=0, sinks=False, lse=False, lens=8),
        # eight long conversations of the same length: the largest
        dict(name="decode 8x14402", kind="decode", heads=32, kv=8, d=128, dtype="fp16", block=16,
             batch=8, lo=14402, hi=14402, queries=1, window=0, sinks=False, lse=False, lens=9),
        # a full server of short conversations
        dict(name="decode 61 short", kind="decode", heads=32, kv=8, d=128, dtype="bf16", block=32,
             batch=61, lo=70, hi=2900, queries=1, window=0, sinks=False, lse=False, lens=10),
        # small heads with a sliding window and sinks, eight query heads per KV head
        dict(name="decode 24 windowed", kind="decode", heads=64, kv=8, d=64, dtype="bf16",
             block=16, batch=24, lo=200, hi=20000, queries=1, window=1024, sinks=True, lse=True,
             lens=11),
        # drafts of five tokens to verify, wide heads: twenty rows per KV head
        dict(name="decode 6x5 drafts", kind="decode", heads=16, kv=4, d=256, dtype="bf16",
             block=64, batch=6, lo=900, hi=9000, queries=5, window=0, sinks=False, lse=False,
             lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "write", "write", "read", "decode", "decode", "decode"])
    d = rng.choice([64, 128, 128, 128, 256])
    c = dict(kind=kind, lens=rng.randint(1, 10 ** 6), d=d, kv=rng.choice([8, 8, 4, 2, 1, 5]),
             dtype=rng.choice(["fp16", "bf16"]))
    if kind in ("rotary", "write"):
        c.update(adjacent=rng.random() < 0.5, far=_log(rng, 100, 1000000),
                 scaled=rng.choice(["none", "linear", "llama3", "yarn"]),
                 rot=rng.choice([d, d, d // 2, d // 4, 3 * d // 4, 2 * rng.randint(1, d // 2)]))
    if kind != "rotary":
        c["block"] = rng.choice([16, 16, 32, 48, 64])
    c["heads"] = c["kv"] * rng.choice([1, 2, 3, 4, 4, 7, 8])
    if kind == "rotary":
        c["tokens"] = _log(rng, 1, 8192 * 40 * 128 // (max(40, c["heads"] + c["kv"]) * d))
    elif kind == "write":
        c.pop("far")
        if rng.random() < 0.4:
            c.update(rot=0, adjacent=False, scaled="none", heads=0)
        c["batch"] = _log(rng, 1, 32)
        most = 2048 * 1024 // (c["kv"] * d * c["batch"])
        c["lo"] = _log(rng, 1, min(most, 4096))
        c["hi"] = rng.choice([c["lo"], rng.randint(c["lo"], min(most, 4096))])
        c["keep"] = rng.random() < 0.5
    elif kind == "read":
        c.pop("heads")
        c["batch"] = _log(rng, 1, 32)
        c["lo"] = _log(rng, 1, min(16000, 30000 * 1024 // (c["kv"] * d * c["batch"])))
        c["hi"] = rng.choice([c["lo"], rng.randint(1, c["lo"])])
        c["lo"], c["hi"] = min(c["lo"], c["hi"]), max(c["lo"], c["hi"])
    else:
        c["batch"], c["queries"] = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, 8])
        rows = c["queries"] * c["heads"] // c["kv"]     # (many of them cost more than the bytes)
        most = min(60000, 110000 * 1024 // (c["kv"] * d * c["batch"] * max(1, rows // 20)))
        c["lo"] = max(c["queries"], _log(rng, 1, most))
        c["hi"] = rng.choice([c["lo"], rng.randint(c["lo"], max(most, c["lo"]))])
        c["window"] = rng.choice([0, 0, _log(rng, 1, 4096)])
        c["sinks"], c["lse"] = rng.random() < 0.4, rng.random() < 0.4
    return c


# ------------------------------------------------------------------------------------ inputs
def _gen(seed, dev="cuda"):
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    return g


def _lens(case, lo, hi, salt=0):
    r = random.Random(case["lens"] * 7 + salt)
    return [r.randint(lo, hi) for _ in range(case["batch"])]


def _i32(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return _i32(at)


def _tokens(n, H, d, g):
    """Keys with eight channels of every head that are larger than the others, and values."""
    k = torch.randn(n, H, d, generator=g, device="cuda")
    k[..., :8] *= 8
    return k, torch.randn(n, H, d, generator=g, device="cuda")


def _tables(lens, block, seed):
    """A block table over a shuffled cache and the cache's block count."""
    need = [-(-n // block) for n in lens]
    total = sum(need) + 4
    perm = torch.randperm(total, generator=_gen(seed, "cpu")).to(torch.int32)
    bt = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for r, k in enumerate(need):
        bt[r, :k] = perm[at:at + k]
        at += k
    return bt.cuda(), total


def _frequencies(rot, scaled):
    """(turns per position of each pair, in 64 bits; factor of the rotated rows)."""
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    theta, amplitude = 500000.0, 1.0
    w = theta ** (-i / rot)
    if scaled == "linear":
        w = w / 4
    elif scaled == "llama3":
        turns = 8192 * w / (2 * math.pi)            # in the context it was trained on
        t = ((turns - 1) / (4 - 1)).clamp(0, 1)
        w = w / 32 * (1 - t) + w * t
    elif scaled == "yarn":
        edge = [rot * math.log(8192 / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32, 1)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
        t = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        w = w / 16 * t + w * (1 - t)
        amplitude = 0.1 * math.log(16) + 1
    return (w / (2 * math.pi)).cuda(), amplitude


def prepare(case, seed):
    s = globals()["_prepare_" + case["kind"]](case, seed)
    s.case = case
    s.err = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


def _prepare_rotary(case, seed):
    g = _gen(seed)
    dt, n = DTYPES[case["dtype"]], case["tokens"]
    turns, amplitude = _frequencies(case["rot"], case["scaled"])
    q = torch.randn(n, case["heads"], case["d"], generator=g, device="cuda").to(dt)
    k = _tokens(n, case["kv"], case["d"], g)[0].to(dt)
    # a few requests' tokens, each in a row from where its context stands
    at = torch.randint(case["far"], (-(-n // 64),), generator=g, device="cuda")
    pos = (at[:, None] + torch.arange(64, device="cuda")).reshape(-1)[:n].contiguous()
    return SimpleNamespace(q=q, k=k, pos=pos, turns=turns, amplitude=amplitude,
                           q_out=torch.empty_like(q), k_out=torch.empty_like(k))


def _prepare_write(case, seed):
    g, H, d, block = _gen(seed), case["kv"], case["d"], case["block"]
    counts = _lens(case, case["lo"], case["hi"])
    before = _lens(case, 0, 700, salt=1)
    bt, blocks = _tables([b + n for b, n in zip(before, counts)], block, seed)
    p = [torch.arange(b, b + n, device="cuda") for b, n in zip(before, counts)]
    slots = torch.cat([bt[r].long()[i // block] * block + i % block for r, i in enumerate(p)])
    dt = DTYPES[case["dtype"]]
    k, v = (x.to(dt) for x in _tokens(sum(counts), H, d, g))
    s = SimpleNamespace(k=k, v=v, slots=slots, pos=torch.cat(p), q=None, q_out=None, k_out=None,
                        v_out=None, page=torch.zeros(blocks, block, H * 33 * d // 16,
                                                     dtype=torch.uint8, device="cuda"))
    if case["rot"]:
        s.turns, s.amplitude = _frequencies(case["rot"], case["scaled"])
        s.q = torch.randn(sum(counts), case["heads"], d, generator=g, device="cuda").to(dt)
        s.q_out = torch.empty_like(s.q)
    if case["keep"]:
        s.k_out = torch.empty(k.shape, dtype=torch.bfloat16, device="cuda")
        s.v_out = torch.empty_like(s.k_out)
    return s


def _store(case, seed, lens):
    """A paged store of requests of `lens` tokens: distinct tiles, dealt out by chance."""
    g, H, d, block = _gen(seed), case["kv"], case["d"], case["block"]
    bt, blocks = _tables(lens, block, seed)
    tiles = min(POOL_TILES, max(1, sum(lens) // 16))
    k, v = _tokens(tiles * 16, H, d, g)
    pool = torch.zeros(tiles, H, 33 * d, dtype=torch.uint8, device="cuda")
    _put(pool, torch.arange(tiles * 16, device="cuda"), *_quantise(k), *_quantise(v))
    pick = torch.randint(tiles, (blocks * block // 16,), generator=g, device="cuda")
    page = pool[pick].reshape(blocks, block, H * 33 * d // 16)
    return g, page, bt


def _prepare_read(case, seed):
    lens = _lens(case, case["lo"], case["hi"])
    _, page, bt = _store(case, seed, lens)
    k = torch.empty(sum(lens), case["kv"], case["d"], dtype=DTYPES[case["dtype"]], device="cuda")
    return SimpleNamespace(page=page, bt=bt, starts=_starts(lens), longest=max(lens), k_out=k,
                           v_out=torch.empty_like(k))


def _prepare_decode(case, seed):
    lens, Q = _lens(case, case["lo"], case["hi"]), case["queries"]
    g, page, bt = _store(case, seed, lens)
    q = torch.randn(len(lens) * Q, case["heads"], case["d"], generator=g, device="cuda")
    q = q.to(DTYPES[case["dtype"]])
    sinks = torch.randn(case["heads"], generator=g, device="cuda") if case["sinks"] else None
    lse = torch.empty(q.shape[:2], device="cuda") if case["lse"] else None
    return SimpleNamespace(page=page, bt=bt, seq=_i32(lens), qsl=_starts([Q] * len(lens)), q=q,
                           longest=max(lens), sinks=sinks, out=torch.empty_like(q), lse=lse,
                           ws=torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda"))


# ------------------------------------------------------------------------------------ passes
def run(state):
    return globals()[("_own_" if own else "_plain_") + state.case["kind"]](state)


def _kernels():
    if "ttkv-vllm_amd" not in sys.path:
        sys.path.insert(0, "ttkv-vllm_amd")
    from vllm_ttkv import kernels
    return kernels


def _layout(s):
    lay = getattr(s, "lay", None)
    if lay is None:
        _kernels()
        from vllm_ttkv.octet import OctetLayout
        lay = s.lay = OctetLayout(H=s.case["kv"], d=s.case["d"])
    return lay


def _rotary(s):
    rotary = getattr(s, "rotary", None)
    if rotary is None:
        _kernels()
        from vllm_ttkv.rope import Rotary
        rotary = s.rotary = Rotary(s.turns, amplitude=s.amplitude, adjacent=s.case["adjacent"])
    return rotary


def _own_rotary(s):
    return list(_kernels().rotary_scaled(s.q, s.k, s.pos, _rotary(s), query_out=s.q_out,
                                         key_out=s.k_out, error_word=s.err))


def _own_write(s):
    kw = {}
    if s.q is not None:
        kw = dict(rotary=_rotary(s), positions=s.pos, query=s.q, query_out=s.q_out)
    _kernels().octet_write_paged(_layout(s), s.k, s.v, s.slots, s.page, key_out=s.k_out,
                                 value_out=s.v_out, error_word=s.err, **kw)
    return _stored(s)


def _own_read(s):
    return list(_kernels().octet_read_paged(_layout(s), s.page, s.case["block"], s.bt, s.starts,
                                            s.longest, key_out=s.k_out, value_out=s.v_out,
                                            error_word=s.err))


def _own_decode(s):
    out = _kernels().octet_decode_paged(
        _layout(s), s.q, s.page, s.case["block"], s.bt, s.seq, s.qsl, s.case["queries"], s.longest,
        s.case["d"] ** -0.5, window=s.case["window"], sinks=s.sinks, out=s.out, lse=s.lse,
        workspace=s.ws, error_word=s.err)
    return [out, s.lse]


def _stored(s):
    """What a write leaves: the cache's codes and powers of two, the queries, the stored values."""
    H, d = s.case["kv"], s.case["d"]
    rec = s.page.reshape(-1, H, 33 * d)
    return dict(codes=rec[..., :32 * d].view(torch.float8_e4m3fn),
                powers=rec[..., 32 * d:].view(torch.float8_e8m0fnu), query=s.q_out, key=s.k_out,
                value=s.v_out)


# ------------------------------------------------------------------------------- plain forms
def _places(d, dev="cuda"):
    """Bytes within a record of [token, dim] codes and of [token, group] powers, keys and values."""
    u, x = torch.arange(16, device=dev)[:, None], torch.arange(d, device=dev)[None, :]
    k = ((x % (d // 4) // 16 * 4 + x // (d // 4)) * 16 + u) * 16 + x % 16
    b = u % 4 * (d // 16) + x % (d // 16)
    v = 16 * d + (b // 16 * 64 + u // 4 * 16 + x // (d // 16)) * 16 + b % 16
    P, g = max(1, d // 128), x[:, :d // 32]
    return k, v, 32 * d + (g // P * 16 + u) * P + g % P, 32 * d + d // 2 + g * 16 + u


def _two(byte):
    """2^(byte - 127) as fp32, from its bits (exp2 and pow are off by a bit at some powers)."""
    return (byte.int() << 23).view(torch.float32)


def _quantise(x):
    """Codes [..., d] as bytes, and the bytes of their groups' powers of two, of x [..., d]."""
    t = x.double().reshape(*x.shape[:-1], -1, 32)
    m, e = torch.frexp(t.abs().amax(-1))            # 448 = 0.875 * 2^9
    byte = torch.where(m == 0, 0, e + 127 - 9 + (m > 0.875)).clamp(min=127 - 117)
    code = (t * _two(254 - byte)[..., None]).float().to(torch.float8_e4m3fn)
    return code.view(torch.uint8).reshape(x.shape), byte.to(torch.uint8)


def _values(code, power):
    """fp32 values of bytes."""
    t = code.view(torch.float8_e4m3fn).float().reshape(*power.shape, 32)
    return (t * _two(power)[..., None]).reshape(code.shape)


def _put(rec, slots, kc, kp, vc, vp):
    """Writes rows of codes and powers into the records rec [tiles, H, 33 d] of their slots."""
    H, d = kc.shape[1:]
    head = torch.arange(H, device=slots.device)[None, :, None]
    tile, u = (slots // 16)[:, None, None], slots % 16
    for row, at in zip((kc, vc, kp, vp), _places(d)):
        rec[tile, head, at[u][:, None, :]] = row


def _turned(x, pos, turns, amplitude, adjacent):
    """x [N, heads, d] rotated in 64 bits (a quantised value can lie next to a border)."""
    half = turns.numel()
    angle = torch.remainder(pos.double()[:, None] * turns, 1.0) * (2 * math.pi)
    c, s = (angle.cos() * amplitude)[:, None], (angle.sin() * amplitude)[:, None]
    y = x.double()
    a, b = (y[..., :2 * half:2], y[..., 1:2 * half:2]) if adjacent else \
        (y[..., :half], y[..., half:2 * half])
    u, v = a * c - b * s, b * c + a * s
    turned = torch.stack([u, v], -1).flatten(-2) if adjacent else torch.cat([u, v], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1)


def _plain_rotary(s):
    return [_turned(x, s.pos, s.turns, s.amplitude, s.case["adjacent"]).to(x.dtype)
            for x in (s.q, s.k)]


def _plain_write(s):
    H, d = s.case["kv"], s.case["d"]
    k = s.k
    if s.q is not None:
        k = _turned(k, s.pos, s.turns, s.amplitude, s.case["adjacent"])
        s.q_out = _turned(s.q, s.pos, s.turns, s.amplitude, s.case["adjacent"]).to(s.q.dtype)
    kc, kp = _quantise(k)
    vc, vp = _quantise(s.v)
    _put(s.page.view(-1, H, 33 * d), s.slots, kc, kp, vc, vp)
    if s.k_out is not None:
        s.k_out, s.v_out = _values(kc, kp).bfloat16(), _values(vc, vp).bfloat16()
    return _stored(s)


def _dense(s, longest):
    """The store's keys and values as fp32 [B, H, longest rounded up to tiles, d]."""
    H, d, block = s.case["kv"], s.case["d"], s.case["block"]
    ids = s.bt[:, :-(-longest // block)].long().clamp(min=0)
    rec = s.page[ids].reshape(ids.shape[0], -1, H, 33 * d)
    k, v, kp, vp = (rec[..., at].permute(0, 2, 1, 3, 4).flatten(2, 3) for at in _places(d))
    return _values(k, kp), _values(v, vp)


def _plain_read(s):
    k, v = _dense(s, s.longest)
    n = (s.starts[1:] - s.starts[:-1])[:, None]
    there = torch.arange(k.shape[2], device="cuda")[None, :] < n
    return [x.transpose(1, 2)[there].to(s.k_out.dtype) for x in (k, v)]


def _plain_decode(s):
    H, d, Q, HQ = s.case["kv"], s.case["d"], s.case["queries"], s.case["heads"]
    B, G = s.seq.numel(), HQ // H
    k, v = _dense(s, s.longest)
    q = s.q.float().reshape(B, Q, H, G, d).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, d)
    w = torch.matmul(q, k.transpose(2, 3).contiguous()) * d ** -0.5
    at = (s.seq[:, None] - Q + torch.arange(Q, device="cuda")).repeat_interleave(G, 1)
    t = torch.arange(k.shape[2], device="cuda")
    hidden = t > at[..., None]
    if s.case["window"]:
        hidden |= t <= at[..., None] - s.case["window"]
    w = w.masked_fill(hidden[:, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    if s.sinks is not None:
        sink = s.sinks.reshape(H, 1, G).repeat(1, Q, 1).reshape(1, H, Q * G, 1)
        top = torch.maximum(top, sink)
    w = torch.exp(w - top)
    total = w.sum(-1, keepdim=True)
    if s.sinks is not None:
        total = total + torch.exp(sink - top)
    o = torch.matmul(w, v) / total
    o = o.reshape(B, H, Q, G, d).permute(0, 2, 1, 3, 4).reshape(s.q.shape).to(s.q.dtype)
    lse = (top + total.log()).reshape(B, H, Q, G).permute(0, 2, 1, 3).reshape(B * Q, HQ)
    return [o, lse if s.case["lse"] else None]


# -------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    return globals()["_exact_" + case["kind"]](case, prepare(case, seed))


def _exact_turn(x, pos, s, adjacent):
    """Every pair as a complex number, turned by its angle."""
    half = s.turns.numel()
    t = pos.double()[:, None] * s.turns
    angle = 2 * math.pi * (t - t.floor())
    w = torch.polar(torch.full_like(angle, s.amplitude), angle)[:, None, :]
    y = x.double().clone()
    first = torch.arange(half, device="cuda") * (2 if adjacent else 1)
    second = first + (1 if adjacent else half)
    z = torch.complex(y[..., first], y[..., second]) * w
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rotary(case, s):
    return [_exact_turn(x, s.pos, s, case["adjacent"]) for x in (s.q, s.k)]


def _exact_power(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_codes(x):
    """(code values, powers of two) of x in 64 bits, by the grid of each value's own exponent."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1)
    e = torch.where(top == 0, -117, torch.frexp(top)[1] - 9).clamp(min=-117)
    e = e + (top > 448 * _exact_power(e)).int()
    y = g / _exact_power(e)[..., None]
    step = _exact_power((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).reshape(x.shape), _exact_power(e)


def _exact_write(case, s):
    H, d = case["kv"], case["d"]
    N, P = d // 16, max(1, d // 128)
    k = _exact_turn(s.k, s.pos, s, case["adjacent"]) if case["rot"] else s.k
    q = _exact_turn(s.q, s.pos, s, case["adjacent"]) if case["rot"] else None
    (kc, kp), (vc, vp) = _exact_codes(k), _exact_codes(s.v)
    rows = s.page.numel() // (33 * H * d // 16)
    kall, vall = torch.zeros(2, rows, H, d, dtype=torch.float64, device="cuda")
    kall[s.slots], vall[s.slots] = kc, vc
    powers = torch.full((2, rows, H, d // 32), 2.0 ** -127, dtype=torch.float64, device="cuda")
    powers[0, s.slots], powers[1, s.slots] = kp, vp
    # [tile, token, head, dims] to the record's order
    kall = kall.reshape(-1, 16, H, 4, d // 64, 16).permute(0, 2, 4, 3, 1, 5)
    vall = vall.reshape(-1, 4, 4, H, 16, N).permute(0, 3, 1, 4, 2, 5)
    vall = vall.reshape(-1, H, 64, N // 4, 16).transpose(2, 3)
    a = powers[0].reshape(-1, 16, H, d // 32 // P, P).permute(0, 2, 3, 1, 4)
    b = powers[1].reshape(-1, 16, H, d // 32).permute(0, 2, 3, 1)
    kv = [(c.reshape(*p.shape, 32) * p[..., None]).reshape(c.shape)
          for c, p in ((kc, kp), (vc, vp))] if case["keep"] else [None, None]
    return dict(codes=torch.cat([kall.flatten(2), vall.flatten(2)], 2),
                powers=torch.cat([a.flatten(2), b.flatten(2)], 2), query=q, key=kv[0],
                value=kv[1])


def _exact_kv(case, s, r, n):
    """Keys and values [n, H, d] of a request, from the bytes' own fields."""
    H, d, block = case["kv"], case["d"], case["block"]
    N, P = d // 16, max(1, d // 128)
    rec = s.page[s.bt[r, :-(-n // block)].long()].reshape(-1, H, 33 * d)
    c = rec[..., :32 * d].int()
    e, m = c % 128 // 8, (c % 8).double()
    c = (1 - 2 * (c // 128)) * torch.where(e == 0, m / 512, (1 + m / 8) * _exact_power(e - 7))
    p = _exact_power(rec[..., 32 * d:].int() - 127)
    k = c[..., :16 * d].reshape(-1, H, d // 64, 4, 16, 16).permute(0, 4, 1, 3, 2, 5)
    v = c[..., 16 * d:].reshape(-1, H, N // 4, 64, 16).transpose(2, 3)
    v = v.reshape(-1, H, 4, 16, 4, N).permute(0, 2, 4, 1, 3, 5)
    a = p[..., :d // 2].reshape(-1, H, d // 32 // P, 16, P).permute(0, 3, 1, 2, 4)
    b = p[..., d // 2:].reshape(-1, H, d // 32, 16).permute(0, 3, 1, 2)
    return [(x.reshape(-1, H, d // 32, 32) * y.reshape(-1, H, d // 32, 1)).reshape(-1, H, d)[:n]
            for x, y in ((k, a), (v, b))]


def _exact_read(case, s):
    n = (s.starts[1:] - s.starts[:-1]).tolist()
    kv = [_exact_kv(case, s, r, m) for r, m in enumerate(n)]
    return [torch.cat([x[i] for x in kv]) for i in (0, 1)]


def _exact_decode(case, s):
    H, HQ, d, Q = case["kv"], case["heads"], case["d"], case["queries"]
    G = HQ // H
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s.q.shape[:2], dtype=torch.float64, device="cuda")
    for r, n in enumerate(s.seq.tolist()):
        k, v = _exact_kv(case, s, r, n)
        t = torch.arange(n, device="cuda")
        for j in range(Q):
            at = n - Q + j
            seen = (t <= at) & (t > at - (case["window"] or n + 1))
            kk, vv = (x[seen].permute(1, 0, 2).contiguous() for x in (k, v))
            qq = s.q[r * Q + j].double().reshape(H, G, d)
            w = (kk[:, None] * qq[:, :, None]).sum(-1) * d ** -0.5 if kk.shape[1] < 64 else \
                torch.bmm(kk, qq.transpose(1, 2).contiguous()).transpose(1, 2) * d ** -0.5
            if s.sinks is not None:
                w = torch.cat([w, s.sinks.double().reshape(H, G, 1)], -1)
            z = torch.logsumexp(w, -1, keepdim=True)
            p = torch.exp(w - z)[..., :kk.shape[1]].contiguous()
            out[r * Q + j] = torch.bmm(p, vv).reshape(HQ, d)
            lse[r * Q + j] = z.reshape(HQ)
    return [out, lse if case["lse"] else None]


def work(case):
    """Positions, slots, lengths, tables, tokens, queries, stored bytes and outputs once; the
    products of the keys that are seen."""
    kind, H, d = case["kind"], case["kv"], case["d"]
    slot = H * 33 * d // 16
    if kind == "rotary":
        n, heads = case["tokens"], case["heads"] + H
        return dict(bytes=n * (heads * d * 4 + 8) + 4 * case["rot"],
                    flops=3 * n * heads * case["rot"])
    lens = _lens(case, case["lo"], case["hi"])
    n = sum(lens)
    if kind == "write":
        turned = case["heads"] * d * 4 + 8 if case["rot"] else 0
        return dict(bytes=n * (2 * H * d * (4 if case["keep"] else 2) + slot + 8 + turned),
                    flops=n * (4 * H * d + 3 * (H + case["heads"]) * case["rot"]))
    if kind == "read":
        return dict(bytes=n * (slot + 4 * H * d), flops=2 * n * H * d)
    Q, W = case["queries"], case["window"] or 1 << 40
    rows = sum(min(m, W + Q - 1) for m in lens)
    seen = sum(min(m - Q + j + 1, W) for m in lens for j in range(Q))
    return dict(bytes=rows * slot + len(lens) * Q * case["heads"] * (4 * d + 4 * case["lse"]),
                flops=4 * case["heads"] * d * seen)

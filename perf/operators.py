"""Performance cases of the 4-bit cache: a step's plan, rotary positions with several axes, the
cache's write and the attention that reads it, one attention layer per pass.

  plan     `kernels.step_plan`: block tables, slot map and positions from the requests' lengths
  rotary   `kernels.rotary_axes`: queries and keys rotated by positions of one to three axes
  write    `kernels.nibble_write_paged`: new keys and values quantised into their slots
  decode   `kernels.nibble_decode_paged`: one query per running request over its whole store
  prefill  `kernels.nibble_prefill_paged`: chunks of prompts over what is stored, causal

`listed()` gives the fixed cases, `draw(rng)` more of the same ranges. A case is a dict of plain
values; `prepare` makes its inputs on the GPU from a seed, `run` is one pass: the package's own
operators where `own` is true, else the same results in plain torch. `exact` gives them in 64 bits,
written apart from both.

The cache holds 4-bit codes with one 16-bit parameter per group of 32 dims. Of a group x:
  lo = min(0, min x), hi = max(0, max x)              (x clamped to +-32640 first)
  s  = (hi - lo) / 15 rounded up to 7 significant bits, at least 2^-14
  z  = rint(-lo / s) in [0, 15],  c = rint(x / s) + z in [0, 15],  value = (c - z) * s
The parameter is s as fp16, whose low four bits are free, with z in them; a group that holds a
value that is not finite has the parameter 0x7e00 and stands for NaN.

Sixteen tokens of a block make a tile; a tile holds one record of 2,304 bytes per KV head:
  0     key codes, dword (qd * 16 + u) * 4 + g of token u: dims 32 g + 8 qd + j, j = 0..7, at bit
        4 (j / 2) + 16 (j % 2)
  1024  value codes, dword ((q4 * 16 + n) * 2 + pair) * 2 + quad: its low half token 4 q4 + 2 pair,
        its high half the next one, each with dims 32 g + 2 n + b, g = 2 quad + gg, at bit
        4 (2 gg + b)
  2048  key parameters, 16 bits at u * 4 + g
  2176  value parameters, 16 bits at (q4 * 4 + g) * 4 + u % 4
"""
from __future__ import annotations

import math
import random
import sys
from types import SimpleNamespace

import torch

own = False

D = 128                     # head dim
GROUP = 32
RECORD = 2304               # bytes of a tile's record of one KV head
HALVES = RECORD // 2
SCALE = D ** -0.5
POOL_TILES = 192            # distinct tiles a store is filled from
WORKSPACE = 64 << 20        # the buffer a server keeps for its reads
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of eight requests: all latency
        dict(name="plan 8x1", kind="plan", reqs=8, qlo=1, qhi=1, clo=900, chi=14000, block=16,
             pad=0, lens=1),
        # a full server's step: decodes beside chunks of prompts, padded to a graph's size
        dict(name="plan 256 mixed", kind="plan", reqs=256, qlo=1, qhi=120, clo=0, chi=16000,
             block=16, pad=37, lens=2),
        # a decode step's queries and keys
        dict(name="rotary 16", kind="rotary", tokens=16, heads=24, kv=8, dtype="fp16", axes=3,
             rot=128, interleaved=False, lens=3),
        # a long prompt with images, axes dealt in turn over the frequencies
        dict(name="rotary 8192", kind="rotary", tokens=8192, heads=32, kv=8, dtype="bf16", axes=3,
             rot=128, interleaved=True, lens=4),
        # one new token of each of eight requests: the smallest write
        dict(name="write 8x1", kind="write", kv=8, dtype="fp16", block=16, batch=8, lo=1, hi=1,
             lens=5),
        # a chunk of a long prompt
        dict(name="write 1x2048", kind="write", kv=8, dtype="bf16", block=16, batch=1, lo=2048,
             hi=2048, lens=6),
        # one user, a short context: the smallest read, all latency
        dict(name="decode 1x1082", kind="decode", heads=24, kv=8, dtype="fp16", block=16, batch=1,
             lo=1082, hi=1082, lens=7),
        # eight long conversations of the same length: the benchmark's lengths, the largest read
        dict(name="decode 8x14402", kind="decode", heads=24, kv=8, dtype="fp16", block=16, batch=8,
             lo=14402, hi=14402, lens=8),
        # a full server of short conversations, four query heads per KV head
        dict(name="decode 61 short", kind="decode", heads=32, kv=8, dtype="bf16", block=32,
             batch=61, lo=70, hi=2900, lens=9),
        # what is left of a step's token budget beside the decodes: short odd chunks, ragged
        dict(name="prefill 3x19 ragged", kind="prefill", heads=32, kv=8, dtype="bf16", block=16,
             batch=3, qlo=7, qhi=19, lo=900, hi=5200, lens=10),
        # four prompts' chunks in one step (the benchmark's continuation)
        dict(name="prefill 4x256 over 7656", kind="prefill", heads=24, kv=8, dtype="fp16",
             block=16, batch=4, qlo=256, qhi=256, lo=7400, hi=7400, lens=11),
        # one long prompt in large chunks: the most arithmetic
        dict(name="prefill 1x2048 over 12345", kind="prefill", heads=24, kv=8, dtype="bf16",
             block=16, batch=1, qlo=2048, qhi=2048, lo=10297, hi=10297, lens=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rotary", "write", "decode", "decode", "decode", "prefill",
                       "prefill"])
    c = dict(kind=kind, lens=rng.randint(1, 10 ** 6))
    if kind == "plan":
        c.update(reqs=_log(rng, 1, 1000), block=rng.choice([16, 32, 48, 64]), qlo=1, clo=0)
        c["qhi"] = _log(rng, 1, max(1, min(2048, 30000 // c["reqs"])))
        c.update(chi=_log(rng, 1, 20000), pad=rng.choice([0, rng.randint(1, 200)]))
        return c
    c.update(kv=rng.choice([8, 8, 4, 2, 1]), dtype=rng.choice(["fp16", "bf16"]),
             block=rng.choice([16, 16, 32, 48, 64]))
    if kind == "write":
        c["batch"] = _log(rng, 1, 32)
        c["lo"] = _log(rng, 1, 2048 // c["batch"])
        c["hi"] = rng.choice([c["lo"], rng.randint(c["lo"], 2048 // c["batch"])])
        return c
    c["heads"] = c["kv"] * rng.choice([1, 2, 3, 4, 4, 7, 8])
    if kind == "rotary":
        c.pop("block")
        c.update(tokens=_log(rng, 1, 8192 * 40 // max(40, c["heads"] + c["kv"])),
                 axes=rng.choice([1, 2, 3, 3]), rot=rng.choice([128, 128, 64, 96]),
                 interleaved=rng.random() < 0.5)
    elif kind == "decode":
        c["batch"] = _log(rng, 1, 64)
        most = min(16000, 110000 // c["batch"])
        c["lo"] = _log(rng, 1, most)
        c["hi"] = rng.choice([c["lo"], rng.randint(c["lo"], most)])
    else:
        c["batch"] = rng.choice([1, 1, 2, 3, 4])
        # (queries times heads, and those times keys, stay below the largest listed case's)
        c["qhi"] = _log(rng, 1, max(2, min(2048, 49152 // (c["heads"] * c["batch"]))))
        c["qlo"] = rng.choice([c["qhi"], rng.randint(1, c["qhi"])])
        c["hi"] = _log(rng, 1, 9000 // c["batch"])
        c["lo"] = rng.choice([c["hi"], rng.randint(0, c["hi"])])
    return c


# ------------------------------------------------------------------------------------ inputs
def _gen(seed, dev="cuda"):
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    return g


def _lens(case, lo, hi, n, salt=0):
    r = random.Random(case["lens"] * 7 + salt)
    return [r.randint(lo, hi) for _ in range(n)]


def _i32(v, dev="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return _i32(at)


def _tokens(n, H, g):
    """Keys with eight channels of every head that are larger than the others, and values."""
    k = torch.randn(n, H, D, generator=g, device="cuda")
    k[..., :8] *= 8
    return k, torch.randn(n, H, D, generator=g, device="cuda")


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


def _store(case, seed, lens):
    """A paged store of requests of `lens` tokens: distinct tiles, dealt out by chance."""
    g, H, block = _gen(seed), case["kv"], case["block"]
    bt, blocks = _tables(lens, block, seed)
    tiles = min(POOL_TILES, max(1, sum(lens) // 16))
    k, v = _tokens(tiles * 16, H, g)
    pool = torch.zeros(tiles, H * HALVES, dtype=torch.int16, device="cuda")
    _put(pool, torch.arange(tiles * 16, device="cuda"), *_quantise(k), *_quantise(v))
    pick = torch.randint(tiles, (blocks * block // 16,), generator=g, device="cuda")
    page = pool[pick].view(torch.uint8).reshape(blocks, block, H * 144)
    return g, page, bt, blocks


def _axis_positions(n, axes, r):
    """Positions [axes, n] of a prompt of texts and images: a text's tokens advance all axes, an
    image's lie on a grid that starts where the text before it ended."""
    rows, at = [], r.randint(0, 3000)
    while len(rows) < n:
        for _ in range(r.randint(1, 400)):
            rows.append((at,) * 3)
            at += 1
        h, w = r.randint(2, 24), r.randint(2, 32)
        rows += [(at, at + i, at + j) for i in range(h) for j in range(w)]
        at += max(h, w)
    return torch.tensor(rows[:n], dtype=torch.int64).t()[:axes].contiguous().cuda()


def _sections(axes, rot, interleaved):
    """How many of the rot / 2 frequencies each axis has."""
    half = rot // 2
    if axes == 1:
        return (half,)
    if axes == 2:
        return (half - half // 2, half // 2)
    side = 5 * half // 16 if interleaved else 3 * half // 8
    return (half - 2 * side, side, side)


def _angles(n, rot):
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    f = torch.outer(torch.arange(n, dtype=torch.float64, device="cuda"), inv)
    return torch.cat([f.cos(), f.sin()], 1).float()


def prepare(case, seed):
    s = globals()["_prepare_" + case["kind"]](case, seed)
    s.case = case
    return s


def _prepare_plan(case, seed):
    g = _gen(seed, "cpu")
    r = random.Random(case["lens"])
    R, block = case["reqs"], case["block"]
    computed = [r.randint(case["clo"], case["chi"]) for _ in range(R)]
    # two of three requests decode where the others have chunks
    counts = [1 if r.random() < 0.66 else r.randint(case["qlo"], case["qhi"]) for _ in range(R)]
    held = [-(-c // block) for c in computed]
    need = [-(-(c + n) // block) for c, n in zip(computed, counts)]
    blocks = sum(need) + 64
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    bt = torch.full((R, max(need)), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(held):
        bt[i, :k] = perm[at:at + k]
        at += k
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    return SimpleNamespace(computed=_i32(computed), counts=_i32(counts), bt=bt.cuda(),
                           free=perm[at:].cuda(), blocks=blocks,
                           tokens=sum(counts) + case["pad"], err=err)


def _prepare_rotary(case, seed):
    g = _gen(seed)
    pos = _axis_positions(case["tokens"], case["axes"], random.Random(seed))
    dt, n = DTYPES[case["dtype"]], case["tokens"]
    q = torch.randn(n, case["heads"], D, generator=g, device="cuda").to(dt)
    k = _tokens(n, case["kv"], g)[0].to(dt)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    return SimpleNamespace(q=q, k=k, pos=pos, angles=_angles(16384, case["rot"]), err=err,
                           sections=_sections(case["axes"], case["rot"], case["interleaved"]),
                           q_out=torch.empty_like(q), k_out=torch.empty_like(k))


def _prepare_write(case, seed):
    g, H, block = _gen(seed), case["kv"], case["block"]
    counts = _lens(case, case["lo"], case["hi"], case["batch"])
    before = _lens(case, 0, 300, case["batch"], salt=1)
    bt, blocks = _tables([b + n for b, n in zip(before, counts)], block, seed)
    p = [torch.arange(b, b + n, device="cuda") for b, n in zip(before, counts)]
    slots = torch.cat([bt[r].long()[i // block] * block + i % block for r, i in enumerate(p)])
    k, v = (x.to(DTYPES[case["dtype"]]) for x in _tokens(sum(counts), H, g))
    page = torch.zeros(blocks, block, H * 144, dtype=torch.uint8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    return SimpleNamespace(k=k, v=v, slots=slots, page=page, err=err,
                           k_out=torch.empty(k.shape, dtype=torch.float16, device="cuda"),
                           v_out=torch.empty(k.shape, dtype=torch.float16, device="cuda"))


def _reads(case):
    """(tokens stored, queries) of each request: a prompt's chunk is stored before it is read."""
    if case["kind"] == "decode":
        lens = _lens(case, case["lo"], case["hi"], case["batch"])
        return lens, [1] * len(lens)
    counts = _lens(case, case["qlo"], case["qhi"], case["batch"])
    before = _lens(case, case["lo"], case["hi"], case["batch"], salt=1)
    return [b + n for b, n in zip(before, counts)], counts


def _prepare_read(case, seed):
    lens, counts = _reads(case)
    g, page, bt, _ = _store(case, seed, lens)
    q = torch.randn(sum(counts), case["heads"], D, generator=g, device="cuda")
    q = q.to(DTYPES[case["dtype"]])
    return SimpleNamespace(page=page, bt=bt, seq=_i32(lens), qsl=_starts(counts), q=q,
                           longest=max(lens), most=max(counts), out=torch.empty_like(q),
                           ws=torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda"),
                           err=torch.zeros(1, dtype=torch.int32, device="cuda"))


_prepare_decode = _prepare_prefill = _prepare_read


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
        from vllm_ttkv.nibble import NibbleLayout
        lay = s.lay = NibbleLayout(H=s.case["kv"])
    return lay


def _own_plan(s):
    p = _kernels().step_plan(s.computed, s.counts, s.bt, s.free, s.case["block"], s.blocks,
                             s.tokens, error_word=s.err)
    return [p.query_start_loc, p.seq_lens, p.slot_mapping, p.positions, p.blocks_used, s.bt]


def _own_rotary(s):
    return list(_kernels().rotary_axes(s.q, s.k, s.pos, s.angles, s.sections,
                                       interleaved=s.case["interleaved"], query_out=s.q_out,
                                       key_out=s.k_out, error_word=s.err))


def _own_write(s):
    _kernels().nibble_write_paged(_layout(s), s.k, s.v, s.slots, s.page, key_out=s.k_out,
                                  value_out=s.v_out, error_word=s.err)
    return dict(key=s.k_out, value=s.v_out, page=s.page)


def _own_decode(s):
    return _kernels().nibble_decode_paged(
        _layout(s), s.q, s.page, s.case["block"], s.bt, s.seq, s.qsl, s.longest, SCALE, out=s.out,
        workspace=s.ws, error_word=s.err)


def _own_prefill(s):
    return _kernels().nibble_prefill_paged(
        _layout(s), s.q, s.page, s.case["block"], s.bt, s.seq, s.qsl, s.most, s.longest, SCALE,
        out=s.out, workspace=s.ws, error_word=s.err)


# ------------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    block, W = s.case["block"], s.bt.shape[1]
    seq = s.computed + s.counts
    have, need = (s.computed + block - 1) // block, (seq + block - 1) // block
    new = need - have
    first = torch.cumsum(new, 0) - new
    qsl = torch.nn.functional.pad(torch.cumsum(s.counts, 0), (1, 0)).to(torch.int32)
    col = torch.arange(W, device="cuda")
    fresh = (col >= have[:, None]) & (col < need[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, s.free.numel() - 1)
    s.bt.copy_(torch.where(fresh, s.free[at], s.bt))
    t = torch.arange(s.tokens, device="cuda", dtype=torch.int32)
    req = torch.searchsorted(qsl[1:].contiguous(), t, right=True)
    live = req < seq.numel()
    req = req.clamp(max=seq.numel() - 1)
    pos = torch.where(live, s.computed[req] + t - qsl[req], 0).long()
    slot = s.bt[req, pos // block].long() * block + pos % block
    return [qsl, seq, torch.where(live, slot, -1), pos, new.sum().to(torch.int32).reshape(1), s.bt]


def _axis_of(sections, interleaved):
    """The axis whose position turns each frequency."""
    A, half = len(sections), sum(sections)
    j = torch.arange(half, device="cuda")
    ends = torch.tensor(sections, device="cuda")
    if interleaved:
        a = j % A
        return torch.where(j < A * ends[a], a, 0)
    return torch.searchsorted(torch.cumsum(ends, 0), j, right=True)


def _plain_rotary(s):
    half = s.case["rot"] // 2
    at = s.pos[_axis_of(s.sections, s.case["interleaved"])].t()          # [N, half]
    j = torch.arange(half, device="cuda")
    c, sn = s.angles[at, j][:, None], s.angles[at, j + half][:, None]

    def turn(x):
        f = x.float()
        a, b = f[..., :half], f[..., half:2 * half]
        return torch.cat([a * c - b * sn, b * c + a * sn, f[..., 2 * half:]], -1).to(x.dtype)
    return [turn(s.q), turn(s.k)]


def _quantise(x):
    """(codes uint8, scales, zero codes, parameters int16) of rows [..., 128] in groups of 32; the
    quotients in 64 bits, since they may lie next to a rounding border."""
    x = x.double().reshape(*x.shape[:-1], D // GROUP, GROUP)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    x = torch.where(bad, 0.0, x.clamp(-32640.0, 32640.0))
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    low = (1 << 46) - 1                              # all but the first seven significant bits
    s = ((((hi - lo) / 15).view(torch.int64) + low) & ~low).view(torch.float64)
    s = s.clamp(min=2.0 ** -14)
    z = torch.round(-lo / s).clamp(0, 15)
    c = (torch.round(x / s) + z).clamp(0, 15)
    par = s.half().view(torch.int16) | z.to(torch.int16)
    par = torch.where(bad, 0x7e00, par).to(torch.int16)
    s = torch.where(bad, float("nan"), s)
    return c.to(torch.int32), s, z, par.squeeze(-1)


def _halves(nibbles):
    """Four nibbles [..., 4], lowest first, as int16."""
    return (nibbles << torch.tensor([0, 4, 8, 12], device="cuda")).sum(-1).to(torch.int16)


def _put(page16, slots, kc, _ks, _kz, kp, vc, _vs, _vz, vp):
    """Codes and parameters of tokens [N, H, 4, 32] into their slots of a cache [tiles, ...]."""
    N, H = kc.shape[:2]
    flat = page16.view(-1)
    ar = lambda *n: [torch.arange(k, device="cuda").reshape([-1] + [1] * (len(n) - 1 - i))  # noqa: E731
                     for i, k in enumerate(n)]
    u = (slots % 16).reshape(N, 1, 1, 1, 1)
    h = torch.arange(H, device="cuda").reshape(1, H, 1, 1, 1)
    base = (slots // 16).reshape(N, 1, 1, 1, 1) * (H * HALVES) + h * HALVES
    g, qd, b = ar(4, 4, 2)
    k = _halves(kc.reshape(N, H, 4, 4, 4, 2).transpose(-1, -2))          # [N, H, g, qd, b]
    flat[base + 2 * ((qd * 16 + u) * 4 + g) + b] = k
    quad, n, _ = ar(2, 16, 1)
    v = vc.reshape(N, H, 2, 2, 16, 2).permute(0, 1, 2, 4, 3, 5)          # [N, H, quad, n, gg, b]
    at = (((u // 4) * 16 + n) * 2 + (u % 4) // 2) * 2 + quad
    flat[base + 512 + 2 * at + u % 2] = _halves(v.reshape(N, H, 2, 16, 4)).unsqueeze(-1)
    base, u, g = base[..., 0], u[..., 0], torch.arange(4, device="cuda").reshape(4, 1)
    flat[base + 1024 + u * 4 + g] = kp.unsqueeze(-1)
    flat[base + 1088 + (u // 4 * 4 + g) * 4 + u % 4] = vp.unsqueeze(-1)


def _plain_write(s):
    k, v = _quantise(s.k), _quantise(s.v)
    _put(s.page.view(torch.int16), s.slots, *k, *v)
    key, value = (((c - z) * sc).half().reshape(s.k.shape) for c, sc, z, _ in (k, v))
    return dict(key=key, value=value, page=s.page)


def _values(params):
    """Scales and zero codes of parameters (int16)."""
    return (params & -16).view(torch.float16).float(), (params & 15).float()


def _stored(page, bt, block, H):
    """Keys and values [B, tokens, H, 128] fp32 of the blocks of a block table."""
    B = bt.shape[0]
    t = page[bt.clamp(min=0).long()].reshape(-1, H, RECORD)              # [B * tiles, H, record]
    T = t.shape[0]
    w = t[..., :2048].view(torch.int32)
    bits = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device="cuda", dtype=torch.int32)
    k = (w[..., :256].reshape(T, H, 4, 16, 4, 1) >> bits) & 15           # [T, H, qd, u, g, 8]
    k = k.permute(0, 3, 1, 4, 2, 5).reshape(T, 16, H, 4, 32)
    bits = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    v = (w[..., 256:].reshape(T, H, 4, 16, 2, 2, 1) >> bits) & 15
    v = v.reshape(T, H, 4, 16, 2, 2, 2, 2, 2)       # [T, H, q4, n, pair, quad, half, gg, b]
    v = v.permute(0, 2, 4, 6, 1, 5, 7, 3, 8).reshape(T, 16, H, 4, 32)
    par = t[..., 2048:].contiguous().view(torch.int16)
    s, z = _values(par[..., :64].reshape(T, H, 16, 4).transpose(1, 2))
    k = (k - z[..., None]) * s[..., None]
    s, z = _values(par[..., 64:].reshape(T, H, 4, 4, 4).permute(0, 2, 4, 1, 3).reshape(T, 16, H, 4))
    v = (v - z[..., None]) * s[..., None]
    return k.reshape(B, -1, H, D), v.reshape(B, -1, H, D)


def _plain_read(s):
    """Causal attention of every request's queries, padded to the longest chunk, in fp32."""
    H, HQ, N = s.case["kv"], s.case["heads"], s.q.shape[0]
    G, Q = HQ // H, s.most
    K, V = _stored(s.page, s.bt, s.case["block"], H)
    B, n = K.shape[:2]
    K, V = K.permute(0, 2, 3, 1).contiguous(), V.permute(0, 2, 1, 3).contiguous()
    tok = torch.arange(N, device="cuda", dtype=torch.int32)
    req = torch.searchsorted(s.qsl[1:].contiguous(), tok, right=True)
    j = tok - s.qsl[req]
    q = torch.zeros(B, Q, HQ, D, device="cuda")
    q[req, j] = s.q.float()
    q = q.reshape(B, Q, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, Q * G, D)
    p = (torch.matmul(q, K) * SCALE).reshape(B, H, Q, G, n)
    first = (s.seq - (s.qsl[1:] - s.qsl[:-1])).reshape(B, 1)             # position of query 0
    last = first + torch.arange(Q, device="cuda")                        # [B, Q]
    t = torch.arange(n, device="cuda")
    hidden = t > last[..., None]
    p.masked_fill_(hidden[:, None, :, None], float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    V = torch.where((t < s.seq[:, None])[:, None, :, None], V, 0.0)
    o = torch.matmul(p.reshape(B, H, Q * G, n), V) / p.sum(-1).reshape(B, H, Q * G, 1)
    o = o.reshape(B, H, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, HQ, D)
    return o[req, j].to(s.q.dtype)


_plain_decode = _plain_prefill = _plain_read


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["kind"]](case, s)


def _exact_plan(case, s):
    return None                                      # whole numbers only


def _exact_rotary(case, s):
    A, half, outs = case["axes"], case["rot"] // 2, []
    for x in (s.q, s.k):
        y = x.double().clone()
        ends, a = list(s.sections), 0
        for j in range(half):
            if case["interleaved"]:
                a = j % A if j < A * s.sections[j % A] else 0
            else:
                while j >= sum(ends[:a + 1]):
                    a += 1
            cs = s.angles[s.pos[a]].double()
            c, sn = cs[:, j, None], cs[:, j + half, None]
            lo, hi = x[:, :, j].double(), x[:, :, j + half].double()
            y[:, :, j], y[:, :, j + half] = lo * c - hi * sn, hi * c + lo * sn
        outs.append(y)
    return outs


def _exact_write(case, s):
    def stands_for(x):
        out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for g in range(0, D, GROUP):
            part = x[..., g:g + GROUP].double()
            low = torch.minimum(part.min(-1).values, torch.zeros((), device="cuda").double())
            high = torch.maximum(part.max(-1).values, torch.zeros((), device="cuda").double())
            step = (high - low) / 15
            unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=2.0 ** -14))) - 6)
            step = (torch.ceil(step / unit) * unit).clamp(min=2.0 ** -14).unsqueeze(-1)
            zero = torch.round(-low.unsqueeze(-1) / step)
            code = torch.clamp(torch.round(part / step) + zero, 0, 15)
            out[..., g:g + GROUP] = (code - zero) * step
        return out
    return dict(key=stands_for(s.k), value=stands_for(s.v), page=None)


def _exact_places():
    """(byte, shift) of every code and (byte) of every parameter of a record, by token and dim."""
    u = torch.arange(16).reshape(16, 1)
    x = torch.arange(D).reshape(1, D)
    g, i = x // 32, x % 32
    bit = 32 * (((i // 8) * 16 + u) * 4 + g) + 4 * ((i % 8) // 2) + 16 * (i % 2)
    key = (bit // 8, bit % 8, 2048 + 2 * (u * 4 + g))
    word = (((u // 4) * 16 + i // 2) * 2 + (u % 4) // 2) * 2 + g // 2
    bit = 32 * word + 16 * (u % 2) + 4 * (2 * (g % 2) + i % 2)
    val = (1024 + bit // 8, bit % 8, 2176 + 2 * ((u // 4 * 4 + g) * 4 + u % 4))
    return [[t.expand(16, D).reshape(-1).cuda() for t in part] for part in (key, val)]


def _exact_decode(case, s):
    H, HQ, block = case["kv"], case["heads"], case["block"]
    G, places = HQ // H, _exact_places()
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    qsl, seq = s.qsl.tolist(), s.seq.tolist()
    for r, n in enumerate(seq):
        a, b = qsl[r], qsl[r + 1]
        ids = s.bt[r, :-(-n // block)].long()
        rec = s.page[ids].reshape(-1, H, RECORD)
        future = (torch.arange(n, device="cuda")[None, :]
                  > n - (b - a) + torch.arange(b - a, device="cuda")[:, None])
        for h in range(H):
            kv = []
            for byte, shift, par in places:
                one = rec[:, h]
                word = one[:, par].int() + 256 * one[:, par + 1].int()
                zero = word % 16
                step = (word - zero).to(torch.int16).view(torch.float16).double()
                code = (one[:, byte].int() >> shift) % 16
                kv.append(((code - zero).double() * step).reshape(-1, D)[:n])
            qs = s.q[a:b, h * G:(h + 1) * G].double().reshape(-1, D)
            w = (qs @ kv[0].t().contiguous() * SCALE).reshape(b - a, G, n)
            w = torch.softmax(w.masked_fill(future[:, None], float("-inf")), -1)
            out[a:b, h * G:(h + 1) * G] = (w.reshape(-1, n) @ kv[1]).reshape(b - a, G, D)
    return out


_exact_prefill = _exact_decode


def work(case):
    """Lengths, tables, tokens, slots, queries and outputs once; the causal products."""
    kind = case["kind"]
    if kind == "plan":
        r, R = random.Random(case["lens"]), case["reqs"]
        block, fresh = case["block"], 0
        computed = [r.randint(case["clo"], case["chi"]) for _ in range(R)]
        counts = [1 if r.random() < 0.66 else r.randint(case["qlo"], case["qhi"])
                  for _ in range(R)]
        for c, n in zip(computed, counts):
            fresh += -(-(c + n) // block) - -(-c // block)
        return dict(bytes=8 * R + 4 * R + 8 * fresh + 8 * R + 16 * (sum(counts) + case["pad"]),
                    flops=0)
    if kind == "rotary":
        n, heads = case["tokens"], case["heads"] + case["kv"]
        return dict(bytes=n * (heads * D * 4 + 8 * case["axes"] + 4 * case["rot"]),
                    flops=3 * n * heads * case["rot"])
    H = case["kv"]
    if kind == "write":
        n = sum(_lens(case, case["lo"], case["hi"], case["batch"]))
        return dict(bytes=n * (2 * H * D * 4 + H * 144 + 8), flops=4 * n * 2 * H * D)
    lens, counts = _reads(case)
    seen = sum(q * (n - q) + q * (q + 1) // 2 for n, q in zip(lens, counts))
    return dict(bytes=sum(lens) * H * 144 + 4 * sum(counts) * case["heads"] * D,
                flops=4 * case["heads"] * D * seen)

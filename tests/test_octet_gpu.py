"""The 8-bit cache's kernels on the GPU against the oracle in 64 bits: scaled rotary positions, written
bytes, rows read back and attention at the lengths, head dims, tables, windows and types where they can
go wrong, and a run of them together.

Tolerances. Rotary: an angle's cosine and sine are off by at most 2^-22 (the radians' rounding to fp32
and the series' own, four of 2^-24) and, of a far position p, by 2 pi 2^-53 p turns; the two products and
their sum round by 2^-24 each: 2^-21 of |x_u| + |x_v|, times the amplitude. Then one rounding to the
type, half a step. A stored rotated key adds half a step of e4m3 at the stored power: 2^-4 of the value,
at least 2^-10 of the power of two.
Attention: scores are sums of d exact products in 32 bits, off by d 2^-24 of sum |q k| * scale, which
moves a weight by that relative amount and the weights' sum with it (twice); a weight is carried in two
16-bit parts, 2^-18 of it; at most n / 4 + 64 additions of weights and of weighted values follow one
another: (n / 4 + 64) 2^-24 of spread = sum p |v|, each. The factor 1.05 covers products of these terms;
fp16 outputs below 2^-14 are spaced 2^-24."""
import math

import pytest
import torch

from oracle import nibble as on
from oracle import octet as oo
from vllm_ttkv import kernels, synth
from vllm_ttkv.octet import OctetLayout
from vllm_ttkv.rope import Rotary, scaled_rotary

pytestmark = pytest.mark.gpu
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _err():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------ rotary
def _turn_tol(x, pos, r, half, dtype):
    """What a turned row may be off by before its rounding."""
    xx = x.double().abs()
    if r.adjacent:
        both = (xx[..., :2 * half:2] + xx[..., 1:2 * half:2]).repeat_interleave(2, -1)
    else:
        both = (xx[..., :half] + xx[..., half:2 * half]).repeat(1, 1, 2)
    far = 2 * math.pi * 2.0 ** -53 * pos.double() * float(r.turns.max())
    tol = (2.0 ** -21 + far)[:, None, None] * both * abs(r.amplitude)
    return torch.cat([tol, torch.zeros_like(xx[..., 2 * half:])], -1)


def _turn_close(got, x, pos, r):
    half = r.turns.numel()
    want = oo.turn(x, pos, r.turns.tolist(), r.amplitude, r.adjacent)
    tol = _turn_tol(x, pos, r, half, got.dtype) + HALF[got.dtype] * want.abs() * 1.01 + 2.0 ** -25
    tol[..., 2 * half:] = 0                                  # copied
    e = (got.cpu().double() - want).abs()
    assert bool((e <= tol).all()), (float(e.max()), float((e / tol.clamp(min=1e-30)).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("N,HQ,H,d,rot", [(1, 1, 1, 64, 64), (3, 4, 2, 128, 128), (5, 3, 1, 128, 32),
                                          (2, 2, 2, 96, 34), (17, 5, 0, 256, 192), (2, 1, 1, 6, 2),
                                          (4, 16, 8, 128, 6), (3, 2, 1, 80, 80)])
def test_rotary(dtype, adjacent, N, HQ, H, d, rot):
    g = _gen(N * d + rot)
    q = torch.randn(N, HQ, d, generator=g).to(dtype)
    k = torch.randn(N, H, d, generator=g).to(dtype) if H else None
    pos = torch.randint(0, 200000, (N,), generator=g)
    pos[0] = 0
    r = scaled_rotary(rot, rule="yarn", factor=8.0, adjacent=adjacent)
    dev = Rotary(r.turns.cuda(), r.amplitude, adjacent)
    err = _err()
    qo, ko = kernels.rotary_scaled(q.cuda(), None if k is None else k.cuda(), pos.cuda(), dev,
                                   error_word=err)
    assert int(err) == 0
    _turn_close(qo, q, pos, r)
    if H:
        _turn_close(ko, k, pos, r)


def test_rotary_far_positions():
    g = _gen(5)
    q = torch.randn(6, 2, 128, generator=g)
    pos = torch.tensor([2 ** 31 - 1, 2 ** 30 + 7, 123456789, 1000003, 2 ** 24 + 1, 1])
    for adjacent in (False, True):
        r = Rotary(scaled_rotary(128, 10000.0).turns, 1.5, adjacent)
        got, _ = kernels.rotary_scaled(q.cuda(), None, pos.cuda(), r._replace(turns=r.turns.cuda()))
        _turn_close(got, q, pos, r)


@pytest.mark.parametrize("dtype,pad,shift", [(torch.bfloat16, 8, 0), (torch.float16, 3, 0),
                                             (torch.float32, 0, 1), (torch.bfloat16, 0, 1)])
def test_rotary_strides_and_in_place(dtype, pad, shift):
    """Rows at any stride and alignment; outputs that are their inputs; what lies between is left."""
    g = _gen(pad + shift)
    N, HQ, d = 9, 3, 128
    flat = torch.randn(N * (HQ * d + pad) + shift, generator=g).to(dtype).cuda()
    q = flat[shift:].as_strided((N, HQ, d), (HQ * d + pad, d, 1))
    before = flat.clone()
    pos = torch.randint(0, 5000, (N,), generator=g)
    for adjacent, rot in ((False, 128), (True, 64), (False, 48), (False, 64)):
        r = scaled_rotary(rot, adjacent=adjacent)
        dev = r._replace(turns=r.turns.cuda())
        x = q.cpu().clone()
        out, _ = kernels.rotary_scaled(q, None, pos.cuda(), dev)
        _turn_close(out, x, pos, r)
        kernels.rotary_scaled(q, None, pos.cuda(), dev, query_out=q)
        assert torch.equal(q, out)
    mask = torch.ones_like(flat, dtype=torch.bool)
    mask[shift:].as_strided((N, HQ, d), (HQ * d + pad, d, 1)).fill_(False)
    assert torch.equal(flat[mask], before[mask])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("adjacent,rot", [(False, 128), (True, 128), (False, 48), (True, 24)])
def test_rotary_of_rows_beyond_the_caches(dtype, adjacent, rot):
    """Past 128 MB of rows read and written: bit for bit as in calls of a few of them."""
    N = 6600 if dtype == torch.float32 else 13200
    gen = torch.Generator(device="cuda").manual_seed(rot)
    q, k = (torch.randn(N, h, 128, generator=gen, device="cuda").to(dtype) for h in (16, 4))
    assert 2 * (q.numel() + k.numel()) * q.element_size() > 128 << 20
    pos = torch.arange(N, device="cuda") * 7
    r = scaled_rotary(rot, rule="yarn", factor=4.0, adjacent=adjacent, device="cuda")
    qo, ko = kernels.rotary_scaled(q, k, pos, r)
    for a in range(0, N, 1100):
        s = slice(a, a + 1100)
        few = kernels.rotary_scaled(q[s], k[s], pos[s], r)
        assert torch.equal(qo[s], few[0]) and torch.equal(ko[s], few[1])
    kernels.rotary_scaled(q, k, pos, r, query_out=q, key_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)


def test_rotary_refused_positions_and_values():
    q = torch.randn(5, 2, 64, generator=_gen(3)).half().cuda()
    q[1, 0, 7], q[1, 1, 40] = float("nan"), float("inf")
    pos = torch.tensor([3, 4, -1, 2 ** 31, 5]).cuda()
    r = scaled_rotary(32, device="cuda")
    err = _err()
    out, _ = kernels.rotary_scaled(q, None, pos, r, error_word=err)
    assert int(err) == 16
    assert bool(torch.isnan(out[2:4]).all())
    for i in (0, 4):
        _turn_close(out[i:i + 1], q[i:i + 1].cpu(), pos[i:i + 1].cpu(), r._replace(turns=r.turns.cpu()))
    assert int(torch.isnan(out[1, 0]).sum()) == 2 and int((~torch.isfinite(out[1, 1])).sum()) == 1
    empty, _ = kernels.rotary_scaled(q[:0], None, pos[:0], r)
    assert empty.shape == (0, 2, 64)


# ------------------------------------------------------------------------------------- write
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,H,n,pad", [(64, 1, 1, 0), (64, 3, 40, 12), (128, 2, 17, 8), (128, 8, 5, 0),
                                       (256, 1, 23, 0), (256, 5, 4, 48), (128, 1, 90, 1)])
def test_write_bytes(dtype, d, H, n, pad):
    """Every byte of the page, also those no token owns; the stored values; padded tokens."""
    g = _gen(n)
    k, v = (torch.randn(n, H, d, generator=g) for _ in range(2))
    k *= 2.0 ** torch.randint(-22, 12, (n, 1, 1), generator=g)
    k[..., 32:64] = torch.where(torch.rand(n, H, 1, generator=g) < 0.3,
                                torch.arange(32) + 432.5, k[..., 32:64])
    v[0, 0, 33], v[-1, -1, 60] = float("nan"), -float("inf")
    v[n // 2, 0, :32] *= 3e4
    if dtype != torch.float16:
        v[n // 3, 0, :32] *= 1e37
        k[n // 3, 0, :32] *= 1e-37
    if n > 2:
        v[2] = 0
        v[1, 0, :32] = -v[1, 0, :32].abs() * 2.0 ** -20
    k, v = k.to(dtype), v.to(dtype)
    stride, n_slots = OctetLayout(H, d).compressed_bytes_per_token() + pad, 96
    slots = torch.randperm(n_slots, generator=g)[:n]
    if n > 20:                                          # a chunk of a prompt, off the tiles' borders
        slots = torch.arange(n) + 3
    if n > 3:
        slots[3] = -1
    page = torch.randint(0, 256, (6, 16, stride), generator=g, dtype=torch.uint8)
    want = page.reshape(-1).clone()
    oo.write(want, stride, slots, k, v)
    dev, err = page.cuda(), _err()
    ko = torch.full((n, H, d), 7.0, dtype=torch.bfloat16, device="cuda")
    vo = ko.clone()
    kernels.octet_write_paged(OctetLayout(H, d), k.cuda(), v.cuda(), slots.cuda(), dev, key_out=ko,
                              value_out=vo, error_word=err)
    assert int(err) == 0
    assert torch.equal(dev.cpu().reshape(-1), want)
    for got, x in ((ko, k), (vo, v)):
        ref = oo.values(x)
        ref[slots < 0] = 7.0
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=-9.0),
                           torch.nan_to_num(ref, nan=-9.0))


def test_write_types_strides_and_bad_slots():
    """Keys and values of different types at their own strides, unaligned; slots past the cache."""
    g = _gen(11)
    n, H, d = 21, 2, 64
    lay = OctetLayout(H, d)
    kf = torch.randn(n * (H * d + 5) + 1, generator=g).cuda()
    vf = torch.randn(n * (H * d + 2), generator=g).bfloat16().cuda()
    k = kf[1:].as_strided((n, H, d), (H * d + 5, d, 1))
    v = vf.as_strided((n, H, d), (H * d + 2, d, 1))
    slots = torch.randperm(64, generator=g)[:n]
    slots[4], slots[9] = 64, 2 ** 40
    page = torch.zeros(4, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8)
    want = page.reshape(-1).clone()
    oo.write(want, lay.compressed_bytes_per_token(), torch.where(slots < 64, slots, -1), k.cpu(),
             v.cpu())
    dev, err = page.cuda(), _err()
    kernels.octet_write_paged(lay, k, v, slots.cuda(), dev, error_word=err)
    assert int(err) == 4 and torch.equal(dev.cpu().reshape(-1), want)


@pytest.mark.parametrize("d,rot,adjacent", [(64, 64, False), (64, 10, True), (128, 128, False),
                                            (128, 64, True), (128, 50, False), (256, 192, False),
                                            (256, 256, True), (128, 2, False)])
@pytest.mark.parametrize("dtype", TYPES)
def test_write_rotates(dtype, d, rot, adjacent):
    """Rotated on the way: each stored key within its own rounding of the exact one, values as they
    come, queries as the rotation by itself gives them; padded tokens' queries rotated too."""
    g = _gen(d + rot)
    n, H, HQ = 37, 2, 6
    lay = OctetLayout(H, d)
    k, v, q = (torch.randn(n, h, d, generator=g).to(dtype) for h in (H, H, HQ))
    pos = torch.arange(n) + 70000
    slots = torch.arange(n) + 5
    slots[7] = -1
    r = scaled_rotary(rot, rule="llama3", factor=32.0, adjacent=adjacent)._replace(amplitude=1.25)
    dev = r._replace(turns=r.turns.cuda())
    page = torch.zeros(4, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8, device="cuda")
    err = _err()
    ko = torch.zeros(n, H, d, dtype=torch.bfloat16, device="cuda")
    qo = kernels.octet_write_paged(lay, k.cuda(), v.cuda(), slots.cuda(), page, rotary=dev,
                                   positions=pos.cuda(), query=q.cuda(), key_out=ko, error_word=err)
    assert int(err) == 0
    alone, _ = kernels.rotary_scaled(q.cuda(), None, pos.cuda(), dev)
    assert torch.equal(qo, alone)
    _turn_close(qo, q, pos, r)
    kept = slots >= 0
    want = oo.turn(k, pos, r.turns.tolist(), r.amplitude, adjacent)[kept]
    off = _turn_tol(k, pos, r, rot // 2, dtype)[kept]
    (kc, kb), (vc, vb) = oo.fields(page, lay.compressed_bytes_per_token(), slots[kept], H, d)
    got, power = oo.combine(kc, kb), 2.0 ** (kb.double() - 127)
    assert torch.equal(got, ko.cpu().double()[kept])
    step = torch.maximum(want.abs() / 16, power.repeat_interleave(32, -1) * 2.0 ** -10)
    e = (got - want).abs()
    assert bool((e <= (step + off) * 1.001).all()), float((e / (step + off)).max())
    # the power is the smallest that holds the group, up to what the rotation may be off by
    top = want.reshape(*kb.shape, 32).abs().amax(-1)
    slack = off.reshape(*kb.shape, 32).amax(-1)
    assert bool((top - slack <= 448 * power).all()) and bool((top + slack > 224 * power).all())
    assert torch.equal(oo.combine(vc, vb), oo.values(v)[kept])


@pytest.mark.parametrize("d,rot,adjacent", [(64, 64, True), (128, 128, False), (128, 50, False), (256, 64, True),
                                            (256, 256, False)])
@pytest.mark.parametrize("kt,vt,qt,pad", [(torch.float32, torch.bfloat16, torch.float16, 3),
                                          (torch.float16, torch.float32, torch.float32, 8),
                                          (torch.bfloat16, torch.bfloat16, torch.float32, 1)])
def test_write_rotates_rows_of_any_type_and_stride(d, rot, adjacent, kt, vt, qt, pad):
    """Keys, values and queries of their own types, in rows of odd strides that start off 16 bytes: the bytes,
    and the stored values of contiguous rows of the same types, which the same kernel takes."""
    g = _gen(d + rot + pad)
    n, H, HQ = 21, 2, 3
    lay = OctetLayout(H, d)

    def rows(h, t):
        flat = torch.randn(n * (h * d + pad) + 1, generator=g).to(t).cuda()
        return flat[1:].as_strided((n, h, d), (h * d + pad, d, 1))

    k, v, q = rows(H, kt), rows(H, vt), rows(HQ, qt)
    pos, slots = torch.arange(n).cuda() * 31 + 5000, torch.arange(n).cuda() + 9
    slots[4] = -1
    r = scaled_rotary(rot, rule="linear", factor=2.0, adjacent=adjacent, device="cuda")
    pages = [torch.zeros(2, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8, device="cuda") for _ in range(2)]
    kept = [torch.zeros(n, H, d, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    err = _err()
    qo = kernels.octet_write_paged(lay, k, v, slots, pages[0], rotary=r, positions=pos, query=q, key_out=kept[0],
                                   value_out=kept[1], error_word=err)
    assert int(err) == 0
    host = r._replace(turns=r.turns.cpu())
    _turn_close(qo, q.cpu(), pos.cpu(), host)
    alone = kernels.octet_write_paged(lay, k.contiguous(), v.contiguous(), slots, pages[1], rotary=r, positions=pos,
                                      query=q.contiguous(), key_out=kept[2], value_out=kept[3])
    _turn_close(alone, q.cpu(), pos.cpu(), host)
    assert torch.equal(pages[0], pages[1])
    assert torch.equal(kept[0], kept[2]) and torch.equal(kept[1], kept[3])
    on = slots.cpu() >= 0
    (kc, kb), _ = oo.fields(pages[0], lay.compressed_bytes_per_token(), slots.cpu()[on], H, d)
    want = oo.turn(k.cpu(), pos.cpu(), host.turns.tolist(), 1.0, adjacent)[on]
    off = _turn_tol(k.cpu(), pos.cpu(), host, rot // 2, kt)[on]
    step = torch.maximum(want.abs() / 16, 2.0 ** (kb.double() - 137).repeat_interleave(32, -1))
    assert bool(((oo.combine(kc, kb) - want).abs() <= (step + off) * 1.001).all())
    assert torch.equal(kept[1].cpu().double()[on], oo.values(v.cpu())[on])


def test_write_rotates_by_refused_positions():
    g = _gen(8)
    lay = OctetLayout(1, 64)
    k, v = (torch.randn(3, 1, 64, generator=g).cuda() for _ in range(2))
    page = torch.zeros(1, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8, device="cuda")
    err = _err()
    kernels.octet_write_paged(lay, k, v, torch.arange(3).cuda(), page,
                              rotary=scaled_rotary(32, device="cuda"),
                              positions=torch.tensor([5, -2, 9]).cuda(), error_word=err)
    assert int(err) == 16
    K, V = oo.read(page.reshape(-1), 132, torch.arange(3), 1, 64)
    assert bool(torch.isnan(K[1]).all()) and bool(torch.isfinite(K[[0, 2]]).all())
    assert torch.equal(V, oo.values(v.cpu()))


def test_write_in_place_queries_and_waiting():
    """query_out may be the query; a call without tokens does nothing."""
    g = _gen(9)
    lay = OctetLayout(2, 128)
    k, v, q = (torch.randn(6, h, 128, generator=g).bfloat16().cuda() for h in (2, 2, 4))
    page = torch.zeros(1, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8, device="cuda")
    r, pos = scaled_rotary(128, device="cuda"), torch.arange(6).cuda() * 100
    want, _ = kernels.rotary_scaled(q, None, pos, r)
    out = kernels.octet_write_paged(lay, k, v, torch.arange(6).cuda(), page, rotary=r, positions=pos,
                                    query=q, query_out=q)
    assert out is q and torch.equal(q, want)
    ko, vo = k.clone(), v.clone()                       # the stored values in the inputs' place
    for rotary in (r, None):
        want = torch.empty_like(k)
        kw = dict(rotary=rotary, positions=pos) if rotary else {}
        kernels.octet_write_paged(lay, k, v, torch.arange(6).cuda(), page, key_out=want, **kw)
        ko.copy_(k), vo.copy_(v)
        kernels.octet_write_paged(lay, ko, vo, torch.arange(6).cuda(), page, key_out=ko, value_out=vo, **kw)
        assert torch.equal(ko, want) and torch.equal(vo.cpu().double(), oo.values(v.cpu()))
    before = page.clone()
    kernels.octet_write_paged(lay, k[:0], v[:0], torch.arange(0).cuda(), page)
    assert torch.equal(page, before)


def test_more_tokens_than_a_launch_has_threads():
    """2^24 tokens and some: each as in a small call of its neighbours."""
    N = 2 ** 24 + 37
    spans = [slice(a, a + 300) for a in (0, 2 ** 22 - 100, 2 ** 23 - 150, 2 ** 23 + 4000, N - 300)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(N, 1, 2, generator=gen, device="cuda").bfloat16()
    pos = torch.arange(N, device="cuda") % 100003
    r, err = scaled_rotary(2, device="cuda"), _err()
    out, _ = kernels.rotary_scaled(x, None, pos, r, error_word=err)
    assert int(err) == 0
    for s in spans:
        assert torch.equal(out[s], kernels.rotary_scaled(x[s], None, pos[s], r)[0])
    del x, out
    lay, r = OctetLayout(1, 64), scaled_rotary(64, device="cuda")
    q = torch.randn(N, 1, 64, generator=gen, device="cuda", dtype=torch.bfloat16)
    slots = torch.full((N,), -1, dtype=torch.int64, device="cuda")
    for i, s in enumerate(spans):
        slots[s] = torch.arange(i * 300, i * 300 + 300, device="cuda")
    pages = [torch.zeros(94, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8, device="cuda") for _ in range(2)]
    out = kernels.octet_write_paged(lay, q, q, slots, pages[0], rotary=r, positions=pos, query=q, error_word=err)
    assert int(err) == 0
    for s in spans:
        small = kernels.octet_write_paged(lay, q[s], q[s], slots[s], pages[1], rotary=r, positions=pos[s],
                                          query=q[s])
        assert torch.equal(out[s], small)
    assert torch.equal(pages[0], pages[1])


# ------------------------------------------------------------------------------------- store
class Store:
    """An 8-bit store of requests of `lens` tokens in a shuffled paged cache, written by the kernel
    (whose bytes have their own test); slots that no token has hold 0xff (NaN codes, exponents that no
    write leaves)."""

    def __init__(self, lens, H, d=128, block=16, seed=0, pad=0, scale=1.0, dtype=torch.float16):
        self.lens, self.H, self.d, self.block = list(lens), H, d, block
        self.lay = OctetLayout(H, d)
        self.stride = self.lay.compressed_bytes_per_token() + pad
        bt, self.blocks = synth.shuffled_block_table([max(n, 1) for n in lens], block, seed=seed,
                                                     extra_blocks=3)
        self.bt = bt.cuda()
        self.page = torch.full((self.blocks, block, self.stride), 255, dtype=torch.uint8,
                               device="cuda")
        g = _gen(seed)
        n = sum(lens)
        k = torch.randn(n, H, d, generator=g)
        k[..., :8] *= 4
        v = torch.randn(n, H, d, generator=g)
        if torch.is_tensor(scale):
            scale = scale[:n].reshape(n, 1, 1)
        self.k, self.v = k.to(dtype), (v * scale).to(dtype)
        self.slots = torch.cat([on.table_slots(bt[r], m, block) for r, m in enumerate(lens)]
                               + [torch.zeros(0, dtype=torch.int64)])
        err = _err()
        kernels.octet_write_paged(self.lay, self.k.cuda(), self.v.cuda(), self.slots.cuda(),
                                  self.page, error_word=err)
        assert int(err) == 0
        self.seq = _i32(self.lens)

    def kv(self, r):
        at = sum(self.lens[:r])
        s = slice(at, at + self.lens[r])
        return oo.values(self.k[s]), oo.values(self.v[s])


# -------------------------------------------------------------------------------------- read
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,H,block,pad", [(64, 3, 16, 0), (128, 2, 32, 16), (256, 1, 48, 0),
                                           (128, 5, 64, 3)])
def test_read_rows(dtype, d, H, block, pad):
    """Whole requests, none, single tokens and parts from any token; rows between and behind left."""
    st = Store([1, 0, 47, 16, 130, 33], H, d, block, seed=d, pad=pad)
    first = [0, 0, 5, 0, 17, 31]
    starts = [2, 3, 3, 45, 61, 174, 176]                    # rows 0, 1 and those past 176: nobody's
    out = [torch.full((180, H, d), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    err = _err()
    got = kernels.octet_read_paged(st.lay, st.page, block, st.bt, _i32(starts), max(st.lens),
                                   first=_i32(first), key_out=out[0], value_out=out[1], error_word=err)
    assert int(err) == 0 and got[0] is out[0]
    want = torch.full((2, 180, H, d), 7.0).double()
    for r in range(6):
        for i, x in enumerate(st.kv(r)):
            m = starts[r + 1] - starts[r]
            want[i, starts[r]:starts[r + 1]] = x[first[r]:first[r] + m]
    for i in (0, 1):
        assert torch.equal(out[i].cpu(), want[i].to(dtype))


@pytest.mark.parametrize("H,d", [(1, 64), (3, 128)])
def test_read_many_requests(H, d):
    """More requests than a wave looks at together, many of them empty; heads that share no wave evenly."""
    lens = [(7 * i) % 53 if i % 3 else 0 for i in range(200)]
    st = Store(lens, H, d, seed=4)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    k, v = kernels.octet_read_paged(st.lay, st.page, 16, st.bt, _i32(starts), max(lens), num_rows=starts[-1])
    assert torch.equal(k.cpu().double(), oo.values(st.k)) and torch.equal(v.cpu().double(), oo.values(st.v))
    # two requests that name the same rows, more than the rows' own number: in bounds, and one of them is there
    err = _err()
    k, _ = kernels.octet_read_paged(st.lay, st.page, 16, st.bt[[1, 2, 4]], _i32([0, 7, 0, 14]), 53, num_rows=14,
                                    error_word=err)
    assert int(err) == 8
    assert torch.equal(k[7:].cpu().double(), st.kv(4)[0][7:14])


def test_read_rows_that_two_requests_name():
    """Each head's row is one request's or the other's as a whole; rows past them are the second's."""
    st = Store([9, 20], 3, 128, seed=4)
    k, v = kernels.octet_read_paged(st.lay, st.page, 16, st.bt[[0, 1, 1]], _i32([0, 7, 0, 14]), 20, num_rows=14)
    for x, i in ((k.cpu().double(), 0), (v.cpu().double(), 1)):
        one, two = ((x[:7] == st.kv(r)[i][:7]).all(-1) for r in (0, 1))
        assert bool((one | two).all()) and torch.equal(x[7:], st.kv(1)[i][7:14])


def test_read_strides_and_defaults():
    st = Store([70, 5], 2, 128)
    k, v = kernels.octet_read_paged(st.lay, st.page, 16, st.bt, _i32([0, 70, 75]), 70, num_rows=75)
    assert k.dtype == torch.bfloat16
    want = [torch.cat(x) for x in zip(st.kv(0), st.kv(1))]
    assert torch.equal(k.cpu().double(), want[0]) and torch.equal(v.cpu().double(), want[1])
    both = torch.full((75, 2, 2, 128), 3.0, dtype=torch.float16, device="cuda")   # rows of k | v
    kernels.octet_read_paged(st.lay, st.page, 16, st.bt, _i32([0, 70, 75]), 70, key_out=both[:, 0],
                             value_out=both[:, 1])
    assert torch.equal(both.cpu()[:, 0], want[0].half()) and torch.equal(both.cpu()[:, 1], want[1].half())
    odd = torch.full((75 * 259 + 1,), 3.0, dtype=torch.float16, device="cuda")    # unaligned rows
    ko = odd[1:].as_strided((75, 2, 128), (259, 128, 1))
    kernels.octet_read_paged(st.lay, st.page, 16, st.bt, _i32([0, 70, 75]), 70, key_out=ko,
                             value_out=both[:, 1])
    assert torch.equal(ko.cpu(), want[0].half())
    assert float(odd[0]) == 3.0 and bool((odd[1:].reshape(75, 259)[:, 256:] == 3.0).all())
    huge = Store([20], 1, 64, scale=torch.full((20,), 1e30), dtype=torch.float32)
    _, v = kernels.octet_read_paged(huge.lay, huge.page, 16, huge.bt, _i32([0, 20]), 20, num_rows=20,
                                    dtype=torch.float16)
    assert torch.equal(v.cpu(), huge.kv(0)[1].half())        # beyond fp16: infinite


def test_read_refused_places():
    """Tokens past max_seq_len or before 0, blocks outside the cache, rows outside the output."""
    st = Store([40, 40, 40], 1, 64)
    bt = st.bt.clone()
    bt[1, 1] = st.blocks
    out = [torch.full((100, 1, 64), 7.0, device="cuda") for _ in range(2)]
    err = _err()
    kernels.octet_read_paged(st.lay, st.page, 16, bt, _i32([0, 40, 80, 200]), 40, key_out=out[0],
                             value_out=out[1], error_word=err)
    assert int(err) == 2 | 8
    k = out[0].cpu().double()
    assert torch.equal(k[:40], st.kv(0)[0])
    assert torch.equal(k[40:56], st.kv(1)[0][:16]) and bool(torch.isnan(k[56:72]).all())
    assert torch.equal(k[72:80], st.kv(1)[0][32:]) and torch.equal(k[80:100], st.kv(2)[0][:20])
    for first, starts, nan in ((-3, [0, 8], 3), (36, [0, 8], 4)):
        err = _err()
        k, _ = kernels.octet_read_paged(st.lay, st.page, 16, st.bt[:1], _i32(starts), 40,
                                        first=_i32([first]), num_rows=8, error_word=err)
        assert int(err) == 8 and int(torch.isnan(k[:, 0, 0]).sum()) == nan
    err = _err()
    out[0].fill_(7.0)
    kernels.octet_read_paged(st.lay, st.page, 16, st.bt[:1], _i32([-5, 10]), 40, key_out=out[0],
                             value_out=out[1], error_word=err)
    assert int(err) == 8
    assert torch.equal(out[0][:10].cpu().double(), st.kv(0)[0][5:15]) and bool((out[0][10:] == 7).all())


@pytest.mark.parametrize("starts,rows", [
    ([-2 ** 31, -2 ** 31 + 1], (0, 0)), ([-2 ** 31, -5], (0, 0)), ([-2 ** 31, 3], (0, 3)),
    ([3, -2 ** 31], (0, 0)), ([2 ** 31 - 1, -5], (0, 0)), ([5, 2 ** 31 - 1], (5, 8)),
    ([2 ** 30, 2 ** 31 - 1], (0, 0)), ([-2 ** 31, 2 ** 31 - 1], (0, 8))])
def test_read_row_starts_at_the_ends_of_their_type(starts, rows):
    """Only rows of the outputs are written; of tokens past the call's lengths, as NaN."""
    st = Store([40], 1, 64)
    out = [torch.full((24, 1, 64), 7.0, device="cuda") for _ in range(2)]
    err = _err()
    kernels.octet_read_paged(st.lay, st.page, 16, st.bt, _i32(starts), 40, key_out=out[0][8:16],
                             value_out=out[1][8:16], error_word=err)
    assert int(err) == 8
    lo, hi = rows
    for x, kept in zip(out, st.kv(0)):
        got = x[8:16].cpu()
        assert bool((x[:8] == 7).all()) and bool((x[16:] == 7).all())
        assert bool((got[:lo] == 7).all()) and bool((got[hi:] == 7).all())
        if starts[0] >= 0:
            assert torch.equal(got[lo:hi].double(), kept[:hi - lo])
        else:
            assert bool(torch.isnan(got[lo:hi]).all())


# ------------------------------------------------------------------------------------ decode
def _close(got, lse, q, K, V, scale, what, **kw):
    want, wlse, spread, score = oo.attend(q, K, V, scale, **kw)
    half, n, d = HALF[got.dtype], K.shape[0], q.shape[2]
    vmax = float(V.abs().max()) if n else 0.0
    adds = (n / 4 + 64) * 2.0 ** -23
    tol = 1.05 * (half * want.abs() + (2.0 ** -18 + 2 * d * 2.0 ** -24 * score + adds) * spread) \
        + 2.0 ** -25 * (1 + vmax)
    e = (got.cpu().double() - want).abs()
    assert bool((e <= tol).all()), (what, float(e.max()), float((e / tol).max()))
    if lse is None:
        return
    lse = lse.cpu().double()
    empty = torch.isinf(wlse)
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all()), what
    tol = 1.05 * (2 * d * 2.0 ** -24 * score[..., 0] + adds + 2.0 ** -22 * (1 + wlse.abs()))
    assert bool(((lse - wlse).abs() <= tol)[~empty].all()), what


def _decode(st, q, counts=None, **kw):
    err = _err()
    counts = [1] * len(st.lens) if counts is None else counts
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    kw.setdefault("max_seq_len", max(st.lens))
    out = kernels.octet_decode_paged(st.lay, q, st.page, st.block, st.bt, st.seq, _i32(at),
                                     kw.pop("max_q_len", max(counts + [1])), kw.pop("max_seq_len"),
                                     st.d ** -0.5, error_word=err, **kw)
    torch.cuda.synchronize()
    return out, int(err), at


def _check(st, q, counts, out, lse, at, **kw):
    for r in range(len(st.lens)):
        rows = slice(at[r], at[r + 1])
        _close(out[rows], None if lse is None else lse[rows], q[rows].cpu(), *st.kv(r), st.d ** -0.5,
               (r, st.lens[r], kw), **kw)


LENS = [1, 15, 16, 17, 0, 31, 32, 33, 64, 97, 128, 129, 300]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,G,block", [(128, 2, 1, 16), (128, 1, 4, 32), (64, 3, 8, 16), (256, 2, 2, 48),
                                         (64, 1, 16, 64), (128, 3, 5, 16), (256, 1, 3, 16), (128, 8, 4, 16)])
def test_decode_lengths(dtype, d, H, G, block):
    st = Store(LENS, H, d, block, seed=G, dtype=dtype)
    q = torch.randn(len(LENS) + 2, H * G, d, generator=_gen(G)).to(dtype).cuda()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    _, err, at = _decode(st, q, out=out, lse=lse)
    assert err == 0
    _check(st, q, None, out, lse, at)
    assert bool((out[len(LENS):] == 7).all()) and bool((lse[len(LENS):] == 7).all())
    assert bool((out[4] == 0).all())


@pytest.mark.parametrize("d,H,G", [(64, 2, 8), (128, 2, 4), (256, 1, 2)])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 32, 33, 100, 299, 300, 2 ** 40])
def test_decode_windows_and_sinks(d, H, G, window):
    st = Store(LENS, H, d, seed=3, dtype=torch.bfloat16)
    g = _gen(window % 1000)
    q = torch.randn(len(LENS), H * G, d, generator=g).bfloat16().cuda()
    sinks = torch.randn(H * G, generator=g) * 3
    sinks[0], sinks[-1] = -math.inf, 60.0
    for s in (None, sinks):
        lse = torch.zeros(q.shape[:2], device="cuda")
        out, err, at = _decode(st, q, window=window, sinks=None if s is None else s.cuda(), lse=lse)
        assert err == 0
        _check(st, q, None, out, lse, at, window=window, sinks=s)


@pytest.mark.parametrize("d,H,G", [(64, 1, 4), (128, 2, 3), (256, 2, 1), (128, 1, 16)])
@pytest.mark.parametrize("window", [0, 5, 40])
def test_decode_drafts(d, H, G, window):
    """Chunks of 1 to 16 queries and waiting requests in one call."""
    counts = [1, 15, 0, 2, 0, 5, 16, 16, 3, 0, 7, 1, 16]
    st = Store(LENS, H, d, seed=5)
    q = torch.randn(sum(counts) + 1, H * G, d, generator=_gen(7)).half().cuda()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    _, err, at = _decode(st, q, counts, out=out, lse=lse, window=window)
    assert err == 0
    _check(st, q, counts, out, lse, at, window=window)
    assert bool((out[-1] == 7).all())


@pytest.mark.parametrize("d,H,G,lens", [(128, 8, 4, [5000]), (128, 1, 8, [9000, 3]), (64, 2, 8, [3000] * 9),
                                        (256, 1, 16, [2500, 700]), (128, 2, 4, [1, 2000, 40] * 30)])
def test_decode_long(d, H, G, lens):
    """Requests whose keys several workgroups share, ragged, at a large and a small batch."""
    st = Store(lens, H, d, 32, seed=9, dtype=torch.bfloat16)
    q = torch.randn(len(lens), H * G, d, generator=_gen(1)).bfloat16().cuda()
    lse = torch.zeros(q.shape[:2], device="cuda")
    out, err, at = _decode(st, q, lse=lse)
    assert err == 0
    _check(st, q, None, out, lse, at)
    again, _, _ = _decode(st, q)
    assert torch.equal(again, out)                       # bit for bit
    counts = [min(n, 3) for n in lens]
    q = torch.randn(sum(counts), H * G, d, generator=_gen(2)).bfloat16().cuda()
    out, err, at = _decode(st, q, counts, window=1500)
    assert err == 0
    _check(st, q, counts, out, None, at, window=1500)


@pytest.mark.parametrize("d,H,G,R", [(64, 8, 4, 36), (128, 8, 4, 36), (256, 4, 3, 44)])
@pytest.mark.parametrize("window", [0, 30])
def test_decode_drafts_of_large_batches(d, H, G, R, window):
    """More than 16 rows per KV head in batches that share a block's keys between two groups of rows; a
    NaN in a value stays with the rows that see it."""
    g = _gen(d + window)
    lens = [8 + int(torch.randint(0, 150, (1,), generator=g)) for _ in range(R)]
    st = Store(lens, H, d, seed=6, dtype=torch.bfloat16)
    v = st.v.clone()
    sick = sum(lens[:5]) + lens[5] - 4                     # the fourth last token of request 5
    v[sick, H - 1, d - 1] = float("nan")
    kernels.octet_write_paged(st.lay, st.k.cuda(), v.cuda(), st.slots.cuda(), st.page)
    counts = [8 if i % 4 else 5 + i % 3 for i in range(R)]
    q = torch.randn(sum(counts), H * G, d, generator=g).bfloat16().cuda()
    lse = torch.zeros(q.shape[:2], device="cuda")
    out, err, at = _decode(st, q, counts, max_q_len=8, lse=lse, window=window)
    assert err == 0
    last, heads = counts[5] - 4, slice((H - 1) * G, H * G)
    sees = out[at[5]:at[6]][last:, heads]                  # the queries from that token's on
    assert bool(torch.isnan(sees[..., d - 32:]).all()) and bool(torch.isfinite(sees[..., :d - 32]).all())
    for r in range(R):
        rows = slice(at[r], at[r + 1])
        if r == 5:
            rows = slice(at[5], at[5] + last)
            K, V = (x[:lens[5] - 4] for x in st.kv(5))
            _close(out[rows], lse[rows], q[rows].cpu(), K, V, d ** -0.5, r, window=window)
        else:
            _close(out[rows], lse[rows], q[rows].cpu(), *st.kv(r), d ** -0.5, r, window=window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,G,Q,R,window", [(128, 8, 8, 5, 24, 0), (64, 8, 8, 8, 20, 0), (128, 4, 16, 3, 48, 9),
                                              (256, 4, 12, 4, 24, 0), (64, 2, 16, 16, 20, 25)])
def test_decode_drafts_of_several_blocks_in_large_batches(d, H, G, Q, R, window, dtype):
    """More than 32 rows per KV head in batches that give a block two groups of rows: blocks that are partly
    filled, requests of fewer queries and waiting ones, keys that are split and that are not."""
    g = _gen(d + Q)
    assert G * Q > 32 and R * H * -(-G * Q // 16) > (256 if d == 256 else 512)
    lens = [Q + int(torch.randint(0, 120, (1,), generator=g)) for _ in range(R)]
    lens[3] = 900
    st = Store(lens, H, d, 32, seed=4, dtype=dtype)
    counts = [Q if i % 3 else i // 3 % (Q + 1) for i in range(R)]
    q = torch.randn(sum(counts) + 1, H * G, d, generator=g).to(dtype).cuda()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    _, err, at = _decode(st, q, counts, max_q_len=Q, out=out, lse=lse, window=window)
    assert err == 0
    _check(st, q, counts, out, lse, at, window=window)
    assert bool((out[-1] == 7).all()) and bool((lse[-1] == 7).all())


@pytest.mark.parametrize("d,R", [(64, 150), (128, 140)])
def test_decode_batches_beyond_the_counters(d, R):
    """8 KV heads of 16 query heads and 16 drafts: more (block, head) pairs than counters, so several launches."""
    g = _gen(R)
    lens = [1 + int(torch.randint(0, 40, (1,), generator=g)) for _ in range(R)]
    lens[R - 2], lens[2] = 600, 500
    counts = [min(n, 16 if i % 9 == 0 else 1 + i % 2) for i, n in enumerate(lens)]
    st = Store(lens, 8, d, seed=5)
    q = torch.randn(sum(counts), 128, d, generator=g).half().cuda()
    ws = kernels.octet_decode_workspace(st.lay, 128, R, 16, 600, "cuda")
    out, err, at = _decode(st, q, counts, max_q_len=16, workspace=ws)
    assert err == 0 and bool((ws[:65536] == 0).all())
    _check(st, q, counts, out, None, at)


@pytest.mark.parametrize("d,H,R,window,Q", [(64, 8, 24, 0, 1), (128, 8, 24, 0, 1), (64, 8, 32, 640, 2),
                                            (128, 8, 21, 600, 3), (128, 4, 60, 0, 1)])
def test_decode_pairs_that_fill_the_chip(d, H, R, window, Q):
    """About as many (request, KV head) pairs as compute units, keys of a middle length."""
    g = _gen(R)
    lens = [int(torch.randint(3, 900 if R < 40 else 700, (1,), generator=g)) for _ in range(R)]
    lens[1] = 1700
    st = Store(lens, H, d, 32, seed=6, dtype=torch.float16)
    q = torch.randn(R * Q, H * 3, d, generator=g).half().cuda()
    sinks = torch.randn(H * 3, generator=g)
    lse = torch.zeros(q.shape[:2], device="cuda")
    out, err, at = _decode(st, q, [Q] * R, lse=lse, window=window, sinks=sinks.cuda())
    assert err == 0
    _check(st, q, None, out, lse, at, window=window, sinks=sinks)


def test_decode_many_requests():
    """More requests than one launch plans for, some of them waiting, one per group long."""
    lens = [1 + 7 * i % 90 for i in range(600)]
    lens[100], lens[400] = 900, 1200
    st = Store(lens, 2, 64, seed=2)
    counts = [0 if i % 5 == 3 else 1 + i % 2 * (lens[i] > 1) for i in range(600)]
    q = torch.randn(sum(counts), 4, 64, generator=_gen(3)).half().cuda()
    out, err, at = _decode(st, q, counts)
    assert err == 0
    _check(st, q, counts, out, None, at)


@pytest.mark.parametrize("factor", [2.0 ** -60, 1e-3, 300.0, 1e18])
def test_decode_scores_and_values_of_any_size(factor):
    """Scores far from 0 and values of any size; every key the same weight at a scale of 0."""
    st = Store([77], 1, 128, seed=4, dtype=torch.float32,
               scale=torch.full((77,), 1.0 if factor < 1 else factor))
    q = torch.randn(1, 4, 128, generator=_gen(5)).bfloat16()
    q = (q.float() * (factor if factor < 1 else min(factor, 300.0))).bfloat16().cuda()
    out, err, at = _decode(st, q)
    assert err == 0
    _check(st, q, None, out, None, at)
    for scale in (0.0, -0.3):
        got = kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, _i32([0, 1]), 1, 77, scale)
        _close(got, None, q.cpu(), *st.kv(0), scale, scale)


def _cancelling(d, H, n, Q, seed):
    """Whole-number keys [n, H, d] and a query [H, d], whose scores are exact in 32 bits, with values of 8 to 15
    in size whose weighted sum nearly cancels for the last of Q queries: (q, k, v)."""
    g = _gen(seed)
    q, k = (torch.randint(-1, 2, s, generator=g).float() for s in ((H, d), (n, H, d)))
    v = torch.empty(n, H, d)
    for h in range(H):
        s = (k[:, h] @ q[h]).double() / 64
        assert float(s.abs().max()) <= 1
        tries = torch.randint(8, 16, (n, 40000), generator=g) * (2 * torch.randint(0, 2, (n, 40000), generator=g) - 1)
        left = (torch.softmax(s, 0) @ tries.double()).abs()
        v[:, h] = tries[:, left.argsort()[:d]].float()
    return q, k, v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,H,G,Q,R", [(64, 4, 1, 1, 3), (128, 4, 4, 1, 3), (256, 4, 2, 1, 3), (64, 2, 16, 2, 130),
                                       (128, 2, 6, 3, 130), (256, 2, 4, 5, 65), (256, 1, 16, 3, 2)])
def test_decode_weights_are_not_rounded_to_fewer_bits(d, H, G, Q, R, dtype):
    """Where values cancel, an output shows what its softmax weights are off by. In units of 2^-24 of the
    spread sum p |v|: a score's product with the scale and that scale's own rounding, at most 1.5 after the
    exponential; its difference to the maximum, at most 2 in size, 1.4; the exponential 2; the additions of six
    products in three parts 8: 12.9 in all, 2^-20.3. The sum of weights and the division scale what is left of
    the values. Weights of 16 bits are off by up to 2^-18 each and fail here (2^-18.7 of the spread)."""
    n = 6
    q, k, v = _cancelling(d, H, n, Q, d + G)
    st = Store([n] * R, H, d, seed=1)
    st.k, st.v = k.half().repeat(R, 1, 1), v.half().repeat(R, 1, 1)
    kernels.octet_write_paged(st.lay, st.k.cuda(), st.v.cuda(), st.slots.cuda(), st.page)
    rows = q.repeat_interleave(G, 0).to(dtype).repeat(R * Q, 1, 1).cuda()
    err, at = _err(), _i32([Q * r for r in range(R + 1)])
    out = kernels.octet_decode_paged(st.lay, rows, st.page, st.block, st.bt, st.seq, at, Q, n, 1 / 64,
                                     out=torch.empty_like(rows, dtype=torch.float16), error_word=err)
    assert int(err) == 0
    want, _, spread, _ = oo.attend(rows[:Q].cpu(), *st.kv(0), 1 / 64)
    last = want[-1].abs()
    assert float((last / spread[-1]).max()) < 2.0 ** -7                  # (they do cancel)
    tol = 2.0 ** -20.25 * spread + 2.0 ** -11 * want.abs() + 2.0 ** -25
    e = (out.cpu().double().reshape(R, Q, H * G, d) - want).abs()
    assert bool((e <= tol).all()), (float((e / spread).max()), float((e / tol).max()))


@pytest.mark.parametrize("d,H,G,n,Q", [(64, 1, 2, 40, 1), (128, 2, 4, 40, 3), (256, 1, 3, 70, 1), (64, 1, 16, 50, 2),
                                       (128, 1, 2, 3000, 1), (256, 2, 2, 2500, 2)])
@pytest.mark.parametrize("sinks", [False, True])
def test_decode_scores_beyond_their_type(d, H, G, n, Q, sinks):
    """Scores of +-2^130 in size: one above the type makes its row NaN, those below weigh nothing, and a row
    that has no other is NaN, or its sink's."""
    g = _gen(n + d)
    for some in (-1.0, 1.0, None):     # the sign of the scores beyond, of about half the keys; None: all, below
        k = torch.randint(-2, 3, (n, H, d), generator=g).float()
        v = torch.randint(-8, 9, (n, H, d), generator=g).float()
        k[..., :32] = 0
        k[..., 0] = torch.where(torch.rand(n, H, generator=g) < 0.5, 2.0 ** 30, 0.0)
        k[n // 2, :, 0] = 2.0 ** 30
        if some is None:
            k[..., 0] = 2.0 ** 30
        st = Store([n], H, d, seed=2)
        st.k, st.v = k, v
        kernels.octet_write_paged(st.lay, k.cuda(), v.cuda(), st.slots.cuda(), st.page)
        assert torch.equal(st.kv(0)[0], k.double())
        q = torch.randint(-1, 2, (Q, H * G, d), generator=g).float()
        q[..., 0] = (some or -1.0) * 2.0 ** 100
        q = q.bfloat16().cuda()
        s = (torch.arange(H * G).float() / 4).cuda() if sinks else None
        lse = torch.full((Q, H * G), 7.0, device="cuda")
        out, err, _ = _decode(st, q, [Q], sinks=s, lse=lse)
        assert err == 0
        if some == 1.0:
            assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())
        elif some is None and not sinks:
            assert bool(torch.isnan(out).all()) and bool(torch.isnan(lse).all())
        elif some is None:
            assert bool((out == 0).all())
            assert bool(((lse - s).abs() <= 2.0 ** -22 * (1 + s)).all())
        else:
            plain = q.clone()
            plain[..., 0] = 0
            for h in range(H):
                kept, heads = k[:, h, 0] == 0, slice(h * G, h * G + G)
                for j in range(Q):
                    seen = kept & (torch.arange(n) <= n - Q + j)
                    _close(out[j:j + 1, heads], lse[j:j + 1, heads], plain[j:j + 1, heads].cpu(),
                           k[seen, h:h + 1].double(), v[seen, h:h + 1].double(), d ** -0.5, (h, j),
                           sinks=s if s is None else s[heads].cpu())


@pytest.mark.parametrize("size", [1e4, 2.0 ** 100, 2.0 ** 127])
def test_decode_sinks_of_any_size(size):
    """A large sink takes all the weight, a low one none; an empty request's lse is its sink."""
    st = Store([40, 0], 1, 64, seed=3)
    q = torch.randn(2, 4, 64, generator=_gen(3)).half().cuda()
    sinks, lse = torch.tensor([size, -size, -math.inf, 0.0]), torch.zeros(2, 4, device="cuda")
    out, err, _ = _decode(st, q, sinks=sinks.cuda(), lse=lse)
    assert err == 0
    _close(out[:1, 1:], lse[:1, 1:], q[:1, 1:].cpu(), *st.kv(0), 0.125, "low", sinks=sinks[1:])
    assert bool((out[0, 0] == 0).all()) and bool((out[1] == 0).all())
    assert float(lse[1, 2]) == -math.inf
    got, want = torch.cat([lse[:1, 0], lse[1, [0, 1, 3]]]).cpu().double(), sinks[[0, 0, 1, 3]].double()
    assert bool(((got - want).abs() <= 2.0 ** -22 * want.abs()).all()), got


def test_decode_bad_blocks_and_lengths():
    st = Store([40, 40, 40, 40, 2], 2, 128)
    bt = st.bt.clone()
    bt[1, 1], bt[2, 0] = st.blocks, -1
    q = torch.randn(8, 4, 128, generator=_gen(1)).half().cuda()
    out, err = torch.full_like(q, 7.0), _err()
    # five requests of one query, but the last of four over its two keys
    kernels.octet_decode_paged(st.lay, q, st.page, 16, bt, st.seq, _i32([0, 1, 2, 3, 4, 8]), 4, 40,
                               128 ** -0.5, out=out, error_word=err)
    assert int(err) == 2 | 8
    assert bool(torch.isnan(out[[1, 2, 4, 5, 6, 7]]).all())
    for r in (0, 3):
        _close(out[r:r + 1], None, q[r:r + 1].cpu(), *st.kv(r), 128 ** -0.5, r)
    # a bad block outside a window is not read
    err = _err()
    got = kernels.octet_decode_paged(st.lay, q[:1], st.page, 16, bt[2:3], st.seq[2:3], _i32([0, 1]), 1, 40,
                                     128 ** -0.5, window=20, error_word=err)
    assert int(err) == 0
    _close(got, None, q[:1].cpu(), *st.kv(2), 128 ** -0.5, "window", window=20)


def test_decode_lengths_beyond_the_call():
    """Clamped, and said so: keys past max_seq_len, queries past max_q_len, rows outside the query."""
    st = Store([50, 20], 1, 64)
    q = torch.randn(5, 2, 64, generator=_gen(1)).half().cuda()
    out, err = torch.full_like(q, 7.0), _err()
    kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, _i32([0, 1, 2]), 1, 32, 0.125, out=out,
                               error_word=err)
    assert int(err) == 8
    K, V = st.kv(0)
    _close(out[:1], None, q[:1].cpu(), K[:32], V[:32], 0.125, "clamped")
    _close(out[1:2], None, q[1:2].cpu(), *st.kv(1), 0.125, "whole")
    assert bool((out[2:] == 7).all())
    out, err = torch.full_like(q, 7.0), _err()
    kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, _i32([0, 4, 5]), 2, 50, 0.125, out=out,
                               error_word=err)
    assert int(err) == 8
    want = oo.attend(q[:4].cpu(), K, V, 0.125)[0]
    assert float((out[:2].cpu().double() - want[:2]).abs().max()) < 2e-3
    assert bool((out[2:4] == 7).all())
    _close(out[4:], None, q[4:].cpu(), *st.kv(1), 0.125, "last")
    out, err = torch.full_like(q, 7.0), _err()
    kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, _i32([-1, 1, 7]), 6, 50, 0.125, out=out,
                               error_word=err)
    assert int(err) == 8 and bool((out[0] != 7).all()) and bool((out[1:] != 7).all())
    err = _err()
    neg = _i32([-5, 20])
    got = kernels.octet_decode_paged(st.lay, q[:2], st.page, 16, st.bt, neg, _i32([0, 1, 2]), 1, 50, 0.125,
                                     error_word=err)
    assert bool((got[0] == 0).all())


def test_decode_rows_partly_outside_the_query():
    """Of a request whose rows begin before the query's or end behind them, those inside are its own."""
    st = Store([50, 20], 1, 64)
    q = torch.randn(5, 2, 64, generator=_gen(1)).half().cuda()
    for window in (0, 7):
        out, err = torch.full_like(q, 7.0), _err()
        kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, _i32([-1, 1, 7]), 6, 50, 0.125,
                                   window=window, out=out, error_word=err)
        assert int(err) == 8
        # row 0 is the second of request 0's two queries, rows 1 .. 4 the first of request 1's six
        K, V = st.kv(0)
        _close(out[:1], None, q[:1].cpu(), K, V, 0.125, "second of two", window=window)
        K, V = st.kv(1)
        _close(out[1:], None, q[1:].cpu(), K[:18], V[:18], 0.125, "four of six", window=window)


@pytest.mark.parametrize("R", [3, 300])
def test_decode_negative_lengths_and_falling_starts(R):
    """Said so; a length below 0 counts as none, starts that fall as a request that waits."""
    st = Store([20] * R, 1, 64)
    q = torch.randn(R, 2, 64, generator=_gen(2)).half().cuda()
    for r in (0, R - 1):
        seq, err, out = st.seq.clone(), _err(), torch.full_like(q, 7.0)
        seq[r] = -2 ** 31 if r else -5
        lse = torch.full((R, 2), 7.0, device="cuda")
        starts = torch.arange(R + 1, dtype=torch.int32, device="cuda")
        kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, seq, starts, 1, 20, 0.125, out=out, lse=lse,
                                   error_word=err)
        assert int(err) == 8
        assert bool((out[r] == 0).all()) and bool((lse[r] == -math.inf).all())
        for i in {0, 1, R - 2, R - 1} - {r}:
            _close(out[i:i + 1], lse[i:i + 1], q[i:i + 1].cpu(), *st.kv(i), 0.125, i)
    # queries of row i + 1 for request i; request R - 2's end before they begin, the last one's is row 0 or none
    for low in (0, -2 ** 31):
        starts, err, out = torch.arange(1, R + 2, dtype=torch.int32, device="cuda"), _err(), torch.full_like(q, 7.0)
        starts[R - 1], starts[R] = low, low + 1
        kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, starts, 1, 20, 0.125, out=out,
                                   error_word=err)
        assert int(err) == 8
        for i in {0, R - 3}:
            _close(out[i + 1:i + 2], None, q[i + 1:i + 2].cpu(), *st.kv(i), 0.125, i)
        if low == 0:
            _close(out[:1], None, q[:1].cpu(), *st.kv(R - 1), 0.125, "last")
        assert bool((out[R - 1:] == 7).all()) and (low == 0 or bool((out[0] == 7).all()))
    # from one end of the type to the other: more than max_q_len, all of its first ones outside
    err, out = _err(), torch.full_like(q, 7.0)
    kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt[:1], st.seq[:1], _i32([-2 ** 31, 2 ** 31 - 1]), 1, 20,
                               0.125, out=out, error_word=err)
    assert int(err) == 8 and bool((out == 7).all())


def test_decode_nan_keys_stay_with_the_rows_that_see_them():
    """A NaN in a stored key or value reaches the rows that see it; behind the last key, in a draft's
    future or before the window it reaches nobody."""
    lens = [60]
    st = Store(lens, 1, 128, dtype=torch.bfloat16)
    for part in ("k", "v"):
        for at in (10, 55, 58):
            k, v = st.k.clone(), st.v.clone()
            (k if part == "k" else v)[at, 0, 70] = float("nan")
            kernels.octet_write_paged(st.lay, k.cuda(), v.cuda(), st.slots.cuda(), st.page)
            q = torch.randn(4, 4, 128, generator=_gen(at)).bfloat16().cuda()
            K, V = oo.values(k), oo.values(v)
            for window in (0, 8):
                out, err, _ = _decode(st, q, [4], window=window)
                assert err == 0
                for j in range(4):
                    p = 56 + j
                    sees = at <= p and (not window or at > p - window)
                    got = out[j].cpu()
                    if not sees:
                        keep = torch.arange(60) != at
                        n = int(keep[:p + 1].sum())
                        lo = max(0, p - window + 1) if window else 0
                        span = torch.arange(lo, p + 1)
                        span = span[span != at]
                        assert n and bool(torch.isfinite(got).all())
                        _close(out[j:j + 1], None, q[j:j + 1].cpu(), K[span], V[span], 128 ** -0.5, (at, j))
                    elif part == "k":
                        assert bool(torch.isnan(got).all())
                    else:
                        assert bool(torch.isnan(got[:, 64:96]).all())
                        assert bool(torch.isfinite(got[:, :64]).all() and torch.isfinite(got[:, 96:]).all())


def test_decode_out_types_strides_and_in_place():
    st = Store([100, 37], 2, 128, pad=24)
    g = _gen(6)
    base = torch.randn(2, 3, 8, 128, generator=g).half().cuda()
    q = base[:, 1]                                             # rows at three times their length
    want, err, at = _decode(st, q.contiguous())
    assert err == 0
    _check(st, q, None, want, None, at)
    bf, _, _ = _decode(st, q, out=torch.empty(2, 8, 128, dtype=torch.bfloat16, device="cuda"))
    _check(st, q, None, bf, None, at)
    wide = torch.full((2, 2, 8, 128), 7.0, dtype=torch.float16, device="cuda")
    _decode(st, q, out=wide[:, 1])
    assert torch.equal(wide[:, 1], want) and bool((wide[:, 0] == 7).all())
    copy = base.clone()
    _decode(st, copy[:, 1], out=copy[:, 1])
    assert torch.equal(copy[:, 1], want) and torch.equal(copy[:, 0], base[:, 0])


def test_decode_far_pages():
    """Blocks whose bytes lie beyond 2^32 of the page's start."""
    st = Store([70], 2, 128, block=32)
    blocks = (5 << 30) // (32 * st.stride)
    page = torch.empty(blocks, 32, st.stride, dtype=torch.uint8, device="cuda")
    bt = torch.tensor([[blocks - 1, 3, blocks - 7]], dtype=torch.int32, device="cuda")
    slots = on.table_slots(bt[0].cpu(), 70, 32)
    r = scaled_rotary(128, device="cuda")
    kernels.octet_write_paged(st.lay, st.k.cuda(), st.v.cuda(), slots.cuda(), page)
    q = torch.randn(1, 8, 128, generator=_gen(2)).half().cuda()
    err = _err()
    out = kernels.octet_decode_paged(st.lay, q, page, 32, bt, st.seq, _i32([0, 1]), 1, 70, 128 ** -0.5,
                                     error_word=err)
    assert int(err) == 0
    _close(out, None, q.cpu(), *st.kv(0), 128 ** -0.5, "far")
    k, v = kernels.octet_read_paged(st.lay, page, 32, bt, _i32([0, 70]), 70, num_rows=70)
    assert torch.equal(k.cpu().double(), st.kv(0)[0]) and torch.equal(v.cpu().double(), st.kv(0)[1])


def test_workspace_serves_calls_in_turn():
    """One workspace for the largest batch; the counters are left zero whatever the calls."""
    big = Store([3000, 900, 40], 2, 128, seed=1)
    small = Store([5, 700], 4, 64, seed=2)
    ws = kernels.octet_decode_workspace(big.lay, 16, 3, 16, 3000, "cuda")
    for i in range(2):
        for st, HQ, counts in ((big, 8, [1, 1, 1]), (small, 16, [3, 2]), (big, 16, [16, 4, 1])):
            q = torch.randn(sum(counts), HQ, st.d, generator=_gen(i)).half().cuda()
            need = kernels.octet_decode_workspace(st.lay, HQ, len(counts), max(counts), max(st.lens), "cuda")
            assert need.numel() <= ws.numel()
            out, err, at = _decode(st, q, counts, workspace=ws)
            assert err == 0 and bool((ws[:65536] == 0).all())
            _check(st, q, counts, out, None, at)
            ws[65536:] = 255


def test_wrapper_refusals():
    st = Store([20], 2, 64)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    one = _i32([0, 1])
    r = scaled_rotary(32, device="cuda")
    pos = torch.zeros(1, dtype=torch.int64, device="cuda")

    def decode(**kw):
        a = dict(query=q, page=st.page, bt=st.bt, seq=st.seq, qsl=one)
        a.update({k: kw.pop(k) for k in list(kw) if k in a})
        return kernels.octet_decode_paged(st.lay, a["query"], a["page"], 16, a["bt"], a["seq"], a["qsl"],
                                          kw.pop("max_q_len", 1), kw.pop("max_seq_len", 20), 0.1, **kw)

    for kw, text in ((dict(query=q.float()), "dtype"), (dict(query=q[..., :32]), "query must be"),
                     (dict(qsl=one[:1]), "query start"), (dict(seq=st.seq.long()), "int32"),
                     (dict(bt=st.bt[:0]), "block table"), (dict(sinks=torch.zeros(3, device="cuda")), "sinks"),
                     (dict(sinks=torch.zeros(4, device="cuda").half()), "sinks"),
                     (dict(lse=torch.zeros(1, 3, device="cuda")), "lse"),
                     (dict(out=torch.zeros(2, 4, 64, device="cuda").half()), "out"),
                     (dict(page=st.page[:, :, :100].contiguous()), "cache row"), (dict(max_seq_len=1000), "blocks"),
                     (dict(max_q_len=17), "16 queries"), (dict(window=-1), "window"),
                     (dict(workspace=torch.zeros(64, dtype=torch.uint8, device="cuda")), "workspace"),
                     (dict(seq=st.seq.cpu()), "device")):
        with pytest.raises((ValueError, RuntimeError), match=text):
            decode(**kw)
    k = torch.zeros(1, 2, 64, device="cuda")
    for kw, text in ((dict(rotary=r), "positions"), (dict(query=q), "rotary"),
                     (dict(rotary=r, positions=pos.int()), "positions"),
                     (dict(rotary=r._replace(turns=r.turns.float()), positions=pos), "fp64"),
                     (dict(rotary=r._replace(turns=r.turns.cpu()), positions=pos), "device"),
                     (dict(rotary=Rotary(torch.zeros(40, device="cuda").double()), positions=pos), "frequencies"),
                     (dict(query_out=q), "query_out"), (dict(key_out=k), "key_out"),
                     (dict(rotary=r, positions=pos, query=q.double()), "dtype")):
        with pytest.raises((ValueError, RuntimeError), match=text):
            kernels.octet_write_paged(st.lay, k, k, pos, st.page, **kw)
    for kw, text in ((dict(), "num_rows"), (dict(key_out=k, value_out=k.half()), "dtype"),
                     (dict(num_rows=2, dtype=torch.int32), "dtype"), (dict(num_rows=2, first=one[:0]), "first")):
        with pytest.raises(ValueError, match=text):
            kernels.octet_read_paged(st.lay, st.page, 16, st.bt, one, 20, **kw)


def test_wrappers_refuse_numbers_beyond_32_bits():
    """(Cut to 32 bits each of these would be a call that runs.)"""
    st = Store([20], 2, 64)
    q, at = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda"), _i32([0, 1])
    for block, longest, most in ((16, 2 ** 32 + 20, 1), (16, 20, 2 ** 32 + 1), (2 ** 32 + 16, 20, 1), (16, 2 ** 31, 1)):
        with pytest.raises(ValueError, match="2.31"):
            kernels.octet_decode_paged(st.lay, q, st.page, block, st.bt, st.seq, at, most, longest, 0.1)
    for block, longest, rows in ((2 ** 32 + 16, 20, 20), (16, 2 ** 32 + 20, 20), (16, 20, 2 ** 32 + 20)):
        with pytest.raises(ValueError, match="2.31"):
            kernels.octet_read_paged(st.lay, st.page, block, st.bt, _i32([0, 20]), longest, num_rows=rows)
    with pytest.raises(ValueError, match="2.31"):
        kernels.octet_decode_workspace(st.lay, 4, 1, 1, 2 ** 32 + 20, "cuda")
    N = 2 ** 32 + 1                                    # rows that are one row, so no memory
    x, ids = q[:, :2].expand(N, 2, 64), torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="2.31"):
        kernels.rotary_scaled(x, None, ids, scaled_rotary(64, device="cuda"))
    with pytest.raises(ValueError, match="2.31"):
        kernels.octet_write_paged(st.lay, x, x, ids, st.page)


# ----------------------------------------------------------------------------------- together
class Serving:
    """A server's layer over the 8-bit cache: each step plans its addresses, rotates and stores its
    tokens and attends to what is stored, all on the device; the oracle follows in 64 bits."""

    def __init__(self, R, H, G, d, window=0, adjacent=False, seed=0):
        self.R, self.H, self.G, self.d, self.window = R, H, G, d, window
        self.lay = OctetLayout(H, d)
        self.blocks, self.block = 40, 16
        self.page = torch.full((self.blocks, 16, self.lay.compressed_bytes_per_token()), 255,
                               dtype=torch.uint8, device="cuda")
        self.bt = torch.full((R, 12), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(self.blocks, generator=_gen(seed)).int().cuda()
        self.computed = torch.zeros(R, dtype=torch.int32, device="cuda")
        self.r = scaled_rotary(d // 2 if adjacent else d, rule="yarn", factor=16.0, adjacent=adjacent)
        self.dev = self.r._replace(turns=self.r.turns.cuda())
        self.ws = kernels.octet_decode_workspace(self.lay, H * G, R, 16, 192, "cuda")
        self.err = _err()

    def step(self, counts, tokens, q, k, v, out, lse=None):
        plan = kernels.step_plan(self.computed, counts, self.bt, self.free, self.block, self.blocks, tokens,
                                 error_word=self.err)
        qr = kernels.octet_write_paged(self.lay, k, v, plan.slot_mapping, self.page, rotary=self.dev,
                                       positions=plan.positions, query=q, error_word=self.err)
        kernels.octet_decode_paged(self.lay, qr, self.page, self.block, self.bt, plan.seq_lens,
                                   plan.query_start_loc, 16, 192, self.d ** -0.5, window=self.window, out=out,
                                   lse=lse, workspace=self.ws, error_word=self.err)
        return plan, qr


@pytest.mark.parametrize("d,window,adjacent", [(64, 0, True), (128, 24, False), (256, 0, False)])
def test_a_run_of_them_together(d, window, adjacent):
    R, H, G = 4, 2, 3
    s = Serving(R, H, G, d, window, adjacent)
    g = _gen(d)
    stored = [([], []) for _ in range(R)]
    for counts in ([16, 3, 0, 1], [1, 16, 9, 2], [1, 1, 1, 1], [4, 0, 16, 1]) * 2:
        n, T = sum(counts), 40
        q, k, v = (torch.randn(T, h, d, generator=g).bfloat16().cuda() for h in (H * G, H, H))
        out = torch.full_like(q, 7.0)
        plan, qr = s.step(_i32(counts), T, q, k, v, out)
        assert int(s.err) == 0
        used = int(plan.blocks_used)
        s.free = s.free[used:].contiguous()
        at, seq = plan.query_start_loc.tolist(), plan.seq_lens.tolist()
        for r in range(R):
            rows = slice(at[r], at[r + 1])
            stored[r][1].append(oo.values(v[rows].cpu()))
            if seq[r] == 0:
                continue
            slots = on.table_slots(s.bt[r], seq[r], 16)
            K, V = oo.read(s.page.reshape(-1), s.lay.compressed_bytes_per_token(), slots, H, d)
            assert torch.equal(V, torch.cat(stored[r][1]))
            _close(out[rows], None, qr[rows].cpu(), K, V, d ** -0.5, (counts, r), window=window)
        assert bool((out[n:] == 7).all())
        # what a prompt's next chunk would attend to densely
        starts = [0]
        for m in seq:
            starts.append(starts[-1] + m)
        _, vals = kernels.octet_read_paged(s.lay, s.page, 16, s.bt, _i32(starts), 192, num_rows=starts[-1])
        want = torch.cat([torch.cat(x[1]) for x in stored if x[1]])
        assert torch.equal(vals.cpu().double(), want)
        s.computed = plan.seq_lens


def test_parts_of_a_context_join_by_their_lse():
    """Attention over a window and over what lies before it, joined by their lse, is the whole's."""
    st = Store([90], 1, 64, seed=3)
    q = torch.randn(1, 4, 64, generator=_gen(4)).half().cuda()
    lse = [torch.zeros(1, 4, device="cuda") for _ in range(3)]
    whole, _, _ = _decode(st, q, lse=lse[0])
    late, _, _ = _decode(st, q, lse=lse[1], window=26)
    st.seq, st.lens = _i32([64]), [64]
    early, _, _ = _decode(st, q, lse=lse[2])
    w = [(x - lse[0]).exp().unsqueeze(-1) for x in lse[1:]]
    got = late.float() * w[0] + early.float() * w[1]
    assert float((got - whole.float()).abs().max()) < 3 * 2.0 ** -11 * float(whole.abs().max()) + 1e-4
    assert float((w[0] + w[1] - 1).abs().max()) < 1e-4


def test_captured_steps_replay():
    """A step captured into a graph, replayed over new inputs and lengths with eager work between,
    each replay against the eager result; two graphs share the workspace in stream order."""
    R, H, G, d = 3, 2, 4, 128
    g = _gen(0)
    eager, graph = Serving(R, H, G, d), Serving(R, H, G, d)
    T = 8
    static = dict(counts=_i32([1, 1, 1]), q=torch.zeros(T, H * G, d, dtype=torch.float16, device="cuda"),
                  k=torch.zeros(T, H, d, dtype=torch.float16, device="cuda"),
                  v=torch.zeros(T, H, d, dtype=torch.float16, device="cuda"),
                  out=torch.zeros(T, H * G, d, dtype=torch.float16, device="cuda"),
                  lse=torch.zeros(T, H * G, device="cuda"))

    def feed(counts):
        static["counts"].copy_(_i32(counts))
        for name in ("q", "k", "v"):
            static[name].copy_(torch.randn(static[name].shape, generator=g).half())

    def run(s):
        plan, _ = s.step(static["counts"], T, static["q"], static["k"], static["v"], static["out"],
                         static["lse"])
        return plan

    feed([1, 1, 1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                 # (the caches of warm-up are thrown away below)
        run(graph)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        cg = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cg):
            plan = run(graph)
        graphs.append((cg, plan))
    graph.page.fill_(255)
    graph.bt.fill_(-1)
    for i, counts in enumerate([[1, 1, 1], [4, 3, 1], [1, 0, 2], [2, 2, 2], [1, 1, 1], [0, 0, 8]]):
        feed(counts)
        static["out"].fill_(7)
        plan = run(eager)
        want, wlse = static["out"].clone(), static["lse"].clone()
        eager.computed.copy_(plan.seq_lens)
        eager.free.copy_(torch.roll(eager.free, -int(plan.blocks_used)))
        static["out"].fill_(7)
        static["lse"].fill_(0)
        cg, held = graphs[i % 2]
        cg.replay()
        torch.cuda.synchronize()
        n = sum(counts)
        assert torch.equal(static["out"], want) and torch.equal(static["lse"][:n], wlse[:n])
        graph.computed.copy_(held.seq_lens)
        graph.free.copy_(torch.roll(graph.free, -int(held.blocks_used)))
        torch.randn(1000, device="cuda").sum().item()
    assert int(eager.err) == 0 and int(graph.err) == 0


def test_other_streams():
    """Two streams at once, a workspace each."""
    st = Store([2000, 150], 2, 128, seed=8)
    q = torch.randn(2, 8, 128, generator=_gen(1)).half().cuda()
    want, _, _ = _decode(st, q)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    wss = [kernels.octet_decode_workspace(st.lay, 8, 2, 1, 2000, "cuda") for _ in range(2)]
    at = _i32([0, 1, 2])
    torch.cuda.synchronize()
    for _ in range(5):
        for s, ws in zip(streams, wss):
            with torch.cuda.stream(s):
                got.append(kernels.octet_decode_paged(st.lay, q, st.page, 16, st.bt, st.seq, at, 1, 2000,
                                                      128 ** -0.5, workspace=ws))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)

"""The 8-bit cache on the CPU: the oracle's quantisation against rational arithmetic, its places, the
layout's sizes, scaled frequencies, and the refusals of the C entry points and the wrappers (nothing
is launched)."""
import math
from fractions import Fraction

import pytest
import torch

from oracle import octet as oo
from vllm_ttkv import _hip, kernels
from vllm_ttkv.octet import OctetLayout
from vllm_ttkv.rope import LLAMA32_3B_ROPE, Rotary, llama3_inv_freq, scaled_rotary

GRID = sorted({m * Fraction(2) ** -9 for m in range(8)}
              | {(8 + m) * Fraction(2) ** (e - 10) for e in range(1, 16) for m in range(8)})[:-1]
assert GRID[-1] == 448 and len(GRID) == 127


def _nearest(t):
    """The e4m3 number nearest to t in [0, 448], ties to the even code."""
    lo = max(i for i, v in enumerate(GRID) if v <= t)
    if lo == len(GRID) - 1:
        return lo
    below, above = t - GRID[lo], GRID[lo + 1] - t
    return lo if below < above or (below == above and lo % 2 == 0) else lo + 1


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantisation_is_the_exact_formula(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(24, 64, generator=g)
    x[:6] *= 2.0 ** torch.randint(-30, 14, (6, 1), generator=g)
    x[6, :32] = torch.arange(32) + 432.5         # at and around the largest code
    x[7, :32], x[7, 0] = (2 * torch.arange(32) + 1) / 1024, 448.0    # on the borders of small codes
    x[8, :32], x[8, 0] = 17 + 2 * torch.arange(32), 448.0            # and of larger ones
    x[9] = 0
    x[10], x[10, 0] = 2.0 ** -20, 1.0            # under the smallest code
    x[11] = -x[11].abs()
    if dtype != torch.float16:
        x[12] *= 1e-36
        x[13, :3] = torch.tensor([3.3e38, -3.3e38, 2.9e38])          # beyond the limit
        x[14] *= 1e37
    x = x.to(dtype)
    code, byte = oo.quantise(x)
    got = oo.values(x)
    for i in range(24):
        for gr in range(2):
            row = [max(min(Fraction(float(v)), Fraction(oo.LIMIT)), -Fraction(oo.LIMIT))
                   for v in x[i, 32 * gr:32 * gr + 32]]
            e = -117
            while max(abs(v) for v in row) > 448 * Fraction(2) ** e:
                e += 1
            assert int(byte[i, gr]) == e + 127
            for k, v in enumerate(row):
                at = 32 * gr + k
                want = _nearest(abs(v) / Fraction(2) ** e)
                assert int(code[i, at]) % 128 == want
                assert int(code[i, at]) // 128 == int(math.copysign(1, float(x[i, at])) < 0)
                val = Fraction(float(got[i, at]))
                assert abs(val) == GRID[want] * Fraction(2) ** e
                assert Fraction(float(got[i, at].to(torch.bfloat16))) == val    # exact in bf16
                assert val == 0 or abs(val) >= Fraction(2) ** -126
                assert abs(val - v) <= max(abs(v) / 16, Fraction(2) ** (e - 10))


def test_a_group_that_is_not_finite_reads_as_nan():
    x = torch.randn(3, 128)
    x[0, 5], x[1, 40], x[2, 127] = float("nan"), float("inf"), -float("inf")
    v, (_, byte) = oo.values(x), oo.quantise(x)
    for i, g in ((0, 0), (1, 1), (2, 3)):
        assert int(byte[i, g]) == 127
        for k in range(4):
            assert bool(torch.isnan(v[i, 32 * k:32 * k + 32]).all()) == (k == g)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_places_fill_the_record(d):
    """Every byte of a record is used once; a lane's share comes in whole pieces of 16 bytes."""
    seen = torch.cat([t.reshape(-1) for t in oo.places(d)])
    assert sorted(seen.tolist()) == list(range(33 * d))
    for u in range(16):
        for x in range(0, d, 16):
            assert oo.key_place(d, u, x) % 16 == 0
            assert oo.key_place(d, u, x + 15) == oo.key_place(d, u, x) + 15


@pytest.mark.parametrize("d", [64, 128, 256])
def test_oracle_write_and_read_agree(d):
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(5, 2, d, generator=g), torch.randn(5, 2, d, generator=g)
    slots, stride = torch.tensor([3, 16, 47, -1, 30]), OctetLayout(2, d).compressed_bytes_per_token()
    page = torch.zeros(48 * stride, dtype=torch.uint8)
    oo.write(page, stride, slots, k, v)
    keep = slots >= 0
    K, V = oo.read(page, stride, slots[keep], 2, d)
    assert torch.equal(K, oo.values(k)[keep]) and torch.equal(V, oo.values(v)[keep])


def test_layout():
    lay = OctetLayout(H=8)
    assert lay.row_bytes == 132 and lay.compressed_bytes_per_token() == 2112
    assert lay.dense_bytes_per_token() == 4096 and abs(lay.ratio() - 4096 / 2112) < 1e-12
    for d in (64, 128, 256):
        assert OctetLayout(3, d).compressed_bytes_per_token() * 16 == 3 * 33 * d
    with pytest.raises(ValueError, match="head dim"):
        OctetLayout(H=8, d=96)
    with pytest.raises(ValueError, match="KV heads"):
        OctetLayout(H=0)


# ------------------------------------------------------------------------- scaled frequencies
def _w(r):
    return r.turns * 2 * math.pi


def test_scaled_frequencies():
    base = 500000.0 ** (-torch.arange(0, 128, 2).double() / 128)
    assert torch.allclose(_w(scaled_rotary(128)), base, rtol=1e-15)
    assert torch.allclose(_w(scaled_rotary(128, rule="linear", factor=4)), base / 4, rtol=1e-15)
    n = _w(scaled_rotary(128, rule="ntk", factor=8))
    assert abs(float(n[0]) - 1) < 1e-12 and abs(float(n[-1] / base[-1]) - 1 / 8) < 1e-12
    three = scaled_rotary(128, LLAMA32_3B_ROPE["theta"], "llama3", 32.0, 8192, 1.0, 4.0)
    assert torch.allclose(_w(three).float(), llama3_inv_freq(128, **LLAMA32_3B_ROPE), rtol=2e-6)
    y = scaled_rotary(64, 10000.0, "yarn", 16.0, 4096)
    base = 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    ratio = _w(y) / base                     # 1 to fast revolutions, 1 / 16 to slow ones, falling
    assert float(ratio[0]) == pytest.approx(1) and float(ratio[-1]) == pytest.approx(1 / 16)
    assert bool((ratio[1:] <= ratio[:-1] + 1e-12).all())
    turns = 4096 * base / (2 * math.pi)
    assert bool((ratio[turns > 40] > 0.999).all()) and bool((ratio[turns < 0.8] < 0.0626).all())
    assert y.amplitude == pytest.approx(0.1 * math.log(16) + 1) and not y.adjacent
    for bad in (dict(rotary_dim=5), dict(rotary_dim=0), dict(rotary_dim=64, factor=0.5),
                dict(rotary_dim=64, rule="other")):
        with pytest.raises(ValueError):
            scaled_rotary(**bad)


# ------------------------------------------------------------------------- C entry refusals
def _refused(rc, code, text):
    msg = _hip.lib().ttkv_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def _rotary(**kw):
    a = dict(q=4096, k=8192, qo=4096, ko=8192, dt=1, n=2, HQ=4, H=2, d=64, qs=256, ks=128, qos=256,
             kos=128, pos=64, turns=64, rot=64, amp=1.0, adj=0, err=16)
    a.update(kw)
    return _hip.lib().ttkv_rotary_scaled(*a.values(), None)


def test_rotary_refusals():
    _refused(_rotary(dt=5), 1, "dtype")
    _refused(_rotary(n=-1), 1, "negative")
    _refused(_rotary(d=0), 1, "negative")
    for rot in (0, 63, 66, -2):
        _refused(_rotary(rot=rot), 1, "rotary dims")
    _refused(_rotary(d=2048, rot=1026, qs=8192, ks=4096, qos=8192, kos=4096), 2, "1024")
    _refused(_rotary(pos=0), 1, "null")
    _refused(_rotary(turns=0), 1, "null")
    _refused(_rotary(turns=68), 1, "8-byte")
    for a in ("q", "k", "qo", "ko", "err"):
        _refused(_rotary(**{a: 0}), 1, "null")
    _refused(_rotary(qo=4096 + 16), 1, "overlaps its input")
    _refused(_rotary(qos=260), 1, "overlaps its input")
    _refused(_rotary(ko=4096), 1, "overlaps")
    _refused(_rotary(qo=8192 + 64, qos=256), 1, "overlaps")
    assert _rotary(n=0) == 0 and _rotary(HQ=0, H=0) == 0


def _write(**kw):
    a = dict(H=8, d=128, key=65536, kt=1, ks=1024, value=131072, vt=1, vs=1024, slots=16, n=4, page=4096,
             n_slots=64, stride=2112, ko=0, vo=0, pos=0, turns=0, rot=0, amp=1.0, adj=0, q=0, qt=0,
             qs=0, HQ=0, qo=0, qos=0, err=16)
    a.update(kw)
    return _hip.lib().ttkv_octet_write_paged(*a.values(), None)


def test_write_refusals():
    _refused(_write(d=96), 2, "head dim")
    _refused(_write(H=0), 1, "H must")
    _refused(_write(page=0), 1, "page")
    _refused(_write(page=4104), 1, "16-byte")
    _refused(_write(stride=2111), 1, "slot stride")
    _refused(_write(n_slots=24), 1, "multiple of 16")
    _refused(_write(n_slots=0), 1, "multiple of 16")
    _refused(_write(kt=3), 1, "dtype")
    _refused(_write(vt=-1), 1, "dtype")
    _refused(_write(n=-1), 1, "negative")
    for a in ("key", "value", "slots", "err"):
        _refused(_write(**{a: 0}), 1, "null")
    _refused(_write(ko=8), 1, "key_out")
    _refused(_write(vo=24), 1, "value_out")
    # outputs: bf16 rows of 2,048 bytes, four of them; the inputs are fp16 rows of as many
    _refused(_write(ko=65536 + 2048), 1, "key_out or value_out overlaps")
    _refused(_write(ko=65536, kt=0), 1, "key_out or value_out overlaps")
    _refused(_write(ko=131072), 1, "key_out or value_out overlaps")
    _refused(_write(vo=65536), 1, "key_out or value_out overlaps")
    _refused(_write(vo=131072 - 16), 1, "key_out or value_out overlaps")
    _refused(_write(ko=1 << 18, vo=(1 << 18) + 4096), 1, "key_out or value_out overlaps")
    rotated = dict(pos=64, turns=64, rot=128)
    _refused(_write(**dict(rotated, rot=130)), 1, "rotary dims")
    _refused(_write(**dict(rotated, rot=-2)), 1, "rotary dims")
    _refused(_write(**dict(rotated, pos=0)), 1, "null")
    _refused(_write(HQ=8, q=1 << 20, qo=1 << 20, qt=1, qs=1024, qos=1024), 1, "queries")
    asked = dict(rotated, HQ=8, q=1 << 20, qo=1 << 20, qt=1, qs=1024, qos=1024)
    _refused(_write(**dict(asked, qt=7)), 1, "query dtype")
    _refused(_write(**dict(asked, q=0)), 1, "null")
    _refused(_write(**dict(asked, qo=(1 << 20) + 256)), 1, "overlaps the query")
    _refused(_write(**dict(asked, qo=65536)), 1, "overlaps the keys")
    _refused(_write(**dict(asked, qo=131072 + 512)), 1, "overlaps the keys")
    _refused(_write(**dict(asked, ko=1 << 20)), 1, "overlaps the keys")
    _refused(_write(**dict(asked, qo=1 << 21, vo=(1 << 20) + 2048)), 1, "overlaps the keys")
    assert _write(n=0) == 0


def _read(**kw):
    a = dict(H=8, d=128, page=4096, n_slots=64, stride=2112, bs=16, bt=16, bts=4, mb=4, starts=16,
             first=0, reqs=1, max_seq=64, rows=8, ko=1 << 16, ks=1024, vo=1 << 17, vs=1024, dt=2, err=16)
    a.update(kw)
    return _hip.lib().ttkv_octet_read_paged(*a.values(), None)


def test_read_refusals():
    _refused(_read(d=80), 2, "head dim")
    _refused(_read(stride=2000), 1, "slot stride")
    _refused(_read(bs=24), 1, "block size")
    _refused(_read(bs=0), 1, "block size")
    _refused(_read(bs=48), 1, "block size")
    _refused(_read(max_seq=65), 1, "blocks")
    _refused(_read(max_seq=(1 << 26) + 1, mb=1 << 23), 2, "2^26")
    for a in ("reqs", "max_seq", "rows"):
        _refused(_read(**{a: -1}), 1, "negative")
    _refused(_read(dt=3), 1, "dtype")
    for a in ("bt", "starts", "ko", "vo", "err"):
        _refused(_read(**{a: 0}), 1, "null")
    _refused(_read(ko=1 << 16, vo=(1 << 16) + 2046), 1, "overlap")
    _refused(_read(ko=1 << 16, vo=(1 << 16) - 16), 1, "overlap")
    assert _read(rows=0) == 0 and _read(reqs=0) == 0


def _decode(**kw):
    a = dict(H=8, HQ=32, d=128, scale=0.1, q=16, qt=1, qs=4096, n=4, page=4096, n_slots=64,
             stride=2112, bs=16, bt=16, bts=4, mb=4, seq=16, qsl=16, reqs=1, max_q=1, max_seq=64,
             window=0, sinks=0, out=16, ot=1, os=4096, lse=0, ws=256, wsb=1 << 30, err=16)
    a.update(kw)
    return _hip.lib().ttkv_octet_decode_paged(*a.values(), None)


def test_decode_refusals():
    _refused(_decode(d=192), 2, "head dim")
    _refused(_decode(HQ=20), 1, "multiple of H")
    _refused(_decode(HQ=8 * 17), 2, "16 query heads")
    _refused(_decode(qt=0), 1, "dtype")
    _refused(_decode(ot=0), 1, "dtype")
    _refused(_decode(bs=40), 1, "block size")
    _refused(_decode(max_seq=65), 1, "blocks")
    for a in ("n", "max_q", "reqs", "max_seq", "mb"):
        _refused(_decode(**{a: -1}), 1, "negative")
    _refused(_decode(max_q=17), 2, "16 queries")
    _refused(_decode(window=-1), 1, "window")
    for a in ("q", "bt", "seq", "qsl", "out", "err"):
        _refused(_decode(**{a: 0}), 1, "null")
    _refused(_decode(q=24), 1, "16-byte")
    _refused(_decode(out=8), 1, "16-byte")
    _refused(_decode(qs=4100), 1, "16-byte")
    _refused(_decode(q=65536, out=65536 + 8192), 1, "overlaps the query")
    _refused(_decode(q=65536, out=65536, os=8192), 1, "overlaps the query")
    _refused(_decode(q=65536, out=65536 - 16), 1, "overlaps the query")
    _refused(_decode(ws=0), 4, "workspace")
    _refused(_decode(ws=128), 4, "workspace")
    _refused(_decode(wsb=16), 4, "workspace")
    assert _decode(reqs=0) == 0 and _decode(n=0) == 0 and _decode(max_q=0) == 0


def test_output_rows_that_overlap_one_another_are_refused():
    for kw in (dict(q=1 << 20, qos=248), dict(q=1 << 20, qos=0), dict(k=1 << 20, kos=-120)):
        _refused(_rotary(**kw), 1, "rows of an output")
    _refused(_write(pos=64, turns=64, rot=128, HQ=8, q=1 << 20, qo=1 << 21, qt=1, qs=1024, qos=1016), 1,
             "rows of query_out")
    for kw in (dict(ks=1016), dict(vs=0)):
        _refused(_read(**kw), 1, "rows of an output")
    for stride in (4088, 0):
        _refused(_decode(q=1 << 20, out=1 << 21, os=stride), 1, "rows of out")


def test_outputs_that_overlap_rows_of_another_stride_are_refused():
    """Rows of unlike strides whose first ones lie apart: packed rows, and an output's at twice their stride from
    the second one on; a packed output behind a strided input's first row."""
    q = 1 << 20
    _refused(_rotary(q=q, qo=q + 512, qos=512), 1, "overlaps its input")
    _refused(_rotary(q=q, qs=512, qo=q + 512, n=4), 1, "overlaps its input")
    _refused(_rotary(q=q, qs=0, qo=q - 512), 1, "overlaps its input")
    _refused(_rotary(q=q, k=q + 512, ks=256, ko=q + 3 * 512, kos=512, n=4), 1, "overlaps")
    asked = dict(pos=64, turns=64, rot=128, HQ=8, q=q, qo=1 << 21, qt=1, qs=1024, qos=1024)
    _refused(_write(**dict(asked, qo=q + 2048, qos=2048)), 1, "overlaps the query")
    _refused(_write(**dict(asked, qo=65536 + 2048, qos=2048)), 1, "overlaps the keys")
    _refused(_write(ko=65536 + 2048, ks=2048), 1, "key_out or value_out overlaps")
    _refused(_write(vo=131072 + 2048, vs=1536), 1, "key_out or value_out overlaps")
    _refused(_read(ko=1 << 16, vo=(1 << 16) + 2048, vs=2048), 1, "overlap")
    _refused(_decode(q=1 << 20, out=(1 << 20) + 8192, os=8192), 1, "overlaps the query")
    _refused(_decode(q=1 << 20, qs=8192, out=(1 << 20) + 8192), 1, "overlaps the query")


def test_overlap_is_found_exactly():
    """Against the rows' bytes one by one, for strides of any sign; a later refusal (keys' output rows that
    overlap one another) takes the calls whose queries lie apart, so that nothing is launched."""
    g = torch.Generator().manual_seed(3)

    def pick(lo, hi):
        return int(torch.randint(lo, hi + 1, (1,), generator=g))

    seen = [0, 0]
    for _ in range(6000):
        n, w, q = pick(2, 7), 2 * pick(1, 4), 1 << 20
        qs, qos = (pick(-12, 12) for _ in range(2))
        if pick(0, 3) == 0:
            qos = qs
        qo = q + 2 * pick(-60, 60)
        rows = [{a + 2 * s * i + b for i in range(n) for b in range(2 * w)} for a, s in ((q, qs), (qo, qos))]
        meets = bool(rows[0] & rows[1]) and not (q == qo and qs == qos)
        seen[meets] += 1
        _refused(_rotary(q=q, qo=qo, qs=qs, qos=qos, n=n, HQ=1, H=1, d=w, rot=2, k=1 << 24, ks=64, ko=1 << 25,
                         kos=0), 1, "overlaps its input" if meets else "rows of an output")
    assert min(seen) > 1000


def test_workspace_sizes_grow_with_every_argument():
    f = _hip.lib().ttkv_octet_decode_workspace_bytes
    for bad in ((0, 8, 128, 1, 1, 64), (8, 12, 128, 1, 1, 64), (8, 8, 96, 1, 1, 64),
                (8, 8, 128, -1, 1, 64), (8, 8, 128, 1, -1, 64), (8, 8, 128, 1, 1, -1)):
        assert f(*bad) == -1
    last = 0
    for a in ((8, 8, 64, 1, 1, 1), (8, 32, 64, 1, 1, 1000), (8, 32, 128, 1, 1, 1000),
              (8, 32, 128, 9, 1, 20000), (8, 32, 256, 9, 5, 20000), (8, 128, 256, 300, 16, 1 << 26)):
        assert f(*a) >= last
        last = f(*a)


# ------------------------------------------------------------------------- wrapper refusals
def test_wrappers_refuse_host_tensors():
    lay = OctetLayout(2, 64)
    k = torch.zeros(3, 2, 64)
    page = torch.zeros(2, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8)
    i = torch.zeros(4, dtype=torch.int32)
    bt, slots = i.reshape(2, 2), torch.zeros(3, dtype=torch.int64)
    r = Rotary(torch.zeros(32, dtype=torch.float64))
    for f in (lambda: kernels.rotary_scaled(k, None, slots, r),
              lambda: kernels.octet_write_paged(lay, k, k, slots, page),
              lambda: kernels.octet_read_paged(lay, page, 16, bt, i[:2], 16, num_rows=3),
              lambda: kernels.octet_decode_paged(lay, k.half(), page, 16, bt, i[:1], i[:2], 1, 16, 1.0)):
        with pytest.raises(RuntimeError, match="device"):
            f()

"""The 4-bit cache on the CPU: the oracle's quantisation against rational arithmetic, its places,
the layout's sizes, and the refusals of the C entry points and the wrappers (nothing is launched)."""
import ctypes
from fractions import Fraction

import pytest
import torch

from oracle import nibble as on
from vllm_ttkv import _hip, kernels
from vllm_ttkv.nibble import NibbleLayout


def _round_half_even(f):
    q, r = divmod(f.numerator, f.denominator)
    twice = 2 * r - f.denominator
    return q + (twice > 0 or (twice == 0 and q % 2 == 1))


def _step(rng):
    """The smallest number of 7 significant bits that is at least rng / 15, at least 2^-14."""
    t = rng / 15
    if t <= Fraction(1, 2 ** 14):
        return Fraction(1, 2 ** 14)
    e = 0
    while t >= Fraction(2) ** (e + 1):
        e += 1
    while t < Fraction(2) ** e:
        e -= 1
    unit = Fraction(2) ** (e - 6)
    return -(-t // unit) * unit


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantisation_is_the_exact_formula(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(40, 128, generator=g)
    x[:10] *= 2.0 ** torch.randint(-20, 14, (10, 1), generator=g)
    x[10, :64] = torch.arange(64) / 4 - 3        # quotients on rounding borders
    x[11] = 0
    x[12] = x[12].abs() + 5                      # one sign
    x[13] = (-x[13].abs() * 1e5).clamp(min=-60000)    # beyond the limit
    x = x.to(dtype)
    c, z, s, par = on.quantise(x)
    for i in range(40):
        for gr in range(4):
            v = [min(max(Fraction(float(t)), Fraction(-32640)), Fraction(32640))
                 for t in x[i, 32 * gr:32 * gr + 32]]
            lo, hi = min(v + [Fraction(0)]), max(v + [Fraction(0)])
            step = _step(hi - lo)
            assert Fraction(float(s[i, gr])) == step
            zero = min(max(_round_half_even(-lo / step), 0), 15)
            assert int(z[i, gr]) == zero
            codes = [min(max(_round_half_even(t / step) + zero, 0), 15) for t in v]
            assert c[i, gr].tolist() == codes
            assert int(par[i, gr]) & 15 == zero
            assert float(torch.tensor(int(par[i, gr]) - zero).to(torch.int16).view(torch.float16)) \
                == float(step)
            # a value is exact in fp16, and at most half a step from its input (a step where both
            # ends of a full range round outwards and the last code is taken back)
            for t, k in zip(v, codes):
                val = (k - zero) * step
                assert Fraction(float(torch.tensor(float(val)).half())) == val
                assert abs(val - t) <= step / 2 + (step / 2 if k == 15 else 0)


def test_a_group_that_is_not_finite_reads_as_nan():
    x = torch.randn(3, 128)
    x[0, 5], x[1, 40], x[2, 127] = float("nan"), float("inf"), -float("inf")
    v, par = on.values(x), on.quantise(x)[3]
    for i, g in ((0, 0), (1, 1), (2, 3)):
        assert int(par[i, g]) == 0x7E00
        for k in range(4):
            assert bool(torch.isnan(v[i, 32 * k:32 * k + 32]).all()) == (k == g)


def test_places_fill_the_record():
    """Every nibble of the codes and every 16-bit word of the parameters is used once."""
    for place, par, lo, plo in ((on.key_place, on.key_par, 0, on.KPAR),
                                (on.value_place, on.value_par, on.VCODES, on.VPAR)):
        seen = {place(u, x) for u in range(16) for x in range(128)}
        assert seen == {(lo + b, s) for b in range(1024) for s in (0, 4)}
        assert {par(u, g) for u in range(16) for g in range(4)} == set(range(plo, plo + 128, 2))


def test_oracle_write_and_read_agree():
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn(5, 2, 128, generator=g), torch.randn(5, 2, 128, generator=g)
    slots = torch.tensor([3, 16, 47, -1, 30])
    page = torch.zeros(48 * 288, dtype=torch.uint8)
    on.write(page, 288, slots, k, v)
    keep = slots >= 0
    K, V = on.read(page, 288, slots[keep], 2)
    assert torch.equal(K, on.values(k)[keep]) and torch.equal(V, on.values(v)[keep])


def test_layout():
    lay = NibbleLayout(H=8)
    assert lay.row_bytes == 72 and lay.compressed_bytes_per_token() == 1152
    assert lay.dense_bytes_per_token() == 4096 and abs(lay.ratio() - 4096 / 1152) < 1e-12
    with pytest.raises(ValueError, match="head dim"):
        NibbleLayout(H=8, d=64)
    with pytest.raises(ValueError, match="KV heads"):
        NibbleLayout(H=0)


# ------------------------------------------------------------------------- C entry refusals
def _refused(rc, code, text):
    msg = _hip.lib().ttkv_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def _write(**kw):
    a = dict(H=8, d=128, key=16, kt=1, ks=1024, value=16, vt=1, vs=1024, slots=16, n=4, page=4096,
             n_slots=64, stride=1152, ko=0, vo=0, err=16)
    a.update(kw)
    return _hip.lib().ttkv_nibble_write_paged(*a.values(), None)


def test_write_refusals():
    _refused(_write(d=64), 2, "head dim")
    _refused(_write(H=0), 1, "H must")
    _refused(_write(page=0), 1, "null page")
    _refused(_write(page=4104), 1, "aligned")
    _refused(_write(stride=1136), 1, "slot stride")
    _refused(_write(stride=1160), 1, "aligned")
    _refused(_write(n_slots=40), 1, "multiple of 16")
    _refused(_write(n_slots=0), 1, "multiple of 16")
    _refused(_write(kt=5), 1, "dtype")
    _refused(_write(n=-1), 1, "negative")
    _refused(_write(key=0), 1, "null")
    _refused(_write(slots=0), 1, "null")
    _refused(_write(err=0), 1, "null")
    _refused(_write(ko=24), 1, "key_out")
    assert _write(n=0) == 0                                        # nothing to do


def _decode(**kw):
    a = dict(H=8, HQ=24, d=128, scale=0.088, q=16, qt=1, qs=24 * 128, page=4096, n_slots=64,
             stride=1152, bs=16, bt=16, bts=4, W=4, seq=16, qsl=16, R=1, max_seq=64, out=16, ot=1,
             os=24 * 128, ws=256, ws_bytes=1 << 30, err=16)
    a.update(kw)
    return _hip.lib().ttkv_nibble_decode_paged(*a.values(), None)


def _prefill(**kw):
    a = dict(H=8, HQ=24, d=128, scale=0.088, q=16, qt=1, qs=24 * 128, page=4096, n_slots=64,
             stride=1152, bs=16, bt=16, bts=4, W=4, seq=16, qsl=16, idx=0, R=1, max_q=8,
             max_seq=64, out=16, ot=1, os=24 * 128, ws=256, ws_bytes=1 << 30, err=16)
    a.update(kw)
    return _hip.lib().ttkv_nibble_prefill_paged(*a.values(), None)


@pytest.mark.parametrize("call", [_decode, _prefill])
def test_read_refusals(call):
    _refused(call(d=96), 2, "head dim")
    _refused(call(HQ=20), 1, "multiple of H")
    _refused(call(HQ=8 * 17), 2, "16 query heads")
    _refused(call(HQ=0), 1, "multiple of H")
    _refused(call(qt=0), 1, "dtype")
    _refused(call(ot=0), 1, "dtype")
    _refused(call(bs=8), 1, "block size")
    _refused(call(bs=48), 1, "block size")                          # 64 slots are not 48s
    _refused(call(max_seq=65), 1, "blocks")
    _refused(call(R=-1), 1, "negative")
    _refused(call(q=0), 1, "null")
    _refused(call(q=24), 1, "aligned")
    _refused(call(qs=24 * 128 + 4), 1, "aligned")
    _refused(call(err=0), 1, "null")
    _refused(call(ws=0), 4, "workspace")
    _refused(call(ws=264), 4, "workspace")
    _refused(call(ws_bytes=16), 4, "workspace")
    _refused(call(stride=1151), 1, "slot stride")
    assert call(R=0) == 0                                           # nothing to do


def test_prefill_refusals():
    _refused(_prefill(max_q=65), 1, "max_q_len")
    _refused(_prefill(max_q=-1), 1, "negative")
    assert _prefill(max_q=0) == 0


def test_workspace_sizes():
    L = _hip.lib()
    assert L.ttkv_nibble_decode_workspace_bytes(8, 20, 1, 100) == -1
    assert L.ttkv_nibble_decode_workspace_bytes(0, 8, 1, 100) == -1
    assert L.ttkv_nibble_decode_workspace_bytes(8, 24, -1, 100) == -1
    assert L.ttkv_nibble_prefill_workspace_bytes(8, 24, 1, -1, 100) == -1
    small = L.ttkv_nibble_decode_workspace_bytes(8, 24, 1, 100)
    assert 0 < small <= L.ttkv_nibble_decode_workspace_bytes(8, 24, 64, 16000)


def test_a_workspace_for_the_largest_batch_serves_smaller_ones():
    L, g = _hip.lib(), torch.Generator().manual_seed(3)

    def draw(most):
        return int(2 ** (float(torch.rand(1, generator=g)) * most))

    for _ in range(300):
        H, G = draw(4), min(draw(5), 16)
        R, q, n = draw(9), draw(12), draw(15)
        q = min(q, n)
        r2, q2, n2 = R + draw(4) - 1, q + draw(8) - 1, n + draw(13)
        assert L.ttkv_nibble_decode_workspace_bytes(H, H * G, R, n) \
            <= L.ttkv_nibble_decode_workspace_bytes(H, H * G, r2, n2)
        a = L.ttkv_nibble_prefill_workspace_bytes(H, H * G, R, q, n)
        assert 256 <= a <= L.ttkv_nibble_prefill_workspace_bytes(H, H * G, r2, q2, max(n2, q2))
        assert a <= 64 << 20
    big = 2 ** 31 - 1
    assert 0 < L.ttkv_nibble_prefill_workspace_bytes(16384, 16384, big, big, big) <= 64 << 20


def _rotary(sections=(16, 24, 24), **kw):
    a = dict(q=16, k=16, qo=16, ko=16, dt=1, N=4, HQ=24, H=8, d=128, qs=24 * 128, ks=1024,
             qos=24 * 128, kos=1024, pos=16, ps=4, axes=len(sections),
             sec=(ctypes.c_int32 * len(sections))(*sections), inter=0, cs=16, max_pos=64, rot=128,
             err=16)
    a.update(kw)
    return _hip.lib().ttkv_rotary_axes(*a.values(), None)


def test_rotary_refusals():
    _refused(_rotary(dt=3), 1, "dtype")
    _refused(_rotary(rot=126), 1, "add up")
    _refused(_rotary(rot=127), 1, "even")
    _refused(_rotary(rot=130), 1, "even")
    _refused(_rotary(sections=(64, 0, 0, 0, 0)), 1, "axes")
    _refused(_rotary(sections=(16, 24, 23)), 1, "add up")
    _refused(_rotary(sections=(70, -6, 0)), 1, "negative section")
    _refused(_rotary(inter=1), 1, "interleaved")                    # 1 + 3 * 23 > 63
    _refused(_rotary(max_pos=0), 1, "cos_sin_cache")
    _refused(_rotary(pos=0), 1, "null")
    _refused(_rotary(ko=0), 1, "null")
    _refused(_rotary(sec=None), 1, "null sections")
    _refused(_rotary(N=-1), 1, "negative")
    assert _rotary(N=0) == 0 and _rotary(HQ=0, H=0) == 0


def _plan(**kw):
    a = dict(c=16, n=16, R=2, bt=16, bts=4, W=4, free=16, F=4, bs=16, blocks=8, T=8, qsl=16,
             seq=16, slots=16, pos=16, used=16, err=16)
    a.update(kw)
    return _hip.lib().ttkv_step_plan(*a.values(), None)


def test_plan_refusals():
    _refused(_plan(R=8001), 2, "8000")
    _refused(_plan(R=-1), 1, "negative")
    _refused(_plan(F=-1), 1, "negative")
    _refused(_plan(bs=0), 1, "block_size")
    _refused(_plan(bts=3), 1, "overlap")
    _refused(_plan(T=1 << 30), 1, "too many")
    _refused(_plan(bt=0), 1, "null")
    _refused(_plan(free=0), 1, "null")
    _refused(_plan(slots=0), 1, "null")
    _refused(_plan(used=0), 1, "null")
    out = dict(qsl=32, seq=48, used=64)
    for name in out:
        for at in ("c", "n"):
            _refused(_plan(**{**out, "c": 80, "n": 96, at: out[name]}), 1, "length inputs")


# --------------------------------------------------------------------------- wrapper refusals
def test_wrappers_refuse_host_tensors():
    lay = NibbleLayout(H=8)
    q, i32 = torch.zeros(1, 24, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    page = torch.zeros(4, 16, 1152, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="device tensors"):
        kernels.nibble_decode_paged(lay, q, page, 16, i32.view(1, 2), i32[:1], i32, 16, 0.1)
    with pytest.raises(RuntimeError, match="device tensors"):
        kernels.nibble_prefill_paged(lay, q, page, 16, i32.view(1, 2), i32[:1], i32, 1, 16, 0.1)
    with pytest.raises(RuntimeError, match="device tensors"):
        kernels.nibble_write_paged(lay, q[:, :8], q[:, :8], torch.zeros(1, dtype=torch.int64), page)
    with pytest.raises(RuntimeError, match="device tensors"):
        kernels.rotary_axes(q, None, torch.zeros(3, 1, dtype=torch.int64), torch.zeros(8, 128),
                            (16, 24, 24))
    with pytest.raises(RuntimeError, match="device tensors"):
        kernels.step_plan(i32, i32, i32.view(2, 1), i32, 16, 4, 4)

"""The 4-bit cache's entry points on the CPU: refusals that go with their edge cases (nothing is
launched)."""
import ctypes

import torch

from vllm_ttkv import _hip


def _refused(rc, code, text):
    msg = _hip.lib().ttkv_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def test_decode_starts_refusals():
    def call(starts, R):
        return _hip.lib().ttkv_nibble_decode_starts_paged(
            8, 24, 128, 0.088, 16, 1, 24 * 128, 4096, 64, 1152, 16, 16, 4, 4, 16, 16, starts, R, 64,
            16, 1, 24 * 128, 256, 1 << 30, 16, None)
    _refused(call(1, 2), 1, "query starts")
    _refused(call(0, 1), 1, "query starts")
    _refused(call(-1, 1), 1, "query starts")
    assert call(0, 0) == 0 and call(1, 0) == 0                      # nothing to do


# ------------------------------------------------------- a plan's outputs and what it reads
def _plan(**kw):
    """Two requests, a table of two rows of 4 at a stride of 8, 6 free ids, 9 tokens, apart from
    one another; a call that is not refused would launch, so each one here is."""
    a = dict(c=0x1000, n=0x2000, R=2, bt=0x3000, bts=8, W=4, free=0x4000, F=6, bs=16, blocks=8, T=9,
             qsl=0x5000, seq=0x6000, slots=0x7000, pos=0x8000, used=0x9000, err=0xa000)
    a.update(kw)
    return _hip.lib().ttkv_step_plan(*a.values(), None)


def test_plan_refuses_outputs_that_lie_in_its_inputs():
    size = dict(qsl=12, seq=8, used=4, slots=72, pos=72)
    for name, n in size.items():
        for at, length in ((0x1000, 8), (0x2000, 8)):               # the lengths, at any offset
            for off in range(-n + 4, length, 4):
                _refused(_plan(**{name: at + off}), 1, "length inputs")
        for off in range(-n + 4, 24, 4):
            _refused(_plan(**{name: 0x4000 + off}), 1, "free list")
        for row in (0x3000, 0x3020):
            for off in range(-n + 4, 16, 4):
                _refused(_plan(**{name: row + off}), 1, "block table")
    _refused(_plan(c=0x300c), 1, "length inputs")
    _refused(_plan(n=0x3020), 1, "length inputs")
    _refused(_plan(free=0x301c), 1, "free list")
    _refused(_plan(pos=0x7040), 1, "overlap")
    _refused(_plan(seq=0x5008), 1, "overlap")
    # query_lens as the tail of the buffer that the starts go to
    _refused(_plan(n=0x5004), 1, "length inputs")


# ------------------------------------------------------------------ rotary outputs and inputs
def _rotary(**kw):
    """Four tokens, four query and two key heads of 8 dims in fp16, inside rows of 8 heads (128 bytes
    a token): queries at 0, keys at 64, values behind; outputs apart unless named."""
    a = dict(q=0x10000, k=0x10040, qo=0x20000, ko=0x30000, dt=1, N=4, HQ=4, H=2, d=8, qs=64, ks=64,
             qos=32, kos=16, pos=16, ps=4, axes=1, sec=(ctypes.c_int32 * 1)(4), inter=0, cs=16,
             max_pos=64, rot=8, err=16)
    a.update(kw)
    return _hip.lib().ttkv_rotary_axes(*a.values(), None)


def test_rotary_refuses_outputs_that_overlap():
    q, k, row = 0x10000, 0x10040, 128
    for off in (-48, -16, 16, 48):                                  # shifted in place
        _refused(_rotary(qo=q + off, qos=64), 1, "without being it")
    for rows in (-3, -1, 1, 3):                                     # by whole rows
        _refused(_rotary(qo=q + rows * row, qos=64), 1, "without being it")
        _refused(_rotary(ko=k + rows * row, kos=64), 1, "without being it")
    _refused(_rotary(qo=q, qos=32), 1, "without being it")          # packed at the same place
    _refused(_rotary(ko=q + 16, kos=64), 1, "overlaps the other")   # key_out in the queries
    _refused(_rotary(qo=k, qos=64), 1, "overlaps the other")
    _refused(_rotary(qo=k - 16, qos=64, N=1), 1, "without being it")
    _refused(_rotary(qo=q, qos=64, ko=q, kos=64), 1, "overlaps the other")
    _refused(_rotary(qo=0x20000, ko=0x20000, qos=32, kos=32), 1, "overlaps the other")
    _refused(_rotary(qo=0x20000, ko=0x20030 + 128, qos=64, kos=64), 1, "overlaps the other")


# ----------------------------------------------------------------------------- workspace sizes
def test_workspaces_grow_with_every_argument():
    """With the KV heads and with the query heads too: one buffer serves layers of unlike heads."""
    L, g = _hip.lib(), torch.Generator().manual_seed(5)

    def draw(most):
        return int(2 ** (float(torch.rand(1, generator=g)) * most))

    for _ in range(400):
        HQ, R, n = 12 * draw(4), draw(9), draw(17)
        q = min(draw(12), n)
        heads = [h for h in range(1, HQ + 1) if HQ % h == 0 and HQ // h <= 16]
        decode = [L.ttkv_nibble_decode_workspace_bytes(h, HQ, R, n) for h in heads]
        prefill = [L.ttkv_nibble_prefill_workspace_bytes(h, HQ, R, q, n) for h in heads]
        assert decode == sorted(decode) and prefill == sorted(prefill) and decode[0] >= 65536
        h = heads[draw(3) % len(heads)]
        for k in (h, 2 * h, 5 * h):                                 # more query heads
            assert L.ttkv_nibble_decode_workspace_bytes(h, HQ, R, n) \
                <= L.ttkv_nibble_decode_workspace_bytes(h, HQ + k, R, n)
            assert L.ttkv_nibble_prefill_workspace_bytes(h, HQ, R, q, n) \
                <= L.ttkv_nibble_prefill_workspace_bytes(h, HQ + k, R, q, n)

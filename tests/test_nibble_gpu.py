"""The 4-bit cache's kernels on the GPU against the oracle in 64 bits: written bytes, reads at the
lengths, head counts, tables and types where they can go wrong, a step's plan, rotary axes, and a
run of them together.

Tolerances. A read rounds each softmax weight to fp16 once (half a step, 2^-11 of it) and its output
to the output's type once (2^-11 or, bf16, 2^-8 half a step: eps / 2); scores are products in 32 bits,
each of their 128 terms off by at most 2^-24 per addition (128 of them): 2^-17 of sum |q k| * scale,
which moves a weight by that relative amount, and the weights' sum with it (twice). So an output is
within  out_eps / 2 * |o| + (2^-11 + 2 * 2^-17 * score) * spread + 2^-24 spread-sized sums, where
spread = sum p |v|; the factor 1.05 covers the products of these terms. Smallest steps: fp16 outputs
below 2^-14 are spaced 2^-24, and weights below it add at most n * 2^-25 * max |v|."""
import pytest
import torch

from oracle import nibble as on
from vllm_ttkv import kernels, synth
from vllm_ttkv.nibble import NibbleLayout

pytestmark = pytest.mark.gpu
D = 128
SCALE = D ** -0.5
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _err():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


class Store:
    """A 4-bit store of requests of `lens` tokens in a shuffled paged cache, written by the kernel
    (whose bytes have their own test); slots that no token has hold 0xff (parameters that are NaN)."""

    def __init__(self, lens, H, block=16, seed=0, pad=0, scale=1.0, dtype=torch.float16):
        self.lens, self.H, self.block = list(lens), H, block
        self.lay = NibbleLayout(H)
        self.stride = self.lay.compressed_bytes_per_token() + pad
        bt, self.blocks = synth.shuffled_block_table([max(n, 1) for n in lens], block, seed=seed,
                                                     extra_blocks=3)
        self.bt = bt.cuda()
        self.page = torch.full((self.blocks, block, self.stride), 255, dtype=torch.uint8,
                               device="cuda")
        g = _gen(seed)
        n = sum(lens)
        k = torch.randn(n, H, D, generator=g)
        k[..., :8] *= 8
        v = torch.randn(n, H, D, generator=g)
        if torch.is_tensor(scale):
            scale = scale[:n].reshape(n, 1, 1)
        self.k, self.v = k.to(dtype), (v * scale).to(dtype)
        self.slots = torch.cat([on.table_slots(bt[r], m, block) for r, m in enumerate(lens)]
                               + [torch.zeros(0, dtype=torch.int64)])
        err = _err()
        kernels.nibble_write_paged(self.lay, self.k.cuda(), self.v.cuda(), self.slots.cuda(),
                                   self.page, error_word=err)
        assert int(err) == 0
        self.seq = _i32(self.lens)

    def kv(self, r):
        at = sum(self.lens[:r])
        s = slice(at, at + self.lens[r])
        return on.values(self.k[s]), on.values(self.v[s])


def _close(got, q, K, V, scale, what):
    want, spread, score = on.attend(q, K, V, scale)
    half, n = HALF[got.dtype], K.shape[0]
    vmax = float(V.abs().max()) if n else 0.0
    tol = 1.05 * (half * want.abs() + (2.0 ** -11 + 2.0 ** -16 * score + 2.0 ** -20) * spread) \
        + 2.0 ** -25 * (1 + n * vmax)
    e = (got.cpu().double() - want).abs()
    assert bool((e <= tol).all()), (what, float(e.max()), float((e / tol).max()))


def _decode(st, q, **kw):
    err = _err()
    B = len(st.lens)
    qsl = kw.pop("qsl", torch.arange(B + 1, dtype=torch.int32, device="cuda"))
    out = kernels.nibble_decode_paged(st.lay, q, st.page, st.block, st.bt, st.seq, qsl,
                                      kw.pop("max_seq", max(st.lens)), SCALE, error_word=err, **kw)
    torch.cuda.synchronize()
    return out, int(err)


# ------------------------------------------------------------------------------------- write
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,n,pad", [(1, 1, 0), (2, 17, 32), (8, 5, 0), (3, 40, 16)])
def test_write_bytes(dtype, H, n, pad):
    """Every byte of the page, also those no token owns; the stored values; padded tokens."""
    g = _gen(n)
    k, v = (torch.randn(n, H, D, generator=g) for _ in range(2))
    k *= 2.0 ** torch.randint(-18, 12, (n, 1, 1), generator=g)
    k[..., :64] = torch.where(torch.rand(n, H, 1, generator=g) < 0.3,
                              torch.arange(64) / 4 - 3, k[..., :64])
    v[0, 0, 33], v[-1, -1, 100] = float("nan"), -float("inf")
    v[n // 2, 0, :32] *= 3e4
    if n > 2:
        v[2] = 0
    k, v = k.to(dtype), v.to(dtype)
    stride, n_slots = 144 * H + pad, 96
    slots = torch.randperm(n_slots, generator=g)[:n]
    if n > 3:
        slots[3] = -1
    page = torch.randint(0, 256, (6, 16, stride), generator=g, dtype=torch.uint8)
    want = page.reshape(-1).clone()
    on.write(want, stride, slots, k, v)
    dev, err = page.cuda(), _err()
    ko = torch.full((n, H, D), 7.0, dtype=torch.float16, device="cuda")
    vo = ko.clone()
    kernels.nibble_write_paged(NibbleLayout(H), k.cuda(), v.cuda(), slots.cuda(), dev, key_out=ko,
                               value_out=vo, error_word=err)
    assert int(err) == 0
    assert torch.equal(dev.cpu().reshape(-1), want)
    for o, x in ((ko, k), (vo, v)):
        ref = on.values(x)
        ref[slots < 0] = 7
        assert torch.equal(o.cpu().double().nan_to_num(1e30), ref.nan_to_num(1e30))


def test_write_strided_rows_and_bad_slots():
    """Rows inside a wider projection; a slot past the cache sets its bit and touches nothing."""
    g, H, n = _gen(3), 8, 9
    qkv = torch.randn(n, 40 * D, generator=g).half()
    k, v = (qkv[:, 24 * D + 8 * D * i:][:, :8 * D].unflatten(1, (H, D)) for i in range(2))
    slots = torch.arange(n) + 20
    slots[4] = 64
    page = torch.zeros(4, 16, 1152, dtype=torch.uint8)
    want = page.reshape(-1).clone()
    keep = slots < 64
    on.write(want, 1152, slots[keep], k[keep], v[keep])
    dev, err, d = page.cuda(), _err(), qkv.cuda()
    kd, vd = (d[:, 24 * D + 8 * D * i:][:, :8 * D].unflatten(1, (H, D)) for i in range(2))
    kernels.nibble_write_paged(NibbleLayout(H), kd, vd, slots.cuda(), dev, error_word=err)
    assert int(err) == 4
    assert torch.equal(dev.cpu().reshape(-1), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,first", [(2048, 0), (700, 7), (333, 16), (64, 5)])
def test_write_chunk(dtype, n, first):
    """A chunk of consecutive slots, from any offset in a tile; keys and values of unlike types."""
    g, H = _gen(n), 2
    k = (torch.randn(n, H, D, generator=g) * 3).to(dtype)
    v = torch.randn(n, H, D, generator=g).half()
    blocks = (n + first + 31) // 32 + 1
    slots = torch.arange(n) + first
    page = torch.full((blocks, 32, 288), 170, dtype=torch.uint8, device="cuda")
    ko = torch.zeros(n, H, D, dtype=torch.float16, device="cuda")
    err = _err()
    kernels.nibble_write_paged(NibbleLayout(H), k.cuda(), v.cuda(), slots.cuda(), page,
                               key_out=ko, error_word=err)
    assert int(err) == 0
    flat = page.reshape(-1)
    K, V = on.read(flat, 288, slots, H)
    assert torch.equal(K, on.values(k)) and torch.equal(V, on.values(v))
    assert torch.equal(ko.cpu().double(), K)
    # slots that were not written hold what they held
    other = torch.tensor([s for s in range(blocks * 32) if s < first or s >= first + n])
    blank = torch.full_like(flat, 170).cpu()
    for got, ref in zip(on.read(flat, 288, other, H), on.read(blank, 288, other, H)):
        assert torch.equal(got, ref)


def test_write_far_slots():
    """Slots whose bytes lie past 4 GiB (and a read of them)."""
    H, lay = 8, NibbleLayout(8)
    blocks = (5 << 30) // (16 * 1152)
    page = torch.empty(blocks, 16, 1152, dtype=torch.uint8, device="cuda")
    n, g = 40, _gen(5)
    ids = [blocks - 1, 3, blocks - 2]
    bt = _i32([ids])
    slots = on.table_slots(bt[0], n, 16)
    k, v = (torch.randn(n, H, D, generator=g).half() for _ in range(2))
    err = _err()
    kernels.nibble_write_paged(lay, k.cuda(), v.cuda(), slots.cuda(), page, error_word=err)
    q = torch.randn(2, 24, D, generator=g).half()
    out = kernels.nibble_decode_paged(lay, q[:1].cuda(), page, 16, bt, _i32([n]), _i32([0, 1]), n,
                                      SCALE, error_word=err)
    _close(out, q[:1], on.values(k), on.values(v), SCALE, "decode")
    out = kernels.nibble_prefill_paged(lay, q.cuda(), page, 16, bt, _i32([n]), _i32([0, 2]), 2, n,
                                       SCALE, error_word=err)
    _close(out, q, on.values(k), on.values(v), SCALE, "prefill")
    assert int(err) == 0


# ------------------------------------------------------------------------------------ decode
@pytest.mark.parametrize("H,HQ", [(8, 24), (8, 32), (4, 28), (1, 8), (2, 2), (1, 16), (3, 15)])
def test_decode_heads(H, HQ):
    st = Store([1, 37, 500, 16, 1201], H, seed=H + HQ)
    q = torch.randn(5, HQ, D, generator=_gen(1)).half()
    out, err = _decode(st, q.cuda())
    assert err == 0
    for r in range(5):
        _close(out[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, (H, HQ, r))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block", [16, 32, 48])
@pytest.mark.parametrize("lens", [[0, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65],
                                  [127, 128, 129, 255, 1, 257], [3001], [2, 0, 9000, 5]])
def test_decode_lengths(dtype, block, lens):
    """Lengths around every tile, block and split border; the slots behind the last token hold
    parameters that are NaN; an empty request gives zeros."""
    st = Store(lens, 2, block, seed=sum(lens), dtype=dtype)
    q = torch.randn(len(lens), 8, D, generator=_gen(2)).to(dtype)
    out, err = _decode(st, q.cuda())
    assert err == 0
    for r in range(len(lens)):
        _close(out[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, lens[r])


def test_decode_many_requests():
    g = _gen(9)
    lens = [int(x) for x in torch.randint(0, 300, (300,), generator=g)]
    st = Store(lens, 1, seed=9)
    q = torch.randn(300, 4, D, generator=g).half()
    out, err = _decode(st, q.cuda())
    assert err == 0
    for r in range(300):
        _close(out[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, r)


def test_decode_rows_strides_and_out():
    """Queries inside a wider row, rows named by query_start_loc, a wide slot, an output of the
    other type whose other rows stay as they were."""
    st = Store([300, 40], 2, seed=4, pad=48)
    buf = torch.randn(6, 8, D, generator=_gen(4)).half().cuda()
    q = buf.reshape(6, 8 * D)[:, :4 * D].unflatten(1, (4, D))
    out = torch.full((6, 4, D), 9.0, dtype=torch.bfloat16, device="cuda")
    got, err = _decode(st, q, out=out, qsl=_i32([4, 1, 6]))
    assert err == 0 and got is out
    for r, row in enumerate((4, 1)):
        _close(out[row:row + 1], q[row:row + 1].cpu(), *st.kv(r), SCALE, r)
    assert bool((out[[0, 2, 3, 5]] == 9).all())


def test_decode_bad_blocks_and_lengths():
    """A block outside the cache makes its request's rows NaN and no other's; a length past
    max_seq_len is cut to it; both set their bits."""
    for bad in (-1, 10 ** 6):
        st = Store([500, 500, 200], 2, seed=6)
        st.bt[1, 17] = bad
        q = torch.randn(3, 6, D, generator=_gen(6)).half()
        out, err = _decode(st, q.cuda())
        assert err == 2
        assert bool(torch.isnan(out[1]).all())
        for r in (0, 2):
            _close(out[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, r)
    st = Store([500, 100], 2, seed=7)
    q = torch.randn(2, 6, D, generator=_gen(7)).half()
    out, err = _decode(st, q.cuda(), max_seq=200)
    assert err == 8
    K, V = st.kv(0)
    _close(out[:1], q[:1], K[:200], V[:200], SCALE, "cut")
    _close(out[1:], q[1:], *st.kv(1), SCALE, "whole")
    st.seq[0] = -5
    out, err = _decode(st, q.cuda(), max_seq=200)
    assert not bool(out[0].any())


def test_decode_large_and_small_values():
    """Value rows whose scales span the format's range, queries that fp16 cannot hold without a
    row scale, and a flat softmax over many tokens."""
    n = 3000
    f = 10.0 ** torch.linspace(-3, 4, n)
    for dtype, scale in ((torch.float16, 1e-3), (torch.float16, f), (torch.bfloat16, f.flip(0))):
        st = Store([n], 1, seed=8, scale=scale, dtype=dtype)
        q = torch.randn(1, 4, D, generator=_gen(8)) * 0.05
        q = q.to(dtype)
        out, err = _decode(st, q.cuda())
        _close(out, q, *st.kv(0), SCALE, "values")
    st = Store([100], 1, seed=10, dtype=torch.bfloat16)
    q = torch.randn(1, 4, D, generator=_gen(10)) * torch.tensor([1e6, 1e-9, 1.0, 3e38 / 8]).reshape(
        1, 4, 1)
    q = q.bfloat16()
    err = _err()
    for scale, heads in ((1e-7, [0, 1]), (1e6, [1]), (SCALE, [2]), (1e-38, [3])):
        out = kernels.nibble_decode_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq,
                                          _i32([0, 1]), 100, scale, error_word=err)
        for p in heads:
            K, V = st.kv(0)
            _close(out[:, p:p + 1], q[:, p:p + 1], K, V, scale, (scale, p))


def test_decode_nan_groups_and_far_scores():
    """A stored NaN reaches the outputs of its own request and KV head alone; scores of which one
    dwarfs the rest, late and early."""
    st = Store([64, 64], 2, seed=11)
    k = st.k.clone().cuda()
    k[10, 1, 3] = float("nan")
    err = _err()
    kernels.nibble_write_paged(st.lay, k, st.v.cuda(), st.slots.cuda(), st.page, error_word=err)
    q = torch.randn(2, 4, D, generator=_gen(11)).half()
    out, _ = _decode(st, q.cuda())
    assert bool(torch.isnan(out[0, 2:]).all())
    _close(out[:1, :2], q[:1, :2], *(x[:, :1] for x in st.kv(0)), SCALE, "other head")
    _close(out[1:], q[1:], *st.kv(1), SCALE, "other request")
    for at in (0, 900, 1999):
        st = Store([2000], 1, seed=12)
        st.k[at] = (st.k[at] * 30).clamp(-30000, 30000)
        kernels.nibble_write_paged(st.lay, st.k.cuda(), st.v.cuda(), st.slots.cuda(), st.page,
                                   error_word=err)
        q = st.k[at:at + 1].expand(1, 2, D) / 30
        out, _ = _decode(st, q.cuda().contiguous())
        _close(out, q, *st.kv(0), SCALE, at)


def test_decode_workspace_serves_other_shapes():
    """One workspace for calls of different shapes in turn, and calls that repeat exactly."""
    shapes = [([9000, 3, 700], 8, 24), ([100] * 40, 2, 8), ([14402], 1, 16)]
    need = max(kernels.nibble_decode_workspace(NibbleLayout(H), HQ, len(l), max(l), "cpu").numel()
               for l, H, HQ in shapes)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for lens, H, HQ in shapes * 2:
        st = Store(lens, H, seed=len(lens))
        q = torch.randn(len(lens), HQ, D, generator=_gen(3)).half()
        out, err = _decode(st, q.cuda(), workspace=ws)
        again, _ = _decode(st, q.cuda(), workspace=ws)
        assert err == 0 and torch.equal(out, again)
        for r in range(0, len(lens), 13):
            _close(out[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, (lens[r], H))


# ----------------------------------------------------------------------------------- prefill
def _prefill(st, q, counts, **kw):
    err = _err()
    qsl = [0]
    for c in counts:
        qsl.append(qsl[-1] + c)
    out = kernels.nibble_prefill_paged(st.lay, q, st.page, st.block, st.bt, st.seq, _i32(qsl),
                                       kw.pop("max_q", max(counts)), kw.pop("max_seq", max(st.lens)),
                                       SCALE, error_word=err, **kw)
    torch.cuda.synchronize()
    return out, int(err), qsl


@pytest.mark.parametrize("H,HQ", [(8, 24), (2, 8), (1, 7), (2, 2), (1, 16), (1, 5)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_heads(H, HQ, dtype):
    lens, counts = [40, 1, 333, 190], [40, 1, 50, 65]     # first chunks and continuations
    st = Store(lens, H, seed=HQ, dtype=dtype)
    q = torch.randn(sum(counts), HQ, D, generator=_gen(1)).to(dtype)
    out, err, qsl = _prefill(st, q.cuda(), counts)
    assert err == 0
    for r in range(4):
        s = slice(qsl[r], qsl[r + 1])
        _close(out[s], q[s], *st.kv(r), SCALE, (H, HQ, r))


@pytest.mark.parametrize("block", [16, 48])
@pytest.mark.parametrize("lens,counts", [
    ([15, 16, 17, 33], [15, 3, 17, 1]), ([64, 65, 63, 128, 129], [64, 64, 63, 2, 129]),
    ([1000], [257]), ([5000, 100], [31, 100]), ([2500], [600])])
def test_prefill_lengths(block, lens, counts):
    st = Store(lens, 2, block, seed=sum(lens))
    q = torch.randn(sum(counts), 6, D, generator=_gen(2)).half()
    out, err, qsl = _prefill(st, q.cuda(), counts)
    assert err == 0
    for r in range(len(lens)):
        s = slice(qsl[r], qsl[r + 1])
        _close(out[s], q[s], *st.kv(r), SCALE, (lens[r], counts[r]))


def test_prefill_picked_rows_and_empty_chunks():
    """req_index picks the rows of the batch; the others' rows, and requests without queries, are
    left as they were."""
    lens, counts = [100, 200, 300, 50], [20, 1, 0, 33]
    st = Store(lens, 2, seed=3)
    q = torch.randn(54, 8, D, generator=_gen(3)).half()
    out = torch.full((54, 8, D), 5.0, dtype=torch.float16, device="cuda")
    _, err, qsl = _prefill(st, q.cuda(), counts, out=out, req_index=_i32([3, 2, 0]))
    assert err == 0
    for r in (3, 0):
        s = slice(qsl[r], qsl[r + 1])
        _close(out[s], q[s], *st.kv(r), SCALE, r)
    assert bool((out[20:21] == 5).all())


@pytest.mark.parametrize("lens,counts", [([300, 4000], [20, 3]), ([300, 4000], [200, 90])])
def test_prefill_of_a_row_picked_twice(lens, counts):
    st = Store(lens, 2, seed=33)
    q = torch.randn(sum(counts), 8, D, generator=_gen(34)).half().cuda()
    want, err, qsl = _prefill(st, q, counts)
    got, err2, _ = _prefill(st, q, counts, req_index=_i32([1, 0, 1]))
    assert err == 0 and err2 == 0
    for r in range(2):
        s = slice(qsl[r], qsl[r + 1])
        _close(got[s], q[s].cpu(), *st.kv(r), SCALE, r)


def test_prefill_refuses_on_the_device():
    """Fewer keys than queries, a block outside the cache, a count past max_q_len."""
    lens, counts = [100, 30, 200, 64], [10, 31, 20, 12]
    st = Store(lens, 2, seed=5)
    st.bt[2, 3] = st.blocks
    q = torch.randn(sum(counts), 8, D, generator=_gen(5)).half()
    out, err, qsl = _prefill(st, q.cuda(), counts)
    assert err == 8 | 2
    assert bool(torch.isnan(out[qsl[1]:qsl[3]]).all())
    for r in (0, 3):
        s = slice(qsl[r], qsl[r + 1])
        _close(out[s], q[s], *st.kv(r), SCALE, r)
    st = Store([100], 2, seed=6)
    q = torch.randn(20, 8, D, generator=_gen(6)).half()
    out = torch.full((20, 8, D), 5.0, dtype=torch.float16, device="cuda")
    _, err, _ = _prefill(st, q.cuda(), [20], max_q=7, out=out)
    assert err == 8
    K, V = st.kv(0)
    _close(out[:7], q[:7], K[:87], V[:87], SCALE, "counted")
    assert bool((out[7:] == 5).all())


def test_prefill_large_and_small_values():
    n = 700
    f = 10.0 ** torch.linspace(-3, 4, n)
    for dtype, scale in ((torch.float16, 1e-3), (torch.float16, f), (torch.bfloat16, f.flip(0))):
        st = Store([n], 1, seed=8, scale=scale, dtype=dtype)
        q = (torch.randn(90, 4, D, generator=_gen(8)) * 0.05).to(dtype)
        out, err, _ = _prefill(st, q.cuda(), [90])
        assert err == 0
        _close(out, q, *st.kv(0), SCALE, "values")
    st = Store([100], 1, seed=10, dtype=torch.bfloat16)
    q = torch.randn(30, 2, D, generator=_gen(10)) * torch.tensor([1e6, 1e-9]).reshape(1, 2, 1)
    q = q.bfloat16()
    err = _err()
    for scale in (1e-7, 1e-6):
        out = kernels.nibble_prefill_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq,
                                           _i32([0, 30]), 30, 100, scale, error_word=err)
        _close(out, q, *st.kv(0), scale, scale)


@pytest.mark.parametrize("H,HQ,n,Q,at", [(1, 4, 300, 100, 230), (1, 4, 70, 70, 3), (1, 2, 90, 8, 85),
                                         (1, 16, 33, 1, 20), (1, 3, 640, 130, 575)])
@pytest.mark.parametrize("what", ["value", "key"])
def test_prefill_nan_stays_behind(H, HQ, n, Q, at, what):
    """A NaN in a token's value (one group) or key reaches the queries that see the token and no
    query before it, in the same tile or not."""
    st = Store([n], H, seed=n, dtype=torch.float16)
    k, v = st.k.clone(), st.v.clone()
    (v if what == "value" else k)[at, 0, 37] = float("nan")
    kernels.nibble_write_paged(st.lay, k.cuda(), v.cuda(), st.slots.cuda(), st.page)
    q = torch.randn(Q, HQ, D, generator=_gen(n)).half()
    out, err, _ = _prefill(st, q.cuda(), [Q])
    assert err == 0
    clear = max(0, min(Q, at - (n - Q)))         # queries before the token
    K, V = st.kv(0)
    if clear:
        _close(out[:clear], q[:clear], K[:n - Q + clear], V[:n - Q + clear], SCALE, "before")
    rest = out[clear:]
    if what == "key":
        assert bool(torch.isnan(rest).all())
    else:
        nan = torch.isnan(rest)
        assert bool(nan[..., 32:64].all()) and not bool(nan[..., :32].any() or nan[..., 64:].any())


@pytest.mark.parametrize("scale", [0.0, -SCALE, 2.0])
def test_scales_of_any_sign(scale):
    """Zero (a plain mean), negative, and large enough that one key takes nearly all."""
    for dtype in (torch.float16, torch.bfloat16):
        st = Store([333, 40], 2, seed=14, dtype=dtype)
        q = torch.randn(2, 8, D, generator=_gen(14)).to(dtype)
        qsl = torch.arange(3, dtype=torch.int32, device="cuda")
        out = kernels.nibble_decode_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq, qsl, 333,
                                          scale)
        for r in range(2):
            _close(out[r:r + 1], q[r:r + 1], *st.kv(r), scale, r)
        q = torch.randn(70, 8, D, generator=_gen(15)).to(dtype)
        out = kernels.nibble_prefill_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq,
                                           _i32([0, 40, 70]), 40, 333, scale)
        for r, s in ((0, slice(0, 40)), (1, slice(40, 70))):
            _close(out[s], q[s], *st.kv(r), scale, r)


def test_prefill_many_requests_and_long_splits():
    """More requests than a launch's plan holds, with chunks of both kernels; one long request whose
    keys are split many times."""
    g = _gen(16)
    for most in (3, 40):
        counts = [int(x) for x in torch.randint(0, most + 1, (300,), generator=g)]
        lens = [c + int(x) for c, x in zip(counts, torch.randint(0, 150, (300,), generator=g))]
        st = Store(lens, 1, seed=most)
        q = torch.randn(sum(counts), 4, D, generator=g).half()
        out, err, qsl = _prefill(st, q.cuda(), counts, max_q=most)
        assert err == 0
        for r in range(0, 300, 7):
            s = slice(qsl[r], qsl[r + 1])
            if counts[r]:
                _close(out[s], q[s], *st.kv(r), SCALE, r)
    for Q in (2, 33):
        st = Store([20011], 1, seed=17)
        q = torch.randn(Q, 5, D, generator=g).half()
        out, err, _ = _prefill(st, q.cuda(), [Q])
        again, _, _ = _prefill(st, q.cuda(), [Q])
        assert err == 0 and torch.equal(out, again)
        _close(out, q, *st.kv(0), SCALE, Q)


@pytest.mark.parametrize("H,HQ,lens,counts", [
    (2, 2, [700] * 17, [700] * 17), (1, 2, [1500] * 18, [1500] * 18), (2, 2, [2001] * 20, [900] * 20),
    (1, 2, [5000] + [70] * 15, [300] + [70] * 15), (1, 2, [5000] + [70] * 39, [300] + [70] * 39),
    (2, 4, [64, 65] * 8, [64, 63] * 8), (1, 4, [9000], [130])])
def test_prefill_batches_write_every_row(H, HQ, lens, counts):
    """Prompts of many row blocks each, and one long among short: every row is written, by whatever
    rows per block and key parts the plan takes."""
    st = Store(lens, H, seed=20)
    q = torch.randn(sum(counts), HQ, D, generator=_gen(21)).half()
    out = torch.full((sum(counts), HQ, D), float("nan"), dtype=torch.float16, device="cuda")
    _, err, qsl = _prefill(st, q.cuda(), counts, out=out)
    assert err == 0
    assert not bool(torch.isnan(out).any())
    for r in (0, len(lens) // 2, len(lens) - 1):
        s = slice(qsl[r], qsl[r + 1])
        _close(out[s], q[s], *st.kv(r), SCALE, r)


@pytest.mark.parametrize("R,H,HQ,most,longest", [
    (70, 4, 16, 7, 300), (33, 8, 24, 10, 90), (300, 1, 5, 5, 70), (140, 2, 4, 16, 33), (3, 8, 32, 8, 26000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_of_many_short_chunks(R, H, HQ, most, longest, dtype):
    """Chunks of 17 to 32 rows per KV head in batches large enough for two groups of 16 rows to share a
    block, ragged, and a NaN in a value that only the queries at or after it may see."""
    g = _gen(R + most)
    counts = [most] + [int(torch.randint(0, most + 1, (1,), generator=g)) for _ in range(R - 1)]
    lens = [longest] + [c + int(torch.randint(0, longest - most, (1,), generator=g)) for c in counts[1:]]
    st = Store(lens, H, seed=40, dtype=dtype)
    q = torch.randn(sum(counts), HQ, D, generator=g).to(dtype)
    out = torch.full((sum(counts), HQ, D), float("nan"), dtype=dtype, device="cuda")
    _, err, qsl = _prefill(st, q.cuda(), counts, out=out)
    assert err == 0 and not bool(torch.isnan(out).any())
    for r in {0, 1, R // 2, R - 1}:
        s = slice(qsl[r], qsl[r + 1])
        if counts[r]:
            _close(out[s], q[s], *st.kv(r), SCALE, (r, lens[r], counts[r]))
    k, v = st.k.clone(), st.v.clone()
    at = lens[0] - most + 2                       # seen by the queries from 2 on
    v[at, 0, 40] = float("nan")
    page = st.page.clone()
    kernels.nibble_write_paged(st.lay, k.cuda(), v.cuda(), st.slots.cuda(), page)
    bad = kernels.nibble_prefill_paged(st.lay, q.cuda(), page, st.block, st.bt, st.seq, _i32(qsl), most,
                                       max(lens), SCALE)
    G = HQ // H
    nan = torch.isnan(bad[:most, :G])
    assert bool(nan[2:, :, 32:64].all()) and not bool(nan[:2].any())
    assert not bool(nan[:, :, :32].any()) and not bool(nan[:, :, 64:].any())
    nan = torch.isnan(bad)
    nan[:most, :G] = False
    assert not bool(nan.any())


def test_prefill_workspace_serves_other_shapes():
    """One workspace for prefill calls of different shapes and for decode calls in turn."""
    shapes = [([5000, 300], 2, 8, [70, 20]), ([900, 64, 30], 1, 4, [3, 1, 2]), ([1200], 4, 12, [400])]
    ws = torch.zeros(max(
        [kernels.nibble_prefill_workspace(NibbleLayout(H), HQ, len(l), max(c), max(l), "cpu").numel()
         for l, H, HQ, c in shapes]
        + [kernels.nibble_decode_workspace(NibbleLayout(2), 8, 3, 2000, "cpu").numel()]),
        dtype=torch.uint8, device="cuda")
    for lens, H, HQ, counts in shapes * 2:
        st = Store(lens, H, seed=len(lens))
        q = torch.randn(sum(counts), HQ, D, generator=_gen(3)).half()
        out, err, qsl = _prefill(st, q.cuda(), counts, workspace=ws)
        assert err == 0
        for r in range(len(lens)):
            s = slice(qsl[r], qsl[r + 1])
            _close(out[s], q[s], *st.kv(r), SCALE, (lens[r], H))
        st, dq, qd, _ = _decode_args(50)
        out, err = _decode(st, dq, workspace=ws)
        assert err == 0
        for r in range(3):
            _close(out[r:r + 1], dq[r:r + 1].cpu(), *st.kv(r), SCALE, r)


def test_the_largest_length_a_call_may_name():
    """max_seq_len of 2^26, as a captured server would have it, over short requests."""
    most = 1 << 26
    st = Store([400, 90], 2, seed=41)
    table = torch.full((2, most // 16), -1, dtype=torch.int32, device="cuda")
    table[:, :st.bt.shape[1]] = st.bt
    st.bt = table
    for counts in ([1, 1], [5, 9], [300, 90]):
        q = torch.randn(sum(counts), 8, D, generator=_gen(42)).half()
        out, err, qsl = _prefill(st, q.cuda(), counts, max_seq=most, max_q=max(counts) + 3)
        assert err == 0
        for r in range(2):
            s = slice(qsl[r], qsl[r + 1])
            _close(out[s], q[s], *st.kv(r), SCALE, (counts, r))
    out, err = _decode(st, q[:2].cuda(), max_seq=most)
    assert err == 0
    for r in range(2):
        _close(out[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, r)


@pytest.mark.parametrize("lens,counts", [([300, 5000], [300, 40]), ([5000, 90], [9, 3]),
                                         ([700], [128]), ([20000, 1], [1, 1])])
def test_the_output_may_be_the_query(lens, counts):
    st = Store(lens, 2, seed=30)
    q = torch.randn(sum(counts), 8, D, generator=_gen(31)).half()
    want, err, qsl = _prefill(st, q.cuda(), counts)
    got = q.cuda()
    _prefill(st, got, counts, out=got)
    assert err == 0 and torch.equal(got, want)
    if counts == [1] * len(counts):
        want, _ = _decode(st, q.cuda())
        got = q.cuda()
        _decode(st, got, out=got)
        assert torch.equal(got, want)


def test_prefill_and_decode_agree_on_one_query():
    st = Store([777, 20], 2, seed=13)
    q = torch.randn(2, 8, D, generator=_gen(13)).half()
    a, _ = _decode(st, q.cuda())
    b, _, _ = _prefill(st, q.cuda(), [1, 1])
    for r in range(2):
        for o in (a, b):
            _close(o[r:r + 1], q[r:r + 1], *st.kv(r), SCALE, r)


# -------------------------------------------------------------------------------- rotary axes
def _angles(n, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
    f = torch.outer(torch.arange(n).double(), inv)
    return torch.cat([f.cos(), f.sin()], 1).float()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sections,interleaved,rot,d", [
    ((64,), False, 128, 128), ((16, 24, 24), False, 128, 128), ((24, 20, 20), True, 128, 128),
    ((12, 10, 10), True, 64, 128), ((10, 0, 38), False, 96, 128), ((20, 15), False, 70, 80),
    ((10, 9, 8, 8), True, 70, 72), ((33, 31), True, 128, 192), ((3, 2), True, 10, 10)])
def test_rotary(dtype, sections, interleaved, rot, d):
    """y within one rounding of the type, and of two products and a sum in 32 bits (3 * 2^-24 of
    |x cos| + |x' sin|)."""
    g, N, HQ, H = _gen(rot), 37, 5, 2
    pos = torch.randint(0, 500, (len(sections), N), generator=g)
    cs = _angles(500, rot)
    q = torch.randn(N, HQ, d, generator=g).to(dtype)
    k = (torch.randn(N, H, d, generator=g) * 8).to(dtype)
    err = _err()
    qo, ko = kernels.rotary_axes(q.cuda(), k.cuda(), pos.cuda(), cs.cuda(), sections,
                                 interleaved=interleaved, error_word=err)
    assert int(err) == 0
    for x, y in ((q, qo), (k, ko)):
        want = on.rotary(x, pos, cs, sections, interleaved)
        both = x.double().abs()
        big = torch.zeros_like(both)
        big[..., :rot // 2] = both[..., :rot // 2] + both[..., rot // 2:rot]
        big[..., rot // 2:rot] = big[..., :rot // 2]
        tol = HALF[dtype] * want.abs() * 1.01 + 3 * 2.0 ** -24 * big + 2.0 ** -25 * (
            dtype == torch.float16)
        assert bool(((y.cpu().double() - want).abs() <= tol).all())
        assert torch.equal(y.cpu()[..., rot:], x[..., rot:])


def test_rotary_in_place_strided_and_alone():
    """In place inside a projection's rows; queries alone; one axis as a vector."""
    g, N = _gen(2), 19
    qkv = torch.randn(N, 40 * D, generator=g).half()
    pos = torch.randint(0, 300, (3, N), generator=g)
    cs = _angles(300, 128)
    d = qkv.cuda()
    q, k = d[:, :24 * D].unflatten(1, (24, D)), d[:, 24 * D:32 * D].unflatten(1, (8, D))
    q1, k1 = kernels.rotary_axes(q.contiguous(), k.contiguous(), pos.cuda(), cs.cuda(),
                                 (16, 24, 24))
    kernels.rotary_axes(q, k, pos.cuda(), cs.cuda(), (16, 24, 24), query_out=q, key_out=k)
    assert torch.equal(q, q1) and torch.equal(k, k1)
    assert torch.equal(d[:, 32 * D:].cpu(), qkv[:, 32 * D:])
    x = qkv[:, :24 * D].unflatten(1, (24, D)).contiguous()
    y, none = kernels.rotary_axes(x.cuda(), None, pos[0].cuda(), cs.cuda(), (64,))
    assert none is None
    three, _ = kernels.rotary_axes(x.cuda(), None, pos[:1].expand(3, N).contiguous().cuda(),
                                   cs.cuda(), (16, 24, 24))
    assert torch.equal(y, three)        # equal positions on every axis are the one position
    assert kernels.rotary_axes(x[:0].cuda(), None, pos[0, :0].cuda(), cs.cuda(),
                               (64,))[0].shape[0] == 0


def test_rotary_bad_positions():
    g, N = _gen(4), 6
    pos = torch.randint(0, 100, (3, N), generator=g)
    pos[1, 2], pos[2, 4] = 100, -1
    cs, q = _angles(100, 64), torch.randn(N, 4, D, generator=g).half()
    err = _err()
    y, _ = kernels.rotary_axes(q.cuda(), None, pos.cuda(), cs.cuda(), (12, 10, 10),
                               error_word=err)
    assert int(err) == 16
    nan = torch.isnan(y).all(-1).all(-1).tolist()
    assert nan == [False, False, True, False, True, False]
    assert bool(torch.isfinite(y[[0, 1, 3, 5]]).all())


# ---------------------------------------------------------------------------------- step plan
def _plan_case(seed, R, block, cmax, qmax):
    g = _gen(seed)
    c = torch.randint(0, cmax + 1, (R,), generator=g)
    n = torch.randint(0, qmax + 1, (R,), generator=g)
    held, need = (c + block - 1) // block, (c + n + block - 1) // block
    W = max(int(need.max()), 1)
    total = int(need.sum()) + 7
    perm = torch.randperm(total, generator=g).to(torch.int32)
    bt = torch.full((R, W), -1, dtype=torch.int32)
    at = 0
    for r in range(R):
        bt[r, :held[r]] = perm[at:at + int(held[r])]
        at += int(held[r])
    return c.int(), n.int(), bt, perm[at:], total, int(n.sum())


def _check_plan(c, n, bt, free, block, blocks, T, want_err=0):
    want = on.plan(c.tolist(), n.tolist(), bt.tolist(), free.tolist(), block, blocks, T)
    dev, err = bt.cuda(), _err()
    p = kernels.step_plan(c.cuda(), n.cuda(), dev, free.cuda(), block, blocks, T, error_word=err)
    got = [t.tolist() for t in p[:4]] + [int(p.blocks_used), dev.tolist()]
    assert int(err) == want_err
    for name, a, b in zip(("qsl", "seq", "slots", "pos", "used", "table"), got, want):
        assert a == b, name


@pytest.mark.parametrize("R,block,cmax,qmax,pad", [
    (1, 16, 0, 1, 0), (1, 16, 100, 40, 5), (8, 16, 300, 1, 0), (63, 32, 200, 30, 100),
    (257, 48, 500, 3, 0), (1000, 16, 60, 9, 31), (8000, 16, 20, 2, 1), (5, 5, 30, 3000, 0)])
def test_plan(R, block, cmax, qmax, pad):
    c, n, bt, free, blocks, total = _plan_case(R, R, block, cmax, qmax)
    _check_plan(c, n, bt, free, block, blocks, total + pad)


def test_plan_conditions():
    """A free list too short, a row too narrow, more tokens than outputs, ids outside the cache, a
    negative length, no requests."""
    c, n, bt, free, blocks, total = _plan_case(3, 20, 16, 100, 40)
    _check_plan(c, n, bt, free[:4], 16, blocks, total, want_err=32)
    _check_plan(c, n, bt[:, :5].contiguous(), free, 16, blocks, total, want_err=8)
    _check_plan(c, n, bt, free, 16, blocks, total - 30, want_err=8)
    _check_plan(c, n, bt, free, 16, blocks - 40, total, want_err=2)
    err = _err()
    c[3], n[5] = -2, -7
    p = kernels.step_plan(c.cuda(), n.cuda(), bt.cuda(), free.cuda(), 16, blocks, total,
                          error_word=err)
    assert int(err) & 8 and int(p.seq_lens[5]) == int(c[5]) and int(p.seq_lens[3]) == int(n[3])
    none = torch.zeros(0, dtype=torch.int32)
    p = kernels.step_plan(none.cuda(), none.cuda(), torch.zeros(0, 4, dtype=torch.int32).cuda(),
                          free.cuda(), 16, blocks, 3)
    assert p.query_start_loc.tolist() == [0] and p.slot_mapping.tolist() == [-1] * 3


# ------------------------------------------------------------------------------ run together
class Serving:
    """A server's loop over the 4-bit cache: plan, rotate, write, attend."""

    def __init__(self, B, H, HQ, block, seed):
        self.B, self.H, self.HQ, self.block = B, H, HQ, block
        self.lay, self.g = NibbleLayout(H), _gen(seed)
        self.blocks = 80
        self.page = torch.full((self.blocks, block, 144 * H), 255, dtype=torch.uint8,
                               device="cuda")
        self.free = torch.randperm(self.blocks, generator=self.g).to(torch.int32).cuda()
        self.bt = torch.full((B, 20), -1, dtype=torch.int32, device="cuda")
        self.computed = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.cs = _angles(4000, D).cuda()
        self.err = _err()
        self.K = [torch.zeros(0, H, D).double() for _ in range(B)]
        self.V = [torch.zeros(0, H, D).double() for _ in range(B)]

    def inputs(self, counts):
        N = sum(counts)
        q, k, v = (torch.randn(N, h, D, generator=self.g).half()
                   for h in (self.HQ, self.H, self.H))
        pos = torch.randint(0, 4000, (3, N), generator=self.g)
        return q, k, v, pos

    def note(self, counts, k, v, pos):
        """The oracle's view of what the step stores."""
        # rotated keys are rounded to fp16 by the operator; its own test bounds that rounding
        kr = kernels.rotary_axes(k.cuda(), None, pos.cuda(), self.cs, (16, 24, 24))[0].cpu()
        at = 0
        for r, c in enumerate(counts):
            self.K[r] = torch.cat([self.K[r], on.values(kr[at:at + c])])
            self.V[r] = torch.cat([self.V[r], on.values(v[at:at + c])])
            at += c

    def step(self, counts, decode):
        q, k, v, pos = self.inputs(counts)
        n = _i32(counts)
        plan = kernels.step_plan(self.computed, n, self.bt, self.free, self.block, self.blocks,
                                 sum(counts) + 3, error_word=self.err)
        qr, kr = kernels.rotary_axes(q.cuda(), k.cuda(), pos.cuda(), self.cs, (16, 24, 24),
                                     error_word=self.err)
        kernels.nibble_write_paged(self.lay, kr, v.cuda(), plan.slot_mapping, self.page,
                                   error_word=self.err)
        self.note(counts, k, v, pos)
        longest = max(len(x) for x in self.K)
        if decode:
            out = kernels.nibble_decode_paged(self.lay, qr, self.page, self.block, self.bt,
                                              plan.seq_lens, plan.query_start_loc, longest, SCALE,
                                              error_word=self.err)
        else:
            out = kernels.nibble_prefill_paged(self.lay, qr, self.page, self.block, self.bt,
                                               plan.seq_lens, plan.query_start_loc, max(counts),
                                               longest, SCALE, error_word=self.err)
        at = 0
        for r, c in enumerate(counts):
            if c:
                _close(out[at:at + c], qr[at:at + c].cpu(), self.K[r], self.V[r], SCALE, r)
            at += c
        assert plan.seq_lens.tolist() == [len(x) for x in self.K]
        self.computed = plan.seq_lens
        self.free = self.free[int(plan.blocks_used):]
        assert int(self.err) == 0


@pytest.mark.parametrize("block", [16, 32])
def test_serving_loop(block):
    s = Serving(3, 2, 8, block, seed=block)
    s.step([37, 5, 64], decode=False)        # first chunks
    s.step([20, 0, 33], decode=False)        # continuations, one request waits
    for _ in range(4):
        s.step([1, 1, 1], decode=True)
    s.step([1, 16, 1], decode=False)         # a chunk beside decodes


def _decode_args(seed, lens=(700, 33, 2000)):
    st = Store(list(lens), 2, seed=seed)
    q = torch.randn(len(lens), 8, D, generator=_gen(seed)).half().cuda()
    return st, q, torch.arange(len(lens) + 1, dtype=torch.int32, device="cuda"), _err()


def test_on_another_stream():
    st, q, qsl, err = _decode_args(21)
    want, _ = _decode(st, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k, v = st.k.cuda(), st.v.cuda()
        page = torch.full_like(st.page, 255)
        kernels.nibble_write_paged(st.lay, k, v, st.slots.cuda(), page)
        out = kernels.nibble_decode_paged(st.lay, q, page, 16, st.bt, st.seq, qsl, 2000, SCALE)
        pre = kernels.nibble_prefill_paged(st.lay, q, page, 16, st.bt, st.seq, qsl, 1, 2000, SCALE)
    side.synchronize()
    assert torch.equal(out, want)
    for r in range(3):
        _close(pre[r:r + 1], q[r:r + 1].cpu(), *st.kv(r), SCALE, r)


def test_captured_step_replays():
    """A whole step in a graph, replayed with new inputs, lengths and blocks, with eager work on
    another workspace between the replays; two graphs that share a workspace in turn."""
    B, H, HQ, W = 3, 2, 8, 8
    lay, g = NibbleLayout(H), _gen(31)
    blocks = 40
    page = torch.full((blocks, 16, 288), 255, dtype=torch.uint8, device="cuda")
    cs = _angles(200, D).cuda()
    computed, ones = _i32([0, 0, 0]), _i32([1, 1, 1])
    bt = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(blocks, generator=g).to(torch.int32).cuda()
    q, k, v = (torch.zeros(B, h, D, dtype=torch.float16, device="cuda") for h in (HQ, H, H))
    pos = torch.zeros(3, B, dtype=torch.int64, device="cuda")
    ws = kernels.nibble_decode_workspace(lay, HQ, B, 16 * W, "cuda")
    ws2 = kernels.nibble_prefill_workspace(lay, HQ, B, 1, 16 * W, "cuda")
    err = _err()

    def step(chunked):
        p = kernels.step_plan(computed, ones, bt, free, 16, blocks, B + 2, error_word=err)
        qr, kr = kernels.rotary_axes(q, k, pos, cs, (16, 24, 24), error_word=err)
        kernels.nibble_write_paged(lay, kr, v, p.slot_mapping, page, error_word=err)
        args = (lay, qr, page, 16, bt, p.seq_lens, p.query_start_loc)
        if chunked:
            return p, qr, kr, kernels.nibble_prefill_paged(*args, 1, 16 * W, SCALE, workspace=ws2,
                                                           error_word=err)
        return p, qr, kr, kernels.nibble_decode_paged(*args, 16 * W, SCALE, workspace=ws,
                                                      error_word=err)

    pools = []
    for chunked in (False, True, False):
        step(chunked)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(chunked)
        pools.append((graph, got))
    page.fill_(255)
    bt.fill_(-1)
    K, V = [[] for _ in range(B)], [[] for _ in range(B)]
    for t in range(12):
        graph, (p, qr, kr, out) = pools[t % 3]
        q.copy_(torch.randn(B, HQ, D, generator=g))
        k.copy_(torch.randn(B, H, D, generator=g))
        v.copy_(torch.randn(B, H, D, generator=g))
        pos.copy_(torch.randint(0, 200, (3, B), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert int(err) == 0
        for r in range(B):
            K[r].append(on.values(kr[r].cpu()))
            V[r].append(on.values(v[r].cpu()))
            _close(out[r:r + 1], qr[r:r + 1].cpu(), torch.stack(K[r]), torch.stack(V[r]), SCALE,
                   (t, r))
        computed.copy_(p.seq_lens)
        taken = int(p.blocks_used)
        free.copy_(torch.cat([free[taken:], free[:taken]]))
        st, qq, _, _ = _decode_args(40 + t, lens=(100, 50))
        _decode(st, qq)


def test_captured_prefill_replays():
    """Chunks in a graph, with lengths that change on the device between the replays and eager calls of
    both reads on the same workspace."""
    st = Store([2000, 700], 2, seed=36)
    qsl = _i32([0, 200, 290])
    q = torch.zeros(290, 8, D, dtype=torch.float16, device="cuda")
    seq = st.seq.clone()
    ws = kernels.nibble_prefill_workspace(st.lay, 8, 2, 200, 2000, "cuda")
    other = kernels.nibble_prefill_workspace(st.lay, 8, 2, 200, 2000, "cuda")
    err, g = _err(), _gen(37)

    def call(w):
        return kernels.nibble_prefill_paged(st.lay, q, st.page, st.block, st.bt, seq, qsl, 200, 2000,
                                            SCALE, workspace=w, error_word=err)

    call(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(ws)
    for lens in ([2000, 700], [200, 90], [1111, 699], [2000, 90]):
        q.copy_(torch.randn(290, 8, D, generator=g))
        seq.copy_(_i32(lens))
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, call(other)) and int(err) == 0
        for r, s in ((0, slice(0, 200)), (1, slice(200, 290))):
            K, V = st.kv(r)
            _close(got[s], q[s].cpu(), K[:lens[r]], V[:lens[r]], SCALE, (lens, r))
        assert torch.equal(call(ws), got)
        kernels.nibble_decode_paged(st.lay, q, st.page, st.block, st.bt, seq, qsl[:2], 2000, SCALE,
                                    workspace=ws, error_word=err)
        assert not bool(ws[:65536].any())

"""The 4-bit cache's operators at calls that their documentation allows and that go wrong easily:
requests without a query, a plan's tensors within one buffer,
positions of other shapes, outputs that lie in inputs, scores of any size,
small weights in numbers, layers of unlike heads, steps without
tokens. Helpers and tolerances are test_nibble_gpu's."""
import pytest
import torch

from oracle import nibble as on
from test_nibble_gpu import D, HALF, SCALE, Store, _close, _err, _gen, _i32
from vllm_ttkv import kernels
from vllm_ttkv.nibble import NibbleLayout

pytestmark = pytest.mark.gpu


# ----------------------------------------------------------------- requests without a query
def _starts(counts):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return at


def _guarded(rows, heads, dtype=torch.float16, fill=9.0):
    """(output rows, the buffer around them with a row before and three behind)."""
    buf = torch.full((rows + 4, heads, D), fill, dtype=dtype, device="cuda")
    return buf[1:rows + 1], buf


@pytest.mark.parametrize("counts", [[1, 0, 1], [1, 1, 0], [0, 0, 1], [0, 1, 0, 0], [1, 0, 0, 1, 0]])
@pytest.mark.parametrize("longest", [60, 9000])
def test_decode_skips_requests_that_wait(counts, longest):
    """A request with tokens stored and no query this step writes no row, neither the next request's
    nor one past the output."""
    lens = [longest - 7 * r for r in range(len(counts))]
    st = Store(lens, 2, seed=longest)
    n, qsl = sum(counts), _starts(counts)
    q = torch.randn(n, 8, D, generator=_gen(50)).half()
    out, buf = _guarded(n, 8)
    err = _err()
    kernels.nibble_decode_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq, _i32(qsl), longest,
                                SCALE, out=out, error_word=err)
    assert int(err) == 0
    for r, c in enumerate(counts):
        if c:
            _close(out[qsl[r]:qsl[r] + 1], q[qsl[r]:qsl[r] + 1], *st.kv(r), SCALE, r)
    assert bool((buf[0] == 9).all()) and bool((buf[n + 1:] == 9).all())


def test_decode_skips_among_many_requests():
    """More requests than a launch's plan holds, waiting ones on both sides of its border; a batch
    in which all wait."""
    g = _gen(51)
    counts = [int(x) for x in torch.randint(0, 2, (300,), generator=g)]
    counts[254:258], counts[-1] = [1, 0, 0, 1], 0
    lens = [int(x) for x in torch.randint(1, 300, (300,), generator=g)]
    st = Store(lens, 1, seed=51)
    n, qsl = sum(counts), _starts(counts)
    q = torch.randn(n, 4, D, generator=g).half()
    out, buf = _guarded(n, 4)
    err = _err()
    kernels.nibble_decode_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq, _i32(qsl), max(lens),
                                SCALE, out=out, error_word=err)
    assert int(err) == 0
    for r, c in enumerate(counts):
        if c:
            _close(out[qsl[r]:qsl[r] + 1], q[qsl[r]:qsl[r] + 1], *st.kv(r), SCALE, r)
    assert bool((buf[0] == 9).all()) and bool((buf[n + 1:] == 9).all())
    out, buf = _guarded(2, 4)
    kernels.nibble_decode_paged(st.lay, q[:2].cuda(), st.page, 16, st.bt[:3], st.seq[:3],
                                _i32([0, 0, 0, 0]), max(lens), SCALE, out=out, error_word=err)
    assert int(err) == 0 and bool((buf == 9).all())


def test_decode_of_a_planned_step_with_waiting_requests():
    """The plan's own starts, a padded batch whose last requests are empty: their rows, which are
    the padding's, stay as they were."""
    lens = [40, 700, 33]
    st = Store(lens, 2, seed=52)
    err = _err()
    bt = torch.cat([st.bt, torch.full_like(st.bt, -1)])
    computed, query = _i32([39, 700, 32, 0, 0, 0]), _i32([1, 0, 1, 0, 0, 0])
    fresh = st.bt[2, 2:3].clone()        # request 2's new token, its 33rd, opens a block
    p = kernels.step_plan(computed, query, bt, fresh, 16, st.blocks, 4, error_word=err)
    q = torch.randn(4, 8, D, generator=_gen(52)).half()
    out, buf = _guarded(4, 8)
    kernels.nibble_decode_paged(st.lay, q.cuda(), st.page, 16, bt, p.seq_lens, p.query_start_loc,
                                700, SCALE, out=out, error_word=err)
    assert int(err) == 0
    for row, r in ((0, 0), (1, 2)):
        _close(out[row:row + 1], q[row:row + 1], *st.kv(r), SCALE, r)
    assert bool((buf[0] == 9).all()) and bool((buf[3:] == 9).all())


# ----------------------------------------------------------- a plan's tensors within one buffer
def test_plan_of_tensors_that_touch():
    """Lengths, free list and outputs side by side in one buffer, the lengths between the table's
    rows: the same plan as of tensors of their own. Starts into whose tail the query lengths are a
    view are refused."""
    R, W, block, blocks, T = 3, 4, 16, 20, 30
    c, n, free = [20, 0, 33], [5, 17, 2], [11, 12, 13, 14]
    table = torch.full((R, W + R), -1, dtype=torch.int32, device="cuda")
    table[0, :2], table[2, :3] = _i32([3, 4]), _i32([5, 6, 7])
    own = table[:, :W].contiguous()
    want = kernels.step_plan(_i32(c), _i32(n), own, _i32(free), block, blocks, T)
    flat = torch.zeros(64, dtype=torch.int32, device="cuda")
    table[1, W:W + R] = _i32(c)                     # in the gap behind row 1
    computed, query, ids = table[1, W:W + R], flat[:R], flat[R:R + 4]
    query.copy_(_i32(n))
    ids.copy_(_i32(free))
    wide = torch.zeros(2 * T, dtype=torch.int64, device="cuda")
    err = _err()
    got = kernels.step_plan(computed, query, table[:, :W], ids, block, blocks, T,
                            query_start_loc=flat[7:11], seq_lens=flat[11:14], blocks_used=flat[14:15],
                            slot_mapping=wide[:T], positions=wide[T:], error_word=err)
    assert int(err) == 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(table[:, :W], own)
    assert table[1, W:].tolist() == c and flat[:7].tolist() == n + free
    starts = torch.zeros(R + 1, dtype=torch.int32, device="cuda")
    for kw in (dict(query_start_loc=starts), dict(seq_lens=starts[:R]), dict(blocks_used=starts[2:3])):
        with pytest.raises(RuntimeError, match="length inputs"):
            kernels.step_plan(_i32(c), starts[1:], own, _i32(free), block, blocks, T, **kw)


# ------------------------------------------------------------------- positions of other shapes
def test_rotary_positions_of_other_shapes():
    """Positions of three dims are taken where they are contiguous and refused where they are not
    (only a matrix's axis stride is passed on); a broadcast or strided matrix, and one token."""
    g, N = _gen(60), 6
    cs = torch.randn(50, D, generator=g).cuda()
    q = torch.randn(N, 4, D, generator=g).half().cuda()
    sections = (16, 24, 24)
    pos = torch.randint(0, 50, (3, N), generator=g).cuda()

    def turn(p, x=q):
        return kernels.rotary_axes(x, None, p, cs, sections)[0]
    want = turn(pos)
    assert torch.equal(turn(pos.reshape(3, 1, N)), want)
    wide = torch.zeros(3, 40, dtype=torch.int64, device="cuda")
    wide[:, 3:3 + N] = pos
    assert torch.equal(turn(wide[:, 3:3 + N]), want)
    assert torch.equal(turn(pos[:1].expand(3, N)), turn(pos[:1].repeat(3, 1)))
    assert torch.equal(turn(pos[:, 2:3], q[2:3]), want[2:3])
    for bad in (pos[:1].reshape(1, 1, N).expand(3, 1, N), wide[:, 3:3 + N].unsqueeze(1),
                pos.t().contiguous().t(), torch.zeros((), dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError, match="positions"):
            turn(bad)


def test_rotary_outputs_beside_inputs():
    """Outputs in the same rows as the inputs, behind them or in place, one of each: the same values."""
    g, N = _gen(61), 9
    cs = torch.randn(50, D, generator=g).cuda()
    pos = torch.randint(0, 50, (3, N), generator=g).cuda()
    rows = torch.randn(N, 12 * D, generator=g).half().cuda()
    part = lambda a, n: rows[:, a * D:(a + n) * D].unflatten(1, (n, D))  # noqa: E731
    q, k = part(0, 4), part(4, 2)
    want = kernels.rotary_axes(q.contiguous(), k.contiguous(), pos, cs, (16, 24, 24))
    before = rows[:, 4 * D:6 * D].clone()
    got = kernels.rotary_axes(q, k, pos, cs, (16, 24, 24), query_out=q, key_out=part(7, 2))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(rows[:, 4 * D:6 * D], before)
    got = kernels.rotary_axes(part(0, 4), k, pos, cs, (16, 24, 24), query_out=part(8, 4), key_out=k)
    assert torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------- large scores
def _levels(n, seed):
    """A store of n tokens of one KV head whose keys are one channel of seven levels, 8 % apart or
    more (the stored ones), and random values; the levels as stored and the values."""
    st = Store([n], 1, seed=seed)
    level = torch.randint(1, 8, (n,), generator=_gen(seed)).half()
    k = torch.zeros(n, 1, D).half()
    k[:, 0, 0] = level
    kernels.nibble_write_paged(st.lay, k.cuda(), st.v.cuda(), st.slots.cuda(), st.page)
    return st, on.values(k)[:, 0, 0], on.values(st.v)[:, 0]


def _winners(level, V, sign, sees):
    """The mean of the values of the largest (smallest) level among the first `sees` tokens."""
    lv = level[:sees] * sign
    return V[:sees][lv == lv.max()].mean(0)


@pytest.mark.parametrize("n,Q", [(70, 1), (9000, 1), (500, 7), (6000, 5), (100, 100), (3000, 130)])
@pytest.mark.parametrize("dtype,peak,scale", [
    (torch.bfloat16, 2.0 ** 12, 1.0), (torch.bfloat16, 2.0 ** 24, 1.0), (torch.bfloat16, 2.0 ** 29, 1.0),
    (torch.bfloat16, 2.0 ** 31, 1.3), (torch.bfloat16, 2.0 ** 60, 0.7), (torch.bfloat16, 2.0 ** 101, 1.1),
    (torch.bfloat16, 2.0 ** 122, 1.0), (torch.float16, 60000.0, 1e4), (torch.float16, 60000.0, 3e25)])
def test_scores_far_beyond_the_weights_range(n, Q, dtype, peak, scale):
    """Scores of up to 2^125, of either sign: neighbours are 2^8 or more apart, so a row is the mean
    of the values of its largest keys, whose scores are equal. Equal weights leave the roundings of
    the mean's sum (n additions of 2^-24) and of the output: half + 2^-24 n of the largest value."""
    st, level, V = _levels(n, n)
    q = torch.zeros(Q, 4, D)
    q[:, :2, 0], q[:, 2:, 0] = peak, -peak
    err = _err()
    if Q == 1:
        out = kernels.nibble_decode_paged(st.lay, q.to(dtype).cuda(), st.page, 16, st.bt, st.seq,
                                          _i32([0, 1]), n, scale, error_word=err)
    else:
        out = kernels.nibble_prefill_paged(st.lay, q.to(dtype).cuda(), st.page, 16, st.bt, st.seq,
                                           _i32([0, Q]), Q, n, scale, error_word=err)
    assert int(err) == 0
    got = out.cpu().double()
    for j in {0, Q // 2, Q - 1}:
        for p, sign in ((0, 1), (1, 1), (2, -1), (3, -1)):
            want = _winners(level, V, sign, n - Q + j + 1)
            tol = HALF[dtype] * want.abs() + 2.0 ** -24 * n * V.abs().max()
            assert bool(((got[j, p] - want).abs() <= tol).all()), (j, p, got[j, p, :3], want[:3])


# ------------------------------------------------------------------ small weights in numbers
def _far_key(n, at, H=2):
    """n tokens whose scores are 0 but for token `at`'s, which is the query's first element; its
    value is 0, the others' are in [1, 2): the output is the sum of the small weights."""
    g = _gen(n + at)
    k, v = torch.zeros(n, H, D), 1 + torch.rand(n, H, D, generator=g)
    k[at, :, 0], v[at] = 1, 0
    k, v = k.half(), v.half()
    lay = NibbleLayout(H)
    blocks = -(-n // 16)
    page = torch.full((blocks, 16, 144 * H), 255, dtype=torch.uint8, device="cuda")
    ids = torch.randperm(blocks, generator=g).to(torch.int32)
    kernels.nibble_write_paged(lay, k.cuda(), v.cuda(), on.table_slots(ids, n, 16).cuda(), page)
    return lay, page, ids.cuda(), on.values(k), on.values(v)


@pytest.mark.parametrize("bits", [15.5, 18.6, 20.4, 22.3, 26.0])
@pytest.mark.parametrize("kind,B,n,Q,at", [
    ("decode", 300, 600, 1, 0), ("decode", 300, 600, 1, 599), ("decode", 2, 9000, 1, 4500),
    ("chunk", 300, 600, 4, 1), ("flash", 20, 2000, 400, 0), ("flash", 20, 2000, 400, 1200),
    ("flash", 1, 5000, 200, 0)])
def test_many_small_weights_beside_a_large_one(kind, B, n, Q, at, bits):
    """Weights of 2^-15 to 2^-26 of the largest: each is rounded to half a step of fp16, 2^-11 of it
    while it is a normal number and 2^-25 below that, where the largest weight is 2^8 (decode and
    short chunks) or 2^4 (long ones): 2^-33 and 2^-29 of the largest. Requests share one table."""
    least = 2.0 ** (-29 if kind == "flash" else -33)
    lay, page, ids, K, V = _far_key(n, at)
    scale = 0.6931471805599453
    H, G = 2, 4 if kind != "flash" else 8
    q = torch.zeros(Q, H * G, D).half()
    q[..., 0] = bits
    all_q = q.repeat(B, 1, 1).cuda()
    bt = ids.repeat(B, 1).contiguous()
    seq, qsl, err = _i32([n] * B), _i32([Q * r for r in range(B + 1)]), _err()
    if kind == "decode":
        out = kernels.nibble_decode_paged(lay, all_q, page, 16, bt, seq, qsl, n, scale,
                                          error_word=err)
    else:
        out = kernels.nibble_prefill_paged(lay, all_q, page, 16, bt, seq, qsl, Q, n, scale,
                                           error_word=err)
    assert int(err) == 0
    for r in {0, B // 2, B - 1}:
        for j in {0, Q // 2, Q - 1}:
            sees = n - Q + j + 1
            want, spread, score = on.attend(q[j:j + 1], K[:sees], V[:sees], scale)
            tol = 1.05 * (2.0 ** -11 * want.abs() + (2.0 ** -11 + 2.0 ** -16 * score + 2.0 ** -20)
                          * spread + sees * least * V.abs().max()) + 2.0 ** -25
            e = (out[r * Q + j].cpu().double() - want[0]).abs()
            assert bool((e <= tol[0]).all()), (r, j, float((e / tol[0]).max()))


# ---------------------------------------------------------- a workspace for layers of unlike heads
def test_one_workspace_for_layers_of_unlike_heads():
    """Sixteen query heads over 16, 4, 2 and 1 KV heads on the buffer of the first's size."""
    lens, HQ = [5000, 300, 40], 16
    for counts in ([1, 1, 1], [9, 2, 5], [150, 300, 40]):
        lay, most = NibbleLayout(16), max(counts)
        ws = torch.zeros(max(kernels.nibble_prefill_workspace(lay, HQ, 3, most, 5000, "cpu").numel(),
                             kernels.nibble_decode_workspace(lay, HQ, 3, 5000, "cpu").numel()),
                         dtype=torch.uint8, device="cuda")
        for H in (16, 4, 1, 2):
            st = Store(lens, H, seed=70 + H)
            q = torch.randn(sum(counts), HQ, D, generator=_gen(71)).half()
            qsl, err = _starts(counts), _err()
            args = (st.lay, q.cuda(), st.page, 16, st.bt, st.seq, _i32(qsl))
            outs = [kernels.nibble_prefill_paged(*args, most, 5000, SCALE, workspace=ws,
                                                 error_word=err)]
            if most == 1:
                outs.append(kernels.nibble_decode_paged(*args, 5000, SCALE, workspace=ws,
                                                        error_word=err))
            assert int(err) == 0
            for out in outs:
                for r in range(3):
                    s = slice(qsl[r], qsl[r + 1])
                    _close(out[s], q[s], *st.kv(r), SCALE, (H, counts, r))


# ------------------------------------------------------------------------ a step without tokens
def test_a_step_without_tokens():
    """Every request waits and nothing is padded: plan, rotation, write and both reads take a step of
    no tokens."""
    st = Store([40, 700], 2, seed=80)
    lay, H, HQ = st.lay, 2, 8
    page, cs = st.page.clone(), torch.randn(50, D).cuda()

    def step():
        err = _err()
        p = kernels.step_plan(st.seq, _i32([0, 0]), st.bt, _i32([0]), 16, st.blocks, 0, error_word=err)
        q, k = (torch.zeros(0, h, D, dtype=torch.float16, device="cuda") for h in (HQ, H))
        pos = torch.zeros(3, 0, dtype=torch.int64, device="cuda")
        qr, kr = kernels.rotary_axes(q, k, pos, cs, (16, 24, 24), error_word=err)
        kernels.nibble_write_paged(lay, kr, k, p.slot_mapping, st.page, error_word=err)
        args = (lay, qr, st.page, 16, st.bt, p.seq_lens, p.query_start_loc)
        outs = [kernels.nibble_decode_paged(*args, 700, SCALE, error_word=err),
                kernels.nibble_prefill_paged(*args, 0, 700, SCALE, error_word=err),
                kernels.nibble_prefill_paged(*args, 64, 700, SCALE, error_word=err),
                kernels.nibble_prefill_paged(*args, 300, 700, SCALE, req_index=_i32([1]),
                                             error_word=err)]
        assert int(err) == 0 and all(tuple(o.shape) == (0, HQ, D) for o in outs)
        assert p.query_start_loc.tolist() == [0, 0, 0] and p.seq_lens.tolist() == [40, 700]
    step()
    assert torch.equal(st.page, page)


# -------------------------------------------------------- more tokens than a launch has threads
def test_rotary_of_more_tokens_than_a_launch_has_threads():
    """2^24 tokens and some: each as in a small call of its neighbours."""
    N = 2 ** 24 + 37
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(N, 1, 2, generator=gen, device="cuda").bfloat16()
    pos = torch.arange(N, device="cuda") % 4001
    cs = torch.rand(4001, 2, generator=gen, device="cuda")
    err = _err()
    out, _ = kernels.rotary_axes(x, None, pos, cs, (1,), error_word=err)
    assert int(err) == 0
    for a in (0, 2 ** 23 - 150, 2 ** 23 + 4000, N - 300):
        s = slice(a, a + 300)
        assert bool((out[s] == kernels.rotary_axes(x[s], None, pos[s], cs, (1,))[0]).all())


def test_write_of_more_tokens_than_a_launch_has_threads():
    """2^23 tokens of 16 heads and some, all of one key and value row; a few, the last ones among them, have a
    slot."""
    H, N = 16, 2 ** 23 + 40
    lay = NibbleLayout(H)
    row = torch.randn(1, H, D, generator=_gen(5)).bfloat16().cuda()
    x = row.expand(N, H, D)
    at = torch.tensor([0, 1, 2 ** 22 + 3, 2 ** 23 - 1, 2 ** 23, 2 ** 23 + 9, N - 1]).cuda()
    slots = torch.full((N,), -1, dtype=torch.int64, device="cuda")
    slots[at] = torch.arange(at.numel(), device="cuda") * 3
    pages = [torch.zeros(2, 16, lay.compressed_bytes_per_token(), dtype=torch.uint8, device="cuda") for _ in range(2)]
    err = _err()
    kernels.nibble_write_paged(lay, x, x, slots, pages[0], error_word=err)
    assert int(err) == 0
    few = row.expand(at.numel(), H, D).contiguous()
    kernels.nibble_write_paged(lay, few, few, slots[at], pages[1])
    assert bool((pages[0] == pages[1]).all()) and bool((pages[0].reshape(32, -1)[18] != 0).any())

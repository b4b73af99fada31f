"""`nibble_prefill_paged` with chunks of more than 256 rows per KV head, which the row blocks of the
long-chunk kernel take whatever the batch: its error paths, scales, types, strides, and single
queries beside long chunks. Keys unsplit and in several parts. Helpers and tolerances are
test_nibble_gpu's; the same paths of the short-chunk kernel are tested there."""
import pytest
import torch

from test_nibble_gpu import D, SCALE, Store, _close, _err, _gen, _i32, _prefill
from vllm_ttkv import kernels

pytestmark = pytest.mark.gpu

UNSPLIT = ([150, 130, 100, 160], [100, 90, 70, 120])
SPLIT = ([6000, 5000], [100, 70])


def _check(st, out, q, qsl, r, take=None, n=None, scale=SCALE):
    """Request r's first `take` rows against the first n of its keys."""
    K, V = st.kv(r)
    n = len(K) if n is None else n
    s = slice(qsl[r], qsl[r + 1] if take is None else qsl[r] + take)
    _close(out[s], q[s], K[:n], V[:n], scale, r)


@pytest.mark.parametrize("lens,counts,at", [(*UNSPLIT, [(1, 0)]), (*UNSPLIT, [(1, 8), (3, 3)]),
                                            (*SPLIT, [(0, 0)]), (*SPLIT, [(0, 200)]),
                                            (*SPLIT, [(1, 311)]), (*SPLIT, [(1, 312), (1, 5)])])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_bad_blocks(lens, counts, at, bad):
    """A block outside the cache, in the first part of the keys or another: the rows that see it
    become NaN, and no other request's."""
    st = Store(lens, 2, seed=1)
    for r, b in at:
        st.bt[r, b] = bad
    q = torch.randn(sum(counts), 8, D, generator=_gen(1)).half()
    out, err, qsl = _prefill(st, q.cuda(), counts)
    assert err == 2
    hit = {r for r, _ in at}
    for r in range(len(lens)):
        if r in hit:
            first = min(b for x, b in at if x == r) * 16       # the first token of a bad block
            sees = [n for n in range(counts[r]) if lens[r] - counts[r] + n >= first]
            rows = out[qsl[r]:qsl[r + 1]][sees]
            assert len(sees) and bool(torch.isnan(rows).all())
        else:
            _check(st, out, q, qsl, r)


def test_fewer_keys_than_queries():
    for lens, counts, bad in (([99, 300, 120], [100, 80, 90], 0), ([6000, 70], [100, 71], 1)):
        st = Store(lens, 2, seed=2)
        q = torch.randn(sum(counts), 8, D, generator=_gen(2)).half()
        out, err, qsl = _prefill(st, q.cuda(), counts)
        assert err == 8
        for r in range(len(lens)):
            if r == bad:
                assert bool(torch.isnan(out[qsl[r]:qsl[r + 1]]).all())
            else:
                _check(st, out, q, qsl, r)


@pytest.mark.parametrize("lens,counts", [UNSPLIT, SPLIT])
def test_counts_past_max_q_len(lens, counts):
    """The first max_q_len queries are taken, in their places; the rows behind stay as they were."""
    st, most = Store(lens, 2, seed=3), max(counts) - 20
    q = torch.randn(sum(counts), 8, D, generator=_gen(3)).half()
    out = torch.full_like(q, 5.0, device="cuda")
    _, err, qsl = _prefill(st, q.cuda(), counts, max_q=most, out=out)
    assert err == 8
    for r, c in enumerate(counts):
        take = min(c, most)
        _check(st, out, q, qsl, r, take, lens[r] - c + take)
        assert bool((out[qsl[r] + take:qsl[r + 1]] == 5).all())


@pytest.mark.parametrize("lens,counts,cut", [(*UNSPLIT, 140), (*SPLIT, 4990), (*SPLIT, 100),
                                             ([400, 90], [9, 3], 200), ([5000, 90], [2, 3], 3000)])
def test_lengths_past_max_seq_len(lens, counts, cut):
    """The first max_seq_len keys are taken, the chunk's queries at their end (also of short chunks)."""
    st = Store(lens, 2, seed=4)
    q = torch.randn(sum(counts), 8, D, generator=_gen(4)).half()
    out, err, qsl = _prefill(st, q.cuda(), counts, max_seq=cut)
    assert err == 8
    for r, n in enumerate(lens):
        _check(st, out, q, qsl, r, n=min(n, cut))


@pytest.mark.parametrize("scale", [0.0, -SCALE, 2.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,counts", [UNSPLIT, SPLIT])
def test_scales_of_any_sign(lens, counts, dtype, scale):
    st = Store(lens, 2, seed=5, dtype=dtype)
    q = torch.randn(sum(counts), 8, D, generator=_gen(5)).to(dtype)
    qsl, err = [0], _err()
    for c in counts:
        qsl.append(qsl[-1] + c)
    out = kernels.nibble_prefill_paged(st.lay, q.cuda(), st.page, 16, st.bt, st.seq, _i32(qsl),
                                       max(counts), max(lens), scale, error_word=err)
    assert int(err) == 0
    for r in range(len(lens)):
        _check(st, out, q, qsl, r, scale=scale)


@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.float16, torch.bfloat16),
                                               (torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("lens,counts", [UNSPLIT, SPLIT])
def test_strided_rows_and_another_type(lens, counts, q_dtype, out_dtype):
    """Queries inside wider rows, outputs of the other type inside wider rows whose rest stays, and
    slots wider than they need be."""
    st, n = Store(lens, 2, 32, seed=6, pad=48, dtype=q_dtype), sum(counts)
    wide = torch.randn(n, 20 * D, generator=_gen(6)).to(q_dtype).cuda()
    q = wide[:, 8 * D:16 * D].unflatten(1, (8, D))
    buf = torch.full((n, 11 * D), 3.0, dtype=out_dtype, device="cuda")
    out, err, qsl = _prefill(st, q, counts, out=buf[:, D:9 * D].unflatten(1, (8, D)))
    assert err == 0
    for r in range(len(lens)):
        _check(st, out, q.cpu(), qsl, r)
    assert bool((buf[:, :D] == 3).all()) and bool((buf[:, 9 * D:] == 3).all())


@pytest.mark.parametrize("H,HQ,singles,longest,chunks", [
    (2, 8, 60, 500, [(700, 300)]), (8, 32, 20, 90, [(512, 512), (3000, 120)]), (1, 7, 280, 40, [(900, 400)])])
def test_single_queries_beside_long_chunks(H, HQ, singles, longest, chunks):
    """A mixed step: a decode token of each of many requests and a long chunk in one call, and the
    same rows in two calls by req_index, each with its own max_q_len."""
    g = _gen(singles)
    lens = [int(x) for x in torch.randint(1, longest, (singles,), generator=g)]
    counts = [1] * singles
    for k, (n, c) in enumerate(chunks):             # between the single ones
        at = (k + 1) * singles // (len(chunks) + 1)
        lens.insert(at, n)
        counts.insert(at, c)
    st = Store(lens, H, seed=singles)
    q = torch.randn(sum(counts), HQ, D, generator=g).half()
    out, err, qsl = _prefill(st, q.cuda(), counts)
    assert err == 0
    picks = [r for r in range(len(lens)) if counts[r] > 1 or r % 9 == 0]
    for r in picks:
        _check(st, out, q, qsl, r)
    apart = torch.full_like(out, float("nan"))
    for keep in ([r for r, c in enumerate(counts) if c == 1], [r for r, c in enumerate(counts) if c > 1]):
        most = max(counts[r] for r in keep)
        _, err, _ = _prefill(st, q.cuda(), counts, out=apart, max_q=most, req_index=_i32(keep),
                             max_seq=max(lens[r] for r in keep))
        assert err == 0
    assert not bool(torch.isnan(apart).any())
    for r in picks:
        _check(st, apart, q, qsl, r)

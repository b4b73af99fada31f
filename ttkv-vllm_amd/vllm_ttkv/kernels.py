"""torch-facing wrappers over the libttkv_hip C ABI.

Each wrapper validates what the host can see, allocates nothing on its own except when the
caller did not pass an output or workspace, and launches on torch's current stream. The tensors
must live on a HIP device; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _hip
from .decoder_pool import DecoderPool, decoder_ranks
from .layout import TTKLayout
from .nibble import NibbleLayout


def _need_device(*ts):
    for t in ts:
        if isinstance(t, DecoderPool):
            _need_device(*t)
        elif t is not None and not t.is_cuda:
            raise RuntimeError("libttkv_hip kernels take device tensors; got a "
                               f"{t.device.type} tensor (there is no CPU implementation)")


def _i32(t, name):
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor, got {t.dtype}")
    return t


def pool_args(lay: TTKLayout, dec_pool: DecoderPool) -> tuple[int, int, int]:
    """(dec_q pointer, dec_scale pointer, slots) of a decoder pool, after checking it has the
    layout's shape: `q [slots, H*d, R]` int8 and `scale [slots, R]` fp32, both contiguous, R =
    decoder_ranks(r1) (see `decoder_pool`)."""
    if not isinstance(dec_pool, DecoderPool):
        raise TypeError("dec_pool must be a DecoderPool (a store's `dec_pool`, or "
                        "decoder_pool.pack_decoders of fp32 decoders)")
    q, sc = dec_pool
    R = decoder_ranks(lay.r1)
    if (q.dtype != torch.int8 or q.dim() != 3 or q.shape[1:] != (lay.H * lay.d, R)
            or not q.is_contiguous()):
        raise ValueError(f"dec_pool.q must be contiguous int8 [slots, {lay.H * lay.d}, {R}], got "
                         f"{q.dtype} {tuple(q.shape)} (a decoder written at one rank cannot be "
                         f"read at another)")
    if sc.dtype != torch.float32 or sc.shape != (q.shape[0], R) or not sc.is_contiguous():
        raise ValueError(f"dec_pool.scale must be contiguous fp32 [{q.shape[0]}, {R}], got "
                         f"{sc.dtype} {tuple(sc.shape)}")
    return q.data_ptr(), sc.data_ptr(), int(q.shape[0])


def page_bytes(page: torch.Tensor, blob: int) -> torch.Tensor:
    """`[n_slots, W]` uint8 view of a paged cache `[num_blocks, (1,) block_size, C]` in any dtype.

    The last dim of a vLLM page counts MODEL-dtype elements (decode.py:125-157), so the row is
    reinterpreted as bytes. W >= blob is accepted (vLLM rounds the row up to whole elements)."""
    u8 = page if page.dtype == torch.uint8 else page.view(torch.uint8)
    if u8.shape[-1] < blob:
        raise ValueError(f"the cache row is {u8.shape[-1]} bytes but the layout needs {blob}")
    if not u8.is_contiguous():
        raise ValueError("the cache page must be contiguous")
    return u8.reshape(-1, u8.shape[-1])


def _page_args(page: torch.Tensor, blob: int) -> tuple[int, int, int]:
    """(pointer, slots, bytes per slot) of a paged cache, as `page_bytes` views it (the same
    refusals, without making the views)."""
    shape = page.shape
    if len(shape) < 2 or not page.is_contiguous():
        flat = page_bytes(page, blob)
        return flat.data_ptr(), flat.shape[0], flat.stride(0)
    last = shape[-1]
    row = last * page.element_size()
    if row < blob:
        raise ValueError(f"the cache row is {row} bytes but the layout needs {blob}")
    return page.data_ptr(), page.numel() // (last or 1), row


def decode_workspace(lay: TTKLayout, num_heads: int, num_reqs: int, max_seq_len: int,
                     device, block_size: int = 16) -> torch.Tensor:
    """A zero-filled workspace sized for this batch shape. Its counter region (the first 64 KiB)
    is left zero by every call, so a buffer this large serves later calls of any shape."""
    n = _hip.lib().ttkv_decode_workspace_bytes(_hip.Layout.of(lay), num_heads, num_reqs,
                                               max_seq_len, block_size)
    if n < 0:
        raise ValueError("invalid layout / head count for the decode workspace")
    return torch.zeros(max(int(n), 256), dtype=torch.uint8, device=device)


def decode_paged(lay: TTKLayout, query: torch.Tensor, page: torch.Tensor, block_size: int,
                 block_table: torch.Tensor, seq_lens: torch.Tensor,
                 query_start_loc: torch.Tensor, max_seq_len: int,
                 dec_slot_of_block: torch.Tensor, dec_pool: DecoderPool,
                 cos_sin_cache: torch.Tensor, scale: float, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None,
                 error_word: torch.Tensor | None = None) -> torch.Tensor:
    """K1: one launch over all decode requests. See `ttkv_decode_paged` in include/ttkv_hip.h.

    query [N, HQ, d]; page: the layer's cache (bytes reinterpreted); block_table [B, max_blocks]
    int32; seq_lens [B] int32; query_start_loc [>=B] int32 (row of request r's query);
    dec_slot_of_block [num_blocks] int32; dec_pool: the decoder pool (`DecoderPool`);
    cos_sin_cache [max_pos, d] fp32 (vLLM layout). Returns `out` [N, HQ, d] with the decode rows
    written."""
    _need_device(query, page, block_table, seq_lens, query_start_loc, dec_slot_of_block,
                 dec_pool, cos_sin_cache)
    L = _hip.lib()
    num_reqs = int(seq_lens.numel())
    N, HQ, d = query.shape
    if d != lay.d:
        raise ValueError(f"query head dim {d} != layout d {lay.d}")
    if query.stride(2) != 1 or query.stride(1) != d:
        raise ValueError("query must be contiguous within a token ([HQ, d] rows)")
    page_ptr, n_slots, slot_bytes = _page_args(page, lay.compressed_bytes_per_token())
    _i32(block_table, "block_table")
    _i32(seq_lens, "seq_lens")
    _i32(query_start_loc, "query_start_loc")
    _i32(dec_slot_of_block, "dec_slot_of_block")
    dq, ds, n_dec = pool_args(lay, dec_pool)
    if cos_sin_cache.dtype != torch.float32 or not cos_sin_cache.is_contiguous():
        raise ValueError("cos_sin_cache must be contiguous fp32 [max_pos, d]")
    if cos_sin_cache.shape[-1] != lay.d:
        raise NotImplementedError(
            f"rotary_dim={cos_sin_cache.shape[-1]} != head_dim={lay.d} (partial rotary) is not "
            f"supported: the kernel pairs (j, j+d/2) across the whole row")
    if out is None:
        out = torch.empty_like(query)
    if out.shape != query.shape or out.stride(2) != 1 or out.stride(1) != d:
        raise ValueError("out must match query's shape with contiguous [HQ, d] rows")
    if out.dtype not in _hip.DTYPE_CODE or query.dtype not in _hip.DTYPE_CODE:
        raise ValueError("query/out dtype must be fp32, fp16 or bf16")
    if workspace is None:
        workspace = decode_workspace(lay, HQ, num_reqs, max_seq_len, query.device, block_size)
    if error_word is None:
        error_word = torch.zeros(1, dtype=torch.int32, device=query.device)
    rc = L.ttkv_decode_paged(
        _hip.Layout.of(lay), HQ, float(scale),
        query.data_ptr(), _hip.DTYPE_CODE[query.dtype], query.stride(0),
        page_ptr, n_slots, slot_bytes,
        int(block_size), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        seq_lens.data_ptr(), query_start_loc.data_ptr(), num_reqs, int(max_seq_len),
        dec_slot_of_block.data_ptr(), dec_slot_of_block.numel(), dq, ds, n_dec,
        cos_sin_cache.data_ptr(), cos_sin_cache.shape[0],
        out.data_ptr(), _hip.DTYPE_CODE[out.dtype], out.stride(0),
        workspace.data_ptr(), workspace.numel(), error_word.data_ptr(),
        _hip.stream_ptr(query.device))
    _hip.check(rc, "ttkv_decode_paged")
    return out


def write_paged(lay: TTKLayout, key: torch.Tensor, value: torch.Tensor,
                slot_mapping: torch.Tensor, query_start_loc: torch.Tensor,
                block_table: torch.Tensor, dec_slot_of_block: torch.Tensor,
                dec_pool: DecoderPool, pinv_pool: torch.Tensor | None, page: torch.Tensor,
                coeff_q_in: torch.Tensor | None = None,
                coeff_scale_in: torch.Tensor | None = None,
                coeff_out: torch.Tensor | None = None, resid_out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None,
                dec_used: torch.Tensor | None = None) -> None:
    """K3: encode + pack `key`/`value` ([N, H, d], raw pre-RoPE keys) into their slots.

    See `ttkv_write_paged` in include/ttkv_hip.h. `pinv_pool` [slots, r1, H*d] fp32 (each decoder's pinv transposed: row a
    is rank a's projection vector) drives the
    frozen projection; `coeff_q_in`/`coeff_scale_in` replace it with a fit's coefficients.
    `dec_used` ([slots] int32, optional) receives 1 for every decoder slot a token used."""
    _need_device(key, value, slot_mapping, query_start_loc, block_table, dec_slot_of_block,
                 dec_pool, pinv_pool, page)
    N = key.shape[0]
    if key.dim() != 3 or key.shape[1:] != (lay.H, lay.d) or value.shape != key.shape:
        raise ValueError(f"key/value must be [N, {lay.H}, {lay.d}], got {tuple(key.shape)} and "
                         f"{tuple(value.shape)}")
    for t, nm in ((key, "key"), (value, "value")):
        if t.stride(2) != 1 or t.stride(1) != lay.d:
            raise ValueError(f"{nm} must be contiguous within a token")
        if t.dtype not in _hip.DTYPE_CODE:
            raise ValueError(f"{nm} dtype must be fp32, fp16 or bf16")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() < N:
        raise ValueError("slot_mapping must be int64 with one id per token")
    _i32(query_start_loc, "query_start_loc")
    _i32(block_table, "block_table")
    _i32(dec_slot_of_block, "dec_slot_of_block")
    dq, ds, n_dec = pool_args(lay, dec_pool)
    if pinv_pool is not None and (pinv_pool.dtype != torch.float32 or
                                  pinv_pool.shape[1:] != (lay.r1, lay.H * lay.d)):
        raise ValueError("pinv_pool must be fp32 [slots, r1, H*d] (each pinv transposed)")
    page_ptr, n_slots, slot_bytes = _page_args(page, lay.compressed_bytes_per_token())
    if error_word is None:
        error_word = torch.zeros(1, dtype=torch.int32, device=key.device)
    if dec_used is not None:
        _i32(dec_used, "dec_used")
        if dec_used.numel() < n_dec:
            raise ValueError("dec_used needs one flag per decoder pool slot")
    cq = None
    if coeff_q_in is not None:
        if lay.qbits != 8:
            raise ValueError("coeff_q_in is the int8 mode's; the fp16 and 4-bit coefficient "
                             "modes quantise the projection themselves (pass pinv_pool)")
        cq = coeff_q_in.to(torch.int8).contiguous()
        if coeff_scale_in is None:
            raise ValueError("coeff_q_in needs coeff_scale_in (fp32)")
        coeff_scale_in = coeff_scale_in.to(torch.float32).contiguous()
    if workspace is None and cq is None:
        workspace = write_workspace(lay, N, key.device)
    rc = _hip.lib().ttkv_write_paged(
        _hip.Layout.of(lay), key.data_ptr(), _hip.DTYPE_CODE[key.dtype], key.stride(0),
        value.data_ptr(), _hip.DTYPE_CODE[value.dtype], value.stride(0),
        slot_mapping.data_ptr(), N, query_start_loc.data_ptr(), query_start_loc.numel() - 1,
        block_table.data_ptr(), block_table.stride(0), dec_slot_of_block.data_ptr(),
        dec_slot_of_block.numel(), dq, ds, _hip.ptr(pinv_pool), n_dec,
        _hip.ptr(dec_used), _hip.ptr(cq), _hip.ptr(coeff_scale_in), page_ptr, n_slots, slot_bytes,
        _hip.ptr(coeff_out), _hip.ptr(resid_out), _hip.ptr(workspace),
        0 if workspace is None else workspace.numel(), error_word.data_ptr(),
        _hip.stream_ptr(key.device))
    _hip.check(rc, "ttkv_write_paged")


def write_workspace(lay: TTKLayout, num_tokens: int, device) -> torch.Tensor:
    """A zero-filled workspace for `write_paged` over `num_tokens` projected tokens."""
    n = _hip.lib().ttkv_write_workspace_bytes(_hip.Layout.of(lay), int(num_tokens))
    if n < 0:
        raise ValueError("invalid layout for the write workspace")
    return torch.zeros(max(int(n), 256), dtype=torch.uint8, device=device)


def _read_checks(lay: TTKLayout, query, page, block_table, seq_lens, query_start_loc,
                 dec_slot_of_block, dec_pool, cos_sin_cache):
    """Host-visible checks shared by the read kernels (K1, K2)."""
    _need_device(query, page, block_table, seq_lens, query_start_loc, dec_slot_of_block,
                 dec_pool, cos_sin_cache)
    if query.dim() != 3 or query.shape[2] != lay.d:
        raise ValueError(f"query must be [N, num_heads, {lay.d}], got {tuple(query.shape)}")
    if query.stride(2) != 1 or query.stride(1) != lay.d:
        raise ValueError("query must be contiguous within a token ([HQ, d] rows)")
    if query.dtype not in _hip.DTYPE_CODE:
        raise ValueError("query dtype must be fp32, fp16 or bf16")
    flat = page_bytes(page, lay.compressed_bytes_per_token())
    _i32(block_table, "block_table")
    _i32(seq_lens, "seq_lens")
    _i32(query_start_loc, "query_start_loc")
    _i32(dec_slot_of_block, "dec_slot_of_block")
    pool_args(lay, dec_pool)
    if cos_sin_cache.dtype != torch.float32 or not cos_sin_cache.is_contiguous():
        raise ValueError("cos_sin_cache must be contiguous fp32 [max_pos, d]")
    if cos_sin_cache.shape[-1] != lay.d:
        raise NotImplementedError(
            f"rotary_dim={cos_sin_cache.shape[-1]} != head_dim={lay.d} (partial rotary) is not "
            f"supported: the kernels pair (j, j+d/2) across the whole row")
    return flat


def prefill_workspace(lay: TTKLayout, num_heads: int, num_reqs: int, max_q_len: int,
                      max_seq_len: int, device, block_size: int = 16) -> torch.Tensor:
    n = _hip.lib().ttkv_prefill_workspace_bytes(_hip.Layout.of(lay), num_heads, num_reqs,
                                                max_q_len, max_seq_len, block_size)
    if n < 0:
        raise ValueError("invalid layout / head count for the prefill workspace")
    return torch.zeros(max(int(n), 256), dtype=torch.uint8, device=device)


def prefill_paged(lay: TTKLayout, query: torch.Tensor, page: torch.Tensor, block_size: int,
                  block_table: torch.Tensor, seq_lens: torch.Tensor,
                  query_start_loc: torch.Tensor, max_q_len: int, max_seq_len: int,
                  dec_slot_of_block: torch.Tensor, dec_pool: DecoderPool,
                  cos_sin_cache: torch.Tensor, scale: float,
                  req_index: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None,
                  error_word: torch.Tensor | None = None) -> torch.Tensor:
    """K2: continuation attention for a batch of chunked-prefill requests, one launch.

    Rows `query_start_loc[r] .. [r+1]` of `query` [N, HQ, d] (post-RoPE) attend causally over the
    `seq_lens[r]` stored keys of request r (p0 = seq_len - q_len). `req_index` picks the batch
    rows to process (default: all `seq_lens.numel()`). See `ttkv_prefill_paged`."""
    flat = _read_checks(lay, query, page, block_table, seq_lens, query_start_loc,
                        dec_slot_of_block, dec_pool, cos_sin_cache)
    if req_index is not None:
        _i32(req_index, "req_index")
        num_reqs = int(req_index.numel())
    else:
        num_reqs = int(seq_lens.numel())
    N, HQ, d = query.shape
    if out is None:
        out = torch.empty_like(query)
    if out.shape != query.shape or out.stride(2) != 1 or out.stride(1) != d:
        raise ValueError("out must match query's shape with contiguous [HQ, d] rows")
    if out.dtype not in _hip.DTYPE_CODE:
        raise ValueError("out dtype must be fp32, fp16 or bf16")
    if workspace is None:
        workspace = prefill_workspace(lay, HQ, num_reqs, max_q_len, max_seq_len, query.device,
                                      block_size)
    if error_word is None:
        error_word = torch.zeros(1, dtype=torch.int32, device=query.device)
    rc = _hip.lib().ttkv_prefill_paged(
        _hip.Layout.of(lay), HQ, float(scale),
        query.data_ptr(), _hip.DTYPE_CODE[query.dtype], query.stride(0),
        flat.data_ptr(), flat.shape[0], flat.stride(0),
        int(block_size), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        seq_lens.data_ptr(), query_start_loc.data_ptr(), _hip.ptr(req_index), num_reqs,
        int(max_q_len), int(max_seq_len),
        dec_slot_of_block.data_ptr(), dec_slot_of_block.numel(), *pool_args(lay, dec_pool),
        cos_sin_cache.data_ptr(), cos_sin_cache.shape[0],
        out.data_ptr(), _hip.DTYPE_CODE[out.dtype], out.stride(0),
        workspace.data_ptr(), workspace.numel(), error_word.data_ptr(),
        _hip.stream_ptr(query.device))
    _hip.check(rc, "ttkv_prefill_paged")
    return out


def multi_scores_paged(lay: TTKLayout, query: torch.Tensor, page: torch.Tensor,
                       block_size: int, block_table: torch.Tensor, seq_lens: torch.Tensor,
                       query_start_loc: torch.Tensor, max_q_len: int, max_seq_len: int,
                       dec_slot_of_block: torch.Tensor, dec_pool: DecoderPool,
                       cos_sin_cache: torch.Tensor, scale: float,
                       scores: torch.Tensor | None = None,
                       error_word: torch.Tensor | None = None,
                       workspace: torch.Tensor | None | bool = None) -> torch.Tensor:
    """K2 scores mode for ONE request (row 0 of block_table / seq_lens / query_start_loc):
    returns `scores` [HQ, Q, n] fp32 with -inf where key t > p0 + j (`krt_multi_from_slots`).
    Q and n are `max_q_len` / `max_seq_len`, which must equal the request's own lengths.
    `workspace`: None allocates `ttkv_multi_scores_workspace_bytes` (a chunk of two or more
    queries then reads every stored key expanded once), False runs the fused kernel."""
    flat = _read_checks(lay, query, page, block_table, seq_lens, query_start_loc,
                        dec_slot_of_block, dec_pool, cos_sin_cache)
    HQ = query.shape[1]
    if scores is None:
        scores = torch.empty(HQ, max_q_len, max_seq_len, dtype=torch.float32,
                             device=query.device)
    if (scores.dtype != torch.float32 or scores.dim() != 3 or scores.shape[0] != HQ
            or scores.shape[1] < max_q_len or scores.shape[2] < max_seq_len
            or scores.stride(2) != 1):
        raise ValueError(f"scores must be fp32 [{HQ}, >= {max_q_len}, >= {max_seq_len}] with "
                         f"contiguous key rows")
    if error_word is None:
        error_word = torch.zeros(1, dtype=torch.int32, device=query.device)
    if workspace is None:
        n = _hip.lib().ttkv_multi_scores_workspace_bytes(_hip.Layout.of(lay), HQ, int(max_q_len),
                                                         int(max_seq_len))
        if n < 0:
            raise ValueError("invalid layout / head count for the scores workspace")
        workspace = torch.empty(int(n), dtype=torch.uint8, device=query.device) if n else False
    ws_ptr, ws_bytes = (0, 0) if workspace is False else (workspace.data_ptr(), workspace.numel())
    rc = _hip.lib().ttkv_multi_scores_paged(
        _hip.Layout.of(lay), HQ, float(scale),
        query.data_ptr(), _hip.DTYPE_CODE[query.dtype], query.stride(0),
        flat.data_ptr(), flat.shape[0], flat.stride(0),
        int(block_size), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        seq_lens.data_ptr(), query_start_loc.data_ptr(), int(max_q_len), int(max_seq_len),
        dec_slot_of_block.data_ptr(), dec_slot_of_block.numel(), *pool_args(lay, dec_pool),
        cos_sin_cache.data_ptr(), cos_sin_cache.shape[0],
        scores.data_ptr(), scores.stride(0), scores.stride(1), ws_ptr, ws_bytes,
        error_word.data_ptr(), _hip.stream_ptr(query.device))
    _hip.check(rc, "ttkv_multi_scores_paged")
    return scores


def dense_decode_paged(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       block_size: int, block_table: torch.Tensor, seq_lens: torch.Tensor,
                       query_start_loc: torch.Tensor, max_seq_len: int, scale: float,
                       out: torch.Tensor | None = None,
                       workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Benchmark comparator: dense paged decode attention over uncompressed caches
    k_cache / v_cache [n_slots, H, d] (fp16 or bf16, same dtype as query). One launch."""
    _need_device(query, k_cache, v_cache, block_table, seq_lens, query_start_loc)
    N, HQ, d = query.shape
    n_slots, H, d2 = k_cache.shape
    if d2 != d or v_cache.shape != k_cache.shape:
        raise ValueError("k_cache / v_cache must be [n_slots, H, d] with the query's d")
    if query.dtype not in (torch.float16, torch.bfloat16) or k_cache.dtype != query.dtype \
            or v_cache.dtype != query.dtype:
        raise ValueError("dense comparator: query and caches must share fp16 or bf16")
    for t in (query, k_cache, v_cache):
        if not t.is_contiguous():
            raise ValueError("dense comparator tensors must be contiguous")
    _i32(block_table, "block_table")
    _i32(seq_lens, "seq_lens")
    _i32(query_start_loc, "query_start_loc")
    B = int(seq_lens.numel())
    if out is None:
        out = torch.empty_like(query)
    if workspace is None:
        n = _hip.lib().ttkv_dense_workspace_bytes(H, HQ, B, int(max_seq_len), int(block_size))
        workspace = torch.zeros(max(int(n), 256), dtype=torch.uint8, device=query.device)
    rc = _hip.lib().ttkv_dense_decode_paged(
        H, HQ, d, float(scale), query.data_ptr(), query.stride(0), k_cache.data_ptr(),
        v_cache.data_ptr(), _hip.DTYPE_CODE[query.dtype], n_slots, int(block_size),
        block_table.data_ptr(), block_table.stride(0), block_table.shape[1], seq_lens.data_ptr(),
        query_start_loc.data_ptr(), B, int(max_seq_len), out.data_ptr(), out.stride(0),
        workspace.data_ptr(), workspace.numel(), _hip.stream_ptr(query.device))
    _hip.check(rc, "ttkv_dense_decode_paged")
    return out


# ---------------------------------------------------------------- the 4-bit cache
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") \
    else torch.cuda.current_device


def _on_device(index: int, fn, *args) -> int:
    """Call a launching C entry with device `index` current: a launch goes to the current device,
    whatever device its stream belongs to. (The guard costs more than the checks, so it is taken only
    where the device differs.)"""
    if index == _current_device():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _one_device(first, *ts) -> int:
    """Refuse host tensors and tensors of another device than the first; returns its index."""
    index = first.get_device()
    if index < 0:
        _need_device(first)
    for t in ts:
        if t is not None and t.get_device() != index:
            _need_device(t)
            raise ValueError(f"tensors on {first.device} and {t.device} in one call")
    return index


def _stream(index: int) -> int:
    """The current stream of device `index`."""
    if _hip._raw_stream is not None:
        return _hip._raw_stream(index)
    return torch.cuda.current_stream(index).cuda_stream


def _error_word(error_word, device):
    if error_word is None:
        return torch.zeros(1, dtype=torch.int32, device=device)
    if error_word.dtype != torch.int32 or error_word.numel() < 1:
        raise ValueError("error_word must be an int32 tensor")
    return error_word


def _rows(t, heads, d, what):
    """Check [N, heads, d] rows, contiguous within a token."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != d:
        raise ValueError(f"{what} must be [N, {heads}, {d}], got {tuple(shape)}")
    if not t.is_contiguous() and t.numel() and (t.stride(2) != 1
                                                or (heads > 1 and t.stride(1) != d)):
        raise ValueError(f"{what} must be contiguous within a token ([heads, {d}] rows)")


class StepPlan(NamedTuple):
    """A step's addresses (`step_plan`)."""
    query_start_loc: torch.Tensor   # [R + 1] int32
    seq_lens: torch.Tensor          # [R] int32, this step's tokens included
    slot_mapping: torch.Tensor      # [num_tokens] int64, -1 past the last token
    positions: torch.Tensor         # [num_tokens] int64, 0 past the last token
    blocks_used: torch.Tensor       # [1] int32, ids taken from the free list


def _table(block_table, want, rows=None):
    """(max_blocks, row stride) of a block table; `rows`: how many it must have."""
    shape = block_table.shape
    if block_table.dtype != torch.int32 or len(shape) != 2 \
            or (rows is not None and shape[0] != rows) \
            or (not block_table.is_contiguous() and shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 {want} with contiguous rows")
    return shape[1], block_table.stride(0)


def _plan_out(t, n, dtype, like, name):
    if t is None:
        return like.new_empty(n, dtype=dtype)
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of {n}")
    return t


def step_plan(computed_lens: torch.Tensor, query_lens: torch.Tensor, block_table: torch.Tensor,
              free_blocks: torch.Tensor, block_size: int, num_blocks: int, num_tokens: int,
              query_start_loc: torch.Tensor | None = None, seq_lens: torch.Tensor | None = None,
              slot_mapping: torch.Tensor | None = None, positions: torch.Tensor | None = None,
              blocks_used: torch.Tensor | None = None,
              error_word: torch.Tensor | None = None) -> StepPlan:
    """Block tables, slot map and positions of a step, from its requests' lengths, in one launch
    with nothing read back. See `ttkv_step_plan` in include/ttkv_hip.h.

    computed_lens / query_lens [R] int32: tokens stored before the step and new in it;
    block_table [R, max_blocks] int32, updated in place; free_blocks [F] int32, taken from the
    front; num_tokens: the (padded) token count of the outputs, at least the sum of query_lens."""
    index = _one_device(computed_lens, query_lens, block_table, free_blocks, query_start_loc,
                        seq_lens, slot_mapping, positions, blocks_used, error_word)
    _i32(computed_lens, "computed_lens")
    _i32(query_lens, "query_lens")
    _i32(free_blocks, "free_blocks")
    R = computed_lens.numel()
    if query_lens.numel() != R:
        raise ValueError(f"{R} computed lengths and {query_lens.numel()} query lengths")
    W, stride = _table(block_table, f"[{R}, max_blocks]", R)
    n = int(num_tokens)
    plan = StepPlan(_plan_out(query_start_loc, R + 1, torch.int32, computed_lens, "query_start_loc"),
                    _plan_out(seq_lens, R, torch.int32, computed_lens, "seq_lens"),
                    _plan_out(slot_mapping, n, torch.int64, computed_lens, "slot_mapping"),
                    _plan_out(positions, n, torch.int64, computed_lens, "positions"),
                    _plan_out(blocks_used, 1, torch.int32, computed_lens, "blocks_used"))
    err = _error_word(error_word, computed_lens.device)
    rc = _on_device(
        index, _hip.lib().ttkv_step_plan, computed_lens.data_ptr(), query_lens.data_ptr(), R, block_table.data_ptr(),
        stride if R > 1 else W, W, free_blocks.data_ptr(), free_blocks.numel(),
        int(block_size), int(num_blocks), n, plan.query_start_loc.data_ptr(),
        plan.seq_lens.data_ptr(), plan.slot_mapping.data_ptr(), plan.positions.data_ptr(),
        plan.blocks_used.data_ptr(), err.data_ptr(), _stream(index))
    _hip.check(rc, "ttkv_step_plan")
    return plan


@functools.lru_cache(maxsize=64)
def _c_sections(sections: tuple) -> ctypes.Array:
    return (ctypes.c_int32 * len(sections))(*sections)


def rotary_axes(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor,
                cos_sin_cache: torch.Tensor, sections, interleaved: bool = False,
                query_out: torch.Tensor | None = None, key_out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None):
    """Rotate query [N, HQ, d] and key [N, H, d] by positions of one to four axes; returns
    (query_out, key_out), each of which may be its input. See `ttkv_rotary_axes` in include/ttkv_hip.h.

    positions [axes, N] (or [N] for one axis) int64; sections: how many of the rotary_dim / 2
    frequencies each axis has, in a row, or dealt in turn where `interleaved`; cos_sin_cache
    [max_pos, rotary_dim] fp32 (vLLM layout)."""
    index = _one_device(query, key, positions, cos_sin_cache, query_out, key_out, error_word)
    if query.dim() != 3:
        raise ValueError(f"query must be [N, heads, d], got {tuple(query.shape)}")
    N, HQ, d = query.shape
    sections = tuple(sections)
    if positions.dtype != torch.int64 or positions.shape[-1:] != (N,) \
            or positions.numel() != len(sections) * N:
        raise ValueError(f"positions must be int64 [{len(sections)}, {N}], got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    if (N > 1 and positions.stride(-1) != 1) or (positions.dim() > 2
                                                 and not positions.is_contiguous()):
        raise ValueError("an axis's positions must be contiguous")
    if cos_sin_cache.dtype != torch.float32 or cos_sin_cache.dim() != 2 \
            or not cos_sin_cache.is_contiguous():
        raise ValueError("cos_sin_cache must be contiguous fp32 [max_pos, rotary_dim]")
    if query.dtype not in _hip.DTYPE_CODE:
        raise ValueError("query dtype must be fp32, fp16 or bf16")
    query_out = torch.empty_like(query) if query_out is None else query_out
    H = 0
    if key is not None:
        H = key.shape[1] if key.dim() == 3 else 0
        key_out = torch.empty_like(key) if key_out is None else key_out
    dtype = query.dtype
    for t, heads, what in ((query, HQ, "query"), (query_out, HQ, "query_out"), (key, H, "key"),
                           (key_out, H, "key_out")):
        if t is None:
            continue
        _rows(t, heads, d, what)
        if t.shape[0] != N or t.dtype != dtype:
            raise ValueError(f"{what} must have the query's {N} tokens and dtype")
    err = _error_word(error_word, query.device)
    rc = _on_device(
        index, _hip.lib().ttkv_rotary_axes, query.data_ptr(), _hip.ptr(key),
        query_out.data_ptr(), _hip.ptr(key_out), _hip.DTYPE_CODE[dtype], N, HQ, H, d,
        query.stride(0),
        0 if key is None else key.stride(0), query_out.stride(0),
        0 if key is None else key_out.stride(0), positions.data_ptr(),
        positions.stride(0) if positions.dim() == 2 else N, len(sections), _c_sections(sections),
        int(bool(interleaved)), cos_sin_cache.data_ptr(), cos_sin_cache.shape[0],
        cos_sin_cache.shape[1], err.data_ptr(), _stream(index))
    _hip.check(rc, "ttkv_rotary_axes")
    return query_out, key_out


def nibble_write_paged(lay: NibbleLayout, key: torch.Tensor, value: torch.Tensor,
                       slot_mapping: torch.Tensor, page: torch.Tensor,
                       key_out: torch.Tensor | None = None,
                       value_out: torch.Tensor | None = None,
                       error_word: torch.Tensor | None = None) -> None:
    """Quantise key / value [N, H, d] (rotated keys) into their slots of a 4-bit cache.

    page: the layer's cache, its last dim one slot (`lay.compressed_bytes_per_token()` bytes or
    more); slot_mapping [>= N] int64, -1 for padded tokens; key_out / value_out (optional, fp16
    [N, H, d], contiguous) receive what the slots then stand for. See `ttkv_nibble_write_paged`."""
    index = _one_device(key, value, slot_mapping, page, key_out, value_out, error_word)
    shape = key.shape
    _rows(key, lay.H, lay.d, "key")
    _rows(value, lay.H, lay.d, "value")
    N = shape[0]
    if value.shape[0] != N:
        raise ValueError(f"{N} keys and {value.shape[0]} values")
    k_code, v_code = _hip.DTYPE_CODE.get(key.dtype), _hip.DTYPE_CODE.get(value.dtype)
    if k_code is None or v_code is None:
        raise ValueError("key / value dtype must be fp32, fp16 or bf16")
    for t, what in ((key_out, "key_out"), (value_out, "value_out")):
        if t is not None and (t.shape != shape or t.dtype != torch.float16
                              or not t.is_contiguous()):
            raise ValueError(f"{what} must be contiguous fp16 [{N}, {lay.H}, {lay.d}]")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() < N \
            or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 with one id per token")
    if not page.is_contiguous():
        raise ValueError("the cache page must be contiguous")
    err = _error_word(error_word, key.device)
    rc = _on_device(
        index, _hip.lib().ttkv_nibble_write_paged, lay.H, lay.d, key.data_ptr(), k_code,
        key.stride(0), value.data_ptr(), v_code, value.stride(0), slot_mapping.data_ptr(), N,
        *_page_args(page, lay.compressed_bytes_per_token()), _hip.ptr(key_out),
        _hip.ptr(value_out), err.data_ptr(), _stream(index))
    _hip.check(rc, "ttkv_nibble_write_paged")


_NIBBLE_DTYPES = {t: _hip.DTYPE_CODE[t] for t in (torch.float16, torch.bfloat16)}


def _nibble_read(lay, query, page, block_table, seq_lens, query_start_loc, out):
    """Checks shared by the 4-bit reads; returns (out, what the C entries take of query and page, of
    the block table and of out)."""
    shape = query.shape
    _rows(query, shape[1] if len(shape) == 3 else 0, lay.d, "query")
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != shape or not out.is_contiguous():
        _rows(out, shape[1], lay.d, "out")
        if out.shape[0] != shape[0]:
            raise ValueError("out must match query's shape")
    q_code, out_code = _NIBBLE_DTYPES.get(query.dtype), _NIBBLE_DTYPES.get(out.dtype)
    if q_code is None or out_code is None:
        raise ValueError(f"{'out' if q_code else 'query'} dtype must be fp16 or bf16")
    table = _table(block_table, "[requests, max_blocks]")
    _i32(seq_lens, "seq_lens")
    _i32(query_start_loc, "query_start_loc")
    if not page.is_contiguous():
        raise ValueError("the cache page must be contiguous")
    return (out, (query.data_ptr(), q_code, query.stride(0),
                  *_page_args(page, lay.compressed_bytes_per_token())),
            (block_table.data_ptr(), table[1], table[0]),
            (out.data_ptr(), out_code, out.stride(0)))


def _nibble_workspace(n: int, device) -> torch.Tensor:
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=device)
    ws[:65536].zero_()
    return ws


def nibble_decode_workspace(lay: NibbleLayout, num_heads: int, num_reqs: int, max_seq_len: int,
                            device) -> torch.Tensor:
    """A workspace for `nibble_decode_paged` over batches of up to this shape. Its first 64 KiB
    (counters) are zero, and every call of either 4-bit read leaves them so: one buffer of the
    larger size serves both, call after call in stream order. Calls that may overlap, on two
    streams, take one each."""
    n = _hip.lib().ttkv_nibble_decode_workspace_bytes(lay.H, num_heads, num_reqs, max_seq_len)
    if n < 0:
        raise ValueError("invalid head count or batch for the decode workspace")
    return _nibble_workspace(int(n), device)


def nibble_decode_paged(lay: NibbleLayout, query: torch.Tensor, page: torch.Tensor,
                        block_size: int, block_table: torch.Tensor, seq_lens: torch.Tensor,
                        query_start_loc: torch.Tensor, max_seq_len: int, scale: float,
                        out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                        error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one query per request (row query_start_loc[r] of query [N, HQ, d], rotated)
    over its seq_lens[r] stored tokens of a 4-bit cache. See `ttkv_nibble_decode_paged` in
    include/ttkv_hip.h. Returns `out` [N, HQ, d] with the decode rows written.

    query_start_loc [B] or, as `step_plan` writes it, [B + 1] (of a longer one its first B + 1): a
    request whose entry equals the next one has no query in this step and is skipped."""
    index = _one_device(query, page, block_table, seq_lens, query_start_loc, out, workspace,
                        error_word)
    out, q_args, bt_args, out_args = _nibble_read(lay, query, page, block_table, seq_lens,
                                                  query_start_loc, out)
    B, HQ = seq_lens.numel(), query.shape[1]
    if block_table.shape[0] < B or query_start_loc.numel() < B:
        raise ValueError(f"{B} sequence lengths need as many block table rows and query rows")
    if query.shape[0] == 0:                     # every request waits
        return out
    if workspace is None:
        workspace = nibble_decode_workspace(lay, HQ, B, max_seq_len, query.device)
    err = _error_word(error_word, query.device)
    rc = _on_device(
        index, _hip.lib().ttkv_nibble_decode_starts_paged, lay.H, HQ, lay.d, float(scale), *q_args,
        int(block_size), *bt_args, seq_lens.data_ptr(), query_start_loc.data_ptr(),
        min(query_start_loc.numel(), B + 1), B,
        int(max_seq_len), *out_args, workspace.data_ptr(), workspace.numel(), err.data_ptr(),
        _stream(index))
    _hip.check(rc, "ttkv_nibble_decode_paged")
    return out


def nibble_prefill_workspace(lay: NibbleLayout, num_heads: int, num_reqs: int, max_q_len: int,
                             max_seq_len: int, device) -> torch.Tensor:
    """A workspace for `nibble_prefill_paged` over batches of up to this shape (see
    `nibble_decode_workspace`)."""
    n = _hip.lib().ttkv_nibble_prefill_workspace_bytes(lay.H, num_heads, num_reqs, max_q_len,
                                                       max_seq_len)
    if n < 0:
        raise ValueError("invalid head count or batch for the prefill workspace")
    return _nibble_workspace(int(n), device)


def nibble_prefill_paged(lay: NibbleLayout, query: torch.Tensor, page: torch.Tensor,
                         block_size: int, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         query_start_loc: torch.Tensor, max_q_len: int, max_seq_len: int,
                         scale: float, req_index: torch.Tensor | None = None,
                         out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                         error_word: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of chunks of queries (rows query_start_loc[r] .. [r + 1] of query
    [N, HQ, d], rotated) over their requests' stored tokens of a 4-bit cache, the chunk's own
    included. `req_index` picks the batch rows to process (default: all). See
    `ttkv_nibble_prefill_paged` in include/ttkv_hip.h."""
    index = _one_device(query, page, block_table, seq_lens, query_start_loc, req_index, out,
                        workspace, error_word)
    out, q_args, bt_args, out_args = _nibble_read(lay, query, page, block_table, seq_lens,
                                                  query_start_loc, out)
    B, HQ = seq_lens.numel(), query.shape[1]
    if block_table.shape[0] < B or query_start_loc.numel() < B + 1:
        raise ValueError(f"{B} sequence lengths need as many block table rows and one more "
                         f"query start")
    if query.shape[0] == 0:
        return out
    if req_index is not None:
        _i32(req_index, "req_index")
        B = req_index.numel()
    if workspace is None:
        workspace = nibble_prefill_workspace(lay, HQ, B, max_q_len, max_seq_len, query.device)
    err = _error_word(error_word, query.device)
    rc = _on_device(
        index, _hip.lib().ttkv_nibble_prefill_paged, lay.H, HQ, lay.d, float(scale), *q_args,
        int(block_size), *bt_args, seq_lens.data_ptr(), query_start_loc.data_ptr(),
        _hip.ptr(req_index), B, int(max_q_len), int(max_seq_len), *out_args,
        workspace.data_ptr(), workspace.numel(), err.data_ptr(), _stream(index))
    _hip.check(rc, "ttkv_nibble_prefill_paged")
    return out

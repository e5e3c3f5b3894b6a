"""Block tables, slot mapping, positions and lengths of a ragged batch, built on the GPU.

One call per step turns request lengths into what the paged operators read: the slots of
``int8_kv_cache_write`` / ``reshape_and_cache_int8`` (vllm_int8/vllm_int8_cache_ops.py:134-210 of
the reference), the block tables and lengths of ``int8_paged_attention``, the positions of the
rotary step, and the request of every token.  Lengths stay on the device, so the call can be
captured into a HIP graph and nothing waits for the host.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _decode, _ext, _lib


class BatchTables(NamedTuple):
    """The outputs of ``build_batch_tables``."""

    query_starts: torch.Tensor  # int32 [requests + 1], first token of each request
    seq_lens: torch.Tensor  # int32 [requests], tokens in the cache after the step
    positions: torch.Tensor  # int64 [tokens], 0 behind the last token
    slot_mapping: torch.Tensor  # int64 [tokens], -1 where nothing is to be written
    token_requests: torch.Tensor  # int32 [tokens], -1 behind the last token
    free_end: torch.Tensor  # int64 [1], free_start plus the blocks taken


def batch_tables_buffers(requests: int, tokens: int, device) -> BatchTables:
    """Buffers for ``build_batch_tables(..., out=)`` (a serving loop keeps one set)."""

    def empty(n, dtype):
        return torch.empty(n, dtype=dtype, device=device)

    return BatchTables(empty(requests + 1, torch.int32), empty(requests, torch.int32),
                       empty(tokens, torch.int64), empty(tokens, torch.int64),
                       empty(tokens, torch.int32), empty(1, torch.int64))


_OUT_DTYPES = (torch.int32, torch.int32, torch.int64, torch.int64, torch.int32, torch.int64)


def build_batch_tables(
    computed_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_tables: torch.Tensor,
    free_blocks: torch.Tensor,
    num_tokens: int,
    *,
    block_size: int = 16,
    free_start: torch.Tensor | None = None,
    out: BatchTables | None = None,
) -> BatchTables:
    """Extends ``block_tables`` by the blocks this step's tokens need and builds their indices.

    Request r has ``computed_lens[r]`` tokens in the cache and brings ``new_lens[r]`` more (int32 or
    int64 [requests]; negative lengths count as 0).  The blocks it lacks are taken from
    ``free_blocks`` (int32), starting at ``free_start`` (int64 [1] on the device, default 0), in
    request order, and written into its row of ``block_tables`` (int32 [requests, width], unit inner
    stride, in place); no other entry changes.  ``num_tokens`` rows of token outputs follow each
    other request by request; rows behind the last token are padding (slot -1), and tokens that
    do not fit are dropped as if their request brought fewer.

    A token's slot is -1 where its block lies past the table's width or the free list ran out
    (``free_end`` then exceeds ``free_blocks.numel()``).  ``out.free_end`` may be ``free_start`` itself;
    no other output may share memory with an input.
    """
    ext = None if _decode.DEBUG_CHECKS else _ext.module()
    if ext is not None:
        if out is None:
            out = batch_tables_buffers(computed_lens.numel(), int(num_tokens), computed_lens.device)
        ext.build_batch_tables(computed_lens, new_lens, block_tables, free_blocks, num_tokens,
                               block_size, free_start, *out)
        return out
    assert computed_lens.dim() == 1 and new_lens.shape == computed_lens.shape
    assert computed_lens.dtype in (torch.int32, torch.int64) and new_lens.dtype == computed_lens.dtype
    requests = computed_lens.numel()
    assert block_tables.dim() == 2 and block_tables.shape[0] == requests
    assert block_tables.dtype == torch.int32
    assert block_tables.stride(1) == 1 or block_tables.shape[1] <= 1 or requests == 0
    assert block_tables.stride(0) >= block_tables.shape[1] or requests <= 1, \
        "rows of block_tables overlap"
    assert free_blocks.dim() == 1 and free_blocks.dtype == torch.int32
    assert 0 <= num_tokens <= 2**31 - 1, "num_tokens must lie in [0, 2^31 - 1]"
    assert 1 <= block_size <= 65536, "block_size must lie in [1, 65536]"
    assert computed_lens.is_cuda, "build_batch_tables needs GPU tensors"
    dev = computed_lens.device
    given = [new_lens, block_tables, free_blocks]
    if free_start is not None:
        assert free_start.dtype == torch.int64 and free_start.numel() == 1
        given.append(free_start)
    if out is None:
        out = batch_tables_buffers(requests, num_tokens, dev)
    sizes = (requests + 1, requests, num_tokens, num_tokens, num_tokens, 1)
    for t, dtype, size in zip(out, _OUT_DTYPES, sizes):
        assert t.dtype == dtype and t.is_contiguous() and t.numel() == size
    assert all(t.device == dev for t in [*given, *out]), "all tensors must be on one device (the GPU)"
    lens = {computed_lens.data_ptr(), new_lens.data_ptr()}
    assert not requests or not any(t.numel() and t.data_ptr() in lens for t in out), \
        "an output shares memory with the lengths"
    if _decode.DEBUG_CHECKS:
        _debug_check(computed_lens, new_lens, block_tables, free_blocks, num_tokens, block_size,
                     free_start)
    computed_lens, new_lens = computed_lens.contiguous(), new_lens.contiguous()
    free_blocks = free_blocks.contiguous()
    lib = _lib.load()
    with torch.cuda.device(dev):
        stream = _lib.stream_handle(dev)
        need = lib.int8kv_batch_tables_workspace_bytes(requests)
        ws = _decode._cached_workspace(dev, stream, need)
        status = lib.int8kv_batch_tables(
            computed_lens.data_ptr(), new_lens.data_ptr(), _lib.DTYPE_CODE[computed_lens.dtype],
            requests, block_tables.data_ptr(), block_tables.shape[1], block_tables.stride(0),
            block_size, free_blocks.data_ptr(), free_blocks.numel(),
            None if free_start is None else free_start.data_ptr(), num_tokens,
            *(t.data_ptr() for t in out), ws.data_ptr(), ws.numel(), stream)
    _lib.check(status, "int8kv_batch_tables")
    return out


def _debug_check(computed_lens, new_lens, block_tables, free_blocks, num_tokens, block_size,
                 free_start) -> None:
    """Host-side checks (INT8KV_DEBUG=1): every token fits the outputs and the tables, and the free
    list holds the blocks the step takes."""
    c, n = computed_lens.to("cpu", torch.int64), new_lens.to("cpu", torch.int64)
    assert bool((c >= 0).all()) and bool((n >= 0).all()), "negative length"
    assert int(n.sum()) <= num_tokens, "num_tokens is less than the new tokens"
    need = (c + n + block_size - 1) // block_size
    assert not need.numel() or int(need.max()) <= block_tables.shape[1], "block_tables is too narrow"
    taken = int((need - (c + block_size - 1) // block_size).sum())
    start = 0 if free_start is None else int(free_start.item())
    assert 0 <= start and start + taken <= free_blocks.numel(), "not enough free blocks"

"""Sampling with temperature, top-k, top-p and min-p from given random numbers.

The counterpart of the greedy ``hip_argmax_rows`` of the decode loop: one call per step, every row
with its own settings, all of them device tensors, so that a captured step follows whatever the
host writes into them between replays.
"""

from __future__ import annotations

import torch

from . import _decode, _ext, _lib

MAX_VOCAB = 1 << 21
MAX_ROWS = 1 << 16


def sample_tokens(
    logits: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    temperature: torch.Tensor | None = None,
    top_k: torch.Tensor | None = None,
    top_p: torch.Tensor | None = None,
    min_p: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """One token (int64) per row of ``logits`` [rows, vocab] (float32, float16 or bfloat16, unit
    inner stride).

    With v a row's logits (NaN counts as -inf) and w_i = exp((v_i - max v) / temperature): the
    tokens are ordered by falling logit, equal ones by index; top-k keeps the first ``top_k``,
    top-p those of them whose preceding weight is below ``top_p`` times theirs altogether, min-p
    those with w >= ``min_p`` (the first one always stays).  The token is the first kept one, in
    index order, at which the kept weight up to it exceeds ``uniforms`` (float32 in [0, 1)) times all of
    it.  Rows with temperature 0, and rows without a finite logit, give the first maximum.

    Settings: float32 (top_k int32) [rows]; None, top_k <= 0, top_p >= 1 and min_p <= 0 switch a
    filter off, temperature None is 1.  The result depends on the inputs alone: weights are
    computed in 64 bits and summed as integers."""
    ext = _ext.module()
    if ext is not None:
        return ext.sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, out)
    assert logits.dim() == 2 and logits.dtype in _decode.QUERY_DTYPES
    rows, vocab = logits.shape
    assert 1 <= vocab <= MAX_VOCAB, "vocab must lie in [1, 2^21]"
    assert rows <= MAX_ROWS, "at most 2^16 rows"
    assert logits.stride(1) == 1 or vocab == 1
    assert logits.stride(0) >= vocab or rows <= 1, "rows of logits overlap"
    assert logits.is_cuda, "sample_tokens needs GPU tensors"
    settings = [uniforms, temperature, top_k, top_p, min_p]
    for i, t in enumerate(settings):
        if t is not None:
            assert t.dtype == (torch.int32 if i == 2 else torch.float32) and t.shape == (rows,)
            assert t.device == logits.device, "all tensors must be on one device (the GPU)"
            settings[i] = t.contiguous()
    if out is None:
        out = torch.empty(rows, dtype=torch.int64, device=logits.device)
    assert out.dtype == torch.int64 and out.is_contiguous() and out.shape == (rows,)
    assert out.device == logits.device, "all tensors must be on one device (the GPU)"
    lib, dev = _lib.load(), logits.device
    with torch.cuda.device(dev):
        stream = _lib.stream_handle(dev)
        ws = _decode._cached_workspace(dev, stream, lib.int8kv_sample_workspace_bytes(rows, vocab))
        status = lib.int8kv_sample_rows(
            logits.data_ptr(), _lib.DTYPE_CODE[logits.dtype], rows, vocab, max(logits.stride(0), vocab),
            *(None if t is None else t.data_ptr() for t in settings), out.data_ptr(), ws.data_ptr(),
            ws.numel(), stream)
    _lib.check(status, "int8kv_sample_rows")
    return out

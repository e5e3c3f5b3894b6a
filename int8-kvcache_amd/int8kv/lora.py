"""Low-rank adapters of many requests beside a shared projection.

A serving step computes the shared projection for all its tokens at once (``hip_linear`` or a
library product) and adds each token's own adapter to it:

    plan = lora_plan(adapter_ids, num_adapters)           # once per step, for all projections
    qkv = hip_linear(h, wqkv, bqkv, ...)
    lora_add(qkv, h, lora_a, lora_b, plan, out=qkv)       # in place

The grouping of tokens by adapter happens on the GPU, so both calls can be captured into a HIP
graph whose replays follow the ids in ``adapter_ids``.
"""

from __future__ import annotations

import torch

from . import _decode, _ext, _lib

MAX_ADAPTERS = 4096
MAX_RANK = 128


class LoraPlan:
    """A step's tokens grouped by adapter (``lora_plan``)."""

    __slots__ = ("buffer", "tokens", "num_adapters")

    def __init__(self, buffer: torch.Tensor, tokens: int, num_adapters: int):
        self.buffer, self.tokens, self.num_adapters = buffer, tokens, num_adapters


def lora_plan(adapter_ids: torch.Tensor, num_adapters: int, plan: LoraPlan | None = None) -> LoraPlan:
    """Groups the tokens of a step by adapter (int32 or int64 ids [tokens]; an id outside
    [0, num_adapters) means none).  ``plan``: an earlier plan of the same sizes to fill again."""
    if plan is not None:
        assert (plan.tokens, plan.num_adapters) == (adapter_ids.numel(), num_adapters), \
            "a plan of other sizes"
    ext = _ext.module()
    if ext is not None:
        buffer = ext.lora_plan(adapter_ids, num_adapters, None if plan is None else plan.buffer)
        return plan if plan is not None else LoraPlan(buffer, adapter_ids.numel(), num_adapters)
    assert adapter_ids.dim() == 1 and adapter_ids.dtype in (torch.int32, torch.int64)
    assert 1 <= num_adapters <= MAX_ADAPTERS, "num_adapters must lie in [1, 4096]"
    assert adapter_ids.is_cuda, "lora_plan needs GPU tensors"
    tokens, dev = adapter_ids.numel(), adapter_ids.device
    assert tokens <= 1 << 24, "at most 2^24 tokens"
    ids = adapter_ids.contiguous()
    lib = _lib.load()
    need = lib.int8kv_lora_plan_bytes(tokens, num_adapters)
    if plan is None:
        plan = LoraPlan(torch.empty(need, dtype=torch.uint8, device=dev), tokens, num_adapters)
    assert plan.buffer.device == dev, "all tensors must be on one device (the GPU)"
    with torch.cuda.device(dev):
        status = lib.int8kv_lora_plan(ids.data_ptr(), _lib.DTYPE_CODE[ids.dtype], tokens,
                                      num_adapters, plan.buffer.data_ptr(), plan.buffer.numel(),
                                      _lib.stream_handle(dev))
    _lib.check(status, "int8kv_lora_plan")
    return plan


def lora_add(
    base: torch.Tensor,
    x: torch.Tensor,
    lora_a: torch.Tensor,
    lora_b: torch.Tensor,
    plan: LoraPlan,
    *,
    scales: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """out = base + scales[a] * (x lora_a[a]^T) lora_b[a]^T for each token's adapter a.

    bf16 [tokens, n] base and out, [tokens, k] x, [num_adapters, rank, k] lora_a and
    [num_adapters, n, rank] lora_b, with unit inner strides and 16-byte aligned rows (views into
    wider rows included); scales float32 [num_adapters].  k, n and rank (at most 128) are multiples
    of 8.  Tokens without an adapter get their base row.  ``out`` may be ``base`` itself, and must
    not otherwise overlap the inputs.  Sums are fp32, rounded once."""
    ext = _ext.module()
    if ext is not None:
        return ext.lora_add(base, x, lora_a, lora_b, plan.buffer, plan.tokens, plan.num_adapters,
                            scales, out)
    for t, dim in ((base, 2), (x, 2), (lora_a, 3), (lora_b, 3)):
        assert t.dim() == dim and t.dtype == torch.bfloat16, "lora_add takes bf16 matrices"
        assert t.stride(-1) == 1, "lora_add takes matrices with a unit inner stride"
    tokens, k = x.shape
    n, (adapters, rank, _) = base.shape[1], lora_a.shape
    assert base.shape[0] == tokens and lora_a.shape[2] == k
    assert lora_b.shape == (adapters, n, rank)
    assert k % 8 == 0 and n % 8 == 0 and rank % 8 == 0 and 8 <= rank <= MAX_RANK and k > 0 and n > 0, \
        "k, n and rank must be multiples of 8, rank at most 128"
    assert (plan.tokens, plan.num_adapters) == (tokens, adapters), "a plan of other sizes"
    assert x.is_cuda, "lora_add needs GPU tensors"
    given = [base, lora_a, lora_b, plan.buffer]
    if scales is not None:
        assert scales.dtype == torch.float32 and scales.shape == (adapters,)
        given.append(scales)
        scales = scales.contiguous()
    if out is None:
        out = torch.empty(tokens, n, dtype=base.dtype, device=base.device)
    assert out.shape == base.shape and out.dtype == torch.bfloat16 and out.stride(1) == 1
    assert all(t.device == x.device for t in [*given, out]), "all tensors must be on one device (the GPU)"
    lib, dev = _lib.load(), x.device
    with torch.cuda.device(dev):
        stream = _lib.stream_handle(dev)
        need = lib.int8kv_lora_workspace_bytes(tokens, adapters, k, rank)
        ws = _decode._cached_workspace(dev, stream, need)
        status = lib.int8kv_lora_add(
            base.data_ptr(), base.stride(0), x.data_ptr(), tokens, k, x.stride(0), lora_a.data_ptr(),
            _lib.strides(lora_a), lora_b.data_ptr(), _lib.strides(lora_b), adapters, rank, n,
            None if scales is None else scales.data_ptr(), plan.buffer.data_ptr(),
            plan.buffer.numel(), out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(), stream)
    _lib.check(status, "int8kv_lora_add")
    return out

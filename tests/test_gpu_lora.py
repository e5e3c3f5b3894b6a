"""lora_plan and lora_add against 64 bits, within the bound that fp32 sums, the two bf16 parts of the
rank-wide vector and one rounding to bf16 allow (serving_cases.lora_ref derives it)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import int8kv
from int8kv import _ext, _lib
from serving_cases import lora_ref

pytestmark = pytest.mark.gpu


def inputs(cuda, tokens, k, n, rank, adapters, seed, ids=None):
    g = torch.Generator().manual_seed(seed)

    def normal(*size, std=1.0):
        return (torch.randn(*size, generator=g) * std).to(torch.bfloat16)

    if ids is None:
        ids = torch.randint(-1, adapters, (tokens,), generator=g)
    d = dict(base=normal(tokens, n), x=normal(tokens, k), a=normal(adapters, rank, k, std=k**-0.5),
             b=normal(adapters, n, rank, std=0.1), scales=torch.rand(adapters, generator=g) * 3 - 1)
    d = {key: t.to(cuda) for key, t in d.items()}
    d["ids"] = ids.to(cuda)
    return d


def check(d, out, scales=True):
    f = {key: d[key].float().cpu().numpy() for key in ("base", "x", "a", "b", "scales")}
    s = f["scales"] if scales else np.ones_like(f["scales"])
    ref, bound = lora_ref(f["base"], f["x"], f["a"], f["b"], d["ids"].cpu().tolist(),
                          s.astype(np.float64))
    off = np.abs(out.float().cpu().numpy().astype(np.float64) - ref)
    assert (off <= bound).all(), float((off - bound).max())


def add(d, **kw):
    plan = int8kv.lora_plan(d["ids"], d["a"].shape[0])
    kw.setdefault("scales", d["scales"])
    return int8kv.lora_add(d["base"], d["x"], d["a"], d["b"], plan, **kw)


@pytest.mark.parametrize("tokens,k,n,rank,adapters", [
    (1, 8, 8, 8, 1),
    (1, 3584, 4608, 16, 8),
    (5, 264, 136, 24, 3),
    (17, 512, 1000, 8, 40),
    (32, 3584, 520, 16, 24),
    (33, 1032, 264, 40, 4),
    (64, 128, 72, 64, 2),
    (100, 640, 392, 72, 5),
    (130, 256, 264, 128, 7),
    (200, 40, 16, 120, 200),
    (700, 520, 328, 32, 9),
    (1030, 264, 520, 104, 3),
])
def test_against_64_bits(cuda, tokens, k, n, rank, adapters):
    d = inputs(cuda, tokens, k, n, rank, adapters, seed=tokens + k)
    check(d, add(d))
    check(d, add(d, scales=None), scales=False)


def test_runs_of_one_adapter_and_none(cuda):
    """Prefill-like runs, all tokens on one adapter, and no token with one."""
    ids = torch.repeat_interleave(torch.tensor([2, -1, 0, 3, 2, 1]), torch.tensor([70, 9, 1, 150, 64, 33]))
    d = inputs(cuda, 327, 264, 136, 16, 4, seed=1, ids=ids)
    check(d, add(d))
    d["ids"] = torch.full((327,), 1, device=cuda)
    check(d, add(d))
    for none in (-1, -(2**31), 4, 2**31 - 1):
        d["ids"] = torch.full((327,), none, device=cuda, dtype=torch.int32)
        assert torch.equal(add(d), d["base"])


def test_rows_without_an_adapter_are_the_base_rows(cuda):
    """Bit for bit, NaN and infinities included; the other rows are not touched by them."""
    d = inputs(cuda, 40, 128, 64, 16, 3, seed=2)
    none = d["ids"] < 0
    clean = add(d)
    d["base"][none] = float("nan")
    d["x"][none] = float("inf")
    out = add(d)
    assert torch.isnan(out[none]).all() and torch.equal(out[~none], clean[~none])


def test_non_finite_rows_stay_their_own(cuda):
    """One token's infinity reaches its own row alone, also among tokens of the same adapter."""
    d = inputs(cuda, 50, 264, 72, 16, 2, seed=3, ids=torch.arange(50) % 2)
    clean = add(d)
    d["x"][7, 5] = float("inf")
    out = add(d)
    keep = torch.arange(50, device=cuda) != 7
    assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[7]).any()


def test_infinite_intermediate_without_sign_conflict(cuda):
    """x A^T infinite and B of one sign: the sum is that infinity, as in plain arithmetic."""
    d = inputs(cuda, 3, 64, 16, 8, 1, seed=4, ids=torch.zeros(3, dtype=torch.int64))
    d["x"].fill_(3.0e38)
    d["a"].fill_(1.0)
    d["b"].fill_(0.5)
    d["scales"].fill_(1.0)
    assert (add(d) == float("inf")).all()


def test_large_intermediate_keeps_its_bits(cuda):
    """A rank-wide vector close to the largest fp32 value: its upper part must not overflow."""
    d = inputs(cuda, 2, 64, 16, 8, 1, seed=5, ids=torch.zeros(2, dtype=torch.int64))
    d["x"].zero_()
    d["x"][:, 0] = 3.3895e38  # the largest bf16 value
    d["a"].zero_()
    d["a"][0, 0, 0] = 1.0
    d["b"].zero_()
    d["b"][0, :, 0] = 2.0**-100
    d["scales"].fill_(1.0)
    out = add(d).float()
    want = d["base"].float() + d["x"][0, 0].float() * 2.0**-100
    assert torch.allclose(out, want, rtol=2.0**-8, atol=0)


def test_views_and_in_place(cuda):
    """Base and out inside wider rows (a slice of a packed projection), weights inside wider
    buffers, int64 ids, out in place; the columns around stay."""
    d = inputs(cuda, 37, 264, 136, 24, 5, seed=6)
    want = add(d)
    packed = torch.full((37, 400), 7.0, dtype=torch.bfloat16, device=cuda)
    packed[:, 64:200] = d["base"]
    view = packed[:, 64:200]
    xs = torch.zeros(37, 512, dtype=torch.bfloat16, device=cuda)
    xs[:, 16:280] = d["x"]
    aw = torch.zeros(5, 32, 512, dtype=torch.bfloat16, device=cuda)
    aw[:, 8:, 8:272] = d["a"]
    bw = torch.zeros(5, 200, 64, dtype=torch.bfloat16, device=cuda)
    bw[:, 3:139, 16:40] = d["b"]
    plan = int8kv.lora_plan(d["ids"].long(), 5)
    got = int8kv.lora_add(view, xs[:, 16:280], aw[:, 8:, 8:272], bw[:, 3:139, 16:40], plan,
                          scales=d["scales"], out=view)
    assert got.data_ptr() == view.data_ptr() and torch.equal(view, want)
    assert (packed[:, :64] == 7).all() and (packed[:, 200:] == 7).all()


def test_ctypes_path_and_other_stream(cuda):
    d = inputs(cuda, 90, 520, 264, 32, 6, seed=7)
    want = add(d)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        got = add(d)
    side.synchronize()
    with _ext.use_ctypes():
        other = add(d)
    assert torch.equal(got, want) and torch.equal(other, want)


def test_repeated_calls_are_bit_identical(cuda):
    d = inputs(cuda, 600, 1032, 264, 16, 30, seed=8)
    want = add(d)
    for _ in range(3):
        assert torch.equal(add(d), want)


def test_captured_plan_follows_the_ids(cuda):
    """Plan and product captured; the ids change between replays, with eager calls in between."""
    d = inputs(cuda, 24, 264, 136, 16, 6, seed=9)
    other = inputs(cuda, 300, 520, 264, 64, 6, seed=10)
    out = torch.empty_like(d["base"])
    plan = int8kv.lora_plan(d["ids"], 6)
    int8kv.lora_add(d["base"], d["x"], d["a"], d["b"], plan, scales=d["scales"], out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        int8kv.lora_plan(d["ids"], 6, plan=plan)
        int8kv.lora_add(d["base"], d["x"], d["a"], d["b"], plan, scales=d["scales"], out=out)
    for step in range(4):
        d["ids"].copy_(torch.randint(-1, 6, (24,), generator=torch.Generator().manual_seed(step)))
        graph.replay()
        check(other, add(other))
        torch.cuda.synchronize()
        check(d, out)


def test_no_tokens(cuda):
    d = inputs(cuda, 0, 64, 16, 8, 2, seed=11)
    assert add(d).shape == (0, 16)


def test_misaligned_rows_are_refused(cuda):
    d = inputs(cuda, 4, 64, 16, 8, 2, seed=12)
    plan = int8kv.lora_plan(d["ids"], 2)
    wide = torch.zeros(4, 73, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(_lib.Int8KVError, match="STRIDE"):
        int8kv.lora_add(d["base"], wide[:, 1:65], d["a"], d["b"], plan)
    with pytest.raises(AssertionError):
        int8kv.lora_add(d["base"][:, ::2], d["x"], d["a"], d["b"], plan)


@pytest.mark.parametrize("tokens,k,n,rank,adapters", [
    (20, 520, 328, 32, 9),      # one launch, rank a multiple of 32
    (23, 1024, 264, 32, 12),    # the longest A that one launch takes
    (40, 1024, 1544, 16, 24),
    (300, 264, 520, 8, 48),
    (9, 4104, 264, 24, 3),      # two launches
    (6, 4104, 1032, 8, 4),      # a little over the longest A
    (70, 2056, 264, 32, 30),
])
def test_small_tiles_of_both_forms(cuda, tokens, k, n, rank, adapters):
    """Tiles of 16 tokens with short and with long adapters: values, infinities in their own row,
    rows without an adapter, and out in place."""
    d = inputs(cuda, tokens, k, n, rank, adapters, seed=tokens + rank)
    want = add(d)
    check(d, want)
    none = (d["ids"] < 0) | (d["ids"] >= adapters)
    marked = int(torch.nonzero(~none)[0])
    d["base"][none] = float("nan")
    d["x"][none] = float("inf")
    d["x"][marked, k - 1] = float("-inf")
    out = add(d, out=d["base"])
    assert out.data_ptr() == d["base"].data_ptr() and torch.isnan(out[none]).all()
    same = ~none
    same[marked] = False
    assert torch.equal(out[same], want[same]) and not torch.isfinite(out[marked]).any()


@pytest.mark.parametrize("tokens,adapters,run", [(17001, 3, 700), (20000, 4000, 1), (33000, 1, 50)])
def test_more_tokens_than_a_plan_holds(cuda, tokens, adapters, run):
    """Plans that count their tokens twice: runs of one adapter, and neighbours of all kinds."""
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, adapters, (tokens // run + 1,), generator=g).repeat_interleave(run)[:tokens]
    d = inputs(cuda, tokens, 40, 24, 8, adapters, seed=13, ids=ids)
    check(d, add(d))


@pytest.mark.parametrize("tokens,k,n,rank,adapters", [
    (200, 264, 136, 24, 3),       # tiles of 64 taken as quarters, one launch
    (130, 4104, 264, 32, 2),      # as quarters, two launches
    (96, 1032, 264, 128, 1),
    (3000, 2048, 264, 128, 5),    # whole tiles (122 MB as quarters), the parts summed beforehand
    (2500, 3000, 520, 56, 40),    # whole tiles, no sums
])
def test_whole_tiles_and_quarters(cuda, tokens, k, n, rank, adapters):
    """Tiles of 64 tokens in both readings, with partly filled ones, out in place and not."""
    d = inputs(cuda, tokens, k, n, rank, adapters, seed=tokens)
    want = add(d)
    check(d, want)
    none = (d["ids"] < 0) | (d["ids"] >= adapters)
    d["x"][none] = float("nan")
    out = add(d, out=d["base"])
    assert out.data_ptr() == d["base"].data_ptr() and torch.equal(out, want)


def test_out_beside_x_in_the_same_rows(cuda):
    """Columns of one buffer: out beside x is fine, out over x or over base's other rows is refused."""
    d = inputs(cuda, 21, 264, 136, 16, 3, seed=14)
    want = add(d)
    packed = torch.zeros(21, 400, dtype=torch.bfloat16, device=cuda)
    packed[:, :264] = d["x"]
    plan = int8kv.lora_plan(d["ids"], 3)
    rest = dict(scales=d["scales"])
    got = int8kv.lora_add(d["base"], packed[:, :264], d["a"], d["b"], plan, out=packed[:, 264:], **rest)
    assert torch.equal(got, want) and torch.equal(packed[:, :264], d["x"])
    wide = torch.zeros(22, 136, dtype=torch.bfloat16, device=cuda)
    for base, x, out in ((d["base"], packed[:, :264], packed[:, 128:264]), (wide[:21], d["x"], wide[1:])):
        with pytest.raises(_lib.Int8KVError, match="STRIDE"):
            int8kv.lora_add(base, x, d["a"], d["b"], plan, out=out, **rest)
        with _ext.use_ctypes(), pytest.raises(_lib.Int8KVError, match="STRIDE"):
            int8kv.lora_add(base, x, d["a"], d["b"], plan, out=out, **rest)

"""build_batch_tables against a token-by-token reference: every output and every table entry equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import int8kv
from int8kv import _decode, _ext, _lib
from serving_cases import batch_tables_ref

pytestmark = pytest.mark.gpu


def make(requests, longest, new, bs, seed, dtype=torch.int32, width=None, zero=0.1):
    g = np.random.default_rng(seed)
    c = g.integers(0, longest + 1, requests)
    n = np.full(requests, new) if new <= 1 else g.integers(0, new + 1, requests)
    c[g.random(requests) < zero] = 0
    n[g.random(requests) < zero] = 0
    width = -(-(longest + max(new, 1)) // bs) if width is None else width
    tables = np.full((requests, width), -7, np.int64)
    pool = g.permutation(requests * width + 64)
    used = 0
    for r in range(requests):
        have = min(width, -(-int(c[r]) // bs))
        tables[r, :have] = pool[used:used + have]
        used += have
    return dict(c=c, n=n, tables=tables, free=pool[used:], dtype=dtype, bs=bs)


def run(case, cuda, tokens, start=None, out=None, tables=None, alias=False):
    """Runs the operator; returns its outputs as numpy beside the reference's."""
    dt = case["dtype"]
    tb = torch.tensor(case["tables"], dtype=torch.int32, device=cuda) if tables is None else tables
    fs = None if start is None else torch.tensor([start], dtype=torch.int64, device=cuda)
    if alias:
        out = int8kv.batch_tables_buffers(len(case["c"]), tokens, cuda)._replace(free_end=fs)
    got = int8kv.build_batch_tables(
        torch.tensor(case["c"], dtype=dt, device=cuda), torch.tensor(case["n"], dtype=dt, device=cuda),
        tb, torch.tensor(case["free"], dtype=torch.int32, device=cuda), tokens,
        block_size=case["bs"], free_start=fs, out=out)
    torch.cuda.synchronize()
    ref = batch_tables_ref(case["c"], case["n"], case["tables"], case["free"], start or 0,
                           case["bs"], tokens)
    return tb, got, ref


def check(tb, got, ref):
    assert np.array_equal(tb.cpu().numpy(), ref["tables"])
    for name in ("query_starts", "seq_lens", "positions", "slot_mapping", "token_requests"):
        assert np.array_equal(getattr(got, name).cpu().numpy(), ref[name]), name
    assert int(got.free_end.item()) == ref["free_end"]


@pytest.mark.parametrize("requests,longest,new,bs,dtype,pad", [
    (1, 1, 1, 16, torch.int32, 0),
    (32, 8192, 1, 16, torch.int32, 0),
    (7, 300, 200, 16, torch.int64, 11),
    (3, 5000, 4000, 64, torch.int32, 1),
    (257, 700, 1, 32, torch.int64, 31),
    (1000, 40, 40, 1, torch.int32, 5),
    (13, 77, 900, 48, torch.int64, 0),  # a block size between the powers of two
    (2048, 100, 3, 16, torch.int32, 7),
    (2049, 100, 3, 16, torch.int64, 7),  # more requests than one launch scans
    (5000, 64, 20, 16, torch.int32, 100),
])
def test_against_reference(cuda, requests, longest, new, bs, dtype, pad):
    case = make(requests, longest, new, bs, seed=requests + longest, dtype=dtype)
    tokens = int(case["n"].sum()) + pad
    check(*run(case, cuda, tokens, start=3))


def test_free_start_in_place(cuda):
    """free_end written over free_start, with one workgroup and with many."""
    for requests, new, seed in ((40, 1, 1), (40, 500, 2), (3000, 9, 3)):
        case = make(requests, 600, new, 16, seed)
        tokens = int(case["n"].sum())
        check(*run(case, cuda, tokens, start=5, alias=True))


def test_free_list_runs_out(cuda):
    case = make(20, 100, 90, 16, seed=4)
    for keep in (0, 1, 17):
        case["free"] = case["free"][:keep]
        check(*run(case, cuda, int(case["n"].sum()), start=0))
    case = make(20, 100, 90, 16, seed=5)
    for start in (-3, len(case["free"]) - 4, 2**40):
        check(*run(case, cuda, int(case["n"].sum()), start=start))


def test_table_narrower_than_the_lengths(cuda):
    case = make(11, 200, 120, 16, seed=6, width=9)
    check(*run(case, cuda, int(case["n"].sum()), start=2))
    case = make(4, 0, 5, 16, seed=7, width=0)
    case["c"][:] = 0
    check(*run(case, cuda, int(case["n"].sum()), start=0))


def test_tokens_that_do_not_fit_are_dropped(cuda):
    for requests in (30, 2100):
        case = make(requests, 90, 70, 16, seed=8)
        total = int(case["n"].sum())
        for tokens in (0, 1, total // 2, total - 1):
            check(*run(case, cuda, tokens, start=1))


def test_odd_lengths(cuda):
    """Negative lengths count as 0, those past 2^31 - 1 as that, and positions pass 2^31."""
    case = make(6, 50, 20, 16, seed=9, dtype=torch.int64)
    case["c"] = np.array([-5, 2**31 - 1, 2**40, 7, 0, 2**31 - 3])
    case["n"] = np.array([4, 3, 2, -(2**33), 0, 6])
    check(*run(case, cuda, 20, start=0))


def test_outputs_over_the_lengths_are_refused(cuda):
    lens = torch.ones(4, dtype=torch.int32, device=cuda)
    tables = torch.zeros(4, 3, dtype=torch.int32, device=cuda)
    free = torch.arange(9, dtype=torch.int32, device=cuda)
    out = int8kv.batch_tables_buffers(4, 4, cuda)
    for bad in (out._replace(seq_lens=lens), out._replace(token_requests=lens)):
        with pytest.raises(AssertionError, match="shares memory"):
            int8kv.build_batch_tables(lens, lens.clone(), tables, free, 4, out=bad)
        with _ext.use_ctypes(), pytest.raises(AssertionError, match="shares memory"):
            int8kv.build_batch_tables(lens, lens.clone(), tables, free, 4, out=bad)


def test_no_requests(cuda):
    case = dict(c=np.zeros(0, np.int64), n=np.zeros(0, np.int64), tables=np.zeros((0, 4), np.int64),
                free=np.arange(3), dtype=torch.int32, bs=16)
    check(*run(case, cuda, 5, start=1))
    check(*run(case, cuda, 0, start=1))


def test_views(cuda):
    """Strided lengths and tables inside wider buffers; what lies around them stays."""
    case = make(25, 300, 60, 16, seed=10)
    wide = torch.full((25, case["tables"].shape[1] + 6), 99, dtype=torch.int32, device=cuda)
    view = wide[:, 2:2 + case["tables"].shape[1]]
    view.copy_(torch.tensor(case["tables"], dtype=torch.int32))
    tb, got, ref = run(case, cuda, int(case["n"].sum()), start=0, tables=view)
    check(tb, got, ref)
    assert (wide[:, :2] == 99).all() and (wide[:, -4:] == 99).all()
    lens = torch.tensor(np.stack([case["c"], case["n"]], 1), dtype=torch.int32, device=cuda)
    got = int8kv.build_batch_tables(lens[:, 0], lens[:, 1], view.contiguous(),
                                    torch.tensor(case["free"], dtype=torch.int32, device=cuda),
                                    int(case["n"].sum()))
    assert np.array_equal(got.slot_mapping.cpu().numpy(), ref["slot_mapping"])


def test_ctypes_path_and_other_stream(cuda):
    case = make(60, 500, 33, 16, seed=11)
    tokens = int(case["n"].sum()) + 2
    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        check(*run(case, cuda, tokens, start=4))
    with _ext.use_ctypes():
        check(*run(case, cuda, tokens, start=4))


def test_captured_decode_steps(cuda):
    """A captured step advances lengths and the free list on the device, step after step, across
    block bounds, with eager work between the replays."""
    bs, requests, width, steps = 4, 9, 40, 25
    g = np.random.default_rng(12)
    c0 = g.integers(0, 30, requests)
    pool = g.permutation(requests * width)
    tables0 = np.full((requests, width), -1, np.int64)
    used = 0
    for r in range(requests):
        have = -(-int(c0[r]) // bs)
        tables0[r, :have] = pool[used:used + have]
        used += have
    free = pool[used:]
    lens = torch.tensor(c0, dtype=torch.int32, device=cuda)
    ones = torch.ones_like(lens)
    tables = torch.tensor(tables0, dtype=torch.int32, device=cuda)
    free_t = torch.tensor(free, dtype=torch.int32, device=cuda)
    head = torch.zeros(1, dtype=torch.int64, device=cuda)
    out = int8kv.batch_tables_buffers(requests, requests, cuda)._replace(free_end=head)

    def step():
        int8kv.build_batch_tables(lens, ones, tables, free_t, requests, block_size=bs,
                                  free_start=head, out=out)
        lens.add_(ones)

    side = torch.cuda.Stream(cuda)
    saved = lens.clone(), tables.clone(), head.clone()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    for t, s in zip((lens, tables, head), saved):
        t.copy_(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    c, tb, h = c0.copy(), tables0, 0
    for _ in range(steps):
        graph.replay()
        torch.cuda.synchronize()
        ref = batch_tables_ref(c, np.ones(requests, np.int64), tb, free, h, bs, requests)
        check(tables, out, ref)
        tb, h, c = ref["tables"], ref["free_end"], c + 1
        run(make(50, 300, 60, 16, seed=13), cuda, 100, start=0)  # eager work in between
    assert int(head.item()) == h and np.array_equal(lens.cpu().numpy(), c)


def test_debug_checks(cuda, monkeypatch):
    monkeypatch.setattr(_decode, "DEBUG_CHECKS", True)
    case = make(5, 60, 20, 16, seed=14)
    total = int(case["n"].sum())
    check(*run(case, cuda, total, start=0))
    with pytest.raises(AssertionError):
        run(case, cuda, total - 1, start=0)
    with pytest.raises(AssertionError):
        run(case, cuda, total, start=len(case["free"]))
    case["c"][0] = 10_000
    with pytest.raises(AssertionError):
        run(case, cuda, total, start=0)
    assert _lib.load() is not None

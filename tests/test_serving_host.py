"""CPU tests of the serving operators: sizes and refusals of the C ABI (nothing is launched) and of
the Python entry points, through the extension and through ctypes."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import int8kv
from int8kv import _ext, _lib
from serving_cases import batch_tables_ref, lora_ref, sample_ref

P = 16  # a fake device pointer: every call below fails validation first


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libint8kv.so is not built")
    return _lib.load()


@pytest.fixture(params=["extension", "ctypes"])
def path(request):
    if request.param == "ctypes":
        with _ext.use_ctypes():
            yield
    else:
        if _ext.module() is None:
            pytest.skip("the torch extension is not built")
        yield


def test_batch_tables_refusals(lib):
    def call(**o):
        a = dict(c=P, n=P, dt=4, r=4, bt=P, w=8, bs_=8, block=16, free=P, nf=9, fs=P, nt=4, qs=P,
                 sl=P, pos=P, slot=P, tr=P, fe=P, ws=P, wsb=1 << 20, stream=None)
        a.update(o)
        return lib.int8kv_batch_tables(*a.values())

    for name in ("c", "n", "bt", "free", "qs", "sl", "pos", "slot", "tr", "fe"):
        assert call(**{name: None}) == -1, name
    assert call(dt=0) == -2 and call(dt=3) == -2
    for bad in (dict(r=-1), dict(r=2**31), dict(w=-1), dict(block=0), dict(block=65537),
                dict(nf=-1), dict(nt=-1), dict(nt=2**31)):
        assert call(**bad) == -3, bad
    assert call(bs_=7) == -4
    assert call(ws=None) == -5 and call(wsb=15) == -5 and call(ws=24) == -5
    assert lib.int8kv_batch_tables_workspace_bytes(100) == 16 + 800
    assert lib.int8kv_batch_tables_workspace_bytes(-1) == 0


def test_lora_refusals(lib):
    two = ctypes.c_int64 * 2

    def call(**o):
        a = dict(base=P, bs=64, x=P, t=4, k=32, xs=32, a=P, ast=two(8 * 32, 32), b=P,
                 bst=two(64 * 8, 8), na=3, rank=8, n=64, scales=P, plan=P, pb=1 << 20, out=P, os=64,
                 ws=P, wsb=1 << 20, stream=None)
        a.update(o)
        return lib.int8kv_lora_add(*a.values())

    for name in ("base", "x", "a", "b", "plan", "out", "ast", "bst"):
        assert call(**{name: None}) == -1, name
    for bad in (dict(t=-1), dict(t=2**24 + 1), dict(k=0), dict(k=12), dict(k=2**20 + 8), dict(na=0),
                dict(na=4097), dict(rank=0), dict(rank=12), dict(rank=136), dict(n=0), dict(n=20),
                dict(n=2**20 + 8)):
        assert call(**bad) == -3, bad
    for bad in (dict(base=24), dict(bs=60), dict(bs=56), dict(x=8), dict(xs=36), dict(xs=24),
                dict(a=40), dict(ast=two(100, 32)), dict(ast=two(256, 24)), dict(b=8),
                dict(bst=two(512, 4)), dict(bst=two(508, 8)), dict(out=24), dict(os=56)):
        assert call(**bad) == -4, bad
    assert call(pb=8) == -5 and call(plan=24) == -5
    assert call(ws=None) == -5 and call(wsb=8) == -5 and call(ws=24) == -5
    assert call(t=0) == 0  # nothing to do
    assert lib.int8kv_lora_plan(None, 4, 4, 3, P, 1 << 20, None) == -1
    assert lib.int8kv_lora_plan(P, 4, 4, 3, None, 1 << 20, None) == -1
    assert lib.int8kv_lora_plan(P, 2, 4, 3, P, 1 << 20, None) == -2
    assert lib.int8kv_lora_plan(P, 4, -1, 3, P, 1 << 20, None) == -3
    assert lib.int8kv_lora_plan(P, 4, 4, 4097, P, 1 << 20, None) == -3
    assert lib.int8kv_lora_plan(P, 4, 4, 3, P, 8, None) == -5
    assert lib.int8kv_lora_plan(P, 4, 4, 3, 24, 1 << 20, None) == -5
    for t, na in ((-1, 3), (2**24 + 1, 3), (4, 0), (4, 4097)):
        assert lib.int8kv_lora_plan_bytes(t, na) == 0
    assert lib.int8kv_lora_workspace_bytes(4, 3, 20, 8) == 0


def test_lora_outputs_over_its_inputs_are_refused(lib):
    """Rows of out that share memory with x, or with base otherwise than in place."""
    two = ctypes.c_int64 * 2
    far = P + (1 << 20)

    def call(base, bs, x, xs, out, os, tokens=4, n=64):
        return lib.int8kv_lora_add(base, bs, x, tokens, 32, xs, P, two(8 * 32, 32), P, two(64 * 8, 8), 3, 8,
                                   n, None, P, 1 << 20, out, os, P, 1 << 20, None)

    assert call(far, 64, P, 32, P, 64) == -4  # x itself
    assert call(far, 64, P, 64, P, 64) == -4
    assert call(P, 64, far, 32, P + 128, 64) == -4  # base's next row
    assert call(P, 64, far, 32, P, 128) == -4  # base in other rows
    assert call(P, 256, far, 32, P + 2 * 56, 256) == -4  # columns 56 .. 119 over 0 .. 63
    assert call(P, 256, far, 32, P - 2 * 56, 256) == -4
    assert call(P, 64, far, 32, P + 2 * 56, 64, tokens=1) == -4


def test_sample_refusals(lib):
    def call(**o):
        a = dict(logits=P, dt=2, rows=4, vocab=100, rs=100, u=P, t=None, k=None, p=None, m=None,
                 out=P, ws=P, wsb=1 << 30, stream=None)
        a.update(o)
        return lib.int8kv_sample_rows(*a.values())

    for name in ("logits", "u", "out"):
        assert call(**{name: None}) == -1, name
    assert call(dt=3) == -2 and call(dt=4) == -2
    for bad in (dict(rows=-1), dict(rows=2**16 + 1), dict(vocab=0), dict(vocab=2**21 + 1, rs=2**23)):
        assert call(**bad) == -3, bad
    assert call(rs=99) == -4 and call(logits=17) == -4 and call(dt=0, logits=18) == -4
    assert call(ws=None) == -5 and call(wsb=8) == -5 and call(ws=24) == -5
    assert call(rows=0) == 0
    assert lib.int8kv_sample_workspace_bytes(4, 0) == 0
    assert lib.int8kv_sample_workspace_bytes(-1, 100) == 0
    assert lib.int8kv_sample_workspace_bytes(4, 2**21 + 1) == 0


def test_python_entry_points_refuse(path):
    """AssertionError before anything is launched (CPU tensors are the last refusal)."""
    i32, bf = torch.int32, torch.bfloat16
    lens, tables, free = torch.ones(3, dtype=i32), torch.zeros(3, 4, dtype=i32), torch.arange(9).int()
    for args, kw in (
        ((lens, lens, tables, free, 3), {}),  # not on a GPU
        ((lens, lens[:2], tables, free, 3), {}),
        ((lens.float(), lens.float(), tables, free, 3), {}),
        ((lens, lens.long(), tables, free, 3), {}),
        ((lens, lens, tables.long(), free, 3), {}),
        ((lens, lens, tables[:2], free, 3), {}),
        ((lens, lens, tables[:, ::2], free, 3), {}),
        ((lens, lens, tables[:1].expand(3, 4), free, 3), {}),
        ((lens, lens, tables, free.long(), 3), {}),
        ((lens, lens, tables, free, -1), {}),
        ((lens, lens, tables, free, 3), {"block_size": 0}),
    ):
        with pytest.raises(AssertionError):
            # (buffers of a valid size, so that the arguments themselves are what is refused)
            int8kv.build_batch_tables(*args, out=int8kv.batch_tables_buffers(3, 3, "cpu"), **kw)
    x, a, b = torch.zeros(4, 32, dtype=bf), torch.zeros(2, 8, 32, dtype=bf), torch.zeros(2, 16, 8, dtype=bf)
    base = torch.zeros(4, 16, dtype=bf)
    plan = int8kv.LoraPlan(torch.zeros(1000, dtype=torch.uint8), 4, 2)
    for args in ((base, x, a, b, plan), (base.float(), x, a, b, plan), (base, x[:3], a, b, plan),
                 (base, x, a[:1], b, plan), (base, x, a, b[:, :8], plan), (base, x, a[:, :4], b, plan),
                 (base.t().contiguous().t(), x, a, b, plan),
                 (base, x, a, b, int8kv.LoraPlan(plan.buffer, 5, 2)),
                 (base, x, a, b, int8kv.LoraPlan(plan.buffer, 4, 3))):
        with pytest.raises(AssertionError):
            int8kv.lora_add(*args)
    with pytest.raises(AssertionError):
        int8kv.lora_plan(torch.zeros(4, dtype=i32), 2)
    with pytest.raises(AssertionError):
        int8kv.lora_plan(torch.zeros(4), 2)
    with pytest.raises(AssertionError):
        int8kv.lora_plan(torch.zeros(4, dtype=i32), 0)
    logits, u = torch.zeros(3, 50), torch.zeros(3)
    for args, kw in (((logits, u), {}), ((logits[0], u), {}), ((logits.double(), u), {}),
                     ((logits, u[:2]), {}), ((logits[:, ::2], u), {}), ((logits, u.double()), {}),
                     ((logits[:1].expand(3, 50), u), {}), ((logits, u), {"top_k": u}),
                     ((logits, u), {"top_p": u.half()})):
        with pytest.raises(AssertionError):
            int8kv.sample_tokens(*args, **kw)


def test_references_by_hand():
    """The references themselves against values worked out by hand."""
    r = batch_tables_ref([3, 0], [2, 5], [[7, -1], [-1, -1]], [9, 4, 6], 1, 4, 8)
    assert r["tables"].tolist() == [[7, 4], [6, -1]] and r["free_end"] == 4
    assert r["positions"].tolist() == [3, 4, 0, 1, 2, 3, 4, 0]
    assert r["slot_mapping"].tolist() == [31, 16, 24, 25, 26, 27, -1, -1]
    v = np.log([0.5, 0.25, 0.125, 0.125])
    assert [sample_ref(v, u)[0] for u in (0.0, 0.49, 0.51, 0.76, 0.99)] == [0, 0, 1, 2, 3]
    assert sample_ref(v, 0.99, top_k=3)[1].tolist() == [0, 1, 2]
    assert sample_ref(v, 0.99, top_p=0.8)[1].tolist() == [0, 1, 2]
    assert sample_ref(v, 0.99, top_k=2, top_p=0.6)[1].tolist() == [0]
    assert sample_ref(v, 0.99, min_p=0.4)[1].tolist() == [0, 1]
    out, _ = lora_ref([[1.0]], [[2.0, 3.0]], [[[4.0, 5.0]]], [[[6.0]]], [0], [0.5])
    assert out.tolist() == [[1 + 0.5 * 6 * 23]]

"""sample_tokens against a 64-bit reference by sorting: the tokens are equal."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import int8kv
from int8kv import _ext
from serving_cases import sample_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = math.inf


def run(cuda, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, **kw):
    rows = logits.shape[0]

    def column(v, dtype):
        if v is None:
            return None
        v = [v] * rows if isinstance(v, (int, float)) else v
        return torch.as_tensor(v).to(dtype).to(cuda)

    got = int8kv.sample_tokens(
        logits.to(cuda), column(u, torch.float32), temperature=column(temperature, torch.float32),
        top_k=column(top_k, torch.int32), top_p=column(top_p, torch.float32),
        min_p=column(min_p, torch.float32), **kw)
    return got.cpu().tolist()


def want(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows = logits.shape[0]
    v = logits.float().cpu().numpy()

    def column(x, off, dtype=np.float32):
        x = off if x is None else x
        return np.broadcast_to(np.asarray(x, dtype), (rows,))

    us, ts, ps = column(u, 0), column(temperature, 1), column(top_p, 1)
    ms, ks = column(min_p, 0), column(top_k, 0, np.int64)
    return [sample_ref(v[r], us[r], ts[r], ks[r], ps[r], ms[r])[0] for r in range(rows)]


def both(cuda, logits, u, **kw):
    got, ref = run(cuda, logits, u, **kw), want(logits, u, **kw)
    assert got == ref, [(r, g, w) for r, (g, w) in enumerate(zip(got, ref)) if g != w][:10]
    return got


def random_logits(rows, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype), torch.rand(rows, generator=g)


FILTERS = [
    {}, {"temperature": 0.7}, {"temperature": 1.9}, {"top_k": 1}, {"top_k": 40},
    {"top_p": 0.9}, {"top_p": 0.999}, {"min_p": 0.05},
    {"temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02},
    {"temperature": 1.3, "top_k": 300, "top_p": 0.5},
    {"temperature": 0.9, "top_p": 0.8, "min_p": 0.3}, {"temperature": 0.0, "top_p": 0.5},
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(4, 7), (3, 64), (5, 1000), (6, 4099), (7, 32000)])
def test_against_64_bits(cuda, rows, vocab, dtype):
    for i, kw in enumerate(FILTERS):
        logits, u = random_logits(rows, vocab, dtype, seed=vocab + i)
        both(cuda, logits, u, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(2, 152064), (40, 50257), (300, 2003), (1, 260001)])
def test_large_vocabularies(cuda, rows, vocab, dtype):
    for i, kw in enumerate((FILTERS[1], FILTERS[4], FILTERS[5], FILTERS[8])):
        logits, u = random_logits(rows, vocab, dtype, seed=rows + i)
        both(cuda, logits, u, **kw)


def test_every_row_its_own_settings(cuda):
    rows, g = 96, np.random.default_rng(1)
    for dtype in DTYPES:
        logits, u = random_logits(rows, 5003, dtype, seed=2)
        both(cuda, logits, u, temperature=g.choice([0.0, 0.3, 1.0, 2.5], rows),
             top_k=g.choice([0, -4, 1, 5, 700, 5003, 9000], rows),
             top_p=g.choice([1.0, 2.0, 0.0, -1.0, 0.3, 0.99], rows),
             min_p=g.choice([0.0, -1.0, 0.01, 0.5, 1.0, 3.0], rows))


def test_flat_rows_and_exact_borders(cuda):
    """Equal logits: the tokens are shares of [0, 1) whose borders are exact, ties cut by index."""
    for dtype in DTYPES:
        for vocab in (8, 64, 4096, 65536):
            logits = torch.full((5, vocab), 1.5, dtype=dtype)
            u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0**-24]
            assert run(cuda, logits, u) == [0, vocab // 4, vocab // 2, 3 * vocab // 4, vocab - 1]
            assert run(cuda, logits, u, top_p=0.5) == \
                [0, vocab // 8, vocab // 4, 3 * vocab // 8, vocab // 2 - 1]
            assert run(cuda, logits, u, top_k=4) == [0, 1, 2, 3, 3]
            assert run(cuda, logits, u, top_k=vocab // 2, top_p=0.5, min_p=1.0) == \
                [0, vocab // 16, vocab // 8, 3 * vocab // 16, vocab // 4 - 1]


def test_many_ties_at_the_cut(cuda):
    """A few distinct values over a large vocabulary: every cut falls into thousands of ties."""
    g = torch.Generator().manual_seed(3)
    for dtype in DTYPES:
        logits = torch.randint(0, 3, (30, 50000), generator=g).to(dtype)
        u = torch.rand(30, generator=g)
        for kw in ({"top_k": 20000}, {"top_p": 0.7}, {"top_k": 40000, "top_p": 0.6},
                   {"top_p": 0.31, "temperature": 0.5}, {"min_p": 0.3, "top_k": 9}):
            both(cuda, logits, u, **kw)


def test_hundreds_of_equal_logits(cuda):
    """Lists whose cut falls among hundreds to thousands of equal logits, put in order by index."""
    g = torch.Generator().manual_seed(17)
    for dtype in DTYPES:
        for vocab, steps in ((9000, 4.0), (30000, 16.0), (152064, 32.0), (152064, 64.0)):
            logits = torch.round(torch.randn(12, vocab, generator=g) * 2.0 * steps) / steps
            u = torch.rand(12, generator=g)
            for kw in ({"top_k": 700}, {"top_k": 3500}, {"top_p": 0.5}, {"top_p": 0.93},
                       {"top_k": 2900, "top_p": 0.8}, {"top_k": 1200, "top_p": 0.999, "min_p": 0.01},
                       {"top_k": 4000, "top_p": 0.4, "temperature": 3.0}):
                both(cuda, logits.to(dtype), u, **kw)


def test_dense_values_at_the_cut(cuda):
    """Many distinct values close together (fp32), far from zero and around it."""
    g = torch.Generator().manual_seed(4)
    for offset, spread in ((100.0, 1e-3), (0.0, 1e-4), (-7.0, 1e-2), (0.0, 1e-30)):
        logits = offset + torch.randn(8, 60000, generator=g) * spread
        u = torch.rand(8, generator=g)
        for kw in ({"top_k": 777}, {"top_p": 0.63}, {"top_k": 30000, "top_p": 0.9}):
            both(cuda, logits, u, **kw)


def test_as_many_as_top_k_stand_apart(cuda):
    """k tokens far above the others, k from a short order to a long one: the cut ends with them."""
    g = torch.Generator().manual_seed(15)
    for dtype in DTYPES:
        for vocab in (5003, 32000):
            for k in (200, 257, 700, 3001, 4096):
                logits = torch.randn(24, vocab, generator=g)
                for r in range(24):
                    at = torch.randperm(vocab, generator=g)[:k]
                    logits[r, at] = 9.0 + torch.rand(k, generator=g) * 4.0
                u = torch.rand(24, generator=g)
                for kw in ({"top_k": k}, {"top_k": k, "temperature": 6.0},
                           {"top_k": k, "temperature": 6.0, "min_p": 0.6}):
                    both(cuda, logits.to(dtype), u, **kw)


def test_cuts_of_every_size(cuda):
    """top-k from one token to the whole vocabulary, beside nuclei from nothing to everything: cuts
    from piece maxima, from bins, and past both lists; masked rows with fewer tokens than top-k."""
    g = torch.Generator().manual_seed(14)
    ks = [1, 2, 15, 16, 17, 60, 70, 127, 128, 129, 700, 4096, 4097, 9000, 30000, 32767, 32768, 50000]
    ps = [1.0, 0.02, 0.3, 0.7, 0.97, 0.9999, 1 - 2.0**-24]
    for dtype in DTYPES:
        for vocab, live in ((32768, 1.0), (32771, 0.2), (32771, 0.001)):
            logits = torch.randn(len(ks), vocab, generator=g) * 2.5
            logits[torch.rand(len(ks), vocab, generator=g) >= live] = -INF
            logits[:, 77] = 1.0
            logits = logits.to(dtype)
            for p in ps:
                u = torch.rand(len(ks), generator=g)
                both(cuda, logits, u, top_k=ks, top_p=p, temperature=0.9)
            both(cuda, logits, u, top_k=ks)  # (without top_p no histogram pass runs)


def test_long_top_k_beside_nuclei(cuda):
    """Rows with a long top-k in a batch where others have a nucleus cut alone, of any spread: their
    lists are gathered beside the others' histograms."""
    g = torch.Generator().manual_seed(16)
    ks = [257, 300, 590, 1000, 1700, 4096, 0, 0, 257, 1500]
    for vocab in (50257, 152064, 300007):
        for dtype in DTYPES:
            logits = torch.randn(len(ks), vocab, generator=g) * \
                torch.tensor([3.0, 1.0, 0.1, 3.0, 8.0, 3.0, 0.3, 3.0, 3.0, 3.0])[:, None]
            logits[8, torch.rand(vocab, generator=g) < 0.999] = -INF  # (fewer than k in all)
            logits[9, vocab // 8:] = -INF
            u = torch.rand(len(ks), generator=g)
            for kw in ({"top_p": 0.9}, {"top_p": 0.97, "min_p": 0.01, "temperature": 1.4}):
                both(cuda, logits.to(dtype), u, top_k=ks, **kw)


def test_live_tokens_in_few_places(cuda):
    """All live tokens in one corner of the row, more and fewer than the list holds."""
    g = torch.Generator().manual_seed(15)
    for lo, n in ((0, 300), (40000, 300), (49000, 1003), (20000, 5000), (0, 20000)):
        logits = torch.full((6, 50003), -INF)
        logits[:, lo:lo + n] = torch.randn(6, n, generator=g)
        u = torch.rand(6, generator=g)
        for kw in ({}, {"top_k": 80}, {"top_k": 80, "top_p": 0.9}, {"top_p": 0.9}, {"top_k": 2000},
                   {"min_p": 0.2}, {"top_k": 30000, "top_p": 0.5}):
            both(cuda, logits, u, **kw)


def test_log_probabilities(cuda):
    """Rows whose maximum is close to zero while the cut lies far below it, at every distance."""
    g = torch.Generator().manual_seed(17)
    for dtype in DTYPES:
        for spread, shift in ((3.0, 0.0), (40.0, 1e-3), (0.5, -1e-4)):
            logits = torch.log_softmax(torch.randn(24, 30011, generator=g) * spread, -1)
            logits = (logits - logits.amax(-1, keepdim=True) + shift).to(dtype)
            u = torch.rand(24, generator=g)
            t = spread / 3 if spread > 1 else 1.0
            for kw in ({"top_k": 100}, {"top_k": 1000}, {"top_p": 0.95}, {"top_p": 0.6, "min_p": 0.01},
                       {"min_p": 1e-3}, {}):
                both(cuda, logits, u, temperature=t, **kw)


def test_more_rows_than_share_a_workspace(cuda):
    logits, u = random_logits(2500, 5003, torch.bfloat16, seed=18)
    for kw in ({}, {"top_p": 0.9}, {"top_k": 30, "top_p": 0.9}):
        both(cuda, logits, u, **kw)
    ks = [0, 1, 50] * 833 + [7]
    both(cuda, logits, u, top_k=ks, top_p=0.8, temperature=0.7)


def test_vocabularies_of_more_pieces_than_tiles(cuda):
    for vocab in (262145, 400003, 2**21):
        logits, u = random_logits(2, vocab, torch.bfloat16, seed=vocab)
        for kw in ({}, {"top_k": 50}, {"top_p": 0.9}, {"top_k": 5000, "top_p": 0.9, "min_p": 0.01},
                   {"min_p": 0.1}, {"temperature": 0.0}):
            both(cuda, logits, u, **kw)


def test_far_and_near_chunks(cuda):
    """Chunks whose maxima lie far below the row's, and equal ones: the plain path's scaling."""
    g = torch.Generator().manual_seed(16)
    logits = torch.randn(64, 40000, generator=g)
    logits += torch.repeat_interleave(torch.tensor([-30.0, 0.0, -3.0, -80.0, -0.5]), 8000)
    both(cuda, logits, torch.rand(64, generator=g))
    both(cuda, logits, torch.rand(64, generator=g), temperature=5.0)
    both(cuda, logits, torch.rand(64, generator=g), temperature=0.1)
    low = torch.full((1, 40000), -1e4)
    low[0, 39999] = 3.0
    assert run(cuda, low.expand(2, -1).contiguous(), [0.0, 1 - 2.0**-24]) == [39999, 39999]


def test_masks(cuda):
    """Tokens at -inf, at the type's lowest value and at NaN: never drawn while another is left;
    one token left; none left."""
    for dtype in DTYPES:
        logits, u = random_logits(12, 3001, dtype, seed=5)
        low = torch.finfo(dtype).min
        g = torch.Generator().manual_seed(6)
        drop = torch.rand(12, 3001, generator=g) < 0.97
        for value in (-INF, low, math.nan):
            masked = logits.masked_fill(drop, value)
            for kw in FILTERS:
                got = both(cuda, masked, u, **kw)
                assert not drop[range(12), got].any()
        one = torch.full((3, 3001), -INF, dtype=dtype)
        one[:, 1234] = -5.0
        for kw in FILTERS:
            assert run(cuda, one, [0.0, 0.5, 0.999], **kw) == [1234] * 3
        for value in (-INF, math.nan):
            empty = torch.full((2, 3001), value, dtype=dtype)
            for kw in FILTERS:
                assert run(cuda, empty, [0.3, 0.9], **kw) == [0, 0]
        lowest = torch.full((2, 3001), low, dtype=dtype)
        assert run(cuda, lowest, [0.0, 0.5]) == [0, 1500]


def test_infinite_logits_and_signed_zeros(cuda):
    for dtype in DTYPES:
        logits, _ = random_logits(3, 500, dtype, seed=7)
        logits[:, 100], logits[:, 300] = INF, INF  # they share all the weight
        assert run(cuda, logits, [0.0, 0.4, 0.6]) == [100, 100, 300]
        assert run(cuda, logits, [0.9, 0.4, 0.6], top_k=1) == [100] * 3
        zeros = torch.zeros(2, 64, dtype=dtype)
        zeros[:, ::2] = -0.0
        assert run(cuda, zeros, [0.0, 0.5], top_k=4) == [0, 2]
        assert run(cuda, zeros, [0.3, 0.5], temperature=0.0) == [0, 0]


def test_odd_settings(cuda):
    logits, _ = random_logits(6, 900, torch.float32, seed=8)
    nan = math.nan
    first = logits.argmax(-1).tolist()
    assert run(cuda, logits, 0.4, temperature=nan) == first
    assert run(cuda, logits, 0.4, temperature=-1.0) == first
    assert run(cuda, logits, 0.999, temperature=1e-30) == first
    assert run(cuda, logits, [0.0, 0.25, 0.5, 0.6, 0.75, 0.999], temperature=INF) == \
        [0, 225, 450, 540, 675, 899]
    plain = run(cuda, logits, 0.4)
    assert run(cuda, logits, 0.4, top_p=nan) == plain and run(cuda, logits, 0.4, min_p=nan) == plain
    low, high = run(cuda, logits, 0.0), run(cuda, logits, 1 - 2.0**-24)
    assert run(cuda, logits, -3.0) == low and run(cuda, logits, nan) == low
    assert run(cuda, logits, 1.0) == high and run(cuda, logits, INF) == high


def test_small_vocabularies(cuda):
    for vocab in (1, 2, 3, 9):
        for dtype in DTYPES:
            logits, u = random_logits(20, vocab, dtype, seed=vocab)
            for kw in FILTERS:
                both(cuda, logits, u, **kw)


def test_rows_at_every_alignment(cuda):
    """Rows of an odd stride inside a wider buffer whose other columns hold larger values."""
    for dtype in DTYPES:
        logits, u = random_logits(16, 1013, dtype, seed=9)
        for lead in range(9):
            wide = torch.full((16, 1013 + 12), 1e4, dtype=dtype, device=cuda)
            wide[:, lead:lead + 1013] = logits.to(cuda)
            got = int8kv.sample_tokens(wide[:, lead:lead + 1013], u.to(cuda)).cpu().tolist()
            assert got == want(logits, u)


def test_distribution(cuda):
    """Evenly spread uniforms reproduce the weights: token i comes out floor-or-ceil of n p_i times."""
    logits = torch.randn(1, 50, generator=torch.Generator().manual_seed(10)) * 2
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    got = run(cuda, logits.expand(n, 50).contiguous(), u)
    counts = np.bincount(got, minlength=50)
    p = torch.softmax(logits[0].double(), -1).numpy() * n
    assert (np.abs(counts - p) <= 1.0).all()


def test_ctypes_path_stream_and_out(cuda):
    logits, u = random_logits(30, 20011, torch.bfloat16, seed=11)
    kw = {"temperature": 0.9, "top_k": 60, "top_p": 0.9}
    ref = both(cuda, logits, u, **kw)
    with _ext.use_ctypes():
        assert run(cuda, logits, u, **kw) == ref
    side = torch.cuda.Stream(cuda)
    with torch.cuda.stream(side):
        assert run(cuda, logits, u, **kw) == ref
    out = torch.empty(30, dtype=torch.int64, device=cuda)
    assert run(cuda, logits, u, out=out, **kw) == ref and out.cpu().tolist() == ref
    assert run(cuda, logits[:0], u[:0]) == []


def test_captured(cuda):
    """Two captured calls, replayed in turn with eager calls between, follow their inputs."""
    a, ua = (t.to(cuda) for t in random_logits(5, 30011, torch.bfloat16, seed=12))
    b, ub = (t.to(cuda) for t in random_logits(70, 9001, torch.float32, seed=13))
    p = torch.full((5,), 0.9, device=cuda)
    k = torch.full((70,), 30, dtype=torch.int32, device=cuda)
    oa = int8kv.sample_tokens(a, ua, top_p=p)
    ob = int8kv.sample_tokens(b, ub, top_k=k)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        int8kv.sample_tokens(a, ua, top_p=p, out=oa)
    with torch.cuda.graph(gb):
        int8kv.sample_tokens(b, ub, top_k=k, out=ob)
    for step in range(4):
        g = torch.Generator().manual_seed(20 + step)
        ua.copy_(torch.rand(5, generator=g))
        ub.copy_(torch.rand(70, generator=g))
        ga.replay()
        gb.replay()
        eager = int8kv.sample_tokens(b, ub, top_k=k)
        torch.cuda.synchronize()
        assert oa.cpu().tolist() == want(a, ua.cpu().numpy(), top_p=0.9)
        assert torch.equal(ob, eager) and ob.cpu().tolist() == want(b, ub.cpu().numpy(), top_k=30)

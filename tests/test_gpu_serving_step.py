"""The serving operators together in the decode loop: blocks taken on demand, per-sequence adapters
and sampled tokens, eagerly and in the captured step.

Each against something independent: on-demand blocks against the loop with blocks handed out in
advance (bit for bit), adapters against the loop with the adapter merged into its weights, sampled
tokens against the 64-bit reference on the step's own logits.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import metrics
from int8kv import decode_loop as DL
from serving_cases import sample_ref

pytestmark = pytest.mark.gpu

SHAPE = DL.QwenShape(hidden=512, layers=2, q_heads=28, kv_heads=4, head_dim=128, ffn=1024, vocab=2048)
B, S, NEW = 5, 29, 12


@pytest.fixture(scope="module")
def model(cuda):
    w = DL.random_weights(SHAPE, cuda, seed=0)
    g = torch.Generator().manual_seed(5)
    scales = DL.calibrate_static_scales(w, torch.randint(0, SHAPE.vocab, (2, 48), generator=g))
    return w, scales, torch.randint(0, SHAPE.vocab, (B, S), generator=g)


def make(model, mode="int8", weights=None, **kw):
    w, scales, _ = model
    return DL.DecodeLoop(weights or w, B, S, NEW, mode, scales=scales if mode == "int8" else None, **kw)


def settings(cuda, seed=3):
    g = torch.Generator().manual_seed(seed)
    return DL.Sampling(
        uniforms=torch.rand(NEW, B, generator=g).to(cuda),
        temperature=torch.tensor([0.8, 1.0, 0.0, 1.5, 0.7], device=cuda),
        top_k=torch.tensor([40, 0, 0, 500, 5], dtype=torch.int32, device=cuda),
        top_p=torch.tensor([0.95, 0.9, 1.0, 1.0, 0.8], device=cuda),
        min_p=torch.tensor([0.0, 0.0, 0.1, 0.02, 0.0], device=cuda))


def drawn(sampling, logits, step):
    rows = logits.float().cpu().numpy()
    get = {k: getattr(sampling, k).cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p")}
    u = sampling.uniforms[step].cpu().numpy()
    return [sample_ref(rows[r], u[r], **{k: v[r] for k, v in get.items()})[0] for r in range(B)]


@pytest.mark.parametrize("mode", DL.MODES)
def test_blocks_on_demand(model, mode):
    """Tokens and logits of the loop with its blocks handed out in advance; every block taken once,
    and only when a token needs it; eagerly and replayed."""
    plain, lazy = make(model, mode), make(model, mode, on_demand=True)
    plain.prefill(model[2])
    lazy.prefill(model[2])
    assert torch.equal(plain.prefill_logits, lazy.prefill_logits)
    saved = [loop.state() for loop in (plain, lazy)]
    for captured in (False, True):
        for loop, state in zip((plain, lazy), saved):
            loop.restore(state)
            if captured:
                loop.capture()
        for step in range(NEW - 1):
            for loop in (plain, lazy):
                loop.replay() if captured else loop.step_eager()
            torch.cuda.synchronize()
            assert torch.equal(plain.logits, lazy.logits) and torch.equal(plain.tokens, lazy.tokens)
            held = -(-(S + step + 1) // 16)
            table = lazy.block_tables.cpu()
            assert (table[:, held:] == -1).all() and int(lazy.free_head.item()) == B * held
            ids = table[:, :held].reshape(-1)
            assert (ids >= 0).all() and ids.unique().numel() == ids.numel()
        assert torch.equal(plain.generated, lazy.generated)


def test_sampled_tokens(cuda, model):
    sampling = settings(cuda)
    loop = make(model, sampling=sampling)
    loop.prefill(model[2])
    assert loop.generated[:, 0].tolist() == drawn(sampling, loop.prefill_logits, 0)
    state = loop.state()
    eager = []
    for step in range(1, NEW):
        loop.step_eager()
        torch.cuda.synchronize()
        eager.append(loop.tokens.tolist())
        assert eager[-1] == drawn(sampling, loop.logits, step)
        assert loop.generated[:, step].tolist() == eager[-1]
    loop.restore(state)
    loop.capture()
    for step in range(1, NEW):
        loop.replay()
        torch.cuda.synchronize()
        assert loop.tokens.tolist() == eager[step - 1]
        make(model, sampling=settings(cuda, 4)).prefill(model[2])  # eager work between the replays


def test_top_k_of_one_is_greedy(cuda, model):
    greedy = make(model)
    one = make(model, sampling=DL.Sampling(uniforms=torch.rand(NEW, B, device=cuda),
                                           top_k=torch.ones(B, dtype=torch.int32, device=cuda)))
    for loop in (greedy, one):
        loop.prefill(model[2])
        loop.decode()
    torch.cuda.synchronize()
    assert torch.equal(greedy.generated, one.generated)


def merged(w, adapters, i):
    """The model's weights with adapter i added (fp32 products, rounded to bf16)."""
    out = DL.ModelWeights(shape=w.shape, embed=w.embed, ln_f=w.ln_f, lm_head=w.lm_head)
    names = {"qkv": "wqkv", "o": "wo", "gate_up": "w_gate_up", "down": "w_down"}
    for lw, layer in zip(w.layers, adapters.layers):
        new = DL.LayerWeights(**vars(lw))
        for name, (a, b) in layer.items():
            weight = getattr(lw, names[name])
            delta = adapters.scales[i] * (b[i].float() @ a[i].float())
            setattr(new, names[name], (weight.float() + delta).to(torch.bfloat16))
        out.layers.append(new)
    return out


@pytest.mark.parametrize("projections", [DL.PROJECTIONS, ("qkv",), ("o", "gate_up"), ("down",)])
def test_adapters(cuda, model, projections):
    """Each sequence's logits are those of the model with its own adapter merged (both round the
    same products in other places: the tolerance of the step's test against an fp32 model), those
    without one are bit for bit the plain model's; the captured step follows new ids."""
    ids = torch.tensor([0, 2, -1, 1, 0], dtype=torch.int32, device=cuda)
    adapters = DL.random_adapters(SHAPE, ids, 3, 16, projections=projections, seed=1, std=0.05)
    loop, plain = make(model, adapters=adapters), make(model)
    refs = {i: make(model, weights=merged(model[0], adapters, i)) for i in range(3)}
    loops = [loop, plain, *refs.values()]

    def compare(attr):
        torch.cuda.synchronize()
        got = getattr(loop, attr).float().cpu().numpy()
        for r, i in enumerate(ids.tolist()):
            ref = getattr(refs[i] if i >= 0 else plain, attr).float().cpu().numpy()[r]
            _, cos, rel = metrics(got[r], ref)
            assert cos >= 0.999 and rel <= 0.05, (attr, r, i, cos, rel)

    for lp in loops:
        lp.prefill(model[2])
    compare("prefill_logits")
    for lp in loops:  # the same tokens from here on
        lp.tokens.copy_(plain.tokens)
    saved = [lp.state() for lp in loops]
    for lp in loops:
        lp.step_eager()
    compare("logits")
    eager = loop.logits.clone()
    loop.restore(saved[0])
    loop.capture()
    loop.replay()
    torch.cuda.synchronize()
    assert torch.equal(loop.logits, eager)
    # No adapter any more: the rows of the captured step follow (their caches were adapted, so only
    # the sequence that never had one is the plain model's).
    loop.restore(saved[0])
    ids.fill_(-1)
    loop.replay()
    torch.cuda.synchronize()
    _, cos, rel = metrics(loop.logits[2].float().cpu().numpy(), plain.logits[2].float().cpu().numpy())
    assert cos >= 0.999 and rel <= 0.05
    assert not torch.equal(loop.logits[0], eager[0])


def test_everything_together(cuda, model):
    """Blocks on demand, adapters and sampling in one captured step, against the same eagerly."""
    def build():
        ids = torch.tensor([1, -1, 0, 1, 3], dtype=torch.int64, device=cuda)
        return make(model, "bf16", on_demand=True, sampling=settings(cuda, 9),
                    adapters=DL.random_adapters(SHAPE, ids, 4, 24, seed=2, std=0.05))

    eager, graph = build(), build()
    for loop in (eager, graph):
        loop.prefill(model[2])
    graph.capture()
    for step in range(1, NEW):
        eager.step_eager()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager.logits, graph.logits)
        assert eager.tokens.tolist() == graph.tokens.tolist() == drawn(eager.sampling, eager.logits, step)
        assert torch.equal(eager.block_tables, graph.block_tables)
    assert torch.equal(eager.generated, graph.generated)

"""The operators of a serving step over many requests, with their cases: block tables and slot maps
built on the GPU from request lengths, low-rank adapters of many requests beside a shared
projection, and sampling from given random numbers.

``listed()`` names the cases and ``draw(rng)`` gives further ones of the same ranges; a case is a
dict of plain values.  ``prepare(case, seed)`` makes its inputs on the GPU from the seed alone,
``run(state)`` is one pass (the plain torch form, or the library's calls where ``own`` is true),
``work(case)`` the bytes and operations a pass cannot do without, and ``exact(case, seed)`` what a
pass returns from the definitions in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "int32": torch.int32, "int64": torch.int64}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int32": 4, "int64": 8}
LONGEST = 2**31 - 1  # lengths are read as clamp(length, 0, LONGEST)


def _library():
    package = str(Path(__file__).resolve().parent.parent / "int8-kvcache_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import int8kv

    return int8kv


# ------------------------------------------------------------------------------------- cases
def _tables(name, requests, longest, new, *, block=16, lens="int32", ragged=True, padding=0):
    """``new``: new tokens of a request, 1 (a decode step) or at most that many (prefill chunks)."""
    return {"name": name, "kind": "tables", "requests": requests, "longest": longest, "new": new,
            "block": block, "lens": lens, "ragged": ragged, "padding": padding}


def _adapter(name, tokens, k, n, rank, adapters, requests, *, none_every=0):
    """``requests`` contiguous runs of tokens, one adapter each; every ``none_every``-th has none."""
    return {"name": name, "kind": "adapter", "tokens": tokens, "k": k, "n": n, "rank": rank,
            "adapters": adapters, "requests": requests, "none_every": none_every}


def _sample(name, rows, vocab, filters, *, logits="bf16", spread=3.0, masked=0.0):
    """``filters``: temperature, top_k, top_p, all, or mixed (each row its own, some greedy).
    ``masked``: share of the tokens a grammar or a ban list leaves out (-inf)."""
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "filters": filters,
            "logits": logits, "spread": spread, "masked": masked}


def listed():
    return [
        # A decode step of the loop's batch: one token more per sequence at about 8k tokens; every
        # sixteenth sequence takes a new block.  Latency only.
        _tables("tables_decode_32", 32, 8320, 1),
        # A large decode batch padded to a captured graph's size, contexts anywhere up to 32k.
        _tables("tables_decode_1021", 1021, 32768, 1, lens="int64", padding=3),
        # Chunked prefill of 61 prompts behind what they have in the cache, vLLM's larger block.
        _tables("tables_prefill_61", 61, 32768, 16384, block=32, padding=1000),
        # One conversation's query projection: the smallest call, one adapter of a small pool.
        _adapter("adapter_1_qkv", 1, 3584, 4608, 16, 8, 1),
        # A layer of a decode step: 32 requests on 24 of the pool's adapters, their grouping
        # (which the other layers reuse) and the query, value, output and down projections.
        {"name": "adapter_layer_32", "kind": "adapter_layer", "tokens": 32, "rank": 16,
         "adapters": 24, "requests": 32, "none_every": 8, "hidden": 3584, "kv": 512, "ffn": 18944},
        # A mixed step, 13 prompt chunks among decodes (some without an adapter), down projection.
        _adapter("adapter_mixed_1100_down", 1100, 18944, 3584, 32, 16, 300, none_every=5),
        # A prefill of ragged prompts through the widest projection at a high rank.
        _adapter("adapter_prefill_6007_gate_up", 6007, 3584, 37888, 64, 5, 9),
        # One request on a small vocabulary, temperature only: launches and latency.
        _sample("sample_1x32000", 1, 32000, "temperature"),
        # The decode loop's batch with the filters a chat service sets.
        _sample("sample_32x152064_all", 32, 152064, "all"),
        # fp32 logits behind a grammar's mask, every request with its own settings.
        _sample("sample_61x152064_mixed_fp32", 61, 152064, "mixed", logits="fp32", masked=0.6),
        # An odd vocabulary (rows at odd addresses) under a nucleus cut that keeps thousands.
        _sample("sample_200x50257_top_p", 200, 50257, "top_p", logits="fp16"),
        # A large batch sampled from the whole distribution.
        _sample("sample_256x152064_temperature", 256, 152064, "temperature", logits="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["tables", "adapter", "adapter", "sample", "sample", "adapter_layer"])
    if kind == "tables":
        new = rng.choice([1, 1, _log_int(rng, 2, 16384)])
        requests = _log_int(rng, 1, 1500 if new == 1 else max(1, min(1000, 61 * 16384 // new)))
        case = _tables("", requests, _log_int(rng, max(16, new), 32768), new,
                       block=rng.choice([16, 16, 32, 64]), lens=rng.choice(["int32", "int64"]),
                       ragged=rng.random() < 0.8, padding=rng.choice([0, 0, rng.randrange(64)]))
    elif kind == "adapter":
        tokens = _log_int(rng, 1, 8192)
        k = rng.choice([512, 1024, 2048, 3584, 4096, 18944, 8 * rng.randrange(16, 600)])
        n = rng.choice([512, 3584, 4608, 4096, 18944, 37888, 8 * rng.randrange(16, 600)])
        # at most the largest listed case's traffic
        tokens = max(1, min(tokens, 6007 * (3584 + 2 * 37888) // (k + 2 * n)))
        case = _adapter("", tokens, k, n, rng.choice([8, 16, 16, 24, 32, 64, 128]),
                        _log_int(rng, 1, 48), rng.choice([tokens, max(1, min(tokens, 9))]),
                        none_every=rng.choice([0, 0, 3, 8]))
    elif kind == "adapter_layer":
        tokens = _log_int(rng, 1, 256)
        hidden = rng.choice([512, 1024, 3584, 4096])
        case = {"kind": kind, "tokens": tokens, "rank": rng.choice([8, 16, 32, 64]),
                "adapters": _log_int(rng, 1, 48), "requests": tokens,
                "none_every": rng.choice([0, 8]), "hidden": hidden, "kv": rng.choice([256, 512]),
                "ffn": rng.choice([1536, 4864, 18944])}
    else:
        vocab = rng.choice([32000, 50257, 128256, 152064, _log_int(rng, 200, 260000)])
        rows = _log_int(rng, 1, min(512, 256 * 152064 // vocab))
        case = _sample("", rows, vocab, rng.choice(["temperature", "top_k", "top_p", "all", "mixed"]),
                       logits=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                       spread=rng.choice([1.0, 2.0, 3.0, 3.0]),
                       masked=rng.choice([0.0, 0.0, rng.random()]))
    case.pop("name", None)
    return case


# ------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)


def _tables_tokens(case):
    """Rows of the token outputs: the most tokens the requests can bring, and the padding."""
    return case["requests"] * case["new"] + case["padding"]


def _prepare_tables(case, seed):
    g = _generator(seed)
    r, bs, longest, new = case["requests"], case["block"], case["longest"], case["new"]
    width = -(-longest // bs)
    if new == 1:
        n = torch.ones(r, dtype=torch.int64, device=DEV)
    elif case["ragged"]:
        n = torch.randint(1, new + 1, (r,), generator=g, device=DEV)
    else:
        n = torch.full((r,), new, dtype=torch.int64, device=DEV)
    most = (longest - n).clamp(min=0)
    if case["ragged"]:
        c = (torch.rand(r, generator=g, device=DEV) * (most + 1)).long().minimum(most)
    else:
        c = most
    # The pool's blocks in the order an allocator left them: those the requests hold, then the
    # free list, with room for what this step takes.
    have = (c + bs - 1) // bs
    pool = torch.randperm(r * width, generator=g, device=DEV).to(torch.int32).view(r, width)
    cols = torch.arange(width, device=DEV)
    tables = torch.where(cols < have[:, None], pool, torch.full_like(pool, -1))
    free = pool[cols >= have[:, None]] if r * width else pool.view(-1)
    free = torch.cat([torch.zeros(5, dtype=torch.int32, device=DEV), free]).contiguous()
    state = {"case": case, "computed": c.to(DTYPES[case["lens"]]), "new": n.to(DTYPES[case["lens"]]),
             "tables": tables.contiguous(), "free": free, "tokens": _tables_tokens(case),
             "free_start": torch.full((1,), 5, dtype=torch.int64, device=DEV)}
    if own:
        lib = _library()
        state["lib"] = lib
        state["out"] = lib.batch_tables_buffers(r, state["tokens"], DEV)
    return state


def _adapter_ids(case, g):
    """Adapter of every token: the requests are runs of tokens and take the pool's adapters in turn
    (a shuffled order), every ``none_every``-th request none (-1)."""
    requests, tokens, pool = case["requests"], case["tokens"], case["adapters"]
    order = torch.randperm(pool, generator=g, device=DEV)
    req = torch.arange(requests, device=DEV)
    of_request = order[req % pool]
    if case["none_every"]:
        of_request = torch.where(req % case["none_every"] == case["none_every"] - 1,
                                 torch.full_like(of_request, -1), of_request)
    if requests >= tokens:
        return of_request[:tokens].to(torch.int32).contiguous()
    cuts = torch.randperm(tokens - 1, generator=g, device=DEV)[:requests - 1].sort().values + 1
    request = torch.searchsorted(cuts, torch.arange(tokens, device=DEV), right=True)
    return of_request[request].to(torch.int32).contiguous()


def _normal(g, *size, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*size, generator=g, device=DEV) * std).to(dtype)


def _adapter_weights(case, k, n, g):
    a = _normal(g, case["adapters"], case["rank"], k, std=k**-0.5)
    b = _normal(g, case["adapters"], n, case["rank"], std=0.05)
    return a, b


def _prepare_adapter(case, seed):
    g = _generator(seed)
    t, k, n = case["tokens"], case["k"], case["n"]
    ids = _adapter_ids(case, g)
    a, b = _adapter_weights(case, k, n, g)
    state = {"case": case, "ids": ids, "x": _normal(g, t, k), "base": _normal(g, t, n), "a": a,
             "b": b, "scales": torch.rand(case["adapters"], generator=g, device=DEV) * 2 + 0.25}
    if own:
        lib = _library()
        state["lib"] = lib
        # A step's grouping of its tokens by adapter, made once for all its projections.
        state["plan"] = lib.lora_plan(ids, case["adapters"])
        state["out"] = torch.empty_like(state["base"])
    return state


def _layer_projections(case):
    """(K, N, columns of the projection's output that the adapter adds to, width of that output)."""
    h, kv, ffn = case["hidden"], case["kv"], case["ffn"]
    qkv = h + 2 * kv
    return [(h, h, slice(0, h), qkv), (h, kv, slice(h + kv, qkv), qkv), (h, h, slice(0, h), h),
            (ffn, h, slice(0, h), h)]


def _prepare_layer(case, seed):
    g = _generator(seed)
    t = case["tokens"]
    state = {"case": case, "ids": _adapter_ids(case, g), "parts": [],
             "scales": torch.rand(case["adapters"], generator=g, device=DEV) * 2 + 0.25}
    for k, n, columns, width in _layer_projections(case):
        a, b = _adapter_weights(case, k, n, g)
        base = _normal(g, t, width)
        part = {"x": _normal(g, t, k), "base": base[:, columns], "a": a, "b": b}
        if own:
            part["out"] = torch.empty_like(base)[:, columns]
        state["parts"].append(part)
    if own:
        state["lib"] = _library()
    return state


def _prepare_sample(case, seed):
    g = _generator(seed)
    rows, vocab, kind = case["rows"], case["vocab"], case["filters"]
    logits = torch.randn(rows, vocab, generator=g, device=DEV).mul_(case["spread"])
    if case["masked"]:
        drop = torch.rand(rows, vocab, generator=g, device=DEV) < case["masked"]
        drop[:, vocab // 2] = False
        logits.masked_fill_(drop, -math.inf)

    def pick(values, dtype):
        t = torch.tensor(values, dtype=dtype, device=DEV)
        return t[torch.randint(0, len(values), (rows,), generator=g, device=DEV)].contiguous()

    mixed = kind == "mixed"
    state = {"case": case, "logits": logits.to(DTYPES[case["logits"]]),
             "u": torch.rand(rows, generator=g, device=DEV),
             "temperature": pick([0.0, 0.6, 0.8, 1.0, 1.3] if mixed else [0.7, 0.8, 1.0], torch.float32),
             "top_k": None, "top_p": None, "min_p": None}
    if mixed or kind in ("top_k", "all"):
        state["top_k"] = pick([0, 1, 20, 50, 1000] if mixed else [20, 40, 50, 100], torch.int32)
    if mixed or kind in ("top_p", "all"):
        state["top_p"] = pick([1.0, 0.95, 0.9, 0.5] if mixed else [0.95, 0.9, 0.8], torch.float32)
    if mixed or kind == "all":
        state["min_p"] = pick([0.0, 0.0, 0.05, 0.1] if mixed else [0.0, 0.02, 0.05], torch.float32)
    if own:
        state["lib"] = _library()
        state["out"] = torch.empty(rows, dtype=torch.int64, device=DEV)
    return state


PREPARE = {"tables": _prepare_tables, "adapter": _prepare_adapter, "adapter_layer": _prepare_layer,
           "sample": _prepare_sample}


def prepare(case, seed):
    return PREPARE[case["kind"]](case, seed)


# ------------------------------------------------------------------------------- plain forms
def _plain_tables(computed, new, tables, free, free_start, bs, tokens):
    r, width = tables.shape
    c = computed.long().clamp(0, LONGEST)
    n = new.long().clamp(0, LONGEST)
    ends = torch.cumsum(n, 0)
    starts = ends - n
    have = ((c + bs - 1) // bs).clamp(max=width)
    need = ((c + n + bs - 1) // bs).clamp(max=width)
    taken = torch.cumsum(need - have, 0)
    cols = torch.arange(width, device=tables.device)
    at = free_start + (taken - (need - have))[:, None] + cols - have[:, None]
    fresh = torch.where((at >= 0) & (at < free.numel()),
                        free[at.clamp(0, free.numel() - 1)], torch.full_like(tables, -1))
    tables = torch.where((cols >= have[:, None]) & (cols < need[:, None]), fresh, tables)
    t = torch.arange(tokens, device=tables.device)
    request = torch.searchsorted(ends, t, right=True)
    held = request < r
    q = request.clamp(max=r - 1)
    position = torch.where(held, c[q] + t - starts[q], torch.zeros_like(t))
    block = position // bs
    ids = tables[q, block.clamp(max=width - 1)].long()
    slot = torch.where(held & (block < width) & (ids >= 0), ids * bs + position % bs,
                       torch.full_like(t, -1))
    query_starts = torch.cat([torch.zeros_like(ends[:1]), ends]).clamp(max=tokens).int()
    return (tables, query_starts, (c + n).clamp(max=LONGEST).int(), position, slot,
            torch.where(held, request, torch.full_like(request, -1)).int(), free_start + taken[-1:])


def _plain_adapter(x, base, a, b, ids, scales):
    """All adapters at once: x times every A, the columns of other adapters cleared, times every B."""
    pool, rank, k = a.shape
    n = b.shape[1]
    hidden = x.float() @ a.float().reshape(pool * rank, k).t()
    of_column = torch.arange(pool * rank, device=x.device) // rank
    keep = (of_column[None, :] == ids[:, None]) * scales.repeat_interleave(rank)[None, :]
    delta = (hidden * keep) @ b.float().permute(0, 2, 1).reshape(pool * rank, n)
    return (base.float() + delta).to(base.dtype)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    rows, vocab = logits.shape
    dev = logits.device
    x = logits.float()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    t = torch.ones(rows, device=dev) if temperature is None else temperature
    # 64 bits: a sum over the vocabulary decides between neighbouring tokens.
    z = torch.where(x == top, torch.zeros_like(x, dtype=torch.float64),
                    (x.double() - top.double()) / t.double()[:, None])
    w = torch.where(x == -math.inf, torch.zeros_like(z), torch.exp(z))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=dev)[None, :]
    keep = torch.ones(rows, vocab, dtype=torch.bool, device=dev)
    if top_k is not None:
        k = torch.where((top_k <= 0) | (top_k > vocab), torch.full_like(top_k, vocab), top_k)
        keep &= rank < k[:, None]
    if top_p is not None:
        before = torch.cumsum(ws, -1) - ws
        total = (ws * keep).sum(-1, keepdim=True)
        p = top_p.double()[:, None]
        keep &= (before < p * total) | ~(p < 1) | (rank == 0)
    if min_p is not None:
        m = min_p.double()[:, None]
        keep &= (ws >= m) | ~(m > 0) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    total = torch.cumsum(w * kept, -1)
    target = u.double()[:, None] * total[:, -1:]
    token = (total <= target).sum(-1).clamp(max=vocab - 1)
    first = (x == top).to(torch.uint8).argmax(-1)  # the first of the largest: greedy rows
    greedy = ~(t > 0) | (top[:, 0] == -math.inf)
    return torch.where(greedy, first, token)


# ------------------------------------------------------------------------------------- a pass
def _run_tables(s):
    bs = s["case"]["block"]
    if own:
        o = s["lib"].build_batch_tables(s["computed"], s["new"], s["tables"], s["free"], s["tokens"],
                                        block_size=bs, free_start=s["free_start"], out=s["out"])
        return [s["tables"], o.query_starts, o.seq_lens, o.positions, o.slot_mapping,
                o.token_requests, o.free_end]
    return list(_plain_tables(s["computed"], s["new"], s["tables"], s["free"], s["free_start"], bs,
                              s["tokens"]))


def _run_adapter(s):
    if own:
        return s["lib"].lora_add(s["base"], s["x"], s["a"], s["b"], s["plan"], scales=s["scales"],
                                 out=s["out"])
    return _plain_adapter(s["x"], s["base"], s["a"], s["b"], s["ids"], s["scales"])


def _run_layer(s):
    if own:
        plan = s["lib"].lora_plan(s["ids"], s["case"]["adapters"])
        return [s["lib"].lora_add(p["base"], p["x"], p["a"], p["b"], plan, scales=s["scales"],
                                  out=p["out"]) for p in s["parts"]]
    return [_plain_adapter(p["x"], p["base"], p["a"], p["b"], s["ids"], s["scales"])
            for p in s["parts"]]


def _run_sample(s):
    if own:
        return s["lib"].sample_tokens(s["logits"], s["u"], temperature=s["temperature"],
                                      top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                      out=s["out"])
    return _plain_sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


RUN = {"tables": _run_tables, "adapter": _run_adapter, "adapter_layer": _run_layer,
       "sample": _run_sample}


def run(state):
    return RUN[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------- work
def _adapter_work(case, k, n):
    t, rank = case["tokens"], case["rank"]
    requests = min(case["requests"], t)
    with_one = requests - (requests // case["none_every"] if case["none_every"] else 0)
    used = min(case["adapters"], with_one)
    share = with_one / max(1, requests)
    return (2 * t * (share * k + 2 * n) + 2 * used * rank * (k + n) + 4 * t,
            2 * t * share * rank * (k + n))


def work(case):
    if case["kind"] == "tables":
        r, bs, new = case["requests"], case["block"], case["new"]
        held = r * ((new + 1) / 2 if case["ragged"] and new > 1 else new)
        taken = held / bs
        read = 2 * r * BYTES[case["lens"]] + 4 * taken + 4 * r
        written = 20 * _tables_tokens(case) + 4 * taken + 8 * r
        return {"bytes": int(read + written), "flops": 0}
    if case["kind"] == "adapter":
        b, f = _adapter_work(case, case["k"], case["n"])
        return {"bytes": int(b), "flops": int(f)}
    if case["kind"] == "adapter_layer":
        parts = [_adapter_work(case, k, n) for k, n, _, _ in _layer_projections(case)]
        return {"bytes": int(sum(p[0] for p in parts)), "flops": int(sum(p[1] for p in parts))}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * (vocab * BYTES[case["logits"]] + 32), "flops": 4 * rows * vocab}


# ----------------------------------------------------------------------------------- 64 bits
def _exact_tables(s):
    bs, tokens = s["case"]["block"], s["tokens"]
    c, n = s["computed"].cpu().numpy().astype(np.int64), s["new"].cpu().numpy().astype(np.int64)
    tables, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy()
    head = int(s["free_start"].item())
    r, width = tables.shape
    starts = np.zeros(r + 1, np.int64)
    position, slot = np.zeros(tokens, np.int64), np.full(tokens, -1, np.int64)
    request = np.full(tokens, -1, np.int64)
    for q in range(r):
        have, need = min(width, -(-c[q] // bs)), min(width, -(-(c[q] + n[q]) // bs))
        for j in range(have, need):
            tables[q, j] = free[head] if 0 <= head < len(free) else -1
            head += 1
        starts[q + 1] = starts[q] + n[q]
        here = slice(starts[q], starts[q + 1])
        p = c[q] + np.arange(n[q])
        ids = tables[q, np.minimum(p // bs, width - 1)].astype(np.int64)
        position[here], request[here] = p, q
        slot[here] = np.where((p // bs < width) & (ids >= 0), ids * bs + p % bs, -1)
    return [tables, starts.astype(np.int32), (c + n).astype(np.int32), position, slot,
            request.astype(np.int32), np.array([head], np.int64)]


def _exact_adapter(x, base, a, b, ids, scales):
    out = base.double()
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().view(-1)
        if rows.numel():
            hidden = x[rows].double() @ a[i].double().t().contiguous()
            out[rows] += scales[i].double() * (hidden @ b[i].double().t().contiguous())
    return out.cpu()


def _exact_sample_row(v, u, t, k, p, m):
    v = np.where(np.isnan(v), -np.inf, v.astype(np.float64))
    top = v.max()
    if not t > 0 or top == -np.inf:
        return int(np.argmax(v))
    w = np.zeros_like(v)
    live = v > -np.inf
    w[live] = 1.0
    below = live & (v < top)
    w[below] = np.exp((v[below] - top) / np.float64(t))
    order = np.argsort(-v, kind="stable")
    ws = w[order]
    kept = len(v) if k <= 0 else min(int(k), len(v))
    sums = np.concatenate([[0.0], np.cumsum(ws)])
    limit = kept
    if p < 1:
        limit = min(limit, max(1, int((sums[:kept] < np.float64(p) * sums[kept]).sum())))
    if m > 0:
        limit = min(limit, max(1, int((ws >= np.float64(m)).sum())))
    index = np.sort(order[:limit])
    mass = np.cumsum(w[index])
    return int(index[min(np.searchsorted(mass, np.float64(u) * mass[-1], side="right"), limit - 1)])


def _exact_sample(s):
    rows, vocab = s["logits"].shape
    v = s["logits"].float().cpu().numpy()

    def column(name, off):
        return [off] * rows if s[name] is None else s[name].cpu().numpy()

    t, k = column("temperature", 1.0), column("top_k", 0)
    p, m = column("top_p", 1.0), column("min_p", 0.0)
    u = s["u"].cpu().numpy()
    return np.array([_exact_sample_row(v[i], u[i], t[i], k[i], p[i], m[i]) for i in range(rows)],
                    np.int64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(s)
    if case["kind"] == "adapter":
        return _exact_adapter(s["x"], s["base"], s["a"], s["b"], s["ids"], s["scales"])
    if case["kind"] == "adapter_layer":
        return [_exact_adapter(p["x"], p["base"], p["a"], p["b"], s["ids"], s["scales"])
                for p in s["parts"]]
    return _exact_sample(s)

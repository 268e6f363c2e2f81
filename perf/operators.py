"""Timed cases of the shared-row (embedding) and budget (eviction) operators.

Four operators:

- ``lookup``      out[n] = scale * table[index[n]]
- ``gradient``    grad_table[v] = scale * sum of grad_out[n] over the n with index[n] = v
- ``accumulate``  out[g, j] = decay * score[g, j] + sum over r of weights[g, r, j]
- ``evict``       keep the `first` first, the `recent` last and the highest-scored entries of every group up to a
                  budget, in order, and gather the kept rows of every field

``own = False`` computes them in elementary torch operations in 32 bits, ``own = True`` through gsx_b200.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
INDEX = {"i32": torch.int32, "i64": torch.int64}
SCENE_FIELDS = (3, 3, 4, 1, 3)  # mean3d, logscale, rotation, opacity, sh0


def listed():
    return [
        # one new token's row of a 64k x 4096 table, scaled by sqrt(4096): the latency of a call
        dict(name="lookup_token", op="lookup", count=1, rows=65536, dim=4096, table="bf16", out="bf16", index="i64",
             scale=64.0, skew=1.0),
        # the base colours of a 3M-Gaussian scene from a codebook of 4096 colours
        dict(name="lookup_colour", op="lookup", count=3_000_000, rows=4096, dim=3, table="f32", out="f32", index="i32",
             scale=1.0, skew=1.5),
        # the 45 view-dependent coefficients of 1M Gaussians from 16-bit codebook rows (90 bytes: no row is aligned)
        dict(name="lookup_sh", op="lookup", count=1_000_000, rows=16384, dim=45, table="bf16", out="f32", index="i32",
             scale=0.5, skew=1.5),
        # the gradient of the colour codebook: 3M rows of 12 bytes into 4096
        dict(name="gradient_colour", op="gradient", count=3_000_000, rows=4096, dim=3, table="f32", out="f32",
             index="i32", scale=1.0, skew=1.5),
        # the gradient of the coefficient codebook, with rows that many Gaussians share (the first has 4% of them)
        dict(name="gradient_sh", op="gradient", count=1_000_000, rows=16384, dim=45, table="f32", out="f32",
             index="i32", scale=0.5, skew=3.0),
        # the gradient of a token table after a batch of 8191 tokens: few rows are touched, all are written
        dict(name="gradient_tokens", op="gradient", count=8191, rows=65536, dim=2048, table="bf16", out="bf16",
             index="i64", scale=45.25, skew=3.0),
        # one decoding step: 32 caches, 4 query heads on each, a ragged batch
        dict(name="accumulate_step", op="accumulate", groups=32, rows=4, length=4097, weights="bf16", decay=1.0,
             ragged=True),
        # a prompt: 8 caches, 4 heads x 512 queries, causal
        dict(name="accumulate_prompt", op="accumulate", groups=8, rows=2048, length=8192, weights="bf16", decay=0.5,
             ragged=False),
        # the blend weights of 8 views onto the 3M Gaussians of a scene
        dict(name="accumulate_views", op="accumulate", groups=1, rows=8, length=3_000_000, weights="f32", decay=0.875,
             ragged=False),
        # a small cache one token over its budget: the latency of a call
        dict(name="evict_step", op="evict", groups=8, length=1025, budget=1024, first=4, recent=64, dim=64,
             table="f16", scene=False, ragged=False),
        # long prompts cut to 4096 entries a head
        dict(name="evict_long", op="evict", groups=32, length=32768, budget=4096, first=4, recent=512, dim=128,
             table="bf16", scene=False, ragged=True),
        # a 3M-Gaussian scene cut to 2M, the last 100k (just grown) protected
        dict(name="evict_scene", op="evict", groups=1, length=3_000_000, budget=2_000_000, first=0, recent=100_000,
             dim=0, table="f32", scene=True, ragged=False),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _drawn(rng):
    op = rng.choice(["lookup", "gradient", "accumulate", "evict"])
    kinds = ["f32", "f16", "bf16"]
    if op in ("lookup", "gradient"):
        if rng.random() < 0.5:  # many short rows: a scene's codebook
            count, rows, dim = _log(rng, 1000, 4_000_000), _log(rng, 16, 65536), rng.choice([1, 3, 4, 9, 15, 24, 45, 48])
        else:  # few long rows: a token table
            count, rows, dim = _log(rng, 1, 16384), _log(rng, 1000, 131072), _log(rng, 64, 8192)
        table = rng.choice(kinds)
        return dict(op=op, count=count, rows=rows, dim=dim, table=table, out=rng.choice([table, "f32"]),
                    index=rng.choice(["i32", "i64"]), scale=round(rng.uniform(0.1, 64.0), 3),
                    skew=rng.choice([1.0, 1.5, 3.0]))
    if op == "accumulate":
        if rng.random() < 0.3:
            groups, rows, length = 1, rng.randint(1, 16), _log(rng, 10000, 4_000_000)
        else:
            groups, rows, length = _log(rng, 1, 128), _log(rng, 1, 4096), _log(rng, 1, 65536)
        return dict(op=op, groups=groups, rows=rows, length=length, weights=rng.choice(kinds),
                    decay=rng.choice([0.0, 0.5, 0.9, 1.0]), ragged=rng.random() < 0.5)
    scene = rng.random() < 0.3
    length = _log(rng, 10000, 3_000_000) if scene else _log(rng, 2, 131072)
    budget = rng.randint(1, length)
    first = min(rng.choice([0, 1, 4, 64]), budget)
    return dict(op=op, groups=1 if scene else _log(rng, 1, 128), length=length, budget=budget, first=first,
                recent=rng.randint(0, (budget - first) // 2), dim=0 if scene else rng.choice([1, 40, 64, 80, 128, 256]),
                table="f32" if scene else rng.choice(kinds), scene=scene, ragged=not scene and rng.random() < 0.5)


def draw(rng):
    while True:
        case = _drawn(rng)
        if work(case)["bytes"] <= 300e6:
            return case


def _index(case, g):
    """Row numbers, the low ones more often than the high ones (u^skew)."""
    u = torch.rand(case["count"], generator=g, device=DEVICE, dtype=torch.float64)
    return (u.pow(case["skew"]) * case["rows"]).long().clamp_(max=case["rows"] - 1).to(INDEX[case["index"]])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEVICE)  # noqa: E731
    op = case["op"]
    s = dict(case)
    if op == "lookup":
        s["t"] = (randn(case["rows"], case["dim"]) * 0.02).to(TYPES[case["table"]])
        s["i"] = _index(case, g)
        s["o"] = torch.empty(case["count"], case["dim"], dtype=TYPES[case["out"]], device=DEVICE)
    elif op == "gradient":
        s["i"] = _index(case, g)
        s["g"] = (randn(case["count"], case["dim"]) * 1e-3).to(TYPES[case["out"]])
        s["o"] = torch.empty(case["rows"], case["dim"], dtype=TYPES[case["table"]], device=DEVICE)
    elif op == "accumulate":
        G, R, L = case["groups"], case["rows"], case["length"]
        if G == 1:  # a scene: each view sees some of the Gaussians
            w = torch.rand(G, R, L, generator=g, device=DEVICE)
            s["w"] = torch.where(w < 0.4, torch.zeros((), device=DEVICE), w.pow(4) * 20.0).to(TYPES[case["weights"]])
        else:  # causal attention weights of the last queries
            w = randn(G, R, L)
            if R >= 64:
                seen = L - 1 - (R - 1 - torch.arange(R, device=DEVICE)) % 512
                w.masked_fill_(torch.arange(L, device=DEVICE)[None, None, :] > seen.clamp(min=0)[None, :, None],
                               float("-inf"))
            s["w"] = torch.softmax(w, dim=-1).to(TYPES[case["weights"]])
        s["s"] = torch.rand(G, L, generator=g, device=DEVICE)
        s["n"] = _lengths(case, g)
        s["o"] = torch.empty(G, L, device=DEVICE)
    else:
        G, L = case["groups"], case["length"]
        # accumulated weights: a few entries hold most of it; some never got any
        s["s"] = torch.where(torch.rand(G, L, generator=g, device=DEVICE) < 0.05, torch.zeros((), device=DEVICE),
                             torch.exp(2.0 * randn(G, L)))
        s["n"] = _lengths(case, g)
        dims = SCENE_FIELDS if case["scene"] else (case["dim"], case["dim"])
        s["f"] = [s["s"].unsqueeze(-1)] + [randn(G, L, d).to(TYPES[case["table"]]) for d in dims]
        s["d"] = [torch.zeros(G, case["budget"], f.shape[-1], dtype=f.dtype, device=DEVICE) for f in s["f"]]
        s["k"] = torch.zeros(G, case["budget"], dtype=torch.int32, device=DEVICE)
        s["c"] = torch.zeros(G, dtype=torch.int32, device=DEVICE)
    return s


def _lengths(case, g):
    """Entries in use of every group: between a half and all, or None where all groups are full."""
    if not case["ragged"]:
        return None
    L = case["length"]
    return torch.randint(L // 2, L + 1, (case["groups"],), generator=g, device=DEVICE, dtype=torch.int32)


def run(state):
    s, op = state, state["op"]
    if own:
        import gsx_b200 as gb
        if op == "lookup":
            return gb.embedding_lookup(s["t"], s["i"], out=s["o"], scale=s["scale"])
        if op == "gradient":
            return gb.embedding_backward(s["g"], s["i"], s["o"], scale=s["scale"])
        if op == "accumulate":
            return gb.budget_accumulate(s["s"], s["w"], out=s["o"], decay=s["decay"], lengths=s["n"])
        keep, kept = gb.budget_select(s["s"], s["budget"], lengths=s["n"], first=s["first"], recent=s["recent"],
                                      keep=s["k"], kept=s["c"])
        gb.budget_gather(list(zip(s["f"], s["d"])), keep, kept)
        return [keep, kept] + s["d"]
    if op == "lookup":
        return (s["t"][s["i"].long()].float() * s["scale"]).to(s["o"].dtype)
    if op == "gradient":
        total = torch.zeros(s["rows"], s["dim"], dtype=torch.float32, device=DEVICE)
        total.index_add_(0, s["i"].long(), s["g"].float())
        return (total * s["scale"]).to(s["o"].dtype)
    if op == "accumulate":
        total = s["s"] * s["decay"] + s["w"].float().sum(1)
        if s["n"] is None:
            return total
        return torch.where(torch.arange(s["length"], device=DEVICE) < s["n"][:, None], total, s["s"])
    return _evict(s)


def _evict(s):
    G, L, budget = s["groups"], s["length"], s["budget"]
    j = torch.arange(L, device=DEVICE)
    n = s["n"].long()[:, None] if s["n"] is not None else torch.full((G, 1), L, device=DEVICE)
    rank = torch.where((j < s["first"]) | (j >= n - s["recent"]), torch.inf, s["s"])
    rank = torch.where(j < n, rank, -torch.inf)
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget]
    kept = n.clamp(max=budget)
    inside = torch.arange(budget, device=DEVICE) < kept
    keep = torch.sort(torch.where(inside, order, L), dim=1).values
    keep = torch.where(inside, keep, 0)
    rows = [torch.where(inside[..., None], torch.gather(f, 1, keep[..., None].expand(-1, -1, f.shape[-1])),
                        torch.zeros((), dtype=f.dtype, device=DEVICE)) for f in s["f"]]
    return [keep.int(), kept[:, 0].int()] + rows


def work(case):
    c = case
    if c["op"] in ("lookup", "gradient"):
        full = c["rows"] if c["op"] == "gradient" else min(c["rows"], c["count"])
        ends = c["count"] * c["dim"] * BYTES[c["out"]] + full * c["dim"] * BYTES[c["table"]]
        return {"bytes": ends + c["count"] * (4 if c["index"] == "i32" else 8), "flops": c["count"] * c["dim"]}
    if c["op"] == "accumulate":
        n = c["groups"] * c["length"] * (0.75 if c["ragged"] else 1.0)
        return {"bytes": n * (c["rows"] * BYTES[c["weights"]] + 8), "flops": n * c["rows"]}
    n = c["groups"] * c["length"] * (0.75 if c["ragged"] else 1.0)
    width = 4 + (4 * sum(SCENE_FIELDS) if c["scene"] else 2 * c["dim"] * BYTES[c["table"]])
    kept = min(n, c["groups"] * c["budget"])
    return {"bytes": n * 4 + kept * (4 + 2 * width), "flops": n}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    host = lambda t: t.double().cpu().numpy()  # noqa: E731
    if op == "lookup":
        return np.take(host(s["t"]), s["i"].cpu().numpy(), axis=0) * float(np.float32(case["scale"]))
    if op == "gradient":
        index, grad = s["i"].cpu().numpy().astype(np.int64), host(s["g"])
        order = np.argsort(index, kind="stable")
        at = np.flatnonzero(np.diff(index[order], prepend=-1))
        out = np.zeros((case["rows"], case["dim"]))
        out[index[order][at]] = np.add.reduceat(grad[order], at, axis=0) * float(np.float32(case["scale"]))
        return out
    if op == "accumulate":
        score, w = host(s["s"]), s["w"].cpu().float().numpy()
        out = score * float(np.float32(case["decay"]))
        for g in range(case["groups"]):
            out[g] += np.add.reduce(w[g], axis=0, dtype=np.float64)
            if s["n"] is not None:
                out[g, int(s["n"][g]):] = score[g, int(s["n"][g]):]
        return out
    score = s["s"].cpu().numpy()
    G, L, budget = case["groups"], case["length"], case["budget"]
    keep, kept = np.zeros((G, budget), np.int32), np.zeros(G, np.int32)
    rows = [np.zeros(d.shape) for d in s["d"]]
    fields = [host(f) for f in s["f"]]
    for g in range(G):
        n = L if s["n"] is None else int(s["n"][g])
        chosen = np.arange(n)
        if n > budget:
            middle = np.arange(case["first"], n - case["recent"])
            best = middle[np.lexsort((middle, -score[g, middle]))][:budget - case["first"] - case["recent"]]
            chosen = np.sort(np.concatenate([np.arange(case["first"]), best, np.arange(n - case["recent"], n)]))
        keep[g, :len(chosen)], kept[g] = chosen, len(chosen)
        for out, f in zip(rows, fields):
            out[g, :len(chosen)] = f[g, chosen]
    return [keep, kept] + rows

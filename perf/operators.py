"""The operators of a budgeted KV cache: attention over packed prompts, the attention weight every key received, the
eviction that keeps the heaviest keys, and the decode step over the kept ones.

``listed()`` gives the fixed cases, ``draw(rng)`` more of the same ranges, ``prepare`` what a program holds before the
call, ``run`` the call, ``work`` the bytes and operations no implementation can avoid, ``exact`` the same outputs in 64
bits. With ``own`` false ``run`` computes the operators from elementary torch operations in 32 bits, with ``own`` true
through this package.

Queries and keys are N(0, 1) with a common direction per KV head: one key in 32 and every sequence's first key lie
further along it, so a few keys gather much of the attention weight, as in a trained model.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- the cases ------------------------------------------------------------------------------------------------------


def _prompt(kind: str, seqs: int, q_lo: int, q_hi: int, past_lo: int, past_hi: int, heads: tuple[int, int], dim: int,
            dtype: str, **more) -> dict:
    return {"kind": kind, "seqs": seqs, "q_lo": q_lo, "q_hi": q_hi, "past_lo": past_lo, "past_hi": past_hi,
            "q_heads": heads[0], "kv_heads": heads[1], "dim": dim, "dtype": dtype, "softcap": 0.0, "sinks": False,
            "window": 0, "tail": 0, **more}


def _evict(seqs: int, lo: int, hi: int, kv_heads: int, dim: int, dtype: str, budget: int, recent: int, first: int) -> dict:
    return {"kind": "evict", "seqs": seqs, "q_lo": lo, "q_hi": hi, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "budget": budget, "recent": recent, "first": first}


def _step(batch: int, heads: tuple[int, int], dim: int, dtype: str, budget: int, recent: int, first: int, fill: float,
          **more) -> dict:
    return {"kind": "step", "batch": batch, "q_heads": heads[0], "kv_heads": heads[1], "dim": dim, "dtype": dtype,
            "budget": budget, "recent": recent, "first": first, "fill": fill, "softcap": 0.0, "sinks": False, **more}


def listed() -> list[dict]:
    cases = [
        # one short prompt on a small model: launch and host time
        ("prompt_one", _prompt("prompt", 1, 190, 190, 0, 0, (8, 2), 64, "bf16")),
        # a serving batch's prompts packed without padding, from one token to 2047, rows behind the last one
        ("prompt_packed", _prompt("prompt", 24, 1, 2047, 0, 0, (32, 8), 128, "bf16", tail=7)),
        # one long document
        ("prompt_long", _prompt("prompt", 1, 32768, 32768, 0, 0, (32, 8), 128, "bf16")),
        # chunks of prompts behind the tokens already cached
        ("prompt_chunks", _prompt("prompt", 6, 100, 612, 4000, 12000, (16, 4), 64, "fp16")),
        # the weight every key of a batch of prompts received, before their cache is cut to a budget
        ("mass_packed", _prompt("mass", 4, 1000, 8192, 0, 0, (32, 8), 128, "bf16")),
        # the same from the last 64 queries of each prompt only (an observation window)
        ("mass_window", _prompt("mass", 16, 501, 8000, 0, 0, (16, 4), 64, "fp16", window=64)),
        # one long document's
        ("mass_long", _prompt("mass", 1, 32768, 32768, 0, 0, (32, 8), 128, "bf16")),
        # one prompt cut to a small budget
        ("evict_one", _evict(1, 1021, 1021, 2, 64, "fp16", 256, 32, 4)),
        # a batch of prompts cut to 1024 entries per head
        ("evict_batch", _evict(16, 6000, 8192, 8, 128, "bf16", 1024, 128, 4)),
        # a decode step of one request on a small model: launch and host time
        ("step_one", _step(1, (8, 2), 64, "bf16", 512, 64, 4, 1.0)),
        # a decode step of a full batch, a third of the rows not at their budget yet
        ("step_batch", _step(32, (32, 8), 128, "bf16", 2048, 256, 4, 0.67)),
        # heads of their own K/V (no groups), wide heads, a large budget
        ("step_wide", _step(16, (16, 16), 256, "fp16", 4096, 512, 0, 1.0)),
    ]
    return [{"name": name, **case} for name, case in cases]


def _spread(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["prompt", "mass", "evict", "step"])
    dtype = rng.choice(["bf16", "fp16"])
    heads = rng.choice([(8, 2), (32, 8), (16, 4), (16, 16), (14, 2), (12, 1)])
    dim = rng.choice([64, 128, 128, 256])
    extra = {"softcap": rng.choice([0.0, 0.0, 0.0, 30.0]), "sinks": rng.random() < 0.25}
    if kind in ("prompt", "mass"):
        total = _spread(rng, 100, 20000)  # rows of queries in all
        seqs = min(_spread(rng, 1, 32), total)
        mean = max(1, total // seqs)
        lo = rng.randint(0, mean) if seqs > 1 else mean
        past = _spread(rng, 1, 8000) if rng.random() < 0.3 else 0
        window = rng.choice([16, 32, 64, 100]) if kind == "mass" and rng.random() < 0.4 else 0
        # a case costs no more than one sequence of 32768 tokens at (32, 8) heads of 128 channels
        return _prompt(kind, seqs, lo, 2 * mean - lo, past // 2, past, heads, dim, dtype, window=window,
                       tail=rng.choice([0, 0, 3]), **extra)
    if kind == "evict":
        budget = _spread(rng, 64, 2048)
        hi = _spread(rng, budget // 2 + 1, 16384)
        recent = rng.randint(1, budget // 2)
        return _evict(_spread(rng, 1, 16), rng.randint(hi // 2, hi), hi, heads[1], dim, dtype, budget, recent,
                      rng.choice([0, 4]))
    budget = _spread(rng, 64, 4096)
    batch = max(1, min(_spread(rng, 1, 32), 16 * 16 * 256 // (heads[1] * dim)))
    return _step(batch, heads, dim, dtype, budget, rng.randint(1, budget // 2), rng.choice([0, 4]),
                 rng.choice([0.5, 1.0]), **extra)


def _lens(n: int, lo: int, hi: int) -> list[int]:
    """n lengths spread evenly over [lo, hi], in a fixed mixed order."""
    lens = [lo + (hi - lo) * i // (n - 1) for i in range(n)] if n > 1 else [hi]
    random.Random(n).shuffle(lens)
    return lens


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Queries and keys of every sequence."""
    nq = _lens(case["seqs"], case["q_lo"], case["q_hi"])
    past = _lens(case["seqs"], case.get("past_lo", 0), case.get("past_hi", 0))
    return nq, [a + b if a else 0 for a, b in zip(nq, past)]


def _starts(lens: list[int]) -> list[int]:
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _counts(case: dict) -> list[int]:
    """Tokens every row of a decode step has seen before it: the last rows are not at the budget yet."""
    c, b = case["budget"], case["batch"]
    full = round(b * case["fill"])
    return [c + 37 * i + 1 if i < full else max(1, c * (i - full + 1) // (b - full + 1)) for i in range(b)]


def work(case: dict) -> dict:
    d = case["dim"]
    if case["kind"] in ("prompt", "mass"):
        nq, nk = _lengths(case)
        hq, hkv, t, tk = case["q_heads"], case["kv_heads"], sum(nq), sum(nk)
        if case["kind"] == "prompt":
            pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(nq, nk))
            return {"bytes": 2 * d * (2 * t * hq + 2 * tk * hkv) + 4 * t * hq, "flops": 4 * d * hq * pairs}
        w = [min(n, case["window"]) if case["window"] else n for n in nq]
        pairs = sum(n * k - n * (n - 1) // 2 for n, k in zip(w, nk))
        return {"bytes": 2 * d * (sum(w) * hq + tk * hkv) + 4 * sum(w) * hq + 4 * tk * hkv, "flops": 2 * d * hq * pairs}
    if case["kind"] == "evict":
        nq, _ = _lengths(case)
        kept = sum(min(n, case["budget"]) for n in nq) * case["kv_heads"]
        return {"bytes": 4 * sum(nq) * case["kv_heads"] + kept * (8 * d + 8), "flops": 0}
    slots = sum(min(n + 1, case["budget"]) for n in _counts(case))
    rows = case["batch"] * (case["q_heads"] + 2 * case["kv_heads"])
    return {"bytes": slots * case["kv_heads"] * (4 * d + 12) + 4 * d * rows, "flops": 4 * d * case["q_heads"] * slots}


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _keys(gen: torch.Generator, u: torch.Tensor, *lead: int) -> torch.Tensor:
    """Keys [*lead, Hkv, D], one in 32 further along the head's direction u [Hkv, D]."""
    k = torch.randn(*lead, *u.shape, generator=gen, device=DEVICE)
    heavy = torch.rand(*lead, u.shape[0], 1, generator=gen, device=DEVICE) < 1 / 32
    return k + 0.5 * heavy * u


def _queries(gen: torch.Generator, u: torch.Tensor, groups: int, *lead: int) -> torch.Tensor:
    q = torch.randn(*lead, u.shape[0], groups, u.shape[1], generator=gen, device=DEVICE)
    return (q + 0.6 * u[:, None]).reshape(*lead, -1, u.shape[1])


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, d, hkv = DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    u = torch.randn(hkv, d, generator=gen, device=DEVICE)
    s = {"case": case, "scale": d ** -0.5, "softcap": case.get("softcap", 0.0), "sinks": None}
    hq = case.get("q_heads", hkv)
    if case.get("sinks"):
        s["sinks"] = torch.randn(hq, generator=gen, device=DEVICE)
    if case["kind"] in ("prompt", "mass"):
        nq, nk = _lengths(case)
        s["nq"], s["nk"] = nq, nk
        s["max_q"], s["max_k"] = max(nq), max(nk)
        s["cu_q"] = torch.tensor(_starts(nq), dtype=torch.int32, device=DEVICE)
        s["cu_k"] = torch.tensor(_starts(nk), dtype=torch.int32, device=DEVICE)
        t, tk = sum(nq) + case["tail"], sum(nk) + case["tail"]
        k = _keys(gen, u, tk)
        heads = [b for b, n in zip(_starts(nk), nk) if n]
        k[heads] += 0.7 * u
        s["q"] = _queries(gen, u, hq // hkv, t).to(dt)
        s["k"] = k.to(dt)
        if case["kind"] == "prompt":
            s["v"] = torch.randn(tk, hkv, d, generator=gen, device=DEVICE).to(dt)
        else:
            s["lse"] = _plain_prompt(s, False)[1]
        return s
    if case["kind"] == "evict":
        nq, _ = _lengths(case)
        t = sum(nq)
        s["nq"], s["max_q"] = nq, max(nq)
        s["cu_q"] = torch.tensor(_starts(nq), dtype=torch.int32, device=DEVICE)
        s["k"] = _keys(gen, u, t).to(dt)
        s["v"] = torch.randn(t, hkv, d, generator=gen, device=DEVICE).to(dt)
        # masses: a few heavy keys over a long tail, and a run of exact ties
        s["mass"] = torch.exp(2 * torch.randn(hkv, t, generator=gen, device=DEVICE))
        s["mass"][:, :: 5] = 0.25
        shape = (len(nq), hkv, case["budget"])
        s["position"] = torch.zeros(shape, dtype=torch.int32, device=DEVICE)
        s["count"] = torch.zeros(shape[:2], dtype=torch.int32, device=DEVICE)
        s["length"] = torch.zeros(shape[0], dtype=torch.int32, device=DEVICE)
        s["score"] = torch.zeros(shape, device=DEVICE)
        s["keys"] = torch.zeros(*shape, d, dtype=dt, device=DEVICE)
        s["values"] = torch.zeros(*shape, d, dtype=dt, device=DEVICE)
    else:
        b, c = case["batch"], case["budget"]
        seen = torch.tensor(_counts(case), dtype=torch.int32, device=DEVICE)
        s["q"] = _queries(gen, u, hq // hkv, b).to(dt)
        s["new_k"] = _keys(gen, u, b).to(dt)
        s["new_v"] = torch.randn(b, hkv, d, generator=gen, device=DEVICE).to(dt)
        s["length"] = seen
        s["count"] = seen.clamp(max=c)[:, None].expand(b, hkv).contiguous()
        # rows past their budget hold the newest tokens and a random choice of the older ones, in mixed slots
        slot = torch.arange(c, device=DEVICE, dtype=torch.int32)
        filled = slot < s["count"][..., None]
        newest = seen[:, None, None] - s["count"][..., None] + slot
        order = torch.rand(b, hkv, c, generator=gen, device=DEVICE).masked_fill(~filled, 2.0).argsort(-1)
        s["position"] = newest.expand(b, hkv, c).gather(2, order).masked_fill(~filled, 0).to(torch.int32)
        s["score"] = torch.exp(torch.randn(b, hkv, c, generator=gen, device=DEVICE)) * filled
        s["keys"] = (_keys(gen, u, b, c).transpose(1, 2) * filled[..., None]).to(dt).contiguous()
        s["values"] = (torch.randn(b, hkv, c, d, generator=gen, device=DEVICE) * filled[..., None]).to(dt)
    if own:
        from economize_amd.eviction import HeavyHitterCache

        s["cache"] = HeavyHitterCache(s["keys"], s["values"], s["score"], s["position"], s["count"], s["length"],
                                      recent=case["recent"], first=case["first"])
    return s


# ---- the operators --------------------------------------------------------------------------------------------------


def run(s: dict):
    case = s["case"]
    kind = case["kind"]
    if not own:
        if kind == "prompt":
            return _plain_prompt(s, True)
        return {"mass": _plain_mass, "evict": _plain_evict, "step": _plain_step}[kind](s)
    cap = s["softcap"] or None
    if kind in ("prompt", "mass"):
        from economize_amd.prompt import attention_mass, prompt_attention

        if kind == "prompt":
            return prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["max_q"], s["scale"], cu_seqlens_k=s["cu_k"],
                                    softcap=cap, sinks=s["sinks"], return_lse=True)
        return attention_mass(s["q"], s["k"], s["lse"], s["cu_q"], s["max_q"], s["scale"], cu_seqlens_k=s["cu_k"],
                              max_seqlen_k=s["max_k"], window=case["window"] or None, softcap=cap)
    from economize_amd.eviction import evict_prompt, heavy_hitter_attention

    if kind == "evict":
        evict_prompt(s["cache"], s["k"], s["v"], s["mass"], s["cu_q"], s["max_q"])
        return _state(s)
    out = heavy_hitter_attention(s["cache"], s["q"], s["new_k"], s["new_v"], s["scale"], softcap=cap, sinks=s["sinks"])
    return {"out": out, **_state(s)}


def _state(s: dict) -> dict:
    return {n: s[n] for n in ("keys", "values", "score", "position", "count", "length")}


def _padded(starts: torch.Tensor, lens: list[int], width: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Row indices [N, width] of every sequence (clamped inside the rows) and which of them exist."""
    n = torch.tensor(lens, device=DEVICE)[:, None]
    i = torch.arange(width, device=DEVICE)
    return starts[:-1, None].long() + torch.minimum(i, (n - 1).clamp(min=0)), i < n


def _capped(x: torch.Tensor, cap: float) -> torch.Tensor:
    return torch.tanh(x / cap) * cap if cap else x


def _scores(s: dict, h: int, q_rows: torch.Tensor, k_rows: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 scores [N, G, queries, keys] of KV head h, and which pairs exist: query i sees keys <= i + nk - nq."""
    g = s["q"].shape[1] // s["k"].shape[1]
    rq, rk = q_rows.clamp(max=s["q"].shape[0] - 1), k_rows.clamp(max=s["k"].shape[0] - 1)
    q = s["q"][:, h * g: (h + 1) * g][rq].float()  # [N, queries, G, D]
    k = s["k"][:, h][rk].float()  # [N, keys, D]
    x = torch.matmul(q.transpose(1, 2), k[:, None].transpose(2, 3).contiguous()) * s["scale"]
    i = (q_rows - s["cu_q"][:-1, None])[:, None, :, None]
    j = (k_rows - s["cu_k"][:-1, None])[:, None, None, :]
    nq, nk = (torch.tensor(s[n], device=DEVICE)[:, None, None, None] for n in ("nq", "nk"))
    width = torch.arange(k_rows.shape[1], device=DEVICE)
    return _capped(x, s["softcap"]), (j <= i + nk - nq) & (width < nk)


def _plain_prompt(s: dict, values: bool):
    hq, hkv, d = s["q"].shape[1], s["k"].shape[1], s["q"].shape[2]
    g = hq // hkv
    q_rows, q_there = _padded(s["cu_q"], s["nq"], s["max_q"])
    k_rows, _ = _padded(s["cu_k"], s["nk"], s["max_k"])
    t = s["q"].shape[0]
    rows = torch.where(q_there, q_rows, t).reshape(-1)  # queries that do not exist go to a row of their own
    out = torch.zeros(t + 1, hq, d, dtype=s["q"].dtype, device=DEVICE) if values else None
    lse = torch.full((hq, t + 1), -math.inf, device=DEVICE)
    for h in range(hkv):  # one KV head at a time: the scores of all would not fit
        x, seen = _scores(s, h, q_rows, k_rows)
        x.masked_fill_(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        if s["sinks"] is not None:
            sink = s["sinks"][h * g: (h + 1) * g].view(1, g, 1, 1)
            top = torch.maximum(top, sink)
        top = top.clamp(min=-1e30)
        x.sub_(top).exp_()
        total = x.sum(-1, keepdim=True)
        if s["sinks"] is not None:
            total = total + torch.exp(sink - top)
        lse[h * g: (h + 1) * g, rows] = (top + total.log())[..., 0].transpose(0, 1).reshape(g, -1)
        if values:
            v = s["v"][:, h][k_rows.clamp(max=s["v"].shape[0] - 1)].float()
            o = torch.matmul(x, v[:, None]) / total.clamp(min=1e-38)
            out[rows, h * g: (h + 1) * g] = o.transpose(1, 2).reshape(-1, g, d).to(out.dtype)
    if values:
        out[t - s["case"]["tail"]:] = 0
    lse[:, t - s["case"]["tail"]:] = -math.inf
    return (out[:t], lse[:, :t]) if values else (None, lse[:, :t].contiguous())


def _plain_mass(s: dict) -> torch.Tensor:
    hkv = s["k"].shape[1]
    g = s["q"].shape[1] // hkv
    nq = torch.tensor(s["nq"], device=DEVICE)
    w = min(s["case"]["window"] or s["max_q"], s["max_q"])
    i = (nq[:, None] - w + torch.arange(w, device=DEVICE))  # the last w queries of every sequence
    q_rows = s["cu_q"][:-1, None].long() + i.clamp(min=0)
    k_rows, k_there = _padded(s["cu_k"], s["nk"], s["max_k"])
    t, tk = s["q"].shape[0], s["k"].shape[0]
    rows = torch.where(k_there, k_rows, tk).reshape(-1)
    mass = torch.zeros(hkv, tk + 1, device=DEVICE)
    for h in range(hkv):
        x, seen = _scores(s, h, q_rows, k_rows)
        lse = s["lse"][h * g: (h + 1) * g, q_rows.clamp(max=t - 1)].transpose(0, 1)[..., None]
        seen = seen & (i >= 0)[:, None, :, None]
        x = x.sub_(lse).masked_fill_(~seen, -math.inf).exp_()
        mass[h, rows] = x.sum((1, 2)).reshape(-1)
    mass[:, tk - s["case"]["tail"]:] = 0
    return mass[:, :tk]


def _plain_evict(s: dict) -> dict:
    case = s["case"]
    c, hkv = case["budget"], case["kv_heads"]
    rows, there = _padded(s["cu_q"], s["nq"], s["max_q"])  # [N, S]
    n = torch.tensor(s["nq"], device=DEVICE)[:, None]
    j = torch.arange(s["max_q"], device=DEVICE)
    rank = torch.nan_to_num(s["mass"][:, rows].transpose(0, 1), nan=-math.inf)  # [N, Hkv, S]
    rank = rank.masked_fill(((j < case["first"]) | (j >= n - case["recent"]))[:, None], math.inf)
    kept_all = n <= c
    rank = torch.where(kept_all[:, None], torch.zeros_like(rank), rank).masked_fill(~there[:, None], -math.inf)
    at = rank.sort(dim=-1, descending=True, stable=True).indices[..., :c]
    at = torch.where(there[:, None].expand_as(rank).gather(2, at), at, s["max_q"]).sort(dim=-1).values
    if at.shape[2] < c:
        at = torch.cat([at, at.new_full((*at.shape[:2], c - at.shape[2]), s["max_q"])], 2)
    valid = at < s["max_q"]
    src = (s["cu_q"][:-1].long()[:, None, None] + at).clamp(max=s["k"].shape[0] - 1)
    h = torch.arange(hkv, device=DEVICE)[:, None]
    s["keys"].copy_(torch.where(valid[..., None], s["k"][src, h], s["keys"]))
    s["values"].copy_(torch.where(valid[..., None], s["v"][src, h], s["values"]))
    s["score"].copy_(torch.where(valid, s["mass"][h, src], s["score"]))
    s["position"].copy_(torch.where(valid, at, s["position"]))
    s["count"].copy_(valid.sum(-1))
    s["length"].copy_(n[:, 0])
    return _state(s)


def _plain_step(s: dict) -> dict:
    case = s["case"]
    c, d = case["budget"], case["dim"]
    b, hkv = s["new_k"].shape[:2]
    g = s["q"].shape[1] // hkv
    slot = torch.arange(c, device=DEVICE)
    pos, t = s["position"], s["length"][:, None, None]
    free = (pos >= case["first"]) & (pos <= t - case["recent"])
    rank = torch.nan_to_num(s["score"], nan=-math.inf).masked_fill(~free, math.inf)
    victim = torch.where(rank == rank.amin(-1, keepdim=True), slot, c).amin(-1)
    to = torch.where(s["count"] < c, s["count"], victim)[..., None].long()
    s["keys"].scatter_(2, to[..., None].expand(b, hkv, 1, d), s["new_k"][:, :, None])
    s["values"].scatter_(2, to[..., None].expand(b, hkv, 1, d), s["new_v"][:, :, None])
    s["score"].scatter_(2, to, 0.0)
    s["position"].scatter_(2, to, t.expand(b, hkv, 1).contiguous())
    s["count"].copy_((s["count"] + 1).clamp(max=c))
    s["length"].add_(1)
    q = s["q"].view(b, hkv, g, d).float()
    x = _capped(torch.matmul(q, s["keys"].float().transpose(2, 3).contiguous()) * s["scale"], s["softcap"])
    valid = slot < s["count"][..., None]
    x = x.masked_fill_(~valid[:, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, hkv, g, 1)
        top = torch.maximum(top, sink)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    p = x / total
    out = torch.matmul(p, s["values"].float()).reshape(b, hkv * g, d).to(s["q"].dtype)
    s["score"].add_(p.sum(2))
    return {"out": out, **_state(s)}


# ---- 64 bits --------------------------------------------------------------------------------------------------------


def _exact_weights(q, k, scale, cap, sink, last):
    """Scores and visibility of queries q [n, D] (float64), the first of them seeing keys <= last."""
    x = scale * (q @ k.T)
    if cap:
        x = cap * torch.tanh(x / cap)
    hidden = torch.arange(k.shape[0], device=DEVICE)[None] > last + torch.arange(q.shape[0], device=DEVICE)[:, None]
    x[hidden] = -math.inf
    lse = torch.logsumexp(x, 1) if sink is None else torch.logaddexp(torch.logsumexp(x, 1), sink)
    return x, lse


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] in ("prompt", "mass"):
        return _exact_prompt(s)
    return _exact_evict(s) if case["kind"] == "evict" else _exact_step(s)


def _exact_prompt(s: dict):
    case = s["case"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    prompt = case["kind"] == "prompt"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE) if prompt else None
    lses = torch.full((hq, s["q"].shape[0]), -math.inf, dtype=torch.float64, device=DEVICE)
    mass = torch.zeros(hkv, s["k"].shape[0], dtype=torch.float64, device=DEVICE)
    q0 = k0 = 0
    for nq, nk in zip(s["nq"], s["nk"]):
        begin = max(0, nq - case["window"]) if case["window"] else 0
        for head in range(hq):
            kv = head * hkv // hq
            k = s["k"][k0: k0 + nk, kv].double()
            sink = None if s["sinks"] is None else s["sinks"][head].double()
            for lo in range(begin, nq, 4096):
                hi = min(nq, lo + 4096)
                see = nk - nq + hi  # no query of the block sees a later key
                x, lse = _exact_weights(s["q"][q0 + lo: q0 + hi, head].double(), k[:see], s["scale"], case["softcap"],
                                        sink, lo + nk - nq)
                if prompt:
                    lses[head, q0 + lo: q0 + hi] = lse
                    out[q0 + lo: q0 + hi, head] = torch.exp(x - lse[:, None]) @ s["v"][k0: k0 + see, kv].double()
                else:
                    given = s["lse"][head, q0 + lo: q0 + hi].double()
                    mass[kv, k0: k0 + see] += torch.exp(x - given[:, None]).sum(0)
        q0, k0 = q0 + nq, k0 + nk
    return (out, lses) if prompt else mass


def _exact_evict(s: dict) -> dict:
    """Counted rather than sorted: a token is kept if fewer than the budget are before it in the order."""
    case = s["case"]
    c, got = case["budget"], {n: s[n].double() for n in ("keys", "values", "score")}
    begin = 0
    for b, n in enumerate(s["nq"]):
        for h in range(case["kv_heads"]):
            m = s["mass"][h, begin: begin + n].double()
            j = torch.arange(n, device=DEVICE)
            must = (j < case["first"]) | (j >= n - case["recent"])
            m = torch.where(must, torch.full_like(m, math.inf), m)
            values, inverse, ties = torch.unique(m, return_inverse=True, return_counts=True)
            above = ties.flip(0).cumsum(0).flip(0)[inverse] - ties[inverse]
            order = torch.argsort(inverse * n + j)  # equal masses by index
            among = torch.empty_like(j)
            among[order] = torch.arange(n, device=DEVICE) - (ties.cumsum(0) - ties)[inverse[order]]
            kept = torch.nonzero(above + among < c)[:, 0]
            got["keys"][b, h, : len(kept)] = s["k"][begin + kept, h].double()
            got["values"][b, h, : len(kept)] = s["v"][begin + kept, h].double()
            got["score"][b, h, : len(kept)] = s["mass"][h, begin + kept].double()
        begin += n
    return {**got, "position": None, "count": None, "length": None}


def _exact_step(s: dict) -> dict:
    case = s["case"]
    c, d, hkv = case["budget"], case["dim"], case["kv_heads"]
    g = case["q_heads"] // hkv
    out = torch.zeros(case["batch"], case["q_heads"], d, dtype=torch.float64, device=DEVICE)
    score = s["score"].double()
    keys, values = s["keys"].double(), s["values"].double()
    for b, seen in enumerate(s["length"].tolist()):
        counts = s["count"][b].tolist()
        for h in range(hkv):
            to = counts[h]
            if to == c:
                old = (s["position"][b, h] >= case["first"]) & (s["position"][b, h] <= seen - case["recent"])
                slots = torch.nonzero(old)[:, 0]
                to = int(slots[torch.sort(score[b, h, slots], stable=True).indices[0]])
            keys[b, h, to], values[b, h, to], score[b, h, to] = s["new_k"][b, h], s["new_v"][b, h], 0.0
            n = min(counts[h] + 1, c)
            x = s["scale"] * (s["q"][b, h * g: (h + 1) * g].double() @ keys[b, h, :n].T)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            lse = torch.logsumexp(x, 1)
            if s["sinks"] is not None:
                lse = torch.logaddexp(lse, s["sinks"][h * g: (h + 1) * g].double())
            p = torch.exp(x - lse[:, None])
            out[b, h * g: (h + 1) * g] = p @ values[b, h, :n]
            score[b, h, :n] += p.sum(0)
    return {"out": out, "keys": keys, "values": values, "score": score, "position": None, "count": None, "length": None}

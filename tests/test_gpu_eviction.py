"""Caches held at a budget (``eco_evict_prompt``, ``eco_heavy_hitter_decode``) against the 64-bit oracle
(``oracle/budget.py``): what stays of a prompt (exactly, ties and NaN included), decode steps and the scores they leave,
rows below and at their budget, and the whole path from a prompt's attention to its decode."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from budget_cases import assert_output, f64, prompt_inputs, score_error
from oracle import budget as ob

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def check_evicted(cache, k, v, mass, cu) -> None:
    cu = cu.tolist()
    m = mass.cpu().numpy()
    for b, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        assert cache.length[b].item() == hi - lo
        for h in range(k.shape[1]):
            kept = ob.evict(m[h, lo:hi].astype(np.float64), cache.budget, cache.recent, cache.first)
            n = len(kept)
            assert cache.count[b, h].item() == n
            assert cache.position[b, h, :n].tolist() == kept.tolist(), (b, h)
            at = torch.from_numpy(kept + lo).to(k.device)
            assert torch.equal(cache.keys[b, h, :n], k[at, h]) and torch.equal(cache.values[b, h, :n], v[at, h])
            assert torch.equal(cache.score[b, h, :n].view(torch.int32), mass[h, at].view(torch.int32))


LENGTHS = [[0, 1, 63], [64, 65], [66, 200, 64], [1000, 4096, 4097], [5000], [16384, 16385, 300], [40000]]


@pytest.mark.parametrize("lens", LENGTHS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("budget,recent,first", [(64, 1, 0), (64, 30, 4), (64, 60, 4), (64, 64, 0), (700, 100, 1)])
def test_evict(lens, budget, recent, first) -> None:
    from economize_amd.eviction import HeavyHitterCache, evict_prompt

    dtype, dim = (BF16, 64) if len(lens) > 1 else (FP16, 128)
    _, k, v, cu, _ = prompt_inputs(1, lens, lens, (4, 2), dim, dtype, tail=3)
    gen = torch.Generator().manual_seed(2)
    mass = torch.exp(2 * torch.randn(2, k.shape[0], generator=gen))
    mass[:, ::3] = 0.5  # many equal ones
    cache = HeavyHitterCache.empty(len(lens), 2, dim, budget, dtype, "cuda", recent, first)
    print(f"evict {lens} to {budget} {recent} {first}", flush=True)
    evict_prompt(cache, k, v, mass.cuda(), cu, max(lens))
    check_evicted(cache, k, v, mass.cuda(), cu)


@pytest.mark.parametrize("kind", ["all_equal", "zeros", "signed", "nan", "inf", "close"])
def test_evict_orders(kind) -> None:
    """Masses in every order of the type: equal ones, zeros of both signs, negative, infinite, NaN, one bit apart."""
    from economize_amd.eviction import HeavyHitterCache, evict_prompt

    n = 3001
    _, k, v, cu, _ = prompt_inputs(3, [n], [n], (2, 2), 64, BF16)
    rng = np.random.default_rng(4)
    m = {"all_equal": np.full((2, n), 1.25), "zeros": rng.choice([0.0, -0.0], (2, n)),
         "signed": rng.standard_normal((2, n)), "nan": rng.choice([np.nan, -np.nan, 1.0, -1.0, -np.inf], (2, n)),
         "inf": rng.choice([np.inf, -np.inf, 0.0, 3.0], (2, n)),
         "close": 1 + rng.integers(0, 64, (2, n)) * 2.0 ** -23}[kind].astype(np.float32)
    mass = torch.from_numpy(m).cuda()
    cache = HeavyHitterCache.empty(1, 2, 64, 500, BF16, "cuda", 10, 2)
    evict_prompt(cache, k, v, mass, cu)
    check_evicted(cache, k, v, mass, cu)


def test_evict_views_and_slots_past_the_count() -> None:
    """Strided K, V and masses, a padded batch, and slots past the count left as they were."""
    from economize_amd.eviction import HeavyHitterCache, evict_prompt

    width = 90
    _, k, v, _, _ = prompt_inputs(5, [width] * 2, [width] * 2, (2, 2), 64, BF16)
    begin = torch.tensor([70, 90], dtype=torch.int32, device="cuda")
    end = torch.tensor([90, 180], dtype=torch.int32, device="cuda")
    mass = torch.rand(2, 200, generator=torch.Generator().manual_seed(6)).cuda()[:, :180]
    cache = HeavyHitterCache.empty(2, 2, 64, 40, BF16, "cuda", 8)
    cache.keys.fill_(9.0)
    cache.score.fill_(-1.0)
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)
    evict_prompt(cache, kt, v, mass, (begin, end))
    assert cache.count.tolist() == [[20, 20], [40, 40]] and cache.length.tolist() == [20, 90]
    assert (cache.keys[0, :, 20:] == 9).all() and (cache.score[0, :, 20:] == -1).all()
    for h in range(2):
        assert torch.equal(cache.keys[0, h, :20], k[70:90, h])
        kept = ob.evict(f64(mass[h, 90:]), 40, 8, 0)
        assert cache.position[1, h].tolist() == kept.tolist()
        assert torch.equal(cache.values[1, h], v[torch.from_numpy(90 + kept).cuda(), h])


def test_evict_bound_and_own_memory() -> None:
    """``max_seqlen`` sizes the launch: longer rows are copied all the same. A cache is no source of its own prompt."""
    from economize_amd.errors import ConfigError
    from economize_amd.eviction import HeavyHitterCache, evict_prompt

    lens = [900, 1, 300]
    _, k, v, cu, _ = prompt_inputs(27, lens, lens, (2, 2), 64, BF16)
    mass = torch.rand(2, sum(lens), generator=torch.Generator().manual_seed(28)).cuda()
    for bound in (0, 1, 40, 900, 10 ** 6, None):
        cache = HeavyHitterCache.empty(3, 2, 64, 512, BF16, "cuda", 8, 4)
        evict_prompt(cache, k, v, mass, cu, bound)
        check_evicted(cache, k, v, mass, cu)
    own = cache.keys[0].transpose(0, 1)
    for args in ((own, v[:512], mass[:, :512]), (k[:512], own, mass[:, :512]), (k[:512], v[:512], cache.score[0])):
        with pytest.raises(ConfigError, match="apart from the cache"):
            evict_prompt(cache, *args, cu)


def make_cache(seed, batch, heads, dim, dtype, budget, recent, first, seen):
    """A cache whose rows have seen ``seen`` tokens, the kept ones in mixed slots."""
    from economize_amd.eviction import HeavyHitterCache

    gen = torch.Generator().manual_seed(seed)
    hkv = heads[1]
    cache = HeavyHitterCache.empty(batch, hkv, dim, budget, dtype, "cuda", recent, first)
    cache.length.copy_(torch.tensor(seen, dtype=torch.int32))
    for b, n in enumerate(seen):
        for h in range(hkv):
            c = min(n, budget)
            old = torch.randperm(max(0, n - recent - first), generator=gen)[: max(0, c - recent - first)] + first
            pos = torch.cat([torch.arange(min(first, n)), old, torch.arange(max(min(first, n), n - recent), n)])[:c]
            pos = pos[torch.randperm(len(pos), generator=gen)]
            cache.count[b, h] = len(pos)
            cache.position[b, h, : len(pos)] = pos.to(torch.int32).cuda()
            cache.score[b, h, : len(pos)] = torch.exp(torch.randn(len(pos), generator=gen)).cuda()
    cache.keys.copy_(torch.randn(cache.keys.shape, generator=gen).to(dtype))
    cache.values.copy_(torch.randn(cache.keys.shape, generator=gen).to(dtype))
    return cache, gen


def states(cache):
    return [dict(keys=f64(cache.keys[b]), values=f64(cache.values[b]), score=f64(cache.score[b]),
                 position=cache.position[b].cpu().numpy().astype(int).copy(),
                 count=cache.count[b].cpu().numpy().astype(int).copy(), length=int(cache.length[b]))
            for b in range(cache.keys.shape[0])]


def step_and_check(cache, q, k, v, **more) -> None:
    from economize_amd.eviction import heavy_hitter_attention

    before = states(cache)
    scale = more.get("scale") or q.shape[-1] ** -0.5
    sinks = more.get("sinks")
    out = heavy_hitter_attention(cache, q, k, v, **more)
    torch.cuda.synchronize()
    after = states(cache)
    error = score_error(q, torch.cat([k[:, :, None], cache.keys], 2), scale, cache.budget)
    for b, state in enumerate(before):
        want, size = ob.heavy_step(state, f64(q[b]), f64(k[b]), f64(v[b]), cache.budget, cache.recent, cache.first,
                                   scale, more.get("softcap"), None if sinks is None else f64(sinks))
        assert_output(out[b], want, size, error)
        for name in ("keys", "values", "position", "count"):
            for h in range(k.shape[1]):
                n = state["count"][h] if name != "count" else None
                assert np.array_equal(after[b][name][h][:n] if n else after[b][name][h],
                                      state[name][h][:n] if n else state[name][h]), (b, h, name)
        assert after[b]["length"] == state["length"]
        for h in range(k.shape[1]):
            n = state["count"][h]
            off = np.abs(after[b]["score"][h, :n] - state["score"][h, :n])
            # weights within 2 error, and an fp32 sum of at most 65 terms
            assert (off <= (2 * error + 65 * 2.0 ** -24) * 1.01 * np.abs(state["score"][h, :n]) + 1e-30).all()


def new_token(gen, batch, heads, dim, dtype):
    return (torch.randn(batch, heads[0], dim, generator=gen).to(dtype).cuda(),
            torch.randn(batch, heads[1], dim, generator=gen).to(dtype).cuda(),
            torch.randn(batch, heads[1], dim, generator=gen).to(dtype).cuda())


@pytest.mark.parametrize("heads,dim", [((8, 2), 64), ((8, 8), 128), ((32, 8), 128), ((17, 1), 64), ((64, 1), 128),
                                       ((4, 2), 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("budget,recent,first,seen", [
    (64, 8, 0, [0, 1, 63, 64, 65]),
    (300, 40, 4, [299, 300, 1000]),
    (33, 1, 0, [10, 50]),
    (130, 130, 0, [400]),
    (1, 1, 0, [0, 7]),
])
def test_steps(budget, recent, first, seen, dtype, heads, dim) -> None:
    cache, gen = make_cache(7, len(seen), heads, dim, dtype, budget, recent, first, seen)
    print(f"steps {heads} {dim} {dtype} {budget} {seen}", flush=True)
    for _ in range(3):
        step_and_check(cache, *new_token(gen, len(seen), heads, dim, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_steps_softcap_sinks_scale(dtype) -> None:
    heads, dim, seen = (12, 4), 128, [5, 700]
    cache, gen = make_cache(8, 2, heads, dim, dtype, 500, 60, 4, seen)
    sinks = (3 * torch.randn(12, generator=gen)).cuda()
    step_and_check(cache, *new_token(gen, 2, heads, dim, dtype), softcap=15.0)
    step_and_check(cache, *new_token(gen, 2, heads, dim, dtype), sinks=sinks)
    step_and_check(cache, *new_token(gen, 2, heads, dim, dtype), sinks=sinks, softcap=30.0, scale=0.7)


def test_step_takes_the_lower_of_equal_scores_and_a_nan_first() -> None:
    cache, gen = make_cache(9, 2, (4, 2), 64, BF16, 64, 4, 0, [500, 500])
    cache.score.fill_(2.0)
    cache.score[1, 0, 40] = math.nan
    cache.score[1, 1] = -math.inf
    step_and_check_positions = [cache.position.clone(), cache.count.clone()]
    from economize_amd.eviction import heavy_hitter_attention

    before = states(cache)
    q, k, v = new_token(gen, 2, (4, 2), 64, BF16)
    heavy_hitter_attention(cache, q, k, v)
    for b in range(2):
        ob.heavy_step(before[b], f64(q[b]), f64(k[b]), f64(v[b]), 64, 4, 0, 0.125)
        assert np.array_equal(cache.position[b].cpu().numpy(), before[b]["position"])
    assert int((cache.position[1, 0] != step_and_check_positions[0][1, 0]).nonzero()) == 40


def test_slots_past_the_count_are_not_read() -> None:
    heads, seen = (8, 2), [10, 100, 33]
    cache, gen = make_cache(10, 3, heads, 128, BF16, 256, 16, 0, seen)
    for b, n in enumerate(seen):
        cache.keys[b, :, n:] = math.nan
        cache.values[b, :, n:] = math.nan
        cache.score[b, :, n:] = math.nan
        cache.position[b, :, n:] = -7
    for _ in range(2):
        step_and_check(cache, *new_token(gen, 3, heads, 128, BF16))


def test_a_step_over_many_slots() -> None:
    """Enough slots that a launch of its own chooses the new token's."""
    cache, gen = make_cache(21, 1, (4, 2), 64, BF16, 16400, 900, 4, [30000])
    for _ in range(2):
        step_and_check(cache, *new_token(gen, 1, (4, 2), 64, BF16))


def test_strided_step_and_out() -> None:
    from economize_amd.eviction import heavy_hitter_attention

    heads, dim = (8, 2), 64
    a, gen = make_cache(11, 2, heads, dim, FP16, 100, 10, 0, [50, 300])
    b, _ = make_cache(11, 2, heads, dim, FP16, 100, 10, 0, [50, 300])
    q, k, v = new_token(gen, 2, heads, dim, FP16)
    want = heavy_hitter_attention(a, q, k, v)
    fused = torch.cat([q.reshape(2, -1), k.reshape(2, -1), v.reshape(2, -1)], 1)
    out = torch.full((2, 10, dim), 3.0, dtype=FP16, device="cuda")
    got = heavy_hitter_attention(b, fused[:, :512].view(2, 8, dim), fused[:, 512:640].view(2, 2, dim),
                                 fused[:, 640:].view(2, 2, dim), out=out[:, 1:9])
    assert torch.equal(got, want) and (out[:, 0] == 3).all() and (out[:, 9] == 3).all()
    for name in ("keys", "values", "score", "position", "count", "length"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_the_path_from_a_prompt_to_its_decode() -> None:
    """Attention over packed prompts, the weight of every key, the cache cut to its budget, decode steps over it; and the
    kept prompt decoded over as compact entries with the prompt's dense slots behind."""
    from economize_amd.eviction import HeavyHitterCache, evict_prompt
    from economize_amd.gathered import gathered_decode_attention
    from economize_amd.prompt import attention_mass, prompt_attention

    lens, heads, dim, budget = [500, 40, 1300], (8, 2), 128, 200
    q, k, v, cu, _ = prompt_inputs(12, lens, lens, heads, dim, BF16)
    out, lse = prompt_attention(q, k, v, cu, max(lens), return_lse=True)
    mass = attention_mass(q, k, lse, cu, max(lens))
    # every query gives a weight of one per head
    for h in range(2):
        np.testing.assert_allclose([float(mass[h, a:b].sum()) for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:])],
                                   [4.0 * n for n in lens], rtol=1e-5)
    cache = HeavyHitterCache.empty(3, 2, dim, budget, BF16, "cuda", 20, 4)
    evict_prompt(cache, k, v, mass, cu, max(lens))
    check_evicted(cache, k, v, mass, cu)

    gen = torch.Generator().manual_seed(13)
    q1, k1, v1 = new_token(gen, 3, heads, dim, BF16)
    width = max(lens) + 1
    dense_k = torch.full((3, 2, width, dim), math.nan, dtype=BF16, device="cuda")
    dense_v = dense_k.clone()
    mask = torch.zeros(3, 1, 1, width, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        dense_k[b, :, n], dense_v[b, :, n] = k1[b], v1[b]
        mask[b, :, :, : n + 1] = True
    dense_k, dense_v = dense_k.nan_to_num(0.0), dense_v.nan_to_num(0.0)
    gathered = gathered_decode_attention(q1[:, :, None], dense_k, dense_v, mask, dim ** -0.5, cache.gathered())
    for b in range(3):
        for h in range(2):
            n = int(cache.count[b, h])
            kk = f64(torch.cat([cache.keys[b, h, :n], k1[b, h][None]]))
            vv = f64(torch.cat([cache.values[b, h, :n], v1[b, h][None]]))
            x = dim ** -0.5 * f64(q1[b, 4 * h: 4 * h + 4]) @ kk.T
            p = np.exp(x - x.max(1, keepdims=True))
            np.testing.assert_allclose(f64(gathered[b, 0, 4 * h: 4 * h + 4]), p / p.sum(1, keepdims=True) @ vv,
                                       atol=2e-3, rtol=1e-2)
    for _ in range(5):
        step_and_check(cache, *new_token(gen, 3, heads, dim, BF16))
    assert int(cache.count.max()) == budget and cache.length.tolist() == [n + 5 for n in lens]


def test_captured_steps_replay() -> None:
    """A captured step advances the cache on the device; every replay equals an eager step on a twin."""
    from economize_amd.eviction import heavy_hitter_attention

    heads, dim = (8, 2), 128
    make = lambda: make_cache(14, 3, heads, dim, BF16, 96, 16, 2, [90, 96, 300])[0]  # noqa: E731
    a, b = make(), make()
    gen = torch.Generator().manual_seed(15)
    q, k, v = new_token(gen, 3, heads, dim, BF16)
    out_a, out_b = torch.empty_like(q), torch.empty_like(q)
    names = ("keys", "values", "score", "position", "count", "length")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        heavy_hitter_attention(a, q, k, v, out=out_a)
    torch.cuda.synchronize()
    heavy_hitter_attention(b, q, k, v, out=out_b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        heavy_hitter_attention(a, q, k, v, out=out_a)
    for i in range(12):  # (the first row reaches its budget on the way)
        for t, new in zip((q, k, v), new_token(gen, 3, heads, dim, BF16)):
            t.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        heavy_hitter_attention(b, q, k, v, out=out_b)
        torch.cuda.synchronize()
        assert torch.equal(out_a, out_b), i
        for name in names:
            assert torch.equal(getattr(a, name), getattr(b, name)), (i, name)


def test_two_caches_on_two_streams() -> None:
    from economize_amd.eviction import heavy_hitter_attention

    heads, dim = (8, 2), 64
    caches = [make_cache(s, 4, heads, dim, BF16, 512, 64, 0, [600, 511, 9, 3000])[0] for s in (16, 17, 16, 17)]
    gen = torch.Generator().manual_seed(18)
    tokens = [new_token(gen, 4, heads, dim, BF16) for _ in range(6)]
    want = [[heavy_hitter_attention(c, *t) for t in tokens] for c in caches[:2]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for t in tokens:
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                got[s].append(heavy_hitter_attention(caches[2 + s], *t))
    torch.cuda.synchronize()
    for s in range(2):
        for a, b in zip(want[s], got[s]):
            assert torch.equal(a, b)


def test_refusals() -> None:
    from economize_amd.errors import ConfigError
    from economize_amd.eviction import HeavyHitterCache, evict_prompt, heavy_hitter_attention

    for more, match in ((dict(head_dim=96), "head dims 64, 128 and 256"), (dict(dtype=torch.float32), "bf16 or fp16"),
                        (dict(recent=0), "recent >= 1"), (dict(recent=60, first=5), "recent \\+ first <= budget"),
                        (dict(budget=0), "at least one row, head and slot")):
        args = dict(batch=2, kv_heads=2, head_dim=64, budget=64, dtype=BF16, device="cuda", recent=8) | more
        with pytest.raises(ConfigError, match=match):
            HeavyHitterCache.empty(**args)
    cache = HeavyHitterCache.empty(2, 2, 64, 64, BF16, "cuda", 8)
    _, k, v, cu, _ = prompt_inputs(19, [5, 6], [5, 6], (4, 2), 64, BF16)
    mass = torch.ones(2, 11, device="cuda")
    for args, match in (((k.half(), v, mass, cu), "for a cache of"), ((k, v[:5], mass, cu), "takes keys and values"),
                        ((k, v, mass[:, :5], cu), "mass must be"), ((k, v, mass.double(), cu), "mass must be"),
                        ((k, v, mass, cu[:2]), "1 sequences for a cache of 2"), ((k, v, mass, cu.long()), "int32")):
        with pytest.raises(ConfigError, match=match):
            evict_prompt(cache, *args)
    gen = torch.Generator().manual_seed(20)
    q, k, v = new_token(gen, 2, (4, 2), 64, BF16)
    for args, more, match in (
        ((q[:1], k, v), {}, "takes queries"), ((q[:, :3], k, v), {}, "not a multiple"), ((q, k[:, :1], v), {}, "the new keys"),
        ((q, k, v.half()), {}, "a step of"), ((q, k, v), {"sinks": torch.zeros(3, device="cuda")}, "sink logits"),
        ((q, k, v), {"scale": -1.0}, "scale must be positive"), ((q, k, v), {"softcap": math.inf}, "softcap"),
        ((q, k, v), {"out": torch.empty(2, 4, 32, dtype=BF16, device="cuda")}, "out must be"),
        ((torch.zeros(2, 130, 64, dtype=BF16, device="cuda"), k, v), {}, "at most 64 query heads"),
    ):
        with pytest.raises(ConfigError, match=match):
            heavy_hitter_attention(cache, *args, **more)
    assert not cache.length.any() and not cache.count.any()
    cache.position = cache.position.transpose(0, 1)
    with pytest.raises(ConfigError, match="position must be contiguous"):
        heavy_hitter_attention(cache, q, k, v)

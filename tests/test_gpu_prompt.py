"""Packed prompt attention (``eco_prompt_attention``) and the attention weight of its keys (``eco_attention_mass``) against
the 64-bit oracle (``oracle/budget.py``): sequence lengths around the tiles' edges, empty sequences, queries behind
cached keys, queries without keys, grouped heads, head dims, strides, padded batches, soft cap, sinks, windows, infinities
and NaN where no query looks, rows of no sequence, other streams, graphs. Tolerances: ``tests/budget_cases.py``."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from budget_cases import assert_output, f64, prompt_inputs, score_error
from oracle import budget as ob

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def run(q, k, v, cu_q, cu_k, lens_q, lens_k, scale=None, softcap=None, sinks=None, **more):
    from economize_amd.prompt import prompt_attention

    return prompt_attention(q, k, v, cu_q, max(lens_q, default=0), scale, cu_seqlens_k=cu_k,
                            max_seqlen_k=max(lens_k, default=0), softcap=softcap, sinks=sinks, **more)


def check(q, k, v, cu_q, cu_k, lens_q, lens_k, scale=None, softcap=None, sinks=None, window=None, rows=None):
    """Attention, its denominators and the keys' masses against the oracle."""
    from economize_amd.prompt import attention_mass

    d = q.shape[-1]
    real = d ** -0.5 if scale is None else scale
    out, lse = run(q, k, v, cu_q, cu_k, lens_q, lens_k, scale, softcap, sinks, return_lse=True)
    torch.cuda.synchronize()
    host = tuple(tuple(f64(x) for x in c) if isinstance(c, tuple) else f64(c) for c in (cu_q, cu_k))
    host = [tuple(x.astype(int) for x in c) if isinstance(c, tuple) else c.astype(int) for c in host]
    want, want_lse, size = ob.prompt_attention(f64(q), f64(k), f64(v), *host, real, softcap,
                                               None if sinks is None else f64(sinks))
    error = score_error(q, k, real, max(lens_k, default=0))
    if rows is None:
        rows = np.ones(q.shape[0], bool)
    assert_output(out[torch.from_numpy(rows).to(out.device)], want[rows], size[rows], error)
    g = f64(lse)
    finite = np.isfinite(want_lse)
    assert np.array_equal(finite, np.isfinite(g)) and np.array_equal(np.isnan(want_lse), np.isnan(g))
    assert np.max(np.abs(g[finite] - want_lse[finite]), initial=0) <= error
    mass = attention_mass(q, k, lse, cu_q, max(lens_q, default=0), scale, cu_seqlens_k=cu_k,
                          max_seqlen_k=max(lens_k, default=0), window=window, softcap=softcap)
    torch.cuda.synchronize()
    want_mass = ob.attention_mass(f64(q), f64(k), f64(lse), *host, real, softcap, window)
    terms = max(lens_q, default=0) * (q.shape[1] // k.shape[1])
    m = f64(mass)
    ok = np.isfinite(want_mass)
    assert np.array_equal(ok, np.isfinite(m))
    assert (np.abs(m - want_mass)[ok] <= (error + (terms / 32 + 32) * 2.0 ** -24) * 1.01 * want_mass[ok] + 1e-30).all()
    return out, lse, mass


LENGTHS = [
    ([1], [1]),
    ([63, 1, 64, 65], None),
    ([127, 128, 0, 129, 2], None),
    ([255, 257, 33], None),
    ([5, 100, 1], [5, 1000, 700]),   # chunks behind cached keys, a single token among them
    ([1, 1, 1], [64, 65, 1]),
    ([70, 200, 3], [10, 130, 0]),    # queries that see no key
    ([700], None),
]


@pytest.mark.parametrize("heads,dim", [((8, 2), 64), ((8, 8), 128), ((8, 2), 128), ((6, 2), 64), ((7, 1), 128),
                                       ((4, 1), 256)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", range(len(LENGTHS)))
def test_lengths(case, dtype, heads, dim) -> None:
    lens_q, lens_k = LENGTHS[case]
    lens_k = lens_k or lens_q
    q, k, v, cu_q, cu_k = prompt_inputs(case, lens_q, lens_k, heads, dim, dtype)
    print(f"prompt {lens_q} behind {lens_k} {heads} {dim} {dtype}", flush=True)
    check(q, k, v, cu_q, cu_k, lens_q, lens_k)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_softcap_sinks_scale_window(dtype, dim) -> None:
    lens = [150, 1, 0, 333]
    q, k, v, cu, _ = prompt_inputs(11, lens, lens, (12, 4), dim, dtype)
    sinks = torch.randn(12, generator=torch.Generator().manual_seed(1)).cuda() * 3
    check(q, k, v, cu, cu, lens, lens, softcap=20.0, window=64)
    check(q, k, v, cu, cu, lens, lens, sinks=sinks, window=1)
    check(q, k, v, cu, cu, lens, lens, scale=0.5, sinks=sinks, softcap=50.0, window=1000)


@pytest.mark.parametrize("lens_q,lens_k", [([1], [9000]), ([3, 130, 0, 1], [2000, 5000, 0, 64]), ([40, 7], [4095, 513]),
                                           ([600], [1700])])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64), (BF16, 256)])
def test_few_queries_behind_many_keys(lens_q, lens_k, dtype, dim) -> None:
    """Too few rows for the GPU: their keys are cut into parts and joined."""
    from economize_amd import _lib

    heads = (6, 2)
    q, k, v, cu_q, cu_k = prompt_inputs(17, lens_q, lens_k, heads, dim, dtype)
    assert _lib.lib().eco_prompt_attention_workspace_size(len(lens_q), sum(lens_q), max(lens_q), max(lens_k), *heads,
                                                          dim) > 0
    sinks = torch.randn(6, generator=torch.Generator().manual_seed(2)).cuda()
    check(q, k, v, cu_q, cu_k, lens_q, lens_k)
    check(q, k, v, cu_q, cu_k, lens_q, lens_k, sinks=sinks, softcap=30.0, window=2)
    out = torch.full((sum(lens_q) + 5, 6, dim), 2.0, dtype=dtype, device="cuda")
    run(torch.cat([q, q[:1].expand(5, -1, -1)]), k, v, cu_q, cu_k, lens_q, lens_k, out=out)
    assert (out[-5:] == 2).all()


@pytest.mark.parametrize("lens_q,lens_k,heads", [([70, 3], [6200, 900], (64, 2)), ([40], [6400], (64, 64))])
def test_many_heads_over_many_keys(lens_q, lens_k, heads) -> None:
    """Enough tiles of keys for 64 of them to a wave of the mass, cut by heads and whole."""
    q, k, v, cu_q, cu_k = prompt_inputs(25, lens_q, lens_k, heads, 128, BF16)
    check(q, k, v, cu_q, cu_k, lens_q, lens_k)


def test_few_rows_of_a_large_buffer() -> None:
    """One chunk in a buffer of many rows: what the rest holds does not matter, and it gives 0."""
    q, k, v, _, _ = prompt_inputs(26, [6000], [6000], (4, 2), 64, BF16)
    q[40:] = math.nan
    k[5000:] = math.nan
    v[5000:] = math.nan
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows, rows_k = (zero, zero + 40), (zero, zero + 5000)
    from economize_amd.prompt import prompt_attention
    out, lse = prompt_attention(q, k, v, rows, 40, cu_seqlens_k=rows_k, max_seqlen_k=5000, return_lse=True)
    assert not out[40:].any() and torch.isneginf(lse[:, 40:]).all()
    cu = np.array([0, 40]), np.array([0, 5000])
    exact, _, size = ob.prompt_attention(f64(q[:40]), f64(k[:5000]), f64(v[:5000]), *cu, 64 ** -0.5)
    assert_output(out[:40], exact, size, score_error(q[:40], k[:5000], 64 ** -0.5, 5000))


def test_unseen_nan_in_a_cut_row() -> None:
    """The keys are cut, and the last tiles hold infinities that only the last queries see."""
    q, k, v, cu_q, cu_k = prompt_inputs(18, [100], [3000], (4, 2), 128, BF16)
    v[2999, 0, 5], v[2950, 1, 9], v[2890, 0, 77] = math.inf, math.nan, -math.inf
    out, _, _ = check(q, k, v, cu_q, cu_k, [100], [3000])
    assert torch.isfinite(out[:99, :2, 5]).all() and torch.isinf(out[99, :2, 5]).all()


def test_sinks_without_keys() -> None:
    """A query without keys attends to its sink alone: 0, and the sink's logit as its denominator's logarithm."""
    q, k, v, cu_q, cu_k = prompt_inputs(2, [70], [5], (4, 2), 64, BF16)
    sinks = torch.tensor([1.0, -2.0, 30.0, 0.0], device="cuda")
    out, lse, _ = check(q, k, v, cu_q, cu_k, [70], [5], sinks=sinks)
    assert not out[:65].any() and torch.allclose(lse[:, :65], sinks[:, None].expand(4, 65), atol=1e-5)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64), (BF16, 256)])
def test_large_scores(dtype, dim) -> None:
    """Scores in the hundreds, maxima that move late: the running maximum rescales what is summed already."""
    lens = [300, 129]
    q, k, v, cu, _ = prompt_inputs(5, lens, lens, (4, 2), dim, dtype)
    k = (k.float() * torch.linspace(0.1, 8, k.shape[0], device="cuda")[:, None, None]).to(dtype)
    check(q, k, v, cu, cu, lens, lens, scale=0.4)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (FP16, 64), (FP16, 256)])
def test_unseen_infinities_and_nan(dtype, dim, value) -> None:
    """Keys and values past what a query sees may hold anything; a query that does see them gets them."""
    lens = [150, 200]
    q, k, v, cu, _ = prompt_inputs(6, lens, lens, (4, 2), dim, dtype, tail=80)
    v[149, 0, 3] = value        # the first sequence's last key: seen by its last query only
    v[150 + 100, 1, 7] = value  # inside the second's
    v[350:] = value             # behind the last sequence
    k[350:] = value
    q[350:] = value
    rows = np.arange(430) < 350
    out, _, mass = check(q, k, v, cu, cu, lens, lens, rows=rows)
    assert torch.isfinite(out[:149]).all() and not torch.isfinite(out[149, :2, 3]).any()
    assert not out[350:].any() and not mass[:, 350:].any()


def test_unseen_nan_keys() -> None:
    lens = [150, 64]
    q, k, v, cu, _ = prompt_inputs(7, lens, lens, (4, 2), 128, BF16)
    k[120, 0] = math.nan
    out, lse = run(q, k, v, cu, cu, lens, lens, return_lse=True)
    assert torch.isfinite(out[:120].float()).all() and torch.isfinite(out[150:].float()).all()
    assert torch.isfinite(out[:, 2:].float()).all() and torch.isnan(out[120:150, :2].float()).all()
    assert torch.isfinite(lse[:, :120]).all() and torch.isnan(lse[:2, 120:150]).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_strides(dim) -> None:
    """Views of a fused projection, a batch-first layout and a head-first layout give what contiguous copies give."""
    lens, heads = [130, 77], (4, 2)
    t = sum(lens)
    q, k, v, cu, _ = prompt_inputs(8, lens, lens, heads, dim, BF16)
    want = run(q, k, v, cu, cu, lens, lens, return_lse=True)
    fused = torch.cat([q.reshape(t, -1), k.reshape(t, -1), v.reshape(t, -1)], 1)
    a, b = 4 * dim, 6 * dim
    views = (fused[:, :a].view(t, 4, dim), fused[:, a:b].view(t, 2, dim), fused[:, b:].view(t, 2, dim))
    heads_first = tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    odd = tuple(torch.cat([x, x], -1)[..., 1:dim + 1].copy_(x) for x in (q, k, v))  # rows off 16 bytes: copied
    for x in (views, heads_first, odd):
        got = run(*x, cu, cu, lens, lens, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out = torch.full((t, 6, dim), 7.0, dtype=BF16, device="cuda")
    run(q, k, v, cu, cu, lens, lens, out=out[:, 1:5])
    assert torch.equal(out[:, 1:5], want[0]) and (out[:, 0] == 7).all() and (out[:, 5] == 7).all()


def test_rows_of_no_sequence_are_left_as_they_are() -> None:
    lens = [40, 100]
    q, k, v, cu, _ = prompt_inputs(9, lens, lens, (4, 2), 64, BF16, tail=30)
    out = torch.full_like(q, 5.0)
    run(q, k, v, cu, cu, lens, lens, out=out)
    assert (out[140:] == 5).all() and not (out[:140] == 5).all(-1).any()
    from economize_amd.prompt import attention_mass

    _, lse = run(q, k, v, cu, cu, lens, lens, return_lse=True)
    assert torch.isneginf(lse[:, 140:]).all()
    mass = torch.full((2, 170), -3.0, device="cuda")
    attention_mass(q, k, lse, cu, 100, out=mass)
    assert (mass[:, 140:] == -3).all() and (mass[:, :140] > 0).all()


def test_padded_batch() -> None:
    """Left-padded rows as (begin, end): the padding gives 0, and what it holds does not matter."""
    lens, width = [30, 64, 1], 64
    q, k, v, _, _ = prompt_inputs(10, [width] * 3, [width] * 3, (4, 2), 64, FP16)
    begin = torch.tensor([64 - 30, 64, 128 + 63], dtype=torch.int32, device="cuda")
    end = torch.tensor([64, 128, 192], dtype=torch.int32, device="cuda")
    pad = torch.ones(192, dtype=torch.bool, device="cuda")
    for b, e in zip(begin.tolist(), end.tolist()):
        pad[b:e] = False
    for x in (q, k, v):
        x[pad] = math.nan
    rows = (begin, end)
    out, lse, mass = check(q, k, v, rows, rows, lens, lens, rows=(~pad).cpu().numpy())
    assert not out[pad].any() and torch.isneginf(lse[:, pad]).all() and not mass[:, pad].any()


def test_bounds_of_the_launch_do_not_bound_the_result() -> None:
    """``max_seqlen`` sizes the launch: longer sequences are computed all the same; bounds outside the rows are clamped."""
    from economize_amd.prompt import attention_mass, prompt_attention

    lens = [900, 1, 300]
    q, k, v, cu, _ = prompt_inputs(12, lens, lens, (4, 1), 128, BF16)
    want, lse = prompt_attention(q, k, v, cu, 900, return_lse=True)
    rows = cu.cpu().numpy()
    exact, _, size = ob.prompt_attention(f64(q), f64(k), f64(v), rows, rows, 128 ** -0.5)
    for bound in (0, 1, 100, 900, None):  # (the bound decides how long rows are cut, so the bits may differ)
        assert_output(prompt_attention(q, k, v, cu, bound), exact, size, score_error(q, k, 128 ** -0.5, 900))
    # (the bound decides how a long walk is cut: the same positive terms, summed in another order, each sum within
    # (terms / 32 + 32) 2^-24 of its value)
    mass = attention_mass(q, k, lse, cu, 900)
    rtol = 2 * (900 * 4 / 32 + 32) * 2.0 ** -24
    for bound in (0, 1, 300, None):
        torch.testing.assert_close(attention_mass(q, k, lse, cu, bound), mass, rtol=rtol, atol=0)
    wild = torch.tensor([-5, 900, 901, 99999], dtype=torch.int32, device="cuda")
    assert torch.equal(prompt_attention(q, k, v, wild, 900), want)


def test_no_rows() -> None:
    from economize_amd.prompt import attention_mass, prompt_attention

    cu = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    k = torch.zeros(0, 2, 64, dtype=BF16, device="cuda")
    out, lse = prompt_attention(q, k, k, cu, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    assert attention_mass(q, k, lse, cu).shape == (2, 0)
    q = torch.ones(5, 4, 64, dtype=BF16, device="cuda")
    out, lse = prompt_attention(q, k, k, torch.tensor([0, 5], dtype=torch.int32, device="cuda"),
                                cu_seqlens_k=torch.tensor([0, 0], dtype=torch.int32, device="cuda"), return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


def test_same_bits_every_time_and_on_another_stream() -> None:
    from economize_amd.prompt import attention_mass

    lens = [513, 64, 1200]
    q, k, v, cu, _ = prompt_inputs(13, lens, lens, (8, 2), 128, BF16)
    want, lse = run(q, k, v, cu, cu, lens, lens, return_lse=True)
    mass = attention_mass(q, k, lse, cu, 1200)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_lse = run(q, k, v, cu, cu, lens, lens, return_lse=True)
        got_mass = attention_mass(q, k, got_lse, cu, 1200)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got_lse, lse) and torch.equal(got_mass, mass)


def test_captured_and_replayed() -> None:
    """A captured call follows the lengths and inputs on the device."""
    from economize_amd.prompt import attention_mass

    heads, dim = (8, 2), 64
    sets = [[300, 20, 150], [1, 400, 69], [470, 0, 0], [156, 157, 157]]
    q, k, v, cu, _ = prompt_inputs(14, sets[0], sets[0], heads, dim, FP16)

    def call():
        out, lse = run(q, k, v, cu, cu, [470], [470], return_lse=True)
        return out, lse, attention_mass(q, k, lse, cu, 470, window=50)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = call()
    for i, lens in enumerate(sets * 2):
        new = prompt_inputs(20 + i, lens, lens, heads, dim, FP16)
        for a, b in zip((q, k, v, cu), new):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, call()):
            assert torch.equal(a, b), i


def test_far_rows() -> None:
    """Rows whose byte offsets pass 32 bits: a sequence at the end of a long buffer of wide rows."""
    rows, pitch = 70000, 32768  # 70000 rows of 64 KiB: 4.6 GB
    lens = [200]
    q, k, v, _, _ = prompt_inputs(15, lens, lens, (2, 1), 64, BF16)
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    want = run(q, k, v, cu, cu, lens, lens, return_lse=True)
    big = torch.empty(rows, pitch, dtype=BF16, device="cuda")
    far = torch.tensor([rows - 200, rows], dtype=torch.int32, device="cuda")
    big[-200:, :64], big[-200:, 64:128] = k[:, 0], v[:, 0]
    kb, vb = big[:, :64].unsqueeze(1), big[:, 64:128].unsqueeze(1)
    from economize_amd.prompt import attention_mass, prompt_attention

    got = prompt_attention(q, kb, vb, cu, 200, cu_seqlens_k=far, max_seqlen_k=200, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    mass = attention_mass(q, kb, got[1], cu, 200, cu_seqlens_k=far, max_seqlen_k=200)
    assert torch.equal(mass[:, -200:], attention_mass(q, k, want[1], cu, 200)) and not mass[:, :-200].any()


def test_refusals() -> None:
    from economize_amd.errors import ConfigError
    from economize_amd.prompt import attention_mass, prompt_attention

    lens = [10, 20]
    q, k, v, cu, _ = prompt_inputs(16, lens, lens, (4, 2), 64, BF16)
    lse = torch.zeros(4, 30, device="cuda")
    for args, more, match in (
        ((q.float(), k.float(), v.float(), cu), {}, "bf16 or fp16"),
        ((q, k.half(), v, cu), {}, "one dtype"),
        ((q[:, :3], k, v, cu), {}, "not a multiple"),
        ((q, k, v[:20], cu), {}, "do not match"),
        ((q[..., :32], k[..., :32], v[..., :32], cu), {}, "head dim must be 64, 128 or 256"),
        ((q, k, v, cu.long()), {}, "int32"),
        ((q, k, v, cu[:1]), {}, "at least one sequence"),
        ((q, k, v, cu.cpu()), {}, "cu_seqlens on cpu"),
        ((q, k[:20], v[:20], cu), {}, "need cu_seqlens_k"),
        ((q, k, v, cu), {"cu_seqlens_k": cu[:2]}, "2 sequences of queries, 1 of keys"),
        ((q, k, v, cu), {"scale": 0.0}, "scale must be positive"),
        ((q, k, v, cu), {"scale": math.nan}, "scale must be positive"),
        ((q, k, v, cu), {"softcap": -1.0}, "softcap"),
        ((q, k, v, cu), {"sinks": torch.zeros(3, device="cuda")}, "sink logits"),
        ((q, k, v, cu), {"out": torch.empty(30, 4, 32, dtype=BF16, device="cuda")}, "out must be"),
    ):
        with pytest.raises(ConfigError, match=match):
            prompt_attention(*args, **more)
    for args, more, match in (
        ((q, k, lse[:, :20], cu), {}, "lse must be"),
        ((q, k, lse, cu), {"window": 0}, "window"),
        ((q, k, lse, cu), {"out": torch.zeros(2, 20, device="cuda")}, "out must be"),
    ):
        with pytest.raises(ConfigError, match=match):
            attention_mass(*args, **more)
    with pytest.raises(RuntimeError, match="run on an AMD GPU"):
        prompt_attention(q.cpu(), k.cpu(), v.cpu(), cu.cpu())

"""The C ABI's refusals of the packed-prompt and budgeted-cache entry points, on the CPU: a call that is well formed but for
one argument returns 1 with a message that names it, before any device work (stand-in addresses, as in
``test_capi_refusals.py``); and what their Python layer refuses of tensors it can look at without a device."""

from __future__ import annotations

import math
import re
from pathlib import Path

import pytest
import torch

from economize_amd import _lib

ROOT = Path(__file__).resolve().parents[1]

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="stand-in addresses: run without a GPU")

FAKE = 1 << 20
ROWS = dict(sequences=2, q_rows=30, k_rows=30, max_queries=20, max_keys=20)
SHAPE = dict(format=_lib.ECO_BF16, q_heads=8, kv_heads=2, head_dim=64, scale=0.125, softcap=0.0)
CACHE = dict(batch=2, kv_heads=2, slots=64, head_dim=64, recent=8, first=4)
BASE = {
    "eco_prompt_attention": dict(
        null=("sinks", "workspace", "stream"), **ROWS, **SHAPE, sq_t=512, sq_h=64, sk_t=128, sk_h=64, sv_t=128, sv_h=64,
        so_t=512, so_h=64, sl_h=30, fill=1, workspace_bytes=1 << 40),
    "eco_attention_mass": dict(
        null=("workspace", "stream"), **ROWS, **SHAPE, sq_t=512, sq_h=64, sk_t=128, sk_h=64, sl_h=30, window=0, sm_h=30,
        fill=1, workspace_bytes=0),
    "eco_evict_prompt": dict(
        null=("stream",), **CACHE, sk_t=128, sk_h=64, sv_t=128, sv_h=64, sm_h=30, rows=30, max_tokens=20),
    "eco_heavy_hitter_decode": dict(
        null=("sinks", "stream"), **{**SHAPE, **CACHE}, sq_b=512, sq_h=64, sk_b=128, sk_h=64, sv_b=128, sv_h=64, so_b=512,
        so_h=64, workspace_bytes=1 << 40),
}
CASES = [
    ("eco_prompt_attention", dict(k=None), "null pointer"),
    ("eco_prompt_attention", dict(q_end=None), "null sequence bounds"),
    ("eco_prompt_attention", dict(format=_lib.ECO_FP32), "bf16 or fp16"),
    ("eco_prompt_attention", dict(q_heads=7), "not a multiple of the KV heads"),
    ("eco_prompt_attention", dict(head_dim=80), "head dim must be 64, 128 or 256"),
    ("eco_prompt_attention", dict(scale=0.0), "scale must be positive"),
    ("eco_prompt_attention", dict(scale=math.inf), "scale must be positive"),
    ("eco_prompt_attention", dict(softcap=math.nan), "softcap must be"),
    ("eco_prompt_attention", dict(sequences=0), "at least one sequence"),
    ("eco_prompt_attention", dict(k_rows=1 << 31), "rows must be"),
    ("eco_prompt_attention", dict(sk_t=132), "keys need strides"),
    ("eco_prompt_attention", dict(sv_t=1 << 24), "values need strides"),
    ("eco_prompt_attention", dict(sq_h=-64), "queries need strides"),
    ("eco_prompt_attention", dict(out=FAKE + 8), "outputs must be 16-byte aligned"),
    ("eco_prompt_attention", dict(sl_h=29), "lse rows are shorter"),
    ("eco_prompt_attention", dict(max_queries=-1), "must not be negative"),
    ("eco_prompt_attention", dict(max_keys=30000, workspace_bytes=0), "workspace is too small"),
    ("eco_prompt_attention", dict(sequences=40000), "too many sequences"),
    ("eco_prompt_attention", dict(q_rows=1 << 30, sl_h=1 << 30), "too many queries"),
    ("eco_prompt_attention", dict(so_t=0), "outputs overlap each other"),
    ("eco_prompt_attention", dict(so_t=64, so_h=1920 - 8), "outputs overlap each other"),
    ("eco_prompt_attention", dict(k_rows=0x7fffffff), "rows must be"),
    ("eco_attention_mass", dict(lse=None), "null pointer"),
    ("eco_attention_mass", dict(max_queries=30000, max_keys=30000), "workspace is too small"),
    ("eco_attention_mass", dict(window=-1), "must not be negative"),
    ("eco_attention_mass", dict(sm_h=29), "mass rows are shorter"),
    ("eco_attention_mass", dict(k=FAKE + 2), "keys must be 16-byte aligned"),
    ("eco_evict_prompt", dict(mass=None), "null pointer"),
    ("eco_evict_prompt", dict(count=None), "null cache"),
    ("eco_evict_prompt", dict(recent=0), "recent >= 1"),
    ("eco_evict_prompt", dict(recent=61), "recent \\+ first <= slots"),
    ("eco_evict_prompt", dict(slots=0), "sizes must be positive"),
    ("eco_evict_prompt", dict(slots=1 << 29), "too many slots"),
    ("eco_evict_prompt", dict(batch=1, kv_heads=1, slots=(1 << 25) + 1), "too many slots"),
    ("eco_evict_prompt", dict(batch=40000), "too many rows"),
    ("eco_evict_prompt", dict(keys=FAKE - 64), "apart from the cache"),
    ("eco_evict_prompt", dict(sm_h=3), "mass rows are shorter"),
    ("eco_evict_prompt", dict(rows=-1), "rows must be"),
    ("eco_heavy_hitter_decode", dict(workspace=None), "null pointer"),
    ("eco_heavy_hitter_decode", dict(workspace_bytes=64), "workspace is too small"),
    ("eco_heavy_hitter_decode", dict(workspace=FAKE + 4), "workspace must be 16-byte aligned"),
    ("eco_heavy_hitter_decode", dict(q_heads=132), "at most 64 query heads"),
    ("eco_heavy_hitter_decode", dict(keys=FAKE + 2), "cache must be 16-byte aligned"),
    ("eco_heavy_hitter_decode", dict(head_dim=512), "head dim must be 64, 128 or 256"),
    ("eco_heavy_hitter_decode", dict(sk_b=4), "keys need strides"),
    ("eco_heavy_hitter_decode", dict(so_h=32), "outputs overlap each other"),
    ("eco_heavy_hitter_decode", dict(batch=70000, kv_heads=1, q_heads=1, slots=12), "too many rows"),
]


def _names(fn: str) -> list[str]:
    text = (ROOT / "include" / "economize_amd.h").read_text()
    m = re.search(r"\bint " + fn + r"\s*\(([^)]*)\)\s*;", text, flags=re.S)
    assert m, fn
    return [re.findall(r"(\w+)\s*$", p.strip())[0] for p in m.group(1).split(",")]


@no_gpu
@pytest.mark.parametrize("fn,bad,message", CASES, ids=[f"{c[0]}-{'-'.join(c[1])}-{i}" for i, c in enumerate(CASES)])
def test_refused_before_any_device_work(fn: str, bad: dict, message: str) -> None:
    base = dict(BASE[fn])
    null = set(base.pop("null"))
    names = _names(fn)
    assert set(bad) <= set(names) and set(base) <= set(names) and null <= set(names)
    args = []
    for name, kind in zip(names, _lib.SIGNATURES[fn][1]):
        if name in bad:
            args.append(bad[name])
        elif name in base:
            args.append(base[name])
        else:
            assert kind is _lib._P, (fn, name)
            args.append(None if name in null else FAKE)
    lib = _lib.lib()
    rc = getattr(lib, fn)(*args)
    error = (lib.eco_last_error() or b"").decode()
    assert rc == 1 and re.search(message, error), (rc, error)


@no_gpu
def test_nothing_to_do_is_no_error() -> None:
    lib = _lib.lib()
    for fn, rows in (("eco_prompt_attention", "q_rows"), ("eco_attention_mass", "k_rows")):
        base = dict(BASE[fn])
        null = set(base.pop("null"))
        base[rows] = 0
        args = [base[n] if n in base else None if n in null else FAKE for n in _names(fn)]
        assert getattr(lib, fn)(*args) == 0


def test_workspaces() -> None:
    lib = _lib.lib()
    assert lib.eco_heavy_hitter_workspace_size(2, 8, 2, 64, 64) > 0
    assert lib.eco_heavy_hitter_workspace_size(2, 7, 2, 64, 64) == 0
    assert lib.eco_prompt_attention_workspace_size(2, 20, 10, 10, 7, 2, 64) == 0
    # few rows in a large buffer: the parts' places for all of its rows stay within half a GiB
    assert 0 < lib.eco_prompt_attention_workspace_size(1, 100, 100, 32768, 32, 8, 128) <= 1 << 29
    assert 0 <= lib.eco_prompt_attention_workspace_size(1, 32768, 100, 32768, 32, 8, 128) <= 1 << 29
    assert lib.eco_prompt_attention_workspace_size(1, 0, 0, 32768, 32, 8, 128) == 0


def test_caches_and_rows_are_checked() -> None:
    from economize_amd.errors import ConfigError
    from economize_amd.eviction import HeavyHitterCache
    from economize_amd.prompt import check_out, prompt_attention, row_bounds

    with pytest.raises(ConfigError, match="recent"):
        HeavyHitterCache.empty(1, 1, 64, 8, torch.bfloat16, "cpu", recent=9)
    cache = HeavyHitterCache.empty(2, 2, 64, 8, torch.float16, "cpu", recent=4, first=4)
    assert cache.budget == 8 and cache.gathered().dropped == 0
    cache.score = cache.score.double()
    with pytest.raises(ConfigError, match="score must be"):
        cache.check()
    cpu = torch.device("cpu")
    cu = torch.tensor([0, 3, 3, 8], dtype=torch.int32)
    assert row_bounds(cu, cpu)[1:] == (cu.data_ptr(), cu.data_ptr() + 4, 3)
    x = torch.zeros(6, 4, 64, dtype=torch.float16)
    for out in (x, x[:, :2], x.transpose(0, 1).contiguous().transpose(0, 1), x[:1], x[:, :1]):
        assert check_out(out, out, "") == (out.data_ptr(), *(s if n > 1 else t for n, s, t in zip(
            out.shape, out.stride(), check_out(out, out, "")[1:])))
    for out in (x[:1].expand(6, 4, 64), x[:, :1].expand(6, 4, 64), x.as_strided((3, 4, 64), (128, 64, 1)), x[..., ::2]):
        with pytest.raises(ConfigError, match="out must be"):
            check_out(out, out, "")
    for rows in (cu.long(), cu[:1], cu[::2], cu[None], (cu, cu[:2]), (cu, cu.float()), (cu,), [0, 8], 8):
        with pytest.raises(ConfigError):
            row_bounds(rows, cpu)
    with pytest.raises(RuntimeError, match="AMD GPU"):
        prompt_attention(torch.zeros(8, 2, 64), torch.zeros(8, 2, 64), torch.zeros(8, 2, 64), cu)

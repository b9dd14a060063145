"""Attention over whole prompts on the GPU: packed sequences of different lengths, and the weight every key received.

The reference's kernels take up to 64 queries (attention/interface.py:243-285) and leave prompts to ``sdpa``, which
takes one padded batch; these take packed rows and give the softmax statistics an eviction by accumulated attention
weight needs (:mod:`economize_amd.eviction`).

Sequences are given by ``cu_seqlens``, int32 ``[N + 1]`` on the device (sequence ``s`` holds rows ``cu[s] .. cu[s + 1]``), or
by a pair ``(begin, end)`` of int32 ``[N]`` (sequences in order and apart, rows between them belonging to none: a padded
batch). ``max_seqlen`` is the longest one (it sizes the launch; the number of rows when it is not known).
"""

from __future__ import annotations

import functools
import math
from typing import Union

import torch

from . import _lib
from .decode import sinks_operand
from .errors import ConfigError

__all__ = ["Rows", "attention_mass", "prompt_attention"]

#: Rows of the sequences: ``cu_seqlens`` or ``(begin, end)``.
Rows = Union[torch.Tensor, tuple[torch.Tensor, torch.Tensor]]

DTYPES = (torch.bfloat16, torch.float16)
#: Strides the kernels take, in elements: a tile's rows lie within 32 bits of its first one.
STRIDE_LIMIT = 1 << 24


def row_bounds(rows: Rows, device: torch.device) -> tuple[object, int, int, int]:
    """What keeps the bounds alive, the addresses of every sequence's first and past-the-end row, and how many sequences
    there are."""
    if isinstance(rows, torch.Tensor):
        shape = rows.shape
        if rows.dtype is not torch.int32 or len(shape) != 1 or shape[0] < 2 or not rows.is_contiguous():
            raise ConfigError("cu_seqlens must be contiguous int32 [sequences + 1] with at least one sequence")
        if rows.device != device:
            raise ConfigError(f"cu_seqlens on {rows.device}, the queries on {device}")
        at = rows.data_ptr()
        return rows, at, at + 4, shape[0] - 1
    if not isinstance(rows, (tuple, list)) or len(rows) != 2:
        raise ConfigError("sequences are given by cu_seqlens or by (begin, end)")
    begin, end = rows
    for t in (begin, end):
        if not torch.is_tensor(t) or t.dtype != torch.int32 or t.dim() != 1 or t.numel() < 1 or t.stride(0) != 1 or t.device != device:
            raise ConfigError(f"begin and end must be contiguous int32 [sequences] on {device}")
    if begin.numel() != end.numel():
        raise ConfigError(f"{begin.numel()} sequences begin, {end.numel()} end")
    return rows, begin.data_ptr(), end.data_ptr(), begin.numel()


def operand(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """``x`` ``[A, B, D]`` of 16-bit elements as the kernels read it, its address and its first two strides: unit channel
    stride, address and strides whole 16 bytes, strides from 0 to below :data:`STRIDE_LIMIT` (a copy only when it is not; the
    stride of an axis of one entry is not used and given as 0)."""
    a, b, c = x.stride()
    at = x.data_ptr()
    if c == 1 and not (at & 15 or a & 7 or b & 7) and 0 <= a < STRIDE_LIMIT and 0 <= b < STRIDE_LIMIT:
        return x, at, a, b
    a, b = (0 if n <= 1 else s for n, s in zip(x.shape, (a, b)))
    if c == 1 and not (at & 15 or a & 7 or b & 7) and 0 <= a < STRIDE_LIMIT and 0 <= b < STRIDE_LIMIT:
        return x, at, a, b
    copy = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    copy.copy_(x)
    return copy, copy.data_ptr(), copy.stride(0), copy.stride(1)


def check_out(out: torch.Tensor, like: torch.Tensor, what: str) -> tuple[int, int, int]:
    """The address and strides of an output buffer the kernels can write."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ConfigError(f"out must be {what} in the query's dtype on its device")
    same, at, a, b = operand(out)
    if same is not out:
        raise ConfigError(f"out must be {what}, channels contiguous and rows on 16 bytes")
    reach = out.shape[2]  # elements up to the end of one entry of the axis before
    for stride, n in sorted(((a, out.shape[0]), (b, out.shape[1]))):
        if n > 1 and stride < reach:
            raise ConfigError(f"out must be {what} with every element apart, not strides {tuple(out.stride())}")
        reach += (n - 1) * stride
    return at, a, b


def _check(what: str, query: torch.Tensor, key: torch.Tensor) -> tuple[int, int, int, int, int, int]:
    """Queries, query heads, head dim, keys, KV heads and the C ABI's format."""
    shape, shape_k, dtype = query.shape, key.shape, query.dtype
    if len(shape) != 3 or len(shape_k) != 3 or shape[2] != shape_k[2]:
        raise ConfigError(f"{what} takes queries [T, Hq, D] and keys [Tk, Hkv, D], got {tuple(shape)} and {tuple(shape_k)}")
    if dtype not in DTYPES or key.dtype is not dtype:
        raise ConfigError(f"{what} takes bf16 or fp16 queries and keys of one dtype, got {dtype} and {key.dtype}")
    tokens, q_heads, head_dim = shape
    keys, kv_heads, _ = shape_k
    if kv_heads == 0 or q_heads % kv_heads or q_heads == 0:
        raise ConfigError(f"{q_heads} query heads are not a multiple of {kv_heads} KV heads")
    return tokens, q_heads, head_dim, keys, kv_heads, _lib.fmt(dtype)


@functools.lru_cache(maxsize=1024)
def _prompt_workspace(*sizes: int) -> int:
    return _lib.lib().eco_prompt_attention_workspace_size(*sizes)


@functools.lru_cache(maxsize=1024)
def _mass_workspace(*sizes: int) -> int:
    return _lib.lib().eco_attention_mass_workspace_size(*sizes)


def _sequences(cu_seqlens: Rows, cu_seqlens_k: Rows | None, tokens: int, keys: int, device: torch.device) -> tuple:
    bounds = row_bounds(cu_seqlens, device)
    if cu_seqlens_k is None:
        if keys != tokens:
            raise ConfigError(f"{keys} keys for {tokens} queries need cu_seqlens_k")
        return bounds, bounds
    bounds_k = bounds if cu_seqlens_k is cu_seqlens else row_bounds(cu_seqlens_k, device)
    if bounds_k[3] != bounds[3]:
        raise ConfigError(f"{bounds[3]} sequences of queries, {bounds_k[3]} of keys")
    return bounds, bounds_k


def prompt_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, cu_seqlens: Rows,
                     max_seqlen: int | None = None, scale: float | None = None, *, cu_seqlens_k: Rows | None = None,
                     max_seqlen_k: int | None = None, softcap: float | None = None, sinks: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, return_lse: bool = False
                     ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of packed sequences: query ``i`` of a sequence of ``nq`` queries and ``nk`` keys sees its keys
    ``j <= i + nk - nq`` (the queries are its last tokens, so a prompt may be given in chunks behind its earlier keys).

    Args:
        query: ``[T, Hq, D]`` (any strides), bf16 or fp16, head dim 64, 128 or 256.
        key, value: ``[Tk, Hkv, D]`` in the query's dtype.
        cu_seqlens: The sequences' query rows (see the module).
        max_seqlen: The longest sequence's queries.
        scale: Multiplier of the scores, positive (``1 / sqrt(D)``).
        cu_seqlens_k: The sequences' key rows, when they are not the query rows.
        max_seqlen_k: The longest sequence's keys.
        softcap: Optional tanh soft cap of the scaled scores.
        sinks: Optional ``[Hq]`` attention-sink logits.
        out: Optional ``[T, Hq, D]`` output buffer apart from the keys and values; rows of no sequence are left as they are.
        return_lse: Also return the logarithm of every softmax denominator, fp32 ``[Hq, T]``.

    Returns:
        ``[T, Hq, D]`` in the query's dtype (and the denominators' logarithms). A query that sees no key, and without
        ``out`` a row of no sequence, gives 0 and ``-inf``. Nothing here is differentiated.
    """
    device = _lib.require_gpu(query, key, value)
    tokens, q_heads, head_dim, keys, kv_heads, form = _check("prompt_attention", query, key)
    if value.shape != key.shape or value.dtype is not key.dtype:
        raise ConfigError(f"values {tuple(value.shape)} {value.dtype} do not match the keys {tuple(key.shape)} {key.dtype}")
    (keep, q_begin, q_end, sequences), (keep_k, k_begin, k_end, _) = _sequences(cu_seqlens, cu_seqlens_k, tokens, keys,
                                                                                device)
    if sinks is not None:
        sinks = sinks_operand(sinks, q_heads)
        if sinks.device != device:
            raise ConfigError(f"sinks on {sinks.device}, the queries on {device}")
    fill = out is None
    if fill:
        out = torch.empty(tokens, q_heads, head_dim, dtype=query.dtype, device=device)
        at, so_t, so_h = out.data_ptr(), q_heads * head_dim, head_dim
    else:
        at, so_t, so_h = check_out(out, query, "[T, Hq, D]")
    lse = None
    if return_lse:
        lse = torch.empty(q_heads, tokens, dtype=torch.float32, device=device)
        if not fill:
            lse.fill_(-math.inf)
    if tokens:
        query, q_at, sq_t, sq_h = operand(query)
        key, k_at, sk_t, sk_h = operand(key)
        value, v_at, sv_t, sv_h = operand(value)
        max_q = tokens if max_seqlen is None else min(int(max_seqlen), tokens)
        max_k = min(int(max_seqlen_k), keys) if max_seqlen_k is not None else max_q if cu_seqlens_k is None else keys
        need = _prompt_workspace(sequences, tokens, max_q, max_k, q_heads, kv_heads, head_dim)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.call_on(
            device, "eco_prompt_attention", q_at, form, sq_t, sq_h, k_at, v_at, sk_t, sk_h, sv_t, sv_h,
            q_begin, q_end, k_begin, k_end, sequences, tokens, keys, max_q, max_k, _lib.ptr(sinks), at, so_t, so_h,
            _lib.ptr(lse), tokens, fill, q_heads, kv_heads, head_dim, head_dim ** -0.5 if scale is None else scale,
            softcap or 0.0, _lib.ptr(ws), need)
    return (out, lse) if return_lse else out


def attention_mass(query: torch.Tensor, key: torch.Tensor, lse: torch.Tensor, cu_seqlens: Rows,
                   max_seqlen: int | None = None, scale: float | None = None, *, cu_seqlens_k: Rows | None = None,
                   max_seqlen_k: int | None = None, window: int | None = None, softcap: float | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """The attention weight every key of packed sequences received, fp32 ``[Hkv, Tk]``: the sum over the queries that see
    the key and the query heads of its KV head of ``exp(score - lse)``, in a fixed order.

    Args:
        query, key, cu_seqlens, max_seqlen, scale, cu_seqlens_k, max_seqlen_k, softcap: As :func:`prompt_attention` took
            them.
        lse: fp32 ``[Hq, T]``, as :func:`prompt_attention` returned it.
        window: Count only the last ``window`` queries of every sequence (an observation window).
        out: Optional fp32 ``[Hkv, Tk]`` output buffer; keys of no sequence are left as they are (without it they give 0).
    """
    device = _lib.require_gpu(query, key, lse)
    tokens, q_heads, head_dim, keys, kv_heads, form = _check("attention_mass", query, key)
    if lse.dtype is not torch.float32 or lse.shape != (q_heads, tokens) or (tokens > 1 and lse.stride(1) != 1) or \
            (q_heads > 1 and lse.stride(0) < tokens):
        raise ConfigError(f"lse must be fp32 [{q_heads}, {tokens}] with contiguous rows apart")
    if window is not None and (isinstance(window, bool) or int(window) != window or window < 1):
        raise ConfigError(f"window must be a positive integer or None, got {window!r}")
    (keep, q_begin, q_end, sequences), (keep_k, k_begin, k_end, _) = _sequences(cu_seqlens, cu_seqlens_k, tokens, keys,
                                                                                device)
    fill = out is None
    if fill:
        out = torch.empty(kv_heads, keys, dtype=torch.float32, device=device)
    elif out.dtype != torch.float32 or tuple(out.shape) != (kv_heads, keys) or out.device != device or \
            (keys > 1 and out.stride(1) != 1) or (kv_heads > 1 and out.stride(0) < keys):
        raise ConfigError(f"out must be fp32 [{kv_heads}, {keys}] with contiguous rows apart on {device}")
    if keys:
        query, q_at, sq_t, sq_h = operand(query)
        key, k_at, sk_t, sk_h = operand(key)
        max_q = tokens if max_seqlen is None else min(int(max_seqlen), tokens)
        max_k = min(int(max_seqlen_k), keys) if max_seqlen_k is not None else max_q if cu_seqlens_k is None else keys
        window = min(int(window or 0), 0x7fffffff)
        need = _mass_workspace(max_q, keys, window, q_heads, kv_heads)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.call_on(
            device, "eco_attention_mass", q_at, form, sq_t, sq_h, k_at, sk_t, sk_h, lse.data_ptr(),
            lse.stride(0) if q_heads > 1 else tokens, q_begin, q_end, k_begin, k_end, sequences, tokens, keys, max_q, max_k,
            window, out.data_ptr(), out.stride(0) if kv_heads > 1 else keys, fill, q_heads, kv_heads, head_dim,
            head_dim ** -0.5 if scale is None else scale, softcap or 0.0, _lib.ptr(ws), need)
    return out

"""A KV cache held at a budget by accumulated attention weight, on the GPU.

The reference reads caches that an eviction compacted (attention/gathered.py:39-64, "H2O as KVCache-Factory runs them")
but holds no eviction; this module makes them and decodes over them. :class:`HeavyHitterCache` keeps at most ``budget``
tokens per row and KV head: :func:`evict_prompt` fills it from a prompt and the weight its keys received
(:func:`economize_amd.prompt.attention_mass`), :func:`heavy_hitter_attention` is the decode step, in which the new token
takes the slot of the least weight and every token it attends to gains the weight it gave it.
:meth:`HeavyHitterCache.gathered` hands the kept prompt over as a :class:`~economize_amd.gathered.GatheredKV` instead, for a
decode that evicts nothing more.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _lib
from .decode import sinks_operand
from .errors import ConfigError
from .gathered import GatheredKV
from .prompt import DTYPES, Rows, check_out, operand, row_bounds

__all__ = ["HeavyHitterCache", "evict_prompt", "heavy_hitter_attention"]


@dataclass
class HeavyHitterCache:
    """One layer's cache of at most ``budget`` tokens per row and KV head.

    Attributes:
        keys, values: ``[B, Hkv, budget, D]``, bf16 or fp16.
        score: fp32 ``[B, Hkv, budget]``: the attention weight each slot's token has received so far.
        position: int32 ``[B, Hkv, budget]``: the token of its row that each slot holds.
        count: int32 ``[B, Hkv]``: filled slots (the first ones).
        length: int32 ``[B]``: tokens the row has seen, kept or not.
        recent: The newest tokens, never evicted (the one being decoded included).
        first: The first tokens of a row, never evicted.
    """

    keys: torch.Tensor
    values: torch.Tensor
    score: torch.Tensor
    position: torch.Tensor
    count: torch.Tensor
    length: torch.Tensor
    recent: int
    first: int = 0

    @classmethod
    def empty(cls, batch: int, kv_heads: int, head_dim: int, budget: int, dtype: torch.dtype,
              device: torch.device | str, recent: int, first: int = 0) -> HeavyHitterCache:
        shape = (batch, kv_heads, budget)
        cache = cls(torch.zeros(*shape, head_dim, dtype=dtype, device=device),
                    torch.zeros(*shape, head_dim, dtype=dtype, device=device),
                    torch.zeros(shape, dtype=torch.float32, device=device),
                    torch.zeros(shape, dtype=torch.int32, device=device),
                    torch.zeros(shape[:2], dtype=torch.int32, device=device),
                    torch.zeros(batch, dtype=torch.int32, device=device), recent, first)
        cache.check()
        return cache

    @property
    def budget(self) -> int:
        return self.keys.shape[2]

    def __setattr__(self, name: str, value: object) -> None:
        object.__setattr__(self, name, value)
        object.__setattr__(self, "_checked", False)  # (a field replaced: the next call looks at all of them again)

    def check(self) -> None:
        """Refuses fields that do not fit together, once after any of them was set."""
        if self._checked:
            return
        if self.keys.dim() != 4 or self.keys.dtype not in DTYPES:
            raise ConfigError(f"a heavy-hitter cache holds bf16 or fp16 keys [B, Hkv, budget, D], got {self.keys.dtype} "
                              f"{tuple(self.keys.shape)}")
        batch, heads, budget, dim = shape = tuple(self.keys.shape)
        if 0 in shape:
            raise ConfigError(f"a heavy-hitter cache needs at least one row, head and slot, got {shape}")
        if dim not in (64, 128, 256):
            raise ConfigError(f"a heavy-hitter cache takes head dims 64, 128 and 256, not {dim}")
        device = self.keys.device
        slots, rows = shape[:3], shape[:2]
        for name, t, dtype, want in (("keys", self.keys, self.keys.dtype, shape),
                                     ("values", self.values, self.keys.dtype, shape),
                                     ("score", self.score, torch.float32, slots),
                                     ("position", self.position, torch.int32, slots),
                                     ("count", self.count, torch.int32, rows),
                                     ("length", self.length, torch.int32, (batch,))):
            if t.dtype != dtype or t.shape != want or not t.is_contiguous() or t.device != device:
                raise ConfigError(f"{name} must be contiguous {dtype} {list(want)} on {device}")
        if self.recent < 1 or self.first < 0 or self.recent + self.first > budget:
            raise ConfigError(f"need recent >= 1, first >= 0 and recent + first <= budget, got {self.recent}, {self.first} "
                              f"and {budget}")
        object.__setattr__(self, "_checked", True)

    def reset(self) -> None:
        self.count.zero_()
        self.length.zero_()

    def gathered(self, dropped: int = 0) -> GatheredKV:
        """The kept entries of a prompt (:func:`evict_prompt`'s, before any decode step) as compact entries in front of
        dense slots, which then follow from each row's length on. ``dropped`` is the least number of tokens a row and
        head lost, when the host knows it (0 is always right; it bounds the keys a call walks over)."""
        self.check()
        return GatheredKV(self.keys, self.values, self.position, self.count, self.length, dropped)

    def _pointers(self) -> tuple:
        return (self.keys.data_ptr(), self.values.data_ptr(), self.score.data_ptr(), self.position.data_ptr(),
                self.count.data_ptr(), self.length.data_ptr())


def evict_prompt(cache: HeavyHitterCache, key: torch.Tensor, value: torch.Tensor, mass: torch.Tensor,
                 cu_seqlens: Rows, max_seqlen: int | None = None) -> None:
    """Fill ``cache`` from packed prompts, row ``b`` from sequence ``b`` (what the cache held before is dropped): a row of at
    most ``budget`` tokens is kept whole; of a longer one every KV head keeps the ``first`` tokens, the newest ``recent`` and
    those of greatest mass among the rest (equal masses: the lower index; a NaN is the least), in token order. Their masses
    become the slots' scores. Slots past a row's count are left as they are.

    Args:
        key, value: ``[T, Hkv, D]`` (any strides) in the cache's dtype, in memory apart from the cache's.
        mass: fp32 ``[Hkv, T]`` (:func:`~economize_amd.prompt.attention_mass`).
        cu_seqlens: One sequence per cache row: ``cu_seqlens`` or ``(begin, end)``.
        max_seqlen: The longest sequence.
    """
    cache.check()
    device = _lib.require_gpu(cache.keys, key, value, mass)
    batch, kv_heads, budget, head_dim = cache.keys.shape
    if key.dim() != 3 or tuple(key.shape[1:]) != (kv_heads, head_dim) or value.shape != key.shape:
        raise ConfigError(f"evict_prompt takes keys and values [T, {kv_heads}, {head_dim}], got {tuple(key.shape)} and "
                          f"{tuple(value.shape)}")
    if key.dtype != cache.keys.dtype or value.dtype != cache.keys.dtype:
        raise ConfigError(f"keys {key.dtype} and values {value.dtype} for a cache of {cache.keys.dtype}")
    tokens = key.shape[0]
    if mass.dtype != torch.float32 or tuple(mass.shape) != (kv_heads, tokens) or (tokens > 1 and mass.stride(1) != 1) or \
            (kv_heads > 1 and mass.stride(0) < tokens):
        raise ConfigError(f"mass must be fp32 [{kv_heads}, {tokens}] with contiguous rows apart")
    keep, begin, end, sequences = row_bounds(cu_seqlens, device)
    if sequences != batch:
        raise ConfigError(f"{sequences} sequences for a cache of {batch} rows")
    if tokens == 0:
        return cache.reset()
    key, k_at, sk_t, sk_h = operand(key)
    value, v_at, sv_t, sv_h = operand(value)
    _lib.call_on(device, "eco_evict_prompt", k_at, v_at, sk_t, sk_h, sv_t, sv_h, mass.data_ptr(),
                 mass.stride(0) if kv_heads > 1 else tokens, begin, end, tokens,
                 tokens if max_seqlen is None else min(int(max_seqlen), tokens), *cache._pointers(), batch, kv_heads, budget,
                 head_dim, cache.recent, cache.first)


@functools.lru_cache(maxsize=1024)
def _step_workspace(*sizes: int) -> int:
    return _lib.lib().eco_heavy_hitter_workspace_size(*sizes)


def heavy_hitter_attention(cache: HeavyHitterCache, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                           scale: float | None = None, softcap: float | None = None,
                           sinks: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One decode step of every row. The new token (position ``length``) takes the next free slot or, when all are filled,
    the slot of least score whose token is neither one of the ``first`` nor, counting the new one, of the newest ``recent``
    (equal scores: the lower slot; a NaN is the least). Its query heads attend over the filled slots, and every slot's
    score grows by the weight it received, summed over the heads of its KV head. The cache is updated in place; everything
    stays on the device, so a step can be captured in a graph.

    Args:
        query: ``[B, Hq, D]`` (any strides) in the cache's dtype, at most 64 heads per KV head.
        key, value: ``[B, Hkv, D]``, the new token's.
        scale: Multiplier of the scores, positive (``1 / sqrt(D)``).
        softcap: Optional tanh soft cap of the scaled scores.
        sinks: Optional ``[Hq]`` attention-sink logits.
        out: Optional ``[B, Hq, D]`` output buffer.

    Returns:
        ``[B, Hq, D]`` in the query's dtype.
    """
    cache.check()
    device = _lib.require_gpu(cache.keys, query, key, value)
    batch, kv_heads, budget, head_dim = cache.keys.shape
    if query.dim() != 3 or query.shape[0] != batch or query.shape[2] != head_dim or query.shape[1] == 0:
        raise ConfigError(f"heavy_hitter_attention takes queries [{batch}, Hq, {head_dim}], got {tuple(query.shape)}")
    q_heads = query.shape[1]
    if q_heads % kv_heads:
        raise ConfigError(f"{q_heads} query heads are not a multiple of {kv_heads} KV heads")
    want, dtype = (batch, kv_heads, head_dim), cache.keys.dtype
    if key.shape != want or value.shape != want:
        raise ConfigError(f"the new keys and values must be {list(want)}, got {tuple(key.shape)} and {tuple(value.shape)}")
    if query.dtype != dtype or key.dtype != dtype or value.dtype != dtype:
        raise ConfigError(f"a step of {query.dtype} queries, {key.dtype} keys and {value.dtype} values over a cache of {dtype}")
    if sinks is not None:
        sinks = sinks_operand(sinks, q_heads)
        if sinks.device != device:
            raise ConfigError(f"sinks on {sinks.device}, the queries on {device}")
    if out is None:
        out = torch.empty(batch, q_heads, head_dim, dtype=query.dtype, device=device)
        at, so_b, so_h = out.data_ptr(), q_heads * head_dim, head_dim
    else:
        at, so_b, so_h = check_out(out, query, "[B, Hq, D]")
    query, q_at, sq_b, sq_h = operand(query)
    key, k_at, sk_b, sk_h = operand(key)
    value, v_at, sv_b, sv_h = operand(value)
    need = _step_workspace(batch, q_heads, kv_heads, budget, head_dim)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call_on(device, "eco_heavy_hitter_decode", q_at, _lib.fmt(query.dtype), sq_b, sq_h, k_at, v_at, sk_b, sk_h, sv_b,
                 sv_h, _lib.ptr(sinks), *cache._pointers(), at, so_b, so_h, batch, q_heads, kv_heads, budget, head_dim,
                 cache.recent, cache.first, head_dim ** -0.5 if scale is None else scale, softcap or 0.0, ws.data_ptr(), need)
    return out

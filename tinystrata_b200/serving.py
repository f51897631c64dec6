"""The operators around the expert layer in a serving step, over the C ABI: block tables and slot maps, the paged 8-bit
key / value cache (append, read back, attention) and the gated delta rule.

A step of a hybrid decoder: ``block_tables`` hands the step's tokens their cache slots, an attention layer appends its
keys and values (``kv8_append``) and attends (``kv8_attention``), a recurrent layer runs ``gated_delta`` on its states,
and both feed a ``MoELayer`` / ``PrefillLayer``.

Every call is asynchronous on ``stream`` (default: the current stream of the tensors' device), takes its workspace and new
outputs from torch's allocator for that stream, and raises ``TsbError`` where an argument is refused.  Tensors may be
strided; the innermost dimension must be contiguous.  There is no backward pass: with autograd on, a tensor that requires
gradients is refused, and tensors that a call writes count as changed in place.  The calls go through ``_serving.so``
(csrc/tsb_pyserving.cpp), built beside libtsb_moe.so; without it they raise.
"""
from __future__ import annotations

import os
from typing import NamedTuple

import torch

from . import HERE, TsbError, lib

_ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}   # ggml ids
EXT_PATH = os.path.join(HERE, "_serving.so")
_native = None


def _load():
    """The native module (raises when it has not been built: there is no fallback)."""
    global _native
    if _native is None:
        lib()
        if not os.path.exists(EXT_PATH):
            raise TsbError(f"{EXT_PATH} is missing: run `python -m tinystrata_b200.build` (no fallback)")
        from . import _serving
        _serving.init(TsbError)
        _native = _serving
    return _native


def _on(stream):
    """A stream other than the current one, for the length of a call: its allocations belong to it."""
    return torch.cuda.stream(stream)


# ------------------------------------------------------------------------------------------------ block tables
class BlockPlan(NamedTuple):
    """What ``block_tables`` hands a step: the lengths after it [R] int32, the bounds of the requests' new tokens in
    packed order [R + 1] int32, their slots [cap_tokens] int64 (-1: refused, or past the last), and the free blocks
    left [1] int32."""
    lens: torch.Tensor
    cu: torch.Tensor
    slots: torch.Tensor
    n_free: torch.Tensor


def block_tables(lens, n_new, table, free, n_free, block_size: int, cap_tokens: int, done=None, stream=None) -> BlockPlan:
    """One step of the cache's block allocator (tsb_block_tables): blocks for the step's new tokens off the stack ``free``
    (its first n_free[0] entries), blocks of the requests with ``done`` back onto it, and every new token's slot.

    lens, n_new int32 [R], table int32 [R, W] (rows that do not overlap), free int32 [blocks], n_free int32 [1], done
    uint8 [R] or None.  ``table`` and ``free`` are updated in place."""
    if stream is not None:
        with _on(stream):
            return block_tables(lens, n_new, table, free, n_free, block_size, cap_tokens, done)
    return BlockPlan._make((_native or _load()).block_tables(lens, n_new, table, free, n_free, block_size, cap_tokens, done))


# ------------------------------------------------------------------------------------------------ the 8-bit cache
class KV8Cache:
    """The paged 8-bit key / value cache of one layer: int8 codes k, v [n_blocks, n_kv_heads, block_size, head_dim] and
    fp32 scales k_scale, v_scale [n_blocks, n_kv_heads] (tsb_kv8).  Made empty from sizes, or around existing tensors."""

    def __init__(self, n_blocks: int | None = None, n_kv_heads: int | None = None, head_dim: int | None = None,
                 block_size: int = 16, device="cuda", *, k=None, v=None, k_scale=None, v_scale=None):
        if k is None:
            shape = (n_blocks, n_kv_heads, block_size, head_dim)
            k, v = (torch.zeros(shape, dtype=torch.int8, device=device) for _ in "kv")
            k_scale, v_scale = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in "kv")
        if k.dim() != 4 or k.shape[2] not in (16, 32, 64) or k.shape[3] not in (64, 128, 256):
            raise TsbError(f"KV8Cache: [n_blocks, n_kv_heads, block_size 16 | 32 | 64, head_dim 64 | 128 | 256] wanted, got "
                           f"{tuple(k.shape)}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        kv8_append(self, k.new_empty((0, self.n_kv_heads, self.head_dim), dtype=torch.float32),
                   k.new_empty((0, self.n_kv_heads, self.head_dim), dtype=torch.float32),
                   k.new_empty(0, dtype=torch.int64))             # checks the four tensors

    n_blocks = property(lambda self: self.k.shape[0])
    n_kv_heads = property(lambda self: self.k.shape[1])
    block_size = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])
    # what the calls take: the tensors as they are now
    _pools = property(lambda self: (self.k, self.v, self.k_scale, self.v_scale))


def kv8_append(cache: KV8Cache, k, v, slots, stream=None) -> None:
    """Keys and values [T, n_kv_heads, head_dim] into the cache at slots int64 [T] (tsb_kv8_append); -1 skips a token.
    Tokens of one block follow one another in slots, ascending, with skipped ones in their places."""
    if stream is not None:
        with _on(stream):
            return kv8_append(cache, k, v, slots)
    (_native or _load()).kv8_append(cache._pools, k, v, slots)


def kv8_read(cache: KV8Cache, slots, dtype=torch.float32, stream=None):
    """The cached tokens at slots as (keys, values) [T, n_kv_heads, head_dim] of dtype (tsb_kv8_read)."""
    if stream is not None:
        with _on(stream):
            return kv8_read(cache, slots, dtype)
    if dtype not in _ELEM:
        raise TsbError(f"kv8_read: {dtype} (float32, float16 or bfloat16)")
    return (_native or _load()).kv8_read(cache._pools, slots, _ELEM[dtype])


def kv8_attention(cache: KV8Cache, q, table, lens, cu_q=None, max_q: int | None = None, window: int = 0, scale: float | None = None,
                  out=None, stream=None):
    """Causal attention of each request's last queries over its cached keys and values (tsb_kv8_attention).

    q [T, q_heads, head_dim]; table int32 [R, W] and lens int32 [R] as ``block_tables`` leaves them (the queries' own keys
    appended; requests may share rows of the table, as samples of one prompt do: ``table.expand``); cu_q int32 [R + 1]
    bounds of the requests' rows in q (None: max_q rows each); max_q at least the most rows of a request (default 1, with
    cu_q all rows of q; a close bound is faster; a request with more rows, or longer than its row of the table, is cut and
    recorded in ``device_error()``); window 0 or the number of last keys a query sees; scale default head_dim ** -0.5.
    Returns out, of q's shape and type (its elements share no memory); rows of no request stay as out had them (a new one:
    undefined)."""
    if stream is not None:
        with _on(stream):
            return kv8_attention(cache, q, table, lens, cu_q, max_q, window, scale, out)
    return (_native or _load()).kv8_attention(cache._pools, q, table, lens, cu_q, max_q, window, scale, out)


# ------------------------------------------------------------------------------------------------ gated delta rule
def gated_delta(q, k, v, g, beta, state, cu_seqlens=None, max_len: int | None = None, state_idx=None, state_out=None,
                scale: float | None = None, qk_norm: bool = False, eps: float = 1e-6, out=None, stream=None):
    """The gated delta rule over packed sequences (tsb_gated_delta).

    q, k [T, k_heads, dim_k], v [T, v_heads, dim_v] of one type; g (log decays) and beta fp32 [T, v_heads], their rows of
    one stride; state fp32 [n_states, v_heads, dim_k, dim_v].  cu_seqlens int32 [B + 1] bounds the sequences (None: T / max_len sequences of
    max_len tokens; max_len default T, else at least the longest one).  state_idx int32 [B] names the sequences' states
    (None: in order; negative: from zeros, not kept).  What they ask beyond max_len, T or the states is left out and
    recorded in ``device_error()``; rows of no sequence stay as out had them (a new one: undefined).  The states after the step go to state_out (default: in place; else
    memory of its own), where states that no sequence names stay as they are.  out shares no memory with q and k.
    scale default dim_k ** -0.5; qk_norm divides q and k by sqrt(sum of squares + eps) first.  Returns (out, states)."""
    if stream is not None:
        with _on(stream):
            return gated_delta(q, k, v, g, beta, state, cu_seqlens, max_len, state_idx, state_out, scale, qk_norm, eps, out)
    return (_native or _load()).gated_delta(q, k, v, g, beta, state, cu_seqlens, max_len, state_idx, state_out, scale, qk_norm,
                                            eps, out)

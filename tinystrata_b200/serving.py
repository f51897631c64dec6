"""The operators around the expert layer in a serving step, over the C ABI: block tables and slot maps, the paged 8-bit
key / value cache (append, read back, attention) and the gated delta rule.

A step of a hybrid decoder: ``block_tables`` hands the step's tokens their cache slots, an attention layer appends its
keys and values (``kv8_append``) and attends (``kv8_attention``), a recurrent layer runs ``gated_delta`` on its states,
and both feed a ``MoELayer`` / ``PrefillLayer``.

Every call is asynchronous on ``stream`` (default: the current stream), takes its workspace and new outputs from torch's
allocator for that stream, and raises ``TsbError`` where an argument is refused.  Tensors may be strided; the innermost
dimension must be contiguous.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import DeltaRuleDesc, Kv8, Kv8Attn, TsbError, last_error, lib

_ELEM = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}   # ggml ids
_BLOCK_SIZES = (16, 32, 64)
_DELTA_BYTES, _DELTA_STEP = C.sizeof(DeltaRuleDesc), 16    # up to 16 tokens a sequence: no workspace


def _need(ok: bool, what: str):
    if not ok:
        raise TsbError(what)


def _raw(rc: int, what: str):
    if rc != 0:
        raise TsbError(f"{what}: status {rc}: {last_error()}")


_current_device, _current_raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


class _On:
    """A device and stream that are not the current ones, for the length of a call (its allocations belong to the stream)."""
    __slots__ = ("ctx", "handle")

    def __init__(self, device: int, stream):
        _need(device >= 0, "the tensors must be on a CUDA device")
        stream = torch.cuda.current_stream(device) if stream is None else stream
        _need(stream.device.index == device, "the stream belongs to another device than the tensors")
        self.ctx, self.handle = torch.cuda.stream(stream), stream.cuda_stream

    def __enter__(self):
        self.ctx.__enter__()
        return self.handle

    def __exit__(self, *a):
        self.ctx.__exit__(*a)


def _elsewhere(device: int, stream) -> bool:
    """Whether a call has to leave the current device or stream."""
    return stream is not None or device < 0 or _current_device() != device


def _bad(t, want: str, what: str):
    raise TsbError(f"{what}: {want} wanted, got {tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")


def _flat(t, dtype, n: int, device: int, what: str):
    """At least n contiguous values of dtype on the device."""
    if t.dtype is not dtype or t.get_device() != device or t.dim() != 1 or t.shape[0] < n or (n > 1 and t.stride(0) != 1):
        _bad(t, f"at least {n} contiguous {dtype} on cuda:{device}", what)


def _is(t, dtype, dims: int, device: int, what: str):
    if t.dtype is not dtype or t.get_device() != device or t.dim() != dims:
        _bad(t, f"{dims}-dimensional {dtype} on cuda:{device}", what)


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

    lens, n_new int32 [R], table int32 [R, W], free int32 [blocks], n_free int32 [1], done uint8 [R] or None.  ``table``
    and ``free`` are updated in place."""
    dev = lens.get_device()
    if _elsewhere(dev, stream):
        with _On(dev, stream):
            return block_tables(lens, n_new, table, free, n_free, block_size, cap_tokens, done)
    R = lens.shape[0]
    _flat(lens, torch.int32, R, dev, "block_tables: lens")
    _flat(n_new, torch.int32, R, dev, "block_tables: n_new")
    _is(table, torch.int32, 2, dev, "block_tables: table")
    rows, width = table.shape
    ld, col = table.stride()
    _need(rows >= R and (width <= 1 or col == 1), "block_tables: a contiguous row for every request")
    blocks = free.shape[0]
    _flat(free, torch.int32, blocks, dev, "block_tables: free")
    _flat(n_free, torch.int32, 1, dev, "block_tables: n_free")
    if done is not None:
        _flat(done, torch.uint8, R, dev, "block_tables: done")
    _need(cap_tokens >= 0, "block_tables: cap_tokens")
    ints = lens.new_empty(2 * R + 2)
    slots = torch.empty(cap_tokens, dtype=torch.int64, device=lens.device)
    at = ints.data_ptr()
    _raw(lib().tsb_block_tables(lens.data_ptr(), n_new.data_ptr(), None if done is None else done.data_ptr(), R,
                                table.data_ptr(), ld if rows > 1 else max(ld, width), width, free.data_ptr(), blocks,
                                n_free.data_ptr(), block_size, at, at + 4 * R, slots.data_ptr(), cap_tokens,
                                at + 8 * R + 4, _current_raw_stream(dev)), "block_tables")
    after, cu, left = ints.split_with_sizes((R, R + 1, 1))
    return BlockPlan(after, cu, slots, left)


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
        dev = k.get_device()
        for t, what in ((k, "k"), (v, "v")):
            _is(t, torch.int8, 4, dev, f"KV8Cache: {what}")
            _need(t.is_contiguous() and t.shape == k.shape, f"KV8Cache: {what} contiguous, of k's shape")
        for t, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            _is(t, torch.float32, 2, dev, f"KV8Cache: {what}")
            _need(t.is_contiguous() and t.shape == k.shape[:2], f"KV8Cache: {what} contiguous [n_blocks, n_kv_heads]")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_blocks, self.n_kv_heads, self.block_size, self.head_dim = k.shape
        _need(self.block_size in _BLOCK_SIZES, f"KV8Cache: block_size {self.block_size} (16, 32 or 64)")
        _need(self.head_dim in (64, 128, 256), f"KV8Cache: head_dim {self.head_dim} (64, 128 or 256)")
        self.device = dev
        self._call = None          # (key, descriptor, workspace bytes) of the last attention call's shape
        self._c = Kv8(C.sizeof(Kv8), self.n_blocks, self.block_size, self.n_kv_heads, self.head_dim, k.data_ptr(),
                      v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._ref = C.byref(self._c)


def _rows(t, shape, dtype, dev: int, what: str):
    """The token and head strides of rows of this shape [n, heads, dim]."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape:
        _bad(t, f"{tuple(shape)} {dtype} on cuda:{dev}", what)
    a, b, c = t.stride()
    if c != 1:
        _bad(t, "a contiguous innermost dimension", what)
    return a, b


def _elem(t, what: str) -> int:
    e = _ELEM.get(t.dtype)
    if e is None:
        raise TsbError(f"{what}: {t.dtype} (float32, float16 or bfloat16)")
    return e


def kv8_append(cache: KV8Cache, k, v, slots, stream=None) -> None:
    """Keys and values [T, n_kv_heads, head_dim] into the cache at slots int64 [T] (tsb_kv8_append); -1 skips a token."""
    dev = cache.device
    if _elsewhere(dev, stream):
        with _On(dev, stream):
            return kv8_append(cache, k, v, slots)
    n = k.shape[0]
    e = _elem(k, "kv8_append")
    shape = (n, cache.n_kv_heads, cache.head_dim)
    k0, k1 = _rows(k, shape, k.dtype, dev, "kv8_append: k")
    v0, v1 = _rows(v, shape, k.dtype, dev, "kv8_append: v")
    _flat(slots, torch.int64, n, dev, "kv8_append: slots")
    _raw(lib().tsb_kv8_append(cache._ref, k.data_ptr(), v.data_ptr(), e, k0, k1, v0, v1, slots.data_ptr(), n,
                              _current_raw_stream(dev)), "kv8_append")


def kv8_read(cache: KV8Cache, slots, dtype=torch.float32, stream=None):
    """The cached tokens at slots as (keys, values) [T, n_kv_heads, head_dim] of dtype (tsb_kv8_read)."""
    dev = cache.device
    if _elsewhere(dev, stream):
        with _On(dev, stream):
            return kv8_read(cache, slots, dtype)
    n = slots.shape[0]
    _flat(slots, torch.int64, n, dev, "kv8_read: slots")
    _need(dtype in _ELEM, f"kv8_read: {dtype} (float32, float16 or bfloat16)")
    k = torch.empty((n, cache.n_kv_heads, cache.head_dim), dtype=dtype, device=slots.device)
    v = torch.empty_like(k)
    _raw(lib().tsb_kv8_read(cache._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _ELEM[dtype],
                            _current_raw_stream(dev)), "kv8_read")
    return k, v


def kv8_attention(cache: KV8Cache, q, table, lens, cu_q=None, max_q: int = 1, window: int = 0, scale: float | None = None,
                  out=None, stream=None):
    """Causal attention of each request's last queries over its cached keys and values (tsb_kv8_attention).

    q [T, q_heads, head_dim]; table int32 [R, W] and lens int32 [R] as ``block_tables`` leaves them (the queries' own keys
    appended); cu_q int32 [R + 1] bounds of the requests' rows in q (None: max_q rows each); max_q at least the most rows
    of a request; window 0 or the number of last keys a query sees; scale default head_dim ** -0.5.  Returns out, of q's
    shape and type."""
    dev = cache.device
    if _elsewhere(dev, stream):
        with _On(dev, stream):
            return kv8_attention(cache, q, table, lens, cu_q, max_q, window, scale, out)
    shape = q.shape
    _need(len(shape) == 3 and shape[2] == cache.head_dim, "kv8_attention: q [T, q_heads, head_dim]")
    dtype = q.dtype
    q0, q1 = _rows(q, shape, dtype, dev, "kv8_attention: q")
    _is(table, torch.int32, 2, dev, "kv8_attention: table")
    R, width = table.shape
    ld, col = table.stride()
    _need(width <= 1 or col == 1, "kv8_attention: the table's rows must be contiguous")
    _flat(lens, torch.int32, R, dev, "kv8_attention: lens")
    if cu_q is not None:
        _flat(cu_q, torch.int32, R + 1, dev, "kv8_attention: cu_q")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
        o0, o1 = shape[1] * shape[2], shape[2]
    else:
        o0, o1 = _rows(out, shape, dtype, dev, "kv8_attention: out")
    L = lib()
    key = (shape, dtype, R, width, ld, max_q, window, scale, q0, q1, o0, o1)
    if cache._call is not None and cache._call[0] == key:
        _, ref, need = cache._call
    else:
        d = Kv8Attn(C.sizeof(Kv8Attn), R, shape[1], _elem(q, "kv8_attention"), max_q, width, window,
                    shape[2] ** -0.5 if scale is None else scale, shape[0], q0, q1, o0, o1, ld if R > 1 else max(ld, width))
        ref = C.byref(d)
        need = L.tsb_kv8_attention_workspace_bytes(cache._ref, ref)
        cache._call = (key, ref, need)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _raw(L.tsb_kv8_attention(cache._ref, ref, q.data_ptr(), table.data_ptr(), lens.data_ptr(),
                             None if cu_q is None else cu_q.data_ptr(), out.data_ptr(),
                             None if ws is None else ws.data_ptr(), need, _current_raw_stream(dev)), "kv8_attention")
    return out


# ------------------------------------------------------------------------------------------------ gated delta rule
def gated_delta(q, k, v, g, beta, state, cu_seqlens=None, max_len: int | None = None, state_idx=None, state_out=None,
                scale: float | None = None, qk_norm: bool = False, eps: float = 1e-6, out=None, stream=None):
    """The gated delta rule over packed sequences (tsb_gated_delta).

    q, k [T, k_heads, dim_k], v [T, v_heads, dim_v] of one type; g (log decays) and beta fp32 [T, v_heads]; state fp32
    [n_states, v_heads, dim_k, dim_v].  cu_seqlens int32 [B + 1] bounds the sequences (None: T / max_len sequences of
    max_len tokens; max_len default T, else at least the longest one).  state_idx int32 [B] names the sequences' states
    (None: in order; negative: from zeros, not kept).  The states after the step go to state_out (default: in place).
    scale default dim_k ** -0.5; qk_norm divides q and k by sqrt(sum of squares + eps) first.  Returns (out, states)."""
    dev = q.get_device()
    if _elsewhere(dev, stream):
        with _On(dev, stream):
            return gated_delta(q, k, v, g, beta, state, cu_seqlens, max_len, state_idx, state_out, scale, qk_norm, eps, out)
    e = _elem(q, "gated_delta")
    dtype, shape, vshape = q.dtype, q.shape, v.shape
    _need(len(shape) == 3 and len(vshape) == 3, "gated_delta: q, k [T, k_heads, dim_k], v [T, v_heads, dim_v]")
    n, hk, dk = shape
    _, hv, dv = vshape
    _need(vshape[0] == n, "gated_delta: q and v of as many tokens")
    q0, q1 = _rows(q, shape, dtype, dev, "gated_delta: q")
    k0, k1 = _rows(k, shape, dtype, dev, "gated_delta: k")
    v0, v1 = _rows(v, vshape, dtype, dev, "gated_delta: v")
    gb = g.stride(0)
    for t, what in ((g, "g"), (beta, "beta")):
        if t.dtype is not torch.float32 or t.get_device() != dev or t.shape != (n, hv) or (hv > 1 and t.stride(1) != 1) or \
                t.stride(0) != gb:
            _bad(t, f"float32 {(n, hv)} on cuda:{dev}, rows contiguous and of one stride", f"gated_delta: {what}")
    state_out = state if state_out is None else state_out
    _is(state, torch.float32, 4, dev, "gated_delta: state")
    slots = state.shape[0]
    _need(state.shape[1:] == (hv, dk, dv) and state.is_contiguous(), f"gated_delta: state contiguous [n_states, {hv}, {dk}, {dv}]")
    if state_out is not state:
        _is(state_out, torch.float32, 4, dev, "gated_delta: state_out")
        _need(state_out.shape == state.shape and state_out.is_contiguous(), "gated_delta: state_out as state, contiguous")
    max_len = n if max_len is None else max_len
    if cu_seqlens is not None:
        B = cu_seqlens.shape[0] - 1
        _need(B >= 0, "gated_delta: cu_seqlens")
        _flat(cu_seqlens, torch.int32, B + 1, dev, "gated_delta: cu_seqlens")
    else:
        B = n // max_len if max_len else 0
        _need(B * max_len == n, f"gated_delta: {n} tokens are not sequences of {max_len}")
    if state_idx is not None:
        _flat(state_idx, torch.int32, B, dev, "gated_delta: state_idx")
    else:
        _need(slots >= B, "gated_delta: a state for every sequence")
    if out is None:
        out = torch.empty(vshape, dtype=dtype, device=q.device)
        o0, o1 = hv * dv, dv
    else:
        o0, o1 = _rows(out, vshape, dtype, dev, "gated_delta: out")
    d = DeltaRuleDesc(_DELTA_BYTES, e, B, max_len, hk, hv, dk, dv, slots, 1 if qk_norm else 0,
                      dk ** -0.5 if scale is None else scale, eps, n, q0, q1, k0, k1, v0, v1, o0, o1, gb)
    L = lib()
    ref = C.byref(d)
    need, ws = 0, None
    if max_len > _DELTA_STEP:
        need = L.tsb_gated_delta_workspace_bytes(ref)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _raw(L.tsb_gated_delta(ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                           state.data_ptr(), state_out.data_ptr(), None if state_idx is None else state_idx.data_ptr(),
                           None if cu_seqlens is None else cu_seqlens.data_ptr(), out.data_ptr(),
                           None if ws is None else ws.data_ptr(), need, _current_raw_stream(dev)), "gated_delta")
    return out, state_out

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


def _need(ok: bool, what: str):
    if not ok:
        raise TsbError(what)


def _raw(rc: int, what: str):
    if rc != 0:
        raise TsbError(f"{what}: status {rc}: {last_error()}")


class _On:
    """The device and stream a call runs on: entered only when they are not the current ones already."""
    __slots__ = ("ctx", "handle")

    def __init__(self, device: int, stream):
        _need(device >= 0, "the tensors must be on a CUDA device")
        if stream is None and torch._C._cuda_getDevice() == device:
            self.ctx = None
            self.handle = torch._C._cuda_getCurrentRawStream(device)
        else:
            stream = torch.cuda.current_stream(device) if stream is None else stream
            _need(stream.device.index == device, "the stream belongs to another device than the tensors")
            self.ctx = torch.cuda.stream(stream)
            self.handle = stream.cuda_stream

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()
        return self.handle

    def __exit__(self, *a):
        if self.ctx is not None:
            self.ctx.__exit__(*a)


def _is(t, dtype, dims: int, device: int, what: str):
    if not (t.dtype is dtype and t.dim() == dims and t.get_device() == device):
        raise TsbError(f"{what}: {dims}-dimensional {dtype} on cuda:{device} wanted, got {tuple(t.shape)} {t.dtype} on "
                       f"{t.device}")


def _flat(t, dtype, n: int, device: int, what: str):
    _is(t, dtype, 1, device, what)
    if t.shape[0] < n or (n > 1 and t.stride(0) != 1):
        raise TsbError(f"{what}: at least {n} contiguous values wanted, got {tuple(t.shape)}")


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
    R = lens.shape[0]
    _flat(lens, torch.int32, R, dev, "block_tables: lens")
    _flat(n_new, torch.int32, R, dev, "block_tables: n_new")
    _is(table, torch.int32, 2, dev, "block_tables: table")
    _need(table.shape[0] >= R and (table.shape[1] <= 1 or table.stride(1) == 1), "block_tables: a row for every request")
    _flat(free, torch.int32, free.shape[0], dev, "block_tables: free")
    _flat(n_free, torch.int32, 1, dev, "block_tables: n_free")
    if done is not None:
        _flat(done, torch.uint8, R, dev, "block_tables: done")
    _need(cap_tokens >= 0, "block_tables: cap_tokens")
    with _On(dev, stream) as st:
        ints = torch.empty(2 * R + 2, dtype=torch.int32, device=lens.device)
        slots = torch.empty(cap_tokens, dtype=torch.int64, device=lens.device)
        out = BlockPlan(ints[:R], ints[R:2 * R + 1], slots, ints[2 * R + 1:])
        at = ints.data_ptr()
        _raw(lib().tsb_block_tables(lens.data_ptr(), n_new.data_ptr(), None if done is None else done.data_ptr(), R,
                                    table.data_ptr(), table.stride(0), table.shape[1], free.data_ptr(), free.shape[0],
                                    n_free.data_ptr(), block_size, at, at + 4 * R, slots.data_ptr(), cap_tokens,
                                    at + 4 * (2 * R + 1), st), "block_tables")
    return out


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
        self._c = Kv8(C.sizeof(Kv8), self.n_blocks, self.block_size, self.n_kv_heads, self.head_dim, k.data_ptr(),
                      v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
        self._ref = C.byref(self._c)


def _rows(t, heads: int, dim: int, n: int, dtype, dev: int, what: str):
    """The token and head strides of [n, heads, dim] rows."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != (n, heads, dim):
        raise TsbError(f"{what}: {(n, heads, dim)} {dtype} on cuda:{dev} wanted, got {tuple(t.shape)} {t.dtype} on {t.device}")
    a, b, c = t.stride()
    if c != 1 and dim > 1:
        raise TsbError(f"{what}: the innermost dimension must be contiguous")
    return a, b


def _elem(t, what: str) -> int:
    e = _ELEM.get(t.dtype)
    if e is None:
        raise TsbError(f"{what}: {t.dtype} (float32, float16 or bfloat16)")
    return e


def kv8_append(cache: KV8Cache, k, v, slots, stream=None) -> None:
    """Keys and values [T, n_kv_heads, head_dim] into the cache at slots int64 [T] (tsb_kv8_append); -1 skips a token."""
    dev, n = cache.device, k.shape[0]
    e = _elem(k, "kv8_append")
    ks = _rows(k, cache.n_kv_heads, cache.head_dim, n, k.dtype, dev, "kv8_append: k")
    vs = _rows(v, cache.n_kv_heads, cache.head_dim, n, k.dtype, dev, "kv8_append: v")
    _flat(slots, torch.int64, n, dev, "kv8_append: slots")
    with _On(dev, stream) as st:
        _raw(lib().tsb_kv8_append(cache._ref, k.data_ptr(), v.data_ptr(), e, ks[0], ks[1], vs[0], vs[1],
                                  slots.data_ptr(), n, st), "kv8_append")


def kv8_read(cache: KV8Cache, slots, dtype=torch.float32, stream=None):
    """The cached tokens at slots as (keys, values) [T, n_kv_heads, head_dim] of dtype (tsb_kv8_read)."""
    dev, n = cache.device, slots.shape[0]
    _flat(slots, torch.int64, n, dev, "kv8_read: slots")
    _need(dtype in _ELEM, f"kv8_read: {dtype} (float32, float16 or bfloat16)")
    with _On(dev, stream) as st:
        shape = (n, cache.n_kv_heads, cache.head_dim)
        k = torch.empty(shape, dtype=dtype, device=cache.k.device)
        v = torch.empty(shape, dtype=dtype, device=cache.k.device)
        _raw(lib().tsb_kv8_read(cache._ref, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _ELEM[dtype], st),
             "kv8_read")
    return k, v


def kv8_attention(cache: KV8Cache, q, table, lens, cu_q=None, max_q: int = 1, window: int = 0, scale: float | None = None,
                  out=None, stream=None):
    """Causal attention of each request's last queries over its cached keys and values (tsb_kv8_attention).

    q [T, q_heads, head_dim]; table int32 [R, W] and lens int32 [R] as ``block_tables`` leaves them (the queries' own keys
    appended); cu_q int32 [R + 1] bounds of the requests' rows in q (None: max_q rows each); max_q at least the most rows
    of a request; window 0 or the number of last keys a query sees; scale default head_dim ** -0.5.  Returns out, of q's
    shape and type."""
    dev = cache.device
    n, hq, dim = q.shape
    e = _elem(q, "kv8_attention")
    qs = _rows(q, hq, cache.head_dim, n, q.dtype, dev, "kv8_attention: q")
    _is(table, torch.int32, 2, dev, "kv8_attention: table")
    R, width = table.shape
    _need(width <= 1 or table.stride(1) == 1, "kv8_attention: the table's rows must be contiguous")
    _flat(lens, torch.int32, R, dev, "kv8_attention: lens")
    if cu_q is not None:
        _flat(cu_q, torch.int32, R + 1, dev, "kv8_attention: cu_q")
    with _On(dev, stream) as st:
        if out is None:
            out = torch.empty((n, hq, dim), dtype=q.dtype, device=q.device)
        os = _rows(out, hq, dim, n, q.dtype, dev, "kv8_attention: out")
        d = Kv8Attn(C.sizeof(Kv8Attn), R, hq, e, max_q, width, window, dim ** -0.5 if scale is None else scale, n, qs[0],
                    qs[1], os[0], os[1], table.stride(0))
        L = lib()
        ref = C.byref(d)
        need = L.tsb_kv8_attention_workspace_bytes(cache._ref, ref)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _raw(L.tsb_kv8_attention(cache._ref, ref, q.data_ptr(), table.data_ptr(), lens.data_ptr(),
                                 None if cu_q is None else cu_q.data_ptr(), out.data_ptr(),
                                 None if ws is None else ws.data_ptr(), need, st), "kv8_attention")
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
    e = _elem(q, "gated_delta")
    n, hk, dk = q.shape
    _need(v.dim() == 3, "gated_delta: v [T, v_heads, dim_v]")
    hv, dv = v.shape[1:]
    qs = _rows(q, hk, dk, n, q.dtype, dev, "gated_delta: q")
    ks = _rows(k, hk, dk, n, q.dtype, dev, "gated_delta: k")
    vs = _rows(v, hv, dv, n, q.dtype, dev, "gated_delta: v")
    for t, what in ((g, "g"), (beta, "beta")):
        _is(t, torch.float32, 2, dev, f"gated_delta: {what}")
        _need(t.shape == (n, hv) and (hv == 1 or t.stride(1) == 1) and t.stride(0) == g.stride(0),
              f"gated_delta: {what} [T, v_heads], rows contiguous and of one stride")
    state_out = state if state_out is None else state_out
    for t, what in ((state, "state"), (state_out, "state_out")):
        _is(t, torch.float32, 4, dev, f"gated_delta: {what}")
        _need(t.shape[1:] == (hv, dk, dv) and t.is_contiguous() and t.shape == state.shape,
              f"gated_delta: {what} contiguous [n_states, {hv}, {dk}, {dv}]")
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
        _need(state.shape[0] >= B, "gated_delta: a state for every sequence")
    with _On(dev, stream) as st:
        if out is None:
            out = torch.empty((n, hv, dv), dtype=q.dtype, device=q.device)
        os = _rows(out, hv, dv, n, q.dtype, dev, "gated_delta: out")
        d = DeltaRuleDesc(C.sizeof(DeltaRuleDesc), e, B, max_len, hk, hv, dk, dv, state.shape[0], int(qk_norm),
                          dk ** -0.5 if scale is None else scale, eps, n, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0],
                          os[1], g.stride(0))
        L = lib()
        ref = C.byref(d)
        need = L.tsb_gated_delta_workspace_bytes(ref)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _raw(L.tsb_gated_delta(ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
                               state.data_ptr(), state_out.data_ptr(), None if state_idx is None else state_idx.data_ptr(),
                               None if cu_seqlens is None else cu_seqlens.data_ptr(), out.data_ptr(),
                               None if ws is None else ws.data_ptr(), need, st), "gated_delta")
    return out, state_out

"""The serving-step operators at the edges of what they accept: shared and overlapping rows, windows and lengths near the
ends of 32 bits, values that are not finite, defaults, and arguments that the caller could get wrong unnoticed."""
import numpy as np
import pytest
import torch

from . import serving_ref as R
from .test_gpu_serving import BF16, F16, F32, T, _attend, _cache, _dev, _hold, _keys_v, _near, _rule_inputs, _tables  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ table rows
@pytest.mark.parametrize("n,dtype", [(1, BF16), (1, F32), (40, BF16), (500, BF16), (500, F32)])
def test_attention_shared_table_rows(T, n, dtype):
    """Requests that share a row of the table, all of one (stride 0) or with rows that overlap (a stride below the
    width), give the outputs of the same rows laid out apart."""
    rng = np.random.default_rng(21)
    H, G, D, bs, L = 4, 4, 64, 16, 700
    NB = 64
    c = _cache(T, rng, NB, H, D, bs)
    ids = _dev(rng.permutation(NB), torch.int32)
    lens = _dev([L, L - 3, n], torch.int32)
    q = torch.randn((3 * n, H * G, D), device="cuda").to(dtype)
    for table in (ids[None, :44].expand(3, 44), ids.as_strided((3, 44), (5, 1))):
        apart = table.contiguous()
        assert table.stride(0) < 44 == apart.stride(0)
        got = T.kv8_attention(c, q, table, lens, max_q=n)
        assert torch.equal(got, T.kv8_attention(c, q, apart, lens, max_q=n))
        ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, apart, lens.tolist(), [0, n, 2 * n, 3 * n], D ** -0.5, 0)
        _hold(got, ref, mag, dtype, _keys_v(c, [L]))
    assert T.device_error() == 0


def test_block_tables_refuses_rows_that_share_memory(T):
    one = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    room = torch.full((16,), -1, dtype=torch.int32, device="cuda")
    kw = dict(free=_dev([0, 1, 2, 3], torch.int32), n_free=_dev([4], torch.int32), block_size=16, cap_tokens=3)
    two = dict(lens=_dev([0, 0], torch.int32), n_new=_dev([1, 2], torch.int32), **kw)
    for table in (one.expand(2, 4), room.as_strided((2, 4), (3, 1))):
        with pytest.raises(T.TsbError, match="block_tables: table"):
            T.block_tables(table=table, **two)
    assert (one == -1).all() and (room == -1).all()
    # a single row has no stride to speak of
    p = T.block_tables(lens=_dev([0], torch.int32), n_new=_dev([3], torch.int32), table=room.as_strided((1, 4), (1, 1)), **kw)
    assert p.slots.tolist() == [48, 49, 50] and room[:2].tolist() == [3, -1]


# ------------------------------------------------------------------------------------------------ windows
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 1 << 30, 700])
@pytest.mark.parametrize("queries,lens,H,G,D", [
    ([4, 1, 3], [1, 700, 0], 2, 4, 128),                # few rows: split over CTAs
    ([300, 300, 40], [1, 400, 0], 8, 4, 64)])           # tiles of rows
def test_attention_windows_as_long_as_all_keys(T, dtype, window, queries, lens, H, G, D):
    """A window that no request fills hides nothing, whatever its size, also where a request has more queries than keys
    (its first rows have positions below zero)."""
    _, _, _, wide = _attend(T, np.random.default_rng(22), lens, queries, H, G, D, 16, dtype, window)
    _, _, _, all_of_them = _attend(T, np.random.default_rng(22), lens, queries, H, G, D, 16, dtype, 0)
    assert torch.equal(wide, all_of_them)
    assert T.device_error() == 0


# ------------------------------------------------------------------------------------------------ block tables
def test_block_tables_requests_that_ask_for_too_much(T):
    """Sums of the asked tokens and blocks beyond 32 bits: the requests that ask for them are refused, the others served,
    and no token of the packed rows takes another request's slot."""
    top = 2 ** 31 - 1
    for new, cu, lens in (([top, top, 5], [0, top, top, top], [20, 3, 12]), ([5, top, top], [0, 5, top, top], [25, 3, 7]),
                          ([0, top, 5], [0, 0, top, top], [20, 3, 12]), ([top, 0, 0], [0, top, top, top], [20, 3, 7])):
        table = _dev([[4, 0, -1], [5, -1, -1], [1, -1, -1]], torch.int32)
        p = T.block_tables(_dev([20, 3, 7], torch.int32), _dev(new, torch.int32), table, _dev([2, 3, 9, 9], torch.int32),
                           _dev([2], torch.int32), 16, 8)
        assert p.cu.tolist() == cu and p.lens.tolist() == lens and p.n_free.tolist() == [2]
        first = [4, 5, 6, 7, 8] if new[0] == 5 else []
        assert p.slots.tolist() == first + [-1] * (8 - len(first))
        assert table.tolist() == [[4, 0, -1], [5, -1, -1], [1, -1, -1]]
    # far more requests than blocks: the first in order are served
    n = 4096
    rows = torch.full((n, 4), -1, dtype=torch.int32, device="cuda")
    p = T.block_tables(torch.zeros(n, dtype=torch.int32, device="cuda"), torch.full((n,), 64, dtype=torch.int32, device="cuda"), rows,
                       torch.arange(10, dtype=torch.int32, device="cuda"), _dev([10], torch.int32), 16, n * 64)
    assert p.lens.tolist() == [64, 64] + [0] * (n - 2) and p.n_free.tolist() == [2]
    assert rows[:2].tolist() == [[9, 8, 7, 6], [5, 4, 3, 2]] and (rows[2:] == -1).all()
    assert (p.slots[128:] == -1).all() and p.slots[0].item() == 9 * 16


# ------------------------------------------------------------------------------------------------ outputs
def test_outputs_that_share_memory_are_refused(T):
    """Rows of out that are one another's, and states after that lie across the states before."""
    c = T.KV8Cache(4, 2, 64)
    q, table, lens = torch.zeros((2, 8, 64), device="cuda"), torch.zeros((2, 2), dtype=torch.int32, device="cuda"), _dev([1, 1], torch.int32)
    room = torch.full((2000,), 7.0, device="cuda")
    for out in (room[:512].view(1, 8, 64).expand(2, 8, 64), room[:128].view(2, 1, 64).expand(2, 8, 64),
                room.as_strided((2, 8, 64), (500, 64, 1)), room.as_strided((2, 8, 64), (512, 60, 1))):
        with pytest.raises(T.TsbError, match="kv8_attention: out.*share memory"):
            T.kv8_attention(c, q, table, lens, out=out)
    x, v = torch.zeros((3, 1, 64), device="cuda"), torch.zeros((3, 2, 32), device="cuda")
    g, S = torch.zeros((3, 2), device="cuda"), torch.full((4, 2, 64, 32), 7.0, device="cuda")
    ok = dict(q=x, k=x, v=v, g=g, beta=g, state=S[:3], max_len=1)
    with pytest.raises(T.TsbError, match="gated_delta: out.*share memory"):
        T.gated_delta(**ok, out=room[:64].view(1, 2, 32).expand(3, 2, 32))
    with pytest.raises(T.TsbError, match="gated_delta: state_out"):
        T.gated_delta(**ok, state_out=S[1:])
    assert (room == 7).all() and (S == 7).all()
    # strided outputs of every order are taken
    for out in (room[:1024].view(8, 2, 64).transpose(0, 1), room.as_strided((2, 8, 64), (900, 65, 1)), room[:1024].view(2, 8, 64)):
        out.fill_(7)
        T.kv8_attention(c, q, table, lens, out=out)
        assert (out == 0).all()


# ------------------------------------------------------------------------------------------------ rows of the requests
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("queries,lens,H,G", [([3, 1, 2], [90, 40, 2], 2, 4), ([300, 5, 140], [400, 5, 140], 8, 4)])
def test_attention_every_row_by_default(T, dtype, queries, lens, H, G):
    """Bounds without max_q leave no row out; with too small a max_q the request is cut, which the device error word says."""
    rng = np.random.default_rng(23)
    c, table, q, got = _attend(T, rng, lens, queries, H, G, 64, 16, dtype)
    cu = _dev([0, *np.cumsum(queries).tolist()], torch.int32)
    out = torch.full_like(q, 7.0)
    T.kv8_attention(c, q, table, _dev(lens, torch.int32), cu_q=cu, out=out)
    assert T.device_error() == 0
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, cu.tolist(), 64 ** -0.5, 0)
    _hold(out, ref, mag, dtype, _keys_v(c, lens))
    T.kv8_attention(c, q, table, _dev(lens, torch.int32), cu_q=cu, max_q=max(queries) - 1)
    assert T.device_error() == 0xC0000002
    T.kv8_attention(c, q[:-1], table, _dev(lens, torch.int32), cu_q=cu, max_q=max(queries))
    assert T.device_error() == 0xC0000002
    # rows of no request stay as they are
    few = _dev([0, *np.cumsum(queries).tolist()[:-1], sum(queries[:-1])], torch.int32)
    out.fill_(7)
    T.kv8_attention(c, q, table, _dev(lens, torch.int32), cu_q=few, out=out)
    assert (out[sum(queries[:-1]):] == 7).all() and torch.isfinite(out).all()
    assert T.device_error() == 0


@pytest.mark.parametrize("n,H,dtype", [(1, 2, BF16), (230, 4, BF16), (230, 8, F32)])
def test_attention_says_when_a_length_passes_its_table(T, n, H, dtype):
    """A length beyond the table's columns is cut, with its queries at its end, which the device error word says."""
    rng = np.random.default_rng(27)
    c = _cache(T, rng, 64, H, 64, 16)
    table = _tables(rng, [400, 300], 16, 64)
    q = torch.randn((2 * n, 4 * H, 64), device="cuda").to(dtype)
    for cu in (None, _dev([0, n, 2 * n], torch.int32)):
        kw = dict(cu_q=cu, max_q=n)
        got = T.kv8_attention(c, q, table, _dev([401, 300], torch.int32), **kw)
        assert T.device_error() == 0xC0000003
        assert torch.equal(got, T.kv8_attention(c, q, table, _dev([400, 300], torch.int32), **kw))
        assert T.device_error() == 0


# ------------------------------------------------------------------------------------------------ gated delta rule
# k heads, v heads, dim_k, dim_v, sequences: two warps a unit (64 and 128 wide), and one (many sequences)
RULE_FORMS = [(1, 2, 64, 64, 1), (2, 4, 128, 128, 1), (4, 8, 128, 128, 30)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [5, 17, 64, 65, 200])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv,B", RULE_FORMS)
def test_delta_norm_without_eps(T, dtype, n, Hk, Hv, Dk, Dv, B):
    """qk_norm with eps 0: the tokens that fill up a chunk are no division by zero."""
    rng = np.random.default_rng(31)
    q, k, v, g, beta, S = _rule_inputs(rng, B * n, Hk, Hv, Dk, Dv, dtype, B)
    q, k = (q.float() * 3).to(dtype), (k.float() * 0.1).to(dtype)
    ro, rs = R.gated_delta(q, k, v, g, beta, S, [b * n for b in range(B + 1)], qk_norm=True, eps=0.0)
    o, s = T.gated_delta(q, k, v, g, beta, S, max_len=n, qk_norm=True, eps=0.0)
    _near(o, ro, {F32: 1e-5, BF16: 5e-3}[dtype])
    _near(s, rs, 1e-5)


@pytest.mark.parametrize("n", [9, 16, 17, 64, 200])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv,B", RULE_FORMS)
def test_delta_gate_that_is_not_a_number(T, n, Hk, Hv, Dk, Dv, B):
    """A NaN decay makes its head's state NaN from its token on, in the recurrence and in chunks alike; -inf empties it."""
    rng = np.random.default_rng(32)
    q, k, v, g, beta, S = _rule_inputs(rng, B * n, Hk, Hv, Dk, Dv, F32, B)
    at = (B - 1) * n + n // 2                               # in the last sequence
    g[at, Hv - 1], g[at, 0] = float("nan"), float("-inf")
    ro, rs = R.gated_delta(q, k, v, g, beta, S, [b * n for b in range(B + 1)])
    o, s = T.gated_delta(q, k, v, g, beta, S, max_len=n)
    assert torch.isnan(o[at:, Hv - 1]).all() and torch.isnan(s[B - 1, Hv - 1]).all()
    o, s, ro, rs = o[:, :Hv - 1], s[:, :Hv - 1], ro[:, :Hv - 1], rs[:, :Hv - 1]
    _near(o, ro, 1e-5)
    _near(s, rs, 1e-5)
    assert T.device_error() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [16, 40, 64, 200])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv,B", RULE_FORMS)
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta", "state"])
def test_delta_values_that_are_not_finite(T, what, dtype, n, Hk, Hv, Dk, Dv, B):
    """A token's NaN or infinity reaches what the recurrence says and nothing else: outputs of earlier tokens, other heads,
    other columns (a value's) and other sequences stay as they are."""
    rng = np.random.default_rng(33)
    cu = [b * n for b in range(B + 1)]
    clean = _rule_inputs(rng, B * n, Hk, Hv, Dk, Dv, dtype, B)
    for at, bad in ((0, "nan"), (n // 2 + 3, "inf"), (n - 1, "nan"), (n // 3, "inf" if what in ("g", "beta") else "-inf")):
        q, k, v, g, beta, S = (x.clone() for x in clean)
        t = (B - 1) * n + at
        if what == "state":
            S[B - 1, Hv - 1, Dk // 2, 5] = float(bad)
        elif what in ("g", "beta"):
            (g if what == "g" else beta)[t, Hv - 1] = float(bad)
        else:
            {"q": q, "k": k, "v": v}[what][t, -1, 9] = float(bad)
        ro, rs = R.gated_delta(q, k, v, g, beta, S, cu)
        o, s = T.gated_delta(q, k, v, g, beta, S, max_len=n)
        for got, ref, tol in ((o, ro, {F32: 1e-5, BF16: 5e-3}[dtype]), (s, rs, 1e-5)):
            good = torch.isfinite(ref)
            assert torch.equal(torch.isfinite(got), good), (at, bad)
            _near(got.where(good, 0), ref.where(good, 0), tol)
    assert T.device_error() == 0


@pytest.mark.parametrize("n", [2, 70])
def test_delta_says_what_it_leaves_out(T, n):
    """A state that there is not, a sequence longer than max_len and one that reaches past the rows: left out, and recorded
    in the device error word."""
    rng = np.random.default_rng(34)
    q, k, v, g, beta, S = _rule_inputs(rng, 2 * n, 2, 4, 128, 64, F32, 3)
    kw = dict(q=q, k=k, v=v, g=g, beta=beta)
    cu = [0, n, 2 * n]
    assert T.device_error() == 0
    for idx, error in (([2, 3], 0xD0000002), ([2, 2 ** 31 - 1], 0xD0000002), ([2, -1], 0), ([2, -7], 0)):
        S2 = S.clone()
        o, _ = T.gated_delta(**kw, state=S2, max_len=n, state_idx=_dev(idx, torch.int32))
        assert T.device_error() == error
        ro, rs = R.gated_delta(q, k, v, g, beta, S, cu, [2, -1])
        _near(o, ro, 1e-5)
        _near(S2, rs, 1e-5)
        assert torch.equal(S2[:2], S[:2])
    for bounds, longest, error in (([0, n, 2 * n], n - 1, 0xD0000003), ([0, n, 2 * n + 1], n + 1, 0xD0000003), ([0, n, 2 * n], n + 5, 0),
                                   ([0, n, n], n, 0)):
        T.gated_delta(**kw, state=S.clone(), cu_seqlens=_dev(bounds, torch.int32), max_len=longest)
        assert T.device_error() == error


# ------------------------------------------------------------------------------------------------ threads
def test_calls_of_threads_with_sizes_of_their_own(T):
    """Host threads whose calls ask for different amounts of shared memory (by their requests) at once, then the largest."""
    import threading
    rng = np.random.default_rng(24)
    c = _cache(T, rng, 8, 1, 64, 16)
    errors = []

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    z = torch.zeros(n, dtype=torch.int32, device="cuda")
                    T.block_tables(z, z, torch.zeros((n, 1), dtype=torch.int32, device="cuda"), z[:1], z[:1], 16, 0)
                    m = min(n, 4096)
                    T.kv8_attention(c, torch.zeros((m, 2, 64), device="cuda"), torch.zeros((m, 1), dtype=torch.int32, device="cuda"), z[:m])
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                # noqa: BLE001
            errors.append((n, e))
    threads = [threading.Thread(target=work, args=(n,)) for n in (8192, 4200, 6000, 5000, 4097, 7000, 8000, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    work(8192)
    assert not errors and T.device_error() == 0


# ------------------------------------------------------------------------------------------------ autograd
def test_gradients_are_refused_and_writes_are_seen(T):
    """There is no backward pass: a tensor that requires gradients is refused where they would be recorded, and autograd
    notices that a call wrote a tensor that it had saved."""
    rng = np.random.default_rng(25)
    c = _cache(T, rng, 4, 2, 64, 16)
    slots = _dev([16, 17], torch.int64)
    x, lens, table = torch.randn((2, 2, 64), device="cuda"), _dev([1, 1], torch.int32), _dev([[1], [2]], torch.int32)
    q, k, v, g, beta, S = _rule_inputs(rng, 2, 2, 4, 64, 32, F32, 1)
    rule = dict(q=q, k=k, v=v, g=g, beta=beta, state=S)
    calls = [lambda y: T.kv8_append(c, y, x, slots), lambda y: T.kv8_append(c, x, y, slots), lambda y: T.kv8_attention(c, y, table, lens),
             lambda y: T.kv8_attention(c, x, table, lens, out=y)]
    for call in calls:
        with pytest.raises(T.TsbError, match="no backward pass"):
            call(x.clone().requires_grad_())
        with torch.no_grad():
            call(x.clone().requires_grad_())
        call(x.clone().requires_grad_().detach())
    for name in rule:
        with pytest.raises(T.TsbError, match="no backward pass"):
            T.gated_delta(**dict(rule, **{name: rule[name].clone().requires_grad_()}))
    with torch.no_grad():
        T.gated_delta(**dict(rule, q=q.clone().requires_grad_()))

    def changed(t, call):
        before = t._version
        call()
        return t._version > before
    append = lambda: T.kv8_append(c, x, x, slots)                     # noqa: E731
    assert all(changed(t, append) for t in (c.k, c.v, c.k_scale, c.v_scale))
    out = torch.empty_like(x)
    assert changed(out, lambda: T.kv8_attention(c, x, table, lens, out=out))
    assert not changed(c.k, lambda: T.kv8_attention(c, x, table, lens)) and not changed(x, append)
    after, o = torch.empty_like(S), torch.empty_like(v)
    assert changed(S, lambda: T.gated_delta(**rule)) and changed(o, lambda: T.gated_delta(**rule, out=o))
    assert changed(after, lambda: T.gated_delta(**rule, state_out=after)) and not changed(S, lambda: T.gated_delta(**rule, state_out=after))
    free, n = _dev([0, 1, 2, 3], torch.int32), _dev([4], torch.int32)
    tables = lambda: T.block_tables(lens, _dev([1, 1], torch.int32), table, free, n, 16, 2)  # noqa: E731
    assert changed(table, tables) and changed(free, tables) and not changed(lens, tables)
    w = torch.ones_like(S, requires_grad=True)
    loss = (w * S).sum()                                               # saves S
    T.gated_delta(**rule)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():                                       # tensors without versions
        T.gated_delta(**dict(rule, state=S.clone(), out=torch.empty_like(v)))
        T.kv8_append(T.KV8Cache(2, 2, 64), x, x, slots)
    assert T.device_error() == 0


def test_delta_one_token_has_no_row_stride(T):
    """The strides of a single row are arbitrary: g from a product of its own beside beta from a wider one."""
    rng = np.random.default_rng(35)
    q, k, v, g, beta, S = _rule_inputs(rng, 1, 2, 4, 64, 32, F32, 1)
    ro, rs = R.gated_delta(q, k, v, g, beta, S, [0, 1])
    wide = torch.zeros((1, 9), device="cuda")
    wide[:, 2:6] = beta
    for row in (wide[:, 2:6], beta.as_strided((1, 4), (77, 1)), beta.as_strided((1, 4), (0, 1))):
        o, s = T.gated_delta(q, k, v, g, row, S, state_out=torch.empty_like(S))
        _near(o, ro, 1e-5)
        _near(s, rs, 1e-5)


# ------------------------------------------------------------------------------------------------ waits
def test_short_wait_limits(T):
    """Under the shortest bound a wait may give up, which the device error word says; the context and the next calls are as
    before."""
    rng = np.random.default_rng(26)
    c = _cache(T, rng, 300, 4, 128, 16)
    lens = [2000, 900]
    table, dl = _tables(rng, lens, 16, 300), _dev(lens, torch.int32)
    q = torch.randn((1600, 16, 128), device="cuda").to(BF16)
    x = _rule_inputs(rng, 600, 8, 8, 128, 128, BF16, 1)
    run = lambda: [T.kv8_attention(c, q, table, dl, max_q=800), *T.gated_delta(*x, state_out=torch.empty_like(x[-1]))]  # noqa: E731
    good = run()
    assert T.device_error() == 0
    T.set_wait_limit_ns(100_000)
    try:
        for _ in range(5):
            short = run()
            if T.device_error() == 0:
                assert all(torch.equal(a, b) for a, b in zip(short, good))
    finally:
        T.set_wait_limit_ns(2_000_000_000)
    assert all(torch.equal(a, b) for a, b in zip(run(), good))
    assert T.device_error() == 0

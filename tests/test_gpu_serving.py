"""The serving-step operators on the GPU against plain statements in 64 bits (tests/serving_ref.py).

Tolerances, from the arithmetic of the operators.  Attention: an output is a sum of p v; weights carry 2^-11 (one fp16
value) or 2^-22 (two) and the fp32 scores' error, so |error| <= half an output step + c * sum p |v| with c = 2^-10 for
16-bit outputs and 4e-5 (scores of magnitude 15 to 2^-22, twice) for fp32; fp16's smallest steps add 2^-25 to an fp16
output and 2^-40 of a step's largest weight to each weight, that is 2^-40 * (keys) * (largest |v|).  Gated delta rule: operands of 16 bits
(2^-17 each) through three chained products give states and fp32 outputs within 1e-5 of their norm; fp16 outputs add
their rounding (2^-12), bf16 outputs 2^-9 of each term and their own rounding.  Codes, scales, slots and tables are
equal bit for bit."""
import numpy as np
import pytest
import torch

from . import serving_ref as R

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def T():
    import tinystrata_b200 as T
    assert torch.cuda.is_available()
    return T


def _dev(x, dtype):
    return torch.tensor(x, dtype=dtype, device="cuda")


# ------------------------------------------------------------------------------------------------ block tables
def _table_case(rng, n, bs, width, longest, add, spare, done_share):
    lens = [int(rng.integers(0, longest + 1)) for _ in range(n)]
    new = [int(rng.integers(0, add + 1)) for _ in range(n)]
    done = [int(rng.random() < done_share) for _ in range(n)]
    used = [R.blocks_of(x, bs) for x in lens]
    pool = sum(used) + spare
    perm = rng.permutation(pool).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for r in range(n):
        table[r, :used[r]] = perm[at:at + used[r]]
        at += used[r]
    free = np.full(pool, -7, np.int32)
    free[:spare] = perm[at:]
    return lens, new, done, table, free, spare


@pytest.mark.parametrize("n,bs,longest,add,spare,done_share,cap_more", [
    (1, 16, 0, 1, 1, 0.0, 0), (1, 16, 16, 1, 0, 0.0, 3), (3, 32, 100, 5, 2, 0.4, -1), (8, 16, 60, 1, 50, 0.2, 9),
    (40, 64, 500, 90, 30, 0.3, 0), (700, 16, 300, 40, 900, 0.1, 5), (1025, 16, 40, 3, 100000, 0.0, 1),
    (33, 16, 20, 0, 4, 1.0, 2), (8192, 16, 5, 2, 3000, 0.05, 0)])
def test_block_tables(T, n, bs, longest, add, spare, done_share, cap_more):
    rng = np.random.default_rng(n + spare)
    width = R.blocks_of(longest + add // 2 + 1, bs)          # some requests do not fit their row
    lens, new, done, table, free, spare = _table_case(rng, n, bs, max(width, R.blocks_of(longest, bs)), longest, add, spare,
                                                      done_share)
    cap = max(sum(new) + cap_more, 0)
    ref = R.block_tables(lens, new, table, free, spare, bs, cap, done)
    dt, df = _dev(table, torch.int32), _dev(free, torch.int32)
    wide = torch.full((n, table.shape[1] + 3), -5, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = dt
    for tab in (dt, wide[:, :table.shape[1]]):                # a packed table and a strided one
        fr = df.clone()
        p = T.block_tables(_dev(lens, torch.int32), _dev(new, torch.int32), tab, fr, _dev([spare], torch.int32), bs, cap,
                           done=_dev(done, torch.uint8))
        assert p.lens.tolist() == ref["lens"] and p.cu.tolist() == ref["cu"]
        assert p.slots.tolist() == ref["slots"] and p.n_free.tolist() == [ref["n_free"]]
        assert np.array_equal(tab.cpu().numpy(), ref["table"]) and np.array_equal(fr.cpu().numpy(), ref["free"])
    assert (wide[:, table.shape[1]:] == -5).all()


def test_block_tables_without_requests_and_negative_counts(T):
    p = T.block_tables(_dev([], torch.int32), _dev([], torch.int32), torch.zeros((0, 4), dtype=torch.int32, device="cuda"),
                       _dev([3, 1], torch.int32), _dev([2], torch.int32), 16, 4)
    assert p.cu.tolist() == [0] and p.slots.tolist() == [-1] * 4 and p.n_free.tolist() == [2]
    tab = _dev([[2, -1]], torch.int32)
    p = T.block_tables(_dev([5], torch.int32), _dev([-3], torch.int32), tab, _dev([3, 1], torch.int32),
                       _dev([2], torch.int32), 16, 2)
    assert p.lens.tolist() == [5] and p.cu.tolist() == [0, 0] and p.slots.tolist() == [-1, -1]


# ------------------------------------------------------------------------------------------------ append and read
def _fill(rng, shape, dtype):
    x = rng.normal(size=shape) * np.exp(rng.normal(size=(1,) * (len(shape) - 1) + shape[-1:]))
    return torch.tensor(x, dtype=F32).to(dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bs,H,D,layout", [(16, 2, 256, "packed"), (32, 1, 64, "fused"), (64, 3, 128, "odd"),
                                           (16, 8, 64, "heads_first")])
def test_append_codes_equal(T, dtype, bs, H, D, layout):
    """Appends of one token, of runs inside a block and over blocks, with skipped tokens, bit for bit; strided and
    unaligned rows among them; and the read back."""
    rng = np.random.default_rng(bs + D)
    NB = 7
    cache = T.KV8Cache(NB, H, D, bs)
    cache.k.copy_(torch.tensor(rng.integers(-127, 128, cache.k.shape), dtype=torch.int8))
    cache.v.copy_(torch.tensor(rng.integers(-127, 128, cache.v.shape), dtype=torch.int8))
    cache.k_scale.fill_(0.01), cache.v_scale.fill_(3.0)
    state = {x: (getattr(cache, x).cpu().numpy(), getattr(cache, x + "_scale").cpu().numpy()) for x in "kv"}
    order = [5, 0, 6, 2, 1, 3, 4]
    pos = [bs * b + o for b in order for o in range(bs)]      # the slots of one request's positions
    for lo, hi in [(0, 1), (1, 2), (2, bs - 1), (bs - 1, 2 * bs + 3), (2 * bs + 3, 5 * bs), (5 * bs, 5 * bs + 9)]:
        n = hi - lo
        rows = {x: _fill(rng, (n, H, D), dtype) for x in "kv"}
        if lo == 2:
            rows["k"][0, 0, :] = 0
            rows["v"] *= 0.001                                # the old scale stays
        slots = pos[lo:hi]
        dev = {}
        for x in "kv":
            if layout == "fused":
                big = torch.zeros((n, 3, H, D), dtype=dtype, device="cuda")
                dev[x] = big[:, 1]
            elif layout == "odd":
                big = torch.zeros(n * H * (D + 1) + 1, dtype=dtype, device="cuda")
                dev[x] = big[1:].view(n, H, D + 1)[..., :D]
            elif layout == "heads_first":
                dev[x] = torch.zeros((H, n, D), dtype=dtype, device="cuda").transpose(0, 1)
            else:
                dev[x] = torch.zeros((n, H, D), dtype=dtype, device="cuda")
            dev[x].copy_(rows[x])
        T.kv8_append(cache, dev["k"], dev["v"], _dev(slots, torch.int64))
        for x in "kv":
            R.append(*state[x], rows[x].float().numpy(), slots, bs)
            assert np.array_equal(getattr(cache, x).cpu().numpy(), state[x][0]), (x, lo)
            assert np.array_equal(getattr(cache, x + "_scale").cpu().numpy(), state[x][1]), (x, lo)
    want = _dev([3, -1, 0, 99999, NB * bs - 1], torch.int64)
    for out in (F32, F16, BF16):
        got = T.kv8_read(cache, want, dtype=out)
        for x, y in zip("kv", got):
            codes, scale = (torch.tensor(z) for z in state[x])
            for i, s in enumerate(want.tolist()):
                ref = codes[s // bs, :, s % bs].float() * scale[s // bs][:, None] if 0 <= s < NB * bs else torch.zeros(H, D)
                assert torch.equal(y[i].cpu(), ref.to(out))


def test_append_skips_and_bad_values(T):
    bs, H, D = 16, 2, 64
    cache = T.KV8Cache(3, H, D, bs)
    rng = np.random.default_rng(0)
    k, v = _fill(rng, (5, H, D), F32), _fill(rng, (5, H, D), F32)
    k[1, 0, 3], k[2, 1, 5], v[1, 0, 0], v[2, 0, 1] = float("nan"), float("inf"), float("-inf"), 0.0
    slots = [16, 17, 18, -1, 48]                              # one skipped, one past the cache
    T.kv8_append(cache, k.cuda(), v.cuda(), _dev(slots, torch.int64))
    for x, rows in (("k", k), ("v", v)):
        codes, scale = np.zeros((3, H, bs, D), np.int8), np.zeros((3, H), np.float32)
        R.append(codes, scale, rows.numpy(), slots, bs)
        assert np.array_equal(getattr(cache, x).cpu().numpy(), codes)
        assert np.array_equal(getattr(cache, x + "_scale").cpu().numpy(), scale)
    T.kv8_append(cache, k[:0].cuda(), v[:0].cuda(), _dev([], torch.int64))


# ------------------------------------------------------------------------------------------------ attention
def _cache(T, rng, NB, H, D, bs, scale_spread=0.5):
    c = T.KV8Cache(NB, H, D, bs)
    for x in "kv":
        getattr(c, x).copy_(torch.tensor(np.clip(np.rint(rng.normal(size=c.k.shape) * 40), -127, 127), dtype=torch.int8))
        getattr(c, x + "_scale").copy_(torch.tensor(0.03 * np.exp(scale_spread * rng.normal(size=(NB, H))), dtype=F32))
    return c


def _tables(rng, lens, bs, NB, width=None):
    width = max([R.blocks_of(x, bs) for x in lens] + [1]) if width is None else width
    perm, at = rng.permutation(NB), 0
    t = np.full((len(lens), width), -1, np.int32)
    for r, n in enumerate(lens):
        m = R.blocks_of(n, bs)
        t[r, :m] = perm[at:at + m]
        at += m
    assert at <= NB
    return _dev(t, torch.int32)


def _hold(got, ref, mag, dtype, keys_v):
    step = {BF16: 2.0 ** -8, F16: 2.0 ** -10, F32: 2.0 ** -22}[dtype]
    c = 4e-5 if dtype is F32 else 2.0 ** -10
    least = 2.0 ** -25 if dtype is F16 else 0.0                # half a step of the smallest fp16 numbers
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all()
    worst = (err - (step * ref.abs()).clamp(min=least) - c * mag).max().item() - 2.0 ** -40 * keys_v
    assert worst <= 1e-30, worst


def _keys_v(c, lens):
    """Most keys a row sees times the cache's largest value."""
    return max(lens) * 127 * float(c.v_scale.max())


def _attend(T, rng, lens, queries, H, G, D, bs, dtype, window=0, spare=2, **kw):
    NB = sum(R.blocks_of(x, bs) for x in lens) + spare
    c = _cache(T, rng, NB, H, D, bs)
    table = _tables(rng, lens, bs, NB)
    cu = np.concatenate([[0], np.cumsum(queries)]).tolist()
    q = (torch.tensor(rng.normal(size=(cu[-1], H * G, D)), dtype=F32) * 1.5).to(dtype).cuda()
    got = T.kv8_attention(c, q, table, _dev(lens, torch.int32), cu_q=_dev(cu, torch.int32), max_q=max(queries), window=window,
                          **kw)
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, cu, kw.get("scale", D ** -0.5), window)
    assert got.dtype is dtype
    _hold(got, ref, mag, dtype, _keys_v(c, lens))
    return c, table, q, got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,G,D", [(2, 8, 256), (1, 1, 64), (3, 5, 128), (2, 24, 64), (4, 2, 128)])
@pytest.mark.parametrize("bs", [16, 64])
def test_attention_single_tokens(T, dtype, H, G, D, bs):
    """Lengths of one token, around block and step ends, and long ones, in one batch."""
    rng = np.random.default_rng(H * 100 + G + D)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 200, 1031]
    _attend(T, rng, lens, [1] * len(lens), H, G, D, bs, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("queries,lens,window", [
    ([3, 1, 2, 4], [3, 90, 1, 700], 0),          # a request whose first query has no key before it; queries > keys
    ([4, 4], [2, 40], 0), ([2, 0, 3], [50, 60, 0], 0), ([1, 3, 2], [500, 333, 64], 17), ([1, 1], [4000, 100], 1),
    ([5, 8], [1000, 17], 16)])
@pytest.mark.parametrize("H,G,D", [(2, 4, 64), (1, 8, 256)])
def test_attention_short_steps(T, dtype, queries, lens, window, H, G, D):
    _attend(T, np.random.default_rng(7), lens, queries, H, G, D, 32, dtype, window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("queries,lens,window,H,G,D,bs", [
    ([300], [300], 0, 2, 2, 64, 16), ([129, 70], [500, 70], 0, 1, 4, 128, 32), ([33], [1000], 0, 2, 8, 256, 64),
    ([200], [200], 50, 1, 3, 256, 16), ([100, 17, 1], [90, 400, 333], 0, 2, 6, 128, 16), ([80], [2000], 300, 4, 1, 64, 64),
    ([256], [256], 1, 1, 8, 64, 16)])
def test_attention_prompts(T, dtype, queries, lens, window, H, G, D, bs):
    _attend(T, np.random.default_rng(11), lens, queries, H, G, D, bs, dtype, window)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("queries,lens,window,H,G,D,bs", [
    ([300, 300, 299], [300, 299, 450], 0, 5, 2, 64, 16), ([129, 70, 400], [500, 70, 400], 0, 4, 4, 128, 32),
    ([33, 90], [1000, 80], 0, 10, 8, 256, 64), ([200], [200], 50, 9, 3, 256, 16),
    ([100, 17, 1], [90, 400, 333], 0, 5, 6, 128, 16), ([80], [2000], 300, 40, 1, 64, 64), ([256], [256], 1, 3, 8, 64, 16)])
def test_attention_prompt_tiles(T, dtype, queries, lens, window, H, G, D, bs):
    """Enough heads and requests that every type walks its keys in tiles of rows."""
    _attend(T, np.random.default_rng(13), lens, queries, H, G, D, bs, dtype, window)


@pytest.mark.parametrize("n", [1, 90])
def test_attention_without_cu_and_strided(T, n):
    """Rows from a fused projection, a strided output, a wider table, and no bounds."""
    rng = np.random.default_rng(3)
    H, G, D, bs, lens = 2, 4, 128, 16, [100, 95, 240]
    NB = 40
    c = _cache(T, rng, NB, H, D, bs)
    table = _tables(rng, lens, bs, NB, width=20)[:, :16]
    big = torch.randn((3 * n, H * G + 2 * H, D), device="cuda").to(BF16)
    q = big[:, 1:1 + H * G]
    out = torch.full((3 * n, 2, H * G, D), 7.0, dtype=BF16, device="cuda")
    got = T.kv8_attention(c, q, table, _dev(lens, torch.int32), max_q=n, out=out[:, 1])
    cu = [0, n, 2 * n, 3 * n]
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, cu, D ** -0.5, 0)
    assert got.data_ptr() == out[:, 1].data_ptr() and (out[:, 0] == 7).all()
    _hold(got, ref, mag, BF16, _keys_v(c, lens))
    odd = torch.empty(3 * n * H * G * (D + 1) + 1, dtype=BF16, device="cuda")[1:].view(3 * n, H * G, D + 1)[..., :D]
    odd.copy_(q)                                               # rows on odd element addresses
    assert torch.equal(T.kv8_attention(c, odd, table, _dev(lens, torch.int32), max_q=n), got)


@pytest.mark.parametrize("n", [1, 64])
def test_attention_ids_outside_the_cache_hide_their_keys(T, n):
    rng = np.random.default_rng(5)
    H, G, D, bs, lens = 1, 2, 64, 16, [200, 130]
    NB = 30
    c = _cache(T, rng, NB, H, D, bs)
    table = _tables(rng, lens, bs, NB)
    table[0, 3], table[0, 5], table[0, 12], table[1, :] = -1, NB, 1 << 30, -1     # request 1 sees nothing
    q = torch.randn((2 * n, G, D), device="cuda")
    got = T.kv8_attention(c, q, table, _dev(lens, torch.int32), max_q=n)
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, [0, n, 2 * n], D ** -0.5, 0)
    _hold(got, ref, mag, F32, _keys_v(c, lens))
    assert (got[n:] == 0).all()


def test_attention_scales_far_apart(T):
    """Blocks whose scales differ by factors of a thousand, rows of large and of tiny queries, a zero row."""
    rng = np.random.default_rng(6)
    H, G, D, bs, lens = 2, 4, 128, 16, [500, 77]
    NB = 40
    c = _cache(T, rng, NB, H, D, bs)
    c.v_scale.copy_(torch.tensor(10.0 ** rng.integers(-3, 4, (NB, H)), dtype=F32))
    table = _tables(rng, lens, bs, NB)
    for dtype in (F32, BF16):
        q = torch.randn((2, H * G, D), device="cuda")
        q[0, 0], q[0, 1], q[0, 2], q[1, 3] = 0.0, q[0, 1] * 1e-30, q[0, 2] * 20, q[1, 3] * 1e-3
        q = q.to(dtype)
        got = T.kv8_attention(c, q, table, _dev(lens, torch.int32))
        ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, [0, 1, 2], D ** -0.5, 0)
        _hold(got, ref, 8 * mag, dtype, _keys_v(c, lens))                        # scores of magnitude 300: 20 times the error of 15


def test_attention_past_32_bit_offsets(T):
    """Blocks whose bytes lie past 2^31 and 2^32 of the pool."""
    H, G, D, bs = 2, 4, 128, 16
    NB = (5 << 30) // (H * D * bs)
    k = torch.empty((NB, H, bs, D), dtype=torch.int8, device="cuda")
    s = torch.full((NB, H), 0.02, device="cuda")
    rng = np.random.default_rng(8)
    ids = [NB - 1, 3, NB // 2 + 1, NB - 2, NB // 2 - 1, NB * 9 // 10]
    for b in ids:
        k[b] = torch.tensor(np.clip(np.rint(rng.normal(size=(H, bs, D)) * 40), -127, 127), dtype=torch.int8)
    c = T.KV8Cache(k=k, v=k, k_scale=s, v_scale=s)
    table = _dev([ids], torch.int32)
    for n in (1, 80):
        q = torch.randn((n, H * G, D), device="cuda")
        got = T.kv8_attention(c, q, table, _dev([6 * bs - 3], torch.int32), max_q=n)
        ref, mag = R.attention(k, k, s, s, q, table, [6 * bs - 3], [0, n], D ** -0.5, 0)
        _hold(got, ref, mag, F32, 6 * bs * 127 * 0.02)
    x = torch.randn((3, H, D), device="cuda")
    slots = _dev([(NB - 1) * bs + 13, (NB - 1) * bs + 14, (NB - 1) * bs + 15], torch.int64)
    T.kv8_append(c, x, x, slots)
    back, _ = T.kv8_read(c, slots)
    step = c.k_scale[NB - 1].max().item()
    assert (back - x).abs().max().item() <= 0.51 * step


def test_attention_repeats_and_captures(T):
    """The same bits twice, on another stream, and replayed from a graph after the lengths changed."""
    rng = np.random.default_rng(9)
    H, G, D, bs, lens = 2, 8, 128, 16, [900, 33, 2]
    c, table, q, got = _attend(T, rng, lens, [1, 1, 1], H, G, D, bs, BF16)
    dl = _dev(lens, torch.int32)
    assert torch.equal(T.kv8_attention(c, q, table, dl), got)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = T.kv8_attention(c, q, table, dl, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, got)
    out = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        T.kv8_attention(c, q, table, dl, out=out)
    dl.copy_(_dev([450, 32, 1], torch.int32))
    g.replay()
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, [450, 32, 1], [0, 1, 2, 3], D ** -0.5, 0)
    _hold(out, ref, mag, BF16, _keys_v(c, lens))


# ------------------------------------------------------------------------------------------------ gated delta rule
def _rule_inputs(rng, n, Hk, Hv, Dk, Dv, dtype, states, decay=1.0, correlated=False):
    q, k = (torch.tensor(rng.normal(size=(n, Hk, Dk)), dtype=F32) for _ in "qk")
    if correlated:                                             # neighbouring keys nearly alike: the hard triangle
        k = k[:1] + 0.05 * k
    q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    v = torch.tensor(rng.normal(size=(n, Hv, Dv)), dtype=F32)
    g = -decay * torch.tensor(rng.exponential(size=(n, Hv)) * np.exp(rng.uniform(-5, 0.5, (1, Hv))), dtype=F32)
    beta = torch.sigmoid(torch.tensor(rng.normal(size=(n, Hv)) + (2 if correlated else 0), dtype=F32))
    S = torch.tensor(rng.normal(size=(states, Hv, Dk, Dv)) * 0.1, dtype=F32)
    return [x.cuda() for x in (q.to(dtype), k.to(dtype), v.to(dtype), g, beta, S)]


def _near(got, ref, tol):
    assert torch.isfinite(got).all()
    err = (got.double() - ref).norm().item()
    assert err <= tol * ref.norm().item() + 1e-30, err / max(ref.norm().item(), 1e-30)


TOL = {F32: 1e-5, F16: 4e-4, BF16: 5e-3}


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Hk,Hv,Dk,Dv", [(2, 4, 128, 128), (1, 3, 64, 64), (2, 2, 64, 128), (1, 2, 128, 16), (3, 3, 128, 48)])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [4, 0, 2, 16], [17], [64], [65, 1, 128], [300], [0, 5, 200, 63, 129]])
def test_delta(T, dtype, Hk, Hv, Dk, Dv, lens):
    rng = np.random.default_rng(sum(lens) + Dk)
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, g, beta, S = _rule_inputs(rng, cu[-1], Hk, Hv, Dk, Dv, dtype, len(lens))
    after = torch.full_like(S, 9.0)
    before = S.clone()
    o, s = T.gated_delta(q, k, v, g, beta, S, cu_seqlens=_dev(cu, torch.int32), max_len=max(lens), state_out=after)
    ro, rs = R.gated_delta(q, k, v, g, beta, S, cu)
    assert torch.equal(S, before) and s.data_ptr() == after.data_ptr() and o.dtype is dtype
    _near(o, ro, TOL[dtype])
    _near(after, rs, 1e-5)
    T.gated_delta(q, k, v, g, beta, S, cu_seqlens=_dev(cu, torch.int32), max_len=max(lens))        # in place
    assert torch.equal(S, after)
    assert T.device_error() == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Dk,Dv", [(128, 128), (64, 112)])
def test_delta_many_sequences(T, dtype, Dk, Dv):
    """So many sequences that each unit of columns is one warp's."""
    rng = np.random.default_rng(Dv)
    lens = [int(x) for x in rng.integers(17, 80, 24)] + [0, 1]
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, g, beta, S = _rule_inputs(rng, cu[-1], 4, 8, Dk, Dv, dtype, len(lens))
    ro, rs = R.gated_delta(q, k, v, g, beta, S, cu)
    o, s = T.gated_delta(q, k, v, g, beta, S, cu_seqlens=_dev(cu, torch.int32), max_len=max(lens))
    _near(o, ro, TOL[dtype])
    _near(s, rs, 1e-5)
    assert T.device_error() == 0


@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_norm_states_and_strides(T, n, dtype):
    """Unnormalised q and k with qk_norm, named states with one from zeros, rows of a fused projection, odd addresses."""
    rng = np.random.default_rng(n)
    Hk, Hv, D, B = 2, 4, 128, 3
    q, k, v, g, beta, S = _rule_inputs(rng, B * n, Hk, Hv, D, D, dtype, 5)
    q, k = (q.float() * 3.7).to(dtype), (k.float() * 0.02).to(dtype)
    big = torch.zeros((B * n, 2 * Hk + Hv, D), dtype=dtype, device="cuda")
    big[:, :Hk], big[:, Hk:2 * Hk], big[:, 2 * Hk:] = q, k, v
    gb = torch.zeros((B * n, 2 * Hv), device="cuda")
    gb[:, :Hv], gb[:, Hv:] = g, beta
    idx = [4, -1, 1]
    ro, rs = R.gated_delta(q, k, v, g, beta, S, [0, n, 2 * n, 3 * n], idx, scale=0.3, qk_norm=True)
    S2 = S.clone()
    o, _ = T.gated_delta(big[:, :Hk], big[:, Hk:2 * Hk], big[:, 2 * Hk:], gb[:, :Hv], gb[:, Hv:], S2, max_len=n,
                         state_idx=_dev(idx, torch.int32), scale=0.3, qk_norm=True)
    _near(o, ro, TOL[dtype])
    _near(S2, rs, 1e-5)
    assert torch.equal(S2[[0, 2, 3]], S[[0, 2, 3]])

    def odd(x):
        y = torch.empty(x.shape[0] * x.shape[1] * (D + 1) + 1, dtype=dtype, device="cuda")[1:]
        y = y.view(x.shape[0], x.shape[1], D + 1)[..., :D]
        return y.copy_(x)
    S3 = S.clone()
    o3, _ = T.gated_delta(odd(q), odd(k), odd(v), g, beta, S3, max_len=n, state_idx=_dev(idx, torch.int32), scale=0.3,
                          qk_norm=True, out=odd(v))
    assert torch.equal(o3, o) and torch.equal(S3, S2)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [16, 500])
def test_delta_hard_inputs(T, n, dtype):
    """Keys nearly alike with beta near one; decays that empty the state (log decay -inf among them); no decay at all."""
    rng = np.random.default_rng(2)
    for decay, kill in ((0.0, False), (30.0, False), (0.5, True)):
        q, k, v, g, beta, S = _rule_inputs(rng, n, 1, 3, 128, 64, dtype, 1, decay=decay, correlated=True)
        if kill:
            g[n // 2] = float("-inf")
            g[n // 3] = -500.0
        ro, rs = R.gated_delta(q, k, v, g, beta, S, [0, n])
        o, s = T.gated_delta(q, k, v, g, beta, S)
        _near(o, ro, 4 * TOL[dtype])       # nearly equal keys: (1 + A)^-1 multiplies errors by a few
        _near(s, rs, 4e-5)


def test_delta_prompt_then_tokens(T):
    """A prompt in one call and the same tokens in pieces of every form leave the same state and outputs."""
    rng = np.random.default_rng(4)
    n = 333
    q, k, v, g, beta, S = _rule_inputs(rng, n, 2, 4, 128, 128, F32, 1)
    ro, rs = R.gated_delta(q, k, v, g, beta, S, [0, n])
    got, at = [], 0
    for m in (1, 200, 16, 17, 64, 4, 31):
        o, _ = T.gated_delta(q[at:at + m], k[at:at + m], v[at:at + m], g[at:at + m], beta[at:at + m], S)
        got.append(o)
        at += m
    assert at == n
    _near(torch.cat(got), ro, 1e-5)
    _near(S, rs, 1e-5)


def test_delta_streams_and_graph(T):
    rng = np.random.default_rng(12)
    for n in (2, 130):
        q, k, v, g, beta, S = _rule_inputs(rng, n, 2, 4, 128, 128, BF16, 1)
        out = torch.empty_like(S)
        o, _ = T.gated_delta(q, k, v, g, beta, S, state_out=out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        s2 = torch.empty_like(S)
        o2, _ = T.gated_delta(q, k, v, g, beta, S, state_out=s2, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(o, o2) and torch.equal(out, s2)
        o3, s3 = torch.empty_like(o), torch.empty_like(S)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            T.gated_delta(q, k, v, g, beta, S, state_out=s3, out=o3)
        graph.replay()
        assert torch.equal(o, o3) and torch.equal(out, s3)

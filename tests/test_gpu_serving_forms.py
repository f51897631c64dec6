"""Every kernel form behind the serving-step operators, reached on purpose: the append of prompts, ids outside the cache,
offsets past 32 bits and scales far apart in the split, in the tiles of fp32 rows and in the tiles of 16-bit rows, queries
that are not finite, scales of zero and below; and bounds as close as the arithmetic is.

Bounds.  fp16 outputs of attention: weights are two fp16 values, so an output is off by its own rounding (2^-11 of itself,
at least 2^-25) and by c * sum p |v| with the 4e-5 of fp32 queries (scores) and 2^-26 a key (two products of 16 keys
whose sums are cut to 24 bits).  The rule: operands are pairs of fp16 under row scales, two roundings of 2^-22 and a left-out
product of 2^-22 for each of five products in a row: 15 * 2^-22 = 3.6e-6 of the norm of states and fp32 outputs, four times
that where nearly equal keys multiply errors."""
import numpy as np
import pytest
import torch

from . import serving_ref as R
from .test_gpu_serving import BF16, F16, F32, T, _attend, _cache, _dev, _fill, _hold, _keys_v, _near, _rule_inputs, _tables  # noqa: F401

pytestmark = pytest.mark.gpu

# queries a request and key / value heads for which a type takes each form (heads of a group: 4)
FORMS = [(1, 2, F32), (1, 2, F16), (1, 2, BF16), (3, 2, F32), (3, 2, BF16),        # split over CTAs, 8 and 16 rows
         (230, 8, F32), (230, 4, F16), (230, 4, BF16)]                             # tiles


# ------------------------------------------------------------------------------------------------ append of prompts
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bs,H,D,layout", [(16, 2, 256, "packed"), (32, 1, 64, "fused"), (64, 2, 128, "odd"), (64, 1, 256, "heads_first"),
                                           (16, 3, 64, "odd")])
def test_append_prompts_codes_equal(T, dtype, bs, H, D, layout):
    """More than 1024 tokens in a call: requests that start inside blocks of a few tokens or of nearly all, whole blocks, runs
    over the kernel's shares of bs tokens, single tokens between skipped ones and blocks past the cache; bit for bit."""
    rng = np.random.default_rng(bs + D)
    NB = 1700 // bs + 12
    cache = T.KV8Cache(NB, H, D, bs)
    state = {}
    for x in "kv":
        codes = rng.integers(-127, 128, cache.k.shape).astype(np.int8)
        scale = np.exp(rng.normal(size=(NB, H)) * 2 - 4).astype(np.float32)
        getattr(cache, x).copy_(torch.tensor(codes)), getattr(cache, x + "_scale").copy_(torch.tensor(scale))
        state[x] = codes, scale
    order, at, slots = rng.permutation(NB).tolist(), 0, []
    for start, n in ((3, 401), (0, 17), (bs - 1, 600), (bs // 2, 1), (1, bs - 1), (0, 300), (5, 2 * bs)):
        pos = np.arange(start, start + n)
        blocks = np.array(order[at:at + (start + n - 1) // bs + 1])
        at += len(blocks)
        slots += (blocks[pos // bs] * bs + pos % bs).tolist()
    slots[100:103] = [-1] * 3                                  # cuts a run
    slots[700] = NB * bs + 5
    slots[711:800:2] = [-1] * len(slots[711:800:2])            # many short runs in a share
    n = len(slots)
    assert n > 1100 and at <= NB
    rows, dev = {x: _fill(rng, (n, H, D), dtype) for x in "kv"}, {}
    rows["v"][50:90] *= 1e-4                                   # a block's own scale stays
    rows["k"][950:970] = 0
    if dtype is not F16:
        rows["k"][30, 0, 3], rows["v"][640, H - 1, D - 1] = float("nan"), float("-inf")
    for x in "kv":
        if layout == "fused":
            dev[x] = torch.zeros((n, 3, H, D), dtype=dtype, device="cuda")[:, 1]
        elif layout == "odd":
            dev[x] = torch.zeros(n * H * (D + 1) + 1, dtype=dtype, device="cuda")[1:].view(n, H, D + 1)[..., :D]
        elif layout == "heads_first":
            dev[x] = torch.zeros((H, n, D), dtype=dtype, device="cuda").transpose(0, 1)
        else:
            dev[x] = torch.zeros((n, H, D), dtype=dtype, device="cuda")
        dev[x].copy_(rows[x])
    T.kv8_append(cache, dev["k"], dev["v"], _dev(slots, torch.int64))
    for x in "kv":
        R.append(*state[x], rows[x].float().numpy(), slots, bs)
        assert np.array_equal(getattr(cache, x + "_scale").cpu().numpy(), state[x][1]), x
        assert np.array_equal(getattr(cache, x).cpu().numpy(), state[x][0]), x


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("n,H,dtype", FORMS)
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 32), (256, 64)])
def test_attention_hides_ids_outside_the_cache(T, n, H, dtype, D, bs):
    rng = np.random.default_rng(41)
    lens = [700, 530, 300]
    NB = sum(R.blocks_of(x, bs) for x in lens)
    c = _cache(T, rng, NB, H, D, bs)
    table = _tables(rng, lens, bs, NB)
    table[0, 0], table[0, 3], table[0, 5], table[2, 1], table[1, :] = -1, NB, 1 << 30, -(1 << 31), -5     # request 1 sees nothing
    q = torch.randn((3 * n, 4 * H, D), device="cuda").to(dtype)
    got = T.kv8_attention(c, q, table, _dev(lens, torch.int32), max_q=n)
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, [0, n, 2 * n, 3 * n], D ** -0.5, 0)
    _hold(got, ref, mag, dtype, _keys_v(c, lens))
    assert (got[n:2 * n] == 0).all() and T.device_error() == 0


@pytest.mark.parametrize("n,dtype", [(1, BF16), (200, F16), (200, BF16), (700, F32)])
def test_attention_offsets_past_32_bits(T, n, dtype):
    """Blocks whose bytes lie past 2^31 and 2^32 of the pools, in the split and in both tile forms."""
    H, G, D, bs = 2, 4, 128, 16
    NB = (5 << 30) // (H * D * bs)
    k = torch.empty((NB, H, bs, D), dtype=torch.int8, device="cuda")
    s = torch.full((NB, H), 0.02, device="cuda")
    rng = np.random.default_rng(42)
    ids = [NB - 1, 3, NB // 2 + 1, NB - 2, NB // 2 - 1, NB * 9 // 10] + [NB // 41 * i + 7 for i in range(40)]
    for b in ids:
        k[b] = torch.tensor(np.clip(np.rint(rng.normal(size=(H, bs, D)) * 40), -127, 127), dtype=torch.int8)
    c = T.KV8Cache(k=k, v=k, k_scale=s, v_scale=s)
    table, L = _dev([ids], torch.int32), len(ids) * bs - 3
    q = torch.randn((n, H * G, D), device="cuda").to(dtype)
    got = T.kv8_attention(c, q, table, _dev([L], torch.int32), max_q=n)
    ref, mag = R.attention(k, k, s, s, q, table, [L], [0, n], D ** -0.5, 0)
    _hold(got, ref, mag, dtype, L * 127 * 0.02)


@pytest.mark.parametrize("n,H,dtype", FORMS)
def test_attention_scales_far_apart_in_every_form(T, n, H, dtype):
    """Blocks whose value scales differ by a factor of up to a million, rows of large, tiny and zero queries."""
    rng = np.random.default_rng(43)
    D, bs, lens = 128, 16, [500, 377]
    NB = sum(R.blocks_of(x, bs) for x in lens)
    c = _cache(T, rng, NB, H, D, bs)
    c.v_scale.copy_(torch.tensor(10.0 ** rng.integers(-4, 3, (NB, H)), dtype=F32))
    table = _tables(rng, lens, bs, NB)
    q = torch.randn((2 * n, 4 * H, D), device="cuda")
    q[0, 0], q[n - 1, 1], q[n, 2], q[2 * n - 1, 3] = 0.0, q[n - 1, 1] * (1e-6 if dtype is F16 else 1e-30), q[n, 2] * 20, q[2 * n - 1, 3] * 1e-3
    q = q.to(dtype)
    got = T.kv8_attention(c, q, table, _dev(lens, torch.int32), max_q=n)
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, [0, n, 2 * n], D ** -0.5, 0)
    _hold(got, ref, 8 * mag, dtype, _keys_v(c, lens))                        # scores of magnitude 300: 20 times the error of 15


@pytest.mark.parametrize("n,H,dtype", FORMS)
@pytest.mark.parametrize("scale", [-0.11, 0.0, 1e-30])
def test_attention_scales_of_the_scores(T, n, H, dtype, scale):
    """Below zero (the farthest keys weigh most), zero and next to it (all keys alike)."""
    _attend(T, np.random.default_rng(44), [700, 400], [n, n], H, 4, 64, 16, dtype, scale=scale)


@pytest.mark.parametrize("n,H,dtype", FORMS)
def test_attention_queries_that_are_not_finite(T, n, H, dtype):
    """A row with a NaN or an infinity is NaN, and zero where it sees no key; other rows, its group's too, are as without."""
    rng = np.random.default_rng(45)
    D, bs, lens = 128, 16, [500, 0, 290]
    NB = sum(R.blocks_of(x, bs) for x in lens)
    c = _cache(T, rng, NB, H, D, bs)
    table = _tables(rng, lens, bs, NB)
    q = torch.randn((3 * n, 4 * H, D), device="cuda").to(dtype)
    kw = dict(table=table, lens=_dev(lens, torch.int32), max_q=n)
    clean = T.kv8_attention(c, q, **kw)
    bad = q.clone()
    rows = [(0, 1, "nan"), (n - 1, 4 * H - 1, "inf"), (n, 0, "nan"), (2 * n, 2, "-inf"), (3 * n - 1, 5, "nan")]
    for t, h, x in rows:
        bad[t, h, int(rng.integers(0, D))] = float(x)
    got = T.kv8_attention(c, bad, **kw)
    lost = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for t, h, _ in rows:
        lost[t, h] = True
    assert torch.equal(got[~lost], clean[~lost])
    seen = torch.ones(3 * n, dtype=torch.bool, device="cuda")
    seen[n:2 * n] = False
    assert torch.isnan(got[lost & seen[:, None]]).all() and (got[lost & ~seen[:, None]] == 0).all()
    assert T.device_error() == 0


@pytest.mark.parametrize("n,H,dtype", FORMS)
def test_attention_forms_repeat_and_capture(T, n, H, dtype):
    """The same bits twice, on another stream, and replayed from a graph after lengths and queries changed."""
    rng = np.random.default_rng(47)
    lens, bs = [700, 400], 16
    NB = sum(R.blocks_of(x, bs) for x in lens)
    c = _cache(T, rng, NB, H, 64, bs)
    table, dl, cu = _tables(rng, lens, bs, NB), _dev(lens, torch.int32), _dev([0, n, 2 * n], torch.int32)
    q = torch.randn((2 * n, 4 * H, 64), device="cuda").to(dtype)
    kw = dict(table=table, lens=dl, cu_q=cu, max_q=n)
    good = T.kv8_attention(c, q, **kw)
    assert torch.equal(T.kv8_attention(c, q, **kw), good)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = T.kv8_attention(c, q, **kw, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, good)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.kv8_attention(c, q, **kw, out=out)
    graph.replay()
    assert torch.equal(out, good)
    dl.copy_(_dev([523, 399], torch.int32))
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, T.kv8_attention(c, q, **kw)) and not torch.equal(out, good)
    assert T.device_error() == 0


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,H", [(1, 2), (3, 2), (230, 4)])
def test_attention_fp16_outputs_keep_their_bits(T, n, H, D):
    """fp16 outputs to their own rounding.  Sharp scores: few keys carry a row, so that weights of one fp16 value would show
    (the same statement with such weights breaks the bound)."""
    rng = np.random.default_rng(46)
    bs, lens = 16, [640, 500, 333]
    NB = sum(R.blocks_of(x, bs) for x in lens)
    c = _cache(T, rng, NB, H, D, bs, scale_spread=0.1)
    table = _tables(rng, lens, bs, NB)
    q = (torch.tensor(rng.normal(size=(3 * n, 4 * H, D)), dtype=F32) * 1.5).half().cuda()
    scale = 2 * D ** -0.5
    got = T.kv8_attention(c, q, table, _dev(lens, torch.int32), max_q=n, scale=scale)
    cu = [0, n, 2 * n, 3 * n]
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, table, lens, cu, scale, 0)
    keys = max(lens)

    def over(x):
        least = 2.0 ** -40 * _keys_v(c, lens)
        return ((x.double() - ref).abs() - (2.0 ** -11 * ref.abs()).clamp(min=2.0 ** -25) - (4e-5 + keys * 2.0 ** -26) * mag).max().item() - least
    assert over(got) <= 0
    one = torch.zeros_like(ref)                                # weights rounded to one fp16 value, all else in 64 bits
    for r in range(3):
        L = lens[r]
        ids = table[r, :R.blocks_of(L, bs)].long()
        see = torch.arange(L, device="cuda") <= (L - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(4 * H):
            k, v = ((x[ids, h // 4].double() * y[ids, h // 4].double()[:, None, None]).reshape(-1, D)[:L]
                    for x, y in ((c.k, c.k_scale), (c.v, c.v_scale)))
            x = (q[cu[r]:cu[r + 1], h].double() @ k.T * scale).masked_fill(~see, float("-inf"))
            w = torch.exp(x - x.amax(-1, keepdim=True))
            one[cu[r]:cu[r + 1], h] = (w.float() * 2.0 ** 11).half().double() @ v / 2.0 ** 11 / w.sum(-1, keepdim=True)
    assert over(one.half()) > 0


# ------------------------------------------------------------------------------------------------ gated delta rule
PAIRS = 15 * 2.0 ** -22


@pytest.mark.parametrize("Hk,Hv,Dk,Dv,lens", [(2, 4, 128, 128, [300]), (1, 3, 64, 64, [65, 1, 128]), (2, 4, 128, 48, [0, 5, 200, 63, 129]),
                                              (4, 8, 128, 128, [70, 64, 33] * 8), (4, 8, 64, 112, [70, 64, 33] * 8)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_delta_keeps_22_bits(T, dtype, Hk, Hv, Dk, Dv, lens):
    rng = np.random.default_rng(sum(lens))
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, g, beta, S = _rule_inputs(rng, cu[-1], Hk, Hv, Dk, Dv, dtype, len(lens))
    ro, rs = R.gated_delta(q, k, v, g, beta, S, cu)
    o, s = T.gated_delta(q, k, v, g, beta, S, cu_seqlens=_dev(cu, torch.int32), max_len=max(lens))
    _near(s, rs, PAIRS)
    if dtype is F32:
        _near(o, ro, PAIRS)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_delta_keeps_22_bits_of_hard_inputs(T, dtype):
    rng = np.random.default_rng(2)
    for decay in (0.0, 30.0, 0.5):
        q, k, v, g, beta, S = _rule_inputs(rng, 500, 1, 3, 128, 64, dtype, 1, decay=decay, correlated=True)
        ro, rs = R.gated_delta(q, k, v, g, beta, S, [0, 500])
        o, s = T.gated_delta(q, k, v, g, beta, S)
        _near(s, rs, 4 * PAIRS)
        if dtype is F32:
            _near(o, ro, 4 * PAIRS)

"""Refusals of the serving-step operators on the GPU (by argument, each before a launch), and the example that runs them
together with the MoE layers: its allocator keeps every block once, its mixers agree with the operators' 64-bit statements,
a step's results repeat bit for bit, and a request that finds no blocks keeps its cache and states."""
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


def _i(*v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _refuses(T, f, match, **kw):
    with pytest.raises(T.TsbError, match=match):
        f(**kw)


def test_block_tables_refusals(T):
    ok = dict(lens=_i(3, 0), n_new=_i(1, 2), table=torch.zeros((2, 4), dtype=torch.int32, device="cuda"), free=_i(0, 1, 2, 3),
              n_free=_i(4), block_size=16, cap_tokens=3)
    for name, value in (("lens", _i(3, 0, dtype=torch.int64)), ("lens", _i(3, 0, 0, 0)[::2]), ("n_new", _i(1)), ("n_new", _i(1, 2).cpu()),
                        ("table", ok["table"].t().contiguous().t()), ("table", ok["table"][:1]), ("free", ok["free"].float()),
                        ("free", _i(0, 1, 2, 3)[::2]), ("n_free", _i(4).view(1, 1)), ("block_size", 0), ("cap_tokens", -1),
                        ("done", _i(1, 0)), ("done", _i(1, dtype=torch.uint8))):
        _refuses(T, T.block_tables, "block_tables", **dict(ok, **{name: value}))
    T.block_tables(**ok)


def test_cache_refusals(T):
    shape = (4, 2, 16, 64)
    k, v = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in "kv")
    s = torch.zeros((4, 2), device="cuda")
    for kw in (dict(k=k.float()), dict(v=v[:3]), dict(v=v.cpu()), dict(k_scale=s.half()), dict(v_scale=s[:3]), dict(k_scale=s.t()),
               dict(k=k.transpose(0, 1).contiguous().transpose(0, 1))):
        _refuses(T, T.KV8Cache, "KV8Cache", **dict(dict(k=k, v=v, k_scale=s, v_scale=s.clone()), **kw))
    c = T.KV8Cache(4, 2, 64)
    x = torch.zeros((3, 2, 64), device="cuda")
    ok = dict(cache=c, k=x, v=x, slots=_i(0, 1, 2, dtype=torch.int64))
    for name, value in (("k", x[:2]), ("v", x.half()), ("k", x.double()), ("v", x[:, :1]), ("k", torch.zeros((3, 2, 128), device="cuda")[..., ::2]),
                        ("k", x.cpu()), ("slots", _i(0, 1, 2)), ("slots", _i(0, dtype=torch.int64))):
        _refuses(T, T.kv8_append, "kv8_append", **dict(ok, **{name: value}))
    _refuses(T, T.kv8_read, "kv8_read", cache=c, slots=_i(0))
    _refuses(T, T.kv8_read, "kv8_read", cache=c, slots=_i(0, dtype=torch.int64), dtype=torch.float64)


def test_attention_refusals(T):
    c = T.KV8Cache(4, 2, 64)
    q = torch.zeros((2, 8, 64), device="cuda")
    ok = dict(cache=c, q=q, table=torch.zeros((2, 2), dtype=torch.int32, device="cuda"), lens=_i(1, 1))
    for name, value in (("q", q.double()), ("q", q[:, :7]), ("q", q[..., :32]), ("q", q.cpu()), ("q", torch.zeros((2, 64, 8), device="cuda").mT),
                        ("table", ok["table"].long()), ("table", torch.zeros((3, 2), dtype=torch.int32, device="cuda").t()),
                        ("lens", _i(1)), ("lens", _i(1, 1).float()), ("cu_q", _i(0, 1)), ("cu_q", _i(0, 1, 2, dtype=torch.int64)),
                        ("max_q", 2), ("max_q", -1), ("max_q", 1 << 40), ("window", -1), ("out", q.half()), ("out", q[:1])):
        _refuses(T, T.kv8_attention, "kv8_attention", **dict(ok, **{name: value}))
    T.kv8_attention(**ok)


def test_attention_workspace_refusals(T):
    """The C ABI's own: a split needs its workspace, on 16 bytes and whole."""
    import ctypes as C
    c = T.KV8Cache(4, 2, 64)
    q = torch.zeros((2, 8, 64), device="cuda")
    table, lens = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), _i(1, 1)
    k8 = T.Kv8(C.sizeof(T.Kv8), 4, 16, 2, 64, *(x.data_ptr() for x in (c.k, c.v, c.k_scale, c.v_scale)))
    d = T.Kv8Attn(C.sizeof(T.Kv8Attn), 2, 8, 0, 1, 2, 0, 0.125, 2, 512, 64, 512, 64, 2)
    need = T.lib().tsb_kv8_attention_workspace_bytes(C.byref(k8), C.byref(d))
    assert need > 0
    ws = torch.empty(need + 64, dtype=torch.uint8, device="cuda")

    def call(ptr, size):
        return T.lib().tsb_kv8_attention(C.byref(k8), C.byref(d), q.data_ptr(), table.data_ptr(), lens.data_ptr(), None, q.data_ptr(),
                                         ptr, size, None)
    assert call(None, need) == -5 and call(ws.data_ptr(), need - 1) == -5
    assert call(ws.data_ptr() + 8, need) == -4
    assert T.device_error() == 0


def test_gated_delta_refusals(T):
    q, v = torch.zeros((6, 2, 64), device="cuda"), torch.zeros((6, 4, 32), device="cuda")
    g, S = torch.zeros((6, 4), device="cuda"), torch.zeros((2, 4, 64, 32), device="cuda")
    ok = dict(q=q, k=q, v=v, g=g, beta=g, state=S, max_len=3)
    for name, value in (("q", q.half()), ("q", q.double()), ("k", q[:5]), ("k", torch.zeros((6, 2, 128), device="cuda")[..., ::2]),
                        ("v", v[:, :3]), ("v", v[..., :24]), ("g", g.half()), ("beta", g[:5]), ("beta", torch.zeros((6, 8), device="cuda")[:, :4]),
                        ("g", torch.zeros((4, 6), device="cuda").t()), ("state", S.bfloat16()), ("state", S[:, :3]), ("state", S[:1]),
                        ("state", S.mT.contiguous().mT), ("state_out", S[:1]), ("max_len", 4), ("max_len", -3), ("cu_seqlens", _i()),
                        ("cu_seqlens", _i(0, 6, dtype=torch.int64)), ("state_idx", _i(0)), ("out", v[:5]), ("out", v.half())):
        _refuses(T, T.gated_delta, "gated_delta", **dict(ok, **{name: value}))
    T.gated_delta(**ok)


# ------------------------------------------------------------------------------------------------ the example
@pytest.fixture(scope="module")
def example():
    from examples import serving_step
    return serving_step


def _model(example, **kw):
    return example.HybridDecoder(**dict(dict(n_layers=4, requests=5, max_tokens=512, pool_blocks=40, max_len=320, n_expert=32), **kw))


def _blocks_once(m):
    """Every block is either on the stack or in one row of the table."""
    used = [m.table[r, :-(-int(n) // m.block_size)] for r, n in enumerate(m.lens.tolist())]
    ids = torch.cat(used + [m.free[:int(m.n_free)]])
    assert torch.equal(ids.sort().values, torch.arange(m.free.numel(), dtype=torch.int32, device="cuda"))


def test_example_steps(T, example):
    """Prompts beside single tokens, a request that ends while others go on, one that finds no blocks; twice, bit for bit."""
    def run():
        gen = torch.Generator(device="cuda").manual_seed(5)
        m, outs = _model(example), []
        for counts, done in (([100, 1, 70, 0, 33], None), ([1, 1, 1, 200, 1], None), ([1, 1, 1, 1, 1], None),
                             ([0, 90, 1, 1, 1], [1, 0, 0, 0, 0]), ([300, 1, 1, 1, 1], None), ([1, 0, 1, 1, 1], [0, 1, 0, 0, 0])):
            x = torch.randn((sum(counts), m.cfg["n_embd"]), generator=gen, device="cuda")
            out, plan = m.step(x, _i(*counts), max(counts), None if done is None else _i(*done, dtype=torch.uint8))
            assert torch.isfinite(out).all()
            assert plan.cu.tolist() == np.concatenate([[0], np.cumsum(counts)]).tolist()
            _blocks_once(m)
            outs.append((out, plan.lens))
        assert T.device_error() == 0
        return m, outs
    m, a = run()
    _, b = run()
    assert all(torch.equal(x, y) and torch.equal(n, o) for (x, n), (y, o) in zip(a, b))
    assert [n.tolist() for _, n in a] == [[100, 1, 70, 0, 33], [101, 2, 71, 200, 34], [102, 3, 72, 201, 35], [0, 93, 73, 202, 36],
                                          [0, 94, 74, 203, 37], [1, 0, 75, 204, 38]]


def test_example_mixers(T, example):
    """The mixers' calls, on the strided rows of their fused projections, against the 64-bit statements."""
    m = _model(example, requests=3)
    counts, H = [120, 1, 40], m.cfg["n_embd"]
    x = torch.randn((sum(counts), H), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    h = example.rms(x).bfloat16()
    plan = T.block_tables(m.lens, _i(*counts), m.table, m.free, m.n_free, m.block_size, len(x))
    cu = plan.cu.tolist()
    layer = m.layers[3]
    c = layer["cache"]
    got = m.attend(layer, h, plan, max(counts)).view(len(x), example.Q_HEADS, example.HEAD_DIM)
    q = (h @ layer["inp"]).view(len(x), -1, example.HEAD_DIM)[:, :example.Q_HEADS]
    ref, mag = R.attention(c.k, c.v, c.k_scale, c.v_scale, q, m.table, counts, cu, example.HEAD_DIM ** -0.5, 0)
    # one bf16 step of the result and 2^-10 of the sum of p |v|
    assert ((got.double() - ref).abs() <= 2 ** -8 * ref.abs() + 2 ** -10 * mag).all()
    layer = m.layers[0]
    got = m.recur(layer, h, plan, max(counts), m.order).view(len(x), example.V_HEADS, example.RULE_DIM)
    z = (h @ layer["inp"]).view(len(x), -1, example.RULE_DIM)
    g, beta = (h @ layer["gates"]).float().split(example.V_HEADS, 1)
    K = example.K_HEADS
    ro, rs = R.gated_delta(z[:, :K], z[:, K:2 * K], z[:, 2 * K:], -torch.nn.functional.softplus(g), torch.sigmoid(beta),
                           torch.zeros_like(layer["states"]), cu, qk_norm=True)
    assert (got.double() - ro).norm() <= 5e-3 * ro.norm() and (layer["states"].double() - rs).norm() <= 1e-5 * rs.norm()


def test_example_refused_request_keeps_its_state(T, example):
    m = _model(example, requests=2, pool_blocks=6)
    H = m.cfg["n_embd"]
    m.step(torch.randn((50, H), device="cuda"), _i(30, 20), 30)            # 4 of 6 blocks
    states = [l["states"].clone() for l in m.layers if "states" in l]
    codes = [l["cache"].k.clone() for l in m.layers if "cache" in l]
    _, plan = m.step(torch.randn((90, H), device="cuda"), _i(0, 90), 90)   # needs 5 more
    assert plan.lens.tolist() == [30, 20] and int(m.n_free) == 2 and (plan.slots == -1).all()
    assert all(torch.equal(a, l["states"]) for a, l in zip(states, (l for l in m.layers if "states" in l)))
    assert all(torch.equal(a, l["cache"].k) for a, l in zip(codes, (l for l in m.layers if "cache" in l)))
    assert T.device_error() == 0


def test_example_command(T, example, capsys):
    example.main(["--layers", "4", "--requests", "3", "--prompt", "40", "--steps", "4"])
    assert "3 requests" in capsys.readouterr().out

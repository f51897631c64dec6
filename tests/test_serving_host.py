"""What the serving-step operators refuse, without a GPU: every status below is decided before any CUDA call (fake, never
dereferenced device addresses), and the Python functions raise TsbError before they reach the library."""
import ctypes as C

import pytest
import torch

import tinystrata_b200 as T
from tinystrata_b200 import serving

OK, ARG, UNSUP, CUDA, ALIGN, WS = 0, -1, -2, -3, -4, -5
A = 1 << 20          # a 16-byte aligned fake device address


@pytest.fixture(scope="module", autouse=True)
def built():
    from tinystrata_b200 import build
    build.build()


def cache(**kw):
    c = T.Kv8(C.sizeof(T.Kv8), 8, 16, 2, 128, A, A, A, A)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def tables(lens=A, n_new=A, done=None, n=4, table=A, stride=8, width=8, free=A, cap=16, n_free=A, bs=16, lens_out=2 * A, cu=A,
           slots=A, cap_tokens=4, left=2 * A):
    return T.lib().tsb_block_tables(lens, n_new, done, n, table, stride, width, free, cap, n_free, bs, lens_out, cu, slots,
                                    cap_tokens, left, None)


def test_block_tables_refusals():
    assert tables(n=-1) == ARG and tables(width=-1) == ARG and tables(cap=-1) == ARG
    assert tables(bs=0) == ARG and tables(cap_tokens=-1) == ARG
    assert tables(n=8193) == UNSUP
    for name in ("lens", "n_new", "table", "free", "n_free", "lens_out", "cu", "slots", "left"):
        assert tables(**{name: None}) == ARG, name
    assert tables(stride=7) == ARG
    assert tables(lens_out=A) == ARG and tables(left=A) == ARG        # the inputs are read by every CTA
    assert "lens_out" in T.last_error()


def append(c=None, k=A, v=A, elem=30, slots=A, n=3):
    return T.lib().tsb_kv8_append(C.byref(c or cache()), k, v, elem, 256, 128, 256, 128, slots, n, None)


@pytest.mark.parametrize("field,value,status", [
    ("struct_size", 4, ARG), ("n_blocks", 0, ARG), ("n_kv_heads", 0, ARG), ("k", None, ARG), ("v", None, ARG), ("k_scale", None, ARG),
    ("v_scale", None, ARG), ("block_size", 8, UNSUP), ("block_size", 48, UNSUP), ("head_dim", 96, UNSUP), ("head_dim", 512, UNSUP),
    ("k", A + 8, ALIGN), ("v", A + 1, ALIGN), ("k_scale", A + 2, ALIGN)])
def test_cache_refusals(field, value, status):
    c = cache(**{field: value})
    assert append(c) == status
    assert T.lib().tsb_kv8_read(C.byref(c), A, 3, A, A, 0, None) == status
    assert attend(c) == status
    assert T.lib().tsb_kv8_attention_workspace_bytes(C.byref(c), C.byref(desc())) == 0


def test_append_and_read_refusals():
    assert append(elem=2) == UNSUP and append(n=-1) == ARG and append(n=0) == OK
    assert append(k=None) == ARG and append(v=None) == ARG and append(slots=None) == ARG
    assert append(k=A + 1) == ALIGN and append(v=A + 2, elem=0) == ALIGN
    assert append(cache(n_kv_heads=65536)) == UNSUP and append(n=1 << 40) == UNSUP

    def read(elem=0, n=3, slots=A, k=A, v=A):
        return T.lib().tsb_kv8_read(C.byref(cache()), slots, n, k, v, elem, None)
    assert read(elem=8) == UNSUP and read(n=-1) == ARG and read(n=0) == OK
    assert read(k=None) == ARG and read(v=None) == ARG and read(slots=None) == ARG
    assert read(k=A + 4) == ALIGN and read(n=1 << 40) == UNSUP


def desc(**kw):
    d = T.Kv8Attn(C.sizeof(T.Kv8Attn), 3, 8, 30, 1, 8, 0, 0.1, 3, 1024, 128, 1024, 128, 8)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def attend(c=None, q=A, table=A, lens=A, cu=A, out=A, ws=A, ws_bytes=1 << 30, **kw):
    return T.lib().tsb_kv8_attention(C.byref(c or cache()), C.byref(desc(**kw)), q, table, lens, cu, out, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,status", [
    (dict(struct_size=8), ARG), (dict(elem_type=2), UNSUP), (dict(n_req=-1), ARG), (dict(max_q=-1), ARG), (dict(table_width=-1), ARG),
    (dict(window=-1), ARG), (dict(n_tok=-1), ARG), (dict(n_req=4097), UNSUP), (dict(q_heads=0), ARG), (dict(q_heads=7), ARG),
    (dict(table_width=1 << 28), UNSUP), (dict(max_q=1 << 28), UNSUP)])
def test_attention_refusals(kw, status):
    assert attend(**kw) == status
    assert "kv8_attention" in T.last_error()
    assert T.lib().tsb_kv8_attention_workspace_bytes(C.byref(cache()), C.byref(desc(**kw))) == 0


def rule(q=A, k=A, v=A, g=A, beta=A, s_in=A, s_out=A, idx=A, cu=A, o=A, ws=A, ws_bytes=1 << 40, **kw):
    d = T.DeltaRuleDesc(C.sizeof(T.DeltaRuleDesc), 30, 2, 100, 2, 4, 128, 128, 2, 0, 0.1, 1e-6, 200, 256, 128, 256, 128, 512, 128, 512,
                        128, 4)
    for name, value in kw.items():
        setattr(d, name, value)
    return T.lib().tsb_gated_delta(C.byref(d), q, k, v, g, beta, s_in, s_out, idx, cu, o, ws, ws_bytes, None), d


@pytest.mark.parametrize("kw,status", [
    (dict(struct_size=8), ARG), (dict(elem_type=8), UNSUP), (dict(n_seq=-1), ARG), (dict(max_len=-1), ARG), (dict(n_tok=-1), ARG),
    (dict(n_states=-1), ARG), (dict(k_heads=0), ARG), (dict(k_heads=3), ARG), (dict(dim_k=96), UNSUP), (dict(dim_k=256), UNSUP),
    (dict(dim_v=24), UNSUP), (dict(dim_v=0), UNSUP), (dict(v_heads=0), ARG),
    (dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(g=None), ARG), (dict(beta=None), ARG), (dict(o=None), ARG),
    (dict(s_in=None), ARG), (dict(s_out=None), ARG), (dict(cu=None, n_tok=199), ARG),
    (dict(q=A + 1), ALIGN), (dict(s_in=A + 4), ALIGN), (dict(s_out=A + 8), ALIGN), (dict(ws=None), WS), (dict(ws_bytes=64), WS),
    (dict(ws=A + 4), ALIGN)])
def test_gated_delta_refusals(kw, status):
    got, _ = rule(**kw)
    assert got == status
    assert "gated_delta" in T.last_error()


def test_gated_delta_workspace():
    """None for token steps, the chunks' tiles above, none for a refused description."""
    size = T.lib().tsb_gated_delta_workspace_bytes
    _, d = rule(ws=None)
    assert size(C.byref(d)) > 0
    four = size(C.byref(d))                     # chunks of 64: two sequences of at most 100 tokens have 4
    d.n_tok, d.max_len = 400, 200
    assert size(C.byref(d)) == 2 * four
    d.max_len = 16
    assert size(C.byref(d)) == 0
    d.max_len, d.dim_k = 100, 100
    assert size(C.byref(d)) == 0


def test_python_refuses_cpu_tensors_and_wrong_kinds():
    i32, x = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2, 128)
    with pytest.raises(T.TsbError, match="CUDA"):
        T.block_tables(i32, i32, i32.view(1, 4), i32, i32, 16, 4)
    with pytest.raises(T.TsbError, match="CUDA"):
        T.gated_delta(x, x, x, torch.zeros(4, 2), torch.zeros(4, 2), torch.zeros(1, 2, 128, 128))
    with pytest.raises(T.TsbError, match="CUDA"):
        T.KV8Cache(4, 2, 128, device="cpu")
    with pytest.raises(T.TsbError, match="block_size"):
        T.KV8Cache(4, 2, 128, block_size=24, device="cpu")
    with pytest.raises(T.TsbError, match="head_dim"):
        T.KV8Cache(4, 2, 80, device="cpu")
    with pytest.raises(T.TsbError, match="a tensor wanted"):
        T.block_tables([1], i32, i32, i32, i32, 16, 4)


def test_missing_native_module_fails_loudly(monkeypatch, tmp_path):
    monkeypatch.setattr(serving, "_native", None)
    monkeypatch.setattr(serving, "EXT_PATH", str(tmp_path / "_serving.so"))
    i32 = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(T.TsbError, match="no fallback"):
        T.block_tables(i32, i32, i32.view(1, 4), i32, i32, 16, 4)

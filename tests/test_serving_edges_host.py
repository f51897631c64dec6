"""What the serving-step operators refuse at the edges of their ranges, without a GPU (every status is decided before any
launch), and the host side of their Python functions."""
import ctypes as C

import pytest
import torch

import tinystrata_b200 as T
from tinystrata_b200 import serving

from .test_serving_host import A, ALIGN, ARG, CUDA, UNSUP, WS, attend, built, cache, desc, rule, tables  # noqa: F401


@pytest.mark.parametrize("block", [16, 32, 64])
def test_attention_lengths_near_the_end_of_32_bits(block):
    """A request's positions, and those of the tiles read ahead of its last one, stay below 2^31."""
    c = cache(block_size=block)
    for over in (-1, 64, 512):
        width = (2 ** 31 - over) // block
        assert attend(c, table_width=width, table_stride=width) == UNSUP
        d = desc(table_width=width, table_stride=width)
        assert T.lib().tsb_kv8_attention_workspace_bytes(C.byref(c), C.byref(d)) == 0


def test_cache_calls_see_the_tensors_it_has(monkeypatch):
    """A pool that was assigned anew is the one the calls get, and sizes are the pools'."""
    seen = []

    class Native:
        kv8_append = staticmethod(lambda pools, *a: seen.append(pools))
        kv8_read = staticmethod(lambda pools, *a: seen.append(pools))
        kv8_attention = staticmethod(lambda pools, *a: seen.append(pools))

    monkeypatch.setattr(serving, "_native", Native)
    c = T.KV8Cache(4, 2, 64, device="cpu")
    x, i = torch.zeros((1, 2, 64)), torch.zeros(1, dtype=torch.int64)
    c.k, c.v = (torch.zeros((6, 3, 32, 128), dtype=torch.int8) for _ in "kv")
    c.k_scale, c.v_scale = (torch.zeros((6, 3)) for _ in "kv")
    del seen[:]
    T.kv8_append(c, x, x, i)
    T.kv8_read(c, i)
    T.kv8_attention(c, x, i, i)
    assert len(seen) == 3
    for pools in seen:
        assert all(a is b for a, b in zip(pools, (c.k, c.v, c.k_scale, c.v_scale)))
    assert (c.n_blocks, c.n_kv_heads, c.block_size, c.head_dim) == (6, 3, 32, 128)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are not real")
def test_no_device_is_an_error():
    """A call that cannot reach a device says so, whatever its size."""
    for n in (1, 4, 5000, 8192):
        assert tables(n=n) == CUDA, n
        assert "block_tables" in T.last_error()
    assert attend() == CUDA and attend(n_req=4000, cu=A, n_tok=8000) == CUDA


def test_native_module_is_rebuilt_for_another_torch(monkeypatch, tmp_path):
    """_serving.so is bound to the torch it was built against: another version makes it stale, the same one does not."""
    from tinystrata_b200 import build
    ext, runs = tmp_path / "_serving.so", []

    class Done:
        returncode = 0

    def run(cmd, **kw):
        runs.append(cmd)
        ext.write_bytes(b"")
        return Done

    monkeypatch.setattr(build, "EXT", str(ext))
    monkeypatch.setattr(build, "EXT_FOR", str(tmp_path / "_serving.torch"))
    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_ext()
    build.build_ext()
    assert len(runs) == 1
    monkeypatch.setattr(torch, "__version__", "99.0")
    build.build_ext()
    build.build_ext()
    assert len(runs) == 2
    Done.returncode, Done.stderr = 1, "no"
    monkeypatch.setattr(torch, "__version__", "99.1")
    for _ in range(2):                              # a build that failed is not taken for one
        with pytest.raises(RuntimeError):
            build.build_ext()
    assert len(runs) == 4

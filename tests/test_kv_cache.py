"""The 8-bit paged KV cache without a GPU: the C entry points' refusals, the Python checks, and the
tests' own float64 rounding against torch's."""

import ctypes

import pytest
import torch

import kv_ref
from duplex import _build, _lib


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _lib.load()


P = 1 << 20   # an aligned address that nothing reads: each call below is refused before any launch


def cache(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, weights=P, n_blocks=8, kv_heads=2, block=64, dim=128, format=0)
    return _lib.KVCache(**{**a, **kw})


def batch(**kw):
    a = dict(block_table=P, kv_len=P, cu_rows=P, width=4, batch=2, n_rows=2)
    return _lib.KVBatch(**{**a, **kw})


def attend(lib, c=None, b=None, q=P, act=0, heads=8, qs=1024, hs=128, scale=0.1, window=0, sinks=0, out=P, ws=P, n=1 << 40):
    return lib.duplex_kv_attend(ctypes.byref(c or cache()), ctypes.byref(b or batch()), q, act, heads, qs, hs, scale,
                                window, sinks, out, None, ws, n, None, None)


def append(lib, c=None, b=None, k=P, act=0, s=(256, 128, 256, 128)):
    return lib.duplex_kv_append(ctypes.byref(c or cache()), ctypes.byref(b or batch()), k, P, act, *s, None, None)


def evict(lib, c=None, b=None, dst=P, width=4, keep=100, sinks=4, recent=8, new=P, ws=P, n=1 << 40):
    return lib.duplex_kv_evict(ctypes.byref(c or cache()), ctypes.byref(b or batch()), dst, width, keep, sinks, recent, new,
                               ws, n, None, None)


ARG, ALIGN, DTYPE, WORKSPACE, UNSUPPORTED = 1, 2, 3, 4, 6


@pytest.mark.parametrize("call", [attend, append, evict])
def test_cache_and_batch_are_checked(lib, call):
    for kw, rc in (({"k": None}, ARG), ({"v_scale": None}, ARG), ({"n_blocks": 0}, ARG), ({"kv_heads": 0}, ARG),
                   ({"format": 2}, DTYPE), ({"dim": 96}, UNSUPPORTED), ({"dim": 256}, UNSUPPORTED),
                   ({"block": 8}, UNSUPPORTED), ({"block": 48}, UNSUPPORTED), ({"v": P + 8}, ALIGN)):
        assert call(lib, c=cache(**kw)) == rc, kw
    for kw, rc in (({"block_table": None}, ARG), ({"kv_len": None}, ARG), ({"width": 0}, ARG), ({"batch": 0}, ARG),
                   ({"n_rows": -1}, ARG), ({"cu_rows": None, "n_rows": 3}, ARG), ({"batch": 5000}, UNSUPPORTED),
                   ({"width": 1 << 26}, UNSUPPORTED)):
        assert call(lib, b=batch(**kw)) == rc, kw


def test_attend_refuses(lib):
    assert attend(lib, act=2) == DTYPE
    assert attend(lib, heads=7) == ARG and attend(lib, heads=0) == ARG
    assert attend(lib, window=-1) == ARG and attend(lib, sinks=-1) == ARG
    assert attend(lib, scale=float("nan")) == ARG and attend(lib, scale=float("inf")) == ARG
    assert attend(lib, q=None) == ARG and attend(lib, out=None) == ARG
    assert attend(lib, q=P + 2) == ALIGN and attend(lib, qs=1028) == ALIGN and attend(lib, hs=100) == ALIGN
    assert attend(lib, ws=None) == WORKSPACE and attend(lib, n=1000) == WORKSPACE and attend(lib, ws=P + 4) == ALIGN
    assert attend(lib, b=batch(n_rows=0), q=None) == 0      # nothing to do
    n = ctypes.c_size_t()
    assert lib.duplex_kv_attend_workspace_bytes(ctypes.byref(cache()), ctypes.byref(batch()), 7, ctypes.byref(n)) == ARG


def test_append_refuses(lib):
    assert append(lib, act=2) == DTYPE and append(lib, k=None) == ARG and append(lib, k=P + 8) == ALIGN
    assert append(lib, s=(256, 128, 257, 128)) == ALIGN
    assert append(lib, b=batch(n_rows=0), k=None) == 0


def test_evict_refuses(lib):
    assert evict(lib, c=cache(weights=None)) == ARG and evict(lib, dst=None) == ARG and evict(lib, new=None) == ARG
    assert evict(lib, keep=0) == ARG and evict(lib, sinks=-1) == ARG and evict(lib, recent=97) == ARG
    assert evict(lib, keep=257) == ARG                       # more than dst_table holds
    assert evict(lib, ws=None) == WORKSPACE and evict(lib, n=8) == WORKSPACE


def test_python_checks():
    from duplex.streaming import kv_cache
    with pytest.raises(RuntimeError):
        kv_cache.PackedKVCache(4, 2, fmt="int4", device="cpu")
    with pytest.raises(RuntimeError):
        kv_cache.PackedKVCache(4, 2, head_dim=96, device="cpu")
    c = kv_cache.PackedKVCache(4, 2, device="cpu")
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CPU"):
        c.attend(q, table, n)
    with pytest.raises(RuntimeError, match="track_weights"):
        c.evict(table, n, table, keep=1)
    with pytest.raises(RuntimeError, match="gradients"):
        c.attend(q.requires_grad_(), table, n)


def test_reference_rounding():
    """kv_ref.rounded is torch's conversion to e4m3 over its whole range, ties included."""
    x = torch.cat([torch.linspace(-448, 448, 100_001, dtype=torch.float64), torch.arange(-512, 513) * 2.0 ** -11,
                   torch.arange(-40, 41) * 2.0 ** -10]).float().double()   # both sides round the same number
    assert torch.equal(kv_ref.rounded(x, "e4m3"), x.float().to(torch.float8_e4m3fn).double())
    for fmt in ("e4m3", "int8"):
        for amax in (1e-40, 2.0 ** -126, 1.0, 127.0, 127.5, 448.0, 449.0, 3.3e38):
            s, top = kv_ref.scale_of(torch.tensor([amax], dtype=torch.float64), fmt), kv_ref.TOP[fmt]
            assert amax <= top * s and (s == 2.0 ** -126 or amax > top * s / 2)

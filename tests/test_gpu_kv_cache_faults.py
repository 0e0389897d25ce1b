"""Calls of the 8-bit paged KV cache at the edge of what its documentation allows, each of which once gave a
wrong result or went unreported: against float64 (kv_ref) with test_gpu_kv_cache.py's bars."""

import pytest
import torch

import kv_ref
from test_gpu_kv_cache import TYPES, cache_args, check_attend, make

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ row offsets that fall
@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("rows,cu", [(1100, [0, 1100, 0, 1100, 0]), (1100, [1100, 0, 0, 0, 1100]), (6, [0, 6, 0, 6, 0]),
                                     (6, [0, 2, 1, 6, 6]), (40, [0, 40, 0, 40, 40])])
def test_offsets_that_fall_do_nothing(cuda, rows, cu, track):
    """Reported; outputs, caches and weights stay, and a next call with rising offsets is right."""
    from duplex import _lib
    from duplex.streaming import kv_cache
    lens = [1200, 1150, 40, 300]
    s = make(cuda, 4, [rows, 0, 0, 0], lens, 8, 1, 128, 16, "int8", torch.float16)
    fall = torch.tensor(cu, dtype=torch.int32, device=cuda)
    weights = torch.rand(s["k"].shape[:3], device=cuda) if track else None
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = torch.full((rows, 8, 128), 7.0, dtype=torch.float16, device=cuda), torch.full((rows, 8), 7.0, device=cuda)
    state = [s[n] for n in ("k", "v", "k_scale", "v_scale")] + ([weights] if track else [])
    before = [t.clone() for t in state]
    for call in ("attend", "append"):
        err.zero_()
        if call == "attend":
            kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=fall, weights=weights, out=out, lse=lse, err=err)
        else:
            kv_cache.kv_append(s["q"][:, :1], s["q"][:, 1:2], *cache_args(s), cu_q=fall, weights=weights, err=err)
        assert int(err) == _lib.DEVERR_OFFSETS
        assert bool((out == 7).all()) and bool((lse == 7).all())
        assert all(torch.equal(a, b) for a, b in zip(before, state))
    base = weights.clone() if track else None
    kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], weights=weights, out=out, lse=lse)
    check_attend(s, [rows, 0, 0, 0], lens, 0, 0, out, lse, weights, base)

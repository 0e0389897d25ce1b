"""Host restatements of sizes that the 8-bit KV cache's kernels take from device arrays, against the room that
the host gives them."""

import random

import pytest


def rows_of(cu, b, n_rows):
    """csrc/kv.cuh: kv_seq's rows of sequence b."""
    row0 = min(max(cu[b], 0), n_rows)
    return min(max(cu[b + 1], row0), n_rows) - row0


def pairs(cu, n_rows, group):
    """csrc/kv_prompt.cu: the (sequence, row tile) pairs that the plan lists."""
    return sum(-(-rows_of(cu, b, n_rows) * group // 256) for b in range(len(cu) - 1))


def room(batch, n_rows, group):
    """csrc/kv_prompt.cu: max_pairs."""
    return n_rows * group // 256 + batch


@pytest.mark.parametrize("seed", range(20))
def test_rising_offsets_fit_the_item_list(seed):
    rng = random.Random(seed)
    for _ in range(200):
        batch, n_rows, group = rng.randint(1, 40), rng.randint(1, 5000), rng.choice([1, 3, 8, 16, 300])
        low, high = rng.choice([(0, n_rows), (-50, n_rows + 50)])
        cu = sorted(rng.randint(low, high) for _ in range(batch + 1))
        assert sum(rows_of(cu, b, n_rows) for b in range(batch)) <= n_rows
        assert pairs(cu, n_rows, group) <= room(batch, n_rows, group)


def test_falling_offsets_would_not():
    """Which is why a call whose offsets fall does nothing."""
    n_rows = 8192
    assert pairs([0, n_rows, 0, n_rows], n_rows, 8) == 512 > room(3, n_rows, 8) + 1


def test_attend_launches_refuses():
    import ctypes

    from duplex import _build, _lib
    from test_kv_cache import batch, cache
    _build.build()
    lib, n = _lib.load(), ctypes.c_int32(7)
    call = lambda c, b, heads=8, window=0, sinks=0, to=ctypes.byref(n): lib.duplex_kv_attend_launches(  # noqa: E731
        ctypes.byref(c), ctypes.byref(b), heads, window, sinks, to)
    assert call(cache(k=None), batch()) == 1 and call(cache(dim=96), batch()) == 6 and call(cache(), batch(width=0)) == 1
    assert call(cache(), batch(), heads=7) == 1 and call(cache(), batch(), window=-1) == 1
    assert call(cache(), batch(), sinks=-1) == 1 and call(cache(), batch(), to=None) == 1
    assert call(cache(), batch(n_rows=0)) == 0 and n.value == 0

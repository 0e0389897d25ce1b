"""The 8-bit paged KV cache on the GPU (csrc/kv_cache.cu, csrc/kv_attend.cu) against float64
restatements (tests/kv_ref.py).

Append and eviction are exact: codes, scales, weights and lengths are equal.  Attention's bars:

* a score is a sum of dim products, exact in the tensor cores' fp32 but for its 8 accumulations,
  each off by at most 2 steps of 2^-23 of the running magnitude: ds = 2^-19 sum |q_i k_i| scale;
  two more fp32 roundings of the score itself and exp2's 2^-22 make a probability off by
  dp = ds + 2^-21 + 2^-21 |score|, relative, where |score| <= bulk = max sum |q_i k_i| scale;
* lse: dp, and the roundings of log2 and its product: 2^-21 (1 + |lse|);
* out: each probability is rounded to fp16 (half a step, 2^-11), the sum to fp32 (its n additions
  are in the same 2^-19), the normaliser has dp too: (2^-11 + 2 dp + 2^-19) sum p |v|, and one
  rounding to the output's type, half a step: eps / 2 |out|;
* a token's weight: sum of p, each off by dp and lse's error, and the fp32 additions 2^-19."""

import math

import pytest
import torch

import kv_ref

pytestmark = pytest.mark.gpu

E4M3_NAN = 0x7F


def make(cuda, B, rows, lens, Hq, H, D, P, fmt, dtype, seed=0, spare=0, extra_rows=0, spread=1.0, width=None):
    """A filled cache with shuffled blocks: everything that no token owns is NaN (e4m3) or 127, every
    table entry past a sequence's end is out of range."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    width = width or max(1, max(-(-n // P) for n in lens))
    nb = sum(-(-n // P) for n in lens) + 2 + spare
    order = torch.randperm(nb, generator=g, device=cuda).to(torch.int32)
    table = torch.full((B, width), 1 << 30, dtype=torch.int32, device=cuda)
    at = 0
    codes = {}
    for name in "kv":
        if fmt == "int8":
            codes[name] = torch.randint(-127, 128, (nb, H, P, D), generator=g, device=cuda, dtype=torch.int32).to(torch.int8)
        else:
            x = torch.randn(nb, H, P, D, generator=g, device=cuda) * 60
            codes[name] = x.clamp(-448, 448).to(torch.float8_e4m3fn)
        codes[name + "_scale"] = torch.exp2(torch.randint(-8, -4, (nb, H), generator=g, device=cuda).float()) * spread
    for b, n in enumerate(lens):
        m = -(-n // P)
        table[b, :m] = order[at: at + m]
        at += m
        if n % P:
            blk = int(table[b, n // P])
            for name in "kv":
                codes[name].view(torch.uint8)[blk, :, n % P:] = E4M3_NAN
    for blk in order[at:].tolist():
        for name in "kv":
            codes[name].view(torch.uint8)[blk] = E4M3_NAN
    N = sum(rows) + extra_rows
    # q inside a wider buffer, as the q|k|v projection writes it
    buf = torch.randn(N, (Hq + 2 * H) * D, generator=g, device=cuda).to(dtype)
    q = buf[:, : Hq * D].view(N, Hq, D)
    cu = torch.tensor([0] + torch.tensor(rows).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
    return {**codes, "table": table, "kv_len": torch.tensor(lens, dtype=torch.int32, device=cuda), "cu": cu, "q": q,
            "buf": buf, "free": order[at:]}


def cache_args(s):
    return s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["kv_len"]


def check_attend(s, rows, lens, window, sinks, out, lse, weights=None, base=None, scale=None):
    q = s["q"]
    N = sum(rows)
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    ro, rl, mean, bulk, rw = kv_ref.attend(q, s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], lens, rows, window,
                                           sinks, scale)
    dp = 2.0 ** -19 * bulk + 2.0 ** -21 * (1 + bulk)
    eps = torch.finfo(q.dtype).eps
    tol = (2.0 ** -11 + 2 * dp + 2.0 ** -19)[..., None] * mean + eps / 2 * ro.abs() + 2.0 ** -24
    err = (out.double() - ro)[:N].abs()
    assert bool((err <= tol[:N]).all()), f"out: {float((err / tol[:N]).max())} of the bar"
    empty = rl[:N] == -math.inf
    assert torch.equal(lse[:N] == -math.inf, empty)
    assert bool((out[:N][empty] == 0).all())
    dl = dp + 2.0 ** -21 * (1 + rl.abs())
    le = torch.where(empty, 0.0, (lse[:N].double() - rl[:N]).abs())
    assert bool((le <= dl[:N]).all() or empty.all()), f"lse: {float((le / dl[:N]).nan_to_num().max())}"
    if weights is not None:
        worst = float(torch.where(torch.isfinite(dl[:N]), dp[:N] + dl[:N], 0.0).max()) + 2.0 ** -19
        d = (weights.double() - base.double() - rw).abs()
        wt = worst * rw + 2.0 ** -23 * (base.double().abs() + rw)
        assert bool((d <= wt).all()), f"weights: {float((d / wt.clamp(min=1e-30)).max())}"


CASES = [
    # B, rows, lens, Hq, H, D, P, fmt, dtype, window, sinks
    (1, [1], [1], 32, 4, 128, 64, "e4m3", "bf16", 0, 0),
    (1, [1], [1999], 32, 4, 128, 64, "e4m3", "bf16", 0, 0),
    (1, [1], [20011], 8, 1, 128, 16, "int8", "fp16", 0, 0),              # many pieces of one row tile
    (3, [1, 1, 1], [17, 400, 63], 4, 4, 64, 16, "e4m3", "fp16", 0, 0),   # one query head each
    (2, [1, 1], [129, 64], 32, 2, 128, 128, "int8", "bf16", 0, 0),       # 16 query heads: two column tiles
    (4, [3, 0, 5, 1], [3, 50, 700, 0], 12, 2, 64, 32, "e4m3", "bf16", 0, 0),   # empty rows, no rows, no tokens
    (2, [7, 2], [4, 2], 6, 1, 128, 16, "e4m3", "fp16", 0, 0),            # more rows than tokens
    (2, [33, 40], [300, 41], 8, 2, 128, 32, "int8", "bf16", 0, 0),
    (1, [1], [5000], 32, 4, 128, 64, "e4m3", "bf16", 100, 4),
    (3, [1, 2, 6], [1000, 63, 9000], 16, 2, 64, 64, "int8", "fp16", 130, 65),
    (2, [70, 10], [500, 2000], 8, 1, 128, 16, "e4m3", "bf16", 1, 0),     # each row sees itself alone
    (2, [40, 90], [4000, 95], 4, 1, 64, 128, "e4m3", "fp16", 257, 3),
    (1, [1], [700], 8, 8, 128, 64, "e4m3", "bf16", 1 << 30, 1 << 30),    # a window of everything
    (64, [1] * 64, [1 + 37 * i % 900 for i in range(64)], 8, 2, 64, 16, "e4m3", "bf16", 0, 0),
    (3, [700, 129, 300], [700, 1500, 333], 16, 2, 128, 64, "e4m3", "bf16", 0, 0),     # prompts
    (2, [260, 515], [1300, 515], 12, 4, 64, 32, "int8", "fp16", 200, 20),
    (1, [1030], [2100], 4, 4, 128, 128, "int8", "bf16", 0, 0),
    (2, [500, 3], [20, 3], 8, 1, 64, 16, "e4m3", "bf16", 30, 5),          # ... and a window
    # prompts long enough for the tensor-core kernel whatever the window
    (2, [1500, 900], [3000, 900], 12, 4, 64, 32, "int8", "fp16", 200, 20),
    (1, [3000], [3100], 8, 1, 128, 16, "e4m3", "bf16", 1, 0),             # each row sees itself alone
    (2, [1300, 1], [5000, 700], 8, 1, 128, 128, "e4m3", "bf16", 300, 150),
    (2, [2000, 1700], [1500, 1700], 4, 1, 64, 64, "e4m3", "fp16", 0, 0),  # more rows than tokens
    (4, [2500, 0, 5, 1], [2600, 700, 0, 1], 16, 2, 128, 16, "int8", "bf16", 0, 0),
    (1, [1537], [1537], 6, 2, 128, 32, "e4m3", "fp16", 1000, 4),
    (2, [2500, 1700], [700, 1700], 8, 1, 128, 64, "e4m3", "bf16", 900, 20),   # rows before token 0, a window, sinks
]
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}-{c[3]}x{c[4]}x{c[5]}-p{c[6]}-{c[7]}-w{c[9]}-{max(c[1])}of{max(c[2])}")
def test_attend(cuda, case, track):
    from duplex import _lib
    from duplex.streaming import kv_cache
    B, rows, lens, Hq, H, D, P, fmt, dt, window, sinks = case
    s = make(cuda, B, rows, lens, Hq, H, D, P, fmt, TYPES[dt], extra_rows=2)
    if window and max(lens) > window + sinks + P:   # blocks that no row sees: their ids are not looked at
        for b, (t, n) in enumerate(zip(rows, lens)):
            a, z = -(-sinks // P), (n - t - window + 1) // P
            if t and a < z:
                s["table"][b, a:z] = -5
    weights = torch.rand(s["k"].shape[:3], device=cuda) if track else None
    base = weights.clone() if track else None
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out = torch.full((sum(rows) + 2, Hq, D), 7.0, dtype=TYPES[dt], device=cuda)
    lse = torch.full((sum(rows) + 2, Hq), 7.0, device=cuda)
    kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=sinks, weights=weights, out=out, lse=lse,
                       err=err)
    assert int(err) == 0
    check_attend(s, rows, lens, window, sinks, out, lse, weights, base)
    assert bool((out[sum(rows):] == 7).all()) and bool((lse[sum(rows):] == 7).all())   # rows of no sequence
    again, lse2 = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=sinks, return_lse=True)
    n = sum(rows)
    assert torch.equal(again[:n], out[:n]) and torch.equal(lse2[:n], lse[:n])           # the same bits on each run
    _lib.check(0, "")


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 300.0])
def test_attend_extreme_sizes(cuda, dt, size):
    """Small and large query rows, block scales far apart: scores stay right whatever the factors."""
    from duplex.streaming import kv_cache
    if dt == "fp16" and size < 1e-4:
        size = 2.0 ** -20   # fp16's subnormals
    rows, lens = [2, 1], [300, 80]
    s = make(cuda, 2, rows, lens, 8, 2, 128, 16, "e4m3", TYPES[dt], seed=3)
    s["q"].mul_(size)
    s["k_scale"] *= torch.exp2(torch.randint(-12, 4, s["k_scale"].shape, device=cuda).float())
    s["v_scale"] *= torch.exp2(torch.randint(-12, 12, s["v_scale"].shape, device=cuda).float())
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], return_lse=True, softmax_scale=0.003)
    # p (times its block's scale over the largest so far) is held to 2^-39 of the largest value seen, at worst
    vmax = float((s["v_scale"].max() * 448).item())
    ro, rl, mean, bulk, _ = kv_ref.attend(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], lens, rows, 0, 0, 0.003)
    dp = 2.0 ** -19 * bulk + 2.0 ** -21 * (1 + bulk)
    tol = (2.0 ** -11 + 2 * dp + 2.0 ** -19)[..., None] * mean + torch.finfo(s["q"].dtype).eps / 2 * ro.abs() + 300 * 2.0 ** -30 * vmax
    fit = ro.abs() < torch.finfo(s["q"].dtype).max
    assert bool(((out.double() - ro).abs() <= tol)[fit].all())
    assert bool(((lse.double() - rl).abs() <= dp + 2.0 ** -21 * (1 + rl.abs())).all())


@pytest.mark.parametrize("rows,lens", [([2, 1], [300, 80]), ([1500, 700], [2900, 700])], ids=["few", "many"])
@pytest.mark.parametrize("fmt,dt", [("e4m3", "bf16"), ("int8", "fp16")])
@pytest.mark.parametrize("window", [0, 150])
def test_attend_scales_of_any_value(cuda, rows, lens, fmt, dt, window):
    """Scales that another writer chose: not powers of two, and up to 2^9 apart."""
    from duplex.streaming import kv_cache
    s = make(cuda, 2, rows, lens, 8, 2, 64, 32, fmt, TYPES[dt], seed=11)
    g = torch.Generator(device=cuda).manual_seed(5)
    for n in ("k_scale", "v_scale"):
        s[n] *= torch.exp2(torch.rand(s[n].shape, generator=g, device=cuda) * 5 - 4)
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=3, return_lse=True)
    ro, rl, mean, bulk, _ = kv_ref.attend(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], lens, rows,
                                          window, 3, 1 / 8)
    # a key's scale is a factor in fp32; a value's is rounded to fp16 and so is its product with the code (half a
    # step each, 2^-11), beside the probability's own rounding
    dp = 2.0 ** -19 * bulk + 2.0 ** -21 * (1 + bulk)
    tol = (3 * 2.0 ** -11 + 2 * dp + 2.0 ** -19)[..., None] * mean + torch.finfo(s["q"].dtype).eps / 2 * ro.abs() + 2.0 ** -24
    assert bool(((lse.double() - rl).abs() <= dp + 2.0 ** -21 * (1 + rl.abs())).all())
    assert bool(((out.double() - ro).abs() <= tol).all())


def test_attend_uniform_rows_and_strides(cuda):
    """cu_q left out; q with strides that need a copy; softmax_scale given."""
    from duplex.streaming import kv_cache
    rows, lens = [2, 2, 2], [40, 2, 333]
    s = make(cuda, 3, rows, lens, 8, 4, 64, 32, "int8", torch.float16, seed=5)
    ref, rlse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], return_lse=True, softmax_scale=0.05)
    check_attend(s, rows, lens, 0, 0, ref, rlse, scale=0.05)
    got = kv_cache.kv_attend(s["q"], *cache_args(s), softmax_scale=0.05)
    assert torch.equal(got, ref)
    odd = torch.empty(6, 8 * 64 + 3, dtype=torch.float16, device=cuda)[:, 1: 1 + 512].view(6, 8, 64)
    odd.copy_(s["q"])
    assert torch.equal(kv_cache.kv_attend(odd, *cache_args(s), softmax_scale=0.05), ref)
    turned = s["q"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(kv_cache.kv_attend(turned, *cache_args(s), softmax_scale=0.05), ref)


@pytest.mark.parametrize("T", [1, 2])
def test_largest_batch(cuda, T):
    """4096 sequences in a call against the same in calls of 128; one more is refused."""
    from duplex.streaming import kv_cache
    B = 4096
    lens = [T + (7 * i) % 40 for i in range(B)]
    s = make(cuda, B, [T] * B, lens, 8, 1, 128, 16, "e4m3", torch.float16, seed=9, width=3)
    out = kv_cache.kv_attend(s["q"], *cache_args(s))
    for b in range(0, B, 128):
        part = kv_cache.kv_attend(s["q"][b * T: (b + 128) * T], *cache_args(s)[:4], s["table"][b: b + 128],
                                  s["kv_len"][b: b + 128])
        assert torch.equal(part, out[b * T: (b + 128) * T])
    kv_cache.kv_append(s["q"][:, :1], s["q"][:, 1:2], *cache_args(s))
    with pytest.raises(RuntimeError):
        kv_cache.kv_attend(s["q"], *cache_args(s)[:4], torch.cat([s["table"], s["table"][:1]]),
                           torch.cat([s["kv_len"], s["kv_len"][:1]]), cu_q=torch.zeros(B + 2, dtype=torch.int32, device=cuda))


def test_rows_before_and_between(cuda):
    """Row offsets that do not begin at 0: the rows before belong to nobody."""
    from duplex.streaming import kv_cache
    s = make(cuda, 2, [40, 3], [60, 33], 4, 1, 64, 16, "int8", torch.float16, extra_rows=70)
    cu = s["cu"] + 65
    q, k = s["q"], s["q"][:, :1]
    ref = [t.clone() for t in (s["k"], s["k_scale"])]
    kv_cache.kv_append(k, k, *cache_args(s), cu_q=cu)
    got = [t.clone() for t in (s["k"], s["k_scale"])]
    s["k"].copy_(ref[0]), s["k_scale"].copy_(ref[1])
    kv_cache.kv_append(k[65:], k[65:], *cache_args(s), cu_q=s["cu"])
    assert torch.equal(got[0], s["k"]) and torch.equal(got[1], s["k_scale"])
    out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
    kv_cache.kv_attend(q, *cache_args(s), cu_q=cu, out=out)
    assert bool((out[:65] == 7).all()) and bool((out[108:] == 7).all())
    assert torch.equal(out[65:108], kv_cache.kv_attend(q[65:], *cache_args(s), cu_q=s["cu"])[:43])


def test_attend_nan_and_inf_rows_stay_alone(cuda):
    from duplex.streaming import kv_cache
    rows, lens = [1, 3], [200, 90]
    s = make(cuda, 2, rows, lens, 8, 2, 128, 64, "e4m3", torch.bfloat16, seed=6)
    ref = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"])
    s["q"][2, 1, 5] = float("nan")
    s["q"][1, 6, 0] = float("inf")
    got = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"])
    assert bool(torch.isnan(got[2, 1]).all()) and bool(torch.isnan(got[1, 6]).all())
    keep = torch.ones(4, 8, dtype=torch.bool, device=cuda)
    keep[2, 1] = keep[1, 6] = False
    assert torch.equal(got[keep], ref[keep])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("P,D", [(16, 64), (64, 128), (128, 128), (32, 64)])
def test_append(cuda, fmt, dt, P, D):
    """Fresh, partly filled and crossed blocks; scales that rise, that do not, and zeros; exact."""
    from duplex.streaming import kv_cache
    rows, lens, H = [1, 0, 5, 2 * P + 3, 1, P, 9], [1, 7, P + 2, 3 * P + 1, P, 2 * P, 4], 3
    s = make(cuda, 7, rows, lens, 6, H, D, P, fmt, TYPES[dt], seed=P, spread=2.0 ** -3, extra_rows=1)
    N = sum(rows)
    buf = s["buf"]
    buf[: N // 2] *= 37.0
    buf[N // 2 + 1] = 0.0
    k_new, v_new = buf[:, 6 * D: (6 + H) * D].view(-1, H, D), buf[:, (6 + H) * D:].view(-1, H, D)
    if fmt == "e4m3":   # the reference wants finite codes in the kept slots alone
        pass
    ref = {n: s[n].double().cpu() for n in ("k", "v", "k_scale", "v_scale")}
    kv_ref.append(ref, k_new.cpu(), v_new.cpu(), s["table"].cpu(), lens, rows, fmt)
    weights = torch.ones(s["k"].shape[:3], device=cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    for _ in range(2):   # storing the same tokens again changes nothing
        kv_cache.kv_append(k_new, v_new, *cache_args(s), cu_q=s["cu"], weights=weights, err=err)
        for n in ("k", "v"):
            assert torch.equal(s[n].double().cpu().nan_to_num(1000.0), ref[n].nan_to_num(1000.0)), n
            assert torch.equal(s[n + "_scale"].double().cpu(), ref[n + "_scale"])
    assert int(err) == 0
    want = torch.ones(s["k"].shape[:3])
    for b, (t, n) in enumerate(zip(rows, lens)):
        for j in range(max(n - t, 0), n):
            want[int(s["table"][b, j // P]), :, j % P] = 0
    assert torch.equal(weights.cpu(), want)


def test_prompt_matches_single_rows(cuda):
    """The tensor-core kernel and the few-rows kernel agree where the first meets what the second is
    tested for: a NaN row, a block id out of range, garbage behind the sequence; rows taken one by one."""
    from duplex import _lib
    from duplex.streaming import kv_cache
    T, n, Hq, H, D, P = 2048, 2300, 8, 2, 128, 64
    s = make(cuda, 1, [T], [n], Hq, H, D, P, "e4m3", torch.bfloat16, seed=11)
    s["q"][700, 3, 9] = float("nan")
    s["table"][0, 20] = -7
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), return_lse=True, err=err)
    assert int(err) == _lib.DEVERR_BLOCK
    assert bool(torch.isnan(out[700, 3]).all()) and int(torch.isnan(out).any(-1).sum()) == 1
    for t in (0, 1, 255, 699, 700, 701, 1027, 1028, 1100, T - 1):
        one, l = kv_cache.kv_attend(s["q"][t: t + 1], *cache_args(s)[:5], s["kv_len"] - T + t + 1, return_lse=True)
        ok = ~torch.isnan(one)
        # both are within the bars of the float64 result: fp16 probabilities, and a rounding to bf16 each
        bar = 2 * (2.0 ** -11 + 2.0 ** -12) * 448 * float(s["v_scale"].max()) + 2.0 ** -8 * one.float().abs()
        assert bool(((out[t] - one[0]).float().abs() <= bar[0])[ok[0]].all())
        assert torch.allclose(lse[t], l[0], rtol=2.0 ** -17, atol=2.0 ** -15, equal_nan=True)


def test_prompt_captured(cuda):
    """A captured prompt call follows lengths, rows and values; two replays side by side."""
    from duplex.streaming import kv_cache
    rows, lens = [1200, 900], [2000, 900]
    s = make(cuda, 2, rows, lens, 8, 1, 128, 32, "int8", torch.float16, seed=12)
    kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"])
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            o = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], return_lse=True)
        graphs.append((g, o))
    for r, n in (([1200, 900], [2000, 900]), ([2100, 0], [2000, 900]), ([300, 1800], [301, 896])):
        s["kv_len"].copy_(torch.tensor(n, dtype=torch.int32))
        s["cu"].copy_(torch.tensor([0, r[0], r[0] + r[1]], dtype=torch.int32))
        s["q"].copy_(torch.randn_like(s["q"]))
        torch.cuda.synchronize()
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        ref = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], return_lse=True)
        k = r[0] + r[1]
        for _, o in graphs:
            assert torch.equal(o[0][:k], ref[0][:k]) and torch.equal(o[1][:k], ref[1][:k])


def test_append_not_finite(cuda):
    from duplex import _lib
    from duplex.streaming import kv_cache
    s = make(cuda, 1, [3], [20], 4, 1, 64, 16, "e4m3", torch.bfloat16)
    k_new = torch.randn(3, 1, 64, device=cuda).bfloat16()
    k_new[0, 0, 3], k_new[2, 0, 60], k_new[1, 0, 0] = float("nan"), float("inf"), -float("inf")
    ref = {n: s[n].double().cpu() for n in ("k", "v", "k_scale", "v_scale")}
    kv_ref.append(ref, k_new.cpu(), k_new.cpu(), s["table"].cpu(), [20], [3], "e4m3")
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv_cache.kv_append(k_new, k_new, *cache_args(s), err=err)
    assert int(err) == _lib.DEVERR_NONFINITE
    assert torch.equal(s["k"].double().cpu().nan_to_num(1000.0), ref["k"].nan_to_num(1000.0))
    assert torch.equal(s["k_scale"].double().cpu(), ref["k_scale"])


def test_append_extreme_values(cuda):
    """bf16's largest and smallest: the scale's exponent at both ends."""
    from duplex.streaming import kv_cache
    for fmt in ("e4m3", "int8"):
        s = make(cuda, 2, [2, 2], [2, 2], 4, 1, 64, 16, fmt, torch.bfloat16)
        k_new = torch.zeros(4, 1, 64, device=cuda).bfloat16()
        k_new[0, 0, 0], k_new[1, 0, 1] = 3.3e38, 1e37
        k_new[2, 0, 0], k_new[3, 0, 1] = 2.0 ** -126, 2.0 ** -130
        ref = {n: s[n].double().cpu() for n in ("k", "v", "k_scale", "v_scale")}
        kv_ref.append(ref, k_new.cpu(), k_new.cpu(), s["table"].cpu(), [2, 2], [2, 2], fmt)
        kv_cache.kv_append(k_new, k_new, *cache_args(s))
        assert torch.equal(s["k"].double().cpu().nan_to_num(1000.0), ref["k"].nan_to_num(1000.0))
        assert torch.equal(s["k_scale"].double().cpu(), ref["k_scale"])


EVICT = [
    # lens, keep, sinks, recent, H, D, P, fmt
    ([100, 37, 5], 40, 4, 10, 2, 64, 16, "e4m3"),
    ([3000, 1025, 64], 1024, 4, 100, 3, 128, 64, "int8"),
    ([20000], 333, 0, 0, 1, 64, 128, "e4m3"),
    ([257, 300], 256, 256, 0, 2, 64, 32, "int8"),        # nothing to choose
    ([130, 0, 1], 100, 30, 70, 1, 128, 32, "e4m3"),
    ([50], 1, 0, 0, 2, 64, 16, "e4m3"),
    ([40_700, 39_000], 5000, 7, 900, 1, 64, 16, "int8"),    # as many keys as shared memory holds
    ([70_000, 3], 9000, 0, 1, 1, 64, 128, "e4m3"),          # and more
]


@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"{max(c[0])}to{c[1]}-{c[7]}")
def test_evict(cuda, case, kind):
    from duplex.streaming import kv_cache
    lens, keep, sinks, recent, H, D, P, fmt = case
    B, width_dst = len(lens), -(-keep // P) + 1
    s = make(cuda, B, [1] * B, lens, H, H, D, P, fmt, torch.float16, spare=B * width_dst, seed=keep)
    g = torch.Generator(device=cuda).manual_seed(1)
    w = torch.rand(s["k"].shape[:3], generator=g, device=cuda)
    if kind == "ties":
        w = torch.floor(w * 3)
        w[w == 0] *= -1      # -0 is 0
    if kind == "odd":
        w = torch.where(w < 0.2, float("nan"), torch.where(w < 0.4, -w, torch.where(w > 0.9, float("inf"), w)))
    dst = torch.full((B, width_dst), -1, dtype=torch.int32, device=cuda)
    dst[:, :-1] = s["free"][: B * (width_dst - 1)].view(B, -1)
    before = {n: s[n].clone() for n in ("k", "v", "k_scale", "v_scale")}
    w0 = w.clone()
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    new = kv_cache.kv_evict(*cache_args(s), w, dst, keep=keep, sinks=sinks, recent=recent, err=err)
    assert int(err) == 0
    assert new.tolist() == [min(n, keep) for n in lens]
    want = {n: before[n].double().cpu() for n in before}
    ww = w0.cpu().clone()
    table, target = s["table"].cpu(), dst.cpu()
    for b, n in enumerate(lens):
        for h in range(H):
            mine = w0[s["table"][b, : -(-n // P)].long(), h].reshape(-1)[:n].tolist()
            at = kv_ref.kept_tokens(mine, n, keep, sinks, recent)
            for i, j in enumerate(at):
                ww[int(target[b, i // P]), h, i % P] = mine[j]
            for name in "kv":
                x = kv_ref.values(before[name], before[name + "_scale"], s["table"][b, : -(-n // P)].long(), h, n).cpu()
                x = x[torch.tensor(at, dtype=torch.long)]
                for i in range(-(-len(at) // P)):
                    part, blk = x[i * P: i * P + P], int(target[b, i])
                    two = kv_ref.scale_of(part, fmt)
                    want[name][blk, h, : len(part)] = kv_ref.rounded(part / two, fmt)
                    want[name + "_scale"][blk, h] = two
    for name in "kv":
        assert torch.equal(s[name].double().cpu().nan_to_num(1000.0), want[name].nan_to_num(1000.0)), name
        assert torch.equal(s[name + "_scale"].double().cpu(), want[name + "_scale"])
    assert torch.equal(w.cpu().nan_to_num(1000.0), ww.nan_to_num(1000.0))


def test_bad_blocks_are_reported(cuda):
    """Ids out of range inside a sequence: reported, their tokens left out, nothing else touched."""
    from duplex import _lib
    from duplex.streaming import kv_cache
    rows, lens = [1, 1], [80, 40]
    s = make(cuda, 2, rows, lens, 4, 1, 64, 16, "int8", torch.float16, spare=8)
    ref = kv_cache.kv_attend(s["q"], *cache_args(s))
    short = kv_cache.kv_attend(s["q"][:1], s["k"], s["v"], s["k_scale"], s["v_scale"],
                               torch.cat([s["table"][:1, :1], s["table"][:1, 2:]], 1).contiguous(), s["kv_len"][:1] - 16)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    s["table"][0, 1] = s["k"].shape[0]
    w = torch.zeros(s["k"].shape[:3], device=cuda)
    out = kv_cache.kv_attend(s["q"], *cache_args(s), weights=w, err=err)
    assert int(err) == _lib.DEVERR_BLOCK
    assert torch.equal(out[1], ref[1])
    torch.testing.assert_close(out[0].float(), short[0].float(), rtol=2 ** -9, atol=2 ** -9 * float(ref.abs().max()))
    for call in ("append", "evict"):
        err.zero_()
        if call == "append":
            s["table"][0, 4] = -1
            kv_cache.kv_append(s["q"][:, :1], s["q"][:, :1], *cache_args(s), err=err)
        else:
            dst = torch.tensor([[-3, 5], [1 << 30, 2]], dtype=torch.int32, device=cuda)
            kv_cache.kv_evict(*cache_args(s), w, dst, keep=32, err=err)
        assert int(err) == _lib.DEVERR_BLOCK


def test_graph_follows_lengths_and_streams(cuda):
    """A captured append + attend + evict replayed with other lengths, tables and rows; and two graphs
    of one capture side by side on two streams."""
    from duplex.streaming.kv_cache import PackedKVCache
    B, H, Hq, D, P = 3, 2, 8, 64, 16
    c = PackedKVCache(64, H, D, P, "e4m3", track_weights=True, device=cuda)
    table = torch.arange(24, dtype=torch.int32, device=cuda).view(B, 8)
    dst = torch.arange(24, 24 + 12, dtype=torch.int32, device=cuda).view(B, 4)
    kv_len = torch.tensor([5, 1, 100], dtype=torch.int32, device=cuda)
    x = torch.randn(B, (Hq + 2 * H) * D, device=cuda).half()
    q, k, v = x[:, : Hq * D].view(B, Hq, D), x[:, Hq * D: (Hq + H) * D].view(B, H, D), x[:, (Hq + H) * D:].view(B, H, D)
    for n in range(1, 100):   # something in every slot
        c.append(torch.randn_like(k), torch.randn_like(v), table, torch.full_like(kv_len, n))

    def step():
        c.append(k, v, table, kv_len)
        out = c.attend(q, table, kv_len, window=40, sinks=2)
        return out, c.evict(table, kv_len, dst, keep=50, sinks=2, recent=8)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, new = step()
    for lens in ([7, 2, 101], [128, 17, 3]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        x.copy_(torch.randn_like(x))
        state = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale, c.weights)]
        graph.replay()
        torch.cuda.synchronize()
        a = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale, c.weights, got, new)]
        for t, o in zip((c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale, c.weights), state):
            t.copy_(o)
        out, n = step()
        e = (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale, c.weights, out, n)
        assert all(torch.equal(i, j) for i, j in zip(a, e))
    ref = c.attend(q, table, kv_len, accumulate=False)
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for st in streams:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            o = c.attend(q, table, kv_len, accumulate=False)
        graphs.append((g, o))
    for _ in range(20):
        for st, (g, o) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for _, o in graphs)
    assert c.device_errors() == 0


def test_session(cuda):
    """The operators as a session runs them: prompt, decode with a window, eviction, decode again;
    attention against float64 over the cache's own values at each point."""
    from duplex.streaming.kv_cache import PackedKVCache
    B, H, Hq, D, P = 2, 4, 32, 128, 64
    c = PackedKVCache(40, H, D, P, "e4m3", track_weights=True, device=cuda)
    table = torch.arange(20, dtype=torch.int32, device=cuda).view(B, 10)
    lens = [0, 0]

    def go(rows, tab, window=0, sinks=0):
        for b in range(B):
            lens[b] += rows[b]
        n = sum(rows)
        x = torch.randn(n, (Hq + 2 * H) * D, device=cuda).bfloat16()
        q = x[:, : Hq * D].view(n, Hq, D)
        kv_len = torch.tensor(lens, dtype=torch.int32, device=cuda)
        cu = torch.tensor([0, rows[0], n], dtype=torch.int32, device=cuda)
        c.append(x[:, Hq * D: (Hq + H) * D].view(n, H, D), x[:, (Hq + H) * D:].view(n, H, D), tab, kv_len, cu)
        base = c.weights.clone()
        out, lse = c.attend(q, tab, kv_len, cu, window=window, sinks=sinks, return_lse=True)
        s = {"q": q, "k": c.k, "v": c.v, "k_scale": c.k_scale, "v_scale": c.v_scale, "table": tab}
        check_attend(s, rows, lens, window, sinks, out, lse, c.weights, base)
        return kv_len

    go([300, 41], table)
    for _ in range(5):
        kv_len = go([1, 1], table, window=128, sinks=4)
    kv_len = go([2, 3], table)
    dst = torch.arange(20, 40, dtype=torch.int32, device=cuda).view(B, 10)
    kv_len = c.evict(table, kv_len, dst, keep=200, sinks=4, recent=64)
    lens[:] = kv_len.tolist()
    assert lens == [200, 49]
    for _ in range(3):
        go([1, 1], dst)
    assert c.device_errors() == 0


def test_far_blocks(cuda):
    """Code offsets past 32 bits: a cache of over 4 GB, its last blocks used."""
    from duplex.streaming import kv_cache
    H, D, P, nb = 2, 128, 128, 140_000
    k = torch.empty(nb, H, P, D, dtype=torch.int8, device=cuda)
    assert k.numel() > 2 ** 32
    s = {"k": k, "v": k.clone(), "k_scale": torch.ones(nb, H, device=cuda), "v_scale": torch.ones(nb, H, device=cuda),
         "table": torch.tensor([[nb - 1, nb - 3, 0]], dtype=torch.int32, device=cuda),
         "kv_len": torch.tensor([300], dtype=torch.int32, device=cuda)}
    x = torch.randn(300, 8, D, device=cuda).half()
    kv_cache.kv_append(x[:, :2], x[:, 2:4], *cache_args(s))
    s["q"] = x[-1:, 4:]
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), return_lse=True)
    check_attend(s, [1], [300], 0, 0, out, lse)
    w = torch.rand(nb, H, P, device=cuda)
    dst = torch.tensor([[nb - 2]], dtype=torch.int32, device=cuda)
    n = kv_cache.kv_evict(*cache_args(s), w, dst, keep=100, sinks=1, recent=99)
    got = kv_ref.values(s["k"], s["k_scale"], dst[0].long(), 0, 100)
    src = kv_ref.values(s["k"], s["k_scale"], s["table"][0].long(), 0, 300)[[0] + list(range(201, 300))]
    assert n.tolist() == [100] and torch.allclose(got, src, rtol=0, atol=float(src.abs().max()) / 100)

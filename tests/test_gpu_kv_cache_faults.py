"""Calls of the 8-bit paged KV cache at the edge of what its documentation allows, each of which once gave a
wrong result or went unreported: against float64 (kv_ref) with test_gpu_kv_cache.py's bars."""

import ctypes
import math

import pytest
import torch

import kv_ref
from test_gpu_kv_cache import cache_args, check_attend, make

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


# ------------------------------------------------------------------ block scales far apart
def spread_scales(s, names, cuts, P, lens, before, after):
    """Blocks that begin at token `cut` of their sequence or later get their scales times `after`, the others times
    `before`; both may be no powers of two."""
    for b, (n, cut) in enumerate(zip(lens, cuts)):
        for col in range(-(-n // P)):
            for name in names:
                s[name + "_scale"][int(s["table"][b, col])] *= after if col * P >= cut else before


def check_rows(s, rows, lens, fmt, window, sinks, out, lse, scale):
    """check_attend with one more term, by what each row sees: a probability times its block's scale over the largest
    scale seen is held in fp16, whose half step is 2^-25 below its normal numbers, and a row's sum of probabilities is
    at least 2^7 (its reference's own), so each token adds up to 2^-32 of top times that scale."""
    ro, rl, mean, bulk, _ = kv_ref.attend(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], lens, rows, window,
                                          sinks, scale)
    P, first = s["k"].shape[2], 0
    step = torch.zeros_like(rl)
    for b, (n, t) in enumerate(zip(lens, rows)):
        p = torch.arange(n - t, n, device=out.device)[:, None]
        j = torch.arange(n, device=out.device)
        seen = (j <= p) & ((j > p - window) | (j < sinks) if window else True)
        blocks = s["table"][b, : -(-n // P)].long()
        blocks = torch.where(torch.nn.functional.pad(seen, (0, -n % P)).view(t, -1, P).any(0).any(-1), blocks, 0)
        for h in range(s["k"].shape[1]):
            top = (seen * s["v_scale"][blocks, h].double().repeat_interleave(P)[:n]).amax(1) * kv_ref.TOP[fmt]
            G = out.shape[1] // s["k"].shape[1]
            step[first: first + t, h * G: h * G + G] = (2.0 ** -32 * top * seen.sum(1))[:, None]
        first += t
    dp = 2.0 ** -19 * bulk + 2.0 ** -21 * (1 + bulk)
    tol = (2.0 ** -11 + 2 * dp + 2.0 ** -19)[..., None] * mean + torch.finfo(out.dtype).eps / 2 * ro.abs() + step[..., None] + 2.0 ** -24
    err = (out.double() - ro).abs()
    assert bool((err <= tol).all()), f"out: {float((err / tol).max())} of the bar"
    le = (lse.double() - rl).abs()
    assert bool((le <= dp + 2.0 ** -21 * (1 + rl.abs())).all()), f"lse: {float((le / dp).max())}"


FAR = [
    # rows, lens, cuts, Hq, H, D, P, fmt, window, sinks
    ([2100], [2100], [300], 8, 2, 128, 64, "e4m3", 0, 0),        # the first rows see the first blocks alone
    ([2100], [2100], [304], 8, 2, 64, 16, "int8", 0, 0),         # ... the border inside a row tile and a tile of tokens
    ([1500, 900], [3001, 900], [1664, 800], 8, 2, 128, 32, "e4m3", 0, 0),
    ([1500], [3001], [1792], 8, 2, 128, 128, "int8", 200, 0),    # windows on both sides of the border
    ([1500], [3001], [1664], 8, 2, 64, 64, "e4m3", 200, 20),
]
SPREADS = {"small first": (2.0 ** -30, 1.0), "small last": (1.0, 2.0 ** -30), "by 1.4, small first": (1.4 * 2.0 ** -22, 1.1)}


@pytest.mark.parametrize("spread", SPREADS)
@pytest.mark.parametrize("names", ["k", "v", "kv"])
@pytest.mark.parametrize("case", FAR, ids=lambda c: f"{c[3]}x{c[4]}x{c[5]}-p{c[6]}-{c[7]}-w{c[8]}-{max(c[0])}of{max(c[1])}")
def test_prompt_rows_that_see_small_blocks(cuda, case, names, spread):
    """A row's result hangs on what it sees: blocks 2^30 below the sequence's largest keep their bits for the
    rows that see no larger ones, keys and values."""
    from duplex.streaming import kv_cache
    rows, lens, cuts, Hq, H, D, P, fmt, window, sinks = case
    before, after = SPREADS[spread]
    s = make(cuda, len(rows), rows, lens, Hq, H, D, P, fmt, torch.bfloat16, seed=21)
    spread_scales(s, names, cuts, P, lens, before, after)
    scale, low = 1 / math.sqrt(D), min(before, after)
    if "k" in names:                           # scores of the usual size for every row, by the largest block that it sees
        scale, at = scale / low, 0
        for t, n, cut in zip(rows, lens, cuts):
            edge = -(-cut // P) * P
            for p in range(n - t, n):
                large = p >= edge if before < after else not window or p - window + 1 < edge or sinks > 0
                s["q"][at] *= low / max(before, after) if large else 1.0
                at += 1
    if "v" in names:
        s["v_scale"] /= low                    # the small ones are of the usual size, the large ones 2^30 of it
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=sinks, softmax_scale=scale,
                                  return_lse=True)
    check_rows(s, rows, lens, fmt, window, sinks, out, lse, scale)


@pytest.mark.parametrize("apart", [2.0 ** 34, 1.7 * 2.0 ** 40])
@pytest.mark.parametrize("case", [
    # rows, lens, cuts, Hq, H, D, P, fmt, window, sinks, whether the large values come first
    ([2], [17], [16], 4, 2, 64, 16, "e4m3", 0, 0, False),              # row 0 does not see the last block
    ([5, 3], [1010, 34], [1008, 32], 4, 1, 128, 16, "int8", 0, 0, False),
    ([5], [1010], [1008], 16, 4, 128, 16, "e4m3", 3, 0, False),
    ([3], [194], [192], 4, 1, 128, 64, "e4m3", 0, 0, False),
    ([6], [2230], [128], 4, 1, 64, 64, "e4m3", 2100, 0, True),         # rows 3 and on do not see the first two blocks
    ([6], [2230], [128], 8, 1, 128, 128, "int8", 2101, 0, True),
    ([5] * 40, [1010] * 40, [1008] * 40, 4, 1, 128, 16, "e4m3", 0, 0, False),     # pieces of row tiles
    ([3], [194], [192], 4, 1, 64, 16, "e4m3", 100, 5, False),
], ids=lambda c: f"{c[3]}x{c[4]}x{c[5]}-p{c[6]}-{c[7]}-w{c[8]}-{max(c[0])}of{max(c[1])}")
def test_few_rows_that_see_small_values(cuda, case, apart):
    """Rows of one tile beside a row that sees a block with values 2^34 times as large: they do not see it."""
    from duplex.streaming import kv_cache
    rows, lens, cuts, Hq, H, D, P, fmt, window, sinks, first = case
    s = make(cuda, len(rows), rows, lens, Hq, H, D, P, fmt, torch.bfloat16, seed=22)
    spread_scales(s, "v", cuts, P, lens, apart if first else 1.0, 1.0 if first else apart)
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=sinks, return_lse=True)
    check_rows(s, rows, lens, fmt, window, sinks, out, lse, 1 / math.sqrt(D))


# ------------------------------------------------------------------ very large scores
def scores(s, b, h, n, t, first, window, scale):
    """[t, group, n] float64 of one sequence and KV head, -inf where a row does not see."""
    P, G = s["k"].shape[2], s["q"].shape[1] // s["k"].shape[1]
    p = torch.arange(n - t, n, device=s["q"].device)[:, None]
    j = torch.arange(n, device=s["q"].device)
    seen = (j <= p) & (j > p - window if window else True)
    blocks = s["table"][b, : -(-n // P)].long()
    blocks = torch.where(torch.nn.functional.pad(seen, (0, -n % P)).view(t, -1, P).any(0).any(-1), blocks, 0)
    k = kv_ref.values(s["k"], s["k_scale"], blocks, h, n).nan_to_num(0, 0, 0)
    x = torch.einsum("tgd,nd->tgn", s["q"][first: first + t, h * G: h * G + G].double(), k) * scale
    return x.masked_fill(~seen[:, None], -math.inf)


@pytest.mark.parametrize("by", [2.0 ** 22, 2.0 ** 27, -2.0 ** 30, 2.0 ** 45])
@pytest.mark.parametrize("rows,lens,window,odd", [([1, 3], [700, 90], 0, 1.0), ([2, 5], [9000, 40], 100, 1.0),
                                                  ([1500, 900], [2900, 900], 0, 1.0), ([1500, 900], [2900, 900], 200, 1.3)])
def test_large_scores(cuda, rows, lens, window, odd, by):
    """Scores of 1e7 to 1e14, whose fp32 steps are far above 1: where one stands out by more than the bars of a score, the
    row is its value alone; elsewhere the result is some mean of values.  The weights' pass computes a score anew, off from
    the attention's by up to 2 ds, where ds is 2^-19 bulk > 8 here: exp(2 ds) leaves of a weight only that it is a number
    from 0 to 1 for each row and head."""
    from duplex.streaming import kv_cache
    s = make(cuda, 2, rows, lens, 8, 2, 128, 32, "e4m3", torch.bfloat16, seed=31)
    s["k_scale"] *= odd
    weights = torch.zeros(s["k"].shape[:3], device=cuda)
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, softmax_scale=by, weights=weights,
                                  return_lse=True)
    ro, rl, mean, bulk, _ = kv_ref.attend(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], lens, rows, window,
                                          0, by)
    ds = 2.0 ** -19 * bulk + 2.0 ** -21 * (1 + bulk)
    assert bool(((lse.double() - rl).abs() <= ds + 2.0 ** -21 * (1 + rl.abs())).all())
    gap, first = torch.zeros_like(rl), 0
    for b, (n, t) in enumerate(zip(lens, rows)):
        for h in range(2):
            top = torch.topk(scores(s, b, h, n, t, first, window, by), 2, -1).values
            gap[first: first + t, 4 * h: 4 * h + 4] = top[..., 0] - top[..., 1]
        first += t
    alone = gap > 2 * ds + 40
    assert float(alone.double().mean()) > 0.5
    tol = (2.0 ** -10 * mean + 2.0 ** -8 * ro.abs() + 2.0 ** -24)
    assert bool(((out.double() - ro).abs() <= tol)[alone].all())
    vmax = float(s["v_scale"].max()) * 448
    assert bool((out.abs() <= vmax * 1.01).all())
    assert float(ds.median()) > 8
    assert bool(((weights >= 0) & (weights <= 4 * sum(rows) * (1 + 2.0 ** -19))).all())
    # as for NaN: it stays in its row
    s["q"][0, 0, 0] = float("nan")
    got = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, softmax_scale=by)
    assert bool(torch.isnan(got[0, 0]).all()) and int(torch.isnan(got).any(-1).sum()) == 1


# ------------------------------------------------------------------ eviction of zeros
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("keep", [16, 17, 37])
def test_evict_zero_tokens(cuda, keep, small, fmt):
    """Zero tokens out of blocks with a large scale: zeros at the smallest scale, in a full block and in a tail of one;
    and beside a small token of another block, which sets the scale."""
    from duplex.streaming import kv_cache
    H, D, P, n = 2, 64, 16, 80
    s = make(cuda, 1, [1], [n], H, H, D, P, fmt, torch.float16, spare=4, seed=3)
    w = torch.zeros(s["k"].shape[:3], device=cuda)
    zero = torch.zeros(H, P, D, device=cuda)
    for col in range(5):
        blk = int(s["table"][0, col])
        for name in "kv":
            code = zero.clone()
            code[:, 5] = 100.0                                   # one large token a block, which is not kept
            if small and col == 1:
                code[:, 7, 3] = 1.0
            s[name][blk] = code.to(s[name].dtype)
            s[name + "_scale"][blk] = 2.0 ** (-100 if small and col == 1 else 100 if small else 3)
        w[blk] = 1.0
        w[blk, :, 5] = 0.0
    dst = s["free"][:3].view(1, 3).contiguous()
    before = {m: s[m].clone() for m in ("k", "v", "k_scale", "v_scale")}
    kv_cache.kv_evict(*cache_args(s), w, dst, keep=keep)
    at = [j for j in range(n) if j % P != 5][:keep]
    for h in range(H):
        for name in "kv":
            x = kv_ref.values(before[name], before[name + "_scale"], s["table"][0].long(), h, n).cpu()[torch.tensor(at)]
            for i in range(-(-keep // P)):
                part, blk = x[i * P: i * P + P], int(dst[0, i])
                two = kv_ref.scale_of(part, fmt)
                got = s[name][blk, h, : len(part)].double().cpu()
                assert torch.equal(got, kv_ref.rounded(part / two, fmt)), (name, i)
                assert float(s[name + "_scale"][blk, h]) == two
    out = kv_cache.kv_attend(s["q"][:1], *cache_args(s)[:4], dst, torch.tensor([keep], dtype=torch.int32, device=cuda))
    assert bool(torch.isfinite(out).all())


# ------------------------------------------------------------------ eviction that writes the lengths in place
def test_evict_lengths_in_place(cuda):
    """duplex_kv_evict with new_len = kv_len: every head reads the old length, however many there are."""
    from duplex import _lib
    from duplex.streaming import kv_cache
    H, D, P, n, keep, B = 400, 64, 16, 48, 20, 2                # more selections than run at once
    s = make(cuda, B, [1] * B, [n] * B, H, H, D, P, "int8", torch.float16, spare=2 * B, seed=4)
    w = torch.rand(s["k"].shape[:3], device=cuda)
    dst = s["free"][: 2 * B].view(B, 2).contiguous()
    names = ("k", "v", "k_scale", "v_scale")
    state = [s[m].clone() for m in names] + [w.clone()]
    new = kv_cache.kv_evict(*cache_args(s), w, dst, keep=keep, sinks=1, recent=3)
    want = [s[m].clone() for m in names] + [w.clone()]
    for m, t in zip(names, state):
        s[m].copy_(t)
    w.copy_(state[-1])
    lib = _lib.load()
    cache = _lib.KVCache(k=s["k"].data_ptr(), v=s["v"].data_ptr(), k_scale=s["k_scale"].data_ptr(),
                         v_scale=s["v_scale"].data_ptr(), weights=w.data_ptr(), n_blocks=s["k"].shape[0], kv_heads=H,
                         block=P, dim=D, format=_lib.KV_INT8)
    batch = _lib.KVBatch(block_table=s["table"].data_ptr(), kv_len=s["kv_len"].data_ptr(), cu_rows=None,
                         width=s["table"].shape[1], batch=B, n_rows=0)
    ws = torch.empty(B * H * keep * 4, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    rc = lib.duplex_kv_evict(ctypes.byref(cache), ctypes.byref(batch), dst.data_ptr(), 2, keep, 1, 3, s["kv_len"].data_ptr(),
                             ws.data_ptr(), ws.numel(), None, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert s["kv_len"].tolist() == new.tolist() == [keep] * B
    for m, t in zip(names, want):
        used = dst.flatten().long()
        assert torch.equal(s[m][used], t[used]), m
    assert torch.equal(w, want[-1])


# ------------------------------------------------------------------ tables that are too narrow
def dense(q, k, v, first, n, window, sinks, scale):
    """Rows q [T, Hq, D] at positions first + t over tokens k, v [H, n, D], float64: out, lse."""
    T, Hq, D = q.shape
    G = Hq // k.shape[0]
    p = first + torch.arange(T, device=q.device)[:, None]
    j = torch.arange(n, device=q.device)
    seen = (j <= p) & ((j > p - window) | (j < sinks) if window else True)
    s = torch.einsum("thd,hnd->thn", q.double(), k.repeat_interleave(G, 0)) * scale
    s = s.masked_fill(~seen[:, None], -math.inf)
    l = torch.logsumexp(s, -1)
    pr = torch.exp(s - torch.where(l == -math.inf, 0, l)[..., None]) * seen[:, None]
    return torch.einsum("thn,hnd->thd", pr, v.repeat_interleave(G, 0)), l, pr


@pytest.mark.parametrize("T,n,W,P,window,sinks", [(5, 35, 2, 16, 0, 0), (5, 35, 2, 16, 8, 2), (1, 40, 2, 16, 0, 0), (1, 40, 2, 16, 3, 1),
                                                  (1500, 2100, 32, 64, 0, 0), (1500, 2100, 32, 64, 100, 5),
                                                  (3, 2 ** 31 - 1, 2, 16, 0, 0), (3, 2 ** 31 - 1, 2, 16, 5, 3),
                                                  (1500, 2 ** 31 - 1, 32, 64, 100, 5)])
def test_table_too_narrow(cuda, T, n, W, P, window, sinks):
    """A length beyond its table: reported; tokens past the table are not stored, and not seen by rows that keep
    their positions; stored tokens and the other sequence stay as they are."""
    from duplex import _lib
    from duplex.streaming import kv_cache
    cap, H, Hq, D = W * P, 2, 8, 64
    s = make(cuda, 2, [T, 1], [cap, 30], Hq, H, D, P, "int8", torch.float16, seed=8)
    s["kv_len"][0] = n
    weights, err = torch.zeros(s["k"].shape[:3], device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    want = {m: s[m].double().cpu() for m in ("k", "v", "k_scale", "v_scale")}
    k_new, v_new = (0.5 * torch.randn(T + 1, H, D, device=cuda).half() for _ in range(2))
    fit = max(cap - (n - T), 0)                                  # rows that the table has room for
    some = [*range(fit), T]
    kv_ref.append(want, k_new[some].cpu(), v_new[some].cpu(), s["table"].cpu(), [min(n, cap), 30], [fit, 1], "int8")
    kv_cache.kv_append(k_new, v_new, *cache_args(s), cu_q=s["cu"], err=err)
    assert int(err) == _lib.DEVERR_LENGTH
    for m in want:
        assert torch.equal(s[m].double().cpu().nan_to_num(1000.0), want[m].nan_to_num(1000.0)), m
    err.zero_()
    out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=sinks, weights=weights,
                                  return_lse=True, err=err)
    assert int(err) == _lib.DEVERR_LENGTH
    blocks = s["table"][0].long()
    k, v = (torch.stack([kv_ref.values(s[m], s[m + "_scale"], blocks, h, cap) for h in range(H)]) for m in "kv")
    ro, rl, pr = dense(s["q"][:T], k, v, n - T, cap, window, sinks, 1 / 8)
    assert torch.equal(lse[:T] == -math.inf, rl == -math.inf)
    some = rl > -math.inf
    big = float(v.abs().max())
    assert bool(((lse[:T] - rl).abs() < 1e-3)[some].all()) and bool(((out[:T] - ro).abs() < 4e-3 * big).all())
    rw = pr.view(T, H, Hq // H, cap).sum((0, 2)).view(H, W, P).transpose(0, 1)
    assert torch.allclose(weights[blocks].double(), rw, rtol=1e-3, atol=1e-3)
    one = kv_cache.kv_attend(s["q"][T:], *cache_args(s)[:4], s["table"][1:], s["kv_len"][1:], window=window, sinks=sinks)
    assert torch.allclose(out[T:].float(), one.float(), rtol=2.0 ** -9, atol=2.0 ** -9 * big)
    new = kv_cache.kv_evict(*cache_args(s), weights, torch.full((2, 1), -1, dtype=torch.int32, device=cuda), keep=1, err=err)
    assert int(err) == _lib.DEVERR_LENGTH | _lib.DEVERR_BLOCK and new.tolist() == [1, 1]


def test_replays_past_the_capacity_are_reported(cuda):
    """A step that the caller captured, replayed more often than the streams have room: nothing stored is lost."""
    from duplex import _lib
    from test_gpu_clock_attention import build
    _, st = build(cuda, 2, tokens=16, fmt="int8")
    x, out = torch.randn(2, 256, device=cuda).half(), torch.zeros(2, 256, device=cuda).half()
    st.step_into(x, out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        st.step_into(x, out)
    state = lambda: [t.clone() for c in st.caches.layers for t in (c.k, c.v, c.k_scale, c.v_scale)]  # noqa: E731
    for _ in range(15):
        x.copy_(torch.randn_like(x))
        g.replay()
    assert st.device_errors() == 0 and st.caches.kv_len.tolist() == [16, 16]
    before = state()
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        g.replay()
    assert st.device_errors() == _lib.DEVERR_LENGTH
    assert all(torch.equal(a, b) for a, b in zip(before, state()))


# ------------------------------------------------------------------ the clock stack's captured steps
def test_capture_warms_the_sessions_kernels(cuda):
    """The step before the capture takes the kernels that the session's tables ask for; a capture that fails leaves the session."""
    from duplex.streaming.kv_cache import PackedKVCache
    from test_gpu_clock_attention import build
    _, st = build(cuda, 2, fmt="int8", tokens=13_000)
    seen, real = [], PackedKVCache.attend

    def attend(self, q, table, *a, **kw):
        seen.append((tuple(table.shape), torch.cuda.is_current_stream_capturing()))
        return real(self, q, table, *a, **kw)

    x = torch.randn(2, 256, device=cuda).half()
    out = torch.zeros_like(x)
    PackedKVCache.attend = attend
    try:
        st.capture()
    finally:
        PackedKVCache.attend = real
    assert {w for w, c in seen if c} == {w for w, c in seen if not c} == {(2, 813)}
    caches = st.caches
    st.x_in.copy_(x)
    st.replay()
    torch.cuda.synchronize()
    got = st.out.clone()
    _, other = build(cuda, 2, fmt="int8", tokens=13_000)
    other.step_into(x, out)
    assert torch.equal(got, out)

    def fails(*a, **kw):
        raise ValueError("no")

    st._chain = fails
    with pytest.raises(ValueError):
        st.capture()
    assert st.caches is caches and caches.kv_len.tolist() == [1, 1]


def captured_kernels(call):
    """The kernel launches of a call, counted in a graph of it."""
    from cuda.bindings import driver
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    raw = driver.CUgraph(g.raw_cuda_graph())
    _, _, n = driver.cuGraphGetNodes(raw)
    _, nodes, n = driver.cuGraphGetNodes(raw, n)
    kernel = driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL
    return sum(driver.cuGraphNodeGetType(v)[1] == kernel for v in nodes[:n])


@pytest.mark.parametrize("tokens,kw", [(None, {}), (64, {}), (64, {"evictable": True}), (13_000, {}), (13_000, {"evictable": True}),
                                       (13_000, {"window": 100})])
def test_kernels_per_step(cuda, tokens, kw):
    """kernels_per_step is the number of this package's kernels in a captured step (the lengths' increment is torch's)."""
    from duplex.clock import ClockStack
    from test_gpu_clock import small_layers
    st = ClockStack.from_arrays(small_layers(2), top_k=4, device=cuda, T=2, fused=False)
    if tokens:
        st.attach_cache(tokens, block=16, head_dim=64, **kw)
    x, out = torch.zeros(2, 256, device=cuda).half(), torch.zeros(2, 256, device=cuda).half()
    st.step_into(x, out)
    torch.cuda.synchronize()
    assert st.kernels_per_step() == captured_kernels(lambda: st.step_into(x, out)) - bool(tokens)


@pytest.mark.parametrize("B,T,width,window,launches", [(1, 1, 4, 0, 1), (40, 1, 4, 0, 2), (1, 1, 1000, 0, 2), (1, 1, 1000, 64, 1),
                                                       (1, 900, 100, 0, 3), (2, 900, 100, 200, 3)])
@pytest.mark.parametrize("track", [False, True])
def test_attend_launches(cuda, B, T, width, window, launches, track):
    """duplex_kv_attend_launches counts what a call launches: clusters, pieces and their join, the prompt kernels, weights."""
    from duplex import _lib
    from duplex.streaming.kv_cache import PackedKVCache
    c = PackedKVCache(8, 1, 128, 16, "int8", track_weights=track, device=cuda)
    table, kv_len = torch.zeros(B, width, dtype=torch.int32, device=cuda), torch.full((B,), 1, dtype=torch.int32, device=cuda)
    q = torch.randn(B * T, 8, 128, device=cuda).half()
    call = lambda: c.attend(q, table, kv_len, window=window)  # noqa: E731
    call()
    torch.cuda.synchronize()
    n, p = ctypes.c_int32(), lambda t: t.data_ptr()
    cache = _lib.KVCache(p(c.k), p(c.v), p(c.k_scale), p(c.v_scale), p(c.weights) if track else None, *c.k.shape, _lib.KV_INT8)
    batch = _lib.KVBatch(p(table), p(kv_len), None, width, B, B * T)
    assert _lib.load().duplex_kv_attend_launches(ctypes.byref(cache), ctypes.byref(batch), 8, window, 0, ctypes.byref(n)) == 0
    assert n.value == launches + track == captured_kernels(call)


def test_offsets_that_fall_are_reported_whatever_else(cuda):
    """Where no sequence has a token to store, and where they fall behind the 256th sequence."""
    from duplex import _lib
    from duplex.streaming import kv_cache
    for B, cu in ((2, [0, 3, 1]), (600, [0] * 400 + [2] + [1] * 200)):
        s = make(cuda, B, [3] + [0] * (B - 1), [16] * B, 2, 1, 64, 16, "int8", torch.float16)
        fall = torch.tensor(cu, dtype=torch.int32, device=cuda)
        before = s["k"].clone()
        for n in (0, 16):
            s["kv_len"].fill_(n)
            err = torch.zeros(1, dtype=torch.int32, device=cuda)
            kv_cache.kv_append(s["q"][:, :1], s["q"][:, 1:2], *cache_args(s), cu_q=fall, err=err)
            assert int(err) == _lib.DEVERR_OFFSETS and torch.equal(s["k"], before)


def test_lse_beside_large_values(cuda):
    """What the values' scales ask of a row's outputs leaves its sum of probabilities alone: lse keeps its last bits."""
    from duplex.streaming import kv_cache
    rows, lens = [300, 777, 777], [350, 777, 778]
    s = make(cuda, 3, rows, lens, 2, 2, 64, 16, "int8", torch.bfloat16, seed=41)
    g = torch.Generator(device=cuda).manual_seed(41)
    s["v_scale"] *= torch.exp2(torch.randint(-60, 1, s["v_scale"].shape, generator=g, device=cuda).float())
    for window, sinks in ((1, 0), (1, 5), (2, 1)):                     # a tile's rows see different blocks, and few tokens
        out, lse = kv_cache.kv_attend(s["q"], *cache_args(s), cu_q=s["cu"], window=window, sinks=sinks, softmax_scale=0.00125,
                                      return_lse=True)
        check_rows(s, rows, lens, "int8", window, sinks, out, lse, 0.00125)

"""The clock stack with its attention core (ClockStack.attach_cache): the int4 linears, the 8-bit KV
cache and attention over it, and the MoE of each layer, step by step, against the numpy restatements
and float64 attention; captured steps; eviction in a running session; refusals.

Each part is checked on the stack's own input to it: a code next to a tie of its rounding, or a router
logit next to the last one chosen, may fall the other way for a last-bit difference before it, and what
follows is then another, equally right, result.  (For the same reason the MoE's output is compared for
tokens whose 4th and 5th logits differ by more than 8 fp16 units.)  Bars are test_gpu_clock.py's,
2e-3 of the largest; for the attention those of test_gpu_kv_cache.py, its fp16 output compared with
float64 before rounding."""

import numpy as np
import pytest
import torch

import kv_ref
from oracle.clock_oracle import moe_layer, rms_norm
from oracle.moe_oracle import packed_linear, round_to, router
from test_gpu_clock import small_layers

pytestmark = pytest.mark.gpu

EPS = 1e-6


def build(cuda, T, layers=2, **kw):
    from duplex.clock import ClockStack
    arrays = small_layers(layers)
    st = ClockStack.from_arrays(arrays, top_k=4, device=cuda, T=T, fused=False)
    st.attach_cache(kw.pop("tokens", 64), block=16, head_dim=32 * 2, **kw)
    return arrays, st


def f16(x):
    return np.asarray(round_to(np.asarray(x), "float16"), np.float32)


@pytest.mark.parametrize("T,fmt,window", [(1, "e4m3", 0), (3, "int8", 5)])
def test_steps_vs_oracle(cuda, T, fmt, window):
    arrays, st = build(cuda, T, fmt=fmt, window=window, sinks=1 if window else 0)
    H, D, heads = 256, 64, 4
    rng = np.random.default_rng(5)
    caches = [{n: (torch.zeros(T * 4, 1, 16, D, dtype=torch.float64) if n in ("k", "v") else
                   torch.ones(T * 4, 1, dtype=torch.float64)) for n in ("k", "v", "k_scale", "v_scale")} for _ in arrays]
    table = torch.arange(T * 4).view(T, 4)
    log = []
    real = st._attention

    def attention(i):
        real(i)
        log.append([st.qkv_buf.clone(), st.attn_buf.clone()])

    st._attention = attention
    for L in st.layers:
        def moe(h1, out, _f=L.moe.forward_into, **kw):
            _f(h1, out, **kw)
            log[-1] += [h1.clone(), out.clone()]
        L.moe.forward_into = moe
    num = lambda t: t.float().cpu().numpy()  # noqa: E731

    def near(got, want):
        assert np.abs(got - want).max() <= 2e-3 * np.abs(want).max()

    for step in range(20):                       # into the second block
        x = rng.standard_normal((T, H)).astype(np.float16)
        out = torch.zeros(T, H, device=cuda, dtype=torch.float16)
        log.clear()
        st.step_into(torch.from_numpy(x).to(cuda), out)
        h = x.astype(np.float32)
        lens, ones = [step + 1] * T, [1] * T
        for i, (d, c, (qkv, attn, h1, y)) in enumerate(zip(arrays, caches, log)):
            near(num(qkv), f16(packed_linear(rms_norm(h, EPS), d["qkv_packed"], d["qkv_scale"], d["qkv_zeros"], None, "float16")))
            qkv = qkv.cpu()
            q, k, v = qkv[:, :256].view(T, heads, D), qkv[:, 256:320].view(T, 1, D), qkv[:, 320:].view(T, 1, D)
            kv_ref.append(c, k, v, table, lens, ones, fmt)
            mine = st.caches.layers[i]
            for name in ("k", "v"):
                assert torch.equal(getattr(mine, name).double().cpu(), c[name])
            a, _, mean, bulk, _ = kv_ref.attend(q, c["k"], c["v"], c["k_scale"], c["v_scale"], table, lens, ones, window,
                                                1 if window else 0, D ** -0.5)
            dp = 2.0 ** -19 * bulk + 2.0 ** -21 * (1 + bulk)
            tol = (2.0 ** -11 + 2 * dp + 2.0 ** -19)[..., None] * mean + 2.0 ** -11 * a.abs() + 2.0 ** -24
            assert bool(((attn.cpu().double().view_as(a) - a).abs() <= tol).all())
            o = np.asarray(packed_linear(num(attn), d["o_packed"], d["o_scale"], d["o_zeros"], None, "float16"), np.float32)
            near(num(h1), f16(o + h))
            xn = rms_norm(num(h1), EPS)
            logits = np.sort(np.asarray(router(xn, d["gate_w"], 4, True, None, "float16")[2], np.float32), axis=1)[:, ::-1]
            clear = logits[:, 3] - logits[:, 4] > 8 * 2.0 ** -10 * np.abs(logits[:, 3])
            want = f16(moe_layer(xn, d, 4)[0] + num(h1))
            if clear.any():
                near(num(y)[clear], want[clear])
            h = num(y)
        assert torch.equal(out, log[-1][3])
    assert st.device_errors() == 0 and st.caches.tokens == 20


def test_captured_session_equals_eager(cuda):
    """decode() with its graph, an eviction in between, against eager steps: the same bits."""
    (_, a), (_, b) = (build(cuda, 2, fmt="e4m3", evictable=True, tokens=48) for _ in range(2))
    xs = torch.randn(70, 2, 256, generator=torch.Generator().manual_seed(1)).half()
    host = torch.empty(2, 256, dtype=torch.float16).pin_memory()
    out = torch.zeros(2, 256, device=cuda, dtype=torch.float16)
    for i, x in enumerate(xs):
        if a.caches.tokens == a.caches.capacity:
            for st in (a, b):
                st.evict(keep=20, sinks=2, recent=4)
            assert a.caches.kv_len.tolist() == [20, 20]
        a.decode(x.pin_memory(), host)
        b.step_into(x.to(cuda), out)
        torch.cuda.synchronize()
        assert torch.equal(host, out.cpu()), i
    assert a.caches.tokens == b.caches.tokens == int(a.caches.kv_len[0])
    for ca, cb in zip(a.caches.layers, b.caches.layers):
        assert torch.equal(ca.weights, cb.weights)
    assert a.device_errors() == 0 and b.device_errors() == 0


def test_capture_leaves_the_session_alone(cuda):
    """Capturing in the middle of a block changes nothing of what is cached, whatever x_in holds."""
    _, st = build(cuda, 2, fmt="int8", evictable=True)
    x = torch.randn(2, 256, device=cuda).half()
    out = torch.zeros_like(x)
    for _ in range(5):
        st.step_into(0.01 * x, out)
    state = lambda: [t.clone() for c in st.caches.layers for t in (c.k, c.v, c.k_scale, c.v_scale, c.weights)] + [  # noqa: E731
        st.caches.kv_len.clone()]
    before = state()
    st.x_in.copy_(1000 * x)
    st.capture()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, state())) and st.caches.tokens == 5
    st.replay()
    torch.cuda.synchronize()
    assert st.caches.kv_len.tolist() == [6, 6]


def test_refusals(cuda):
    from duplex.clock import ClockStack
    arrays, st = build(cuda, 1, tokens=16)
    x, out = torch.zeros(1, 256, device=cuda).half(), torch.zeros(1, 256, device=cuda).half()
    for _ in range(16):
        st.step_into(x, out)
    st.capture()
    for call in (lambda: st.step_into(x, out), st.replay, lambda: st.evict(keep=4)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(RuntimeError, match="heads"):
        st.attach_cache(16, head_dim=128)
    with pytest.raises(RuntimeError, match="fused=False"):
        ClockStack(st.layers, 256, 256, device=cuda, fused=True).attach_cache(16)

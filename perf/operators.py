"""The streaming KV cache's operators as measurable cases: what a decoder layer runs between its q|k|v and its o
projection.  `kv_append` stores new keys and values in 8 bits, `kv_attend` is attention over that cache (whole context,
or a sliding window with sink tokens; with or without accumulated attention weights), `kv_evict` keeps the tokens with
the largest accumulated weights.

The cache is paged: k, v [n_blocks, kv_heads, block, dim] in e4m3 or int8, one scale per (block, head), a power of two.
block_table [batch, width] names a sequence's blocks in order, kv_len [batch] counts its tokens (the new ones
included), cu_q [batch + 1] says which rows of q (or of the new keys and values) are whose.
"""

import random
import sys

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
#: the largest code of each format, as (mantissa in [0.5, 1), exponent): 448 and 127
TOP = {"e4m3": (0.875, 9), "int8": (0.9921875, 7)}


def _kv():
    """The framework's module, for `own` alone."""
    if "qwen3-omni-duplex_b200" not in sys.path:
        sys.path.insert(0, "qwen3-omni-duplex_b200")
    from duplex.streaming import kv_cache
    return kv_cache


# ------------------------------------------------------------------ cases
def _case(name, op, batch, rows, kv, **more):
    c = {"name": name, "op": op, "batch": batch, "rows": rows, "kv": kv, "ragged": True, "heads": 32, "kv_heads": 4,
         "dim": 128, "block": 64, "type": "bf16", "codes": "e4m3", "window": 0, "sinks": 0, "weights": False, "keep": 0,
         "recent": 0}
    c.update(more)
    return c


def listed():
    return [
        # attention over the 8-bit cache.  One conversation, one 80 ms frame: latency is all that counts.
        _case("decode 1 x 2k", "attend", 1, 1, 1999),
        # a serving batch at its largest: the cache's bytes are the cost.
        _case("decode 64 x 12k", "attend", 64, 1, 12288),
        # a few drafted tokens a sequence, small heads, small pages, the other code.
        _case("draft 7 x 5, int8", "attend", 7, 5, 3001, heads=16, kv_heads=2, dim=64, block=16, type="fp16", codes="int8"),
        # a prompt's next chunk over what is cached already, ragged.
        _case("chunk 3 x 500 of 6k", "attend", 3, 509, 6100, block=32),
        # a whole long prompt, from an empty cache.
        _case("prompt 8k", "attend", 1, 8192, 8192, ragged=False),
        # sliding window with sinks: long sessions, of which each frame reads the last 4096 tokens and the first 4.
        _case("window decode 48 x 32k", "attend", 48, 1, 32768, window=4096, sinks=4),
        # ... and a prompt under the same kind of mask.
        _case("window prompt 2 x 2k", "attend", 2, 2047, 5000, window=1024, sinks=16, type="fp16", block=128),
        # decode that accumulates its attention weights for a later eviction.
        _case("decode 16 x 6k, weights", "attend", 16, 1, 6000, weights=True),
        # eviction: one conversation that went a little over its budget, and a batch that is halved.
        _case("evict 1 x 4k", "evict", 1, 0, 4203, keep=4000, sinks=4, recent=512, codes="int8"),
        _case("evict 12 x 16k", "evict", 12, 0, 16384, keep=8192, sinks=16, recent=1024),
        # storing: one token each for a batch, and a prompt.
        _case("append 64 x 1", "append", 64, 1, 4097, type="fp16", codes="int8"),
        _case("append 4 x 4k", "append", 4, 4099, 6000, block=32),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attend"] * 5 + ["evict"] * 2 + ["append"] * 2)
    group, kv_heads = rng.choice([1, 4, 6, 8, 16]), rng.choice([1, 2, 4, 5, 8])
    c = {"op": op, "ragged": rng.random() < 0.8, "heads": group * kv_heads, "kv_heads": kv_heads,
         "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64, 128]), "type": rng.choice(["bf16", "fp16"]),
         "codes": rng.choice(["e4m3", "e4m3", "int8"]), "window": 0, "sinks": 0, "weights": False, "keep": 0, "recent": 0,
         "batch": _spread(rng, 1, 64), "rows": 1, "kv": _spread(rng, 64, 32768)}
    if op == "attend":
        if rng.random() < 0.5:
            c["rows"] = _spread(rng, 2, 4096)
        if rng.random() < 0.4:
            c["window"], c["sinks"] = _spread(rng, 16, 8192), rng.choice([0, 1, 4, 16, 100])
        c["weights"] = rng.random() < 0.3
    elif op == "evict":
        c["rows"] = 0
        c["keep"] = max(8, int(c["kv"] * rng.uniform(0.2, 1.0)))
        c["sinks"] = rng.choice([0, 1, 4])
        c["recent"] = rng.randint(0, c["keep"] // 2)
    else:
        c["rows"] = _spread(rng, 1, 4096)
    c["kv"] = max(c["kv"], c["rows"])
    # no more than the largest listed case, in cache and in products
    while c["batch"] > 1 and (c["batch"] * c["kv"] * c["kv_heads"] * c["dim"] > 64 * 12288 * 4 * 128
                              or c["batch"] * max(1, c["rows"]) * c["kv"] * c["heads"] * c["dim"] > 8192 * 4096 * 32 * 128):
        c["batch"] = max(1, c["batch"] // 2)
    while max(1, c["rows"]) * c["kv"] * c["heads"] * c["dim"] > 8192 * 4096 * 32 * 128:
        c["rows"], c["kv"] = c["rows"] // 2, c["kv"] // 2
    return c


def _sizes(c):
    """(rows, lengths) of the sequences: by the case alone, whatever the seed."""
    rng = random.Random("%(op)s %(batch)d %(rows)d %(kv)d %(block)d" % c)
    if not c["ragged"]:
        return [c["rows"]] * c["batch"], [c["kv"]] * c["batch"]
    rows = [c["rows"]] + [rng.randint(min(1, c["rows"]), c["rows"]) for _ in range(c["batch"] - 1)]
    lens = [c["kv"]] + [max(t, rng.randint(c["kv"] // 4, c["kv"])) for t in rows[1:]]
    return rows, lens


def _up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = case
    dev, g = torch.device("cuda"), torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, lens = _sizes(c)
    B, H, D, P = c["batch"], c["kv_heads"], c["dim"], c["block"]
    width = _up(max(lens), P)
    width_dst = _up(c["keep"], P) if c["op"] == "evict" else 0
    n_blocks = B * (width + width_dst) + 3
    order = torch.randperm(n_blocks, generator=g, device=dev).to(torch.int32)
    s = {"case": c, "rows": max(rows), "table": order[: B * width].view(B, width).contiguous(),
         "kv_len": torch.tensor(lens, dtype=torch.int32, device=dev)}
    cu = [0]
    for t in rows:
        cu.append(cu[-1] + t)
    s["cu_q"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    N = cu[-1]

    def noise(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def coded(spread):
        """A filled cache: channels of unlike size, blocks of unlike size, in codes and scales."""
        x = noise(n_blocks, H, P, D)
        x *= spread * (0.3 + noise(H, 1, D).abs())
        x *= torch.exp2(0.7 * noise(n_blocks, H, 1, 1))
        e = _exponent(x.abs().amax((2, 3)), c["codes"])
        return _code(x * torch.exp2(-e)[..., None, None], c["codes"]), torch.exp2(e)

    s["k"], s["k_scale"] = coded(1.0)
    s["v"], s["v_scale"] = coded(0.5)
    t = TYPES[c["type"]]
    if c["op"] == "attend":
        s["q"] = (2.0 * noise(N, c["heads"], D)).to(t)
        if c["weights"]:
            s["weights0"] = noise(n_blocks, H, P).abs() * 0.01
            s["weights"] = s["weights0"].clone()
    elif c["op"] == "append":
        # new rows lie in one q|k|v buffer, as the projection writes them
        qkv = noise(N, (c["heads"] + 2 * H) * D).to(t)
        s["k_new"] = qkv[:, c["heads"] * D: (c["heads"] + H) * D].view(N, H, D)
        s["v_new"] = qkv[:, (c["heads"] + H) * D:].view(N, H, D)
    else:
        s["dst"] = order[B * width: B * (width + width_dst)].view(B, width_dst).contiguous()
        # few heavy tokens, many light ones, and many that were never looked at (equal: ties)
        w = torch.exp(2.0 * noise(n_blocks, H, P) - 4.0)
        s["weights"] = torch.where(w < 0.01, torch.zeros_like(w), w)
    return s


# ------------------------------------------------------------------ plain forms
def _exponent(amax, codes):
    """The scale's exponent: the least e with amax <= top * 2^e, at least -126."""
    m, e = torch.frexp(amax.float())
    top, at = TOP[codes]
    e = e - at + (m > top)
    return torch.where(amax > 0, e, -126).clamp(min=-126).float()


def _code(x, codes):
    """Codes of values that a scale brought into the format's range, ties to even."""
    return x.to(torch.float8_e4m3fn) if codes == "e4m3" else torch.round(x).to(torch.int8)


def _gathered(s, name, scale):
    """A sequence's values in order: [batch, kv_heads, width * block, dim] in 32 bits."""
    x = s[name][s["table"].long()].float() * s[scale][s["table"].long()][..., None, None]
    B, W, H, P, D = x.shape
    return x.transpose(1, 2).reshape(B, H, W * P, D)


def _plain_attend(s):
    c, dev = s["case"], s["q"].device
    H, G, D, P = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["block"]
    N, B, T = s["q"].shape[0], c["batch"], s["rows"]
    cu, n = s["cu_q"].long(), s["kv_len"].long()
    row = torch.arange(N, device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    q = torch.zeros(B, T, c["heads"], D, device=dev)
    q[seq, row - cu[seq]] = s["q"].float()
    q = q.view(B, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    k, v = _gathered(s, "k", "k_scale"), _gathered(s, "v", "v_scale")
    score = (q @ k.transpose(2, 3)).view(B, H, G, T, -1) * D ** -0.5
    at = (n - (cu[1:] - cu[:-1]))[:, None] + torch.arange(T, device=dev)      # position of each row, [B, T]
    j = torch.arange(k.shape[2], device=dev)
    seen = j <= at[..., None]
    if c["window"]:
        seen &= (j > at[..., None] - c["window"]) | (j < c["sinks"])
    seen &= (torch.arange(T, device=dev) < (cu[1:] - cu[:-1])[:, None])[..., None]   # rows of other sequences
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    score /= total.clamp(min=1e-38)
    lse = (top + total.log()).squeeze(-1)
    # a masked value is not looked at: it may be anything
    v = v.masked_fill_((j >= n[:, None])[:, None, :, None], 0.0)
    out = (score.view(B, H, G * T, -1) @ v).view(B, H, G, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, c["heads"], D)
    got = {"out": out[seq, row - cu[seq]].to(s["q"].dtype),
           "lse": lse.permute(0, 3, 1, 2).reshape(B, T, c["heads"])[seq, row - cu[seq]]}
    if c["weights"]:
        add = score.sum((2, 3)).view(B, H, -1, P).transpose(1, 2)
        got["weights"] = s["weights0"].index_put((s["table"].long(),), add, accumulate=True)
    return got


def _plain_append(s):
    c, dev = s["case"], s["k_new"].device
    P, N = c["block"], s["k_new"].shape[0]
    cu, n, table = s["cu_q"].long(), s["kv_len"].long()[:, None], s["table"].long()
    start = n - (cu[1:] - cu[:-1])[:, None]
    # the blocks that new tokens touch; one more than there are stands for the last once more
    col = start // P + torch.arange((s["rows"] - 1) // P + 2, device=dev)
    col = torch.minimum(col, (n - 1) // P).clamp(min=0)
    block = table.gather(1, col)
    slot = col[..., None] * P + torch.arange(P, device=dev)
    old, new = slot < start[..., None], (slot >= start[..., None]) & (slot < n[..., None])
    row = (cu[:-1, None, None] + slot - start[..., None]).clamp(0, N - 1)
    some = new.any(-1)[..., None]
    for x, codes, scales in ((s["k_new"], s["k"], s["k_scale"]), (s["v_new"], s["v"], s["v_scale"])):
        x = (x[row].float() * new[..., None, None]).transpose(2, 3)                          # [B, W, H, P, D]
        was = scales[block]
        e = torch.maximum(_exponent(x.abs().amax((3, 4)), c["codes"]),
                          torch.where(old.any(-1)[..., None], torch.log2(was), -126.0))
        e = torch.where(some, e, torch.log2(was))
        kept = codes[block].float() * (was * torch.exp2(-e))[..., None, None]
        x = torch.where(old[:, :, None, :, None], kept, x * torch.exp2(-e)[..., None, None])
        hold = (old | new)[:, :, None, :, None]
        raw = codes.view(torch.uint8)
        raw[block] = torch.where(hold, _code(x, c["codes"]).view(torch.uint8), raw[block])
        scales[block] = torch.exp2(e)
    return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"]}


def _plain_evict(s):
    c, dev = s["case"], s["k"].device
    B, H, P, D, keep = c["batch"], c["kv_heads"], c["block"], c["dim"], c["keep"]
    n, dst = s["kv_len"].long()[:, None, None], s["dst"].long()
    w = s["weights"][s["table"].long()].transpose(1, 2).reshape(B, H, -1)
    j = torch.arange(w.shape[2], device=dev)
    held = (j < c["sinks"]) | (j >= n - c["recent"])
    rank = torch.where(j < n, torch.where(held, 3e38, w), -3e38)
    at = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values  # [B, H, keep]
    have = torch.arange(dst.shape[1] * P, device=dev) < n.clamp(max=keep)                            # [B, 1, slots]
    at = torch.nn.functional.pad(at, (0, dst.shape[1] * P - at.shape[2])).expand(B, H, -1)
    used = have.view(B, 1, -1, P).any(-1).transpose(1, 2).expand(B, -1, H)
    mask = have.view(B, 1, -1, P).transpose(1, 2).expand(B, -1, H, P)

    def put(into, x):
        into[dst] = torch.where(mask, x.view(B, H, -1, P).transpose(1, 2), into[dst])

    for name in ("k", "v"):
        x = torch.gather(_gathered(s, name, name + "_scale"), 2, at[..., None].expand(-1, -1, -1, D))
        x = (x * have[..., None]).view(B, H, -1, P, D).transpose(1, 2)
        e = _exponent(x.abs().amax((3, 4)), c["codes"])
        x = _code(x * torch.exp2(-e)[..., None, None], c["codes"]).view(torch.uint8)
        raw = s[name].view(torch.uint8)
        raw[dst] = torch.where(mask[..., None], x, raw[dst])
        s[name + "_scale"][dst] = torch.where(used, torch.exp2(e), s[name + "_scale"][dst])
    put(s["weights"], torch.gather(w, 2, at))
    return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"], "weights": s["weights"],
            "kv_len": s["kv_len"].clamp(max=keep)}


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict}[c["op"]](s)
    kv = _kv()
    cache = (s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["kv_len"])
    if c["op"] == "attend":
        if c["weights"]:
            s["weights"].copy_(s["weights0"])     # a pass starts from the same sums each time
        out, lse = kv.kv_attend(s["q"], *cache, cu_q=s["cu_q"], window=c["window"], sinks=c["sinks"],
                                weights=s.get("weights"), return_lse=True)
        got = {"out": out, "lse": lse}
        if c["weights"]:
            got["weights"] = s["weights"]
        return got
    if c["op"] == "append":
        kv.kv_append(s["k_new"], s["v_new"], *cache, cu_q=s["cu_q"])
        return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"]}
    n = kv.kv_evict(*cache, s["weights"], s["dst"], keep=c["keep"], sinks=c["sinks"], recent=c["recent"])
    return {"k": s["k"], "k_scale": s["k_scale"], "v": s["v"], "v_scale": s["v_scale"], "weights": s["weights"],
            "kv_len": n}


# ------------------------------------------------------------------ the least work
def _seen(c, t, n):
    """(tokens that some row of a sequence sees, pairs of a row and a token that it sees)."""
    pairs = 0
    for p in range(n - t, n):
        lo = max(0, p + 1 - c["window"]) if c["window"] else 0
        pairs += p + 1 - lo + min(lo, c["sinks"])
    lo = max(0, n - t + 1 - c["window"]) if c["window"] else 0
    return n - lo + min(lo, c["sinks"]), pairs


def work(case):
    c = case
    rows, lens = _sizes(c)
    H, D, P = c["kv_heads"], c["dim"], c["block"]
    if c["op"] == "attend":
        tokens, pairs = (sum(x) for x in zip(*(_seen(c, t, n) for t, n in zip(rows, lens))))
        n = tokens * H * (2 * D + 8 / P) + sum(rows) * c["heads"] * (4 * D + 4) + (8 * tokens * H if c["weights"] else 0)
        return {"bytes": int(n), "flops": 4 * D * c["heads"] * pairs}
    if c["op"] == "append":
        return {"bytes": int(sum(rows) * H * (2 * 2 * D + 2 * D + 8 / P)), "flops": 2 * sum(rows) * H * D}
    kept = sum(min(n, c["keep"]) for n in lens)
    return {"bytes": int(sum(lens) * H * 4 + kept * H * (4 * D + 4)), "flops": 2 * kept * H * D}


# ------------------------------------------------------------------ 64 bits
def _exact_round(x, codes):
    """The nearest value of the format, ties to even, for |x| within its range."""
    if codes == "int8":
        return torch.round(x)
    step = torch.exp2((torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3))
    return torch.round(x / step) * step


def _exact_scale(x, codes):
    """2^e of the definition, for the values of one block and head."""
    top, e = {"e4m3": 448.0, "int8": 127.0}[codes], -126
    amax = float(x.abs().max()) if x.numel() else 0.0
    while amax > top * 2.0 ** e:
        e += 1
    return 2.0 ** e


def exact(case, seed):
    c = case
    rows, lens = _sizes(c)
    H, G, D, P = c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"], c["block"]
    if c["op"] == "attend" and sum(t * n for t, n in zip(rows, lens)) * c["heads"] > 3e9:
        return None
    if c["op"] != "attend" and sum(max(t, c["keep"] and n) for t, n in zip(rows, lens)) * H // P > 6000:
        return None
    s = prepare(case, seed)
    if c["op"] == "attend":
        out = torch.zeros(sum(rows), c["heads"], D, dtype=torch.float64, device="cuda")
        lse = torch.zeros(sum(rows), c["heads"], dtype=torch.float64, device="cuda")
        weights = s["weights0"].double() if c["weights"] else None
        first = 0
        for b, (t, n) in enumerate(zip(rows, lens)):
            blocks = s["table"][b, : _up(n, P)].long()
            at = torch.arange(n - t, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")
            hidden = j > at
            if c["window"]:
                hidden = hidden | ((j <= at - c["window"]) & (j >= c["sinks"]))
            for h in range(H):
                k = (s["k"][blocks, h].double() * s["k_scale"][blocks, h].double()[:, None, None]).reshape(-1, D)[:n]
                v = (s["v"][blocks, h].double() * s["v_scale"][blocks, h].double()[:, None, None]).reshape(-1, D)[:n]
                total = torch.zeros(n, dtype=torch.float64, device="cuda")
                for i in range(h * G, h * G + G):
                    q = s["q"][first: first + t, i].double()
                    score = (q @ k.T / D ** 0.5).masked_fill(hidden, float("-inf"))
                    lse[first: first + t, i] = torch.logsumexp(score, 1)
                    p = torch.softmax(score, 1)
                    out[first: first + t, i] = p @ v
                    total += p.sum(0)
                if weights is not None:
                    pad = torch.zeros(blocks.numel() * P, dtype=torch.float64, device="cuda")
                    pad[:n] = total
                    weights[blocks, h] += pad.view(-1, P)
            first += t
        got = {"out": out, "lse": lse}
        return got | {"weights": weights} if c["weights"] else got
    got = {"kv_len": None, "weights": s["weights"].double()} if c["op"] == "evict" else {}
    table, target, w = s["table"].cpu(), s.get("dst", s["table"]).cpu(), s["weights"].cpu() if c["op"] == "evict" else None
    picks = {}
    for b, n in enumerate(lens):
        for h in range(H if c["op"] == "evict" else 0):
            mine = w[table[b].long(), h].reshape(-1)[:n].tolist()
            middle = sorted(range(c["sinks"], max(c["sinks"], n - c["recent"])), key=lambda i: (-mine[i], i))
            held = [i for i in range(n) if i < c["sinks"] or i >= n - c["recent"]]
            picks[b, h] = sorted(held + middle[: c["keep"] - len(held)]) if n > c["keep"] else list(range(n))
            for i, p in enumerate(picks[b, h]):
                got["weights"][target[b, i // P], h, i % P] = mine[p]
    for name in ("k", "v"):
        codes, scale = s[name].cpu().double(), s[name + "_scale"].cpu().double()
        new_codes, new_scale = codes.clone(), scale.clone()
        first = 0
        for b, (t, n) in enumerate(zip(rows, lens)):
            for h in range(H):
                if c["op"] == "evict":
                    at = torch.tensor(picks[b, h])
                    page = table[b][at // P].long()
                    x, lo = codes[page, h, at % P] * scale[page, h][:, None], 0
                else:
                    x, lo = s[name + "_new"][first: first + t, h].cpu().double(), n - t
                for i in range(lo // P, _up(lo + len(x), P)):
                    page, a, z = int(target[b, i]), max(lo, i * P), min(lo + len(x), i * P + P)
                    part = x[a - lo: z - lo]
                    two = _exact_scale(part, c["codes"])
                    if a > i * P:
                        two = max(two, float(scale[page, h]))
                        new_codes[page, h, : a - i * P] = _exact_round(codes[page, h, : a - i * P] * float(scale[page, h]) / two, c["codes"])
                    new_codes[page, h, a - i * P: z - i * P] = _exact_round(part / two, c["codes"])
                    new_scale[page, h] = two
            first += t
        got[name], got[name + "_scale"] = (new_codes if c["codes"] == "e4m3" else None), new_scale
    return got

"""The 8-bit paged KV cache's operators in 64 bits, sequence by sequence, for the tests: no code of
the package, and rounding to e4m3 / int8 written out."""

import math

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def rounded(x, fmt):
    """Nearest code value of a float64 tensor within the format's range, ties to even."""
    if fmt == "int8":
        return torch.round(x)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    return torch.round(x / torch.exp2(e - 3)) * torch.exp2(e - 3)


def scale_of(x, fmt):
    """2^e, the least e >= -126 with max|x| <= top * 2^e."""
    amax = float(x.abs().max()) if x.numel() else 0.0
    e = -126 if amax == 0 else max(-126, math.ceil(math.log2(amax / TOP[fmt])) - 1)
    while amax > TOP[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def values(codes, scale, blocks, h, n):
    """Tokens [0, n) of one head: float64 [n, dim]."""
    x = codes[blocks, h].double() * scale[blocks, h].double()[:, None, None]
    return x.reshape(-1, codes.shape[-1])[:n]


def append(cache, k_new, v_new, table, kv_len, rows, fmt):
    """cache: dict of CPU tensors k, v (float64 code values), k_scale, v_scale (float64); in place."""
    P, first = cache["k"].shape[2], 0
    for b, (n, t) in enumerate(zip(kv_len, rows)):
        for name, new in (("k", k_new), ("v", v_new)):
            x = new[first: first + t].double()
            x = torch.where(torch.isfinite(x), x, 0.0)
            for h in range(x.shape[1]):
                for col in range(max(n - t, 0) // P, -(-n // P)):
                    a, z = max(n - t, col * P), min(n, col * P + P)
                    if a >= z:
                        continue
                    blk = int(table[b][col])
                    part = x[a - (n - t): z - (n - t), h]
                    s = scale_of(part, fmt)
                    if a > col * P:
                        old = float(cache[name + "_scale"][blk, h])
                        s = max(s, old)
                        kept = cache[name][blk, h, : a - col * P]
                        cache[name][blk, h, : a - col * P] = rounded(kept * (old / s), fmt)
                    cache[name][blk, h, a - col * P: z - col * P] = rounded(part / s, fmt)
                    cache[name + "_scale"][blk, h] = s
        first += t


def attend(q, k, v, k_scale, v_scale, table, kv_len, rows, window, sinks, scale):
    """Per row and head in float64: out, lse, mean = sum p |v|, bulk = max over seen tokens of
    sum |q_i k_i| * scale; and weights [n_blocks, heads, block] (what a call adds).  Rows that belong
    to no sequence are left at 0."""
    N, Hq, D = q.shape
    H, P = k.shape[1], k.shape[2]
    G = Hq // H
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    out, mean, lse, bulk = z(N, Hq, D), z(N, Hq, D), z(N, Hq), z(N, Hq)
    weights = z(*k.shape[:3])
    first = 0
    for b, (n, t) in enumerate(zip(kv_len, rows)):
        cols = -(-n // P)
        pos = torch.arange(n - t, n, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)
        seen = j <= pos
        if window:
            seen = seen & ((j > pos - window) | (j < sinks))
        blocks = table[b][:cols].long()
        hidden_cols = ~torch.nn.functional.pad(seen, (0, cols * P - n)).view(t, cols, P).any(0).any(-1) if t else None
        blocks = torch.where(hidden_cols, 0, blocks) if t else blocks * 0
        for h in range(H if t else 0):
            kk, vv = values(k, k_scale, blocks, h, n), values(v, v_scale, blocks, h, n)
            kk, vv = kk.nan_to_num(0, 0, 0), vv.nan_to_num(0, 0, 0)
            total = z(cols * P)
            for i in range(h * G, h * G + G):
                x = q[first: first + t, i].double()
                s = (x @ kk.T * scale).masked_fill(~seen, -math.inf)
                l = torch.logsumexp(s, 1)
                p = torch.where(seen, torch.exp(s - torch.where(l == -math.inf, 0, l)[:, None]), 0.0)
                out[first: first + t, i] = p @ vv
                mean[first: first + t, i] = p @ vv.abs()
                lse[first: first + t, i] = l
                if n:
                    bulk[first: first + t, i] = (x.abs() @ kk.abs().T * abs(scale) * seen).amax(1)
                total[:n] += p.sum(0)
            weights.index_put_((blocks, torch.full_like(blocks, h)), total.view(-1, P) * ~hidden_cols[:, None], accumulate=True)
        first += t
    return out, lse, mean, bulk, weights


def kept_tokens(w, n, keep, sinks, recent):
    """The tokens that eviction keeps of one (sequence, head), in order; w: its weights as floats."""
    if n <= keep:
        return list(range(n))
    held = [i for i in range(n) if i < sinks or i >= n - recent]
    big = lambda x: math.inf if x != x else x  # noqa: E731
    middle = sorted(range(sinks, n - recent), key=lambda i: (0 if w[i] != w[i] else 1, -big(w[i]), i))
    return sorted(held + middle[: keep - len(held)])

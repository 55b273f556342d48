"""Paged E4M3 cache in plain 64-bit torch on the CPU: the formulas of the header, one sequence, block and head at a time."""
import math

import torch

F64 = torch.float64


def codes(t):
    """E4M3 bytes -> values."""
    return t.view(torch.float8_e4m3fn).to(F64)


def rope_table(rows, d, base=10000.0):
    angle = torch.arange(rows, dtype=F64)[:, None] * base ** (-torch.arange(0, d, 2, dtype=F64) / d)
    return torch.stack([angle.cos(), angle.sin()], -1).reshape(rows, d).to(torch.float32)


def rotate(x, rope, halves):
    """x (tokens, heads, d) float64, rope (tokens, d)."""
    cos, sin = rope[:, None, 0::2].to(F64), rope[:, None, 1::2].to(F64)
    d = x.shape[-1]
    lo, hi = (slice(0, d // 2), slice(d // 2, d)) if halves else (slice(0, d, 2), slice(1, d, 2))
    y = x.clone()
    y[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    y[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return y


def pages(lens, block, pool, seed, width=None):
    """Block table with entries in random order; -1 behind a sequence's last block."""
    g = torch.Generator().manual_seed(seed)
    need = [(max(n, 0) + block - 1) // block for n in lens]
    assert sum(need) <= pool
    ids = torch.randperm(pool, generator=g)[:sum(need)].tolist()
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(ids[:n], dtype=torch.int32)
        ids = ids[n:]
    return table


def attention(q, kc, vc, ks, vs, table, cu, lens, scale, cap=0.0, window=0, causal=True):
    """q (tokens, hq, d); caches of bytes.  (o, lse, mean of |v| under the weights, sum of |q||k| scale) in 64 bits."""
    tokens, hq, d = q.shape
    hkv, block = kc.shape[1], kc.shape[2]
    o = torch.zeros(tokens, hq, d, dtype=F64)
    size = torch.zeros(tokens, hq, d, dtype=F64)
    lse = torch.full((hq, tokens), -math.inf, dtype=F64)
    reach = torch.zeros(hq, tokens, dtype=F64)
    for b, n_all in enumerate(lens):
        new = cu[b + 1] - cu[b]
        for h in range(hkv):
            ids = [(j, int(table[b, j // block])) for j in range(n_all)]
            ids = [(j, p) for j, p in ids if 0 <= p < kc.shape[0]]
            if not ids:
                continue
            at = torch.tensor([j for j, _ in ids])
            pg = torch.tensor([p for _, p in ids])
            k = codes(kc[pg, h, at % block]) * ks[pg, h].to(F64)[:, None]
            v = codes(vc[pg, h, at % block]) * vs[pg, h].to(F64)[:, None]
            for i in range(new):
                pos = n_all - new + i
                seen = torch.ones(len(at), dtype=torch.bool)
                if causal:
                    seen &= at <= pos
                if window:
                    seen &= at > pos - window
                if not seen.any():
                    continue
                for hh in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    x = q[cu[b] + i, hh].to(F64)
                    s = k[seen] @ x * scale
                    if cap:
                        s = cap * torch.tanh(s / cap)
                    w = torch.softmax(s, 0)
                    o[cu[b] + i, hh] = w @ v[seen]
                    size[cu[b] + i, hh] = w @ v[seen].abs()
                    lse[hh, cu[b] + i] = torch.logsumexp(s, 0)
                    reach[hh, cu[b] + i] = (k[seen].abs() @ x.abs()).max() * scale
    return o, lse, size, reach

"""Plain statements, in Python integers and 64-bit floats on the CPU, of the operators around a decode step with drafted tokens."""
import numpy as np
import torch

F64 = torch.float64


def e4m3(x):
    """Nearest E4M3 value, ties to even: 3 bits behind the leading one, steps of 2^-9 below 2^-6, at most 448; NaN: -448."""
    x = torch.where(x.isnan(), -448.0, x).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def fp8_groups(x):
    """bf16 (rows, dim) -> values of the codes (fp64), scales (groups, rows) fp32."""
    rows, dim = x.shape
    g = (dim + 127) // 128
    v = torch.zeros(rows, g * 128, dtype=F64)
    v[:, :dim] = x.to(F64)
    v = v.view(rows, g, 128)
    top = torch.where(v.isfinite(), v.abs(), 0.0).amax(2).clamp_min(float(torch.tensor(448e-12)))      # the header's bound, an fp32 number
    codes = e4m3(v * 448 / top[:, :, None]).view(rows, g * 128)[:, :dim]
    return codes, (top.float() / 448.0).t().contiguous()


def block_product(a, w, a_scale, w_scale):
    """Codes as values in fp64, scales in fp32 -> (product in fp64, sum of magnitudes)."""
    m, k = a.shape
    n = w.shape[0]
    sw = w_scale.to(F64).repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    sa = a_scale.to(F64).t().repeat_interleave(128, 1)[:, :k]
    x, y = a.to(F64) * sa, w.to(F64) * sw
    return x @ y.T, x.abs() @ y.abs().T


def softmax_rows(x, t):
    x = torch.where(x.isnan(), -torch.inf, x.to(F64))
    out = torch.zeros(x.shape, dtype=F64)
    for r in range(x.shape[0]):
        top = float(x[r].max())
        if top == -np.inf:
            continue
        if not t[r] > 0:
            out[r, int((x[r] == top).nonzero()[0])] = 1.0
        elif top == np.inf:
            hit = x[r] == top
            out[r] = hit / hit.sum()
        else:
            e = torch.where(x[r] == -torch.inf, 0.0, torch.exp((x[r] - top) / float(t[r])))
            out[r] = e / e.sum()
    return out


def verify(p, q, tokens, cu, lens, u, v):
    """Lists of (out, or None behind and in front of the sequences), accepted, kept; p and q fp32 arrays."""
    n, vocab = p.shape
    out, accepted, kept = [None] * n, [], []
    for b in range(len(cu) - 1):
        t, end = cu[b], cu[b + 1] - 1
        if t < 0 or end + 1 > n or end < t:
            accepted.append(0)
            kept.append(lens[b])
            continue
        stood = 0
        while t < end:
            d = tokens[t + 1]
            if not (0 <= d < vocab and float(u[t]) * (float(q[t, d]) if q is not None else 1.0) < float(p[t, d])):
                break
            out[t] = d
            t, stood = t + 1, stood + 1
        w = p[t].astype(np.float64)
        if t < end:
            r = w.copy()
            if q is not None:
                r = np.maximum(r - q[t].astype(np.float64), 0.0)
            elif 0 <= tokens[t + 1] < vocab:
                r[tokens[t + 1]] = 0.0
            if r.sum() > 0:
                w = r
        token = -1
        if w.sum() > 0:
            upto = np.cumsum(w)
            at = min(max(float(v[b]), 0.0), float(np.float32(0.99999994))) if v[b] == v[b] else 0.0
            token = min(int(np.searchsorted(upto, at * upto[-1], side="right")), int(np.nonzero(w)[0][-1]))
        out[t] = token
        for i in range(t + 1, end + 1):
            out[i] = -1
        accepted.append(stood)
        kept.append(lens[b] - (end - t))
    return out, accepted, kept


def blocks_of(n, bs):
    return -(-max(n, 0) // bs)


def release(kept, lens, table, free, count, pool, bs):
    """Changes `table` (a list of rows) and `free`; returns the new count."""
    stride = len(table[0]) if table else 0
    count = min(max(count, 0), pool)
    gone = []
    for b, row in enumerate(table):
        for j in range(blocks_of(kept[b], bs), min(blocks_of(lens[b], bs), stride)):
            if 0 <= row[j] < pool:
                gone.append(row[j])
                row[j] = -1
    for i, page in enumerate(reversed(gone)):
        if count + i < pool:
            free[count + i] = page
    return min(count + len(gone), pool)


def plan(kept, new, table, free, count, pool, bs, tokens):
    """Changes `table`; returns (count, cu, lens, positions, slots, refused)."""
    stride = len(table[0]) if table else 0
    count = min(max(count, 0), pool)
    cu, lens, pos, slot, refused, full, took, asked = [0], [], [], [], 0, False, 0, 0
    for b, row in enumerate(table):
        k, n = kept[b], new[b]
        fits = k >= 0 and n >= 0 and blocks_of(k + n, bs) <= stride and k + n < 2 ** 31
        need = blocks_of(k + n, bs) - blocks_of(k, bs) if fits else 0
        asked += n if fits else 0
        full = full or took + need > count or asked > tokens
        if full or not fits:
            refused += 1
            lens.append(max(k, 0))
            cu.append(cu[-1])
            continue
        for j in range(blocks_of(k, bs), blocks_of(k + n, bs)):
            took += 1
            row[j] = free[count - took]
        for at in range(k, k + n):
            page = row[at // bs]
            pos.append(at)
            slot.append(page * bs + at % bs if 0 <= page < pool else -1)
        lens.append(k + n)
        cu.append(cu[-1] + n)
    pad = [-1] * (tokens - len(pos))
    return count - took, cu, lens, pos + pad, slot + pad, refused

"""Operators of 8-bit language-model serving, as they are measured: plain forms, the library's calls, definitions in 64 bits.

``append``   new tokens of a packed QKV projection: queries rotated, keys rotated, keys and values stored in a paged E4M3 cache
             with one scale per (block, head)
``attend``   attention of those queries over that cache: one token per sequence, a few, or a chunk of a prompt
``project``  activations quantised to 8-bit integers with a scale per token, then the product with 8-bit integer weights that
             have a scale per output channel

``own`` False: ``run`` is the plain form (elementary torch operations in fp32).  ``own`` True: the library's entry points.
"""
import math

import torch

own = False

BF16, E4M3, F32, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64
HEADS = ((8, 1), (32, 8), (8, 8), (12, 2), (40, 8), (28, 4), (16, 1))     # (query, key/value) heads


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one control step of a robot policy's language backbone (8 query heads on one KV head of 256) writes its next token
        {"name": "append_one_token", "op": "append", "batch": 1, "new": 1, "ctx": 819, "hq": 8, "hkv": 1, "d": 256, "block": 16, "halves": False},
        # a full decode batch, every sequence at a length of its own
        {"name": "append_decode_batch", "op": "append", "batch": 96, "new": 1, "ctx": 4099, "hq": 32, "hkv": 8, "d": 128, "block": 32, "halves": True},
        # prompts of uneven lengths entering the cache at once
        {"name": "append_prompts", "op": "append", "batch": 5, "new": 2731, "ctx": 2731, "hq": 32, "hkv": 8, "d": 128, "block": 64, "halves": True},
        # decode of one short sequence: the smallest call
        {"name": "attend_one_token", "op": "attend", "batch": 1, "new": 1, "ctx": 819, "hq": 8, "hkv": 1, "d": 256, "block": 16, "cap": 0.0, "window": 0, "causal": True},
        # a decode batch of ordinary lengths
        {"name": "attend_decode_batch", "op": "attend", "batch": 64, "new": 1, "ctx": 6001, "hq": 32, "hkv": 8, "d": 128, "block": 32, "cap": 0.0, "window": 0, "causal": True},
        # two very long documents: the work has to be split along the keys
        {"name": "attend_long_context", "op": "attend", "batch": 2, "new": 1, "ctx": 131071, "hq": 32, "hkv": 8, "d": 128, "block": 128, "cap": 0.0, "window": 0, "causal": True},
        # drafted tokens checked against a model with capped scores and a sliding window
        {"name": "attend_drafted", "op": "attend", "batch": 16, "new": 5, "ctx": 3777, "hq": 28, "hkv": 4, "d": 128, "block": 16, "cap": 50.0, "window": 2048, "causal": True},
        # a chunk of a long prompt behind what the cache holds already: the largest
        {"name": "attend_prompt_chunk", "op": "attend", "batch": 2, "new": 2048, "ctx": 8191, "hq": 32, "hkv": 8, "d": 128, "block": 64, "cap": 0.0, "window": 0, "causal": True},
        # one token through a backbone's QKV projection (2048 -> 2560)
        {"name": "project_one_token", "op": "project", "m": 1, "n": 2560, "k": 2048, "bias": False},
        # a decode batch through its gate|up projection (2048 -> 32768)
        {"name": "project_decode_batch", "op": "project", "m": 96, "n": 32768, "k": 2048, "bias": False},
        # a policy's prefix through its down projection (16384 -> 2048), odd row count
        {"name": "project_prefix", "op": "project", "m": 817, "n": 2048, "k": 16384, "bias": True},
        # prompts of a batch
        {"name": "project_prompts", "op": "project", "m": 8191, "n": 4096, "k": 4096, "bias": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "project"))
    if op == "project":
        while True:
            c = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 32768), "k": 16 * _log(rng, 4, 1024), "bias": rng.random() < 0.5}
            if c["m"] * c["n"] * c["k"] <= 8191 * 4096 * 4096 and c["n"] * c["k"] <= 1 << 27:
                return c
    hq, hkv = rng.choice(HEADS)
    c = {"op": op, "hq": hq, "hkv": hkv, "d": rng.choice((64, 128, 256)), "block": rng.choice((16, 32, 64, 128))}
    if op == "append":
        new = rng.choice((1, 1, _log(rng, 2, 4096)))
        batch = _log(rng, 1, max(1, min(128, 8192 // new)))
        return {**c, "batch": batch, "new": new, "ctx": new + (0 if rng.random() < 0.3 else _log(rng, 1, 4096)), "halves": rng.random() < 0.5}
    c.update(cap=rng.choice((0.0, 0.0, 30.0)), causal=rng.random() < 0.85)
    while True:
        new = rng.choice((1, 1, _log(rng, 2, 8), _log(rng, 9, 2048)))
        batch, ctx = _log(rng, 1, 128), _log(rng, new, 131072)
        if batch * ctx * hkv * c["d"] <= 1 << 28 and batch * hq * new * ctx <= 1 << 30 and batch * hq * new * ctx * c["d"] <= 1 << 37:
            window = _log(rng, 16, 4096) if c["causal"] and rng.random() < 0.3 else 0
            return {**c, "batch": batch, "new": new, "ctx": ctx, "window": window}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(case):
    """(new tokens, tokens after this call) of every sequence: the first one has the case's figures, the others lie evenly spread
    below them, in no order; prompts of more than 8 tokens are ragged too."""
    new, ctx = [case["new"]], [case["ctx"]]
    for i in range(1, case["batch"]):
        f, g = (i * 0.6180339887) % 1.0, (i * 0.7548776662) % 1.0
        n = case["new"] if case["new"] <= 8 else max(1, int(case["new"] * (0.25 + 0.75 * g)))
        new.append(n)
        ctx.append(n + int((case["ctx"] - case["new"]) * (0.25 + 0.75 * f)))
    return new, ctx


def _pages(ctx, block, g):
    """A pool with some blocks more than needed, handed out in random order; entries behind a sequence's last block are -1."""
    need = [(n + block - 1) // block for n in ctx]
    total = sum(need)
    pool = total + 3 + total // 16
    ids = torch.randperm(pool, generator=g, device="cuda")[:total].to(torch.int32)
    n = torch.tensor(need, device="cuda")
    col = torch.arange(max(need), device="cuda")
    table = torch.full((len(ctx), max(need)), -1, dtype=torch.int32, device="cuda")
    table[col[None] < n[:, None]] = ids
    return pool, table


def _rows(shape, g):
    """Activations of a projection: normal, with a spread of channels and a few strong ones."""
    chan = torch.exp(0.4 * torch.randn(shape[-1], generator=g, device="cuda"))
    chan[torch.randint(0, shape[-1], (max(1, shape[-1] // 256),), generator=g, device="cuda")] *= 6.0
    return torch.randn(shape, generator=g, device="cuda") * chan


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] == "project":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _rows((m, k), g).to(BF16)
        s["w"] = torch.randn(n, k, generator=g, device="cuda").mul_(40.0).clamp_(-127, 127).to(torch.int8)
        s["w_scale"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / (40.0 * math.sqrt(k))
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(BF16) if case["bias"] else None
        if own:
            from flashrt_b200 import flash_rt_kernels as fvk
            s["gemm"] = fvk.GemmRunner()
            s["q"] = torch.empty(m, k, dtype=torch.int8, device="cuda")
            s["x_scale"] = torch.empty(m, dtype=F32, device="cuda")
            s["out"] = torch.empty(m, n, dtype=BF16, device="cuda")
        return s
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    new, ctx = _lengths(case)
    tokens = sum(new)
    pool, s["table"] = _pages(ctx, block, g)
    s["max_new"], s["max_ctx"], s["tokens"] = max(new), max(ctx), tokens
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    s["cu"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    # what earlier calls left in the pool: per block and head the largest value is near the type's end
    for name in ("k", "v"):
        s[name + "_scale"] = (2.5 + 2.0 * torch.rand(pool, hkv, generator=g, device="cuda")) / 448.0
        code = torch.randn(pool, hkv, block, d, generator=g, device="cuda", dtype=BF16)
        code.div_(s[name + "_scale"][:, :, None, None].to(BF16)).clamp_(-448, 448)
        s[name] = code.to(E4M3)
    if case["op"] == "append":
        s["qkv"] = torch.randn(tokens, (hq + 2 * hkv) * d, generator=g, device="cuda").to(BF16)
        angle = torch.arange(max(ctx), dtype=F64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=F64, device="cuda") / d)
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).reshape(-1, d).to(F32)       # [cos0, sin0, cos1, sin1, ...]
        if own:
            s["q"] = torch.empty(tokens, hq * d, dtype=BF16, device="cuda")
        return s
    s["q"] = torch.randn(tokens, hq * d, generator=g, device="cuda").to(BF16)
    if own:
        from flashrt_b200 import flash_rt_fa2 as fa2
        s["o"] = torch.empty(tokens, hq * d, dtype=BF16, device="cuda")
        s["lse"] = torch.empty(hq, tokens, dtype=F32, device="cuda")
        n = fa2.paged_workspace_bytes(tokens, case["batch"], s["max_new"], hq, hkv, d)
        s["work"] = torch.zeros(n, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"append": _append, "attend": _attend, "project": _project}[s["case"]["op"]](s)


def _append(s):
    c = s["case"]
    hq, hkv, d, block = c["hq"], c["hkv"], c["d"], c["block"]
    out = {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if own:
        from flashrt_b200 import flash_rt_kernels as fvk
        fvk.paged_kv_append_fp8(s["qkv"].data_ptr(), s["rope"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                                s["k_scale"].data_ptr(), s["v_scale"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                                0 if s["max_new"] == 1 else s["cu"].data_ptr(), s["ctx"].data_ptr(), s["tokens"], c["batch"],
                                s["k"].shape[0], block, hq, hkv, d, s["rope"].shape[0], torch.cuda.current_stream().cuda_stream,
                                halves=c["halves"])
        return {**out, "q": s["q"]}
    x = s["qkv"].float()
    at = torch.arange(x.shape[0], device="cuda")
    seq = torch.searchsorted(s["cu"], at, right=True, out_int32=True).long() - 1
    pos = (s["ctx"][seq] - (s["cu"][seq + 1] - at)).long()
    rope = s["rope"][pos].view(-1, 1, d // 2, 2)
    cos, sin = rope[..., 0], rope[..., 1]

    def turn(y, heads):
        y = y.view(-1, heads, 2, d // 2).transpose(2, 3) if c["halves"] else y.view(-1, heads, d // 2, 2)
        z = torch.stack([y[..., 0] * cos - y[..., 1] * sin, y[..., 1] * cos + y[..., 0] * sin], -1)
        return (z.transpose(2, 3) if c["halves"] else z).reshape(-1, heads, d)

    out["q"] = turn(x[:, :hq * d], hq).reshape(-1, hq * d).to(BF16)
    page, slot = s["table"][seq, pos // block].long(), pos % block
    first = torch.full((s["k"].shape[0],), block, dtype=torch.long, device="cuda").index_reduce_(0, page, slot, "amin")
    touched = torch.nonzero(first < block)[:, 0]
    held = torch.arange(block, device="cuda")[None, :] < first[touched][:, None]                   # (touched, block)
    for name, y in (("k", turn(x[:, hq * d:(hq + hkv) * d], hkv)), ("v", x[:, (hq + hkv) * d:].reshape(-1, hkv, d))):
        cache, scale = s[name].view(torch.uint8), s[name + "_scale"]
        top = torch.where(y.isfinite(), y.abs(), 0.0).amax(-1)
        grown = torch.zeros_like(scale).index_reduce_(0, page, top, "amax")[touched] / 448.0
        old = torch.where(held[:, :1], scale[touched], 0.0)
        now = torch.maximum(old, grown).clamp_min(1e-12)
        was = cache[touched]
        back = (was.view(E4M3).float() * (old / now)[:, :, None, None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
        cache[touched] = torch.where(held[:, None, :, None], back, was)
        scale[touched] = now
        code = (y * (1.0 / scale[page])[:, :, None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
        cache[page, :, slot] = code
    return out


def _attend(s):
    c = s["case"]
    hq, hkv, d, block, cap = c["hq"], c["hkv"], c["d"], c["block"], c["cap"]
    if own:
        from flashrt_b200 import flash_rt_fa2 as fa2
        fa2.paged_fwd_fp8(s["q"].data_ptr(), s["o"].data_ptr(), s["lse"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                          s["k_scale"].data_ptr(), s["v_scale"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1],
                          0 if s["max_new"] == 1 else s["cu"].data_ptr(), s["ctx"].data_ptr(), s["tokens"], c["batch"], s["max_new"],
                          s["k"].shape[0], block, hq, hkv, d, 1.0 / math.sqrt(d), s["work"].data_ptr(), s["work"].numel(),
                          torch.cuda.current_stream().cuda_stream, softcap=cap, window=c["window"], causal=c["causal"])
        return {"o": s["o"], "lse": s["lse"]}
    group = hq // hkv
    page = s["table"].long().clamp_min(0)
    batch, keys = page.shape[0], page.shape[1] * block
    k, v = ((s[n][page].float() * s[n + "_scale"][page][..., None, None]).transpose(1, 2).reshape(batch, hkv, keys, d) for n in ("k", "v"))
    n_new = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(s["max_new"], device="cuda")
    there = i[None] < n_new[:, None]                                                               # (batch, new)
    token = torch.where(there, s["cu"][:-1, None] + i[None], 0).long()
    q = s["q"].float()[token].view(batch, -1, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)).view(batch, hkv, group, -1, keys).mul_(1.0 / math.sqrt(d))
    if cap:
        score = torch.tanh(score / cap) * cap
    key, length = torch.arange(keys, device="cuda"), s["ctx"][:, None]
    pos = (length - n_new[:, None] + i[None])[:, :, None]
    seen = (key < length)[:, None, :].expand(-1, s["max_new"], -1)
    if c["causal"]:
        seen = seen & (key <= pos)
        if c["window"]:
            seen = seen & (key > pos - c["window"])
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(batch, hkv, -1, keys), v).view(batch, hkv, group, -1, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, -1, hq * d)[there].to(BF16)
    lse = (top + total.log()).squeeze(-1).permute(1, 2, 0, 3).reshape(hq, batch, -1)[:, there]
    return {"o": o, "lse": lse}


def _project(s):
    if own:
        st = torch.cuda.current_stream().cuda_stream
        from flashrt_b200 import flash_rt_kernels as fvk
        m, n, k = s["case"]["m"], s["case"]["n"], s["case"]["k"]
        fvk.quantize_int8_rows(s["x"].data_ptr(), s["q"].data_ptr(), s["x_scale"].data_ptr(), m, k, st)
        s["gemm"].int8_nt(s["q"].data_ptr(), s["w"].data_ptr(), s["out"].data_ptr(), m, n, k, s["x_scale"].data_ptr(),
                          s["w_scale"].data_ptr(), st, bias=s["bias"].data_ptr() if s["bias"] is not None else 0)
        return s["out"]
    x = s["x"].float()
    scale = (torch.where(x.isfinite(), x.abs(), 0.0).amax(1, keepdim=True) / 127.0).clamp_min(1e-12)
    q = torch.round(x * (1.0 / scale)).clamp(-127, 127)
    y = torch.matmul(q, s["w"].float().t()) * scale * s["w_scale"]
    return (y if s["bias"] is None else y + s["bias"].float()).to(BF16)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "project":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    hq, hkv, d, block = case["hq"], case["hkv"], case["d"], case["block"]
    new, ctx = _lengths(case)
    tokens, batch = sum(new), case["batch"]
    if case["op"] == "append":
        blocks = sum((c - 1) // block - (c - n) // block + 1 for n, c in zip(new, ctx))
        return {"bytes": tokens * d * (2 * (hq + 2 * hkv) + 4 + 2 * hq + 2 * hkv) + blocks * (8 * hkv + 4) + 4 * batch,
                "flops": tokens * d * (3 * (hq + hkv) + 4 * hkv)}
    seen = read = 0                                                    # (query, key) pairs; keys that any query sees
    for n, c in zip(new, ctx):
        w = case["window"] or c
        seen += sum(min(w, c - n + i + 1) for i in range(n)) if case["causal"] else n * c
        read += min(c, w + n - 1)
    return {"bytes": int(read * hkv * (2 * d + 8 / block) + 4 * read / block + tokens * hq * (4 * d + 4) + 8 * batch),
            "flops": hq * seen * (4 * d + 5)}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append64, "attend": _attend64, "project": _project64}[case["op"]](s)


def _e4m3(x):
    """Nearest E4M3 value, ties to even: 3 bits behind the leading one, steps of 2^-9 below 2^-6, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _append64(s):
    c = s["case"]
    hq, hkv, d, block = c["hq"], c["hkv"], c["d"], c["block"]
    cu, ctx, table = s["cu"].tolist(), s["ctx"].tolist(), s["table"].tolist()
    out = {"q": torch.zeros(s["tokens"], hq * d, dtype=F64, device="cuda")}
    for name in ("k", "v"):
        out[name], out[name + "_scale"] = s[name].to(F64), s[name + "_scale"].to(F64)
    lo, hi = (slice(0, d // 2), slice(d // 2, d)) if c["halves"] else (slice(0, d, 2), slice(1, d, 2))
    for b in range(c["batch"]):
        x = s["qkv"][cu[b]:cu[b + 1]].to(F64).view(-1, hq + 2 * hkv, d)
        p0, p1 = ctx[b] - x.shape[0], ctx[b]
        cos, sin = (s["rope"][p0:p1, j::2].to(F64)[:, None] for j in (0, 1))
        r = x[:, :hq + hkv].clone()
        r[..., lo] = x[:, :hq + hkv, lo] * cos - x[:, :hq + hkv, hi] * sin
        r[..., hi] = x[:, :hq + hkv, hi] * cos + x[:, :hq + hkv, lo] * sin
        out["q"][cu[b]:cu[b + 1]] = r[:, :hq].reshape(-1, hq * d)
        for j in range(p0 // block, (p1 + block - 1) // block):
            page, a, e = table[b][j], max(p0, j * block), min(p1, (j + 1) * block)
            keep = a - j * block
            for name, y in (("k", r[a - p0:e - p0, hq:]), ("v", x[a - p0:e - p0, hq + hkv:])):
                old = out[name + "_scale"][page].clone() if keep else torch.zeros(hkv, dtype=F64, device="cuda")
                now = torch.maximum(old, y.abs().amax((0, 2)) / 448).clamp_min(1e-12)
                cache = out[name][page]
                if keep:
                    cache[:, :keep] = _e4m3(cache[:, :keep] * (old / now)[:, None, None])
                cache[:, keep:e - j * block] = _e4m3(y.transpose(0, 1) / now[:, None, None])
                out[name + "_scale"][page] = now
    return out


def _attend64(s):
    c = s["case"]
    hq, hkv, d, block = c["hq"], c["hkv"], c["d"], c["block"]
    group = hq // hkv
    cu, ctx = s["cu"].tolist(), s["ctx"].tolist()
    o = torch.zeros(s["tokens"], hq, d, dtype=F64, device="cuda")
    lse = torch.zeros(hq, s["tokens"], dtype=F64, device="cuda")
    for b in range(c["batch"]):
        n, length = cu[b + 1] - cu[b], ctx[b]
        page = s["table"][b, :(length + block - 1) // block].long()
        key = torch.arange(length, device="cuda")
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = torch.zeros(n, length, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden = key > pos
            if c["window"]:
                hidden |= key <= pos - c["window"]
        for h in range(hkv):
            k, v = ((s[m][page, h].to(F64) * s[m + "_scale"][page, h].to(F64)[:, None, None]).reshape(-1, d)[:length] for m in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                w = s["q"][cu[b]:cu[b + 1], j * d:(j + 1) * d].to(F64) @ k.T / math.sqrt(d)
                if c["cap"]:
                    w = c["cap"] * torch.tanh(w / c["cap"])
                w = w.masked_fill(hidden, -math.inf)
                lse[j, cu[b]:cu[b + 1]] = torch.logsumexp(w, -1)
                o[cu[b]:cu[b + 1], j] = torch.softmax(w, -1) @ v
    return {"o": o.view(-1, hq * d), "lse": lse}


def _project64(s):
    x = s["x"].to(F64)
    scale = (x.abs().amax(1) / 127).clamp_min(1e-12)
    q = torch.round(x / scale[:, None]).clamp(-127, 127)
    y = (q @ s["w"].to(F64).T) * scale[:, None] * s["w_scale"].to(F64)
    return y if s["bias"] is None else y + s["bias"].to(F64)

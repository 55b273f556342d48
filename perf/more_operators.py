"""Operators around a language model's decode step with drafted tokens, as they are measured: plain forms, the library's calls,
definitions in 64 bits.

``project``  activations quantised to E4M3 with a scale for each row and group of 128, then the product with E4M3 weights that have a
             scale for each 128 x 128 block
``probs``    logits to probabilities, a temperature for each row (0: all on the largest)
``verify``   drafted tokens against those probabilities, from given random numbers: how many stand, and the token behind them
``blocks``   between two steps of a server: blocks of dropped tokens go back to the paged cache's free list, the next tokens get theirs;
             block table, packed offsets, positions and slots

``own`` False: ``run`` is the plain form (elementary torch operations; fp32, fp64 where tokens are chosen).  ``own`` True: the library's
entry points.
"""
import math

import torch

own = False

BF16, E4M3, F32, F64, I32, I64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64, torch.int32, torch.int64


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a robot policy's language backbone through its QKV projection (2048 -> 2560): the smallest product
        {"name": "project_one_token", "op": "project", "m": 1, "n": 2560, "k": 2048, "bias": False, "f32": False},
        # a decode batch through the gate|up projection (2048 -> 32768)
        {"name": "project_decode_batch", "op": "project", "m": 96, "n": 32768, "k": 2048, "bias": False, "f32": False},
        # sixteen sequences with four drafted tokens each into the logits of a large vocabulary
        {"name": "project_logits", "op": "project", "m": 80, "n": 131072, "k": 2048, "bias": False, "f32": True},
        # a policy's prefix through its down projection (16384 -> 2048), odd row count
        {"name": "project_prefix", "op": "project", "m": 817, "n": 2048, "k": 16384, "bias": True, "f32": False},
        # prompts of a batch: the largest
        {"name": "project_prompts", "op": "project", "m": 8191, "n": 4096, "k": 4096, "bias": False, "f32": False},
        # the next token of one sequence, an odd vocabulary
        {"name": "probs_one_row", "op": "probs", "rows": 1, "vocab": 50257, "f32": False},
        # 64 sequences with five drafted tokens each, every sequence at a temperature of its own
        {"name": "probs_drafted_batch", "op": "probs", "rows": 384, "vocab": 131072, "f32": True},
        # one sequence with four drafted tokens
        {"name": "verify_one", "op": "verify", "batch": 1, "drafts": 4, "vocab": 50257, "q": True},
        # the batch of 64 with five drafted tokens each
        {"name": "verify_batch", "op": "verify", "batch": 64, "drafts": 5, "vocab": 131072, "q": True},
        # one sequence whose drafted tokens did not stand
        {"name": "blocks_one", "op": "blocks", "batch": 1, "ctx": 819, "new": 5, "block": 16},
        # a full batch with six tokens a step, some slots with the prompt of a new request
        {"name": "blocks_drafted_batch", "op": "blocks", "batch": 256, "ctx": 8191, "new": 6, "block": 32},
        # requests with long prompts take the place of ended ones
        {"name": "blocks_prompts", "op": "blocks", "batch": 61, "ctx": 65536, "new": 4096, "block": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("project", "project", "probs", "verify", "blocks"))
    while op == "project":
        c = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 131072), "k": 16 * _log(rng, 4, 1024), "bias": rng.random() < 0.5,
             "f32": rng.random() < 0.3}
        if c["m"] * c["n"] * c["k"] <= 8191 * 4096 * 4096 and c["n"] * c["k"] <= 1 << 28 and c["m"] * c["n"] <= 1 << 25:
            return c
    while op == "probs":
        c = {"op": op, "rows": _log(rng, 1, 4096), "vocab": _log(rng, 500, 262144), "f32": rng.random() < 0.5}
        if c["rows"] * c["vocab"] <= 384 * 131072:
            return c
    while op == "verify":
        c = {"op": op, "batch": _log(rng, 1, 256), "drafts": rng.randint(0, 16), "vocab": _log(rng, 500, 262144), "q": rng.random() < 0.7}
        if c["batch"] * (c["drafts"] + 1) * c["vocab"] <= 384 * 131072:
            return c
    while True:
        c = {"op": op, "batch": _log(rng, 1, 1024), "ctx": _log(rng, 1, 131072), "new": rng.choice((1, rng.randint(2, 8), _log(rng, 9, 8192))),
             "block": rng.choice((16, 32, 64, 128))}
        if c["batch"] * (c["ctx"] + c["new"]) <= 1 << 24 and c["batch"] * c["new"] <= 1 << 18:
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(m, k, g):
    """Normal, with a spread of channels and a few strong ones."""
    chan = torch.exp(0.4 * torch.randn(k, generator=g, device="cuda"))
    chan[torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] *= 6.0
    return (torch.randn(m, k, generator=g, device="cuda") * chan).to(BF16)


def _logits(rows, vocab, g):
    """A spread of ordinary ones and some that lead."""
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.0)
    lead = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    return x.scatter_add_(1, lead, torch.rand(rows, 24, generator=g, device="cuda") * 12.0)


def _seq_rows(case):
    """Rows of every sequence: the token in front and its drafts, ragged from the second sequence on."""
    d = case["drafts"]
    return [d + 1 if i % 5 == 0 else 1 + (d * (i * 7 + 3)) % (d + 1) for i in range(case["batch"])]


def _requests(case):
    """(tokens that stay, tokens of the next step) of every slot: where new tokens are few, most slots decode at lengths of their own and
    every sixteenth starts a prompt of up to 256; where they are many, every slot starts one behind what a shared part left."""
    kept, new = [], []
    for i in range(case["batch"]):
        f, h = (i * 0.6180339887) % 1.0, (i * 0.7548776662) % 1.0
        if case["new"] <= 8 and i % 16 != 15:
            kept.append(int(case["ctx"] * (1.0 - 0.75 * f)))
            new.append(case["new"] if i % 7 else 1 + (case["new"] - 1) // 2)
        elif case["new"] <= 8:
            kept.append(0)
            new.append(1 + int(255 * h))
        else:
            kept.append(0 if i % 3 else int(case["ctx"] * (1.0 - f)))
            new.append(max(1, int(case["new"] * (0.25 + 0.75 * h))))
    return kept, new


def prepare(case, seed):
    return {"project": _prep_project, "probs": _prep_probs, "verify": _prep_verify, "blocks": _prep_blocks}[case["op"]](case, _gen(seed))


def _prep_project(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    nb, kb = (n + 127) // 128, (k + 127) // 128
    s = {"case": case, "x": _activations(m, k, g)}
    s["w"] = torch.randn(n, k, generator=g, device="cuda", dtype=BF16).mul_(110.0).clamp_(-448, 448).to(E4M3)
    s["w_scale"] = torch.exp(0.5 * torch.randn(nb, kb, generator=g, device="cuda")) / (110.0 * math.sqrt(k))
    s["bias"] = torch.randn(n, generator=g, device="cuda").to(BF16) if case["bias"] else None
    s["q"] = torch.empty(m, k, dtype=E4M3, device="cuda")
    s["x_scale"] = torch.empty(kb, m, dtype=F32, device="cuda")
    s["out"] = torch.empty(m, n, dtype=F32 if case["f32"] else BF16, device="cuda")
    return s


def _prep_probs(case, g):
    rows, vocab = case["rows"], case["vocab"]
    s = {"case": case, "x": _logits(rows, vocab, g).to(F32 if case["f32"] else BF16)}
    s["t"] = 0.5 + torch.rand(rows, generator=g, device="cuda")
    s["t"][7::8] = 0.0
    s["p"] = torch.empty(rows, vocab, dtype=F32, device="cuda")
    return s


def _softmax_in_place(x):
    x.sub_(x.amax(1, keepdim=True)).exp_()
    return x.div_(x.sum(1, keepdim=True))


def _prep_verify(case, g):
    rows, batch, vocab = _seq_rows(case), case["batch"], case["vocab"]
    total = sum(rows)
    s = {"case": case, "total": total, "max_rows": max(rows)}
    s["cu"] = torch.tensor([0] + rows, device="cuda").cumsum(0).to(I32)
    x = _logits(total, vocab, g)
    y = (x + 0.7 * torch.randn(total, vocab, generator=g, device="cuda")) if case["q"] else x.clone()
    s["p"], q = _softmax_in_place(x), _softmax_in_place(y)
    # drafted tokens: from the draft's probabilities; row t answers with token t + 1
    drafted = torch.multinomial(q, 1, generator=g)[:, 0]
    if batch > 3:                                                       # every fourth sequence decodes at temperature zero
        seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), torch.tensor(rows, device="cuda"))
        zero = torch.nonzero(seq % 4 == 3)[:, 0]
        drafted[zero] = q[zero].argmax(1)
        for z in (s["p"], q):
            top = z[zero].argmax(1)
            z[zero] = 0.0
            z[zero, top] = 1.0
    s["q"] = q if case["q"] else None
    s["tokens"] = torch.cat([torch.randint(0, vocab, (1,), generator=g, device="cuda"), drafted[:-1]]).to(I32)
    s["lens"] = s["cu"][1:] - s["cu"][:-1] + torch.randint(0, 4096, (batch,), generator=g, device="cuda", dtype=I32)
    s["u"] = torch.rand(total, generator=g, device="cuda")
    s["v"] = torch.rand(batch, generator=g, device="cuda")
    s["out"] = torch.empty(total, dtype=I32, device="cuda")
    s["accepted"], s["kept"] = (torch.empty(batch, dtype=I32, device="cuda") for _ in range(2))
    return s


def _prep_blocks(case, g):
    """As a server has it in front of a step: the table holds the blocks of the step that ended."""
    kept, new = _requests(case)
    batch, block = case["batch"], case["block"]
    held = [(a + b + block - 1) // block for a, b in zip(kept, new)]
    used = sum(held)
    pool = used + 5 + used // 8
    order = torch.randperm(pool, generator=g, device="cuda").to(I32)
    s = {"case": case, "pool": pool, "capacity": sum(new) + 3}
    s["kept"] = torch.tensor(kept, dtype=I32, device="cuda")
    s["new"] = torch.tensor(new, dtype=I32, device="cuda")
    s["lens"] = s["kept"] + s["new"]
    stride = max(held) + 3
    s["table"] = torch.full((batch, stride), -1, dtype=I32, device="cuda")
    s["table"][torch.arange(stride, device="cuda")[None] < torch.tensor(held, device="cuda")[:, None]] = order[:used]
    s["free"] = torch.cat([order[used:], torch.full((used,), -1, dtype=I32, device="cuda")])
    s["count"] = torch.tensor([pool - used], dtype=I32, device="cuda")
    s["between"] = torch.zeros(1, dtype=I32, device="cuda")
    s["cu"] = torch.zeros(batch + 1, dtype=I32, device="cuda")
    s["pos"] = torch.zeros(s["capacity"], dtype=I32, device="cuda")
    s["slot"] = torch.zeros(s["capacity"], dtype=I64, device="cuda")
    s["refused"] = torch.zeros(1, dtype=I32, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"project": _project, "probs": _probs, "verify": _verify, "blocks": _blocks}[s["case"]["op"]](s)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _project(s):
    c = s["case"]
    m, n, k = c["m"], c["n"], c["k"]
    if own:
        from flashrt_b200 import flash_rt_kernels as fvk
        fvk.quantize_fp8_groups(s["x"].data_ptr(), s["q"].data_ptr(), s["x_scale"].data_ptr(), m, k, _stream())
        fvk.GemmRunner().fp8_block_nt(s["q"].data_ptr(), s["w"].data_ptr(), s["out"].data_ptr(), m, n, k, s["x_scale"].data_ptr(),
                                      s["w_scale"].data_ptr(), _stream(), bias=s["bias"].data_ptr() if s["bias"] is not None else 0,
                                      d_f32=c["f32"])
        return s["out"]
    nb, kb = s["w_scale"].shape
    x = torch.nn.functional.pad(s["x"].float(), (0, kb * 128 - k)).view(m, kb, 128)
    top = torch.where(x.isfinite(), x.abs(), 0.0).amax(2, keepdim=True).clamp_min(448e-12)
    q = ((x * (448.0 / 1024.0)) / (top / 1024.0)).clamp(-448, 448)      # x 448 / top, rounded once: halves between two codes stay halves
    q = q.to(E4M3).float().mul_(top / 448.0).view(m, kb * 128)[:, :k]
    w = s["w"].float()
    w *= s["w_scale"].repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    y = torch.matmul(q, w.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y if c["f32"] else y.to(BF16)


def _probs(s):
    rows, vocab = s["x"].shape
    if own:
        from flashrt_b200 import flash_rt_kernels as fvk
        fvk.softmax_rows(s["x"].data_ptr(), s["p"].data_ptr(), rows, vocab, _stream(), temperature=s["t"].data_ptr(),
                         in_f32=s["case"]["f32"])
        return s["p"]
    x, t = s["x"].float(), s["t"][:, None]
    top, at = x.max(1, keepdim=True)
    p = ((x - top) / torch.where(t > 0, t, 1.0)).exp()
    p = p / p.sum(1, keepdim=True)
    first = torch.where(x == top, torch.arange(vocab, device="cuda"), vocab).amin(1, keepdim=True)
    hot = (torch.arange(vocab, device="cuda") == first).float()
    return torch.where(t > 0, p, hot)


def _verify(s):
    c, total = s["case"], s["total"]
    batch, vocab = c["batch"], c["vocab"]
    if own:
        from flashrt_b200 import flash_rt_kernels as fvk
        fvk.verify_drafts(s["p"].data_ptr(), s["q"].data_ptr() if c["q"] else 0, s["tokens"].data_ptr(), s["cu"].data_ptr(),
                          s["lens"].data_ptr(), s["u"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), s["accepted"].data_ptr(),
                          s["kept"].data_ptr(), total, batch, vocab, _stream())
        return {"tokens": s["out"], "accepted": s["accepted"], "kept": s["kept"]}
    cu = s["cu"].long()
    n = cu[1:] - cu[:-1] - 1                                            # drafts of each sequence
    at = torch.arange(s["max_rows"], device="cuda")
    row = (cu[:-1, None] + at).clamp_max(total - 1)                     # (batch, rows)
    draft = s["tokens"].long()[(row + 1).clamp_max(total - 1)]
    pd = s["p"][row, draft].double()
    qd = s["q"][row, draft].double() if c["q"] else torch.ones_like(pd)
    stands = (at < n[:, None]) & (s["u"][row].double() * qd < pd)
    accepted = stands.long().cumprod(1).sum(1)
    last = cu[:-1] + accepted
    p = s["p"][last].double()
    rejected = (accepted < n)[:, None]
    if c["q"]:
        rest = torch.where(rejected, (p - s["q"][last].double()).clamp_min(0.0), p)
    else:
        its = s["tokens"].long()[(last + 1).clamp_max(total - 1)][:, None]
        rest = torch.where(rejected & (torch.arange(vocab, device="cuda") == its), 0.0, p)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    upto = rest.cumsum(1)
    token = (upto <= s["v"].double()[:, None] * upto[:, -1:]).sum(1)
    behind = torch.where(rest > 0, torch.arange(vocab, device="cuda"), -1).amax(1)
    token = torch.minimum(token, behind)
    out = torch.where(at < accepted[:, None], draft, torch.where(at == accepted[:, None], token[:, None], -1))
    return {"tokens": out[at <= n[:, None]].to(I32), "accepted": accepted.to(I32), "kept": (s["lens"] - n + accepted).to(I32)}


def _blocks(s):
    c, pool, capacity = s["case"], s["pool"], s["capacity"]
    batch, block, stride = c["batch"], c["block"], s["table"].shape[1]
    out = {"table": s["table"], "free": s["free"], "count": s["count"], "lens": s["lens"], "cu": s["cu"], "pos": s["pos"],
           "slot": s["slot"], "refused": s["refused"]}
    if own:
        from flashrt_b200 import flash_rt_kernels as fvk
        fvk.paged_release(s["kept"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(), stride, s["free"].data_ptr(),
                          s["count"].data_ptr(), s["between"].data_ptr(), batch, pool, block, _stream())
        fvk.paged_plan(s["kept"].data_ptr(), s["new"].data_ptr(), s["table"].data_ptr(), stride, s["free"].data_ptr(),
                       s["between"].data_ptr(), s["count"].data_ptr(), s["cu"].data_ptr(), s["lens"].data_ptr(), s["pos"].data_ptr(),
                       s["slot"].data_ptr(), s["refused"].data_ptr(), capacity, batch, pool, block, _stream())
        return out
    table, col = s["table"], torch.arange(stride, device="cuda")[None]
    # blocks behind the tokens that stay: the last one of them goes on the list first
    stay, held = ((s[name][:, None] + block - 1) // block for name in ("kept", "lens"))
    drop = (col >= stay) & (col < held) & (table >= 0) & (table < pool)
    nth = drop.view(-1).cumsum(0).view_as(drop)
    between = s["count"] + nth[-1, -1]
    room = torch.cat([s["free"], s["free"][:1]])
    room.scatter_(0, torch.where(drop, between - nth, pool).view(-1).long(), table.view(-1))
    s["free"].copy_(room[:pool])
    table.copy_(torch.where(drop, -1, table))
    # blocks of the next tokens: from the list's end, in order; from the first sequence that does not fit, none get any
    new = s["new"].long()
    last = (s["kept"] + s["new"])[:, None] + block - 1
    fits = (last // block <= stride)[:, 0]
    need = torch.where(fits, (last // block - stay)[:, 0], 0).long()
    new = torch.where(fits, new, 0)
    served = (need.cumsum(0) <= between) & (new.cumsum(0) <= capacity)
    need, new = torch.where(served, need, 0), torch.where(served, new, 0)
    first = need.cumsum(0) - need
    take = (col >= stay) & (col < stay + need[:, None])
    nth = between - 1 - (first[:, None] + col - stay)
    table.copy_(torch.where(take, s["free"][torch.where(take, nth, 0).long()], table))
    s["count"].copy_(between - need.sum())
    s["cu"][1:] = new.cumsum(0)
    s["lens"].copy_(s["kept"] + new)
    s["refused"].copy_((~(fits & served)).sum())
    t = torch.arange(capacity, device="cuda", dtype=I32)
    seq = torch.searchsorted(s["cu"], t, right=True) - 1
    there = seq < batch
    seq = seq.clamp_max(batch - 1)
    pos = s["kept"][seq] + t - s["cu"][seq]
    page = table[seq, torch.where(there, pos // block, 0).long()].long()
    s["pos"].copy_(torch.where(there, pos, -1))
    s["slot"].copy_(torch.where(there, page * block + pos % block, -1))
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "project":
        m, n, k = case["m"], case["n"], case["k"]
        nb, kb = (n + 127) // 128, (k + 127) // 128
        return {"bytes": 2 * m * k + n * k + 4 * nb * kb + (4 if case["f32"] else 2) * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "probs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (8 if case["f32"] else 6) + 4 * case["rows"], "flops": 5 * n}
    if case["op"] == "verify":
        rows, batch = sum(_seq_rows(case)), case["batch"]
        return {"bytes": batch * case["vocab"] * (8 if case["q"] else 4) + rows * 20 + batch * 20, "flops": 4 * batch * case["vocab"]}
    kept, new = _requests(case)
    block, batch = case["block"], case["batch"]
    moved = sum((a + b + block - 1) // block - (a + block - 1) // block for a, b in zip(kept, new))
    return {"bytes": moved * 16 + sum(new) * 12 + batch * 24, "flops": 2 * sum(new)}


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"project": _project64, "probs": _probs64, "verify": _verify64, "blocks": _blocks64}[case["op"]](s)


def _e4m3(x):
    """Nearest E4M3 value, ties to even: 3 bits behind the leading one, steps of 2^-9 below 2^-6, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _project64(s):
    m, k = s["x"].shape
    n = s["w"].shape[0]
    y = torch.zeros(m, n, dtype=F64, device="cuda")
    rows = torch.arange(n, device="cuda") // 128
    for j in range(0, k, 128):
        x = s["x"][:, j:j + 128].to(F64)
        top = x.abs().amax(1, keepdim=True).clamp_min(448e-12)
        y += (_e4m3(x * 448 / top) * (top / 448)) @ s["w"][:, j:j + 128].to(F64).T * s["w_scale"][rows, j // 128].to(F64)
    return y if s["bias"] is None else y + s["bias"].to(F64)


def _probs64(s):
    out = torch.zeros(s["x"].shape, dtype=F64, device="cuda")
    hot = s["t"] == 0
    cold = ~hot
    out[cold] = torch.softmax(s["x"][cold].to(F64) / s["t"][cold].to(F64)[:, None], 1)
    x = s["x"][hot].cpu().float().numpy()
    if x.size:
        out[torch.nonzero(hot)[:, 0], torch.tensor(x.argmax(1), device="cuda")] = 1.0       # numpy: the first of the largest
    return out


def _verify64(s):
    c = s["case"]
    cu, tokens, lens, u, v = (s[k].tolist() for k in ("cu", "tokens", "lens", "u", "v"))
    out, accepted, kept = [], [], []
    for b in range(c["batch"]):
        t, end, ids = cu[b], cu[b + 1] - 1, []
        while t < end:
            d = tokens[t + 1]
            if not u[t] * (float(s["q"][t, d]) if c["q"] else 1.0) < float(s["p"][t, d]):
                break
            ids.append(d)
            t += 1
        w = s["p"][t].double()
        if t < end:
            r = w.clone()
            if c["q"]:
                r = (r - s["q"][t].double()).clamp_min(0)
            else:
                r[tokens[t + 1]] = 0
            w = r if float(r.sum()) > 0 else w
        w = w.cpu().numpy()
        upto = w.cumsum()
        token = min(int(upto.searchsorted(v[b] * upto[-1], side="right")), int(w.nonzero()[0][-1]))
        accepted.append(len(ids))
        kept.append(lens[b] - (end - cu[b]) + len(ids))
        out += ids + [token] + [-1] * (end - t)
    return {"tokens": torch.tensor(out, dtype=I32, device="cuda"), "accepted": torch.tensor(accepted, dtype=I32, device="cuda"),
            "kept": torch.tensor(kept, dtype=I32, device="cuda")}


def _blocks64(s):
    block, stride = s["case"]["block"], s["table"].shape[1]
    kept, new, lens, table = (s[k].tolist() for k in ("kept", "new", "lens", "table"))
    free = s["free"].tolist()
    room, n = free[:], int(s["count"])
    gone = []
    for b, row in enumerate(table):
        for j in range(-(-kept[b] // block), -(-lens[b] // block)):
            if 0 <= row[j] < s["pool"]:
                gone.append(row[j])
                row[j] = -1
    for p in reversed(gone):
        room[n] = p
        n += 1
    cu, pos, slot, refused, full = [0], [], [], 0, False
    for b, row in enumerate(table):
        have, need = -(-kept[b] // block), -(-(kept[b] + new[b]) // block)
        full = full or need - have > n or cu[-1] + new[b] > s["capacity"]
        if full or need > stride:
            refused += 1
            lens[b] = kept[b]
            cu.append(cu[-1])
            continue
        for j in range(have, need):
            n -= 1
            row[j] = room[n]
        for p in range(kept[b], kept[b] + new[b]):
            pos.append(p)
            slot.append(row[p // block] * block + p % block)
        lens[b] = kept[b] + new[b]
        cu.append(cu[-1] + new[b])
    pad = [-1] * (s["capacity"] - len(pos))
    as_ = lambda x, t=I32: torch.tensor(x, dtype=t, device="cuda")  # noqa: E731
    return {"table": as_(table), "free": as_(room), "count": as_([n]), "lens": as_(lens), "cu": as_(cu), "pos": as_(pos + pad),
            "slot": as_(slot + pad, I64), "refused": as_([refused])}

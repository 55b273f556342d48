"""The operators of 8-bit serving as they are used: the attention block of a language model (int8 products, paged E4M3 cache), a
prompt in two chunks and then single tokens, for a batch of sequences that join one behind the other."""
import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


class Block:
    """x -> quantise -> QKV product -> append -> attention -> quantise -> output product, all through the public entry points."""

    def __init__(self, hidden, hq, hkv, d, block, num_blocks, batch, width, max_tokens, seed):
        from flashrt_b200 import flash_rt_fa2 as fa2, flash_rt_kernels as fvk
        self.fa2, self.fvk, self.gemm = fa2, fvk, fvk.GemmRunner()
        g = torch.Generator().manual_seed(seed)
        self.hidden, self.hq, self.hkv, self.d, self.block, self.num_blocks, self.batch, self.width = hidden, hq, hkv, d, block, num_blocks, batch, width
        rows = (hq + 2 * hkv) * d
        int8 = lambda n, k: torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()  # noqa: E731
        self.wqkv, self.wo = int8(rows, hidden), int8(hidden, hq * d)
        self.sqkv = ((0.5 + torch.rand(rows, generator=g)) / (73 * math.sqrt(hidden))).cuda()
        self.so = ((0.5 + torch.rand(hidden, generator=g)) / (73 * math.sqrt(hq * d))).cuda()
        self.bias = (torch.randn(rows, generator=g) * 0.1).to(BF16).cuda()
        z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
        T = max_tokens
        self.x, self.x8, self.xs = z(T, hidden), z(T, hidden, dtype=torch.int8), z(T, dtype=F32)
        self.qkv, self.q, self.o = z(T, rows), z(T, hq * d), z(T, hq * d)
        self.o8, self.os, self.y = z(T, hq * d, dtype=torch.int8), z(T, dtype=F32), z(T, hidden)
        self.k, self.v = (z(num_blocks, hkv, block, d, dtype=torch.uint8) for _ in "kv")
        self.ks, self.vs = z(num_blocks, hkv, dtype=F32), z(num_blocks, hkv, dtype=F32)
        self.rope = R.rope_table(width * block, d).cuda()
        self.table, self.cu, self.lens = torch.full((batch, width), -1, dtype=I32, device="cuda"), z(batch + 1, dtype=I32), z(batch, dtype=I32)
        self.n_work = max(fa2.paged_workspace_bytes(T, batch, n, hq, hkv, d) for n in (1, T))
        self.work = z(self.n_work, dtype=torch.uint8)

    def step(self, tokens, max_new, packed):
        fvk, st = self.fvk, torch.cuda.current_stream().cuda_stream
        hq, hkv, d, H = self.hq, self.hkv, self.d, self.hidden
        cu = self.cu.data_ptr() if packed else 0
        fvk.quantize_int8_rows(self.x.data_ptr(), self.x8.data_ptr(), self.xs.data_ptr(), tokens, H, st)
        self.gemm.int8_nt(self.x8.data_ptr(), self.wqkv.data_ptr(), self.qkv.data_ptr(), tokens, self.wqkv.shape[0], H, self.xs.data_ptr(),
                          self.sqkv.data_ptr(), st, bias=self.bias.data_ptr(), pdl=True)
        fvk.paged_kv_append_fp8(self.qkv.data_ptr(), self.rope.data_ptr(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(),
                                self.ks.data_ptr(), self.vs.data_ptr(), self.table.data_ptr(), self.width, cu, self.lens.data_ptr(), tokens,
                                self.batch, self.num_blocks, self.block, hq, hkv, d, self.rope.shape[0], st, halves=True)
        self.fa2.paged_fwd_fp8(self.q.data_ptr(), self.o.data_ptr(), 0, self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(),
                               self.vs.data_ptr(), self.table.data_ptr(), self.width, cu, self.lens.data_ptr(), tokens, self.batch, max_new,
                               self.num_blocks, self.block, hq, hkv, d, d ** -0.5, self.work.data_ptr(), self.n_work, st)
        fvk.quantize_int8_rows(self.o.data_ptr(), self.o8.data_ptr(), self.os.data_ptr(), tokens, hq * d, st)
        self.gemm.int8_nt(self.o8.data_ptr(), self.wo.data_ptr(), self.y.data_ptr(), tokens, H, hq * d, self.os.data_ptr(), self.so.data_ptr(), st,
                          pdl=True)


def quantized(x):
    """The quantiser's fp32 operations."""
    x = x.float()
    s = (x.abs().amax(1) / 127.0).clamp_min(1e-12)
    return torch.round(x * (1.0 / s)[:, None]).clamp(-127, 127).to(torch.int8), s


@pytest.mark.parametrize("hq,hkv,d,block", [(8, 2, 128, 32), (8, 1, 256, 16), (6, 2, 64, 64)])
def test_block_from_prompt_to_tokens(hq, hkv, d, block):
    """Each stage against its formula on what the stage in front left, so that nothing is compared through a quantiser's step: the products'
    integers exactly, the cache within half a code of the appended values, attention over the cache as it stands."""
    hidden, batch, width = 512, 3, 256 // block
    b = Block(hidden, hq, hkv, d, block, 3 * width, batch, width, 128, seed=d)
    b.table.copy_(torch.randperm(3 * width, generator=torch.Generator().manual_seed(1))[:batch * width].view(batch, width))
    g = torch.Generator().manual_seed(2)
    lens = [0] * batch
    plan = [[60, 1, 0], [25, 50, 30], [1, 1, 1], [1, 1, 1], [3, 1, 40], [1, 1, 1]]
    history = [[] for _ in range(batch)]                   # rotated keys and values that were appended, in 64 bits
    for new in plan:
        lens = [a + n for a, n in zip(lens, new)]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        T = cu[-1]
        b.x[:T] = torch.randn(T, hidden, generator=g).to(BF16)
        b.cu.copy_(torch.tensor(cu, dtype=I32))
        b.lens.copy_(torch.tensor(lens, dtype=I32))
        b.step(T, max(new), new != [1] * batch)
        torch.cuda.synchronize()
        assert b.fvk.tensor_core_status() == 0
        xq, xs = quantized(b.x[:T].cpu())
        assert torch.equal(b.x8[:T].cpu(), xq) and torch.equal(b.xs[:T].cpu(), xs)
        acc = xq.to(F64) @ b.wqkv.cpu().to(F64).T
        want = acc * xs.to(F64)[:, None] * b.sqkv.cpu().to(F64) + b.bias.cpu().to(F64)
        qkv = b.qkv[:T].cpu()
        # half a bf16 step of the value, three fp32 roundings of the product in front of the bias
        assert ((qkv.to(F64) - want).abs() <= want.abs() * 2.0 ** -8 + (want - b.bias.cpu().to(F64)).abs() * 3 * 2.0 ** -24).all()
        rope = b.rope.cpu()
        for s in range(batch):
            if not new[s]:
                continue
            rows = qkv[cu[s]:cu[s + 1]].to(F64).view(-1, hq + 2 * hkv, d)
            at = rope[lens[s] - new[s]:lens[s]]
            q = R.rotate(rows[:, :hq], at, True)
            pair = q.abs() + rows[:, :hq].abs() + torch.roll(rows[:, :hq].abs(), d // 2, -1)
            assert ((b.q[cu[s]:cu[s + 1]].cpu().to(F64).view(-1, hq, d) - q).abs() <= q.abs() * 2.0 ** -8 + pair * 2.0 ** -21).all()
            k, v = R.rotate(rows[:, hq:hq + hkv], at, True), rows[:, hq + hkv:]
            history[s] += [(k[i], v[i]) for i in range(new[s])]
        table, kc, vc, ks, vs = b.table.cpu(), b.k.cpu(), b.v.cpu(), b.ks.cpu(), b.vs.cpu()
        for s in range(batch):
            for j, (k, v) in enumerate(history[s]):
                page = int(table[s, j // block])
                for y, c, sc in ((k, kc, ks), (v, vc, vs)):
                    got = R.codes(c[page, :, j % block]) * sc[page].to(F64)[:, None]
                    # half a code's step at the scale of now, and one more for each time the block's scale may have grown since
                    bar = y.abs() * 2.0 ** -4 + sc[page].to(F64)[:, None] * 2.0 ** -10
                    assert ((got - y).abs() <= bar * (1 + 1.1 * len(plan))).all()
        o = b.o[:T].cpu()
        wo, _, size, _ = R.attention(b.q[:T].cpu().view(-1, hq, d), kc, vc, ks, vs, table, cu, lens, d ** -0.5)
        assert ((o.to(F64).view(wo.shape) - wo).abs() <= wo.abs() * 2.0 ** -8 + size * 2.0 ** -10).all()
        oq, osc = quantized(o)
        assert torch.equal(b.o8[:T].cpu(), oq) and torch.equal(b.os[:T].cpu(), osc)
        y = ((oq.to(F64) @ b.wo.cpu().to(F64).T).to(F32) * osc[:, None] * b.so.cpu()).to(BF16)
        assert torch.equal(b.y[:T].cpu(), y)


def test_captured_decode_step_serves_other_lengths():
    """One graph of the six launches, replayed while sequences grow, one slot idle: the bits of eager calls on a copy of the state."""
    mk = lambda: Block(512, 8, 2, 128, 16, 64, 4, 16, 64, seed=3)  # noqa: E731
    a, e = mk(), mk()
    for b in (a, e):
        b.table.copy_(torch.randperm(64, generator=torch.Generator().manual_seed(1))[:64].view(4, 16))
    a.lens.fill_(0)
    a.step(4, 1, False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(4, 1, False)
    for t in (a.k, a.v, a.ks, a.vs, a.q, a.o, e.q, e.o):
        t.zero_()
    g = torch.Generator().manual_seed(5)
    for i in range(20):
        x = torch.randn(4, 512, generator=g).to(BF16)
        lens = torch.tensor([i + 1, 2 * i + 1, 0 if i % 3 else i + 1, i + 100 if i > 0 else 1], dtype=I32)
        for b in (a, e):
            b.x[:4] = x.cuda()
            b.lens.copy_(lens)
        graph.replay()
        e.step(4, 1, False)
        torch.cuda.synchronize()
        assert torch.equal(a.y[:4], e.y[:4]) and torch.equal(a.k, e.k) and torch.equal(a.v, e.v) and torch.equal(a.ks, e.ks)

"""A decode step with drafted tokens, all of it on the device in one graph: blocks released and planned, block-scaled projections, the paged
cache's append and attention, logits, probabilities, verification.  Replayed over steps whose lengths only the device knows."""
import numpy as np
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
BF16, E4M3, F32, F64, I32, I64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64, torch.int32, torch.int64
HQ, HKV, D, DIM, VOCAB, BS = 8, 2, 64, 512, 1003, 16


def _stream():
    return torch.cuda.current_stream().cuda_stream


class Step:
    """One attention block and an output projection over `batch` slots of at most `drafts` + 1 tokens."""

    def __init__(self, batch, drafts, pool, stride, seed):
        from flashrt_b200 import flash_rt_fa2 as fa2
        from flashrt_b200 import flash_rt_kernels as fvk
        self.fvk, self.fa2, self.batch, self.pool, self.stride = fvk, fa2, batch, pool, stride
        self.rows = batch * (drafts + 1)
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.embed = rnd(VOCAB, DIM).to(BF16)
        self.w = {}
        for name, n, k in (("qkv", (HQ + 2 * HKV) * D, DIM), ("out", VOCAB, HQ * D)):
            self.w[name] = ((rnd(n, k) * 80).clamp(-448, 448).to(E4M3), torch.rand((n + 127) // 128, k // 128, generator=g, device="cuda") * 0.02 / k ** 0.5 * 8)
        angle = torch.arange(stride * BS, dtype=F64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, D, 2, dtype=F64, device="cuda") / D)
        self.rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(-1, D).to(F32).contiguous()
        z = lambda *s, t=I32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        self.kept, self.new, self.lens, self.cu, self.refused = z(batch), z(batch), z(batch), z(batch + 1), z(1)
        self.table = torch.full((batch, stride), -1, dtype=I32, device="cuda")
        self.free = torch.randperm(pool, generator=g, device="cuda").to(I32)
        self.count, self.between = torch.tensor([pool], dtype=I32, device="cuda"), z(1)
        self.pos, self.slot = z(self.rows), z(self.rows, t=I64)
        self.tokens, self.out, self.accepted = z(self.rows), z(self.rows), z(batch)
        self.x, self.qkv = z(self.rows, DIM, t=BF16), z(self.rows, (HQ + 2 * HKV) * D, t=BF16)
        self.x8, self.xs = z(self.rows, DIM, t=E4M3), z(DIM // 128, self.rows, t=F32)
        self.q, self.o = z(self.rows, HQ * D, t=BF16), z(self.rows, HQ * D, t=BF16)
        self.o8, self.os = z(self.rows, HQ * D, t=E4M3), z(HQ * D // 128, self.rows, t=F32)
        self.k, self.v = (z(pool, HKV, BS, D, t=torch.uint8) for _ in range(2))
        self.ks, self.vs = (z(pool, HKV, t=F32) for _ in range(2))
        self.logits, self.p = z(self.rows, VOCAB, t=F32), z(self.rows, VOCAB, t=F32)
        self.temp, self.u, self.uv = z(self.rows, t=F32), z(self.rows, t=F32), z(batch, t=F32)
        self.bytes = fa2.paged_workspace_bytes(self.rows, batch, drafts + 1, HQ, HKV, D)
        self.work = z(self.bytes, t=torch.uint8)
        self.max_new = drafts + 1

    def blocks(self):
        f = self.fvk
        f.paged_release(self.kept.data_ptr(), self.lens.data_ptr(), self.table.data_ptr(), self.stride, self.free.data_ptr(), self.count.data_ptr(),
                        self.between.data_ptr(), self.batch, self.pool, BS, _stream())
        f.paged_plan(self.kept.data_ptr(), self.new.data_ptr(), self.table.data_ptr(), self.stride, self.free.data_ptr(), self.between.data_ptr(),
                     self.count.data_ptr(), self.cu.data_ptr(), self.lens.data_ptr(), self.pos.data_ptr(), self.slot.data_ptr(),
                     self.refused.data_ptr(), self.rows, self.batch, self.pool, BS, _stream())

    def layer(self):
        f, n = self.fvk, self.rows
        self.x.copy_(self.embed[self.tokens.long().clamp(0, VOCAB - 1)])
        gemm = f.GemmRunner()
        f.quantize_fp8_groups(self.x.data_ptr(), self.x8.data_ptr(), self.xs.data_ptr(), n, DIM, _stream())
        gemm.fp8_block_nt(self.x8.data_ptr(), self.w["qkv"][0].data_ptr(), self.qkv.data_ptr(), n, (HQ + 2 * HKV) * D, DIM, self.xs.data_ptr(),
                          self.w["qkv"][1].data_ptr(), _stream(), pdl=True)
        f.paged_kv_append_fp8(self.qkv.data_ptr(), self.rope.data_ptr(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(),
                              self.vs.data_ptr(), self.table.data_ptr(), self.stride, self.cu.data_ptr(), self.lens.data_ptr(), n, self.batch, self.pool,
                              BS, HQ, HKV, D, self.rope.shape[0], _stream())
        self.fa2.paged_fwd_fp8(self.q.data_ptr(), self.o.data_ptr(), 0, self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(),
                               self.table.data_ptr(), self.stride, self.cu.data_ptr(), self.lens.data_ptr(), n, self.batch, self.max_new, self.pool, BS,
                               HQ, HKV, D, D ** -0.5, self.work.data_ptr(), self.bytes, _stream())
        f.quantize_fp8_groups(self.o.data_ptr(), self.o8.data_ptr(), self.os.data_ptr(), n, HQ * D, _stream())
        gemm.fp8_block_nt(self.o8.data_ptr(), self.w["out"][0].data_ptr(), self.logits.data_ptr(), n, VOCAB, HQ * D, self.os.data_ptr(),
                          self.w["out"][1].data_ptr(), _stream(), d_f32=True, pdl=True)

    def verify(self):
        f = self.fvk
        f.softmax_rows(self.logits.data_ptr(), self.p.data_ptr(), self.rows, VOCAB, _stream(), temperature=self.temp.data_ptr(), in_f32=True)
        f.verify_drafts(self.p.data_ptr(), 0, self.tokens.data_ptr(), self.cu.data_ptr(), self.lens.data_ptr(), self.u.data_ptr(), self.uv.data_ptr(),
                        self.out.data_ptr(), self.accepted.data_ptr(), self.kept.data_ptr(), self.rows, self.batch, VOCAB, _stream())

    def step(self):
        self.blocks()
        self.layer()
        self.verify()


def test_steps_in_one_graph():
    batch, drafts, stride = 7, 3, 12
    pool = batch * stride // 2
    a, b = Step(batch, drafts, pool, stride, 1), Step(batch, drafts, pool, stride, 1)      # b: eager, blocks in another order
    b.free.copy_(torch.arange(pool - 1, -1, -1, dtype=I32, device="cuda"))
    rng = np.random.default_rng(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()                                                     # lengths of zero: an empty step
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a.step()
    torch.cuda.synchronize()
    assert a.cu.tolist() == [0] * (batch + 1) and a.accepted.tolist() == [0] * batch

    table, free, count, lens = a.table.tolist(), a.free.tolist(), pool, [0] * batch
    kept = [0] * batch
    text = [[int(rng.integers(VOCAB))] for _ in range(batch)]       # tokens whose keys are not cached yet: the last of each sequence
    for i in range(14):
        for s in range(batch):                                       # now and then a sequence ends and another starts; slots idle
            if rng.random() < 0.08:
                kept[s], text[s] = 0, [int(rng.integers(VOCAB))]
        new = [0 if (i + s) % 9 == 8 else int(rng.integers(1, drafts + 2)) for s in range(batch)]
        packed = []
        for s in range(batch):
            packed += text[s][-1:] + [int(t) for t in rng.integers(0, VOCAB, max(0, new[s] - 1))] if new[s] else []
        temp = np.zeros(a.rows, np.float32) if i % 2 else (0.2 + rng.random(a.rows)).astype(np.float32)
        u, uv = rng.random(a.rows, dtype=np.float32), rng.random(batch, dtype=np.float32)

        def put(m):
            m.kept.copy_(torch.tensor(kept, dtype=I32))
            m.new.copy_(torch.tensor(new, dtype=I32))
            m.tokens.copy_(torch.tensor(packed + [0] * (m.rows - len(packed)), dtype=I32))
            m.temp.copy_(torch.tensor(temp))
            m.u.copy_(torch.tensor(u))
            m.uv.copy_(torch.tensor(uv))

        put(a)
        put(b)
        torch.cuda.synchronize()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        # blocks: plain lists
        mid = R.release(kept, lens, table, free, count, pool, BS)
        count, cu, lens, pos, slot, refused = R.plan(kept, new, table, free, mid, pool, BS, a.rows)
        assert refused == 0 and int(a.refused) == 0
        assert (a.table.tolist(), a.free.tolist(), int(a.count)) == (table, free, count)
        assert (a.cu.tolist(), a.lens.tolist(), a.pos.tolist(), a.slot.tolist()) == (cu, lens, pos, slot)
        # what the step computes does not depend on which blocks hold the keys, nor on the graph
        n = cu[-1]
        assert torch.equal(a.logits[:n], b.logits[:n]) and torch.equal(a.out[:n], b.out[:n])
        # the projections' and the probabilities' own statements
        codes, scales = R.fp8_groups(a.x[:n].cpu())
        assert torch.equal(a.x8[:n].cpu().to(F64), codes) and torch.equal(a.xs[:, :n].cpu(), scales)
        want, size = R.block_product(a.o8[:n].to(F64).cpu(), a.w["out"][0].to(F64).cpu(), a.os[:, :n].cpu(), a.w["out"][1].cpu())
        assert ((a.logits[:n].cpu().to(F64) - want).abs() <= size * (128 * 2.0 ** -23 + 15 * 2.0 ** -24)).all()
        probs = R.softmax_rows(a.logits[:n].cpu(), temp[:n])
        # arguments of up to 2^7 with three roundings, the exponential, factor and sum: as in the softmax's own test
        assert ((a.p[:n].cpu().to(F64) - probs).abs() <= probs * (2.0 ** -24 * 4 * 128 + 4 * 2.0 ** -22 + 2.0 ** -18) + 2.0 ** -120).all()
        out, accepted, stay = R.verify(a.p.cpu().numpy(), None, a.tokens.tolist(), cu, lens, u, uv)
        assert a.accepted.tolist() == accepted and a.kept.tolist() == stay and a.out[:n].tolist() == out[:n]
        for s in range(batch):
            if new[s]:
                text[s] = [t for t in out[cu[s]:cu[s + 1]] if t >= 0]
        kept = stay
    from flashrt_b200 import flash_rt_kernels as fvk
    assert fvk.tensor_core_status() == 0


def test_drafts_that_the_model_itself_would_answer_stand():
    """The step's own answers, given back as drafts until they no longer change: then every draft stands, at temperature zero and with
    random numbers that accept only what is certain."""
    batch = 3
    m = Step(batch, 4, batch * 8, 8, 5)
    tokens = torch.tensor([[11, 0, 0, 0, 0], [700, 0, 0, 0, 0], [1002, 0, 0, 0, 0]], dtype=I32)
    m.u.fill_(0.999)
    for i in range(20):
        m.kept.zero_()
        m.new.fill_(5)
        m.tokens.copy_(tokens.view(-1))
        m.step()
        torch.cuda.synchronize()
        best = m.logits.argmax(1).view(batch, 5).cpu().to(I32)
        stood = [int((best[s, :4] == tokens[s, 1:]).int().cumprod(0).sum()) for s in range(batch)]
        assert m.accepted.tolist() == stood
        out = m.out.view(batch, 5)
        for s in range(batch):
            assert out[s, :stood[s] + 1].tolist() == best[s, :stood[s] + 1].tolist() and (out[s, stood[s] + 1:] == -1).all()
        if stood == [4] * batch:
            break
        tokens[:, 1:] = best[:, :4]
    assert stood == [4] * batch and m.kept.tolist() == [5] * batch

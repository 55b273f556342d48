"""E4M3 products with a scale for each block of 128, and their quantiser, against 64 bits."""
import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
BF16, E4M3, F32, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64


def _stream():
    return torch.cuda.current_stream().cuda_stream


def quantize(x, stride=0, rows=None, dim=None, scale_stride=0):
    from flashrt_b200 import flash_rt_kernels as fvk
    rows, dim = rows or x.shape[0], dim or x.shape[1]
    g = (dim + 127) // 128
    q = torch.full((rows + 1, dim), 0x5a, dtype=torch.uint8, device="cuda")
    s = torch.full((g * (scale_stride or rows) + 3,), -1.0, device="cuda")
    fvk.quantize_fp8_groups(x.data_ptr(), q.data_ptr(), s.data_ptr(), rows, dim, _stream(), in_stride=stride, scale_stride=scale_stride)
    torch.cuda.synchronize()
    assert (q[rows] == 0x5a).all() and (s[-3:] == -1).all()         # nothing behind the last row
    s = s[:-3].view(g, -1)
    assert (s[:, rows:] == -1).all()
    return q[:rows].view(E4M3), s[:, :rows].contiguous()


def check_codes(x, q, s):
    """The 64-bit definition code for code: a quotient of two 8-bit significands times 7 that is not a middle of two codes is at least
    2^-17 away from it (relative), and the kernel's is off by 2^-24.  Scales: one correctly rounded division."""
    codes, scales = R.fp8_groups(x)
    assert torch.equal(s.cpu(), scales)
    assert torch.equal(q.cpu().to(F64), codes)


@pytest.mark.parametrize("rows,dim", [(1, 16), (1, 2048), (3, 48), (7, 1024), (5, 1040), (130, 2064), (9, 4096), (4, 16384), (2, 40000),
                                      (2000, 128), (1300, 4112), (700, 112), (3000, 1024)])
def test_quantize_groups(rows, dim):
    g = torch.Generator().manual_seed(rows + dim)
    x = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(rows, 1, generator=g) * 3)).to(BF16)
    x[rows // 2] = 0
    check_codes(x, *quantize(x.cuda()))


@pytest.mark.parametrize("rows,dim", [(31, 4112), (32, 4112), (33, 160), (63, 80000), (64, 80000), (9001, 528)])
def test_quantize_blocks_of_rows(rows, dim):
    """Rows on both sides of a block of 32, an odd number of groups, more rows than whole blocks have."""
    test_quantize_groups(rows, dim)


def test_quantize_every_significand():
    """Every pair of bf16 significands (value, largest) at four exponents: all quotients that the definition can meet."""
    sig = (1.0 + torch.arange(128) / 128).to(F64)
    for e in (-60, -1, 0, 40):
        x = torch.zeros(128 * 3, 128, dtype=F64)
        x[:, :127] = torch.cat([sig[None, :127] * 2.0 ** (e + k) for k in (0, -3, -7)])[:, None].expand(3, 128, 127).reshape(384, 127)
        top = sig.repeat(3) * 2.0 ** (e + 1)
        x[:, 127] = top
        x = x.to(BF16)
        check_codes(x, *quantize(x.cuda()))


def test_quantize_strided_and_special_values():
    x = torch.randn(6, 512, generator=torch.Generator().manual_seed(0)).to(BF16)
    x[0, 3], x[1, 4], x[1, 5], x[2, 6] = float("inf"), -float("inf"), 1e30, float("nan")
    x[3] = float("nan")
    x[4] = 1e-30
    x[5, :128], x[5, 130] = float("inf"), 3.3895e38
    q, s = quantize(x.cuda(), stride=512, rows=6, dim=272)
    check_codes(x[:, :272], q, s)
    v = q.cpu().float()
    assert v[0, 3] == 448 and v[1, 4] == -448 and v[2, 6] == -448 and (v[3] == -448).all() and (v[5, :128] == 448).all() and v[5, 130] == 448
    wide = torch.randn(9, 328, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    check_codes(wide[:, :320].cpu(), *quantize(wide, stride=328, rows=9, dim=320, scale_stride=13))


def operands(m, n, k, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(m, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    w = (torch.randn(n, k, generator=g) * 100).clamp(-448, 448).to(E4M3)
    kb, nb = (k + 127) // 128, (n + 127) // 128
    sa = torch.exp(spread * torch.randn(kb, m, generator=g)) * 0.01
    sw = torch.exp(spread * torch.randn(nb, kb, generator=g)) * 0.01 / k ** 0.5
    return a, w, sa, sw, torch.randn(n, generator=g).to(BF16)


def product(a, w, sa, sw, bias=None, f32=False, pdl=False, stride=0):
    from flashrt_b200 import flash_rt_kernels as fvk
    m, k = a.shape
    n = w.shape[0]
    out = torch.full((m * n + 64,), -7.0, dtype=F32 if f32 else BF16, device="cuda")
    fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, sa.data_ptr(), sw.data_ptr(), _stream(),
                                  bias=bias.data_ptr() if bias is not None else 0, a_scale_stride=stride, d_f32=f32, pdl=pdl)
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    assert (out[m * n:] == -7.0).all()
    return out[:m * n].view(m, n)


def close(got, want, size, kb, bias, f32):
    """Sums of a block: 128 products in the tensor core, each addition off by at most a last place (2^-23) of the block's magnitudes; then
    two roundings of the scale, one of each block's fma, eight of parts of K, one of the bias (2^-24 each); the store in bf16: half a step."""
    bound = size * (128 * 2.0 ** -23 + (kb + 11) * 2.0 ** -24)
    if bias is not None:
        want, bound = want + bias.to(F64), bound + bias.to(F64).abs() * 2.0 ** -23
    if not f32:
        bound = bound * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    off = (got.to(F64) - want).abs()
    assert (off <= bound).all(), (off / bound).max()


def check(m, n, k, bias=True, f32=False, pdl=False):
    a, w, sa, sw, b = operands(m, n, k, m + n + k)
    b = b if bias else None
    got = product(a.cuda(), w.cuda(), sa.cuda(), sw.cuda(), b.cuda() if bias else None, f32, pdl)
    want, size = R.block_product(a.to(F64).cuda(), w.to(F64).cuda(), sa.cuda(), sw.cuda())
    close(got.cpu(), want.cpu(), size.cpu(), sa.shape[0], b, f32)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 300, 511, 600])
def test_rows(m):
    check(m, 640, 1024)
    check(m, 1000, 528, bias=False, f32=True)


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (3, 7, 16), (70, 5, 48), (130, 1, 128), (5, 127, 144), (129, 129, 112), (1, 2560, 2048),
                                   (96, 4096, 2048), (16, 33000, 256), (64, 40000, 272), (70, 40000, 272), (817, 2048, 1040), (1024, 1024, 4096),
                                   (300, 256, 16384), (8, 256, 16384), (40, 130, 16400), (100, 200, 8208), (4096, 1001, 512), (2500, 2050, 640)])
def test_shapes(m, n, k):
    check(m, n, k)
    check(m, n, k, bias=False, f32=True, pdl=True)


@pytest.mark.parametrize("m,n,k", [(65, 2048, 2048), (96, 130, 7168), (97, 4096, 2064), (128, 1000, 4096), (129, 2048, 2048), (192, 500, 8192),
                                   (193, 1030, 4112), (300, 512, 7168), (257, 1000, 4100 // 16 * 16), (385, 7, 4096), (512, 130, 2048)])
def test_tiles_of_tokens_that_share_k(m, n, k):
    """Few tiles and a long K: four or eight CTAs share it, the last tile of tokens may have one row."""
    check(m, n, k)
    check(m, n, k, bias=False, f32=True, pdl=True)


def test_scales_far_apart():
    """Blocks whose scales lie ten orders of magnitude apart, and scales of zero."""
    for m in (9, 90, 300):
        a, w, sa, sw, _ = operands(m, 384, 1024, m, spread=6.0)
        sa[3], sw[1, 2] = 0.0, 0.0
        got = product(a.cuda(), w.cuda(), sa.cuda(), sw.cuda(), f32=True).cpu()
        want, size = R.block_product(a.to(F64), w.to(F64), sa, sw)
        close(got, want, size, 8, None, True)


def test_exact_products_and_the_same_bits_again():
    """Small whole codes and scales that are powers of two: every sum is exact in fp32, so every form of the kernel gives the same bits; any
    call gives the same bits twice."""
    g = torch.Generator().manual_seed(3)
    for m, n, k in ((4, 500, 2048), (50, 500, 2048), (100, 500, 2048), (400, 500, 2048), (400, 500, 8192)):
        a, w = (torch.randint(-4, 5, (r, k), generator=g).float().to(E4M3) for r in (m, n))
        sa = 2.0 ** torch.randint(-2, 3, (k // 128, m), generator=g)
        sw = 2.0 ** torch.randint(-2, 3, ((n + 127) // 128, k // 128), generator=g)
        want, _ = R.block_product(a.to(F64), w.to(F64), sa, sw)
        got = product(a.cuda(), w.cuda(), sa.cuda(), sw.cuda(), f32=True)
        assert torch.equal(got.cpu().to(F64), want)
    a, w, sa, sw, b = (t.cuda() for t in operands(300, 1000, 4096, 1))
    first = product(a, w, sa, sw, b)
    for _ in range(5):
        assert torch.equal(first, product(a, w, sa, sw, b))


def test_rows_do_not_depend_on_their_neighbours():
    """NaN codes, infinite scales: they stay in their own row or column.  Strided scales."""
    for m in (20, 100, 300):
        a, w, sa, sw, _ = operands(m, 700, 512, m)
        clean = product(a.cuda(), w.cuda(), sa.cuda(), sw.cuda(), f32=True)
        a8, w8 = a.view(torch.uint8).clone(), w.view(torch.uint8).clone()
        a8[3, 7], w8[500, 100] = 0x7f, 0xff
        wide = torch.full((4, m + 5), float("nan"))
        wide[:, :m] = sa
        wide[2, 5] = float("inf")
        got = product(a8.view(E4M3).cuda(), w8.view(E4M3).cuda(), wide.cuda(), sw.cuda(), f32=True, stride=m + 5)
        assert got[3].isnan().all() and got[:, 500].isnan().all() and not got[5].isfinite().any()
        rows = [i for i in range(m) if i not in (3, 5)]
        cols = [i for i in range(700) if i != 500]
        assert torch.equal(got[rows][:, cols], clean[rows][:, cols])


def test_bias_and_output_at_odd_places():
    """A bias that starts two bytes behind a boundary, an output 16 bytes behind one of 32."""
    from flashrt_b200 import flash_rt_kernels as fvk
    for m, n, k in ((5, 640, 512), (70, 640, 512), (300, 640, 512), (128, 1024, 4096)):
        a, w, sa, sw, _ = (t.cuda() for t in operands(m, n, k, m + 1))
        wide = torch.randn(n + 1, device="cuda").to(BF16)
        for f32 in (False, True):
            out = torch.full((m * n + 64,), -7.0, dtype=F32 if f32 else BF16, device="cuda")
            at = 4 if f32 else 8
            fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), out.data_ptr() + 16, m, n, k, sa.data_ptr(), sw.data_ptr(), _stream(),
                                          bias=wide.data_ptr() + 2, d_f32=f32)
            torch.cuda.synchronize()
            assert (out[:at] == -7).all() and (out[at + m * n:] == -7).all()
            want, size = R.block_product(a.to(F64), w.to(F64), sa, sw)
            close(out[at:at + m * n].view(m, n).cpu(), want.cpu(), size.cpu(), k // 128, wide[1:].cpu(), f32)


def test_two_calls_at_once():
    """Products, large and small, on two streams at the same time: nothing is shared."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    jobs = [operands(m, n, k, m) for m, n, k in ((3000, 1024, 2048), (40, 8192, 1024), (100, 4096, 4096), (1, 2560, 2048))]
    jobs = [tuple(t.cuda() for t in j) for j in jobs]
    want = [product(*j[:4], j[4]) for j in jobs]
    from flashrt_b200 import flash_rt_kernels as fvk
    outs = [[torch.zeros_like(w) for w in want] for _ in sides]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, mine in zip(sides, outs):
            with torch.cuda.stream(s):
                for (a, w, sa, sw, b), o in zip(jobs, mine):
                    fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), o.data_ptr(), *o.shape, a.shape[1], sa.data_ptr(), sw.data_ptr(),
                                                  _stream(), bias=b.data_ptr())
    torch.cuda.synchronize()
    for mine in outs:
        for o, w in zip(mine, want):
            assert torch.equal(o, w)
    assert fvk.tensor_core_status() == 0


def test_streams_and_graph():
    from flashrt_b200 import flash_rt_kernels as fvk
    m, n, k = 70, 1500, 2048
    x = torch.randn(m, k, device="cuda").to(BF16)
    _, w, _, sw, _ = (t.cuda() for t in operands(2, n, k, 5))
    q, s, out = torch.empty(m, k, dtype=E4M3, device="cuda"), torch.empty(k // 128, m, device="cuda"), torch.empty(m, n, device="cuda")

    def step():
        fvk.quantize_fp8_groups(x.data_ptr(), q.data_ptr(), s.data_ptr(), m, k, _stream())
        fvk.GemmRunner().fp8_block_nt(q.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, s.data_ptr(), sw.data_ptr(), _stream(), d_f32=True, pdl=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for seed in (1, 2):
        x.copy_(torch.randn(m, k, generator=torch.Generator().manual_seed(seed)).to(BF16))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and got.abs().max() > 0
    assert fvk.tensor_core_status() == 0


@pytest.mark.parametrize("m,n,k", [(5, 700, 4096), (48, 1001, 1024), (96, 4096, 512), (130, 4096, 4096), (817, 2048, 4096), (2100, 1800, 640)])
def test_settled_weights_behind_the_quantiser(m, n, k):
    """Weights read early, activations not: quantiser and product in turn over one pair of buffers give the bits of products that wait for all."""
    from flashrt_b200 import flash_rt_kernels as fvk
    _, w, _, sw, _ = (t.cuda() for t in operands(2, n, k, m))
    xs = [torch.randn(m, k, generator=torch.Generator().manual_seed(i)).to(BF16).cuda() for i in range(8)]
    q, s = torch.empty(m, k, dtype=E4M3, device="cuda"), torch.empty((k + 127) // 128, m, device="cuda")
    outs = {pdl: [torch.zeros(m, n, dtype=BF16, device="cuda") for _ in xs] for pdl in (False, True)}

    def chain(pdl):
        for x, out in zip(xs, outs[pdl]):
            fvk.quantize_fp8_groups(x.data_ptr(), q.data_ptr(), s.data_ptr(), m, k, _stream())
            fvk.GemmRunner().fp8_block_nt(q.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, s.data_ptr(), sw.data_ptr(), _stream(), pdl=pdl)
    chain(False)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        chain(True)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for plain, early in zip(outs[False], outs[True]):
        assert torch.equal(plain, early) and plain.abs().max() > 0
    assert fvk.tensor_core_status() == 0

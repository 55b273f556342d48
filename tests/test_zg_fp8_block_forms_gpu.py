"""Every form of the block-scaled product against 64 bits, the form read from the launch: whole and part tiles, outputs by TMA (N % 8 == 0), in
vectors and value by value, K that ends inside a block, more tiles than places."""
import ctypes
import re

import pytest
import torch

import decode_ref as R

pytestmark = pytest.mark.gpu
BF16, E4M3, F32, F64 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.float64

FORMS = [
    # pairs of 256 columns, K not shared: more tiles than pairs, by TMA; a part tile; odd rows
    ("tile_kernel<2, 256, 1>", [(3000, 2048, 1040), (2100, 1800, 640), (8191, 4096, 512), (2500, 2050, 640)]),
    ("tile_kernel<1, 256, 1>", [(570, 6528, 128), (1627, 2752, 1344), (2599, 1603, 1440)]),
    ("tile_kernel<2, 128, 1>", [(817, 2048, 4096), (811, 2300, 2192), (251, 5248, 3104), (251, 5247, 3104)]),
    ("tile_kernel<1, 128, 1>", [(1000, 1024, 640), (600, 1000, 528), (2264, 7, 1568)]),
    # K shared by two or four
    ("tile_kernel<1, 128, 2>", [(988, 800, 2016), (68, 4736, 2000), (68, 4735, 2000)]),
    ("tile_kernel<2, 128, 2>", [(130, 2560, 8192), (132, 2368, 7312), (132, 2366, 7312), (300, 1601, 8736)]),
    ("tile_kernel<1, 256, 2>", [(817, 2048, 16384), (270, 5888, 7200), (270, 5887, 7200)]),
    ("tile_kernel<1, 256, 4>", [(65, 6144, 14336), (65, 6146, 14336), (65, 6143, 14336)]),
    # weights on the lanes
    ("lane_kernel<16>", [(5, 640, 528), (5, 40000, 272), (16, 4608, 3584), (16, 2561, 8192)]),
    ("lane_kernel<32>", [(17, 640, 4096), (30, 9000, 4096), (31, 40001, 272)]),
    ("lane_kernel<64>", [(40, 640, 1024), (64, 40000, 272), (60, 9001, 4096)]),
    ("lane_kernel<96>", [(96, 640, 2048), (70, 300, 8192), (129, 501, 8208)]),
    ("lane_kernel<128>", [(97, 512, 4096), (128, 2048, 8192), (97, 511, 4112)]),
]


def operands(m, n, k, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    a, w = ((torch.randn(r, k, generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3) for r in (m, n))
    kb, nb = (k + 127) // 128, (n + 127) // 128
    sa = torch.exp(torch.randn(kb, m, generator=g, device="cuda")) * 0.01
    sw = torch.exp(torch.randn(nb, kb, generator=g, device="cuda")) * 0.01 / k ** 0.5
    return a, w, sa, sw, torch.randn(n, generator=g, device="cuda").to(BF16)


def product(a, w, sa, sw, bias, f32, pdl):
    from flashrt_b200 import flash_rt_kernels as fvk
    m, n, k = a.shape[0], w.shape[0], a.shape[1]
    out = torch.full((m * n + 64,), -7.0, dtype=F32 if f32 else BF16, device="cuda")
    fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, sa.data_ptr(), sw.data_ptr(),
                                  torch.cuda.current_stream().cuda_stream, bias=bias.data_ptr() if bias is not None else 0, d_f32=f32, pdl=pdl)
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    assert (out[m * n:] == -7.0).all()
    return out[:m * n].view(m, n)


class KernelNode(ctypes.Structure):
    """CUDA_KERNEL_NODE_PARAMS_v2 of the driver's interface."""
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3), ("shared", ctypes.c_uint),
                ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p), ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


def form_of(a, w, sa, sw):
    """The kernel of a product's launch, read from a graph that holds nothing else."""
    from flashrt_b200 import flash_rt_kernels as fvk
    m, n, k = a.shape[0], w.shape[0], a.shape[1]
    out = torch.empty(m, n, device="cuda")
    graph, side = torch.cuda.CUDAGraph(keep_graph=True), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), out.data_ptr(), m, n, k, sa.data_ptr(), sw.data_ptr(), side.cuda_stream, d_f32=True)
    cuda = ctypes.CDLL("libcuda.so.1")
    handle, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert cuda.cuGraphGetNodes(handle, None, ctypes.byref(count)) == 0 and count.value == 1
    nodes, node, name = (ctypes.c_void_p * 1)(), KernelNode(), ctypes.c_char_p()
    assert cuda.cuGraphGetNodes(handle, nodes, ctypes.byref(count)) == 0
    assert cuda.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(nodes[0]), ctypes.byref(node)) == 0
    if node.func:
        assert cuda.cuFuncGetName(ctypes.byref(name), ctypes.c_void_p(node.func)) == 0
    else:
        assert cuda.cuKernelGetName(ctypes.byref(name), ctypes.c_void_p(node.kern)) == 0
    kind, numbers = re.search(r"gemm_fp8_block_(\w+?_kernel)I((?:Li\d+E)+)E", name.value.decode()).groups()
    return f"{kind}<{', '.join(re.findall(r'[0-9]+', numbers))}>"


@pytest.mark.parametrize("form,m,n,k", [(f, *s) for f, shapes in FORMS for s in shapes])
def test_form(form, m, n, k):
    a, w, sa, sw, bias = operands(m, n, k, m + n)
    assert form_of(a, w, sa, sw) == form
    plain = product(a, w, sa, sw, None, True, False)
    want, size = R.block_product(a, w, sa, sw)
    # a block's 128 additions in the tensor core (2^-23 of its magnitudes each); two roundings of the scale, one of each block's fma, eight of
    # parts of K, one of the bias (2^-24 each); bf16: half a step
    bound = size * (128 * 2.0 ** -23 + (sa.shape[0] + 11) * 2.0 ** -24)
    assert ((plain.to(F64) - want).abs() <= bound).all()
    assert torch.equal(plain, product(a, w, sa, sw, None, True, True))
    wide = want + bias.to(F64)
    bound = bound + bias.to(F64).abs() * 2.0 ** -23
    got = product(a, w, sa, sw, bias, True, True)
    assert ((got.to(F64) - wide).abs() <= bound).all()
    half = product(a, w, sa, sw, bias, False, False)
    assert torch.equal(half, got.to(BF16))                           # the same sums, rounded once


@pytest.mark.parametrize("form", [f for f, _ in FORMS])
def test_two_products_of_a_form_at_once(form):
    """On two streams, each a product of its own: nothing is shared."""
    m, n, k = dict(FORMS)[form][0]
    jobs = [operands(m, n, k, seed) for seed in (1, 2)]
    want = [product(*j[:4], j[4], True, False) for j in jobs]
    from flashrt_b200 import flash_rt_kernels as fvk
    outs = [[torch.full_like(w, -7.0) for _ in range(4)] for w in want]
    sides = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for i in range(4):
        for side, (a, w, sa, sw, b), mine in zip(sides, jobs, outs):
            fvk.GemmRunner().fp8_block_nt(a.data_ptr(), w.data_ptr(), mine[i].data_ptr(), m, n, k, sa.data_ptr(), sw.data_ptr(), side.cuda_stream,
                                          bias=b.data_ptr(), d_f32=True)
    torch.cuda.synchronize()
    assert fvk._lib.call_status("frt_b200_gemm_status", 1) == 0
    for w, mine in zip(want, outs):
        assert all(torch.equal(w, o) for o in mine)

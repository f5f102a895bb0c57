"""dsmoe_set_gemm_sm_limit and the MXFP4 products: what a call launches, read
from its captured graph. A CTA of a product takes a whole SM's shared memory
(one CTA per SM), so that its grid is the number of SMs it holds."""
import ctypes
import itertools

import pytest
import torch

from dsmoe import MXFP4Experts, MXFP4Weight, mxfp4_grouped_linear, mxfp4_linear, mxfp4_matmul, mxfp4_moe, \
    mxfp4_quantize, mxfp4_status
from dsmoe._lib import set_gemm_sm_limit

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
GEMM_THREADS = 640
CLUSTER = 8  # most CTAs of a cluster that shares one tile's K


class KernelNode(ctypes.Structure):
    _fields_ = [("func", ctypes.c_void_p), ("grid", ctypes.c_uint * 3), ("block", ctypes.c_uint * 3),
                ("smem", ctypes.c_uint), ("params", ctypes.c_void_p), ("extra", ctypes.c_void_p),
                ("kern", ctypes.c_void_p), ("ctx", ctypes.c_void_p)]


class Edge(ctypes.Structure):
    _fields_ = [("from_port", ctypes.c_ubyte), ("to_port", ctypes.c_ubyte), ("type", ctypes.c_ubyte),
                ("reserved", ctypes.c_ubyte * 5)]


def launches(fn):
    """[(CTAs, threads of a CTA, may start before its predecessor has ended)] of
    the kernels of ``fn()``, in order, and its result after one replay."""
    fn()  # scratch sizes are asked for once
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = fn()
    cu = ctypes.CDLL("libcuda.so.1")
    g = ctypes.c_void_p(graph.raw_cuda_graph())
    n = ctypes.c_size_t(0)
    assert cu.cuGraphGetNodes(g, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cu.cuGraphGetNodes(g, nodes, ctypes.byref(n)) == 0
    m = ctypes.c_size_t(64)
    src, dst, data = (ctypes.c_void_p * 64)(), (ctypes.c_void_p * 64)(), (Edge * 64)()
    assert cu.cuGraphGetEdges_v2(g, src, dst, data, ctypes.byref(m)) == 0
    after = {src[i]: (dst[i], data[i].type) for i in range(m.value)}
    assert m.value == n.value - 1 == len(after)  # a chain
    (node,) = set(nodes) - set(dst[:m.value])
    early, found = False, []
    while node is not None:
        kind = ctypes.c_int(-1)
        assert cu.cuGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        if kind.value == 0:
            p = KernelNode()
            assert cu.cuGraphKernelNodeGetParams_v2(ctypes.c_void_p(node), ctypes.byref(p)) == 0
            found.append((p.grid[0] * p.grid[1] * p.grid[2], p.block[0], early))
        node, kind = after.get(node, (None, 0))
        early = kind == 1
    graph.instantiate()
    graph.replay()
    torch.cuda.synchronize()
    return found, out


def cases():
    g = torch.Generator(device=DEV)
    g.manual_seed(9)

    def w(*shape):
        return MXFP4Weight(*mxfp4_quantize(torch.randn(*shape, generator=g, device=DEV) * 0.02))

    def x(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16)

    long, wide, narrow = w(7168, 16384), w(2048, 4096), w(576, 7168)
    x1, x24, x100, x40 = x(1, 16384), x(24, 7168), x(100, 4096), x(40, 7168)
    q1, q129 = mxfp4_quantize(x1), mxfp4_quantize(x(129, 7168))
    st, off = w(9, 512, 1024), torch.tensor([0, 0, 3, 40, 40, 41, 100, 120, 299, 300], dtype=torch.int32, device=DEV)
    xg = x(300, 1024)
    ex = MXFP4Experts(w(17, 256, 512), w(17, 256, 512), w(17, 512, 256))
    r = {}
    for t in (3, 200, 1200):
        idx = torch.rand(t, 16, generator=g, device=DEV).topk(4, dim=1).indices
        r[t] = x(t, 512), idx, torch.rand(t, 4, generator=g, device=DEV)
    return {
        "linear 1 x 7168 x 16384": lambda: mxfp4_linear(x1, long),
        "linear 24 x 576 x 7168": lambda: mxfp4_linear(x24, narrow),
        "linear 40 x 576 x 7168": lambda: mxfp4_linear(x40, narrow),
        "linear 100 x 2048 x 4096": lambda: mxfp4_linear(x100, wide),
        "product 1 x 7168 x 16384": lambda: mxfp4_matmul(*q1, long),
        "product 129 x 576 x 7168": lambda: mxfp4_matmul(*q129, narrow),
        "grouped 300 rows": lambda: mxfp4_grouped_linear(xg, st, off),
        **{f"ffn {t} tokens": lambda t=t: mxfp4_moe(*r[t], ex, 1.5) for t in r},
    }


@pytest.mark.parametrize("limit", [1, 5, 37, 100])
def test_the_limit_holds(limit):
    """No launch of more CTAs than the limit (or one cluster), and the same bits."""
    for name, fn in cases().items():
        _, want = launches(fn)
        try:
            set_gemm_sm_limit(limit)
            capped, got = launches(fn)
        finally:
            set_gemm_sm_limit(0)
        gemms = [k for k in capped if k[1] == GEMM_THREADS]
        assert gemms and all(k[0] <= max(limit, CLUSTER) for k in gemms), (name, gemms)
        if limit >= CLUSTER:
            assert all(k[0] <= limit for k in gemms), (name, gemms)
        assert torch.equal(got, want), name
    assert mxfp4_status(DEV) == 0


@pytest.mark.parametrize("limit", [5, 100])
def test_no_kernel_of_a_capped_call_waits_on_the_other_sms(limit):
    """Launched before its predecessor has ended, a kernel would hold the SMs
    that the limit leaves free while it waits: a capped call's products and what
    comes behind them start in turn."""
    for name, fn in cases().items():
        free, _ = launches(fn)
        try:
            set_gemm_sm_limit(limit)
            capped, _ = launches(fn)
        finally:
            set_gemm_sm_limit(0)
        behind = list(itertools.dropwhile(lambda k: k[1] != GEMM_THREADS, capped))
        assert behind and not any(early for _, _, early in behind), (name, capped)
        if "ffn" in name:  # chained where nothing is to be left free
            assert any(early for _, threads, early in free if threads == GEMM_THREADS)

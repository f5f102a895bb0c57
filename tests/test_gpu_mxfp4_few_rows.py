"""MXFP4 products of a few rows, which prepare their rows inside the product
(bf16 rows up to 32, MXFP4 rows in small token tiles), against the 64-bit
oracle: several work units per CTA, K longer than the ring of stages, odd
numbers of K blocks, rows apart, K split over a cluster.

Element bound as in test_gpu_mxfp4.py: one rounding to bf16 (2^-8 relative),
fp32 sums (K 2^-23 S for S = sum |x w|, truncation included), and what the split
of bf16 rows leaves out, at most 2^-12 S for the normal data here."""
import pytest
import torch

from dsmoe import MXFP4Weight, mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize, mxfp4_status
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def gen(*key):
    g = torch.Generator(device=DEV)
    g.manual_seed(sum(int(k) * (i + 7) for i, k in enumerate(key)))
    return g


def check(y, x, w):
    ref, s = O.linear(x, w), x.abs() @ w.abs().T
    bound = 2.0 ** -8 * ref.abs() + (x.shape[1] * 2.0 ** -23 + 2.0 ** -12) * s
    assert bool(((y.double() - ref).abs() <= bound).all())


SHAPES = [(40200, 1152), (38400, 640), (520, 4224), (256, 128), (2056, 32768)]


@pytest.mark.parametrize("N,K", SHAPES)
def test_linear(N, K):
    g = gen(N, K)
    c = mxfp4_quantize(torch.randn(N, K, generator=g, device=DEV) * 0.02)
    w, wd = MXFP4Weight(*c), O.dequantize(*c)
    big = torch.randn(33, K + 24, generator=g, device=DEV).to(torch.bfloat16)
    for T in (1, 4, 5, 8, 9, 15, 16, 17, 23, 24, 25, 32, 33):
        x = big[:T, 8:K + 8]  # rows apart, 16-byte aligned
        y = mxfp4_linear(x, w)
        check(y, x.double(), wd)
        assert torch.equal(mxfp4_linear(x.contiguous(), w), y)
    assert mxfp4_status(DEV) == 0


@pytest.mark.parametrize("N,K", SHAPES)
def test_matmul(N, K):
    g = gen(N, K, 1)
    c = mxfp4_quantize(torch.randn(N, K, generator=g, device=DEV) * 0.02)
    w, wd = MXFP4Weight(*c), O.dequantize(*c)
    for T in (1, 31, 33, 64, 65, 130):
        xq = mxfp4_quantize(torch.randn(T, K, generator=g, device=DEV))
        y = mxfp4_matmul(*xq, w)
        xd = O.dequantize(*xq)
        assert torch.equal(mxfp4_dequantize(*xq, torch.float32).double(), xd)
        check(y, xd, wd)
    assert mxfp4_status(DEV) == 0


def test_rows_that_are_not_numbers_stay_alone():
    g = gen(3)
    w = MXFP4Weight(*mxfp4_quantize(torch.randn(512, 1024, generator=g, device=DEV)))
    x = torch.randn(16, 1024, generator=g, device=DEV).to(torch.bfloat16)
    clean = mxfp4_linear(x, w)
    x[2, 1000], x[9, 0], x[15, 512] = float("nan"), float("inf"), float("-inf")
    y = mxfp4_linear(x, w)
    bad = torch.zeros(16, dtype=torch.bool, device=DEV)
    bad[[2, 9, 15]] = True
    assert bool(torch.isnan(y[bad]).all()) and torch.equal(y[~bad], clean[~bad])


def test_many_calls_in_a_graph_and_on_two_streams():
    """No call uses another's memory: the calls have no scratch of their own."""
    g = gen(4)
    w = MXFP4Weight(*mxfp4_quantize(torch.randn(4096, 2048, generator=g, device=DEV) * 0.02))
    xs = [torch.randn(t, 2048, generator=g, device=DEV).to(torch.bfloat16) for t in (1, 3, 32, 7)]
    qs = [mxfp4_quantize(x) for x in xs]
    want = [(mxfp4_linear(x, w), mxfp4_matmul(*q, w)) for x, q in zip(xs, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 4, mxfp4_linear(xs[i % 4], w), mxfp4_matmul(*qs[i % 4], w)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for i, a, b in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [(mxfp4_linear(x, w), mxfp4_matmul(*q, w)) for x, q in zip(xs, qs)]
    for _ in range(3):
        for pair in out:
            for t in pair:
                t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) and torch.equal(b, d) for (a, b), (c, d) in zip(out, want))
    assert mxfp4_status(DEV) == 0

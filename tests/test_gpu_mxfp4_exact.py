"""MXFP4 operators on data whose results are exact, so that one wrong code, one
K block too many or too few, or a lost term of an activation shows: products of
e4m3 checkpoint numbers right beside a rounding border, and long sums of small
whole numbers. And ragged and routed products on activations with outliers."""
import math

import pytest
import torch

from dsmoe import (MXFP4Experts, MXFP4Weight, mxfp4_grouped_linear, mxfp4_linear, mxfp4_matmul, mxfp4_moe,
                   mxfp4_quantize, mxfp4_status)
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TIES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def gen(*key):
    g = torch.Generator(device=DEV)
    g.manual_seed(sum(int(k) * (i + 11) for i, k in enumerate(key)))
    return g


def near_ties():
    """(w, m, s, side): e4m3 w and m, fp32 s with 4 <= m s < 8 (scale 1), where
    w s is not a tie of the grid but rounds to it in fp32, and the even code at
    the tie is not the nearest of w s (which lies on ``side`` of it)."""
    found = []
    for i, tie in enumerate(TIES):
        side = 1 if i % 2 == 0 else -1  # the even code is below ties 0, 2, 4, 6 and above 1, 3, 5
        for w in range(9, 16):
            near = torch.tensor(tie / w, dtype=torch.float32)
            for s in (near, torch.nextafter(near, torch.tensor(0.0)), torch.nextafter(near, torch.tensor(9.0))):
                exact = w * float(s)  # 28 bits
                if float(torch.tensor(float(w)) * s) == tie and (exact - tie) * side > 0:
                    found.append((w, 2.0 ** math.ceil(math.log2(4 / float(s))), float(s), side))
    return found


@pytest.mark.parametrize("power", [-130, -100, 0, 90])
def test_quantize_fp8_beside_ties(power):
    """Rounding the product to fp32 first gives another code in every one of these blocks."""
    cases = near_ties()
    assert len({c[3] for c in cases}) == 2 and len(cases) >= 10
    x = torch.zeros(len(cases), 1, 32)
    s = torch.zeros(len(cases), 1, 1)
    for i, (w, m, scale, _) in enumerate(cases):
        x[i, 0, 0], x[i, 0, 1::2], x[i, 0, 2::2] = m, w, -w
        s[i] = scale
    sp = torch.ldexp(s.double(), torch.tensor(power)).float()
    if power > -126:
        assert torch.equal(sp.double(), torch.ldexp(s.double(), torch.tensor(power)))
    q = x.to(torch.float8_e4m3fn)
    assert torch.equal(q.float(), x)
    rc, rs = O.quantize(q, sp)
    if power > -126:
        assert bool((rs == 127 + power).all())
        nc, ns = O.quantize(x * sp)  # the fp32 product
        assert torch.equal(ns, rs) and bool((nc != rc).flatten(1).any(1).all())
    codes, scales = mxfp4_quantize(q.to(DEV), sp.to(DEV))
    assert torch.equal(scales.cpu(), rs) and torch.equal(codes.cpu(), rc)


def whole_weight(g, N, K):
    """Codes of whole numbers (0, 1, 2, 3 and negatives) under scale 1."""
    table = torch.tensor([0, 2, 4, 5, 8, 10, 12, 13], dtype=torch.uint8, device=DEV)
    c = table[torch.randint(0, 8, (N, K // 2, 2), generator=g, device=DEV)]
    codes = c[..., 0] | (c[..., 1] << 4)
    scales = torch.full((N, K // 32), 127, dtype=torch.uint8, device=DEV)
    return codes, scales


SHAPES = [(2056, 32768), (264, 32640), (520, 4224), (7168, 2048)]


@pytest.mark.parametrize("N,K", SHAPES)
def test_whole_numbers(N, K):
    """One number of 0, 1 or -1 in 32 is not 0. Every partial sum, in whatever
    order, is a whole number of at most sum |x w| < 2^12: exact in far fewer bits
    than an fp32 sum's 24, and so is the result but for its rounding to bf16.
    128 numbers more or less change it by several."""
    g = gen(N, K)
    c = whole_weight(g, N, K)
    w, wd = MXFP4Weight(*c), O.dequantize(*c)
    x = torch.zeros(700, K // 32, 32, device=DEV)
    pick = torch.randint(0, 32, (700, K // 32, 1), generator=g, device=DEV)
    x.scatter_(2, pick, torch.randint(-1, 2, pick.shape, generator=g, device=DEV).float())
    x = x.view(700, K)
    for T in (1, 5, 16, 17, 32, 33, 64, 65, 130, 300, 700):
        xt = x[:T]
        s = xt.double().abs() @ wd.abs().T
        assert float(s.max()) < 2 ** 12
        want = O.linear(xt, wd).float().to(torch.bfloat16)
        assert torch.equal(mxfp4_linear(xt.to(torch.bfloat16), w), want), T
        assert torch.equal(mxfp4_matmul(*mxfp4_quantize(xt), w), want), T
    assert mxfp4_status(DEV) == 0


@pytest.mark.parametrize("N,K", SHAPES[:3])
@pytest.mark.parametrize("T", [1, 16, 32, 64, 160])
def test_one_number_per_row_in_every_k_block(T, N, K):
    """Each row has one number other than 0, in another K block from row to row
    and from call to call: the result is that number times its weight. bf16 rows
    take numbers of eight significant bits, whose upper and lower terms both
    count: (128 .. 255) * (0, 1, 2 or 3) has ten bits and is rounded once."""
    g = gen(T, N, K)
    c = whole_weight(g, N, K)
    w, wd = MXFP4Weight(*c), O.dequantize(*c)
    rows = torch.arange(T, device=DEV)
    blocks = K // 128
    for at in range(0, blocks, T):
        col = (at + rows) % blocks * 128 + torch.randint(0, 128, (T,), generator=g, device=DEV)
        v = torch.randint(128, 256, (T,), generator=g, device=DEV).double()
        want = (wd[:, col].T * v[:, None]).float().to(torch.bfloat16)
        x = torch.zeros(T, K, dtype=torch.bfloat16, device=DEV)
        x[rows, col] = v.to(torch.bfloat16)
        assert torch.equal(mxfp4_linear(x, w), want), at
        x[rows, col] = 1.0
        assert torch.equal(mxfp4_matmul(*mxfp4_quantize(x), w), wd[:, col].T.to(torch.bfloat16)), at
    assert mxfp4_status(DEV) == 0


def outliers(g, rows, K):
    """Normal activations with a channel in forty 256 times as large: most
    numbers of such a block are below 2^-9 of its largest, or close to it."""
    x = torch.randn(rows, K, generator=g, device=DEV)
    x[:, ::40] *= 256.0
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("E,R,N,K", [(8, 40, 264, 384), (4, 200, 512, 1024), (3, 1500, 256, 512)])
def test_grouped_linear_with_outliers(E, R, N, K):
    """Element bound: one rounding to bf16, fp32 sums, and what the split leaves
    of numbers below 2^-9 of their block's largest, 2^-17 of it each."""
    g = gen(E, R, N, K)
    c = mxfp4_quantize(torch.randn(E, N, K, generator=g, device=DEV) * 0.02)
    wd = O.dequantize(*c)
    x = outliers(g, R, K)
    cuts = torch.randint(0, R + 1, (E - 1,), generator=g, device=DEV).sort().values.tolist()
    off = [0, *cuts, R]
    y = mxfp4_grouped_linear(x, MXFP4Weight(*c), torch.tensor(off, dtype=torch.int32, device=DEV)).double()
    for e in range(E):
        xe, we = x[off[e]:off[e + 1]].double(), wd[e]
        ref, s = O.linear(xe, we), xe.abs() @ we.abs().T
        left = 2.0 ** -17 * xe.view(-1, K // 32, 32).abs().amax(-1) @ we.view(N, K // 32, 32).abs().sum(-1).T
        bound = 2.0 ** -8 * ref.abs() + K * 2.0 ** -23 * s + left
        assert bool(((y[off[e]:off[e + 1]] - ref).abs() <= bound).all())
    assert mxfp4_status(DEV) == 0


@pytest.mark.parametrize("T", [1, 40, 700])
def test_moe_with_outliers(T):
    """Mean square, relative to the terms of the sum without cancellation: h to
    2^-9, an expert's row and the result to 2^-8 each. The split's share: what it
    leaves out of a row is at most 2^-17 sqrt(32) = 2^-14.5 of the row's norm,
    hence as much of gate's and up's mean square for weights of random sign, and
    with |silu'| < 1.1 less than 2^-12 of h's."""
    H, F, E, k = 512, 256, 16, 4
    g = gen(T, H)
    pairs = [mxfp4_quantize(torch.randn(E + 1, *s, generator=g, device=DEV) * 0.02) for s in ((F, H), (F, H), (H, F))]
    deq = [O.dequantize(*p) for p in pairs]
    x = outliers(g, T, H)
    idx = torch.rand(T, E, generator=g, device=DEV).topk(k, dim=1).indices
    w = torch.rand(T, k, generator=g, device=DEV) + 0.1
    y = mxfp4_moe(x, idx, w, MXFP4Experts(*(MXFP4Weight(*p) for p in pairs)), scale=1.5).double()
    ref = O.moe(x, idx, w, *deq, True, 1.5)
    terms = O.ffn(x, deq[0][0], deq[1][0], deq[2][0]).pow(2)
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            v = O.ffn(x[t], deq[0][e + 1], deq[1][e + 1], deq[2][e + 1])
            terms.index_add_(0, t, (1.5 * w[t, j].double().unsqueeze(1) * v).pow(2))
    err = float((y - ref).pow(2).mean().sqrt() / terms.mean().sqrt())
    assert err <= (2.0 ** -9 + 2.0 ** -12 + 2 * 2.0 ** -8) / math.sqrt(3), err
    assert mxfp4_status(DEV) == 0

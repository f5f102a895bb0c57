"""MXFP4 operators on the GPU against the 64-bit oracle (oracle/mxfp4.py).

Tolerances, fixed by arithmetic:
  * quantise, dequantise: exact (power-of-two scales make every step exact but
    the one rounding, whose ties go to the even code).
  * products: every output is rounded once to bf16 (relative 2^-8 at most,
    2^-8 / sqrt(3) in the mean square), the sums are fp32. With
    S = sum_k |x_k w_k| a sum of K fp32 terms is off by at most K 2^-23 S even
    if each addition truncates, and the activations' split leaves out at most
    2^-17 of a block's largest number (only numbers below 2^-9 of it), at most
    2^-17 * 32 * S_block-max <= 2^-12 S for the data here, whose blocks keep
    sum |x_k w_k| >= max|x| max|w| / 4. Element bound: 2^-8 |ref| + (K 2^-23 +
    2^-12) S; mean square: 2^-8 / sqrt(3) of the reference's plus K 2^-24 of
    S's (errors of random sign).
  * routed FFN: h is kept to 2^-9 relative, each expert's row is rounded to
    bf16 (2^-8), the output once more (2^-8): mean square (2^-9 + 2 * 2^-8) /
    sqrt(3) of a sum without cancellation, and at most 3 times that for a sum
    of up to 9 random-sign terms whose mean square is compared term by term.
"""
import math
import zlib

import pytest
import torch

from dsmoe import (MXFP4Experts, MXFP4Weight, mxfp4_dequantize, mxfp4_grouped_linear, mxfp4_linear, mxfp4_matmul,
                   mxfp4_moe, mxfp4_quantize, mxfp4_status)
from dsmoe.synthetic import block_quantize
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def gen(*key):
    g = torch.Generator(device=DEV)
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def weight(g, *shape, std=0.02):
    return mxfp4_quantize(torch.randn(*shape, generator=g, device=DEV) * std)


def check_product(y, x, w):
    """y against x @ w.T: x, w float64 (rows of x times one weight)."""
    ref = O.linear(x, w)
    s = x.abs() @ w.abs().T
    K = x.shape[1]
    err = (y.double() - ref).abs()
    bound = 2.0 ** -8 * ref.abs() + (K * 2.0 ** -23 + 2.0 ** -12) * s
    assert bool((err <= bound).all()), float((err / bound).max())
    if ref.numel() >= 256:
        rms = math.sqrt(float(err.pow(2).mean()))
        lim = 2.0 ** -8 / math.sqrt(3) * math.sqrt(float(ref.pow(2).mean())) + \
            K * 2.0 ** -24 * math.sqrt(float(s.pow(2).mean()))
        assert rms <= lim, (rms, lim)


# ------------------------------------------------------------------ quantise
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(32,), (1, 64), (3, 5, 96), (130, 7168), (0, 64), (4099, 32)])
def test_quantize_exact(dtype, shape):
    g = gen("q", str(dtype), shape)
    x = (torch.randn(*shape, generator=g, device=DEV) * torch.exp2(
        torch.randint(-12, 5, (*shape[:-1], 1), generator=g, device=DEV).float())).to(dtype)
    codes, scales = mxfp4_quantize(x)
    rc, rs = O.quantize(x.cpu())
    assert torch.equal(scales.cpu(), rs)
    assert torch.equal(codes.cpu(), rc)
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(mxfp4_dequantize(codes, scales, out).cpu().double(), O.dequantize(rc, rs))


def test_quantize_borders():
    """Ties of every grid interval, saturation, zeros, the type's extremes,
    subnormals, blocks with infinities and NaN."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99])
    rows = []
    for e in (-140, -127, -126, -3, 0, 7, 124, 125):
        r = torch.zeros(32, dtype=torch.float64)
        r[0] = 4.0 + (3.99 if e % 2 else 0.0)
        r[1:11], r[11:21] = mids, -mids
        r[21:31] = mids * (1 + 2.0 ** -20)
        rows.append(torch.ldexp(r, torch.tensor(e)).clamp(-3.4e38, 3.4e38))
    rows.append(torch.zeros(32, dtype=torch.float64))
    rows.append(-torch.zeros(32, dtype=torch.float64))
    tiny = torch.full((32,), 2.0 ** -149, dtype=torch.float64)
    rows.append(tiny)
    rows.append(torch.full((32,), torch.finfo(torch.float32).max, dtype=torch.float64))
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.ones(32, dtype=torch.float64)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows).float()
    codes, scales = mxfp4_quantize(x.to(DEV))
    rc, rs = O.quantize(x)
    assert torch.equal(scales.cpu(), rs)
    assert torch.equal(codes.cpu(), rc)
    y, ref = mxfp4_dequantize(codes, scales, torch.float32).cpu().double(), O.dequantize(rc, rs)
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    assert torch.equal(y.nan_to_num(7.0), ref.nan_to_num(7.0))
    h = mxfp4_dequantize(codes, scales, torch.float16).cpu()
    assert torch.equal(h.nan_to_num(7.0), ref.float().half().nan_to_num(7.0))


@pytest.mark.parametrize("shape", [(1, 32), (130, 160), (3, 129, 320), (2, 576, 7168)])
def test_quantize_fp8_checkpoint(shape):
    g = gen("f8", shape)
    x = (torch.randn(*shape, generator=g, device=DEV) * 90).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.rand(*shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128), generator=g, device=DEV) * 3e-4 + 1e-5
    codes, scales = mxfp4_quantize(x, s)
    rc, rs = O.quantize(x.cpu(), s.cpu())
    assert torch.equal(scales.cpu(), rs) and torch.equal(codes.cpu(), rc)


def test_quantize_fp8_rounds_the_exact_product():
    """Products next to a tie: fp32 would round them onto it."""
    x = torch.zeros(1, 32)
    x[0, 0], x[0, 1:] = 416.0, 13.0
    q = x.to(torch.float8_e4m3fn)
    # 13 s is next to a tie of the grid, 416 s = 32 * 13 s sets the scale
    for tie in (0.25, 0.75):
        for d in range(-3, 4):
            s = torch.tensor([[tie / 13.0]]).float()
            s = torch.nextafter(s, torch.full_like(s, math.copysign(1e9, d))) if d else s
            codes, scales = mxfp4_quantize(q.to(DEV), s.to(DEV))
            rc, rs = O.quantize(q, s)
            assert torch.equal(codes.cpu(), rc) and torch.equal(scales.cpu(), rs)


def test_quantize_strides():
    g = gen("st")
    big = torch.randn(40, 6, 256, generator=g, device=DEV).to(torch.bfloat16)
    for v in (big[:, 2], big[:, :, 32:96], big[::3, 1, :64], big.transpose(0, 1), big.expand(2, 40, 6, 256),
              big[:, 0, 1:33], big[5:6, 0, 3:35]):
        a, b = mxfp4_quantize(v)
        rc, rs = O.quantize(v.cpu())
        assert torch.equal(a.cpu(), rc) and torch.equal(b.cpu(), rs)
    t = torch.randn(64, 33, generator=g, device=DEV).T  # K strided
    a, b = mxfp4_quantize(t)
    rc, rs = O.quantize(t.cpu())
    assert torch.equal(a.cpu(), rc) and torch.equal(b.cpu(), rs)


# ------------------------------------------------------------------ products
@pytest.mark.parametrize("T", [1, 2, 17, 31, 32, 33, 64, 65, 96, 97, 113, 128, 160, 161, 257, 700])
@pytest.mark.parametrize("N,K", [(256, 128), (8, 256), (576, 1152), (392, 2048)])
def test_linear(T, N, K):
    g = gen("lin", T, N, K)
    x = torch.randn(T, K, generator=g, device=DEV).to(torch.bfloat16)
    codes, scales = weight(g, N, K)
    y = mxfp4_linear(x, MXFP4Weight(codes, scales))
    assert y.shape == (T, N) and mxfp4_status(DEV) == 0
    check_product(y, x.double(), O.dequantize(codes, scales))


@pytest.mark.parametrize("T,N,K", [(1, 7168, 16384), (3, 2048, 7168), (48, 24576, 1536), (512, 7168, 2048),
                                   (1000, 1536, 7168)])
def test_linear_model_shapes(T, N, K):
    g = gen("lm", T, N, K)
    x = torch.randn(T, K, generator=g, device=DEV).to(torch.bfloat16)
    codes, scales = weight(g, N, K)
    w = MXFP4Weight(codes, scales)
    y = mxfp4_linear(x, w)
    assert mxfp4_status(DEV) == 0
    check_product(y, x.double(), O.dequantize(codes, scales))
    assert torch.equal(y, mxfp4_linear(x, w))  # also with K split over CTAs


@pytest.mark.parametrize("T", [1, 16, 63, 65, 128, 129, 192, 193, 400])
@pytest.mark.parametrize("N,K", [(256, 128), (8, 256), (576, 1152), (392, 2048)])
def test_matmul(T, N, K):
    g = gen("mm", T, N, K)
    ac, asc = weight(g, T, K, std=1.0)
    codes, scales = weight(g, N, K)
    y = mxfp4_matmul(ac, asc, MXFP4Weight(codes, scales))
    assert y.shape == (T, N) and mxfp4_status(DEV) == 0
    check_product(y, O.dequantize(ac, asc), O.dequantize(codes, scales))


def test_linear_strides_and_leading_dims():
    g = gen("ls")
    codes, scales = weight(g, 264, 384)
    w, wd = MXFP4Weight(codes, scales), O.dequantize(codes, scales)
    big = torch.randn(7, 5, 1024, generator=g, device=DEV).to(torch.bfloat16)
    for x in (big[..., :384], big[:, 1, 640:], big[..., 5:389], big.transpose(0, 1)[..., 128:512],
              big[:1, :1, :384].expand(3, 4, 384), big[0, 0, :384]):
        y = mxfp4_linear(x, w)
        assert y.shape == (*x.shape[:-1], 264)
        check_product(y.reshape(-1, 264), x.reshape(-1, 384).double(), wd)
    assert mxfp4_linear(big[:0, :, :384], w).shape == (0, 5, 264)


def test_linear_magnitudes():
    """Rows of very different size, blocks with one large number, zeros, the
    smallest bf16: each row's error is bounded by its own sums."""
    g = gen("mag")
    codes, scales = weight(g, 512, 1024)
    scales = (scales.int() + torch.randint(-20, 20, scales.shape, generator=g, device=DEV)).to(torch.uint8)
    x = torch.randn(64, 1024, generator=g, device=DEV)
    x *= torch.exp2(torch.randint(-60, 60, (64, 1), generator=g, device=DEV).float())
    x[5], x[6] = 0.0, 2.0 ** -133
    x[7:20, ::40] *= 1000.0
    x = x.to(torch.bfloat16)
    xd, wd = x.double(), O.dequantize(codes, scales)
    y = mxfp4_linear(x, MXFP4Weight(codes, scales)).double()
    ref, s = O.linear(xd, wd), xd.abs() @ wd.abs().T
    amax = xd.view(64, -1, 32).abs().amax(-1)
    left = 2.0 ** -17 * amax @ wd.view(512, -1, 32).abs().sum(-1).T  # numbers below 2^-9 of their block
    # results below the smallest normal bf16 (2^-126) round to its subnormal step
    bound = 2.0 ** -8 * ref.abs() + 1024 * 2.0 ** -23 * s + left + 2.0 ** -133
    assert bool(((y - ref).abs() <= bound).all())
    assert bool((y[5] == 0).all())


def test_split_is_exact_near_the_block_maximum():
    """The identity as the weight: a bf16 comes back as it was, whatever its
    place in the block, down to 2^-9 of the block's largest number."""
    K = 256
    codes = torch.zeros(K, K // 2, dtype=torch.uint8, device=DEV)
    i = torch.arange(K, device=DEV)
    codes[i, i // 2] = torch.where(i % 2 == 0, 2, 2 << 4).to(torch.uint8)  # the identity
    scales = torch.full((K, K // 32), 127, dtype=torch.uint8, device=DEV)
    w = MXFP4Weight(codes, scales)
    g = gen("id")
    m = torch.randint(128, 256, (300, K), generator=g, device=DEV).float()
    e = torch.randint(-9, 1, (300, K), generator=g, device=DEV).float()
    e[:, ::32], m[:, ::32] = 1.0, 128.0  # the block's largest
    x = (m * torch.exp2(e) * (1 - 2 * torch.randint(0, 2, (300, K), generator=g, device=DEV).float())).to(torch.bfloat16)
    # The block's largest is 2^8, so a split step is 2 * 2^-9 = 2^-8: a bf16 of
    # at least 2^-9 of it (0.5, whose last bit is 2^-8) is a multiple of the
    # step and exact; the data's smaller ones (0.25 to 0.5) round to a multiple
    # of it, off by at most 2^-9, and that multiple is a bf16.
    big = x.abs() >= 0.5
    for T in (300, 1, 20, 50, 150):
        y = mxfp4_linear(x[:T], w)
        assert torch.equal(y[big[:T]], x[:T][big[:T]])
        assert float((y.double() - x[:T].double()).abs().max()) <= 2.0 ** -9


def test_non_finite():
    g = gen("nf")
    codes, scales = weight(g, 256, 256)
    w = MXFP4Weight(codes, scales)
    x = torch.randn(40, 256, generator=g, device=DEV).to(torch.bfloat16)
    clean = mxfp4_linear(x, w)
    x[3, 70], x[35, 0] = float("nan"), float("inf")
    y = mxfp4_linear(x, w)
    rest = torch.ones(40, dtype=torch.bool, device=DEV)
    rest[3] = rest[35] = False
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[35]).all())
    assert torch.equal(y[rest], clean[rest])
    s2 = scales.clone()
    s2[17, 3] = 255  # a weight block that is NaN: that output feature only
    y = mxfp4_linear(x, MXFP4Weight(codes, s2))
    keep = torch.arange(256, device=DEV) != 17
    assert bool(torch.isnan(y[:, 17]).all()) and torch.equal(y[rest][:, keep], clean[rest][:, keep])


# ------------------------------------------------------------------- grouped
def segments(kind, E, R, g):
    if kind == "one":
        c = [0] * E
        c[E // 2] = R
    elif kind == "uniform":
        c = torch.bincount(torch.randint(0, E, (R,), generator=g, device=DEV), minlength=E).tolist()
    else:  # a few experts take most rows, many none
        c = torch.bincount((torch.rand(R, generator=g, device=DEV) ** 4 * E).long(), minlength=E).tolist()
    off = [0]
    for n in c:
        off.append(off[-1] + n)
    return off


@pytest.mark.parametrize("kind", ["one", "uniform", "skewed"])
@pytest.mark.parametrize("E,R", [(1, 5), (3, 1), (8, 200), (17, 600), (64, 64), (300, 90), (512, 2000)])
def test_grouped_linear(kind, E, R):
    g = gen("gr", kind, E, R)
    N, K = 264, 384
    codes, scales = weight(g, E, N, K)
    off = segments(kind, E, R, g)
    tail = 3
    x = torch.randn(R + tail, K, generator=g, device=DEV).to(torch.bfloat16)
    x[R:] = float("nan")  # rows behind the last segment are not read into any result
    w, wd = MXFP4Weight(codes, scales), O.dequantize(codes, scales)
    offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
    y = mxfp4_grouped_linear(x, w, offsets)
    assert mxfp4_status(DEV) == 0
    for e in range(E):
        if off[e + 1] > off[e]:
            check_product(y[off[e]:off[e + 1]], x[off[e]:off[e + 1]].double(), wd[e])
    assert bool((y[R:] == 0).all())
    out = torch.full_like(y, 7.0)
    assert mxfp4_grouped_linear(x, w, offsets, out=out) is out
    assert torch.equal(out[:R], y[:R]) and bool((out[R:] == 7).all())


def test_grouped_rows_before_the_first_segment():
    g = gen("gb")
    codes, scales = weight(g, 2, 256, 256)
    x = torch.randn(50, 256, generator=g, device=DEV).to(torch.bfloat16)
    y = mxfp4_grouped_linear(x, MXFP4Weight(codes, scales), torch.tensor([10, 30, 41], dtype=torch.int32, device=DEV))
    wd = O.dequantize(codes, scales)
    check_product(y[10:30], x[10:30].double(), wd[0])
    check_product(y[30:41], x[30:41].double(), wd[1])
    assert bool((y[:10] == 0).all()) and bool((y[41:] == 0).all())


@pytest.mark.parametrize("off", [[0, 40, 20, 50], [-5, 10, 20, 50], [0, 10, 20, 90], [60, 70, 80, 90],
                                 [2 ** 31 - 1, -2 ** 31, 5, 6]])
def test_grouped_bad_offsets_are_reported(off):
    """Clamped to the rows, never read or written past them; reported once."""
    g = gen("bo")
    codes, scales = weight(g, 3, 256, 256)
    x = torch.randn(50, 256, generator=g, device=DEV).to(torch.bfloat16)
    w = MXFP4Weight(codes, scales)
    out = torch.full((52, 256), 3.0, dtype=torch.bfloat16, device=DEV)
    mxfp4_grouped_linear(x, w, torch.tensor(off, dtype=torch.int32, device=DEV), out=out[:50])
    assert mxfp4_status(DEV) == 6 and mxfp4_status(DEV) == 0
    assert bool((out[50:] == 3).all())
    good = torch.tensor([0, 10, 20, 50], dtype=torch.int32, device=DEV)
    check_product(mxfp4_grouped_linear(x, w, good)[:10], x[:10].double(), O.dequantize(codes, scales)[0])
    assert mxfp4_status(DEV) == 0


# ---------------------------------------------------------------- routed FFN
def routing(g, T, E, k):
    idx = torch.rand(T, E, generator=g, device=DEV).topk(k, dim=1).indices
    w = torch.rand(T, k, generator=g, device=DEV) + 0.1
    return idx, w / w.sum(1, keepdim=True)


def experts(g, G, H, F):
    pairs = [weight(g, G, F, H), weight(g, G, F, H), weight(g, G, H, F)]
    return [MXFP4Weight(*p) for p in pairs], [O.dequantize(*p) for p in pairs]


def check_moe(y, x, idx, w, deq, shared, scale):
    ref = O.moe(x, idx, w, *deq, shared, scale)
    # size of the terms each output is a sum of, without cancellation
    base = int(shared)
    terms = O.ffn(x, deq[0][0], deq[1][0], deq[2][0]).pow(2) if shared else torch.zeros_like(ref)
    for e in range(deq[0].shape[0] - base):
        t, k = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            v = O.ffn(x[t], deq[0][base + e], deq[1][base + e], deq[2][base + e])
            terms.index_add_(0, t, (scale * w[t, k].double().unsqueeze(1) * v).pow(2))
    err = (y.double() - ref).pow(2).mean().sqrt()
    assert float(err) <= (2.0 ** -9 + 2 * 2.0 ** -8) / math.sqrt(3) * float(terms.mean().sqrt()), \
        float(err / terms.mean().sqrt())


@pytest.mark.parametrize("T,E,k,H,F,shared", [
    (1, 8, 1, 128, 128, False), (1, 32, 8, 512, 256, True), (5, 9, 3, 384, 640, True), (64, 256, 8, 256, 128, True),
    (33, 4, 4, 256, 384, False), (300, 16, 2, 512, 256, True), (700, 5, 5, 256, 256, True), (1100, 8, 2, 384, 128, False),
    (200, 511, 8, 128, 128, True), (130, 1, 1, 256, 256, True)])
def test_moe(T, E, k, H, F, shared):
    g = gen("moe", T, E, k, H, F)
    ws, deq = experts(g, E + int(shared), H, F)
    x = torch.randn(T, H, generator=g, device=DEV).to(torch.bfloat16) * 3
    idx, w = routing(g, T, E, k)
    ex = MXFP4Experts(*ws, shared=shared)
    y = mxfp4_moe(x, idx, w, ex, scale=2.5)
    assert mxfp4_status(DEV) == 0
    check_moe(y, x, idx, w, deq, shared, 2.5)
    assert torch.equal(y, mxfp4_moe(x, idx, w, ex, scale=2.5))  # the same bits every time


def test_moe_ids_outside_and_repeated():
    g = gen("moe-ids")
    ws, deq = experts(g, 7, 256, 128)
    x = torch.randn(9, 256, generator=g, device=DEV).to(torch.bfloat16)
    idx, w = routing(g, 9, 6, 4)
    idx[0] = -1               # a token without an expert: the shared expert only
    idx[1, 2], idx[2, 0] = 6, 1 << 40
    idx[3, :] = 4             # the same expert four times
    y = mxfp4_moe(x, idx, w, MXFP4Experts(*ws), scale=1.5)
    check_moe(y, x, idx, w, deq, True, 1.5)
    alone = mxfp4_moe(x, idx[:, :1] * 0 - 1, w[:, :1], MXFP4Experts(*ws))
    assert torch.equal(alone[0], y[0])


def test_moe_one_nan_token_stays_alone():
    g = gen("moe-nan")
    ws, _ = experts(g, 9, 256, 256)
    x = torch.randn(50, 256, generator=g, device=DEV).to(torch.bfloat16)
    idx, w = routing(g, 50, 8, 2)
    ex = MXFP4Experts(*ws)
    clean = mxfp4_moe(x, idx, w, ex)
    x[11, 5] = float("nan")
    y = mxfp4_moe(x, idx, w, ex)
    rest = torch.arange(50, device=DEV) != 11
    assert bool(torch.isnan(y[11]).all()) and torch.equal(y[rest], clean[rest])


# --------------------------------------------------------- streams and graphs
def test_graphs_and_streams():
    """Captured calls replay on new inputs; two graphs replayed on two streams
    at the same time do not share scratch."""
    g = gen("graph")
    ws, _ = experts(g, 17, 512, 256)
    ex = MXFP4Experts(*ws)
    lw = MXFP4Weight(*weight(g, 512, 2048))
    xs = [torch.randn(64, 512, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    zs = [torch.randn(3, 2048, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    routes = [routing(g, 64, 16, 4) for _ in range(2)]
    want = [(mxfp4_moe(x, *r, ex), mxfp4_linear(z, lw)) for x, r, z in zip(xs, routes, zs)]
    graphs, bufs = [], []
    for i in range(2):
        x, z = torch.zeros_like(xs[0]), torch.zeros_like(zs[0])
        idx, w = routes[0][0].clone(), routes[0][1].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = (mxfp4_moe(x, idx, w, ex), mxfp4_linear(z, lw))
        graphs.append(gr)
        bufs.append((x, z, idx, w, out))
    for rep in range(10):
        for i, (x, z, idx, w, _) in enumerate(bufs):
            j = (i + rep) % 2
            x.copy_(xs[j]), z.copy_(zs[j]), idx.copy_(routes[j][0]), w.copy_(routes[j][1])
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for i, b in enumerate(bufs):
            j = (i + rep) % 2
            assert torch.equal(b[4][0], want[j][0]) and torch.equal(b[4][1], want[j][1])
    assert mxfp4_status(DEV) == 0


def test_quantised_weight_from_the_checkpoint_runs_together():
    """FP8 checkpoint weight -> MXFP4 -> quantised activations -> product,
    against the same steps in 64 bits."""
    g = gen("run")
    q, s = block_quantize(torch.randn(576, 512, generator=g, device=DEV) * 0.02)
    w = MXFP4Weight.quantize(q, s)
    rc, rs = O.quantize(q, s)
    x = torch.randn(130, 512, generator=g, device=DEV).to(torch.bfloat16)
    xc, xs = mxfp4_quantize(x)
    check_product(mxfp4_matmul(xc, xs, w), O.dequantize(*O.quantize(x)), O.dequantize(rc, rs))
    check_product(mxfp4_linear(x, w), x.double(), O.dequantize(rc, rs))


# ------------------------------------------------------------------ refusals
def test_python_refusals():
    g = gen("ref")
    bf = torch.bfloat16
    w = MXFP4Weight(*weight(g, 64, 256))
    st = MXFP4Weight(*weight(g, 3, 64, 256))
    x = torch.zeros(4, 256, dtype=bf, device=DEV)
    off = torch.zeros(4, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError):
        mxfp4_linear(x.float(), w)
    with pytest.raises(ValueError):
        mxfp4_linear(x[:, :128], w)
    with pytest.raises(ValueError):
        mxfp4_linear(x, st)
    with pytest.raises(RuntimeError, match="CUDA"):
        mxfp4_linear(x.cpu(), w)
    with pytest.raises(RuntimeError, match="backward"):
        mxfp4_linear(x.clone().requires_grad_(), w)
    with torch.no_grad():
        mxfp4_linear(x.clone().requires_grad_(), w)
    with pytest.raises(ValueError):
        mxfp4_grouped_linear(x, w, off)
    with pytest.raises(ValueError):
        mxfp4_grouped_linear(x, st, off[:3])
    with pytest.raises(ValueError):
        mxfp4_grouped_linear(x, st, off.long())
    with pytest.raises(ValueError):
        mxfp4_grouped_linear(x.view(2, 2, 256), st, off)
    with pytest.raises(ValueError):
        mxfp4_grouped_linear(x, st, off, out=torch.empty(4, 72, dtype=bf, device=DEV)[:, :64])
    with pytest.raises(ValueError):
        MXFP4Weight(*weight(g, 64, 160))      # in % 128
    with pytest.raises(ValueError):
        MXFP4Weight(*weight(g, 12, 256))      # out % 8
    with pytest.raises(ValueError):
        mxfp4_quantize(torch.zeros(4, 40, device=DEV))
    with pytest.raises(TypeError):
        mxfp4_quantize(torch.zeros(4, 64, dtype=torch.float64, device=DEV))
    with pytest.raises(TypeError):
        mxfp4_quantize(torch.zeros(4, 64, device=DEV).to(torch.float8_e4m3fn))
    with pytest.raises(ValueError):
        mxfp4_quantize(torch.zeros(4, 64, device=DEV).to(torch.float8_e4m3fn), torch.ones(2, 1, device=DEV))
    c, s = weight(g, 8, 256)
    with pytest.raises(ValueError):
        mxfp4_dequantize(c, s[:, :4])
    with pytest.raises(TypeError):
        mxfp4_dequantize(c, s, torch.float64)
    with pytest.raises(ValueError):
        mxfp4_matmul(c[:, :64], s[:, :4], w)
    ex = MXFP4Experts(MXFP4Weight(*weight(g, 3, 128, 256)), MXFP4Weight(*weight(g, 3, 128, 256)),
                      MXFP4Weight(*weight(g, 3, 256, 128)))
    idx, tw = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.ones(4, 2, device=DEV)
    mxfp4_moe(x, idx, tw, ex)
    with pytest.raises(TypeError):
        mxfp4_moe(x, idx.int(), tw, ex)
    with pytest.raises(ValueError):
        mxfp4_moe(x, idx[:3], tw[:3], ex)
    with pytest.raises(RuntimeError):  # top_k > 8
        mxfp4_moe(x, idx.repeat(1, 5), tw.repeat(1, 5), ex)
    with pytest.raises(ValueError):
        MXFP4Experts(st, st, st)
    assert mxfp4_status(DEV) == 0


def test_current_device_and_default_stream_are_left_alone():
    w = MXFP4Weight(*weight(gen("dev"), 64, 256))
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    want = mxfp4_linear(x, w)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = mxfp4_linear(x, w)
        assert torch.cuda.current_stream() == side
    side.synchronize()
    assert torch.equal(y, want) and torch.cuda.current_device() == 0


# ------------------------------------------------- calls at the edge of the rules
def test_no_rows_for_any_expert():
    g = gen("none")
    w = MXFP4Weight(*weight(g, 5, 256, 256))
    x = torch.randn(40, 256, generator=g, device=DEV).to(torch.bfloat16)
    off = torch.zeros(6, dtype=torch.int32, device=DEV)
    assert bool((mxfp4_grouped_linear(x, w, off) == 0).all())
    assert mxfp4_grouped_linear(x[:0], w, off).shape == (0, 256)
    ws, _ = experts(g, 8, 256, 128)
    idx = torch.full((40, 3), -1, dtype=torch.int64, device=DEV)
    tw = torch.ones(40, 3, device=DEV)
    assert bool((mxfp4_moe(x, idx, tw, MXFP4Experts(*ws, shared=False)) == 0).all())
    assert mxfp4_moe(x[:0], idx[:0], tw[:0], MXFP4Experts(*ws)).shape == (0, 256)
    assert mxfp4_status(DEV) == 0


def test_matmul_nan_scale_is_one_row():
    g = gen("mmnan")
    ac, asc = weight(g, 70, 512, std=1.0)
    w = MXFP4Weight(*weight(g, 264, 512))
    clean = mxfp4_matmul(ac, asc, w)
    asc[33, 7] = 255
    y = mxfp4_matmul(ac, asc, w)
    rest = torch.arange(70, device=DEV) != 33
    assert bool(torch.isnan(y[33]).all()) and torch.equal(y[rest], clean[rest])


def test_matmul_leading_dims_and_strides():
    g = gen("mmst")
    ac, asc = weight(g, 6, 4, 256, std=1.0)
    codes, scales = weight(g, 64, 256)
    w = MXFP4Weight(codes, scales)
    wd = O.dequantize(codes, scales)
    y = mxfp4_matmul(ac, asc, w)
    assert y.shape == (6, 4, 64)
    check_product(y.view(24, 64), O.dequantize(ac, asc).view(24, 256), wd)
    assert torch.equal(mxfp4_matmul(ac[:, 1], asc[:, 1], w), y[:, 1])
    assert torch.equal(mxfp4_matmul(ac.transpose(0, 1), asc.transpose(0, 1), w), y.transpose(0, 1))
    assert mxfp4_matmul(ac[:0], asc[:0], w).shape == (0, 4, 64)


def test_results_do_not_depend_on_the_sm_limit():
    from dsmoe._lib import set_gemm_sm_limit
    g = gen("lim")
    ws, _ = experts(g, 17, 256, 256)
    ex, lw = MXFP4Experts(*ws), MXFP4Weight(*weight(g, 512, 1024))
    x = torch.randn(200, 256, generator=g, device=DEV).to(torch.bfloat16)
    z = torch.randn(300, 1024, generator=g, device=DEV).to(torch.bfloat16)
    r = routing(g, 200, 16, 4)
    want = mxfp4_moe(x, *r, ex), mxfp4_linear(z, lw)
    try:
        for n in (1, 37, 100):
            set_gemm_sm_limit(n)
            assert torch.equal(mxfp4_moe(x, *r, ex), want[0]) and torch.equal(mxfp4_linear(z, lw), want[1])
    finally:
        set_gemm_sm_limit(0)


def test_two_threads_on_two_streams():
    import threading
    g = gen("thr")
    ws, _ = experts(g, 33, 256, 256)
    ex = MXFP4Experts(*ws)
    xs = [torch.randn(n, 256, generator=g, device=DEV).to(torch.bfloat16) for n in (5, 300)]
    rs = [routing(g, n, 32, 4) for n in (5, 300)]
    want = [mxfp4_moe(x, *r, ex) for x, r in zip(xs, rs)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                y = mxfp4_moe(xs[i], *rs[i], ex)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)

    t = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [a.start() for a in t]
    [a.join() for a in t]
    assert not bad and mxfp4_status(DEV) == 0


def test_first_call_inside_a_capture():
    """A fresh process whose first product runs inside a graph capture."""
    import subprocess
    import sys
    code = (
        "import sys, torch; sys.path.insert(0, 'deepseek-on-one-gpu_b200')\n"
        "from dsmoe import *\n"
        "w = MXFP4Weight(*mxfp4_quantize(torch.ones(256, 512, device='cuda')))\n"
        "e = [MXFP4Weight(*mxfp4_quantize(torch.full(s, 0.25, device='cuda'))) for s in ((5, 128, 512), (5, 128, 512), (5, 512, 128))]\n"
        "e = MXFP4Experts(*e)\n"
        "x = torch.ones(3, 512, dtype=torch.bfloat16, device='cuda')\n"
        "i, t = torch.zeros(3, 2, dtype=torch.int64, device='cuda'), torch.ones(3, 2, device='cuda')\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    y, z = mxfp4_linear(x, w), mxfp4_moe(x, i, t, e)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert bool((y == 512).all()) and torch.equal(z, mxfp4_moe(x, i, t, e)) and mxfp4_status('cuda') == 0\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("off", [[0, 900, 200, 1500], [-3, 10, 1499, 1900], [100, 700, 700, 1400]])
def test_grouped_many_rows_with_odd_offsets(off):
    """More rows than the one-kernel form of the segment tables takes: the same
    clamping, and rows outside every segment."""
    g = gen("bo2")
    codes, scales = weight(g, 3, 256, 256)
    x = torch.randn(1500, 256, generator=g, device=DEV).to(torch.bfloat16)
    w = MXFP4Weight(codes, scales)
    y = mxfp4_grouped_linear(x, w, torch.tensor(off, dtype=torch.int32, device=DEV))
    bad = off[0] < 0 or off[-1] > 1500 or any(a > b for a, b in zip(off, off[1:]))
    assert mxfp4_status(DEV) == (6 if bad else 0)
    clean = [min(max(o, 0), 1500) for o in off]
    for i in range(1, 4):
        clean[i] = max(clean[i], clean[i - 1])
    wd = O.dequantize(codes, scales)
    for e in range(3):
        if clean[e + 1] > clean[e]:
            check_product(y[clean[e]:clean[e + 1]], x[clean[e]:clean[e + 1]].double(), wd[e])
    assert bool((y[:clean[0]] == 0).all()) and bool((y[clean[3]:] == 0).all())
    # the one-kernel form on the first rows
    n = 1000
    part = torch.tensor([min(c, n) for c in clean], dtype=torch.int32, device=DEV)
    small = mxfp4_grouped_linear(x[:n], w, part)
    check_product(small[int(part[0]):int(part[1])], x[int(part[0]):int(part[1])].double(), wd[0])

"""MXFP4 operators at the ends of their number range, with copied weights and
with calls of different sizes at the same time. Everything here is exact: a
format conversion, a product of one non-zero term, or the same call twice."""
import copy
import pickle
import threading

import pytest
import torch

from dsmoe import (DeepSeekConfig, MXFP4Experts, MXFP4Weight, mxfp4_dequantize, mxfp4_grouped_linear, mxfp4_linear,
                   mxfp4_matmul, mxfp4_moe, mxfp4_quantize, mxfp4_status)
from dsmoe.mxfp4 import moe_forward
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def weight(g, *shape):
    return mxfp4_quantize(torch.randn(*shape, generator=g, device=DEV) * 0.02)


def experts(g, n, hidden, inter, shared=True):
    return MXFP4Experts(MXFP4Weight(*weight(g, n, inter, hidden)), MXFP4Weight(*weight(g, n, inter, hidden)),
                        MXFP4Weight(*weight(g, n, hidden, inter)), shared)


@pytest.mark.parametrize("s", [1e-45, 1e-40, 2.0 ** -126, 1e-30, 2.0 ** 63, 2.0 ** 64, 2.0 ** 100, 2.0 ** 112, 7e35,
                               2.0 ** 119, 2.0 ** 121, 1.7e38, 3.4028234663852886e38, 0.0, -1e38, -3e38, -1e-42,
                               float("inf"), float("-inf"), float("nan")])
def test_quantize_fp8_scales_over_all_of_fp32(s):
    g = gen(1)
    w = torch.randn(64, 128, generator=g, device=DEV)
    w[:16] *= 400.0
    w[16:32] *= 2.0 ** -8
    w[3, :32] = 0.0
    w[4, 5], w[5, 40] = 448.0, 2.0 ** -9
    q = w.clamp(-448, 448).to(torch.float8_e4m3fn)
    sc = torch.full((1, 1), s, device=DEV)
    codes, scales = mxfp4_quantize(q, sc)
    rc, rs = O.quantize(q.cpu(), sc.cpu())
    assert torch.equal(scales.cpu(), rs) and torch.equal(codes.cpu(), rc)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequantize_every_scale_and_code(dtype):
    codes = torch.arange(16, dtype=torch.uint8, device=DEV)
    codes = (codes | (codes << 4)).expand(256, 16).contiguous()
    scales = torch.arange(256, dtype=torch.int32, device=DEV).to(torch.uint8).view(256, 1)
    y = mxfp4_dequantize(codes, scales, dtype)
    ref = O.dequantize(codes, scales)
    want = ref.to(torch.float32).to(dtype)  # fp32 holds all but the infinite ones exactly
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    ok = ~torch.isnan(ref)
    assert torch.equal(y[ok], want[ok])


def test_zeros_under_large_scales_add_nothing():
    """Feature n's only non-zero weight is 0.5 * 2^127 at k = 0; x_0 = 2^-120.
    Elsewhere the weights are 0 with scale 2^127 and x is 2^120."""
    N, K = 128, 256
    codes = torch.zeros(N, K // 2, dtype=torch.uint8, device=DEV)
    codes[:, 0] = 1
    w = MXFP4Weight(codes, torch.full((N, K // 32), 254, dtype=torch.uint8, device=DEV))
    x = torch.zeros(3, K, device=DEV)
    x[:, 0], x[:, 32:] = 2.0 ** -120, 2.0 ** 120
    y = mxfp4_linear(x.to(torch.bfloat16), w)
    assert bool((y == 64.0).all())
    y = mxfp4_matmul(*mxfp4_quantize(x), w)
    assert bool((y == 64.0).all())


def test_copies_are_weights_of_their_own():
    g = gen(2)
    x = torch.randn(6, 256, generator=g, device=DEV).to(torch.bfloat16)
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device=DEV)
    idx = torch.randint(0, 4, (6, 2), generator=g, device=DEV)
    tw = torch.rand(6, 2, generator=g, device=DEV)
    w, st, ex = MXFP4Weight(*weight(g, 64, 256)), MXFP4Weight(*weight(g, 2, 64, 256)), experts(g, 5, 256, 128)

    def run(w, st, ex):
        return mxfp4_linear(x, w), mxfp4_grouped_linear(x, st, off), mxfp4_moe(x, idx, tw, ex)

    want = run(w, st, ex)
    copies = [[copy.deepcopy(v) for v in (w, st, ex)], [pickle.loads(pickle.dumps(v)) for v in (w, st, ex)]]
    for t in (w.codes, w.atoms, st.codes, st.atoms, ex.gate_codes, ex.up_codes, ex.gate_up_atoms, ex.down_codes,
              ex.down_atoms):
        t.zero_()
    for c in copies:
        for a, b in zip(run(*c), want):
            assert torch.equal(a, b)
    assert all(bool((a == 0).all()) for a in run(w, st, ex))


def test_weights_keep_their_tensors():
    """The library is handed addresses taken once: another tensor cannot be put in their place."""
    g = gen(3)
    w, ex = MXFP4Weight(*weight(g, 64, 256)), experts(g, 3, 128, 128)
    for v, names in ((w, ("codes", "atoms")),
                     (ex, ("gate_codes", "up_codes", "gate_up_atoms", "down_codes", "down_atoms"))):
        for n in names:
            with pytest.raises(AttributeError):
                setattr(v, n, getattr(v, n).clone())


def test_moe_forward_refuses_what_it_would_misread():
    cfg = DeepSeekConfig(hidden_size=256, moe_intermediate_size=128)
    E = cfg.n_routed_experts
    ex = MXFP4Experts._empty(E + 1, 256, 128, DEV)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)
    gate = torch.zeros(E, 256, dtype=torch.bfloat16, device=DEV)
    out, idx, tw = moe_forward(x, gate, None, cfg, ex)
    assert out.shape == x.shape and bool((out == 0).all())
    with pytest.raises(ValueError):
        moe_forward(torch.zeros(4, 512, dtype=torch.bfloat16, device=DEV)[:, ::2], gate, None, cfg, ex)
    with pytest.raises(ValueError):
        moe_forward(x.view(2, 2, 256), gate, None, cfg, ex)
    with pytest.raises(ValueError):
        moe_forward(x, gate[:-1], None, cfg, ex)
    with pytest.raises(ValueError):
        moe_forward(x, gate.t().contiguous().t(), None, cfg, ex)
    with pytest.raises(TypeError):
        moe_forward(x, gate.float(), None, cfg, ex)
    v3 = DeepSeekConfig(hidden_size=256, moe_intermediate_size=128, router_mode="v3")
    with pytest.raises(TypeError):
        moe_forward(x, gate, torch.zeros(E, dtype=torch.bfloat16, device=DEV), v3, ex)
    with pytest.raises(ValueError):
        moe_forward(x, gate, torch.zeros(E - 1, device=DEV), v3, ex)
    assert mxfp4_status(DEV) == 0


def test_threads_with_different_expert_counts():
    """The planner's shared memory follows the number of experts; two threads
    that launch it for 512 and for 400 do not disturb one another."""
    g = gen(4)
    sets = []
    for n in (512, 400):
        x = torch.randn(256, 128, generator=g, device=DEV).to(torch.bfloat16)
        idx = torch.randint(0, n, (256, 8), generator=g, device=DEV)
        sets.append((x, idx, torch.rand(256, 8, generator=g, device=DEV), experts(g, n, 128, 128, shared=False)))
    want = [mxfp4_moe(*s) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(400):
                    y = mxfp4_moe(*sets[i])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)
        except RuntimeError as e:
            bad.append(str(e))

    t = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [a.start() for a in t]
    [a.join() for a in t]
    assert not bad and mxfp4_status(DEV) == 0

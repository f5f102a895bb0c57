"""moe_block and moe_layer_ffn on MXFP4 experts (GPUTransfer(...,
expert_format="mxfp4")): the same routing as the FP8 block, the FFN of the
64-bit oracle on the experts quantised by the oracle from the store's FP8
weights, and the FP8 block left as it was."""
import math

import pytest
import torch

from dsmoe import DeepSeekConfig, GPUTransfer, SyntheticWeightStore, moe_block, moe_layer_ffn, mxfp4_status, rms_norm
from dsmoe.synthetic import PROJS, activations
from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
H, F, LAYER = 512, 256, 3


def setup(router="ref"):
    cfg = DeepSeekConfig(hidden_size=H, moe_intermediate_size=F, router_mode=router)
    store = SyntheticWeightStore(cfg, seed=21, device=DEV, pin_memory=False, gen_device="cuda")
    return cfg, store, GPUTransfer(cfg, store, DEV, expert_format="mxfp4")


def oracle_stacks(store, cfg):
    ex = [store.get_shared_expert_weights(LAYER)] + [store.device_expert(LAYER, e) for e in range(cfg.n_routed_experts)]
    return [torch.stack([O.dequantize(*O.quantize(*e[p])) for e in ex]) for p in PROJS]


@pytest.mark.parametrize("router", ["ref", "v3"])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_moe_block(T, router):
    cfg, store, gt = setup(router)
    x = activations(22, T, H).to(DEV)
    out, idx, w = moe_block(x.view(1, T, H), LAYER, store, gt, cfg, return_routing=True)
    assert out.shape == (1, T, H) and mxfp4_status(DEV) == 0
    fp8 = GPUTransfer(cfg, store, DEV)
    ref8, idx8, w8 = moe_block(x.view(1, T, H), LAYER, store, fp8, cfg, return_routing=True)
    assert torch.equal(idx, idx8) and torch.equal(w, w8)
    gate, up, down = oracle_stacks(store, cfg)
    scale = 1.0 if router == "v3" else cfg.routed_scaling_factor
    ref = O.moe(x, idx[0], w[0], gate, up, down, True, scale)
    # h is kept to 2^-9, each expert's row is rounded to bf16 (2^-8) and the sum
    # once more; the terms of the sum are within 3 times it in the mean square
    # (9 terms of random sign)
    err = float((out[0].double() - ref).norm() / ref.norm())
    assert err <= 3 * (2.0 ** -9 + 2 * 2.0 ** -8) / math.sqrt(3), err
    # 4-bit experts are another model than the FP8 ones, by no more than e2m1's
    # error on normal weights (a quarter of a number at most, three projections)
    diff = float((out.double() - ref8.double()).norm() / ref8.double().norm())
    assert 0.01 < diff < 0.75, diff
    assert torch.equal(ref8, moe_block(x.view(1, T, H), LAYER, store, fp8, cfg))


def test_layer_ffn_is_norm_block_residual():
    cfg, store, gt = setup()
    x = activations(23, 33, H).to(DEV)
    out = moe_layer_ffn(x.view(1, 33, H), LAYER, store, gt, cfg)
    normed = rms_norm(x, store.get_layer_norm_weights(LAYER)[1], cfg.rms_norm_eps)
    assert torch.equal(out[0], x + moe_block(normed, LAYER, store, gt, cfg))


def test_bank_bytes_and_refusals():
    cfg, store, gt = setup()
    bank = gt.bank(LAYER)
    assert bank.fully_resident
    assert bank.nbytes == 257 * 3 * H * F * 17 // 32
    assert gt.ensure_resident(LAYER, [1, 2]) is bank and gt.prefetch(LAYER, [4]) == 0
    with pytest.raises(TypeError):
        gt.transfer_experts(LAYER, torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        GPUTransfer(cfg, store, DEV, slots_per_layer=40, expert_format="mxfp4")
    with pytest.raises(ValueError):
        GPUTransfer(cfg, store, DEV, device_slots=True, expert_format="mxfp4")
    with pytest.raises(ValueError):
        GPUTransfer(cfg, store, DEV, expert_format="int4")
    with pytest.raises(ValueError):
        bank.write_slot(1, {p: (w[:, :128].contiguous(), s[:, :1].contiguous())
                            for p, (w, s) in store.device_expert(LAYER, 0).items()})


def test_captured_block():
    cfg, store, gt = setup()
    xs = [activations(24 + i, 16, H).to(DEV) for i in range(3)]
    want = [moe_block(x, LAYER, store, gt, cfg) for x in xs]
    buf = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = moe_block(buf, LAYER, store, gt, cfg)
    for x, y in zip(xs[1:] + xs[:1], want[1:] + want[:1]):
        buf.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)


def test_two_captured_blocks_at_once_and_a_larger_call_between():
    """Two graphs replayed on two streams share no scratch, and a larger call
    made after the captures takes none of theirs away."""
    cfg, store, gt = setup()
    xs = [activations(30 + i, 64, H).to(DEV) for i in range(2)]
    want = [moe_block(x, LAYER, store, gt, cfg) for x in xs]
    graphs = []
    for x in xs:
        buf, g = x.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = moe_block(buf, LAYER, store, gt, cfg)
        graphs.append((g, buf, out))
    moe_block(activations(40, 3000, H).to(DEV), LAYER, store, gt, cfg)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for _, _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        for (g, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, out), y in zip(graphs, want):
            assert torch.equal(out, y)
    assert mxfp4_status(DEV) == 0


def test_no_tokens():
    cfg, store, gt = setup()
    assert moe_block(torch.zeros(0, H, dtype=torch.bfloat16, device=DEV), LAYER, store, gt, cfg).shape == (0, H)


def test_quantise_one_layer_and_run_it_by_hand():
    """The operators one after the other, as a caller without moe_block uses
    them: checkpoint experts to MXFP4, route, the routed FFN; and the FFN out
    of ragged products, with the same result up to its roundings."""
    from dsmoe import (MXFP4Experts, MXFP4Weight, mxfp4_grouped_linear, mxfp4_linear, mxfp4_moe, route)
    cfg, store, gt = setup()
    x = activations(50, 90, H).to(DEV)
    ex = [store.get_shared_expert_weights(LAYER)] + [store.device_expert(LAYER, e) for e in range(256)]
    stacks = [MXFP4Weight.quantize(torch.stack([e[p][0] for e in ex]), torch.stack([e[p][1] for e in ex])) for p in PROJS]
    idx, w = route(x, store.get_gate_weight(LAYER), cfg)
    y = mxfp4_moe(x, idx, w, MXFP4Experts(*stacks), cfg.routed_scaling_factor)
    assert torch.equal(y, moe_block(x, LAYER, store, gt, cfg))
    # by ragged products: rows sorted by expert, silu and the sum in torch
    flat = idx.reshape(-1)
    order = torch.argsort(flat, stable=True)
    rows = x[order // 8]
    offsets = torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=256).cumsum(0)]).int()
    routed = [MXFP4Weight.quantize(torch.stack([e[p][0] for e in ex[1:]]), torch.stack([e[p][1] for e in ex[1:]]))
              for p in PROJS]
    g, u = (mxfp4_grouped_linear(rows, s, offsets).float() for s in routed[:2])
    out = mxfp4_grouped_linear((torch.nn.functional.silu(g) * u).bfloat16(), routed[2], offsets).float()
    acc = torch.zeros_like(x, dtype=torch.float32).index_add_(0, order // 8, out * w.reshape(-1)[order, None])
    one = [MXFP4Weight.quantize(*ex[0][p]) for p in PROJS]
    sh = mxfp4_linear((torch.nn.functional.silu(mxfp4_linear(x, one[0]).float()) *
                       mxfp4_linear(x, one[1]).float()).bfloat16(), one[2]).float()
    z = acc * cfg.routed_scaling_factor + sh
    # g, u, h and each row are rounded to bf16 (2^-8 each) where mxfp4_moe keeps
    # fp32 or 2^-9, both sides round their rows: 6 roundings of at most 2^-8
    # between them, and the terms of a sum are within 3 times it
    err = float((y.float() - z).norm() / z.norm())
    assert err <= 3 * 6 * 2.0 ** -8 / math.sqrt(3), err

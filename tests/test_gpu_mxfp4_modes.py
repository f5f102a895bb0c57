"""MXFP4 operators under torch's modes: inference mode, forward-mode
differentiation."""
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

from dsmoe import (DeepSeekConfig, GPUTransfer, MXFP4Experts, MXFP4Weight, SyntheticWeightStore, moe_block, moe_layer_ffn,
                   mxfp4_dequantize, mxfp4_grouped_linear, mxfp4_linear, mxfp4_matmul, mxfp4_moe, mxfp4_quantize)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def test_first_call_in_inference_mode():
    """A process whose first weights and bank are made in inference mode: the
    error word can be read and cleared, and the bank written, outside of it."""
    code = (
        "import sys, torch; sys.path.insert(0, 'deepseek-on-one-gpu_b200')\n"
        "from dsmoe import *\n"
        "cfg = DeepSeekConfig(hidden_size=256, moe_intermediate_size=128)\n"
        "store = SyntheticWeightStore(cfg, seed=1, device=torch.device('cuda', 0), pin_memory=False, gen_device='cuda')\n"
        "gt = GPUTransfer(cfg, store, 'cuda', expert_format='mxfp4')\n"
        "x = torch.ones(4, 256, dtype=torch.bfloat16, device='cuda')\n"
        "with torch.inference_mode():\n"
        "    w = MXFP4Weight(*mxfp4_quantize(torch.ones(1, 256, 256, device='cuda')))\n"
        "    mxfp4_grouped_linear(x, w, torch.tensor([0, 9], dtype=torch.int32, device='cuda'))\n"
        "    a = moe_block(x, 3, store, gt, cfg)\n"
        "assert mxfp4_status('cuda') == 6 and mxfp4_status('cuda') == 0\n"
        "bank = gt.bank(3)\n"
        "for e in range(257):\n"
        "    bank.write_slot(e, store.device_expert(3, 0))\n"
        "b = moe_block(x, 3, store, gt, cfg)\n"
        "for e in range(256):\n"
        "    bank.write_slot(e + 1, store.device_expert(3, e))\n"
        "bank.write_slot(0, store.get_shared_expert_weights(3))\n"
        "c = moe_block(x, 3, store, gt, cfg)\n"
        "assert torch.equal(a, c) and not torch.equal(a, b)\n")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stderr[-2000:]


def weight(*shape):
    g = torch.Generator(device=DEV)
    g.manual_seed(sum(shape))
    return mxfp4_quantize(torch.randn(*shape, generator=g, device=DEV))


def test_forward_mode_tangents_are_refused():
    """The operators have no derivative of either kind: a dual number is not
    answered with a result that has lost its tangent."""
    w, st = MXFP4Weight(*weight(64, 256)), MXFP4Weight(*weight(2, 64, 256))
    ex = MXFP4Experts(MXFP4Weight(*weight(3, 128, 256)), MXFP4Weight(*weight(3, 128, 256)),
                      MXFP4Weight(*weight(3, 256, 128)))
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=DEV)
    off = torch.tensor([0, 1, 4], dtype=torch.int32, device=DEV)
    idx, tw = torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.ones(4, 2, device=DEV)
    pair = mxfp4_quantize(x)

    def calls(x, tw):
        return [lambda: mxfp4_quantize(x), lambda: mxfp4_linear(x, w), lambda: mxfp4_grouped_linear(x, st, off),
                lambda: mxfp4_moe(x, idx, tw, ex)]

    want = [f() for f in calls(x, tw)]
    with forward_ad.dual_level():
        dual, dual_tw = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, tw))
        for f in calls(dual, tw) + calls(x, dual_tw)[3:]:
            with pytest.raises(RuntimeError, match="tangent"):
                f()
        for f, y in zip(calls(x, tw), want):  # numbers without a tangent are taken as ever
            got = f()
            assert all(torch.equal(a, b) for a, b in zip(got, y)) if isinstance(y, tuple) else torch.equal(got, y)
        mxfp4_matmul(*pair, w), mxfp4_dequantize(*pair)


def test_layer_ffn_has_no_derivative_either():
    """Not one through its residual alone."""
    cfg = DeepSeekConfig(hidden_size=256, moe_intermediate_size=128)
    store = SyntheticWeightStore(cfg, seed=2, device=DEV, pin_memory=False, gen_device="cuda")
    gt = GPUTransfer(cfg, store, DEV, expert_format="mxfp4")
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=DEV)
    want = moe_layer_ffn(x, 3, store, gt, cfg)
    for call in (moe_layer_ffn, moe_block):
        with pytest.raises(RuntimeError, match="backward"):
            call(x.clone().requires_grad_(), 3, store, gt, cfg)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
            call(forward_ad.make_dual(x, torch.ones_like(x)), 3, store, gt, cfg)
    with torch.no_grad():
        assert torch.equal(moe_layer_ffn(x.clone().requires_grad_(), 3, store, gt, cfg), want)

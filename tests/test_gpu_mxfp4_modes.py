"""MXFP4 operators under torch's modes."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


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

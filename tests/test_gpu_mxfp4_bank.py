"""A layer's bank whose filling failed (a shard that could not be read, say) is
filled again by the next call: no expert is taken for loaded that is not."""
import pytest
import torch

from dsmoe import DeepSeekConfig, GPUTransfer, SyntheticWeightStore, moe_block, moe_layer_ffn
from dsmoe.synthetic import activations

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
H, F, LAYER = 512, 256, 3


class FailsOnce:
    """A weight store that gives its experts one by one and fails at one of them, once."""

    def __init__(self, store, at):
        self.store, self.at = store, at

    def __getattr__(self, name):
        if name == "fill_bank":
            raise AttributeError(name)
        return getattr(self.store, name)

    def get_expert(self, layer, e):
        if e == self.at:
            self.at = None
            raise OSError("expert not readable")
        return self.store.device_expert(layer, e)


class FillFailsOnce(FailsOnce):
    """The same with ``fill_bank``."""

    def __getattr__(self, name):
        return getattr(self.store, name)

    def fill_bank(self, layer, bank):
        if self.at is not None:
            self.store.fill_bank(layer, bank, range(self.at))
            self.at = None
            raise OSError("expert not readable")
        self.store.fill_bank(layer, bank)


@pytest.mark.parametrize("fmt", ["mxfp4", "fp8"])
@pytest.mark.parametrize("kind", [FailsOnce, FillFailsOnce])
@pytest.mark.parametrize("call", [moe_block, moe_layer_ffn])
def test_a_bank_that_could_not_be_filled_is_filled_again(call, kind, fmt):
    cfg = DeepSeekConfig(hidden_size=H, moe_intermediate_size=F)
    store = SyntheticWeightStore(cfg, seed=31, device=DEV, pin_memory=False, gen_device="cuda")
    x = activations(32, 700, H).to(DEV)
    want = call(x, LAYER, store, GPUTransfer(cfg, store, DEV, expert_format=fmt), cfg)
    broken = kind(store, 100)
    gt = GPUTransfer(cfg, broken, DEV, expert_format=fmt)
    with pytest.raises(OSError):
        call(x, LAYER, broken, gt, cfg)
    assert torch.equal(call(x, LAYER, broken, gt, cfg), want)
    assert gt.bank(LAYER).fully_resident

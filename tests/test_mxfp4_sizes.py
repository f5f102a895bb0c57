"""Sizes that a 32-bit argument of the library does not hold: refused before
any call (2^32 + n would arrive as n). Without a GPU: the device check and the
copies are stood in for, and a library call fails the test."""
import pytest
import torch

from dsmoe import mxfp4

WRAP = 1 << 32


@pytest.fixture
def no_calls(monkeypatch):
    def call(*args):
        raise AssertionError("the library was called")

    monkeypatch.setattr(mxfp4, "_call", call)
    monkeypatch.setattr(mxfp4, "_require", lambda what, *tensors: None)
    monkeypatch.setattr(mxfp4, "_rows", lambda x: x)
    monkeypatch.setattr(mxfp4, "_dense", lambda t, align: t)
    monkeypatch.setattr(torch.Tensor, "contiguous", lambda t: t)
    monkeypatch.setattr(mxfp4, "_device_status", lambda device: torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("cols", [WRAP + 64, 1 << 31])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_refuses_rows_beyond_int32(no_calls, cols, dtype):
    with pytest.raises(ValueError, match="last dimension"):
        mxfp4.mxfp4_quantize(torch.zeros(1, 1, dtype=dtype).expand(1, cols))


def test_quantize_fp8_refuses_rows_beyond_int32(no_calls):
    x = torch.zeros(1, 1).to(torch.float8_e4m3fn).expand(1, WRAP + 64)
    with pytest.raises(ValueError, match="last dimension"):
        mxfp4.mxfp4_quantize(x, torch.ones(1, 1).expand(1, (WRAP + 64 + 127) // 128))


def test_weight_refuses_features_beyond_int32(no_calls):
    byte = torch.zeros(1, 1, dtype=torch.uint8)
    for out, k in ((8, WRAP + 128), (WRAP + 8, 128)):
        with pytest.raises(ValueError, match="features"):
            mxfp4.MXFP4Weight(byte.expand(out, k // 2), byte.expand(out, k // 32))


def test_weight_refuses_experts_beyond_int32(no_calls):
    byte = torch.zeros(1, 1, 1, dtype=torch.uint8)
    with pytest.raises(ValueError, match="expert"):
        mxfp4.MXFP4Weight(byte.expand(WRAP + 2, 8, 64), byte.expand(WRAP + 2, 8, 4))


def test_moe_refuses_top_k_beyond_int32(no_calls):
    ex = mxfp4.MXFP4Experts.__new__(mxfp4.MXFP4Experts)
    ex.hidden, ex.inter, ex.n_routed, ex.shared, ex.device = 256, 128, 4, True, torch.device("cpu")
    ex.desc, ex.status = None, torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    idx, w = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1)
    with pytest.raises(ValueError, match="top_k"):
        mxfp4.mxfp4_moe(x, idx.expand(2, WRAP + 1), w.expand(2, WRAP + 1), ex)

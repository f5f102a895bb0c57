"""MXFP4 operators without a GPU: the oracle against the format's own numbers,
and what the C ABI and the Python functions refuse (no CUDA call is reached)."""
import ctypes

import pytest
import torch

import dsmoe
from dsmoe import _lib
from oracle import mxfp4 as O

BIG = 1 << 40


def test_oracle_format():
    codes = torch.tensor([[0x10 * ((2 * i + 1) % 16) + (2 * i) % 16 for i in range(16)]], dtype=torch.uint8)
    v = O.dequantize(codes, torch.tensor([[127]], dtype=torch.uint8))
    grid = [0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6]
    assert v.tolist() == [grid + grid]
    assert float(O.dequantize(codes, torch.tensor([[130]], dtype=torch.uint8))[0, 7]) == 48.0
    assert float(O.dequantize(codes, torch.tensor([[0]], dtype=torch.uint8))[0, 2]) == 2.0 ** -127
    assert bool(torch.isnan(O.dequantize(codes, torch.tensor([[255]], dtype=torch.uint8))).all())


def test_oracle_rounding():
    x = torch.zeros(1, 32)
    x[0, :10] = torch.tensor([7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -5.01, 0.2501])
    codes, scales = O.quantize(x)
    assert scales.tolist() == [[127]]
    assert O.dequantize(codes, scales)[0, :10].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -6, 0.5]
    for scale in (-100, 3, 60):
        c2, s2 = O.quantize(x.double() * 2.0 ** scale)
        assert torch.equal(c2, codes) and s2.tolist() == [[127 + scale]]


def test_oracle_ragged_and_moe():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 32, generator=g)
    w = torch.randn(2, 8, 32, generator=g)
    y = O.grouped_linear(x, w, [0, 4, 5])
    assert torch.equal(y[:4], O.linear(x[:4], w[0])) and torch.equal(y[4], O.linear(x[4:5], w[1])[0])
    assert bool((y[5] == 0).all())
    gate, up, down = (torch.randn(3, 32, 32, generator=g) for _ in range(3))
    idx, wt = torch.tensor([[0, 1]] * 6), torch.full((6, 2), 0.5)
    m = O.moe(x, idx, wt, gate, up, down, True, 2.0)
    want = sum(O.ffn(x, gate[e], up[e], down[e]) for e in range(3))
    assert torch.allclose(m, want)


@pytest.mark.parametrize("args,code", [
    ((64, 9, 4, 64, 64, None, 0, 64, 64, None), -1),      # dtype
    ((64, 0, 4, 48, 48, None, 0, 64, 64, None), -4),      # cols % 32
    ((64, 0, -1, 64, 64, None, 0, 64, 64, None), -1),     # rows
    ((64, 0, 4, 64, 63, None, 0, 64, 64, None), -1),      # rows overlap
    ((64, 0, 4, 64, 68, None, 0, 64, 64, None), -1),      # rows off 16 bytes
    ((72, 0, 4, 64, 64, None, 0, 64, 64, None), -1),      # x off 16 bytes
    ((None, 0, 4, 64, 64, None, 0, 64, 64, None), -1),
    ((64, 0, 4, 64, 64, None, 0, None, 64, None), -1),
    ((64, 0, 4, 64, 64, None, 0, 64, None, None), -1),
    ((64, 0, 4, 64, 64, 64, 4, 64, 64, None), -1),        # scale_inv without e4m3
    ((64, 3, 4, 64, 64, None, 4, 64, 64, None), -1),      # e4m3 without scale_inv
    ((64, 3, 4, 64, 64, 64, 3, 64, 64, None), -1),        # rows_per_matrix
    ((64, 0, BIG, 64, 64, None, 0, 64, 64, None), -4),
    ((64, 0, 0, 64, 64, None, 0, 64, 64, None), 0),
])
def test_quantize_rejects(args, code):
    L = _lib.lib()
    assert L.dsmoe_mxfp4_quantize(*args) == code
    assert code == 0 or b"mxfp4_quantize" in L.dsmoe_last_error()


def test_dequantize_and_atoms_reject():
    L = _lib.lib()
    assert L.dsmoe_mxfp4_dequantize(64, 64, 4, 3, 64, None) == -1
    assert L.dsmoe_mxfp4_dequantize(66, 64, 4, 0, 64, None) == -1
    assert L.dsmoe_mxfp4_dequantize(64, 64, 4, 0, 72, None) == -1
    assert L.dsmoe_mxfp4_dequantize(64, 64, -1, 0, 64, None) == -1
    assert L.dsmoe_mxfp4_dequantize(None, None, 0, 0, None, None) == 0
    assert L.dsmoe_mxfp4_scale_atoms_bytes(2, 576, 256) == 2 * 3 * 2 * 1024
    assert L.dsmoe_mxfp4_scale_atoms_bytes(0, 576, 256) == 0
    assert L.dsmoe_mxfp4_scale_atoms_bytes(2, 576, 192) == 0
    assert L.dsmoe_mxfp4_scale_atoms_bytes(2, 12, 256) == 0
    assert L.dsmoe_mxfp4_scale_atoms(64, 0, 576, 256, 64, None) == -1
    assert L.dsmoe_mxfp4_scale_atoms(64, 1, 576, 256, 72, None) == -1
    assert L.dsmoe_mxfp4_scale_atoms(62, 1, 576, 256, 64, None) == -1


def linear(L, **kw):
    a = dict(x=256, stride=512, t=4, k=512, n=256, codes=256, atoms=256, out=256, ws=256, bytes=BIG, st=256)
    a.update(kw)
    return L.dsmoe_mxfp4_linear(a["x"], a["stride"], a["t"], a["k"], a["n"], a["codes"], a["atoms"], a["out"], a["ws"],
                                a["bytes"], a["st"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(k=500), -4), (dict(k=0), -4), (dict(k=32896), -4), (dict(n=12), -4), (dict(n=0), -4), (dict(t=-1), -1),
    (dict(t=1 << 23), -4), (dict(codes=272), -1), (dict(codes=None), -1), (dict(atoms=None), -1), (dict(x=264), -1),
    (dict(out=264), -1), (dict(st=None), -1), (dict(stride=511), -1), (dict(stride=516), -1), (dict(ws=None), -1),
    (dict(ws=272), -1), (dict(bytes=100), -3), (dict(t=0, x=None, out=None), 0),
])
def test_linear_rejects(kw, code):
    L = _lib.lib()
    assert linear(L, **kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(k=500), -4), (dict(n=12), -4), (dict(t=-1), -1), (dict(xc=264), -1), (dict(xs=258), -1), (dict(codes=272), -1),
    (dict(out=None), -1), (dict(st=258), -1), (dict(ws=272), -1), (dict(bytes=100), -3), (dict(t=0), 0),
])
def test_matmul_rejects(kw, code):
    a = dict(xc=256, xs=256, t=4, k=512, n=256, codes=256, atoms=256, out=256, ws=256, bytes=BIG, st=256)
    a.update(kw)
    assert _lib.lib().dsmoe_mxfp4_matmul(a["xc"], a["xs"], a["t"], a["k"], a["n"], a["codes"], a["atoms"], a["out"],
                                         a["ws"], a["bytes"], a["st"], None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(e=0), -4), (dict(e=513), -4), (dict(k=500), -4), (dict(n=12), -4), (dict(r=-1), -1), (dict(off=None), -1),
    (dict(off=258), -1), (dict(x=None), -1), (dict(stride=500), -1), (dict(out=264), -1), (dict(st=None), -1),
    (dict(ws=None), -1), (dict(bytes=100), -3), (dict(r=0), 0),
])
def test_grouped_rejects(kw, code):
    a = dict(x=256, stride=512, r=4, k=512, n=256, e=3, off=256, codes=256, atoms=256, out=256, ws=256, bytes=BIG, st=256)
    a.update(kw)
    assert _lib.lib().dsmoe_mxfp4_grouped_linear(a["x"], a["stride"], a["r"], a["k"], a["n"], a["e"], a["off"],
                                                 a["codes"], a["atoms"], a["out"], 1, a["ws"], a["bytes"], a["st"],
                                                 None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(h=500), -4), (dict(h=132), -4), (dict(f=500), -4), (dict(f=0), -4), (dict(e=0), -4), (dict(e=512), -4),
    (dict(shared=2), -1), (dict(k=0), -4), (dict(k=9), -4), (dict(scale=float("inf")), -1), (dict(t=-1), -1),
    (dict(gate=272), -1), (dict(down=None), -1), (dict(idx=260), -1), (dict(w=None), -1), (dict(x=264), -1),
    (dict(out=None), -1), (dict(stride=516), -1), (dict(ws=272), -1), (dict(bytes=100), -3), (dict(t=0), 0),
])
def test_moe_rejects(kw, code):
    a = dict(x=256, stride=512, t=4, h=512, f=256, e=8, shared=1, gate=256, down=256, idx=256, w=256, k=2, scale=1.0,
             out=256, ws=256, bytes=BIG, st=256)
    a.update(kw)
    L = _lib.lib()
    d = _lib.MXFP4ExpertsDesc(hidden=a["h"], inter=a["f"], n_routed=a["e"], shared=a["shared"], gate_codes=a["gate"],
                              up_codes=256, gate_up_atoms=256, down_codes=a["down"], down_atoms=256)
    assert L.dsmoe_mxfp4_moe(a["x"], a["stride"], a["t"], ctypes.byref(d), a["idx"], a["w"], a["k"], a["scale"],
                             a["out"], a["ws"], a["bytes"], a["st"], None) == code
    assert L.dsmoe_mxfp4_moe(256, 512, 4, None, 256, 256, 2, 1.0, 256, 256, BIG, 256, None) == -1


def test_moe_forward_rejects():
    L = _lib.lib()

    def call(cfg=None, d=None, gate=256, bias=None, x=256, t=4, out=256, idx=256, w=256, ws=256, nbytes=BIG, st=256):
        c = _lib.MoeConfig(**{**dict(hidden=512, inter=256, n_routed=64, n_group=2, topk_group=1, top_k=4, router_mode=0,
                                     norm_topk_prob=1, routed_scaling_factor=2.5), **(cfg or {})})
        e = _lib.MXFP4ExpertsDesc(**{**dict(hidden=512, inter=256, n_routed=64, shared=1, gate_codes=256, up_codes=256,
                                            gate_up_atoms=256, down_codes=256, down_atoms=256), **(d or {})})
        return L.dsmoe_mxfp4_moe_forward(c, gate, bias, ctypes.byref(e), x, t, out, idx, w, ws, nbytes, st, None)

    assert call(t=-1) == -1 and call(t=0) == 0
    assert call(d=dict(shared=0)) == -1 and call(d=dict(n_routed=32)) == -1 and call(d=dict(hidden=256)) == -1
    assert call(cfg=dict(topk_group=3)) == -4
    assert call(idx=None) == -1 and call(w=None) == -1 and call(st=None) == -1
    assert call(ws=272) == -1 and call(nbytes=1000) == -3
    assert call(gate=None) == -1 and call(x=264) == -1
    assert call(cfg=dict(router_mode=1)) == -1  # the bias-corrected router needs the bias
    assert L.dsmoe_mxfp4_moe_forward(None, 256, None, None, 256, 4, 256, 256, 256, 256, BIG, 256, None) == -1


def test_workspace_sizes():
    L = _lib.lib()
    assert L.dsmoe_mxfp4_linear_workspace_size(4096, 7168, 2048) >= 2 * 4096 * 7168
    assert L.dsmoe_mxfp4_linear_workspace_size(0, 7168, 2048) == 0
    assert L.dsmoe_mxfp4_linear_workspace_size(4, 7100, 2048) == 0
    assert L.dsmoe_mxfp4_matmul_workspace_size(4096, 7168, 2048) >= 4096 * 7168 // 32
    assert L.dsmoe_mxfp4_grouped_linear_workspace_size(100, 7168, 2048, 513) == 0
    assert L.dsmoe_mxfp4_grouped_linear_workspace_size(100, 7168, 2048, 64) >= 200 * 7168
    assert L.dsmoe_mxfp4_moe_workspace_size(64, 7168, 2048, 256, 1, 8) >= 64 * 9 * 2 * (7168 + 2048 + 7168)
    assert L.dsmoe_mxfp4_moe_workspace_size(64, 7168, 2048, 512, 1, 8) == 0


def test_python_refuses_cpu_tensors_and_wrong_types():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    c, s = torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(8, 8, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        dsmoe.mxfp4_quantize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        dsmoe.mxfp4_dequantize(c, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        dsmoe.MXFP4Weight(c, s)
    with pytest.raises(TypeError):
        dsmoe.mxfp4_linear(x, c)
    with pytest.raises(TypeError):
        dsmoe.mxfp4_matmul(c, s, c)
    with pytest.raises(TypeError):
        dsmoe.mxfp4_grouped_linear(x, c, c)
    with pytest.raises(TypeError):
        dsmoe.mxfp4_moe(x, c, s, None)
    with pytest.raises(TypeError):
        dsmoe.MXFP4Experts(c, c, c)

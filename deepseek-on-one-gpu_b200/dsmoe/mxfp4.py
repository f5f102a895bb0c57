"""MXFP4 experts and projections: 4-bit weights with a power-of-two scale per
32 numbers (the OCP microscaling format), 17/32 of the FP8 checkpoint's bytes.

The reference knows FP8 weights only (``inference/ops.py:15-44``); these
operators stand beside ``fp8_linear``, ``expert_ffn`` and ``moe_block`` for
users who halve the expert memory and the bytes a decode step reads:

  * ``mxfp4_quantize`` / ``mxfp4_dequantize``  tensors to and from MXFP4, also
    straight from the checkpoint's ``(weight, weight_scale_inv)``;
  * ``MXFP4Weight``            a weight (or a stack of experts) laid out for
    the products, once;
  * ``mxfp4_linear``           bf16 activations times an MXFP4 weight;
  * ``mxfp4_matmul``           MXFP4 activations times an MXFP4 weight;
  * ``mxfp4_grouped_linear``   rows sorted by expert times each expert's weight;
  * ``MXFP4Experts`` / ``mxfp4_moe``  the routed FFN after ``route``;
  * ``MXFP4LayerBank``         a layer's experts, filled from FP8 weights.

``GPUTransfer(..., expert_format="mxfp4")`` makes ``moe_block`` and
``moe_layer_ffn`` run on 4-bit experts. Every call goes through
``libdsmoe.so`` on the current stream of the tensors' device, with scratch
from torch's allocator (private to the call, also in a captured graph). There
is no CPU path and no derivative: tensors that require a gradient or carry a
forward-mode tangent are rejected.
"""
from __future__ import annotations

import ctypes
import threading

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib, ptr

BLOCK = 32
_INT_MAX = 2 ** 31 - 1  # of the library's sizes: ctypes hands on the lower 32 bits of a larger one
_IDLE = 256  # bytes of the workspace of calls that use none
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, torch.float8_e4m3fn: 3}
_status: dict[int, torch.Tensor] = {}
_status_lock = threading.Lock()


def _device_status(device: torch.device) -> torch.Tensor:
    """The device error word of this module's kernels (int32, first error wins)."""
    t = _status.get(device.index)
    if t is None:
        with _status_lock:
            t = _status.get(device.index)
            if t is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first MXFP4 call on a device must come before a graph capture")
                with torch.inference_mode(False):  # cleared later, also outside the mode of the first call
                    t = torch.zeros(1, dtype=torch.int32, device=device)
                torch.cuda.current_stream(device).synchronize()
                _status[device.index] = t
    return t


def mxfp4_status(device) -> int:
    """Read (synchronously) and clear the device error code of the MXFP4
    kernels: 0, or the first error since the last read (6: offsets of
    ``mxfp4_grouped_linear`` that decrease or leave the rows)."""
    t = _device_status(_index(torch.device(device)))
    torch.cuda.synchronize(t.device)
    code = int(t.item())
    if code:
        t.zero_()
    return code


def _index(device: torch.device) -> torch.device:
    return device if device.index is not None else torch.device("cuda", torch.cuda.current_device())


def stream_handle(device: torch.device) -> int:
    """The device's current stream, without building a Stream object."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _call(device: torch.device, name: str, *args) -> None:
    """One library call on ``device``'s current stream (the last argument),
    with the device current."""
    fn = getattr(lib(), name)
    if torch._C._cuda_getDevice() == device.index:
        rc = fn(*args, stream_handle(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream_handle(device))
    if rc:
        check(rc, name)


def _require(what: str, *tensors: torch.Tensor) -> None:
    dev, grad = None, torch.is_grad_enabled()
    dual = forward_ad._current_level >= 0  # inside a forward-mode level
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what} expects tensors")
        if not t.is_cuda:
            raise RuntimeError("dsmoe runs on CUDA tensors only (no CPU fallback)")
        if grad and t.requires_grad:
            raise RuntimeError(f"{what} has no backward: detach the inputs or call it under torch.no_grad()")
        if dual and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no derivative: a tangent would be lost")
        d = t.device
        if dev is None:
            dev = d
        elif d != dev:
            raise RuntimeError(f"{what}: tensors on different devices ({dev}, {d})")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as (rows, K) with unit column stride, rows that do not overlap
    and start on 16 bytes; a copy only where the strides need one."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    rows, K = x.shape
    step, unit = x.stride()
    if (unit != 1 and K > 1) or x.data_ptr() % 16 or (rows > 1 and (step < K or step * x.element_size() % 16)):
        return x.clone(memory_format=torch.contiguous_format)
    return x


def _dense(t: torch.Tensor, align: int) -> torch.Tensor:
    if not t.is_contiguous():
        t = t.contiguous()
    return t.clone() if t.data_ptr() % align else t


def _scratch(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def _quantize_into(x: torch.Tensor, scale_inv: torch.Tensor | None, codes: torch.Tensor, scales: torch.Tensor) -> None:
    K = x.shape[-1]
    fp8 = x.dtype == torch.float8_e4m3fn
    x2 = _rows(x)
    per = x.shape[-2] if fp8 else 1
    _call(x.device, "dsmoe_mxfp4_quantize", x2.data_ptr(), _DTYPES[x.dtype], x2.shape[0], K, x2.stride(0),
          ptr(scale_inv), max(per, 1), codes.data_ptr(), scales.data_ptr())


def mxfp4_quantize(x: torch.Tensor, scale_inv: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``x`` [..., K] (K a multiple of 32) -> codes uint8 [..., K/2] and scales
    uint8 [..., K/32]. Per block of 32 numbers with largest magnitude a:
    scale 2^(floor(log2 a) - 2), from 2^-127 to 2^127, codes rounded to nearest
    even, saturating at 6; a block with an infinity or a NaN becomes NaN.

    ``x`` is bf16, fp16 or fp32, or e4m3 [..., O, I] with the checkpoint's
    ``scale_inv`` fp32 [..., ceil(O/128), ceil(I/128)] (the products are
    rounded as exact numbers)."""
    _require("mxfp4_quantize", x, scale_inv)
    if x.dtype not in _DTYPES:
        raise TypeError("mxfp4_quantize expects bf16, fp16, fp32 or e4m3")
    *lead, K = x.shape or (0,)
    if K == 0 or K % BLOCK or K > _INT_MAX:
        raise ValueError(f"the last dimension must be a multiple of {BLOCK} below 2^31")
    if x.dtype == torch.float8_e4m3fn:
        if scale_inv is None or scale_inv.dtype != torch.float32:
            raise TypeError("e4m3 needs fp32 scale_inv")
        if x.dim() < 2:
            raise ValueError("e4m3 weights are (..., out, in)")
        want = (*x.shape[:-2], -(-x.shape[-2] // 128), -(-K // 128))
        if tuple(scale_inv.shape) != want:
            raise ValueError(f"scale_inv must be {want}, is {tuple(scale_inv.shape)}")
        scale_inv = scale_inv.contiguous()
    elif scale_inv is not None:
        raise TypeError("scale_inv goes with e4m3 only")
    codes = torch.empty(*lead, K // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(*lead, K // BLOCK, dtype=torch.uint8, device=x.device)
    if x.numel():
        _quantize_into(x, scale_inv, codes, scales)
    return codes, scales


def _check_pair(what: str, codes: torch.Tensor, scales: torch.Tensor) -> int:
    _require(what, codes, scales)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"{what} expects uint8 codes and scales")
    c, s = codes.shape, scales.shape
    if len(c) < 1 or c[:-1] != s[:-1] or len(c) != len(s) or c[-1] != 16 * s[-1]:
        raise ValueError(f"{what}: codes [..., K/2] {tuple(c)} do not go with scales [..., K/32] {tuple(s)}")
    return 2 * c[-1]


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The numbers MXFP4 data stands for, in bf16 or fp32 (exact) or fp16
    (rounded); beyond the type's range infinite."""
    K = _check_pair("mxfp4_dequantize", codes, scales)
    if out_dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError("mxfp4_dequantize produces bf16, fp16 or fp32")
    codes, scales = _dense(codes, 4), scales.contiguous()
    out = torch.empty(*codes.shape[:-1], K, dtype=out_dtype, device=codes.device)
    if out.numel():
        _call(codes.device, "dsmoe_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), scales.numel(),
              _DTYPES[out_dtype], out.data_ptr())
    return out


def _pack_scales(scales: torch.Tensor, mats: int, out_features: int, in_features: int, atoms: torch.Tensor) -> None:
    _call(scales.device, "dsmoe_mxfp4_scale_atoms", scales.data_ptr(), mats, out_features, in_features,
          atoms.data_ptr())


def _interleave(gate: torch.Tensor, up: torch.Tensor, mats: int, out_features: int, in_features: int) -> torch.Tensor:
    """Scale atoms of gate and up [mats, pairs, K/128, 2, 512] -> [mats, out/128, K/128, (gate, up), 512]."""
    tiles, kb = out_features // 128, in_features // 128

    def by_tile(a):
        return a.view(mats, -1, kb, 2, 512).transpose(2, 3).reshape(mats, -1, kb, 512)[:, :tiles]

    return torch.stack([by_tile(gate), by_tile(up)], dim=3)


class MXFP4Weight:
    """An MXFP4 weight ``[out, in]`` or a stack of experts ``[E, out, in]``,
    held for the products: the codes as they are (not copied when dense and
    32-byte aligned) and the scales in the tensor core's layout. in features
    a multiple of 128, out features of 8."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        K = _check_pair("MXFP4Weight", codes, scales)
        if codes.dim() not in (2, 3):
            raise ValueError("a weight is (out, in/2) or (experts, out, in/2)")
        self.in_features, self.out_features = K, codes.shape[-2]
        self.experts = codes.shape[0] if codes.dim() == 3 else None
        mats = 1 if self.experts is None else self.experts
        nbytes = 0
        if max(mats, self.out_features, K) <= _INT_MAX:
            nbytes = lib().dsmoe_mxfp4_scale_atoms_bytes(mats, self.out_features, K)
        if nbytes == 0:
            raise ValueError("MXFP4Weight: in features must be a multiple of 128 up to 32768, out features a multiple "
                             "of 8 up to 2^18, with at least one expert")
        self._codes = _dense(codes, 32)
        self._atoms = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
        self._bind()
        _pack_scales(_dense(scales, 4), mats, self.out_features, K, self._atoms)

    def _bind(self) -> None:
        """What follows from where the tensors are."""
        self.device = self._codes.device
        self.status = _device_status(self.device)
        self._ptrs = self._codes.data_ptr(), self._atoms.data_ptr(), self.status.data_ptr()
        self._need: dict[tuple, int] = {}  # scratch bytes by call form and rows
        self._idle = self._codes.new_empty(_IDLE)

    # The tensors cannot be replaced: calls use the addresses in _ptrs. A copy or
    # an unpickled weight finds its own.
    codes = property(lambda self: self._codes)
    atoms = property(lambda self: self._atoms)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("device", "status", "_ptrs", "_need", "_idle")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    @classmethod
    def quantize(cls, weight: torch.Tensor, scale_inv: torch.Tensor | None = None) -> "MXFP4Weight":
        """From a bf16, fp16 or fp32 weight, or the checkpoint's e4m3 weight
        with its ``weight_scale_inv``."""
        return cls(*mxfp4_quantize(weight, scale_inv))

    def _scratch(self, form: str, rows: int) -> torch.Tensor:
        need = self._need.get((form, rows))
        if need is None:
            sizes = (rows, self.in_features, self.out_features) + (() if self.experts is None else (self.experts,))
            with torch.cuda.device(self.device):
                need = getattr(lib(), form + "_workspace_size")(*sizes)
            if len(self._need) >= 1024:
                self._need.clear()
            self._need[form, rows] = need
        return self._idle if need <= _IDLE else self._codes.new_empty(need)

    @property
    def nbytes(self) -> int:
        return self._codes.numel() + self._atoms.numel()


def _check_weight(what: str, w: MXFP4Weight, stacked: bool) -> None:
    if not isinstance(w, MXFP4Weight):
        raise TypeError(f"{what} expects an MXFP4Weight")
    if (w.experts is not None) != stacked:
        raise ValueError(f"{what} expects " + ("a stack of experts" if stacked else "a single weight (out, in)"))


def _check_x(what: str, x: torch.Tensor, K: int, device: torch.device, *others: torch.Tensor) -> None:
    _require(what, x, *others)
    if x.device != device:
        raise RuntimeError(f"{what}: activations on {x.device}, weights on {device}")
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{what} expects bf16 activations")
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"{what}: activations end in {x.shape[-1] if x.dim() else 'no'} features, the weight has {K}")


def mxfp4_linear(x: torch.Tensor, weight: MXFP4Weight) -> torch.Tensor:
    """``bf16(x @ W.T)`` for bf16 ``x`` [..., in], fp32 sums. Numbers of ``x``
    below 2^-9 of the largest of their block of 32 are taken with an error of at
    most 2^-17 of it, all others exactly. A row with an infinity or a NaN comes
    out as NaN."""
    _check_weight("mxfp4_linear", weight, False)
    K, N = weight.in_features, weight.out_features
    _check_x("mxfp4_linear", x, K, weight.device)
    x2 = _rows(x)
    T = x2.shape[0]
    out = torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device)
    if T:
        codes, atoms, status = weight._ptrs
        ws = weight._scratch("dsmoe_mxfp4_linear", T)
        _call(weight.device, "dsmoe_mxfp4_linear", x2.data_ptr(), x2.stride(0), T, K, N, codes, atoms, out.data_ptr(),
              ws.data_ptr(), ws.numel(), status)
    return out


def mxfp4_matmul(codes: torch.Tensor, scales: torch.Tensor, weight: MXFP4Weight) -> torch.Tensor:
    """``bf16(x @ W.T)`` for MXFP4 activations (``mxfp4_quantize``'s codes
    [..., in/2] and scales [..., in/32]), fp32 sums."""
    _check_weight("mxfp4_matmul", weight, False)
    K = _check_pair("mxfp4_matmul", codes, scales)
    if codes.device != weight.device:
        raise RuntimeError(f"mxfp4_matmul: activations on {codes.device}, weights on {weight.device}")
    if K != weight.in_features:
        raise ValueError(f"mxfp4_matmul: activations have {K} features, the weight {weight.in_features}")
    shape, N = codes.shape[:-1], weight.out_features
    c2, s2 = _dense(codes, 16), _dense(scales, 4)
    T = c2.numel() // c2.shape[-1]
    out = torch.empty(*shape, N, dtype=torch.bfloat16, device=codes.device)
    if T:
        wc, wa, status = weight._ptrs
        ws = weight._scratch("dsmoe_mxfp4_matmul", T)
        _call(weight.device, "dsmoe_mxfp4_matmul", c2.data_ptr(), s2.data_ptr(), T, K, N, wc, wa, out.data_ptr(),
              ws.data_ptr(), ws.numel(), status)
    return out


def mxfp4_grouped_linear(x: torch.Tensor, weight: MXFP4Weight, offsets: torch.Tensor,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows sorted by expert: rows ``offsets[e] .. offsets[e + 1]`` of ``x``
    [R, in] (bf16) times expert e's weight -> bf16 [R, out]. ``offsets`` is
    int32 [E + 1] on the device, never read by the host. Rows outside every
    segment are zero in a new output and left as they are in ``out`` (dense
    bf16 [R, out], which must not overlap ``x``). Small numbers of a row and
    infinities and NaN are as in ``mxfp4_linear``."""
    _check_weight("mxfp4_grouped_linear", weight, True)
    _check_x("mxfp4_grouped_linear", x, weight.in_features, weight.device, offsets, out)
    if x.dim() != 2:
        raise ValueError("mxfp4_grouped_linear expects (rows, in) activations")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() != weight.experts + 1:
        raise ValueError(f"offsets must be int32 with {weight.experts + 1} entries")
    R, K, N = x.shape[0], weight.in_features, weight.out_features
    clear = out is None
    if clear:
        out = torch.empty(R, N, dtype=torch.bfloat16, device=x.device)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (R, N) or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be a dense, 16-byte aligned bf16 tensor ({R}, {N})")
    if R:
        x2, off = _rows(x), offsets.contiguous()
        codes, atoms, status = weight._ptrs
        ws = weight._scratch("dsmoe_mxfp4_grouped_linear", R)
        _call(weight.device, "dsmoe_mxfp4_grouped_linear", x2.data_ptr(), x2.stride(0), R, K, N, weight.experts,
              off.data_ptr(), codes, atoms, out.data_ptr(), int(clear), ws.data_ptr() or None, ws.numel(), status)
    return out


class MXFP4Experts:
    """The expert weights of one MoE layer: stacks ``gate`` and ``up``
    [G, inter, hidden] and ``down`` [G, hidden, inter]; with ``shared`` matrix
    0 is the shared expert and 1 + e routed expert e."""

    def __init__(self, gate: MXFP4Weight, up: MXFP4Weight, down: MXFP4Weight, shared: bool = True):
        for w in (gate, up, down):
            _check_weight("MXFP4Experts", w, True)
        self.hidden, self.inter = gate.in_features, gate.out_features
        if (up.in_features, up.out_features) != (self.hidden, self.inter) or \
                (down.in_features, down.out_features) != (self.inter, self.hidden) or \
                not gate.experts == up.experts == down.experts:
            raise ValueError("MXFP4Experts: gate and up are (G, inter, hidden), down is (G, hidden, inter)")
        if not gate.device == up.device == down.device:
            raise RuntimeError("MXFP4Experts: weights on different devices")
        if self.hidden % 128 or self.inter % 128:
            raise ValueError("MXFP4Experts: hidden and inter must be multiples of 128")
        self._set_up(gate.codes, up.codes, down.codes, _interleave(gate.atoms, up.atoms, gate.experts, self.inter,
                                                                   self.hidden), down.atoms, shared)

    def _set_up(self, gate, up, down, gate_up_atoms, down_atoms, shared: bool) -> None:
        self.shared = bool(shared)
        self.n_routed = gate.shape[0] - int(self.shared)
        if self.n_routed < 1:
            raise ValueError("MXFP4Experts: no routed expert")
        self._tensors = gate, up, down, gate_up_atoms, down_atoms
        self._bind()

    def _bind(self) -> None:
        gate, up, down, gate_up_atoms, down_atoms = self._tensors
        self.device = gate.device
        self.status = _device_status(self.device)
        self.desc = _lib.MXFP4ExpertsDesc(
            hidden=self.hidden, inter=self.inter, n_routed=self.n_routed, shared=int(self.shared),
            gate_codes=ptr(gate), up_codes=ptr(up), gate_up_atoms=ptr(gate_up_atoms), down_codes=ptr(down),
            down_atoms=ptr(down_atoms))

    # As with MXFP4Weight: not replaced, and a copy describes its own tensors.
    gate_codes = property(lambda self: self._tensors[0])
    up_codes = property(lambda self: self._tensors[1])
    down_codes = property(lambda self: self._tensors[2])
    gate_up_atoms = property(lambda self: self._tensors[3])
    down_atoms = property(lambda self: self._tensors[4])

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("device", "status", "desc")}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()

    @classmethod
    def _empty(cls, experts: int, hidden: int, inter: int, device: torch.device) -> "MXFP4Experts":
        """Room for ``experts`` matrices (the shared expert first), to be
        written one by one (``_write``)."""
        self = cls.__new__(cls)
        self.hidden, self.inter = hidden, inter

        def room(*shape):
            return torch.zeros(*shape, dtype=torch.uint8, device=device)

        with torch.inference_mode(False):  # _write may come outside the caller's mode
            self._set_up(room(experts, inter, hidden // 2), room(experts, inter, hidden // 2),
                         room(experts, hidden, inter // 2), room(experts, inter // 128, hidden // 128, 2, 512),
                         room(experts, -(-hidden // 256), inter // 128, 2, 512), True)
        return self

    def _write(self, slot: int, gate, up, down) -> None:
        """Quantise one expert's FP8 ``(weight, scale_inv)`` pairs into ``slot``."""
        packed = []
        for (w, s), codes in ((gate, self.gate_codes), (up, self.up_codes), (down, self.down_codes)):
            N, K = codes.shape[1], 2 * codes.shape[2]
            if tuple(w.shape) != (N, K) or w.dtype != torch.float8_e4m3fn:
                raise ValueError(f"expert weight is {w.dtype} {tuple(w.shape)}, the bank holds e4m3 {(N, K)}")
            if tuple(s.shape) != (-(-N // 128), K // 128):
                raise ValueError("scale_inv does not go with the weight")
            scales = torch.empty(N, K // BLOCK, dtype=torch.uint8, device=self.device)
            _quantize_into(w, s, codes[slot], scales)
            atoms = torch.empty(-(-N // 256), K // 128, 2, 512, dtype=torch.uint8, device=self.device)
            _pack_scales(scales, 1, N, K, atoms)
            packed.append(atoms)
        self.gate_up_atoms[slot].copy_(_interleave(packed[0], packed[1], 1, self.inter, self.hidden)[0])
        self.down_atoms[slot].copy_(packed[2])

    @property
    def nbytes(self) -> int:
        return sum(t.numel() for t in self._tensors)


def mxfp4_moe(hidden: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor, experts: MXFP4Experts,
              scale: float = 1.0) -> torch.Tensor:
    """The routed FFN of a MoE layer on ``route``'s result (``topk_idx`` int64
    and ``topk_w`` fp32, [..., top_k], top_k <= 8):
    ``bf16(scale * sum_k w_k E_k(hidden) + E_shared(hidden))``,
    ``E(x) = down(silu(gate(x)) * up(x))``, for bf16 ``hidden`` [..., hidden].
    silu, its product with up and the sum over experts are fp32; in between, the
    down projection takes that product to 8 or 9 significant bits (two e4m3 terms,
    as ``mxfp4_linear`` takes bf16, by way of fp16) and each expert's output row
    is rounded to bf16. An id outside the routed experts adds nothing."""
    if not isinstance(experts, MXFP4Experts):
        raise TypeError("mxfp4_moe expects MXFP4Experts")
    _check_x("mxfp4_moe", hidden, experts.hidden, experts.device, topk_idx, topk_w)
    if topk_idx.dtype != torch.int64 or topk_w.dtype != torch.float32:
        raise TypeError("mxfp4_moe expects int64 indices and fp32 weights")
    lead = tuple(hidden.shape[:-1])
    if topk_idx.dim() < 1 or topk_idx.shape != topk_w.shape or tuple(topk_idx.shape[:-1]) != lead:
        raise ValueError(f"mxfp4_moe: indices {tuple(topk_idx.shape)} and weights {tuple(topk_w.shape)} do not go with "
                         f"hidden {tuple(hidden.shape)}")
    if topk_idx.shape[-1] > _INT_MAX:
        raise ValueError("mxfp4_moe: top_k must be in [1, 8]")
    x2 = _rows(hidden)
    T, H, K = x2.shape[0], experts.hidden, topk_idx.shape[-1]
    out = torch.empty(*lead, H, dtype=torch.bfloat16, device=hidden.device)
    if T:
        idx, w = topk_idx.contiguous(), topk_w.contiguous()
        ws = _scratch(lib().dsmoe_mxfp4_moe_workspace_size(T, H, experts.inter, experts.n_routed, int(experts.shared),
                                                           K), hidden.device)
        _call(experts.device, "dsmoe_mxfp4_moe", x2.data_ptr(), x2.stride(0), T, experts.desc, idx.data_ptr(),
              w.data_ptr(), K, float(scale), out.data_ptr(), ws.data_ptr() or None, ws.numel(), ptr(experts.status))
    return out


def moe_forward(x: torch.Tensor, gate_weight: torch.Tensor, bias: torch.Tensor | None, config,
                experts: MXFP4Experts) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``moe_block``'s work on MXFP4 experts: dense bf16 ``x`` [T, hidden] ->
    output, routing indices and weights. Scratch is private to the call."""
    _check_x("moe_forward", x, experts.hidden, experts.device, gate_weight, bias)
    cfg = _lib.moe_config(config)
    if x.dim() != 2 or not x.is_contiguous():
        raise ValueError("moe_forward expects dense (tokens, hidden) activations")
    if gate_weight.dtype != torch.bfloat16 or (bias is not None and bias.dtype != torch.float32):
        raise TypeError("moe_forward expects a bf16 gate weight and an fp32 bias")
    if tuple(gate_weight.shape) != (cfg.n_routed, cfg.hidden) or not gate_weight.is_contiguous() or \
            (bias is not None and (bias.numel() != cfg.n_routed or not bias.is_contiguous())):
        raise ValueError(f"moe_forward expects a dense gate weight {(cfg.n_routed, cfg.hidden)} and a bias of "
                         f"{cfg.n_routed}")
    T, K = x.shape[0], cfg.top_k
    out = torch.empty_like(x)
    idx = torch.empty(T, K, dtype=torch.int64, device=x.device)
    w = torch.empty(T, K, dtype=torch.float32, device=x.device)
    ws = _scratch(lib().dsmoe_mxfp4_moe_forward_workspace_size(cfg, T), x.device)
    _call(experts.device, "dsmoe_mxfp4_moe_forward", cfg, ptr(gate_weight), ptr(bias), experts.desc, x.data_ptr(), T,
          out.data_ptr(), idx.data_ptr(), w.data_ptr(), ws.data_ptr() or None, ws.numel(), ptr(experts.status))
    return out, idx, w


class MXFP4LayerBank:
    """Every expert of one MoE layer in MXFP4 on the device (6.0 GB per
    DeepSeek-R1 layer, against 11.3 GB in FP8), written expert by expert from
    the checkpoint's FP8 weights. Stands where ``GPUTransfer`` keeps a
    ``LayerBank``; every expert is resident, group 0 is the shared expert."""

    def __init__(self, config, device: torch.device):
        E, H, F = config.n_routed_experts, config.hidden_size, config.moe_intermediate_size
        self.n_slots = self.n_groups = E + 1
        self.device = _index(torch.device(device))
        self.experts = MXFP4Experts._empty(E + 1, H, F, self.device)
        self.slot_of_host = [-1] * (E + 1)
        self.last_use: torch.cuda.Event | None = None
        self.pending: torch.cuda.Event | None = None

    @property
    def fully_resident(self) -> bool:
        return all(s >= 0 for s in self.slot_of_host)

    @property
    def nbytes(self) -> int:
        return self.experts.nbytes

    def assign(self, group: int, pinned=None) -> int:
        self.slot_of_host[group] = group
        return group

    def write_slot(self, slot: int, expert: dict, non_blocking: bool = False) -> int:
        """Quantise one FP8 expert ``{proj: (weight, scale_inv)}``, on the host
        or the device, into ``slot``; returns the FP8 bytes read."""
        n, pairs = 0, []
        for p in ("gate_proj", "up_proj", "down_proj"):
            w, s = expert[p]
            if isinstance(w, dict):  # ExpertCache entry form
                w, s = w["weight"], w["weight_scale_inv"]
            n += w.nbytes + s.nbytes
            pairs.append((w.to(self.device, non_blocking=non_blocking),
                          s.to(self.device, torch.float32, non_blocking=non_blocking).contiguous()))
        self.experts._write(slot, *pairs)
        return n

    def sync_table(self, non_blocking: bool = True) -> None:
        """Nothing to bring up to date: slot g is group g."""

"""The MXFP4 operators as measurable cases.

MXFP4 (the OCP microscaling format): a row of K numbers is held as K e2m1
codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; two codes per byte, the
even element in the low nibble) and one power-of-two scale (e8m0: a byte b
stands for 2^(b - 127)) per 32 consecutive numbers.

Operators:
  * ``quant``   quantise a tensor (bf16, fp16, fp32, or the checkpoint's e4m3
                with one fp32 scale per 128x128 block) and read it back:
                scale = 2^(floor(log2(block amax)) - 2), codes rounded to
                nearest even, saturating at 6;
  * ``linear``  bf16 activations times an MXFP4 weight;
  * ``matmul``  MXFP4 activations times an MXFP4 weight;
  * ``grouped`` bf16 rows sorted by expert times each expert's MXFP4 weight,
                ragged segments given by offsets on the device, rows behind
                the last segment come out as zeros;
  * ``moe``     the routed FFN: scale * sum_k w_k down_k(silu(gate_k x) *
                up_k x) + the shared expert, every projection MXFP4.

``run`` computes them in elementary torch operations; with ``own`` set it
calls the framework.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _api():
    pkg = os.path.join(os.getcwd(), "deepseek-on-one-gpu_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import dsmoe
    return dsmoe


# --------------------------------------------------------------------- cases
def listed():
    return [
        # the activations of a decode batch, quantised for a 4-bit product
        {"name": "quant_act_bf16_t64", "op": "quant", "type": "bf16", "rows": 64, "k": 7168},
        # an fp32 weight of a dense layer's shape, with one row more
        {"name": "quant_weight_fp32", "op": "quant", "type": "fp32", "rows": 7169, "k": 18432},
        # 32 experts of an FP8 checkpoint turned into 4-bit experts
        {"name": "quant_fp8_experts", "op": "quant", "type": "fp8", "mats": 32, "rows": 2048, "k": 7168},
        # one token through an attention output projection
        {"name": "linear_t1", "op": "linear", "t": 1, "n": 7168, "k": 16384},
        # a prefill chunk through the dense FFN's down projection
        {"name": "linear_t4096", "op": "linear", "t": 4096, "n": 7168, "k": 18432},
        # a ragged batch, both sides 4-bit, through a small odd-sized projection
        {"name": "matmul_t129", "op": "matmul", "t": 129, "n": 576, "k": 7168},
        # a prefill chunk through the dense FFN's gate projection, both sides 4-bit
        {"name": "matmul_t4096", "op": "matmul", "t": 4096, "n": 18432, "k": 7168},
        # a decode batch's rows over all experts, some of them without a row
        {"name": "grouped_r512", "op": "grouped", "e": 256, "r": 512, "n": 7168, "k": 2048, "skew": 0.0, "tail": 0},
        # a prefill chunk's rows over all experts, skewed, in a padded buffer
        {"name": "grouped_r32768", "op": "grouped", "e": 256, "r": 32768, "n": 2048, "k": 7168, "skew": 0.6,
         "tail": 100},
        # decode, one token, DeepSeek's expert shape
        {"name": "moe_t1", "op": "moe", "t": 1, "e": 256, "top": 8, "h": 7168, "f": 2048, "shared": True, "skew": 0.0},
        # a decode batch
        {"name": "moe_t64", "op": "moe", "t": 64, "e": 256, "top": 8, "h": 7168, "f": 2048, "shared": True,
         "skew": 0.0},
        # a prefill chunk
        {"name": "moe_t4096", "op": "moe", "t": 4096, "e": 256, "top": 8, "h": 7168, "f": 2048, "shared": True,
         "skew": 0.0},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    op = rng.choice(["quant", "linear", "matmul", "grouped", "moe"])
    if op == "quant":
        typ = rng.choice(["bf16", "fp16", "fp32", "fp8"])
        if typ == "fp8":
            return {"op": op, "type": typ, "mats": _log(rng, 1, 32), "rows": _log(rng, 64, 2048, 8),
                    "k": _log(rng, 128, 7168, 32)}
        return {"op": op, "type": typ, "rows": _log(rng, 1, 7169), "k": _log(rng, 32, 18432, 32)}
    if op in ("linear", "matmul"):
        return {"op": op, "t": _log(rng, 1, 4096), "n": _log(rng, 64, 18432, 8) if op == "matmul"
                else _log(rng, 64, 7168, 8), "k": _log(rng, 128, 7168 if op == "matmul" else 18432, 128)}
    if op == "grouped":
        return {"op": op, "e": _log(rng, 1, 256), "r": _log(rng, 1, 32768), "n": _log(rng, 64, 2048, 8),
                "k": _log(rng, 128, 7168, 128), "skew": rng.choice([0.0, 0.5, 1.1]), "tail": rng.choice([0, 0, 37])}
    top = rng.randint(1, 8)
    return {"op": op, "t": _log(rng, 1, 4096), "e": max(top, _log(rng, 8, 256)), "top": top,
            "h": _log(rng, 128, 7168, 128), "f": _log(rng, 128, 2048, 128), "shared": rng.random() < 0.7,
            "skew": rng.choice([0.0, 0.5, 1.1])}


def _wbytes(n, k):
    return n * (k // 2 + k // 32)


def _touched(e, picks, rows):
    return e * (1.0 - (1.0 - picks / e) ** rows)


def work(case):
    op = case["op"]
    if op == "quant":
        n = case.get("mats", 1) * case["rows"] * case["k"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}[case["type"]]
        return {"bytes": n * (size + 2), "flops": 0}
    if op in ("linear", "matmul"):
        t, n, k = case["t"], case["n"], case["k"]
        x = 2 * t * k if op == "linear" else _wbytes(t, k)
        return {"bytes": x + _wbytes(n, k) + 2 * t * n, "flops": 2 * t * n * k}
    if op == "grouped":
        r, n, k = case["r"], case["n"], case["k"]
        live = min(case["e"], _touched(case["e"], 1, r))
        return {"bytes": int(2 * r * k + live * _wbytes(n, k) + 2 * (r + case["tail"]) * n),
                "flops": 2 * r * n * k}
    t, h, f = case["t"], case["h"], case["f"]
    live = _touched(case["e"], case["top"], t) + (1 if case["shared"] else 0)
    rows = t * (case["top"] + (1 if case["shared"] else 0))
    return {"bytes": int(live * (2 * _wbytes(f, h) + _wbytes(h, f)) + 4 * t * h + 12 * t * case["top"]),
            "flops": 6 * rows * h * f}


# -------------------------------------------------------------------- inputs
def _gen(seed, salt=0):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + salt * 7919 + 17) & 0x7FFFFFFFFFFF)
    return g


def _pool(g):
    """2^17 words of 16 codes: normal blocks of 32, quantised."""
    v = torch.randn(1 << 16, 32, generator=g, device=DEV)
    m, e = torch.frexp(v.abs().amax(1, keepdim=True))
    a = v / torch.exp2((e - 3).float())
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)
    c = torch.bucketize(a.abs(), mid).to(torch.uint8) | ((a < 0).to(torch.uint8) << 3)
    c = c.view(-1, 16, 2)
    return (c[..., 0] | (c[..., 1] << 4)).view(-1, 16).contiguous().view(torch.int64).view(-1)


def _weight(g, pool, mats, n, k):
    """MXFP4 weights of about N(0, 0.02): codes [mats, n, k/2], scales [mats, n, k/32]."""
    codes = torch.empty(mats, n, k // 2, dtype=torch.uint8, device=DEV)
    words = n * k // 16
    for m in range(mats):
        pick = torch.randint(0, pool.numel(), (words,), generator=g, device=DEV, dtype=torch.int32)
        codes[m].view(-1).view(torch.int64).copy_(pool.index_select(0, pick))
    scales = torch.randint(118, 122, (mats, n, k // 32), generator=g, device=DEV, dtype=torch.uint8)
    return codes, scales


def _segments(g, e, r, skew):
    """Rows per expert: a multinomial over weights rank^-skew in random order."""
    w = torch.arange(1, e + 1, device=DEV, dtype=torch.float64) ** -skew
    w = w[torch.randperm(e, generator=g, device=DEV)]
    pick = torch.multinomial(w / w.sum(), r, replacement=True, generator=g)
    return torch.bincount(pick, minlength=e)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "quant":
        rows, k = case["rows"], case["k"]
        if case["type"] == "fp8":
            m = case["mats"]
            x = torch.empty(m, rows, k, dtype=torch.float8_e4m3fn, device=DEV)
            for i in range(m):
                w = torch.randn(rows, k, generator=g, device=DEV)
                x[i].copy_((w * 90.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn))
            s["x"] = x
            s["scale_inv"] = 2e-4 * (0.7 + 0.6 * torch.rand(m, -(-rows // 128), -(-k // 128), generator=g, device=DEV))
        else:
            x = torch.randn(rows, k, generator=g, device=DEV)
            if case["type"] == "bf16":  # activations: a few channels far above the rest
                x[:, torch.randint(0, k, (max(1, k // 500),), generator=g, device=DEV)] *= 20.0
            else:
                x *= 0.02
            s["x"] = x.to(TYPES[case["type"]])
        return s
    pool = _pool(g)
    if op in ("linear", "matmul"):
        t, n, k = case["t"], case["n"], case["k"]
        codes, scales = _weight(g, pool, 1, n, k)
        s["w"] = (codes[0], scales[0])
        if op == "linear":
            s["x"] = torch.randn(t, k, generator=g, device=DEV).to(torch.bfloat16)
        else:
            codes, _ = _weight(g, pool, 1, t, k)
            s["a"] = (codes[0], torch.randint(125, 128, (t, k // 32), generator=g, device=DEV, dtype=torch.uint8))
        if own:
            s["weight"] = _api().MXFP4Weight(*s["w"])
        return s
    if op == "grouped":
        e, r, n, k = case["e"], case["r"], case["n"], case["k"]
        s["w"] = _weight(g, pool, e, n, k)
        counts = _segments(g, e, r, case["skew"])
        s["counts"] = counts.tolist()
        s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        s["x"] = torch.randn(r + case["tail"], k, generator=g, device=DEV).to(torch.bfloat16)
        if own:
            s["weight"] = _api().MXFP4Weight(*s["w"])
        return s
    t, e, top, h, f = case["t"], case["e"], case["top"], case["h"], case["f"]
    m = e + (1 if case["shared"] else 0)  # the shared expert first
    s["gate"], s["up"] = _weight(g, pool, m, f, h), _weight(g, pool, m, f, h)
    s["down"] = _weight(g, pool, m, h, f)
    s["x"] = torch.randn(t, h, generator=g, device=DEV).to(torch.bfloat16)
    load = -case["skew"] * torch.log(torch.arange(1, e + 1, device=DEV).float())
    load = load[torch.randperm(e, generator=g, device=DEV)]
    noise = -torch.log(-torch.log(torch.rand(t, e, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-6)))
    s["idx"] = (load + noise).topk(top, dim=1).indices
    w = torch.rand(t, top, generator=g, device=DEV) + 0.1
    s["w"] = w / w.sum(1, keepdim=True)
    s["scale"] = 2.5
    s["counts"] = torch.bincount(s["idx"].reshape(-1), minlength=e).tolist()
    if own:
        api = _api()
        s["experts"] = api.MXFP4Experts(api.MXFP4Weight(*s["gate"]), api.MXFP4Weight(*s["up"]),
                                        api.MXFP4Weight(*s["down"]), shared=case["shared"])
    return s


# ---------------------------------------------------------------- plain form
def _read(codes, scales):
    """The fp32 numbers that codes [..., k/2] and scales [..., k/32] stand for."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=codes.device)
    pairs = torch.stack([codes & 15, codes >> 4], dim=-1)
    v = table[pairs.to(torch.int32)].reshape(*scales.shape, 32)
    return (v * torch.exp2(scales.float() - 127.0).unsqueeze(-1)).reshape(*codes.shape[:-1], -1)


def _round_blocks(v):
    """Numbers of v [..., k], rounded to MXFP4 and back, in v's type."""
    b = v.reshape(*v.shape[:-1], -1, 32)
    amax = b.abs().amax(dim=-1, keepdim=True)
    e = torch.frexp(amax).exponent - 3
    s = torch.where(amax > 0, torch.exp2(e.clamp(-127, 127).to(v.dtype)), torch.ones_like(amax))
    q = b / s
    a = q.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(v.dtype)
    r = (torch.round(a / step) * step).clamp(max=6.0)
    return (torch.copysign(r, q) * s).reshape(v.shape)


def _plain_quant(s):
    x = s["x"]
    if "scale_inv" not in s:
        return _round_blocks(x.float()).to(torch.bfloat16)
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    rows, k = x.shape[1:]
    for i in range(x.shape[0]):  # in 64 bits: products next to a rounding border
        sc = s["scale_inv"][i].double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)[:, :k]
        out[i] = _round_blocks(x[i].double() * sc).to(torch.bfloat16)
    return out


def _plain_grouped(s):
    codes, scales = s["w"]
    x = s["x"]
    out = torch.zeros(x.shape[0], codes.shape[1], dtype=torch.bfloat16, device=x.device)
    at = 0
    for e, c in enumerate(s["counts"]):
        if c:
            out[at:at + c] = (x[at:at + c].float() @ _read(codes[e], scales[e]).T).to(torch.bfloat16)
            at += c
    return out


def _plain_ffn(s, m, x):
    def w(p):
        return _read(s[p][0][m], s[p][1][m]).T
    gate = x @ w("gate")
    return (gate * torch.sigmoid(gate) * (x @ w("up"))) @ w("down")


def _plain_moe(s):
    x, idx = s["x"].float(), s["idx"]
    base = 1 if s["case"]["shared"] else 0
    flat = idx.reshape(-1)
    order = torch.argsort(flat, stable=True)
    token, weight = order // idx.shape[1], s["w"].reshape(-1)[order]
    acc = torch.zeros_like(x)
    at = 0
    for e, c in enumerate(s["counts"]):
        if c:
            t = token[at:at + c]
            acc.index_add_(0, t, _plain_ffn(s, base + e, x[t]) * weight[at:at + c, None])
            at += c
    acc *= s["scale"]
    if base:
        acc += _plain_ffn(s, 0, x)
    return acc.to(torch.bfloat16)


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        api = _api()
        if op == "quant":
            return api.mxfp4_dequantize(*api.mxfp4_quantize(s["x"], s.get("scale_inv")))
        if op == "linear":
            return api.mxfp4_linear(s["x"], s["weight"])
        if op == "matmul":
            return api.mxfp4_matmul(*s["a"], s["weight"])
        if op == "grouped":
            return api.mxfp4_grouped_linear(s["x"], s["weight"], s["offsets"])
        return api.mxfp4_moe(s["x"], s["idx"], s["w"], s["experts"], scale=s["scale"])
    if op == "quant":
        return _plain_quant(s)
    if op == "linear":
        return (s["x"].float() @ _read(*s["w"]).T).to(torch.bfloat16)
    if op == "matmul":
        return (_read(*s["a"]) @ _read(*s["w"]).T).to(torch.bfloat16)
    if op == "grouped":
        return _plain_grouped(s)
    return _plain_moe(s)


# ------------------------------------------------------------------- exact
def _exact_read(codes, scales):
    """64-bit numbers of MXFP4 data, from the fields of each code: sign, two
    exponent bits (0 is subnormal), one mantissa bit."""
    n = torch.empty(*codes.shape, 2, dtype=torch.int64, device=codes.device)
    n[..., 0] = codes.bitwise_and(0x0F)
    n[..., 1] = codes.bitwise_right_shift(4)
    n = n.flatten(-2)
    e, m = (n >> 1) & 3, (n & 1).double()
    mag = torch.where(e == 0, 0.5 * m, torch.ldexp(1.0 + 0.5 * m, (e - 1).double()))
    val = mag * (1 - 2 * (n >> 3)).double()
    return torch.ldexp(val, (scales.double() - 127).repeat_interleave(32, dim=-1))


def _exact_quant(v):
    """Nearest MXFP4 number by distance to every grid point; a tie goes to the
    even code."""
    b = v.reshape(-1, 32)
    amax = b.abs().amax(1)
    e = torch.floor(torch.log2(amax.clamp(min=1e-300)))
    e = torch.where(torch.exp2(e) > amax, e - 1, torch.where(torch.exp2(e + 1) <= amax, e + 1, e))
    s = torch.where(amax > 0, torch.exp2((e - 2).clamp(-127, 127)), torch.ones_like(amax)).unsqueeze(1)
    a = b.abs() / s
    best = torch.zeros_like(a)
    dist = a.clone()
    for code, point in enumerate(GRID[1:], start=1):
        d = (a - point).abs()
        take = (d < dist) | ((d == dist) & (code % 2 == 0))
        best = torch.where(take, torch.full_like(best, point), best)
        dist = torch.where(take, d, dist)
    return (torch.where(b < 0, -best, best) * s).reshape(v.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        x = s["x"]
        if "scale_inv" not in s:
            return _exact_quant(x.double())
        rows, k = x.shape[1:]
        out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        row, col = torch.arange(rows, device=DEV) // 128, torch.arange(k, device=DEV) // 128
        for i in range(x.shape[0]):
            out[i] = _exact_quant(x[i].double() * s["scale_inv"][i].double()[row][:, col])
        return out
    if op == "linear":
        return s["x"].double() @ _exact_read(*s["w"]).T
    if op == "matmul":
        return _exact_read(*s["a"]) @ _exact_read(*s["w"]).T
    if op == "grouped":
        codes, scales = s["w"]
        off = s["offsets"].tolist()
        out = torch.zeros(s["x"].shape[0], codes.shape[1], dtype=torch.float64, device=DEV)
        for e in range(codes.shape[0]):
            if off[e + 1] > off[e]:
                out[off[e]:off[e + 1]] = s["x"][off[e]:off[e + 1]].double() @ _exact_read(codes[e], scales[e]).T
        return out
    x = s["x"].double()
    base = 1 if case["shared"] else 0

    def ffn(m, rows):
        g = rows @ _exact_read(s["gate"][0][m], s["gate"][1][m]).T
        u = rows @ _exact_read(s["up"][0][m], s["up"][1][m]).T
        return (g / (1.0 + torch.exp(-g)) * u) @ _exact_read(s["down"][0][m], s["down"][1][m]).T

    out = ffn(0, x) if base else torch.zeros_like(x)
    for e in range(case["e"]):
        t, k = (s["idx"] == e).nonzero(as_tuple=True)
        if t.numel():
            out.index_add_(0, t, ffn(base + e, x[t]) * (s["scale"] * s["w"][t, k].double()).unsqueeze(1))
    return out

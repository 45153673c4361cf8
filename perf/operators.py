"""Timed cases of the NVFP4 feed-forward operators.

Four operators, each in a plain form (elementary torch operations in fp32) and as the package's kernels:

  linear   D = residual + act(alpha * A B^T + bias) on packed NVFP4 operands       (``nvfp4_gemm_epilogue``)
  grouped  the same product per group of rows, ragged groups, one weight each       (``nvfp4_grouped_gemm``)
  experts  routed feed-forward: quantize per expert, two grouped products, weighted sum (``moe_ffn.expert_ffn``)
  norm     gated residual between the norm after a block and the norm before the next  (``gated_add_rmsnorm_fp4quant``)

NVFP4: E2M1 values, two per byte, one E4M3 scale per 16 values along the row, an fp32 encode scale per tensor.  Scale
bytes lie in 128 x 4 tiles of 512 bytes; a group's rows start on a tile of their own, tile ``offsets[g] // 128 + g``.
"""

import functools
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EPS = 1e-6


# ---- cases ------------------------------------------------------------------------------------------------------


def listed():
    return [
        # decode step of an output projection: 16 sequences, bias and residual; bound by the weight's bytes
        {"name": "linear_decode_16", "op": "linear", "m": 16, "n": 8192, "k": 8192, "act": "none", "bias": True, "residual": True, "dtype": "bfloat16"},
        # a ragged prompt batch: rows and columns that end inside tiles, K that ends inside a slab, fp16 output
        {"name": "linear_ragged_1000", "op": "linear", "m": 1000, "n": 3592, "k": 7104, "act": "gelu", "bias": True, "residual": False, "dtype": "float16"},
        # prefill, down projection with the residual added
        {"name": "linear_prefill_4096", "op": "linear", "m": 4096, "n": 8192, "k": 4096, "act": "none", "bias": True, "residual": True, "dtype": "bfloat16"},
        # the sharded FFN's projection on one GPU, with its activation
        {"name": "linear_ffn_8192", "op": "linear", "m": 8192, "n": 28672, "k": 8192, "act": "silu", "bias": False, "residual": False, "dtype": "bfloat16"},
        # decode through experts: a few rows each, some groups empty; bound by the weights that are touched
        {"name": "grouped_decode_96", "op": "grouped", "rows": 96, "groups": 64, "n": 4096, "k": 2048, "act": "none", "bias": False, "dtype": "bfloat16"},
        # seven uneven groups of an odd batch, sizes that end inside every tile
        {"name": "grouped_ragged_777", "op": "grouped", "rows": 777, "groups": 7, "n": 1352, "k": 1088, "act": "gelu_tanh", "bias": True, "dtype": "float16"},
        # prefill through experts
        {"name": "grouped_prefill_16384", "op": "grouped", "rows": 16384, "groups": 16, "n": 4096, "k": 4096, "act": "none", "bias": False, "dtype": "bfloat16"},
        # one token through its 8 experts of 64: latency
        {"name": "experts_token_1", "op": "experts", "tokens": 1, "experts": 64, "topk": 8, "hidden": 4096, "inner": 1024, "dtype": "bfloat16"},
        # a prompt of 4096 tokens through 4 of 32 experts
        {"name": "experts_prefill_4096", "op": "experts", "tokens": 4096, "experts": 32, "topk": 4, "hidden": 2048, "inner": 1408, "dtype": "bfloat16"},
        # one decode step's row, quantized for the next product: latency
        {"name": "norm_row_1", "op": "norm", "m": 1, "h": 8192, "rows_per_gate": 1, "post": True, "gate": True, "quantize": True, "swizzled": True, "dtype": "bfloat16"},
        # a middling batch, quantized with row-major scales, no gate
        {"name": "norm_quant_500", "op": "norm", "m": 500, "h": 5136, "rows_per_gate": 1, "post": True, "gate": False, "quantize": True, "swizzled": False, "dtype": "float16"},
        # prefill: four sequences of 2048 tokens with a gate row each, 16-bit output
        {"name": "norm_prefill_8192", "op": "norm", "m": 8192, "h": 7168, "rows_per_gate": 2048, "post": True, "gate": True, "quantize": False, "swizzled": False, "dtype": "bfloat16"},
    ]


def _log(rng, low, high, step=1):
    """A multiple of `step` in [low, high], spread evenly over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    op = rng.choice(["linear", "grouped", "experts", "norm"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if op == "linear":
        return {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 64, 16384, 8), "k": _log(rng, 64, 8192, 64),
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.6,
                "residual": rng.random() < 0.5, "dtype": dtype}
    if op == "grouped":
        groups, n = _log(rng, 1, 64), _log(rng, 64, 8192, 8)
        k = _log(rng, 64, min(8192, (1 << 30) // (groups * n) // 64 * 64), 64)
        return {"op": op, "rows": _log(rng, 1, 16384), "groups": groups, "n": n, "k": k,
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.5, "dtype": dtype}
    if op == "experts":
        experts = _log(rng, 4, 64)
        return {"op": op, "tokens": _log(rng, 1, 4096), "experts": experts, "topk": rng.randint(1, min(8, experts)),
                "hidden": _log(rng, 256, 4096, 64), "inner": _log(rng, 128, 1408, 64), "dtype": dtype}
    quantize = rng.random() < 0.4
    m = _log(rng, 1, 8192)
    return {"op": op, "m": m, "h": _log(rng, 64, 7168, 16), "rows_per_gate": _log(rng, 1, m), "post": rng.random() < 0.7,
            "gate": rng.random() < 0.7, "quantize": quantize, "swizzled": rng.random() < 0.5, "dtype": dtype}


# ---- inputs -----------------------------------------------------------------------------------------------------


def _dtype(case):
    return {"bfloat16": torch.bfloat16, "float16": torch.float16}[case["dtype"]]


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=DEVICE) * std


def _round_e2m1(v):
    """Magnitudes of E2M1 nearest to `v`, ties to the even code, the largest for what is beyond it."""
    a = v.abs()
    low = torch.where(a <= 0.25, 0.0, torch.where(a < 0.75, 0.5, torch.where(a <= 1.25, 1.0, 1.5)))
    high = torch.where(a <= 2.5, 2.0, torch.where(a < 3.5, 3.0, torch.where(a <= 5.0, 4.0, 6.0)))
    return torch.copysign(torch.where(a < 1.75, low, high), v)


def _quantize(x, gs):
    """fp32 [..., k] -> (E2M1 values, E4M3 scales [..., k/16]); gs broadcasts against [..., k/16]."""
    blocks = x.unflatten(-1, (-1, 16))
    scale = (gs * (blocks.abs().amax(-1) * (1.0 / 6.0))).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float()
    inverse = torch.where(s == 0, torch.zeros_like(s), 1.0 / (s * (1.0 / gs)))
    return _round_e2m1(blocks * inverse[..., None]).flatten(-2), scale


def _pack(values):
    """E2M1 values -> bytes, the even element in the low nibble."""
    a = values.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(values).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _swizzle(scale, rows):
    """E4M3 [..., rows, cols] -> bytes of its 128 x 4 tiles, padding zero; rows is a multiple of 128."""
    lead, cols = scale.shape[:-2], scale.shape[-1]
    full = torch.zeros(*lead, rows, -(-cols // 4) * 4, dtype=torch.uint8, device=scale.device)
    full[..., : scale.shape[-2], :cols] = scale.view(torch.uint8)
    tiles = full.unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))  # [..., tile, 4, 32, cols/4, 4]
    return tiles.movedim(-2, -4).movedim(-3, -2).contiguous().flatten()


def _up(v, step):
    return -(-v // step) * step


def _weights(g, groups, n, k, std=0.02):
    """Quantized N(0, std) weights of every group: packed, scale tiles, encode scale per group."""
    packed = torch.empty(groups, n, k // 2, dtype=torch.uint8, device=DEVICE)
    tiles = torch.empty(groups, _up(n, 128) * _up(k // 16, 4), dtype=torch.uint8, device=DEVICE)
    gs = torch.empty(groups, device=DEVICE)
    step = max(1, (1 << 27) // (n * k))
    for at in range(0, groups, step):
        w = _randn(g, min(step, groups - at), n, k, std=std).to(torch.bfloat16).float()
        amax = w.flatten(1).abs().amax(1)
        gs[at : at + step] = 2688.0 / amax
        v, s = _quantize(w, gs[at : at + step, None, None])
        packed[at : at + step] = _pack(v)
        tiles[at : at + step] = _swizzle(s, _up(n, 128)).view(w.shape[0], -1)
    return packed, tiles.view(-1), gs


def _grouped_rows(offsets, rows):
    """Group of every row, and the row of the scale tiles that it has: a group starts on a tile of its own."""
    r = torch.arange(rows, device=offsets.device)
    group = torch.searchsorted(offsets.long(), r, right=True) - 1
    first = offsets.long()[group]
    return group, (first // 128 + group) * 128 + r - first


def _popular(g, count):
    """Uneven shares, as routers give them."""
    return torch.softmax(0.5 * _randn(g, count), 0)


def prepare(case, seed):
    g = _generator(seed)
    dtype = _dtype(case)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = _randn(g, m, k).to(torch.bfloat16).float()
        gs = 2688.0 / x.abs().amax()
        v, s = _quantize(x, gs)
        b, sfb, gsb = _weights(g, 1, n, k)
        return {"case": case, "a": _pack(v), "sfa": _swizzle(s, _up(m, 128)), "b": b[0], "sfb": sfb, "alpha": 1.0 / (gs * gsb),
                "bias": _randn(g, n, std=0.5).to(dtype) if case["bias"] else None,
                "residual": _randn(g, m, n).to(dtype) if case["residual"] else None}
    if case["op"] == "grouped":
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        member = torch.multinomial(_popular(g, groups), rows, replacement=True, generator=g)
        sizes = torch.bincount(member, minlength=groups)
        offsets = torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)
        x = _randn(g, rows, k).to(torch.bfloat16).float()
        gs = 2688.0 / x.abs().amax()
        v, s = _quantize(x, gs)
        padded = torch.zeros((rows // 128 + groups) * 128, k // 16, dtype=torch.uint8, device=DEVICE)
        padded[_grouped_rows(offsets, rows)[1]] = s.view(torch.uint8)
        b, sfb, gsb = _weights(g, groups, n, k)
        return {"case": case, "a": _pack(v), "sfa": _swizzle(padded.view(torch.float8_e4m3fn), padded.shape[0]), "b": b, "sfb": sfb,
                "alpha": 1.0 / (gs * gsb), "offsets": offsets, "largest": int(sizes.max()),
                "bias": _randn(g, groups, n, std=0.5).to(dtype) if case["bias"] else None}
    if case["op"] == "experts":
        t, e, topk, h, f = (case[name] for name in ("tokens", "experts", "topk", "hidden", "inner"))
        noise = -torch.log(-torch.log(torch.rand(t, e, generator=g, device=DEVICE).clamp(1e-6, 1 - 1e-6)))
        score, ids = (_popular(g, e).log() + noise).topk(topk, dim=-1)
        w1, sf1, gsw1 = _weights(g, e, 2 * f, h)
        w2, sf2, gsw2 = _weights(g, e, h, f)
        gs1 = torch.full((e,), 2688.0 / 5.3, device=DEVICE)
        gs2 = 2688.0 / ((8.0 + torch.rand(e, generator=g, device=DEVICE)) * 0.02**2 * h)  # the largest products of two N(0, 0.02 sqrt(h))
        return {"case": case, "x": _randn(g, t, h).to(dtype), "ids": ids.to(torch.int32), "gates": torch.softmax(score, -1),
                "w1": w1, "sf1": sf1, "alpha1": 1.0 / (gs1 * gsw1), "gs1": gs1, "w2": w2, "sf2": sf2, "alpha2": 1.0 / (gs2 * gsw2), "gs2": gs2,
                "largest": int(torch.bincount(ids.flatten(), minlength=e).max())}
    m, h = case["m"], case["h"]
    gates = -(-m // case["rows_per_gate"])
    pairs = torch.tensor([_fp8_code(i & 15) | _fp8_code(i >> 4) << 8 for i in range(256)], dtype=torch.int32)
    return {"case": case, "x": (_randn(g, m, h) * (0.5 + torch.rand(m, 1, generator=g, device=DEVICE))).to(dtype), "residual": _randn(g, m, h, std=2.0).to(dtype),
            "w_post": (1.0 + _randn(g, h, std=0.1)).to(dtype) if case["post"] else None,
            "gate": _randn(g, gates, h, std=0.5).to(dtype) if case["gate"] else None,
            "w_pre": (1.0 + _randn(g, h, std=0.1)).to(dtype), "scale": 0.8 + 0.2 * (seed % 7) / 7.0,
            "gs": 300.0 + 100.0 * torch.rand(1, generator=g, device=DEVICE), "pairs": pairs.to(torch.int16).to(DEVICE)}


def _fp8_code(nibble):
    """The E4M3 byte with the value of an E2M1 code."""
    exponent, mantissa = (nibble >> 1) & 3, nibble & 1
    if exponent:
        magnitude = (exponent + 6) << 3 | mantissa << 2
    else:
        magnitude = 0x30 if mantissa else 0
    return (nibble & 8) << 4 | magnitude


# ---- plain forms ------------------------------------------------------------------------------------------------


def _values(packed):
    """Bytes -> E2M1 values in fp32."""
    table = torch.tensor(E2M1 + [-v for v in E2M1], device=packed.device)
    return torch.stack((table[(packed & 15).int()], table[(packed >> 4).int()]), -1).flatten(-2)


def _scales(tiles, rows, cols):
    """Scale tiles -> fp32 [tile rows, cols]; `rows` is a multiple of 128."""
    t = tiles.view(rows // 128, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rows, -1)
    return t[:, :cols].contiguous().view(torch.float8_e4m3fn).float()


def _decode(packed, scale):
    return (_values(packed).unflatten(-1, (-1, 16)) * scale[..., None]).flatten(-2)


def _activate(v, act):
    if act == "relu":
        return v.clamp(min=0.0)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _decode_weights(packed, tiles):
    groups, n, half = packed.shape
    scale = _scales(tiles, groups * _up(n, 128), half // 8).view(groups, -1, half // 8)[:, :n]
    return _decode(packed, scale)


def _grouped_product(a, b, offsets, largest):
    """Rows of `a` by the weight of their group, fp32: groups padded to the largest, one batched product."""
    rows = a.shape[0]
    group = _grouped_rows(offsets, rows)[0]
    first = offsets.long()
    at = (first[:-1, None] + torch.arange(largest, device=a.device)).clamp(max=rows - 1)
    return torch.bmm(a[at], b.transpose(1, 2))[group, torch.arange(rows, device=a.device) - first[group]]


def _run_linear(s):
    case = s["case"]
    a = _decode(s["a"], _scales(s["sfa"], _up(case["m"], 128), case["k"] // 16)[: case["m"]])
    d = (a @ _decode_weights(s["b"][None], s["sfb"])[0].T) * s["alpha"]
    if s["bias"] is not None:
        d = d + s["bias"].float()
    d = _activate(d, case["act"])
    if s["residual"] is not None:
        d = d + s["residual"].float()
    return d.to(_dtype(case))


def _run_grouped(s):
    case = s["case"]
    group, at = _grouped_rows(s["offsets"], case["rows"])
    a = _decode(s["a"], _scales(s["sfa"], (case["rows"] // 128 + case["groups"]) * 128, case["k"] // 16)[at])
    d = _grouped_product(a, _decode_weights(s["b"], s["sfb"]), s["offsets"], s["largest"]) * s["alpha"][group, None]
    if s["bias"] is not None:
        d = d + s["bias"].float()[group]
    return _activate(d, case["act"]).to(_dtype(case))


def _run_experts(s):
    case = s["case"]
    e, topk, f, dtype = case["experts"], case["topk"], case["inner"], _dtype(case)
    flat = s["ids"].flatten().long()
    order = torch.sort(flat, stable=True).indices
    offsets = torch.cat([flat.new_zeros(1), torch.bincount(flat, minlength=e).cumsum(0)])
    expert = flat[order]
    v, scale = _quantize(s["x"][order // topk].float(), s["gs1"][expert, None])
    y = _grouped_product((v.unflatten(-1, (-1, 16)) * scale.float()[..., None]).flatten(-2), _decode_weights(s["w1"], s["sf1"]), offsets, s["largest"])
    y = (y * s["alpha1"][expert, None]).to(dtype).float()
    y = (_activate(y[:, :f], "silu") * y[:, f:]).to(dtype).float()
    v, scale = _quantize(y, s["gs2"][expert, None])
    z = _grouped_product((v.unflatten(-1, (-1, 16)) * scale.float()[..., None]).flatten(-2), _decode_weights(s["w2"], s["sf2"]), offsets, s["largest"])
    z = (z * s["alpha2"][expert, None]).to(dtype).float()
    back = torch.empty_like(z)
    back[order] = z
    return (back.view(case["tokens"], topk, -1) * s["gates"][..., None]).sum(1).to(dtype)


def _run_norm(s):
    case = s["case"]
    dtype = _dtype(case)
    u = s["x"].float()
    if s["w_post"] is not None:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * s["w_post"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()[torch.arange(case["m"], device=u.device) // case["rows_per_gate"]]
    h = (s["scale"] * s["residual"].float() + u).to(dtype)
    y = h.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["w_pre"].float()
    if not case["quantize"]:
        return {"residual": h, "y": y.to(dtype)}
    v, scale = _quantize(y, s["gs"])
    return {"residual": h, "y": v.to(torch.float8_e4m3fn), "scales": scale}


# ---- the package's kernels --------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _package():
    path = os.path.join(os.getcwd(), "tirx-kernels_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from tirx_kernels.basic import gated_add_rmsnorm_fp4quant, moe_ffn, nvfp4_gemm_epilogue, nvfp4_grouped_gemm
    from tirx_kernels.runner import compile_kernel

    return {"linear": nvfp4_gemm_epilogue, "grouped": nvfp4_grouped_gemm, "experts": moe_ffn, "norm": gated_add_rmsnorm_fp4quant,
            "compile": compile_kernel}


@functools.lru_cache(maxsize=None)
def _executable(op, **config):
    return _package()["compile"](_package()[op].get_kernel(**config))


def _own_linear(s):
    c = s["case"]
    ex = _executable("linear", M=c["m"], N=c["n"], K=c["k"], activation=c["act"], out_dtype=c["dtype"])
    d = torch.empty(c["m"], c["n"], dtype=_dtype(c), device=DEVICE)
    ex(s["a"], s["b"], s["sfa"], s["sfb"], s["alpha"], s["bias"], s["residual"], d)
    return d


def _own_grouped(s):
    c = s["case"]
    ex = _executable("grouped", rows=c["rows"], groups=c["groups"], N=c["n"], K=c["k"], activation=c["act"], out_dtype=c["dtype"])
    d = torch.empty(c["rows"], c["n"], dtype=_dtype(c), device=DEVICE)
    ex(s["a"], s["b"], s["sfa"], s["sfb"], s["alpha"], s["offsets"], s["bias"], d)
    return d


def _own_experts(s):
    moe = _package()["experts"]
    weights = moe.ExpertWeights(s["w1"], s["sf1"], s["alpha1"], s["gs1"], s["w2"], s["sf2"], s["alpha2"], s["gs2"])
    return moe.expert_ffn(s["x"], s["ids"], s["gates"], weights)


def _own_norm(s):
    c = s["case"]
    m, h = c["m"], c["h"]
    ex = _executable("norm", input_dtype=c["dtype"], M=m, H=h, quantize=c["quantize"], swizzled=c["swizzled"], rows_per_gate=c["rows_per_gate"])
    out = torch.empty(m, h, dtype=_dtype(c), device=DEVICE)
    if not c["quantize"]:
        y = torch.empty_like(out)
        ex(s["x"], s["residual"], s["w_post"], s["gate"], s["w_pre"], out, y, None, None, s["scale"], EPS)
        return {"residual": out, "y": y}
    y = torch.empty(m, h // 2, dtype=torch.uint8, device=DEVICE)
    rows = _up(m, 128)
    sf = torch.empty(rows * _up(h // 16, 4) if c["swizzled"] else m * (h // 16), dtype=torch.uint8, device=DEVICE)
    ex(s["x"], s["residual"], s["w_post"], s["gate"], s["w_pre"], out, y, sf, s["gs"], s["scale"], EPS)
    if c["swizzled"]:
        sf = sf.view(rows // 128, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rows, -1)[:m, : h // 16].contiguous()
    values = s["pairs"][y.view(-1).int()].view(torch.float8_e4m3fn)
    return {"residual": out, "y": values.view(m, h), "scales": sf.view(m, h // 16).view(torch.float8_e4m3fn)}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "grouped": _own_grouped, "experts": _own_experts, "norm": _own_norm}[op](state)
    return {"linear": _run_linear, "grouped": _run_grouped, "experts": _run_experts, "norm": _run_norm}[op](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------


def _fp4_bytes(count):
    return count / 2 + count / 16


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        extra = (2 * n if case["bias"] else 0) + (2 * m * n if case["residual"] else 0)
        return {"bytes": _fp4_bytes((m + n) * k) + 2 * m * n + extra, "flops": 2.0 * m * n * k}
    if case["op"] == "grouped":
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        touched = groups * (1.0 - (1.0 - 1.0 / groups) ** rows)
        return {"bytes": _fp4_bytes(rows * k + touched * n * k) + 2 * rows * n + (2 * touched * n if case["bias"] else 0), "flops": 2.0 * rows * n * k}
    if case["op"] == "experts":
        t, e, topk, h, f = (case[name] for name in ("tokens", "experts", "topk", "hidden", "inner"))
        touched = e * (1.0 - (1.0 - topk / e) ** t)
        return {"bytes": 4 * t * h + 8 * t * topk + _fp4_bytes(touched * 3 * f * h), "flops": 6.0 * t * topk * f * h}
    m, h = case["m"], case["h"]
    out = m * h * (0.5 + 1 / 16) if case["quantize"] else 2 * m * h
    gates = -(-m // case["rows_per_gate"]) if case["gate"] else 0
    return {"bytes": 6 * m * h + out + 2 * h * (1 + case["post"] + gates), "flops": 12.0 * m * h}


# ---- from the definitions, in 64 bits ---------------------------------------------------------------------------


def _x_values(packed):
    codes = torch.empty(*packed.shape[:-1], packed.shape[-1] * 2, dtype=torch.int64, device=packed.device)
    codes[..., 0::2], codes[..., 1::2] = packed.long() % 16, packed.long() // 16
    exponent, mantissa = codes // 2 % 4, (codes % 2).double()
    magnitude = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * torch.pow(2.0, exponent.double() - 1))
    return torch.where(codes >= 8, -magnitude, magnitude)


def _x_scale(tiles, row, cols):
    """Scales of the tile rows `row` (int64), read one by one by their place in the tiles."""
    c = torch.arange(cols, device=tiles.device)
    row = row[:, None]
    at = row // 128 * (128 * _up(cols, 4)) + c // 4 * 512 + row % 32 * 16 + row % 128 // 32 * 4 + c % 4
    byte = tiles[at].long()
    exponent, mantissa = byte // 8 % 16, (byte % 8).double() / 8
    return torch.where(exponent == 0, mantissa * 2.0**-6, (1 + mantissa) * torch.pow(2.0, exponent.double() - 7))


def _x_matrix(packed, tiles, row):
    return _x_values(packed) * _x_scale(tiles, row, packed.shape[-1] // 8).repeat_interleave(16, -1)


def _x_activate(v, act):
    f = torch.nn.functional
    return {"none": lambda: v, "relu": lambda: f.relu(v), "gelu": lambda: f.gelu(v), "gelu_tanh": lambda: f.gelu(v, approximate="tanh"),
            "silu": lambda: f.silu(v)}[act]()


def _x_quantize(x, gs):
    """Values that a row block stands for after quantization, in the units of the encode scale."""
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    b = x.view(x.shape[0], -1, 16)
    scale = (gs * b.abs().amax(-1) / 6).clamp(max=448).to(torch.float32).to(torch.float8_e4m3fn).double()
    v = torch.where(scale[..., None] == 0, torch.zeros_like(b), b * gs[..., None] / scale[..., None].clamp(min=1e-30))
    above = torch.bucketize(v.abs().clamp(max=6.0), grid).clamp(max=7)
    below = (above - 1).clamp(min=0)
    up, down = grid[above] - v.abs().clamp(max=6.0), v.abs().clamp(max=6.0) - grid[below]
    code = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return torch.copysign(grid[code], v).view_as(x), scale


def exact(case, seed):
    s = prepare(case, seed)
    dtype = _dtype(case)
    if case["op"] == "linear":
        rows = torch.arange(max(case["m"], case["n"]), device=DEVICE)
        b = _x_matrix(s["b"], s["sfb"], rows[: case["n"]])
        d = torch.empty(case["m"], case["n"], dtype=torch.float64, device=DEVICE)
        for at in range(0, case["m"], 1024):
            r = rows[at : min(at + 1024, case["m"])]
            d[r] = _x_activate(_x_matrix(s["a"][r], s["sfa"], r) @ b.T * s["alpha"].double() + (0 if s["bias"] is None else s["bias"].double()), case["act"])
        return d if s["residual"] is None else d + s["residual"].double()
    if case["op"] == "grouped":
        ends = s["offsets"].tolist()
        d = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEVICE)
        for group, (first, last) in enumerate(zip(ends, ends[1:])):
            r = torch.arange(last - first, device=DEVICE)
            a = _x_matrix(s["a"][first:last], s["sfa"], (first // 128 + group) * 128 + r)
            b = _x_matrix(s["b"][group], s["sfb"], group * _up(case["n"], 128) + torch.arange(case["n"], device=DEVICE))
            d[first:last] = _x_activate(a @ b.T * s["alpha"][group].double() + (0 if s["bias"] is None else s["bias"][group].double()), case["act"])
        return d
    if case["op"] == "experts":
        h, f = case["hidden"], case["inner"]
        out = torch.zeros(case["tokens"], h, dtype=torch.float64, device=DEVICE)
        for e in range(case["experts"]):
            token, slot = torch.nonzero(s["ids"] == e, as_tuple=True)
            if not token.numel():
                continue
            v, scale = _x_quantize(s["x"][token].double(), s["gs1"][e].double().view(1, 1))
            w = _x_matrix(s["w1"][e], s["sf1"], e * _up(2 * f, 128) + torch.arange(2 * f, device=DEVICE))
            y = ((v * scale.repeat_interleave(16, -1)) @ w.T * s["alpha1"][e].double()).to(dtype).double()
            y = (torch.nn.functional.silu(y[:, :f]) * y[:, f:]).to(dtype).double()
            v, scale = _x_quantize(y, s["gs2"][e].double().view(1, 1))
            w = _x_matrix(s["w2"][e], s["sf2"], e * _up(h, 128) + torch.arange(h, device=DEVICE))
            z = ((v * scale.repeat_interleave(16, -1)) @ w.T * s["alpha2"][e].double()).to(dtype).double()
            out.index_add_(0, token, z * s["gates"][token, slot].double()[:, None])
        return out
    x, r = s["x"].double(), s["residual"].double()
    if case["post"]:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w_post"].double()
    if case["gate"]:
        x = x * s["gate"].double().repeat_interleave(case["rows_per_gate"], 0)[: case["m"]]
    h = s["scale"] * r + x
    y = h.to(dtype).double()
    y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * s["w_pre"].double()
    if not case["quantize"]:
        return {"residual": h, "y": y}
    v, scale = _x_quantize(y, s["gs"].double().view(1, 1))
    return {"residual": h, "y": v, "scales": scale}

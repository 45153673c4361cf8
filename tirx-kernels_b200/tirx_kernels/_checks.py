"""Torch-side helpers shared by the kernel modules' ``run_test`` / ``run_gpu``.

Byte-format decoding (packed E2M1, E4M3 / UE8M0 block scales, the three scale-factor
layouts), guard regions, and the roofline annotation of benchmark records.  Everything
here runs on whatever device its tensors live on; none of it is on the launch path.
"""

from __future__ import annotations

import json
import os
from pathlib import Path

E2M1_TABLE = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
GUARD_ELEMENTS = 128
GUARD_BYTE = 0xA5


def ceil_div(a: int, b: int) -> int:
    return -(-a // b)


def padded_sf_cols(sf_cols: int) -> int:
    return ceil_div(sf_cols, 4) * 4


def sf_numel(m: int, sf_cols: int, layout: str) -> int:
    if layout == "linear":
        return m * sf_cols
    tile = 8 if layout == "8x4" else 128
    return ceil_div(m, tile) * tile * padded_sf_cols(sf_cols)


def sf_offsets(layout: str, m: int, sf_cols: int, device):
    """int64 [m, sf_cols] byte offsets of the logical scale (r, c) inside a layout's buffer."""
    import torch

    rows = torch.arange(m, device=device, dtype=torch.int64)[:, None]
    cols = torch.arange(sf_cols, device=device, dtype=torch.int64)[None, :]
    pad = padded_sf_cols(sf_cols)
    if layout == "linear":
        return rows * sf_cols + cols
    if layout == "128x4":
        return (rows // 128) * (128 * pad) + (cols // 4) * 512 + (rows % 32) * 16 + ((rows % 128) // 32) * 4 + cols % 4
    if layout == "8x4":
        return (rows // 8) * (ceil_div(pad, 4) * 32) + (cols // 4) * 32 + (rows % 8) * 4 + cols % 4
    raise ValueError(f"unknown sf layout {layout!r}")


def logical_scale_bytes(sf, m: int, sf_cols: int, layout: str):
    return sf.reshape(-1)[sf_offsets(layout, m, sf_cols, sf.device)]


def unpack_e2m1(packed):
    """uint8 [m, k/2] -> float32 [m, k]; the low nibble holds the even element."""
    import torch

    m = packed.shape[0]
    nibbles = torch.stack((packed & 0x0F, packed >> 4), dim=-1).reshape(m, 2 * packed.shape[1]).long()
    table = torch.tensor(E2M1_TABLE, device=packed.device, dtype=torch.float32)
    return table[nibbles]


def dequantize(packed, sf, layout: str, *, block_size: int = 16, scale_format: str = "e4m3", global_scale=1.0):
    """value = e2m1 * scale (E4M3 scale divided by the global encode scale, or 2**(UE8M0 - 127))."""
    import torch

    values = unpack_e2m1(packed)
    m, k = values.shape
    raw = logical_scale_bytes(sf, m, k // block_size, layout)
    if scale_format == "e4m3":
        scales = raw.view(torch.float8_e4m3fn).float() / float(global_scale)
    else:
        scales = torch.pow(2.0, raw.int() - 127)
    return (values.view(m, -1, block_size) * scales[..., None]).reshape(m, k)


def dequantized_matmul_fp32(A_fp4, B_fp4, A_sf, B_sf, alpha: float, *, row_chunk: int = 2048):
    """bf16 [M, N] of alpha * dequantize(A) @ dequantize(B)^T in fp32 with TF32 off, on the device of
    the operands: the checker the GEMM is held to at sizes a CPU oracle cannot afford in full.  A is
    decoded in row chunks so that the temporaries stay small beside the operands."""
    import torch

    M, N = A_fp4.shape[0], B_fp4.shape[0]
    k = A_fp4.shape[1] * 2
    tf32 = torch.backends.cuda.matmul.allow_tf32
    precision = torch.get_float32_matmul_precision()
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.set_float32_matmul_precision("highest")
    try:
        b = torch.empty(N, k, dtype=torch.float32, device=B_fp4.device)
        sf_b = logical_scale_bytes(B_sf, N, k // 16, "128x4").view(torch.float8_e4m3fn)
        for r0 in range(0, N, row_chunk):
            r1 = min(N, r0 + row_chunk)
            b[r0:r1] = (unpack_e2m1(B_fp4[r0:r1]).view(r1 - r0, -1, 16) * sf_b[r0:r1].float()[..., None]).reshape(r1 - r0, k)
        out = torch.empty(M, N, dtype=torch.bfloat16, device=A_fp4.device)
        sf_a = logical_scale_bytes(A_sf, M, k // 16, "128x4").view(torch.float8_e4m3fn)
        for r0 in range(0, M, row_chunk):
            r1 = min(M, r0 + row_chunk)
            a = (unpack_e2m1(A_fp4[r0:r1]).view(r1 - r0, -1, 16) * sf_a[r0:r1].float()[..., None]).reshape(r1 - r0, k)
            out[r0:r1] = (torch.mm(a, b.t()) * float(alpha)).to(torch.bfloat16)
        return out
    finally:
        torch.backends.cuda.matmul.allow_tf32 = tf32
        torch.set_float32_matmul_precision(precision)


def tensor_spec(name: str, dtype: str, shape, optional: bool = False) -> tuple:
    """One argument of an executable: its name, dtype, shape (a tuple, or an int: that many elements, -1: any number), whether
    it may be None."""
    import torch

    return name, getattr(torch, dtype), shape, optional


_torch = None


def require_tensors(specs, tensors) -> int:
    """ValueError unless every tensor is what its spec says, contiguous and on the current device; returns that device."""
    global _torch
    if _torch is None:
        import torch

        _torch = torch
    device = _torch._C._cuda_getDevice() if _torch.cuda.is_initialized() else -2  # no device yet: no tensor is there
    for spec, t in zip(specs, tensors):
        _, dtype, shape, optional = spec
        if t is None and optional:
            continue
        try:
            if (t.dtype is dtype and t.get_device() == device and t.is_contiguous()
                    and (t.shape == shape if shape.__class__ is tuple else shape < 0 or t.numel() == shape)):
                continue
        except AttributeError:
            pass
        _refuse(spec, t, device)
    return device


def _refuse(spec, t, device: int):
    import torch

    name, dtype, shape, _ = spec
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if isinstance(shape, tuple) and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if isinstance(shape, int) and 0 <= shape != t.numel():
        raise ValueError(f"{name} must have {shape} elements, got {t.numel()}")
    if not t.is_cuda:
        raise ValueError(f"{name}: all tensors must be CUDA tensors")
    if not t.is_contiguous():
        raise ValueError(f"{name}: all tensors must be contiguous")
    raise ValueError(f"{name} is on {t.device}, but the current device is cuda:{device}")


def grouped_sf_numel(rows: int, groups: int, k: int) -> int:
    """Bytes of the grouped 128x4 scale layout: group g begins at tile offsets[g] // 128 + g."""
    return (rows // 128 + groups) * 128 * (k // 16)


def grouped_sf_rows(offsets, rows: int):
    """(group of every row, its row in the grouped scale tiles); rows outside every group are not meaningful."""
    import torch

    r = torch.arange(rows, device=offsets.device)
    ends = offsets.long()
    group = (torch.searchsorted(ends, r, right=True) - 1).clamp(0, offsets.numel() - 2)
    first = ends[group]
    return group, (first // 128 + group) * 128 + r - first


def dequantize_rows(packed, sf, sf_rows):
    """float64 values of packed rows whose scales are at the rows `sf_rows` of 128x4 tiles (no encode scale)."""
    import torch

    cols = packed.shape[1] // 8
    tile_rows = sf.numel() // padded_sf_cols(cols)
    scales = logical_scale_bytes(sf, tile_rows, cols, "128x4")[sf_rows].view(torch.float8_e4m3fn).double()
    values = unpack_e2m1(packed).double()
    return (values.view(values.shape[0], cols, 16) * scales[..., None]).reshape(values.shape)


def activation(v, name: str):
    """The epilogue's activations in the type of `v`."""
    from torch.nn import functional as F

    return {"none": lambda: v, "relu": lambda: F.relu(v), "gelu": lambda: F.gelu(v),
            "gelu_tanh": lambda: F.gelu(v, approximate="tanh"), "silu": lambda: F.silu(v)}[name]()


def padding_mask(m: int, sf_cols: int, layout: str, device):
    """bool mask over a swizzled buffer: True where no logical (row < m, col < sf_cols) scale lives."""
    import torch

    mask = torch.ones(sf_numel(m, sf_cols, layout), dtype=torch.bool, device=device)
    mask[sf_offsets(layout, m, sf_cols, device).reshape(-1)] = False
    return mask


def with_guard(numel: int, dtype, device, fill):
    """A tensor of `numel` elements followed by GUARD_ELEMENTS guard elements set to `fill`."""
    import torch

    backing = torch.empty(numel + GUARD_ELEMENTS, dtype=dtype, device=device)
    backing[numel:].fill_(fill)
    return backing, backing[:numel]


# ---- roofline annotation ---------------------------------------------------------------------
FALLBACK_PEAKS = {"hbm_gbs": 6650.0, "bf16_tflops": 1590.0, "bf16_tflops_sustained": 1400.0}
NOMINAL_NVFP4_TFLOPS = 9000.0  # dense; 4x the dense bf16 rate of the same tensor cores


def measured_peaks() -> tuple[dict, str]:
    """(peaks, "measured" | "fallback"): the pool's measured copy bandwidth and bf16 GEMM rate."""
    candidates = [os.environ.get("B200_MEASURED_PEAKS")] if os.environ.get("B200_MEASURED_PEAKS") else []
    here = Path(__file__).resolve()
    candidates += [str(parent / "MEASURED_PEAKS.json") for parent in here.parents[:4]]
    for candidate in candidates:
        try:
            with open(candidate) as handle:
                data = json.load(handle)
            if "hbm_gbs" in data:
                return data, "measured"
        except (OSError, ValueError):
            continue
    return dict(FALLBACK_PEAKS), "fallback"


def roofline_hbm(algorithmic_bytes: int, microseconds: float) -> dict:
    peaks, source = measured_peaks()
    achieved = algorithmic_bytes / (microseconds * 1e-6) / 1e9
    return {"bound": "hbm", "achieved": achieved, "peak": peaks["hbm_gbs"], "unit": "GB/s",
            "frac": achieved / peaks["hbm_gbs"], "peak_source": source, "algorithmic_bytes": algorithmic_bytes}


def roofline_nvfp4(flops: int, microseconds: float) -> dict:
    """Tensor roofline of the block-scaled FP4 GEMM.

    The pool measures a dense bf16 GEMM; the dense NVFP4 rate of the same tensor cores is 4x
    the bf16 rate, so the denominator is 4 x the measured bf16 burst figure.  The fraction of
    the nominal 9 PFLOP/s is reported beside it.
    """
    peaks, source = measured_peaks()
    achieved = flops / (microseconds * 1e-6) / 1e12
    peak = 4.0 * peaks["bf16_tflops"]
    return {"bound": "tensor", "achieved": achieved, "peak": peak, "unit": "TFLOP/s",
            "frac": achieved / peak, "peak_source": f"4 x {source} bf16 burst",
            "frac_of_nominal_9pf": achieved / NOMINAL_NVFP4_TFLOPS, "flops": flops}

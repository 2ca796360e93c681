"""4-bit weights with group scales and their products with a few tokens (``csrc/int4.cu``).

A weight [N, K] is kept as two values a byte along K (``pack_int4``'s order, low nibble first) in [N, K / 2]
uint8, with one scale per output channel and ``group_size`` inputs, [N, ceil(K / group_size)], in the
activations' type. Symmetric weights hold two's complement values -8 .. 7; weights with zero points hold
0 .. 15 and a uint8 zero point per group: w = scale * (value - zero).

``int4_linear`` reads the packed weight itself: its cost is the weight's bytes, a quarter of a bf16 Linear's,
for as few tokens as decoding has. On CPU the same contract is evaluated by dequantising in float32.
"""
from __future__ import annotations

import torch

from ..ops._common import dtype_code, launch, no_backward, ptr, rows2d, same_device


_SLAB = 32768  # inputs that one launch covers: longer rows go in several, their sums kept in float32


def _check_group(K: int, group_size: int) -> None:
    if group_size <= 0 or group_size % 32:
        raise ValueError(f"group size {group_size} is not a positive multiple of 32")
    if K <= 0 or K % 32 or K > 2 ** 20:
        raise ValueError(f"{K} input features: a multiple of 32 up to 2^20 is needed")
    if K > _SLAB and _SLAB % group_size:
        raise ValueError(f"group size {group_size} does not divide {_SLAB}, as more inputs than that need it to")


def _scale(wanted: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Group scales in their type. Its subnormals are far apart (f16's begin at 6e-5, where small weights lie), so these
    round up: a scale rounded down by up to half would cut the largest values off. f32's own are not used."""
    info = torch.finfo(dtype)
    least = max(info.tiny * info.eps, 2.0 ** -126)
    up = torch.ceil(wanted / least).clamp_min(1) * least
    return torch.where(wanted < info.tiny, up, wanted).to(dtype)


def quantize_int4(w: torch.Tensor, group_size: int = 128, symmetric: bool = True,
                  scale_dtype: torch.dtype = torch.bfloat16):
    """w [N, K] -> (packed [N, K / 2] uint8, scales [N, groups], zeros [N, groups] uint8 or None). The scale is
    max |w| / 7 of its group, or (max - min) / 15 with zero points (of a range that holds 0), rounded to
    ``scale_dtype`` before the values are (up, where it is subnormal there; at least 2^-126 and what the type can hold); the
    last group of a K that ``group_size`` does not divide is shorter."""
    if w.dim() != 2:
        raise ValueError(f"quantize_int4 takes a [N, K] weight, not {tuple(w.shape)}")
    N, K = w.shape
    _check_group(K, group_size)
    if scale_dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"quantize_int4: scales are bfloat16 or float16, not {scale_dtype}")
    groups = -(-K // group_size)
    x = torch.nn.functional.pad(w.detach().float(), (0, groups * group_size - K)).view(N, groups, group_size)
    if symmetric:
        scales = _scale(x.abs().amax(-1) / 7, scale_dtype)
        q = torch.round(x / scales.float()[..., None]).clamp(-8, 7)
        zeros = None
    else:
        lo, hi = x.amin(-1).clamp_max(0), x.amax(-1).clamp_min(0)
        scales = _scale((hi - lo) / 15, scale_dtype)
        z = torch.round(-lo / scales.float()).clamp(0, 15)
        q = torch.round(x / scales.float()[..., None] + z[..., None]).clamp(0, 15)
        zeros = z.to(torch.uint8)
    u = q.view(N, -1)[:, :K].to(torch.int16) & 0xF
    return (u[:, 0::2] | (u[:, 1::2] << 4)).to(torch.uint8), scales, zeros


def _check_weight(packed, scales, zeros, group_size):
    if packed.dim() != 2 or packed.dtype != torch.uint8:
        raise ValueError(f"packed int4 weight: [N, K / 2] uint8 is needed, not {tuple(packed.shape)} {packed.dtype}")
    N, K = packed.shape[0], packed.shape[1] * 2
    if N > 2 ** 30:
        raise ValueError(f"packed int4 weight: {N} output features, 2^30 are taken")
    _check_group(K, group_size)
    groups = -(-K // group_size)
    if scales.shape != (N, groups) or (zeros is not None and zeros.shape != (N, groups)):
        raise ValueError(f"int4 weight [{N}, {K}] in groups of {group_size}: scales {tuple(scales.shape)}, zeros "
                         f"{None if zeros is None else tuple(zeros.shape)}, expected {(N, groups)}")
    if zeros is not None and zeros.dtype != torch.uint8:
        raise TypeError(f"int4 zero points are uint8, not {zeros.dtype}")
    same_device(packed, scales, zeros)
    return N, K


def dequantize_int4(packed, scales, zeros=None, group_size: int = 128) -> torch.Tensor:
    """The float32 weight [N, K] that ``packed`` stands for."""
    N, K = _check_weight(packed, scales, zeros, group_size)
    q = torch.stack([packed & 0xF, packed >> 4], -1).view(N, K)
    q = (q ^ 8).float() - 8 if zeros is None else q.float() - zeros.float().repeat_interleave(group_size, 1)[:, :K]
    return q * scales.float().repeat_interleave(group_size, 1)[:, :K]


def int4_linear(x, packed, scales, zeros=None, bias=None, group_size: int = 128) -> torch.Tensor:
    """y = x @ W^T (+ bias) for x [..., K] bf16 or f16 and a packed 4-bit W (:func:`quantize_int4`); scales and
    bias are of x's type. Values are exact, products and sums f32, and y is rounded once. The weight is read once for
    every 16 tokens (8 of up to 8): for few of them. Its rows have to start on 16 bytes. Inference only."""
    N, K = _check_weight(packed, scales, zeros, group_size)
    if x.dim() == 0 or x.shape[-1] != K:
        raise ValueError(f"int4_linear: x {tuple(x.shape)} for a weight [{N}, {K}]")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"int4_linear: bias {tuple(bias.shape)} for a weight [{N}, {K}]")
    code = dtype_code("int4_linear", x, (torch.bfloat16, torch.float16) if x.is_cuda else
                      (torch.bfloat16, torch.float16, torch.float32))
    if x.dtype != torch.float32 and (scales.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype)):
        raise TypeError(f"int4_linear: scales and bias are of x's type, {x.dtype}")
    no_backward("int4_linear", x, scales, bias)
    same_device(x, packed, scales, zeros, bias)
    if not x.is_cuda:
        y = x.float() @ dequantize_int4(packed, scales, zeros, group_size).t()
        return (y if bias is None else y + bias.float()).to(x.dtype)
    if packed.stride(1) != 1 or packed.stride(0) % 16 or packed.data_ptr() % 16:
        raise ValueError("int4_linear: the packed weight's rows have to be adjacent bytes that start on 16 bytes")
    x2 = rows2d(x)
    M = x2.shape[0]
    if x2.stride(0) % 8 or x2.data_ptr() % 16:  # the kernel copies 16 bytes at a time
        x2 = x2.clone(memory_format=torch.contiguous_format)
    # held until the launch: a copy let go of earlier could be given to the next one
    scales, zeros = scales.contiguous(), None if zeros is None else zeros.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = x.new_empty((M, N))
    sums = x.new_empty((M, N), dtype=torch.float32) if K > _SLAB else None
    launch(x, "brain_int4_linear", code, x2.data_ptr(), x2.stride(0), packed.data_ptr(), packed.stride(0),
           scales.data_ptr(), ptr(zeros), ptr(bias), y.data_ptr(), ptr(sums), M, N, K, group_size)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


class Int4Linear(torch.nn.Module):
    """Inference Linear on :func:`int4_linear`. ``from_linear`` quantises a float Linear."""

    def __init__(self, packed, scales, zeros=None, bias=None, group_size: int = 128):
        super().__init__()
        self.out_features, self.in_features = _check_weight(packed, scales, zeros, group_size)
        self.group_size = group_size
        self.register_buffer("packed", packed)
        self.register_buffer("scales", scales)
        self.register_buffer("zeros", zeros)
        self.register_buffer("bias", bias)

    @classmethod
    def from_linear(cls, lin: torch.nn.Module, group_size: int = 128, symmetric: bool = True) -> "Int4Linear":
        w = lin.weight.detach()
        dt = w.dtype if w.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
        b = lin.bias.detach().to(dt) if getattr(lin, "bias", None) is not None else None
        return cls(*quantize_int4(w, group_size, symmetric, dt), b, group_size)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int4_linear(x, self.packed, self.scales, self.zeros, self.bias, self.group_size)

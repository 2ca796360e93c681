"""Helpers shared by the op modules: signatures, streams, parameter-gradient accumulation."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from .. import _native

# Signatures of the kernel entry points (see csrc/*.cu). Codes: p pointer, i int32, l int64,
# f float32, s cudaStream_t.
_native.register({
    "brain_norm_fwd": ("brain_kernels", "iplplppplplppiifs"),
    "brain_norm_bwd_partials": ("brain_kernels", "i"),
    "brain_colsum_partials": ("brain_kernels", "i"),
    "brain_colsum_bf16": ("brain_kernels", "pliipiips"),
    "brain_gemm_bf16_gelu_dual": ("brain_kernels", "plplplpliiips"),
    "brain_gemm_bf16_gelu_grad": ("brain_kernels", "plpliplpliiis"),
    "brain_norm_bwd": ("brain_kernels", "iplplpppplplppiipiis"),
    "brain_swiglu_fwd": ("brain_kernels", "plpllis"),
    "brain_swiglu_bwd": ("brain_kernels", "plplpllis"),
    "brain_gelu_fwd": ("brain_kernels", "ppls"),
    "brain_gelu_bwd": ("brain_kernels", "pppls"),
    "brain_rope": ("brain_kernels", "piiiilllppifs"),
    "brain_embedding_fwd": ("brain_kernels", "pppiplils"),
    "brain_embedding_bwd": ("brain_kernels", "ppppilils"),
    "brain_pos_grad": ("brain_kernels", "ppilii" + "s"),
    "brain_ce_fwd": ("brain_kernels", "plppplilfs"),
    "brain_ce_bwd": ("brain_kernels", "plppppfpllilfs"),
    "brain_adamw": ("brain_kernels", "pppppiplffffffffipps"),
    "brain_grad_stats": ("brain_kernels", "pilfpips"),
    "brain_step_guard": ("brain_kernels", "pfpps"),
    "brain_sgd": ("brain_kernels", "pppiplffffiifps"),
    "brain_sumsq": ("brain_kernels", "pilfpipps"),
    "brain_scale": ("brain_kernels", "pilpfs"),
    "brain_clip_coef": ("brain_kernels", "pfps"),
    "brain_cast_bf16": ("brain_kernels", "ppls"),
    "brain_attn_fwd": ("brain_kernels", "pppppppiiiiiifis"),
    "brain_attn_bwd": ("brain_kernels", "pppppppppppppppp" + "iiiiiifis"),
    "brain_attn_fwd_tc": ("brain_kernels", "pppppppiiiiiifis"),
    "brain_status_attention_tc": ("brain_kernels", "pi"),
    "brain_attn_bwd_tc": ("brain_kernels", "pppppppppppppppp" + "iiiiiifis"),
    "brain_attn_fwd_tc_masked": ("brain_kernels", "pppppppiiiiiifipps"),
    "brain_attn_bwd_tc_masked": ("brain_kernels", "pppppppppppppppp" + "iiiiiifipps"),
    "brain_status_attention_bwd_tc": ("brain_kernels", "pi"),
    "brain_status_norms": ("brain_kernels", "pi"),
    "brain_status_elementwise": ("brain_kernels", "pi"),
    "brain_status_ce": ("brain_kernels", "pi"),
    "brain_status_optim": ("brain_kernels", "pi"),
    "brain_status_attention": ("brain_kernels", "pi"),
    "brain_norm_fp8": ("brain_kernels", "iplplppppliifs"),
    "brain_distill_rows": ("brain_kernels", "iplpppppplppiiiliifps"),
    "brain_distill_count": ("brain_kernels", "ppliipis"),
    "brain_distill_reduce": ("brain_kernels", "pplpips"),
    "brain_status_distill": ("brain_kernels", "pi"),
    "brain_verify_draft": ("brain_kernels", "ipllpllpppppliis"),
    "brain_status_int4": ("brain_kernels", "pi"),
    "brain_int4_linear": ("brain_kernels", "iplplpppppiiiis"),
})

STATUS_TAGS = ["gemm", "norms", "elementwise", "ce", "optim", "attention", "attention_tc", "attention_bwd_tc",
               "attention_decode", "decode_tp", "distill", "int4"]


def same_device(ref: torch.Tensor, *others) -> None:
    """Raise unless every tensor in ``others`` (None skipped) lives on ``ref``'s device: a kernel given a
    pointer into another device's (or the host's) memory would fault."""
    device = ref.device
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"tensor on {t.device} passed to a kernel running on {ref.device}")


# codes of csrc/elem.cuh::BrainDtype
DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def dtype_code(name: str, t: torch.Tensor, allowed=(torch.bfloat16, torch.float16, torch.float32)) -> int:
    """The C code of ``t``'s type; TypeError naming the op for a type that its kernels do not take."""
    if t.dtype not in allowed:
        raise TypeError(f"{name} takes {', '.join(str(d)[6:] for d in allowed)} tensors, not {str(t.dtype)[6:]}")
    return DTYPE_CODES[t.dtype]


def launch(t: torch.Tensor, name: str, *args) -> None:
    """``_native.call`` with ``t``'s device current (a launch goes to the current device) and that device's
    current stream as the last argument."""
    index = t.get_device()
    if index == torch.cuda.current_device():
        _native.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            _native.call(name, *args, _raw_stream(index))


# the stream of a device as an integer, without the Stream object around it (2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: _native.stream_ptr(torch.device("cuda", index)))


def has_tangent(t: torch.Tensor) -> bool:
    """Whether forward-mode differentiation follows ``t``. What a kernel makes of its address would lose that."""
    # without a level there is none, and unpacking costs 0.7 us
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def no_backward(name: str, *tensors) -> None:
    """Raise when autograd, backward or forward, would record an inference op: its result would carry no derivative,
    silently."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0 and any(t is not None and has_tangent(t) for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative: call it on unpacked tensors")


def stream(t: torch.Tensor) -> int:
    return _native.stream_ptr(t.device)


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def i64_array(vals) -> ctypes.Array:
    arr = (ctypes.c_int64 * len(vals))(*[int(v) for v in vals])
    return arr


def check_status() -> list[tuple[str, int, int]]:
    """Read and clear every kernel status word; returns the non-zero entries (tag, code, where)."""
    bad = []
    for tag in STATUS_TAGS:
        code, where = _native.status(tag, clear=True)
        if code:
            bad.append((tag, code, where))
    return bad


def has_main_grad(p: torch.Tensor) -> bool:
    return getattr(p, "main_grad", None) is not None


def main_grad_beta(p: torch.Tensor) -> float:
    """Weight of the existing contents of ``p.main_grad`` for the next gradient written into it: 0.0
    for the first write since the flat buffer's ``zero_grad`` (which marks parameters instead of
    clearing memory, so the first producer overwrites), 1.0 afterwards (accumulate)."""
    if getattr(p, "_main_grad_fresh", False):
        p._main_grad_fresh = False
        return 0.0
    return 1.0


def rows2d(x: torch.Tensor) -> torch.Tensor:
    """View x as [rows, last] with unit last-dim stride (copying only if needed)."""
    if x.dim() == 2 and x.stride(1) == 1 and x.shape[1] > 0:  # reshape refuses rows without values
        return x
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    return x2

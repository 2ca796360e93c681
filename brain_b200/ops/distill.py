"""Distillation from a teacher's stored top logits (``csrc/distill.cu``).

A teacher that was run once keeps, for each token, its k largest logits and their ids. With temperature T,
p = softmax(teacher_logits / T) over the kept entries and q = softmax(logits / T) over the whole vocabulary,

    loss = T^2 * sum_i p_i (log p_i - log q_{id_i}),    dloss/dlogits = T (q - p at its ids).

``topk_distillation`` is the loss with autograd: its backward pass reads the logits again.
``topk_distillation_grad`` gives loss and gradient of one pass over the logits, for a loop that drives the
backward pass itself (``logits.backward(grad)``), in place if asked to. ``linear_topk_distillation`` is the LM
head: like ``linear_cross_entropy`` it turns its one [tokens, vocab] buffer of logits into their gradient.

An id of -1 is no entry (teachers that keep fewer than k), nor is a logit of -inf; a token without entries has
loss and gradient 0 and does not count in the mean. On CUDA an id at or above the vocabulary's size is taken as
no entry and recorded in the status words (``ops.check_status``); on the CPU it raises.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._common import DTYPE_CODES, dtype_code, has_main_grad, has_tangent, launch, main_grad_beta, ptr, rows2d, same_device
from .gemm import gemm

MAX_TOP = 1024


def _check(name, logits, teacher_logits, teacher_ids, temperature, reduction):
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unknown reduction {reduction!r}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{name}: temperature {temperature} is not in [1e-6, 1e6]")
    shape, kept = logits.shape, teacher_ids.shape
    if not shape or not 0 < shape[-1] <= 2 ** 30:
        raise ValueError(f"{name}: logits {tuple(shape)} have no vocabulary dimension of 1 to 2^30 ids")
    if teacher_logits.shape != kept or len(kept) != len(shape) or kept[:-1] != shape[:-1]:
        raise ValueError(f"{name}: logits {tuple(shape)}, teacher_logits {tuple(teacher_logits.shape)}, "
                         f"teacher_ids {tuple(kept)}")
    if not 1 <= kept[-1] <= MAX_TOP:
        raise ValueError(f"{name}: {kept[-1]} teacher entries a token, 1 to {MAX_TOP} are taken")
    if teacher_ids.dtype is not torch.int64 and (
            teacher_ids.is_floating_point() or teacher_ids.is_complex() or teacher_ids.dtype is torch.bool):
        raise TypeError(f"{name}: teacher_ids are whole numbers")
    if teacher_logits.dtype is not torch.float32 and not teacher_logits.is_floating_point():
        raise TypeError(f"{name}: teacher_logits are floating-point numbers")
    if teacher_logits.requires_grad and torch.is_grad_enabled() or has_tangent(teacher_logits):
        raise RuntimeError(f"{name} gives the teacher no gradient: detach teacher_logits")
    same_device(logits, teacher_logits, teacher_ids)


def _teacher(teacher_logits, teacher_ids):
    """The entries as contiguous float32 and int64 (their leading dimensions do not matter to the kernels)."""
    t, ids = teacher_logits, teacher_ids
    if t.dtype is not torch.float32 or not t.is_contiguous():
        t = t.float().contiguous()
    if ids.dtype is not torch.int64 or not ids.is_contiguous():
        ids = ids.long().contiguous()
    return t, ids


def _rows(l2, t, ids, temperature, loss, lse, counts, dz, grad=None, n=None, parts=0, grad_rows=0, count=0, total=None):
    """All but logits, entries and ``dz`` are addresses; those of empty tensors are None or never used."""
    launch(l2, "brain_distill_rows", DTYPE_CODES[l2.dtype], l2.data_ptr(), l2.stride(0), t.data_ptr(), ids.data_ptr(),
           loss, lse, counts, ptr(dz), 0 if dz is None else dz.stride(0), grad, n, parts, count, grad_rows, l2.shape[0],
           t.shape[-1], l2.shape[1], temperature, total)


def _parts(M):
    """In how many parts the tokens that have an entry are counted."""
    return min(max(-(-M // 256), 1), 128)


def _loss(l2, t, ids, temperature, reduction):
    """The loss, and a buffer whose second and last parts the backward pass reads: losses [M], log-sum-exps [M], which
    tokens count [M], how many do [1] (an int32)."""
    M = l2.shape[0]
    own = t.new_empty(3 * M + 1)
    at = own.data_ptr()
    if reduction == "none":
        loss = t.new_empty(M)
        _rows(l2, t, ids, temperature, loss.data_ptr(), at + 4 * M, None, None)
        return loss, own
    total = t.new_empty(())
    mean = reduction == "mean"
    _rows(l2, t, ids, temperature, at, at + 4 * M, at + 8 * M if mean else None, None, None, at + 12 * M if mean else None,
          1 if mean else 0, total=total.data_ptr())
    return total, own


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, t, ids, temperature, reduction):
        loss, own = _loss(rows2d(logits), t, ids, temperature, reduction)
        ctx.save_for_backward(logits, t, ids, own)
        ctx.meta = temperature, reduction
        return loss.view(logits.shape[:-1]) if reduction == "none" else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, t, ids, own = ctx.saved_tensors
        temperature, reduction = ctx.meta
        l2 = rows2d(logits)
        M = l2.shape[0]
        out = torch.empty_like(l2, memory_format=torch.contiguous_format)
        if g.dtype is not torch.float32 or not g.is_contiguous():
            g = g.float().contiguous()
        at = own.data_ptr()
        mean = reduction == "mean"
        _rows(l2, t, ids, temperature, None, at + 4 * M, None, out, g.data_ptr(), at + 12 * M if mean else None,
              1 if mean else 0, 1 if reduction == "none" else 0)
        return out if l2 is logits else out.view(logits.shape), None, None, None, None


def topk_distillation_ref(logits, teacher_logits, teacher_ids, temperature=1.0, reduction="mean"):
    """Torch operations in float32 (float64 for float64 logits), differentiable."""
    ct = torch.float64 if logits.dtype == torch.float64 else torch.float32
    V = logits.shape[-1]
    if teacher_ids.numel() and int(teacher_ids.max()) >= V:
        raise ValueError(f"teacher id {int(teacher_ids.max())} outside the vocabulary of {V}")
    t = teacher_logits.detach().to(ct)
    on = (teacher_ids >= 0) & (t != float("-inf"))
    t = (t / temperature).clamp_min(torch.finfo(ct).min)  # one that overflows is still an entry
    some = on.any(-1)
    t = torch.where(on, t, torch.full_like(t, float("-inf")))
    t = torch.where(some[..., None], t, torch.zeros_like(t))
    logp = torch.log_softmax(t, -1)
    p = torch.where(on, logp.exp(), torch.zeros_like(logp))
    logq = torch.log_softmax(logits.to(ct) / temperature, -1).gather(-1, teacher_ids.long().clamp_min(0))
    used = on & (p != 0)
    loss = torch.where(used, p * (torch.where(used, logp, 0.0) - torch.where(used, logq, 0.0)), 0.0).sum(-1)
    loss = loss * temperature ** 2
    if reduction == "none":
        return loss
    return loss.sum() / some.sum().clamp_min(1) if reduction == "mean" else loss.sum()


def topk_distillation(logits, teacher_logits, teacher_ids, temperature: float = 1.0, reduction: str = "mean"):
    """Distillation loss of ``logits`` [..., V] against a teacher's kept ``teacher_logits`` [..., k] at
    ``teacher_ids`` [..., k] (any order, at most 1024 of them); float32. ``"mean"`` is over the tokens that have
    an entry, ``"none"`` gives the loss of each. To capture its backward pass into a CUDA graph, let go of every
    eager loss of the same leaf first: autograd ties a leaf to the stream of its oldest living graph."""
    _check("topk_distillation", logits, teacher_logits, teacher_ids, temperature, reduction)
    if not logits.is_cuda:
        return topk_distillation_ref(logits, teacher_logits, teacher_ids, temperature, reduction)
    dtype_code("topk_distillation", logits)
    t, ids = _teacher(teacher_logits, teacher_ids)
    if torch.is_grad_enabled() and logits.requires_grad or has_tangent(logits):  # which raises for the latter
        return _DistillFn.apply(logits, t, ids, float(temperature), reduction)
    loss = _loss(rows2d(logits), t, ids, float(temperature), reduction)[0]
    return loss.view(logits.shape[:-1]) if reduction == "none" else loss


def _apart(out, logits):
    """Whether every element of ``out`` is its own, and none is another element of ``logits``."""
    span = 1
    for size, stride in sorted(zip(out.shape, out.stride()), key=lambda x: x[1]):
        if size > 1 and stride < span:
            return False
        span += (size - 1) * stride
    if out.numel() == 0 or out.untyped_storage().data_ptr() != logits.untyped_storage().data_ptr() \
            or (out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()):
        return True
    size = out.element_size()
    other = 1 + sum((n - 1) * s for n, s in zip(logits.shape, logits.stride()))
    lo, lo2 = out.data_ptr(), logits.data_ptr()
    return lo + span * size <= lo2 or lo2 + other * size <= lo


def _plain(out):
    """``out`` for the caller, without the history that it may have as logits."""
    return out.detach() if out.requires_grad else out


def _written(out, given):
    """What was written by address into a caller's tensor is told to autograd: a graph that saved its values raises in
    its backward pass, as after any write in place."""
    if given and not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return _plain(out)


def topk_distillation_grad(logits, teacher_logits, teacher_ids, temperature: float = 1.0, reduction: str = "mean",
                           out: torch.Tensor | None = None):
    """(loss, dloss/dlogits) of :func:`topk_distillation` (with ``"none"`` the gradient of the losses' sum),
    outside autograd. ``out`` takes the gradient: of logits' shape and type with adjacent columns, or logits
    itself, whose own history stays (``logits.backward(grad)``); autograd sees the write, so a graph that saved the
    values of ``out`` raises in its backward pass."""
    name = "topk_distillation_grad"
    _check(name, logits, teacher_logits, teacher_ids, temperature, reduction)
    if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or out.stride(-1) != 1):
        raise ValueError(f"{name}: out {tuple(out.shape)} {out.dtype} for logits {tuple(logits.shape)} {logits.dtype}")
    same_device(logits, out)
    if out is not None and not _apart(out, logits):
        raise ValueError(f"{name}: out shares memory with itself or with logits without being logits")
    if not logits.is_cuda:
        with torch.inference_mode(False), torch.enable_grad():
            z = (logits.clone() if logits.is_inference() else logits).detach().requires_grad_()
            loss = topk_distillation_ref(z, teacher_logits, teacher_ids, temperature, reduction)
            grad = torch.autograd.grad(loss.sum(), z)[0]
        if out is not None:
            out.detach().copy_(grad)
        return loss.detach(), grad if out is None else _plain(out)
    dtype_code(name, logits)
    if logits.requires_grad:
        logits = logits.detach()
    t, ids = _teacher(teacher_logits, teacher_ids)
    l2 = rows2d(logits)
    given = out is not None
    if not given:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    o2 = out if out.dim() == 2 else out.detach().view(-1, out.shape[-1])
    M = l2.shape[0]
    if reduction == "none":
        loss = t.new_empty(M)
        _rows(l2, t, ids, float(temperature), loss.data_ptr(), None, None, o2)
        return loss.view(logits.shape[:-1]), _written(out, given)
    total, parts = t.new_empty(()), _parts(M) if reduction == "mean" else 0
    own = t.new_empty(M + parts)  # the losses, then numbers of the tokens that have an entry (int32)
    at = own.data_ptr()
    _rows(l2, t, ids, float(temperature), at, None, None, o2, None, at + 4 * M if parts else None, parts,
          count=1 if parts else 0, total=total.data_ptr())
    return total, _written(out, given)


class _LinearDistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, t, ids, temperature, chunk):
        h2 = rows2d(h)
        M, V = h2.shape[0], w.shape[0]
        chunk = min(chunk, M) if chunk else M
        dlogits = torch.empty(M, -(-V // 8) * 8, device=h.device, dtype=torch.bfloat16)[:, :V]  # 16-byte rows
        loss = torch.empty(M, device=h.device, dtype=torch.float32)
        k = t.shape[-1]
        t, ids = t.view(M, k), ids.view(M, k)
        n = t.new_empty(_parts(M), dtype=torch.int32)
        launch(t, "brain_distill_count", t.data_ptr(), ids.data_ptr(), M, k, V, n.data_ptr(), n.numel())
        for s0 in range(0, M, max(chunk, 1)):
            rows = slice(s0, min(M, s0 + chunk))
            gemm(h2[rows], w, trans_b=True, out=dlogits[rows])
            _rows(dlogits[rows], t[rows], ids[rows], temperature, loss[rows].data_ptr(), None, None, dlogits[rows], None,
                  n.data_ptr(), n.numel())
        ctx.save_for_backward(h2, w, dlogits)
        ctx.hshape = h.shape
        total = loss.new_empty(())
        launch(loss, "brain_distill_reduce", loss.data_ptr(), None, M, n.data_ptr(), n.numel(), total.data_ptr())
        return total

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        h2, w, dlogits = ctx.saved_tensors
        alpha = float(g)  # scalar loss: fold the upstream gradient into the GEMM alpha
        dh = gemm(dlogits, w, alpha=alpha).view(ctx.hshape) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            if has_main_grad(w):
                gemm(dlogits, h2, trans_a=True, out=w.main_grad, beta=main_grad_beta(w), alpha=alpha)
            else:
                dw = gemm(dlogits, h2, trans_a=True, out_dtype=torch.float32, alpha=alpha).to(w.dtype)
        return dh, dw, None, None, None, None


def linear_topk_distillation(h, w, teacher_logits, teacher_ids, temperature: float = 1.0, chunk: int = 0):
    """Mean :func:`topk_distillation` of the logits ``h @ w.T`` (h [..., D], w [V, D], bf16 on CUDA), with the
    logits held once and turned into their gradient in place, optionally ``chunk`` tokens at a time."""
    if h.shape[-1] != w.shape[-1] or w.dim() != 2 or h.dim() < 1:
        raise ValueError(f"linear_topk_distillation: h {tuple(h.shape)}, w {tuple(w.shape)}")
    if chunk < 0:
        raise ValueError(f"linear_topk_distillation: chunk {chunk}")
    _check("linear_topk_distillation", h, teacher_logits, teacher_ids, temperature, "mean")
    same_device(h, w)
    if not h.is_cuda:
        logits = torch.nn.functional.linear(h.float(), w.float())
        return topk_distillation_ref(logits, teacher_logits, teacher_ids, temperature)
    for x in (h, w):
        dtype_code("linear_topk_distillation", x, (torch.bfloat16,))
    t, ids = _teacher(teacher_logits, teacher_ids)
    with torch.cuda.device(h.device):  # the GEMM launches on the current one
        return _LinearDistillFn.apply(h, w, t, ids, float(temperature), chunk)

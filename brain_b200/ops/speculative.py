"""Verification of drafted tokens (``csrc/verify.cu``), the step of speculative decoding that decides how many
tokens of a cheap draft the target model keeps, and draws the one that follows.
"""
from __future__ import annotations

import torch

from ._common import dtype_code, launch, ptr, same_device


def verify_draft(target_probs, draft_tokens, uniforms, draft_probs=None, draft_lens=None):
    """Which drafted tokens the target's probabilities accept -> (tokens [B, K + 1], accepted [B]), int64.

    ``target_probs`` [B, K + 1, V] (up to 65535 sequences and 2^30 ids): the target's probabilities after the
    context and each drafted token; ``draft_tokens`` [B, K]; ``draft_probs`` [B, K, V]: what each token was drawn from (None: the draft was
    certain of its tokens); ``draft_lens`` [B]: how many of the K were drafted (None: all); ``uniforms``
    [B, K + 1] in [0, 1): one number a drafted token, the last for the token that follows.

    Token i is accepted while ``uniforms[i] * q_i < p_i``. Row b of ``tokens`` holds the accepted tokens, then
    one drawn from max(p - q, 0) at the first refusal (from p where that is empty, or where nothing was
    refused) as the first id whose running sum exceeds ``uniforms[b, K]`` times the whole, then -1. Sums are
    taken in 64 bits. Probabilities need not sum to one; negative, infinite and NaN ones count as 0 throughout (so a
    token without any probability of the target's is refused, whatever the draft's), a drafted id outside the
    vocabulary is refused, and a row without any weight gives token -1."""
    if target_probs.dim() != 3 or draft_tokens.dim() != 2:
        raise ValueError("verify_draft takes target_probs [B, K + 1, V] and draft_tokens [B, K]")
    B, K1, V = target_probs.shape
    K = K1 - 1
    if not 0 < V <= 2 ** 30 or K < 0 or B > 65535 or draft_tokens.shape != (B, K) or uniforms.shape != (B, K1):
        raise ValueError(f"verify_draft: target_probs {tuple(target_probs.shape)}, draft_tokens "
                         f"{tuple(draft_tokens.shape)}, uniforms {tuple(uniforms.shape)}")
    if draft_probs is not None and draft_probs.shape != (B, K, V):
        raise ValueError(f"verify_draft: draft_probs {tuple(draft_probs.shape)}, expected {(B, K, V)}")
    if draft_lens is not None and draft_lens.shape != (B,):
        raise ValueError(f"verify_draft: draft_lens {tuple(draft_lens.shape)}, expected {(B,)}")
    code = dtype_code("verify_draft", target_probs)
    if draft_probs is not None and draft_probs.dtype != target_probs.dtype:
        raise TypeError("verify_draft: target_probs and draft_probs are of one type")
    for t in (draft_tokens, draft_lens):
        if t is not None and (t.is_floating_point() or t.is_complex() or t.dtype == torch.bool):
            raise TypeError("verify_draft: token ids and lengths are whole numbers")
    if uniforms.dtype != torch.float32:
        raise TypeError("verify_draft: uniforms are float32")
    same_device(target_probs, draft_tokens, uniforms, draft_probs, draft_lens)
    if not target_probs.is_cuda:
        return verify_draft_ref(target_probs, draft_tokens, uniforms, draft_probs, draft_lens)
    p = target_probs if target_probs.stride(2) == 1 else target_probs.contiguous()
    q = draft_probs
    if q is not None and q.stride(2) != 1:
        q = q.contiguous()
    drafted = draft_tokens if draft_tokens.dtype == torch.int64 else draft_tokens.long()
    drafted = drafted.contiguous()
    lens = draft_lens
    if lens is not None:
        lens = (lens if lens.dtype == torch.int32 else lens.long().clamp(0, K).int()).contiguous()
    u = uniforms.contiguous()
    tokens = drafted.new_empty((B, K1))
    count = drafted.new_empty(B)
    ps, qs = p.stride(), (0, 0) if q is None else q.stride()
    launch(p, "brain_verify_draft", code, p.data_ptr(), ps[0], ps[1], ptr(q), qs[0], qs[1], drafted.data_ptr(),
           ptr(lens), u.data_ptr(), tokens.data_ptr(), count.data_ptr(), B, K, V)
    return tokens, count


def verify_draft_ref(target_probs, draft_tokens, uniforms, draft_probs=None, draft_lens=None):
    """The same, a sequence at a time in float64 torch operations."""
    B, K1, V = target_probs.shape
    K = K1 - 1
    u = uniforms.double()
    tokens = torch.full((B, K1), -1, dtype=torch.int64, device=target_probs.device)
    count = torch.zeros(B, dtype=torch.int64, device=target_probs.device)

    def weights(t):
        t = t.double()
        return torch.where((t > 0) & (t < float("inf")), t, torch.zeros_like(t))

    for b in range(B):
        n, length = 0, K if draft_lens is None else min(max(int(draft_lens[b]), 0), K)
        while n < length:
            x = int(draft_tokens[b, n])
            if not 0 <= x < V:
                break
            q = 1.0 if draft_probs is None else float(weights(draft_probs[b, n, x]))
            if not float(u[b, n]) * q < float(weights(target_probs[b, n, x])):
                break
            tokens[b, n] = x
            n += 1
        w = weights(target_probs[b, n])
        if n < length:
            if draft_probs is not None:
                left = (w - weights(draft_probs[b, n])).clamp_min(0)
            else:
                left = w.clone()
                if 0 <= int(draft_tokens[b, n]) < V:
                    left[int(draft_tokens[b, n])] = 0
            w = left if bool((left > 0).any()) else w
        some = (w > 0).nonzero()
        if len(some):
            sums = w.cumsum(0)
            over = (sums > u[b, K] * sums[-1]).nonzero()
            tokens[b, n] = over[0, 0] if len(over) else some[-1, 0]
        count[b] = n
    return tokens, count

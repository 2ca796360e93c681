"""The operators of speculative serving together: a draft model's head learns from a target's kept logits, is cut to
4 bits, drafts tokens; the target reads them through its fp8 head and verifies them."""
import pytest
import torch

from brain_b200 import ops
from brain_b200 import quantization as Q

D, V, K, TOP = 256, 1024, 4, 32


def target_probs(h, r, norm, head):
    """The target's probabilities of [B, n, D] states: residual, norm and projection in e4m3."""
    q, scale, s = ops.add_rms_norm_fp8(h, r, norm, 1e-5)
    y = Q.fp8_gemm_rowwise(q.view(-1, D), scale.view(-1), *head)
    return torch.softmax(y.float(), -1).view(*h.shape[:-1], V), s


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_train_draft_verify(device):
    g = torch.Generator().manual_seed(0)

    def rnd(*shape):
        return torch.randn(*shape, generator=g).to(device).bfloat16()

    norm, weight = (1 + 0.1 * rnd(D)).bfloat16(), rnd(V, D) * 0.1
    head = Q.quantize_fp8_rowwise(weight)
    # what the teacher kept of 512 tokens, and the draft's gradient from it
    h, r = rnd(4, 128, D), rnd(4, 128, D)
    teacher, s = target_probs(h, r, norm, head)
    kept = torch.topk(teacher.log(), TOP)
    draft_w = rnd(V, D) * 0.02
    states = ops.rms_norm(s, norm, 1e-5)
    for step in range(2):
        w = draft_w.detach().requires_grad_()
        loss = ops.linear_topk_distillation(states, w, kept.values, kept.indices, 2.0)
        loss.backward()
        assert torch.isfinite(loss) and torch.isfinite(w.grad).all() and (w.grad != 0).any()
        draft_w = (w - 5.0 * w.grad).detach().bfloat16()
    # the draft's head in 4 bits proposes K tokens for each of 6 sequences
    small = Q.Int4Linear(*Q.quantize_int4(draft_w, 64), group_size=64).to(device)
    h, r = rnd(6, K + 1, D), rnd(6, K + 1, D)
    p, s = target_probs(h, r, norm, head)
    with torch.no_grad():
        q = torch.softmax(small(ops.rms_norm(s[:, :K].contiguous(), norm, 1e-5)).float(), -1)
    x = torch.multinomial(q.cpu().view(-1, V), 1, generator=g).view(6, K).to(device)
    u = torch.rand(6, K + 1, generator=g).to(device)
    lens = torch.tensor([4, 4, 3, 1, 0, 4], device=device)
    tokens, n = ops.verify_draft(p, x, u, q, lens)
    want = ops.verify_draft(p.cpu(), x.cpu(), u.cpu(), q.cpu(), lens.cpu())
    assert torch.equal(tokens.cpu(), want[0]) and torch.equal(n.cpu(), want[1])
    assert (n <= lens).all()
    at = torch.arange(K + 1, device=device)
    assert ((tokens >= 0) == (at <= n[:, None])).all() and (tokens < V).all()
    assert ops.check_status() == [] if device == "cuda" else True

"""Distillation from a teacher's kept logits: loss and gradient against the formula in 64 bits and differences."""
import math
import threading

import pytest
import torch

from brain_b200 import _native, losses, ops
from brain_b200.models import LlamaLite, LlamaLiteConfig

gpu = pytest.mark.gpu
INF = float("inf")


def data(rows, V, k, dtype, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, V, generator=g) * scale).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(rows)]) if rows else torch.zeros(0, k, dtype=torch.long)
    t = torch.randn(rows, k, generator=g) * 3 + 5
    return z, t, ids


def formula(z, t, ids, T):
    """Row losses, their gradients, which rows count and the size of what a gradient adds up, in 64 bits, entry by
    entry."""
    z = z.double()
    rows, V = z.shape
    loss, grad, some = torch.zeros(rows).double(), torch.zeros(rows, V).double(), torch.zeros(rows, dtype=torch.bool)
    size = torch.zeros(rows, V).double()
    for r in range(rows):
        keep = [(int(i), float(v) / T) for i, v in zip(ids[r], t[r]) if i >= 0 and v != -INF]
        if not keep:
            continue
        some[r] = True
        top = max(v for _, v in keep)
        total = sum(math.exp(v - top) for _, v in keep)
        lse = torch.logsumexp(z[r] / T, 0)
        grad[r] = torch.exp(z[r] / T - lse)
        size[r] = grad[r]
        for i, v in keep:
            p = math.exp(v - top) / total
            if p:
                loss[r] += p * (v - top - math.log(total) - (z[r, i] / T - lse))
            grad[r, i] -= p
            size[r, i] += p
    return loss * T * T, grad * T, some, size * T


def reduced(loss, grad, some, reduction):
    n = max(1, int(some.sum())) if reduction == "mean" else 1
    return (loss if reduction == "none" else loss.sum() / n), grad / n


def tolerances(z, grad, size, T, dtype):
    """f32: an argument of 2^x off by 3 roundings of its size f, 2^x by 2^-22, up to 64 roundings in the sums; a
    loss adds terms of size f. A gradient is rounded by half a step of its type; f16 ends at 2^-24, f32 at 2^-126."""
    f = z.double().abs()
    f = float(f[f < INF].max()) / T * 1.5 + 20 if f.numel() else 20
    rel = (3 * f + 64) * 2.0 ** -24
    return T * T * rel * f, torch.finfo(dtype).eps / 2 * grad.abs() + rel * size + \
        (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -125)


def check(got_loss, got_grad, z, t, ids, T, reduction, dtype):
    loss, grad, some, size = formula(z, t, ids, T)
    want, grad = reduced(loss, grad, some, reduction)
    n = max(1, int(some.sum())) if reduction == "mean" else 1
    tl, tg = tolerances(z, grad, size / n, T, dtype)
    if reduction == "sum":
        tl *= max(1, z.shape[0])
    assert got_loss.dtype == torch.float32 and got_loss.shape == want.shape
    assert ((got_loss.detach().cpu().double() - want).abs() <= tl).all(), (got_loss, want, tl)
    if got_grad is not None:
        assert got_grad.dtype == dtype
        assert ((got_grad.cpu().double() - grad).abs() <= tg).all(), ((got_grad.cpu().double() - grad).abs() / tg).max()
        assert (got_grad.cpu()[~some] == 0).all()


# ------------------------------------------------------------------ CPU
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("T", [1.0, 2.5])
def test_cpu_path(reduction, T):
    z, t, ids = data(6, 40, 5, torch.float32)
    ids[1, 2:] = -1
    ids[2] = -1
    t[3] = -INF
    ids[4, 3] = ids[4, 0]  # one id twice
    z.requires_grad_()
    loss = ops.topk_distillation(z, t, ids, T, reduction)
    (grad,) = torch.autograd.grad(loss.sum(), z)
    check(loss, grad, z.detach(), t, ids, T, reduction, torch.float32)
    both = ops.topk_distillation_grad(z.detach(), t, ids, T, reduction)
    assert torch.equal(both[0], loss) and torch.equal(both[1], grad)


def test_gradient_against_differences():
    z, t, ids = data(4, 30, 6, torch.float64)
    ids[1] = -1
    ids[2, 4] = ids[2, 1]
    z.requires_grad_()
    assert torch.autograd.gradcheck(lambda v: ops.topk_distillation(v, t, ids, 1.7), (z,))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_teacher_masked_with_the_lowest_value(device, reduction):
    # below one, the temperature takes it out of f32's range: an entry all the same, where it is the only one
    z, t, ids = data(4, 40, 5, torch.float32)
    t[0, 1:] = t[1] = torch.finfo(torch.float32).min
    ids[1, 1:] = -1
    ids[2] = -1
    loss, grad = ops.topk_distillation_grad(z.to(device), t.to(device), ids.to(device), 0.5, reduction)
    check(loss, grad, z, t, ids, 0.5, reduction, torch.float32)
    v = z.to(device).requires_grad_()
    loss = ops.topk_distillation(v, t.to(device), ids.to(device), 0.5, reduction)
    (grad,) = torch.autograd.grad(loss.sum(), v)
    check(loss, grad, z, t, ids, 0.5, reduction, torch.float32)


def test_is_distillation_loss_when_everything_is_kept():
    z, teacher = torch.randn(5, 16), torch.randn(5, 16)
    ids = torch.arange(16).expand(5, 16)
    want = losses.DistillationLoss(2.0)(z, teacher)
    torch.testing.assert_close(losses.TopKDistillationLoss(2.0)(z, teacher, ids), want)
    labels = torch.randint(0, 16, (5,))
    torch.testing.assert_close(losses.TopKDistillationLoss(2.0, 0.3)(z, teacher, ids, labels),
                               losses.DistillationLoss(2.0, 0.3)(z, teacher, labels))
    assert losses.LOSSES["TopKDistillationLoss"] is losses.TopKDistillationLoss


def test_refusals():
    z, t, ids = data(3, 20, 4, torch.float32)
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=INF), dict(temperature=math.nan),
                dict(reduction="batchmean")):
        with pytest.raises(ValueError):
            ops.topk_distillation(z, t, ids, **bad)
    for temperature in (1e-7, 1e-50, 1e7):
        with pytest.raises(ValueError):
            ops.topk_distillation(z, t, ids, temperature)
    with pytest.raises(ValueError):
        ops.topk_distillation(z[:1, :1].expand(1, 2 ** 30 + 1), t[:1], ids[:1])
    for a in ((z, t[:, :3], ids), (z[:2], t, ids), (z, t[:, :0], ids[:, :0]), (z[:, :0], t, ids), (z[None], t, ids),
              (z, t.repeat(1, 300), ids.repeat(1, 300))):
        with pytest.raises(ValueError):
            ops.topk_distillation(*a)
    with pytest.raises(TypeError):
        ops.topk_distillation(z, t, ids.float())
    with pytest.raises(TypeError):
        ops.topk_distillation(z, t.long(), ids)
    with pytest.raises(ValueError):
        ops.topk_distillation(z, t, ids + 20)
    with pytest.raises(RuntimeError):
        ops.topk_distillation(z, t.clone().requires_grad_(), ids)
    with pytest.raises(ValueError):
        ops.topk_distillation_grad(z, t, ids, out=torch.empty(3, 21))
    both = torch.zeros(7, 20)
    both[:3] = z
    for out in (both[1:4], torch.empty(1, 20).expand(3, 20), both[:3].t().reshape(3, 20).t().t()[:, :0]):
        with pytest.raises(ValueError):
            ops.topk_distillation_grad(both[:3], t, ids, out=out)
    want = ops.topk_distillation_grad(z, t, ids)[1]
    assert torch.equal(ops.topk_distillation_grad(both[:3], t, ids, out=both[3:6])[1], want)
    assert torch.equal(ops.topk_distillation_grad(both[:3], t, ids, out=both[:3])[1], want)
    with pytest.raises(ValueError):
        ops.linear_topk_distillation(torch.randn(3, 8), torch.randn(20, 9), t, ids)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradient_in_place_of_logits_with_a_history(device, reduction):
    dtype = torch.float32
    _, t, ids = (x.to(device) for x in data(6, 40, 5, dtype, 12))
    g = torch.Generator().manual_seed(13)
    h, w = torch.randn(6, 8, generator=g).to(device), torch.randn(40, 8, generator=g).to(device).requires_grad_()
    grads = []
    for there in (False, True):
        z = h @ w.t()
        before = z.detach().clone()
        loss, grad = ops.topk_distillation_grad(z, t, ids, 1.5, reduction, out=z if there else None)
        assert not loss.requires_grad and not grad.requires_grad
        assert (z.data_ptr() == grad.data_ptr()) == there and (there or torch.equal(z, before))
        z.backward(grad)
        grads.append(w.grad)
        w.grad = None
    assert (grads[0] != 0).any() and torch.equal(*grads)
    # what was saved before the write is no longer there (on the CPU the loss saves none of it)
    z = h @ w.t()
    pending, square = ops.topk_distillation(z, t, ids, 1.5), z * z
    kept = torch.tanh(z)
    ops.topk_distillation_grad(z, t, ids, 1.5, reduction, out=z)
    for saved in (square.sum(), pending)[:1 if device == "cpu" else 2]:
        with pytest.raises(RuntimeError):
            saved.backward()
    ops.topk_distillation_grad(h @ w.t(), t, ids, 1.5, reduction, out=kept)
    with pytest.raises(RuntimeError):
        kept.sum().backward()
    leaf = z.detach().requires_grad_()
    want = ops.topk_distillation_grad(leaf, t, ids, 1.5, reduction)[1]
    grad = ops.topk_distillation_grad(leaf, t, ids, 1.5, reduction, out=leaf)[1]
    assert torch.equal(grad, want) and leaf.requires_grad and leaf.is_leaf


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_gradient_under_inference_mode(device):
    z, t, ids = (x.to(device) for x in data(6, 40, 5, torch.float32, 14))
    want = ops.topk_distillation_grad(z, t, ids, 1.5)
    with torch.inference_mode():
        for args in ((z, t, ids), (z.clone(), t.clone(), ids.clone())):
            got = ops.topk_distillation_grad(*args, 1.5)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        there = z.clone()
        assert ops.topk_distillation_grad(there, t, ids, 1.5, out=there)[1] is there and torch.equal(there, want[1])


def test_refusals_of_the_entry_point():
    """Before anything is launched: an upstream gradient belongs to the backward pass, which needs it and the row's
    log-sum-exp; sizes and temperatures out of range. The addresses are never used."""
    def call(loss=16, lse=16, dz=16, grad=None, grad_rows=0, M=1, k=1, V=8, T=1.0, total=None):
        return _native.fn("brain_distill_rows")(2, 16, V, 16, 16, loss, lse, None, dz, V, grad, None, 0, 0, grad_rows, M, k, V,
                                                T, total, None)
    for bad in (dict(grad=16), dict(grad_rows=1), dict(loss=None), dict(loss=None, grad=16, lse=None),
                dict(loss=None, grad=16, dz=None), dict(loss=None, grad=16, total=16), dict(k=0), dict(k=1025), dict(V=0),
                dict(V=2 ** 30 + 1), dict(M=-1), dict(M=2 ** 31), dict(T=0.0)):
        assert call(**bad) == 1, bad  # cudaErrorInvalidValue


# ------------------------------------------------------------------ kernels
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V,k,T", [
    (1, 1, 1, 1.0), (3, 7, 7, 2.0), (2, 33, 1, 0.5), (5, 1000, 20, 1.0), (4, 1003, 64, 4.0), (3, 32000, 128, 1.0),
    (2, 50257, 100, 2.0), (2, 128256, 256, 1.0), (1, 128256, 1024, 1.5), (2, 200003, 5, 1.0), (200, 515, 9, 1.0),
    (1, 900001, 3, 1.0), (1300, 130, 5, 1.0), (1200, 4003, 2, 1.5), (301, 33000, 7, 1.0), (170, 50257, 20, 2.0), (160, 128256, 5, 1.0),
    (0, 64, 4, 1.0)])
def test_loss_and_gradients(dtype, rows, V, k, T):
    z, t, ids = data(rows, V, k, dtype, rows + V)
    zc, tc, ic = z.cuda(), t.cuda(), ids.cuda()
    for reduction in ("mean", "sum", "none"):
        leaf = zc.clone().requires_grad_()
        loss = ops.topk_distillation(leaf, tc, ic, T, reduction)
        (grad,) = torch.autograd.grad(loss.sum() * 1.0, leaf)
        check(loss, grad, z, t, ids, T, reduction, dtype)
        l2, g2 = ops.topk_distillation_grad(zc, tc, ic, T, reduction)
        check(l2, g2, z, t, ids, T, reduction, dtype)
        l3, g3 = ops.topk_distillation_grad(zc, tc, ic, T, reduction)
        assert torch.equal(l2, l3) and torch.equal(g2, g3)
        with torch.no_grad():
            assert torch.equal(ops.topk_distillation(zc, tc, ic, T, reduction), loss)
    here = zc.clone()
    l4, g4 = ops.topk_distillation_grad(here, tc, ic, T, "none", out=here)
    assert g4 is here and torch.equal(here, g2) and torch.equal(l4, l2)
    assert ops.check_status() == []


@gpu
def test_rows_without_entries_and_masked_logits():
    z, t, ids = data(9, 300, 6, torch.bfloat16, 3)
    ids[0] = -1
    ids[1, 1:] = -1
    t[2] = -INF
    t[3, :3] = -INF
    ids[4, 5] = ids[4, 2] = ids[4, 0]
    z[5] = torch.where(torch.isin(torch.arange(300), ids[5]), z[5].float(), -INF).bfloat16()  # only teacher ids left
    z[6, 17] = -INF if 17 not in ids[6] else z[6, 17]
    z[0, 3] = math.nan
    t[7] = 1e30
    ids[8, 0] = 299
    zc = z.cuda()
    for reduction in ("none", "mean"):
        loss, grad = ops.topk_distillation_grad(zc, t.cuda(), ids.cuda(), 1.0, reduction)
        some = formula(torch.where(z.isnan(), 0.0, z), t, ids, 1.0)[2]
        assert some.tolist() == [False, True, False] + [True] * 6
        check(loss, grad, torch.where(z.isnan(), 0.0, z), t, ids, 1.0, reduction, torch.bfloat16)
    # nothing to learn from at all
    none = torch.full_like(ids, -1)
    loss, grad = ops.topk_distillation_grad(zc, t.cuda(), none.cuda(), 1.0)
    assert loss.item() == 0 and (grad == 0).all()
    # a teacher id that the student masks: an infinite loss; NaN logits: NaN, in their rows alone
    z2, t2, i2 = data(4, 64, 3, torch.float32, 4)
    z2[1, i2[1, 0]] = -INF
    z2[2, 5] = math.nan
    t2[3, 1] = math.nan
    loss, grad = ops.topk_distillation_grad(z2.cuda(), t2.cuda(), i2.cuda(), 1.0, "none")
    assert torch.isfinite(loss[0]) and loss[1] == INF and loss[2].isnan() and loss[3].isnan()
    assert torch.isfinite(grad[:2]).all() and grad[2].isnan().all() and grad[3].isnan().any()
    assert ops.check_status() == []


@gpu
def test_ids_outside_the_vocabulary_are_recorded():
    z, t, ids = data(3, 50, 4, torch.bfloat16, 5)
    ids[1, 2] = 50
    loss = ops.topk_distillation(z.cuda(), t.cuda(), ids.cuda(), 1.0, "none")
    assert [b[0] for b in ops.check_status()] == ["distill"]
    ids[1, 2] = -1
    check(loss, None, z, t, ids, 1.0, "none", torch.bfloat16)
    assert ops.check_status() == []


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_types_and_shapes(dtype):
    z, t, ids = data(6, 403, 5, dtype, 6)
    wide = torch.zeros(6, 420, dtype=dtype)
    wide[:, 5:408] = z
    w = wide.cuda()[:, 5:408]
    out = torch.full((6, 411), 7.0, device="cuda", dtype=dtype)
    loss, grad = ops.topk_distillation_grad(w, t.cuda(), ids.cuda(), 2.0, out=out[:, 2:405])
    check(loss, grad, z, t, ids, 2.0, "mean", dtype)
    assert (out[:, :2] == 7).all() and (out[:, 405:] == 7).all()  # the neighbours stay
    leaf = w.view(2, 3, 403).detach().requires_grad_()
    loss = ops.topk_distillation(leaf, t.double().view(2, 3, 5).cuda(), ids.int().view(2, 3, 5).cuda(), 2.0)
    loss.backward()
    check(loss, leaf.grad.view(6, 403), z, t, ids, 2.0, "mean", dtype)
    turned = z.cuda().t().contiguous().t().requires_grad_()
    loss = ops.topk_distillation(turned, t.cuda(), ids.cuda(), 2.0, "none")
    up = torch.rand(6, device="cuda")
    (grad,) = torch.autograd.grad(loss, turned, up)
    _, gf, _, size = formula(z, t, ids, 2.0)
    by = up.cpu().double()[:, None]
    assert ((grad.cpu().double() - gf * by).abs() <= tolerances(z, gf * by, size * by, 2.0, dtype)[1]).all()


@gpu
@pytest.mark.parametrize("T", [1.0, 1.7])
@pytest.mark.parametrize("offset", [0.0, -3000.0, 2.0 ** 16, -2.0 ** 18])
def test_loss_of_logits_with_an_offset(offset, T):
    """What a row's logits have in common changes neither the loss nor how far it is off."""
    z, t, ids = data(40, 1000, 12, torch.float32, 16)
    z = z + offset  # rounded to f32, exactly the same for both sides
    loss = ops.topk_distillation(z.cuda(), t.cuda(), ids.cuda(), T, "none").cpu().double()
    want = formula(z, t, ids, T)[0]
    near = z.double() - z.double().amax(-1, keepdim=True)
    assert ((loss - want).abs() <= tolerances(near.float(), want, want, T, torch.float32)[0]).all(), (loss - want).abs().max()


@gpu
def test_gradient_along_a_direction():
    """The kernel's gradient against differences of the loss in 64 bits."""
    z, t, ids = data(5, 700, 12, torch.float32, 7)
    _, grad = ops.topk_distillation_grad(z.cuda(), t.cuda(), ids.cuda(), 1.5)
    d = torch.randn(5, 700, generator=torch.Generator().manual_seed(8)).double()
    h = 1e-5
    hi, lo = (ops.topk_distillation(z.double() + s * h * d, t.double(), ids, 1.5) for s in (1, -1))
    slope = float((hi - lo) / (2 * h))
    assert abs(float((grad.cpu().double() * d).sum()) - slope) <= 1e-5 * float((grad.cpu().double() * d).abs().sum())


@gpu
def test_two_graphs_of_the_same_leaf_and_repeated_backward():
    z, t, ids = (x.cuda() for x in data(8, 600, 10, torch.bfloat16, 9))
    leaf = z.requires_grad_()
    loss = ops.topk_distillation(leaf, t, ids, 2.0)
    (a,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (b,) = torch.autograd.grad(loss * 0.5, leaf, retain_graph=True)
    (c,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(a, c) and torch.equal(a, b * 2)
    with torch.no_grad():
        leaf.mul_(2)
    want = torch.autograd.grad(ops.topk_distillation(leaf, t, ids, 2.0), leaf)[0]
    with torch.no_grad():
        leaf.div_(2)
    del loss  # an eager graph of the leaf that lives on would tie the captured backward pass to its stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got_loss, got = ops.topk_distillation_grad(leaf.detach(), t, ids, 2.0)
            (auto,) = torch.autograd.grad(ops.topk_distillation(leaf, t, ids, 2.0), leaf)
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        leaf.mul_(2)
    graph.replay()
    graph.replay()
    assert torch.equal(auto, want)
    assert torch.equal(got, ops.topk_distillation_grad(leaf.detach(), t, ids, 2.0)[1])


@gpu
@pytest.mark.parametrize("rows,V", [(1, 120000), (160, 25000)])
def test_calls_of_several_threads(rows, V):
    """Few and many kept entries at once, on streams of their own: each call gets the shared memory that it needs. The
    entry point itself is called, as the host time around it would keep the threads apart."""
    call, kept = _native.fn("brain_distill_rows"), (1024, 1, 1024, 1)
    cases = [tuple(x.cuda() for x in data(rows, V, k, torch.float32, k)) for k in kept]
    want = [ops.topk_distillation(*c, 2.0, "none") for c in cases]
    losses, streams = [torch.zeros(rows, device="cuda") for _ in kept], [torch.cuda.Stream() for _ in kept]
    torch.cuda.synchronize()
    gate, failed = threading.Barrier(len(kept)), []

    def calls(i):
        z, t, ids = cases[i]
        gate.wait()
        for j in range(3000):
            rc = call(2, z.data_ptr(), V, t.data_ptr(), ids.data_ptr(), losses[i].data_ptr(), None, None, None, 0, None,
                      None, 0, 0, 0, rows, kept[i], V, 2.0, None, streams[i].cuda_stream)
            if rc:
                failed.append((kept[i], j, rc))
            if j % 200 == 199:
                streams[i].synchronize()

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(len(kept))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    assert all(torch.equal(a, b) for a, b in zip(losses, want))


@gpu
@pytest.mark.parametrize("V,chunk,main", [(512, 0, False), (515, 40, False), (512, 33, True)])
def test_linear(V, chunk, main):
    z, t, ids = data(100, V, 8, torch.float32, 10)
    ids[::7] = -1
    g = torch.Generator().manual_seed(11)
    h = (torch.randn(4, 25, 128, generator=g)).bfloat16().cuda().requires_grad_()
    w = (torch.randn(V, 128, generator=g) * 0.1).bfloat16().cuda().requires_grad_()
    if main:
        w.main_grad = torch.ones(V, 128, device="cuda")
    tt, ii = t.view(4, 25, 8).cuda(), ids.view(4, 25, 8).cuda()
    loss = ops.linear_topk_distillation(h, w, tt, ii, 1.5, chunk)
    (loss * 2).backward()
    hd, wd = (x.detach().cpu().double().requires_grad_() for x in (h, w))
    want = ops.topk_distillation(hd.view(100, 128) @ wd.t(), t.double(), ids, 1.5)
    (want * 2).backward()
    # logits and their gradient are rounded to bf16 on the way (half a step each, 2^-8)
    assert abs(loss.item() - want.item()) < 2.0 ** -7 * max(1.0, want.item())
    dw = w.main_grad - 1 if main else w.grad
    for a, b in ((h.grad, hd.grad.view(4, 25, 128)), (dw, wd.grad)):
        assert (a.cpu().double() - b).norm() <= 3 * 2.0 ** -8 * b.norm()
    assert main == (w.grad is None)


@gpu
@pytest.mark.multigpu
def test_tensors_of_another_device_than_the_current_one():
    z, t, ids = data(40, 64, 4, torch.float32, 15)
    h, w = (torch.randn(n, 32, generator=torch.Generator().manual_seed(n)).bfloat16() for n in (40, 64))
    got = []
    for device in ("cuda:0", "cuda:1"):
        with torch.cuda.device(0):
            tc, ic = t.to(device), ids.to(device)
            loss, grad = ops.topk_distillation_grad(z.to(device), tc, ic)
            hd, wd = h.to(device).requires_grad_(), w.to(device).requires_grad_()
            head = ops.linear_topk_distillation(hd, wd, tc, ic)
            head.backward()
            got.append([x.cpu() for x in (loss, grad, head, hd.grad, wd.grad)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@gpu
@pytest.mark.parametrize("chunk", [0, 4])
def test_linear_without_tokens(chunk):
    h = torch.zeros(2, 0, 32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(64, 32, device="cuda").bfloat16().requires_grad_()
    loss = ops.linear_topk_distillation(h, w, torch.zeros(2, 0, 3, device="cuda"), torch.zeros(2, 0, 3, device="cuda").long(),
                                        chunk=chunk)
    loss.backward()
    assert loss.item() == 0 and h.grad.shape == h.shape and (w.grad == 0).all()


@gpu
def test_a_language_model_learns_from_it():
    cfg = LlamaLiteConfig(vocab_size=256, hidden_dim=128, num_layers=1, num_heads=2, num_kv_heads=2, head_dim=64,
                          intermediate_dim=256, max_seq_len=64)
    model = LlamaLite(cfg, device="cuda", dtype=torch.bfloat16, seed=0)
    tokens = torch.randint(0, 256, (2, 32), device="cuda")
    logits = model(tokens)
    with torch.no_grad():
        top = torch.topk(LlamaLite(cfg, device="cuda", dtype=torch.bfloat16, seed=1)(tokens).float(), 16)
    loss = losses.TopKDistillationLoss(2.0)(logits, top.values, top.indices)
    loss.backward()
    grads = [p.grad for p in model.parameters() if p.grad is not None]
    assert grads and all(torch.isfinite(g).all() for g in grads) and any((g != 0).any() for g in grads)

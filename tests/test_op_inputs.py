"""What the ops' shared helpers refuse and count, whichever op calls them."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from brain_b200 import _native, ops
from brain_b200 import quantization as Q
from brain_b200.ops._common import rows2d

gpu = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(3, 0), (2, 3, 0), (0, 0), (0,)])
def test_rows_without_values_are_refused(shape):
    with pytest.raises(RuntimeError):
        rows2d(torch.empty(shape))


@pytest.mark.parametrize("shape,rows", [((3, 5), 3), ((0, 5), 0), ((2, 0, 5), 0), ((5,), 1), ((2, 3, 5), 6)])
def test_rows_of_a_tensor(shape, rows):
    x = torch.randn(shape)
    assert torch.equal(rows2d(x), x.reshape(rows, 5)) and rows2d(x).stride(1) == 1
    turned = torch.randn(5, 4).t()
    assert torch.equal(rows2d(turned), turned) and rows2d(turned).stride(1) == 1


@gpu
@pytest.mark.parametrize("call", [
    lambda x: ops.rms_norm(x, x[0]), lambda x: ops.layer_norm(x, x[0], x[0]), lambda x: ops.add_rms_norm(x, x, x[0]),
    lambda x: ops.cross_entropy(x, torch.zeros(3, device="cuda", dtype=torch.long)), lambda x: ops.rms_norm_fp8(x, x[0]),
], ids=["rms_norm", "layer_norm", "add_rms_norm", "cross_entropy", "rms_norm_fp8"])
def test_ops_refuse_rows_without_values(call):
    with pytest.raises((RuntimeError, ValueError)):
        call(torch.empty(3, 0, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_followed_or_refused(device, grad_mode):
    """A dual tensor that asks for no gradient: its tangent must not get lost, with or without a backward pass."""
    g = torch.Generator().manual_seed(0)
    x, z = (torch.randn(4, 128, generator=g).to(device) for _ in range(2))
    t, ids = torch.randn(4, 3, generator=g).to(device), torch.tensor([[0, 1, 5]] * 4, device=device)
    packed, scales, _ = Q.quantize_int4(torch.randn(8, 128, generator=g), 64)
    packed, scales = packed.to(device), scales.to(device)
    w = torch.ones(128, device=device)
    with fwd.dual_level(), torch.set_grad_enabled(grad_mode):
        d, half = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(x.bfloat16(), torch.ones_like(x).bfloat16())
        for call in (lambda: ops.rms_norm_fp8(d, w), lambda: ops.add_rms_norm_fp8(x, d, w),
                     lambda: ops.rms_norm_fp8(x, fwd.make_dual(w, w)), lambda: Q.int4_linear(half, packed, scales, group_size=64),
                     lambda: ops.topk_distillation(z, fwd.make_dual(t, t), ids)):
            with pytest.raises(RuntimeError):
                call()
        if device == "cuda":
            with pytest.raises(NotImplementedError):
                ops.topk_distillation(d, t, ids)
        else:
            h = 1e-3
            slope = fwd.unpack_dual(ops.topk_distillation(d * d, t, ids, 1.5)).tangent
            hi, lo = (ops.topk_distillation((x.double() + s * h) ** 2, t, ids, 1.5) for s in (1, -1))
            # differences are off by h^2 times a third derivative of order 100, f32 by a few 2^-24 of it
            assert abs(float(slope - (hi - lo) / (2 * h))) < 1e-3
        # tensors without a tangent are taken as before
        ops.rms_norm_fp8(x, w), Q.int4_linear(x.bfloat16(), packed, scales, group_size=64), ops.topk_distillation(z, t, ids)


@gpu
@pytest.mark.parametrize("rows", [0, 3])
def test_launches_are_counted(rows):
    """Each operator's kernels, by what its call asks for."""
    some = int(rows > 0)
    z, t = (torch.zeros(rows, n, device="cuda", requires_grad=n == 64) for n in (64, 2))
    ids = torch.zeros(rows, 2, device="cuda", dtype=torch.long)
    flat = z.detach()
    h, w = (torch.zeros(n, 64, device="cuda", dtype=torch.bfloat16) for n in (rows, 64))
    x = torch.zeros(rows, 40960, device="cuda", dtype=torch.bfloat16)
    packed, scales = torch.zeros(4, 20480, device="cuda", dtype=torch.uint8), torch.ones(4, 320, device="cuda").bfloat16()
    p, ones = torch.ones(rows, 3, 8, device="cuda"), torch.ones(64, device="cuda")
    for call, kernels in (
            (lambda: ops.topk_distillation(flat, t, ids, reduction="none"), some),
            (lambda: ops.topk_distillation(flat, t, ids), some + 1),
            (lambda: ops.topk_distillation(z, t, ids).backward(), 2 * some + 1),
            (lambda: ops.topk_distillation_grad(flat, t, ids, reduction="none"), some),
            (lambda: ops.topk_distillation_grad(flat, t, ids, reduction="sum"), some + 1),
            (lambda: ops.topk_distillation_grad(flat, t, ids), some + 2),
            (lambda: ops.linear_topk_distillation(h, w, t, ids), 2 * some + 2),
            (lambda: ops.linear_topk_distillation(h, w, t, ids, chunk=1), 2 * rows + 2),
            (lambda: Q.int4_linear(x, packed, scales), 2 * some),
            (lambda: Q.int4_linear(x[:, :1024], packed[:, :512].contiguous(), scales[:, :8]), some),
            (lambda: ops.rms_norm_fp8(flat, ones), some),
            (lambda: ops.verify_draft(p, ids, p[..., 0]), some)):
        with _native.launch_counter() as counter:
            call()
        assert counter.count == kernels
    torch.cuda.synchronize()

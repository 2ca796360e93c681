"""RMSNorm with e4m3 output: the kernel against the definition in 64 bits."""
import pytest
import torch

from brain_b200 import ops
from brain_b200.quantization import fp8 as F8

gpu = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def data(shape, dtype, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(torch.randn((*shape[:-1], 1), generator=g))
    r = torch.randn(shape, generator=g)
    w = 1 + 0.3 * torch.randn(shape[-1], generator=g)
    return x.to(dtype), r.to(dtype) if residual else None, w.to(dtype)


def check(q, scale, s, x, r, w, eps, scaling):
    D = x.shape[-1]
    want_s = x if r is None else (x.float() + r.float()).to(x.dtype)
    if r is not None:
        assert torch.equal(s.cpu(), want_s)
    v = want_s.double()
    y = v * (v.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    cut = y.view(*x.shape[:-1], -1, 128) if scaling == "block" else y[..., None, :]
    amax = cut.abs().amax(-1)
    want = torch.where(amax > 0, (amax / 448).clamp_min(2.0 ** -126), 1.0)
    got = scale.cpu().double().view(want.shape)
    # f32: up to D / 256 + 16 additions follow one another in the mean (which enters by its root), then a
    # reciprocal root of 2 ulp, two products and a division
    tol = (D / 256 + 16) * 2.0 ** -24 / 2 + 8 * 2.0 ** -24
    assert ((got - want).abs() <= tol * want).all()
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    back = q.cpu().double().view(cut.shape) * got[..., None]
    # half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale below 2^-6 of it
    assert ((back - cut).abs() <= (2.0 ** -4 + 4 * tol) * cut.abs() + 2.0 ** -10 * got[..., None]).all()


@pytest.mark.parametrize("scaling", ["rowwise", "block"])
@pytest.mark.parametrize("residual", [False, True])
def test_cpu_path(scaling, residual):
    x, r, w = data((3, 5, 256), torch.bfloat16, residual=residual)
    out = ops.add_rms_norm_fp8(x, r, w, 1e-5, scaling) if residual else (*ops.rms_norm_fp8(x, w, 1e-5, scaling), None)
    check(*out, x, r, w, 1e-5, scaling)


def test_refusals():
    x, r, w = data((4, 96), torch.bfloat16)
    with pytest.raises(ValueError):
        ops.rms_norm_fp8(x, w, scaling="tensor")
    with pytest.raises(ValueError):
        ops.rms_norm_fp8(x, w, scaling="block")  # 96 is not a multiple of 128
    with pytest.raises(ValueError):
        ops.add_rms_norm_fp8(x, r[:3], w)
    with pytest.raises(ValueError):
        ops.rms_norm_fp8(x, w[:95])
    with pytest.raises(ValueError):
        ops.rms_norm_fp8(x[:, :0], w[:0])
    with pytest.raises(ValueError):
        ops.rms_norm_fp8(x[:1, :1].expand(1, 2 ** 30 + 128), w[:1].expand(2 ** 30 + 128))
    with pytest.raises(TypeError):
        ops.rms_norm_fp8(x, w.float())
    with pytest.raises(TypeError):
        ops.rms_norm_fp8(x.double(), w.double())
    with pytest.raises(RuntimeError):
        ops.rms_norm_fp8(x.requires_grad_(), w)
    with torch.no_grad():
        ops.rms_norm_fp8(x, w)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape,scaling", [
    ((1, 4096), "rowwise"), ((1, 128), "block"), ((7, 8192), "block"), ((3, 5, 768), "rowwise"), ((65, 16), "rowwise"),
    ((5, 1), "rowwise"), ((33, 1001), "rowwise"), ((2, 16384), "rowwise"), ((3, 40960), "block"), ((2, 65537), "rowwise"),
    ((300, 384), "block"), ((129, 1024), "rowwise"), ((11, 2056), "rowwise"),
    ((70, 333), "rowwise"), ((41, 7), "rowwise"), ((19, 4097), "rowwise"), ((9, 8191), "rowwise"), ((5, 12003), "rowwise"), ((0, 256), "rowwise")])
def test_kernel(dtype, residual, shape, scaling):
    x, r, w = data(shape, dtype, 1, residual)
    args = [t.cuda() for t in (x, r, w) if t is not None]
    out = ops.add_rms_norm_fp8(*args, 1e-5, scaling) if residual else (*ops.rms_norm_fp8(*args, 1e-5, scaling), None)
    if shape[0]:
        check(*out, x, r, w, 1e-5, scaling)
    else:
        assert out[0].shape == x.shape and out[1].numel() == 0


@gpu
@pytest.mark.parametrize("scaling", ["rowwise", "block"])
def test_strided_and_unaligned_rows(scaling):
    x, r, w = data((9, 640), torch.bfloat16, 2)
    for at, width in ((0, 512), (3, 384), (8, 512)):
        xs, rs, ws = x[:, at:at + width], r[:, 1:1 + width], w[at:at + width]
        out = ops.add_rms_norm_fp8(x.cuda()[:, at:at + width], r.cuda()[:, 1:1 + width], w.cuda()[at:at + width], 1e-6, scaling)
        check(*out, xs, rs, ws, 1e-6, scaling)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width,step", [(1001, 1009), (1001, 1001 + 32), (1003, 1004), (77, 200), (5, 13)])
def test_odd_rows_of_wider_tensors(dtype, width, step):
    x, r, w = data((9, step), dtype, 4)
    xs, rs, ws = x.cuda()[:, :width], r.cuda()[:, :width], w.cuda()[1:1 + width]
    ws = ws if len(ws) == width else w.cuda()[:width]
    out = ops.add_rms_norm_fp8(xs, rs, ws, 1e-5)
    check(*out, xs.cpu(), rs.cpu(), ws.cpu(), 1e-5, "rowwise")
    check(*ops.rms_norm_fp8(xs, ws, 1e-5), None, xs.cpu(), None, ws.cpu(), 1e-5, "rowwise")


@gpu
@pytest.mark.parametrize("D", [512, 500])
@pytest.mark.parametrize("scaling", ["rowwise", "block"])
def test_odd_rows(D, scaling):
    """Zeros, subnormal rows, infinities and NaN stay in their own rows (and blocks)."""
    if scaling == "block" and D % 128:
        pytest.skip("blocks of 128")
    x, _, w = data((6, D), torch.bfloat16, 3, False)
    x[1] = 0
    x[2] = 1e-39
    x[3, 7] = float("inf")
    x[4, 9] = float("nan")
    w[5] = 0
    q, scale = ops.rms_norm_fp8(x.cuda(), w.cuda(), 1e-6, scaling)
    qr, sr = ops.rms_norm_fp8(x, w, 1e-6, scaling)
    check(q[::5], scale[::5], None, x[::5], None, w, 1e-6, scaling)
    assert (q[1].float() == 0).all() and (scale[1] == 1).all()
    assert torch.isfinite(q[2].float()).all() and torch.isfinite(scale[2]).all()
    assert torch.equal(q[3:5].cpu().isnan(), qr[3:5].isnan()) and torch.equal(scale[3:5].cpu().isnan(), sr[3:5].isnan())
    assert q[4].isnan().all()


@gpu
def test_feeds_the_fp8_gemms_and_a_graph():
    x, r, w = (t.cuda() for t in data((64, 512), torch.bfloat16, 4))
    lin = torch.randn(256, 512, generator=torch.Generator().manual_seed(5)).cuda().bfloat16()
    wq, ws = F8.quantize_fp8_rowwise(lin)
    bq, bs = F8.quantize_fp8_weight_blocks(lin)
    torch.cuda.synchronize()

    def step():
        q, s, h = ops.add_rms_norm_fp8(x, r, w, 1e-5)
        b, bsc, _ = ops.add_rms_norm_fp8(x, r, w, 1e-5, "block")
        return F8.fp8_gemm_rowwise(q, s, wq, ws), F8.fp8_gemm_blockscaled(b, bsc, bq, bs), h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.mul_(2).add_(r)
    graph.replay()
    again = step()
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    y = ops.rms_norm(want[2], w, 1e-5).float() @ lin.float().t()
    for out in want[:2]:
        assert (out.float() - y).norm() < 0.06 * y.norm()  # e4m3 on both sides: 2^-4 each at most


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [512, 500, 4096, 5001])
@pytest.mark.parametrize("scaling", ["rowwise", "block"])
def test_rows_of_subnormal_size(dtype, D, scaling):
    """Rows so small that scales stop at 2^-126, and 1 / scale times the row's factor passes f32's range."""
    if scaling == "block" and D % 128:
        pytest.skip("blocks of 128")
    x, _, w = data((4, D), torch.float32, 6, False)
    x = x / x.abs().amax(-1, keepdim=True) * torch.tensor([1e-39, 2e-40, 1e-38, 1.0])[:, None]
    x, w = x.to(dtype), w.to(dtype)
    q, scale = ops.rms_norm_fp8(x.cuda(), w.cuda(), 1e-6, scaling)
    check(q, scale, None, x, None, w, 1e-6, scaling)
    assert (scale[:2] == 2.0 ** -126).all() and (q[:3].float() != 0).any(-1).all()
    # one row offset from 16 bytes against the weight: the kernel for any alignment
    if scaling == "rowwise":
        wide = torch.zeros(4, D + 3, dtype=dtype)
        wide[:, 1:D + 1] = x
        check(*ops.rms_norm_fp8(wide.cuda()[:, 1:D + 1], w.cuda(), 1e-6), None, x, None, w, 1e-6, scaling)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,ldx,ldr", [(1001, 1001, 1009), (1001, 1009, 1001), (1001, 1002, 1010), (77, 85, 80), (4097, 4105, 4097),
                                       (1024, 1032, 1024), (1024, 1024, 1025)])
def test_residual_of_another_row_stride(dtype, D, ldx, ldr):
    x, r, w = data((7, max(ldx, ldr)), dtype, 5)
    xs, rs = (t[:, :n].contiguous().cuda()[:, :D] for t, n in ((x, ldx), (r, ldr)))
    assert xs.stride(0) == ldx and rs.stride(0) == ldr
    out = ops.add_rms_norm_fp8(xs, rs, w[:D].cuda(), 1e-5)
    check(*out, x[:, :D], r[:, :D], w[:D], 1e-5, "rowwise")

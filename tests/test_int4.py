"""4-bit weights: quantiser, packing and the few-token product against the definition in 64 bits."""
import pytest
import torch

from brain_b200 import ops
from brain_b200 import quantization as Q

gpu = pytest.mark.gpu


def weight(N, K, G, zeros, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // G)
    packed = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand(N, groups, generator=g) * 0.02 + 0.001).to(dtype)
    z = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None
    return packed, scales, z


def dense(packed, scales, zeros, G):
    """The weight in 64 bits, value by value as the format says."""
    N, K = packed.shape[0], packed.shape[1] * 2
    v = torch.empty(N, K, dtype=torch.float64)
    v[:, 0::2] = (packed % 16).double()
    v[:, 1::2] = (packed // 16).double()
    g = torch.arange(K) // G
    v = torch.where(v > 7, v - 16, v) if zeros is None else v - zeros.double()[:, g]
    return v * scales.double()[:, g]


def check(y, x, w, bias, dtype):
    xd = x.double()
    want = xd @ w.t() + (0 if bias is None else bias.double())
    # half a step of the output's type, and K / 16 sums of 16 products that each may lose 2^-22 of all their size
    size = xd.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (x.shape[-1] / 16 + 16) * 2.0 ** -22 * size + 2.0 ** -24
    assert y.shape == want.shape and y.dtype == dtype
    assert ((y.cpu().double() - want).abs() <= tol).all(), ((y.cpu().double() - want).abs() / tol).max()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("K,G", [(256, 128), (160, 128), (96, 32), (64, 64)])
def test_quantiser(symmetric, K, G):
    w = torch.randn(9, K, generator=torch.Generator().manual_seed(1))
    w[3] = 0
    w[4] = w[4].abs() + 1
    packed, scales, zeros = Q.quantize_int4(w, G, symmetric)
    assert (zeros is None) == symmetric and packed.shape == (9, K // 2)
    back = Q.dequantize_int4(packed, scales, zeros, G)
    assert torch.equal(back.double(), dense(packed, scales, zeros, G).float().double())
    step = scales.float().repeat_interleave(G, 1)[:, :K]
    # half a step; a scale that bf16 rounds down by 2^-8 leaves the ends of the range 15 x 2^-8 of a step further
    # out, and a rounded zero point moves them by another half
    assert ((back - w).abs() <= step * (0.5 + 15 * 2.0 ** -8 + (0 if symmetric else 0.5))).all()
    assert (back[3] == 0).all()
    if symmetric and K % G == 0:
        flat = Q.pack_int4(torch.round(w / step).clamp(-8, 7).to(torch.int8))
        assert torch.equal(flat.view(9, -1), packed)  # the byte order of pack_int4


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1.0, 1e-4, 3e-6, 2.0 ** -24, 1e-9, 0.0])
def test_scales_of_small_weights(device, symmetric, dtype, size):
    """No value is further from its weight than half a step, of a scale that is no larger than the group asks for and the
    type lets it be."""
    w = torch.randn(5, 256, generator=torch.Generator().manual_seed(3)) * size
    packed, scales, zeros = Q.quantize_int4(w.to(device), 64, symmetric, dtype)
    assert scales.dtype == dtype and (scales > 0).all() and torch.isfinite(scales).all()
    cut = w.view(5, 4, 64).double()
    lo, hi = cut.amin(-1).clamp_max(0), cut.amax(-1).clamp_min(0)
    wanted = cut.abs().amax(-1) / 7 if symmetric else (hi - lo) / 15
    info = torch.finfo(dtype)
    got, least = scales.cpu().double(), max(info.tiny * info.eps, 2.0 ** -126)
    # normal scales round by half a step, subnormal ones up by less than one; f32 on the way adds 2^-23
    assert (got <= wanted * (1 + info.eps / 2 + 2.0 ** -23) + least).all()
    assert (got >= wanted * (1 - info.eps / 2 - 2.0 ** -23)).all()
    back = Q.dequantize_int4(packed, scales, zeros, 64).cpu().double().view_as(cut)
    # as in test_quantiser: what a scale rounded down leaves out at the ends, and a rounded zero point
    far = 0.5 + 15 * (info.eps / 2 + 2.0 ** -22) + (0 if symmetric else 0.5)
    assert ((back - cut).abs() <= far * got[..., None]).all()


def test_small_weights_keep_their_levels_in_f16():
    w = torch.randn(64, 1024, generator=torch.Generator().manual_seed(4))
    for symmetric in (True, False):
        error = [float((Q.dequantize_int4(*Q.quantize_int4(w * size, 128, symmetric, torch.float16), 128) / size - w).norm() / w.norm())
                 for size in (1.0, 1e-4)]
        # scales of about 4e-5 are steps of 2^-24 apart: at most 2^-24 / 2e-5 = 0.3 % larger
        assert error[1] <= error[0] * 1.01


@pytest.mark.parametrize("zeros", [False, True])
def test_cpu_path(zeros):
    packed, scales, z = weight(33, 160, 64, zeros, torch.bfloat16)
    x = torch.randn(2, 3, 160).bfloat16()
    b = torch.randn(33).bfloat16()
    check(Q.int4_linear(x, packed, scales, z, b, 64), x, dense(packed, scales, z, 64), b, torch.bfloat16)


def test_refusals():
    packed, scales, z = weight(8, 128, 64, True, torch.bfloat16)
    x = torch.randn(2, 128).bfloat16()
    for bad in (lambda: Q.int4_linear(x[:, :96], packed, scales, z, group_size=64),
                lambda: Q.int4_linear(x, packed, scales[:, :1], z, group_size=64),
                lambda: Q.int4_linear(x, packed, scales, z[:7], group_size=64),
                lambda: Q.int4_linear(x, packed, scales, z, group_size=48),
                lambda: Q.int4_linear(x, packed, scales, z, torch.zeros(7).bfloat16(), 64),
                lambda: Q.int4_linear(x, packed.int(), scales, z, group_size=64),
                lambda: Q.int4_linear(x, packed[:1, :1].expand(2 ** 30 + 1, 64), scales[:1, :1].expand(2 ** 30 + 1, 2),
                                      group_size=64),
                lambda: Q.quantize_int4(torch.zeros(4, 48), 32),
                lambda: Q.quantize_int4(torch.zeros(1, 96 * 384), 96),
                lambda: Q.quantize_int4(torch.zeros(64), 32)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: Q.int4_linear(x, packed, scales.half(), z, group_size=64),
                lambda: Q.int4_linear(x, packed, scales, z.int(), group_size=64),
                lambda: Q.int4_linear(x.double(), packed, scales, z, group_size=64),
                lambda: Q.int4_linear(x, packed, scales, z, torch.zeros(8), 64),
                lambda: Q.quantize_int4(torch.zeros(4, 64), 32, scale_dtype=torch.float32)):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(RuntimeError):
        Q.int4_linear(x.requires_grad_(), packed, scales, z, group_size=64)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,G", [
    (1, 1, 32, 32), (1, 17, 96, 64), (2, 128, 128, 128), (8, 64, 4096, 128), (3, 100, 1376, 128), (5, 33, 4128, 32),
    (9, 48, 256, 64), (16, 250, 1024, 32), (17, 40, 2048, 96), (31, 70, 160, 4096), (33, 513, 512, 128), (64, 31, 384, 256),
    (130, 65, 640, 64), (1, 4096, 4096, 128), (4, 1024, 14336, 128), (8, 2049, 8192, 64), (1, 3, 28672, 32),
    (3, 20, 40960, 128)])
def test_kernel(dtype, zeros, M, N, K, G):
    packed, scales, z = weight(N, K, G, zeros, dtype, M + N)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(2)).to(dtype)
    b = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(dtype) if M % 2 else None
    c = [None if t is None else t.cuda() for t in (x, packed, scales, z, b)]
    y = Q.int4_linear(*c, group_size=G)
    check(y, x, dense(packed, scales, z, G), b, dtype)
    assert torch.equal(y, Q.int4_linear(*c, group_size=G))


@gpu
@pytest.mark.parametrize("M", [1, 3, 12])
def test_strided_inputs_and_shapes(M):
    packed, scales, z = weight(50, 384, 128, True, torch.bfloat16)
    x = torch.randn(M, 2, 400).bfloat16()
    xs = x[..., 3:387]  # rows on odd addresses
    w = dense(packed, scales, z, 128)
    wide = torch.zeros(50, 208, dtype=torch.uint8)
    wide[:, 16:] = packed
    big = wide.cuda()
    y = Q.int4_linear(x.cuda()[..., 3:387], big[:, 16:], scales.cuda(), z.cuda())
    check(y, xs, w, None, torch.bfloat16)
    y = Q.int4_linear(x.cuda().transpose(0, 1)[..., 3:387], packed.cuda(), scales.t().contiguous().cuda().t(), z.cuda())
    check(y, xs.transpose(0, 1), w, None, torch.bfloat16)
    # copies of both, each of the other's size, and zero points outside 0 .. 15
    g = torch.Generator().manual_seed(9)
    z = torch.randint(0, 256, (50, 3), generator=g, dtype=torch.uint8)
    y = Q.int4_linear(x.cuda()[..., 3:387], packed.cuda(), scales.t().contiguous().cuda().t(),
                      z.t().contiguous().cuda().t())
    check(y, xs, dense(packed, scales, z, 128), None, torch.bfloat16)
    for off in (1, 8):
        with pytest.raises(ValueError):
            Q.int4_linear(x.cuda()[..., 3:387], big[:, off:off + 192], scales.cuda(), z.cuda())
    assert Q.int4_linear(x.cuda()[:0, :, 3:387], packed.cuda(), scales.cuda(), z.cuda()).shape == (0, 2, 50)


@gpu
def test_non_finite_tokens_stay_in_their_rows():
    packed, scales, _ = weight(64, 256, 64, False, torch.bfloat16)
    x = torch.randn(8, 256).bfloat16()
    x[2, 5], x[5, 200] = float("inf"), float("nan")
    y = Q.int4_linear(x.cuda(), packed.cuda(), scales.cuda(), group_size=64).cpu()
    keep = [0, 1, 3, 4, 6, 7]
    check(y[keep], x[keep], dense(packed, scales, None, 64), None, torch.bfloat16)
    assert y[5].isnan().all() and not torch.isfinite(y[2]).any()


@gpu
@pytest.mark.parametrize("zeros", [True, False])
def test_tokens_of_any_size(zeros):
    # bf16 covers f32's range: each token for itself, and values far below a token's largest
    packed, scales, z = weight(70, 544, 64, zeros, torch.bfloat16)
    x = torch.randn(6, 544, generator=torch.Generator().manual_seed(2))
    x = (x * torch.tensor([2.0 ** -130, 2.0 ** -60, 1, 2.0 ** 60, 2.0 ** 115, 1])[:, None]).bfloat16()
    x[5, ::2] *= 2.0 ** -20
    y = Q.int4_linear(x.cuda(), packed.cuda(), scales.cuda(), None if z is None else z.cuda(), group_size=64).cpu()
    w = dense(packed, scales, z, 64)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    # as in check, with the smallest step of bf16's range in place of its fixed term
    tol = 2.0 ** -8 * want.abs() + (544 / 16 + 16) * 2.0 ** -22 * size + 2.0 ** -133
    assert torch.isfinite(y).all() and ((y.double() - want).abs() <= tol).all()


@gpu
@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("M,G", [(3, 32), (6, 64), (11, 128)])
@pytest.mark.parametrize("top,small", [(1.0, 2.0 ** -12), (1.0, 2.0 ** -36), (1.0, 2.0 ** -42), (2.0 ** 60, 2.0 ** -20),
                                       (2.0 ** 100, 2.0 ** -10)])
def test_small_tokens_beside_a_large_one_on_a_weight_of_zero(zeros, M, G, top, small):
    """The large ones add nothing, so the small ones are all of the sum: its bound is theirs."""
    K = 800
    packed, scales, z = weight(70, K, G, zeros, torch.bfloat16)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(5)) * small
    for k in range(5, K, 96):
        x[:, k] = top * (1 if k % 2 else -1)
        none = z[:, k // G] if zeros else torch.zeros(70, dtype=torch.uint8)
        byte = packed[:, k // 2]
        packed[:, k // 2] = byte & 0x0F | none << 4 if k % 2 else byte & 0xF0 | none
    x = x.bfloat16()
    y = Q.int4_linear(x.cuda(), packed.cuda(), scales.cuda(), None if z is None else z.cuda(), group_size=G).cpu()
    w = dense(packed, scales, z, G)
    assert (w[:, 5::96] == 0).all()
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    tol = 2.0 ** -8 * want.abs() + (K / 16 + 16) * 2.0 ** -22 * size + 2.0 ** -133  # as above
    assert ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() / tol).max()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,G", [(2, 32), (7, 64), (15, 128)])
def test_zero_points_of_every_size(dtype, M, G):
    """All 256 of them, next to one another and in whole tiles of the one or the other side of 128."""
    packed, scales, _ = weight(512, 1024, G, False, dtype, 6)
    groups = 1024 // G
    z = torch.arange(512 * groups).view(groups, 512).t().contiguous() % 256
    z[:64] = 128
    z[64:128] = 129
    z[128:192] = 255
    z[192:256] = 0
    z = z.to(torch.uint8)
    x = torch.randn(M, 1024, generator=torch.Generator().manual_seed(7)).to(dtype)
    y = Q.int4_linear(x.cuda(), packed.cuda(), scales.cuda(), z.cuda(), group_size=G)
    check(y, x, dense(packed, scales, z, G), None, dtype)


@gpu
@pytest.mark.parametrize("symmetric", [True, False])
def test_module(symmetric):
    lin = torch.nn.Linear(512, 96).cuda().bfloat16()
    m = Q.Int4Linear.from_linear(lin, 64, symmetric)
    x = torch.randn(3, 512, device="cuda").bfloat16()
    with torch.no_grad():
        y = m(x)
        full = lin(x).float()
    check(y, x.cpu(), dense(m.packed.cpu(), m.scales.cpu(), None if symmetric else m.zeros.cpu(), 64), m.bias.cpu(), torch.bfloat16)
    assert (y.float() - full).norm() < 0.2 * full.norm()
    other = Q.Int4Linear.from_linear(torch.nn.Linear(512, 96).cuda().bfloat16(), 64, symmetric)
    other.load_state_dict(m.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), y)
    assert ops.check_status() == []


@gpu
def test_captured_graph_on_another_stream():
    packed, scales, z = (t.cuda() for t in weight(300, 1024, 128, True, torch.bfloat16))
    x = torch.randn(4, 1024, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        Q.int4_linear(x, packed, scales, z)
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1, stream=side):
            y1 = Q.int4_linear(x, packed, scales, z)
        with torch.cuda.graph(g2, stream=side):
            y2 = Q.int4_linear(x * 2, packed, scales, z)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    x.neg_()
    torch.cuda.synchronize()
    for _ in range(3):  # two graphs at once share nothing
        with torch.cuda.stream(side):
            g1.replay()
        with torch.cuda.stream(other):
            g2.replay()
    torch.cuda.synchronize()
    want = Q.int4_linear(x, packed, scales, z)
    assert torch.equal(y1, want) and torch.equal(y2, 2 * want)

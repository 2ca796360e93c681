"""Verification of drafted tokens: the kernel against the definition, id by id."""
import pytest
import torch

from brain_b200 import ops
from brain_b200.ops.speculative import verify_draft_ref

gpu = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def data(B, K, V, dtype=torch.float32, seed=0, near=1.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(B, K + 1, V, generator=g) * 3
    p = torch.softmax(z, -1).to(dtype)
    q = torch.softmax(z[:, :K] + near * torch.randn(B, K, V, generator=g), -1).to(dtype)
    x = torch.multinomial(q.float().reshape(B * K, V), 1, generator=g).view(B, K) if B * K else torch.zeros(B, K, dtype=torch.long)
    return p, x, torch.rand(B, K + 1, generator=g), q


def same(got, want):
    assert got[0].dtype == got[1].dtype == torch.int64
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1]), (got, want)


# ------------------------------------------------------------------ CPU
def test_definition_by_hand():
    p = torch.tensor([[[0.5, 0.25, 0.25], [0.125, 0.75, 0.125], [0.25, 0.25, 0.5]]])
    q = torch.tensor([[[0.25, 0.5, 0.25], [0.5, 0.25, 0.25]]])
    x = torch.tensor([[0, 0]])
    # the first is certain (p > q); the second is kept while u < 0.125 / 0.5
    tokens, n = ops.verify_draft(p, x, torch.tensor([[0.9, 0.2, 0.3]]), q)
    assert tokens.tolist() == [[0, 0, 1]] and n.tolist() == [2]
    tokens, n = ops.verify_draft(p, x, torch.tensor([[0.9, 0.25, 0.3]]), q)  # refused: max(p - q, 0) is (0, .5, 0)
    assert tokens.tolist() == [[0, 1, -1]] and n.tolist() == [1]
    tokens, n = ops.verify_draft(p, x, torch.tensor([[0.5, 0.0, 0.25]]))  # a certain draft: u < p, without its id
    assert tokens.tolist() == [[1, -1, -1]] and n.tolist() == [0]
    tokens, n = ops.verify_draft(p, x, torch.tensor([[0.9, 0.9, 0.5]]), q, torch.tensor([0]))  # no draft: p itself
    assert tokens.tolist() == [[1, -1, -1]] and n.tolist() == [0]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("p0,q0,kept", [(INF, 0.5, False), (NAN, 0.5, False), (-0.5, 0.5, False), (0.0, -0.5, False),
                                        (0.0, INF, False), (0.0, NAN, False), (0.5, NAN, True), (0.5, INF, True),
                                        (0.5, -0.5, True), (0.5, 0.0, True), (-0.25, -0.5, False), (INF, NAN, False)])
@pytest.mark.parametrize("u", [0.0, 0.5])
def test_acceptance_of_weights_that_are_none(device, p0, q0, kept, u):
    """A drafted id whose probability is negative, infinite or NaN on either side: 0 there, as in the sums. A refused
    one is followed by id 1, all that is left, an accepted one by id 2."""
    p = torch.tensor([[[p0, 0.5, 0.0], [0.0, 0.0, 1.0]]], device=device)
    q = torch.tensor([[[q0, 0.25, 0.0]]], device=device)
    x, us = torch.tensor([[0]], device=device), torch.tensor([[u, 0.5]], device=device)
    tokens, n = ops.verify_draft(p, x, us, q)
    assert tokens.tolist() == ([[0, 2]] if kept else [[1, -1]]) and n.tolist() == [int(kept)]
    if q0 == 0.5 and kept is False:  # a certain draft
        tokens, n = ops.verify_draft(p, x, us)
        assert tokens.tolist() == [[1, -1]] and n.tolist() == [0]


def test_samples_are_the_targets():
    """Over many draws the emitted first token has the target's probabilities."""
    g = torch.Generator().manual_seed(3)
    n = 4000
    p = torch.tensor([0.5, 0.2, 0.3]).expand(n, 2, 3)
    q = torch.tensor([0.2, 0.5, 0.3]).expand(n, 1, 3)
    x = torch.multinomial(q[:, 0], 1, generator=g)
    tokens, _ = ops.verify_draft(p, x, torch.rand(n, 2, generator=g), q)
    share = torch.bincount(tokens[:, 0], minlength=3) / n
    assert (share - p[0, 0]).abs().max() < 5 * (0.25 / n) ** 0.5  # five standard deviations


def test_refusals():
    p, x, u, q = data(2, 3, 10)
    for bad in ((p[0], x, u, q), (p, x[:, :2], u, q), (p, x, u[:, :3], q), (p, x, u, q[..., :9]),
                (p, x, u, q, torch.zeros(3, dtype=torch.int32)), (p[..., :0], x, u, q[..., :0]), (p[:, :0], x, u),
                (p[:1, :1, :1].expand(1, 1, 2 ** 30 + 1), x[:1, :0], u[:1, :1])):
        with pytest.raises(ValueError):
            ops.verify_draft(*bad)
    for bad in ((p.double(), x, u, q.double()), (p, x.float(), u, q), (p, x, u.double(), q), (p, x, u, q.half()),
                (p, x, u, q, torch.ones(2))):
        with pytest.raises(TypeError):
            ops.verify_draft(*bad)


# ------------------------------------------------------------------ kernel
@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 4, 32000), (3, 0, 100), (5, 2, 7), (40, 7, 1003), (9, 40, 257), (2, 3, 128256),
                                   (1, 2, 300001), (300, 1, 64), (0, 3, 50), (17, 5, 4099)])
def test_kernel(dtype, draft, B, K, V):
    p, x, u, q = data(B, K, V, dtype, B + V)
    lens = torch.randint(0, K + 1, (B,), generator=torch.Generator().manual_seed(1), dtype=torch.int32) if B % 2 else None
    q = q if draft else None
    want = verify_draft_ref(p, x, u, q, lens)
    cuda = [None if t is None else t.cuda() for t in (p, x, u, q, lens)]
    same(ops.verify_draft(*cuda), want)


@gpu
@pytest.mark.parametrize("V", [5, 1000, 70000])
@pytest.mark.parametrize("u", [0.0, 0.25, 0.5, 1 - 2.0 ** -24, 1.0])
def test_borders(V, u):
    """Numbers at the ends and on the borders between ids; weights that are exact in 64 bits."""
    p = torch.zeros(6, 2, V)
    p[0, :, 0] = 1
    p[1, :, -1] = 1
    p[2] = 2.0 ** -20
    p[3, :, V // 2:V // 2 + 2] = 0.5
    p[4, :, ::2] = 2.0 ** -10
    p[5, :, [0, -1]] = 0.5
    x = torch.zeros(6, 1, dtype=torch.long)
    us = torch.full((6, 2), u)
    for q in (None, p[:, :1].clone(), torch.zeros(6, 1, V)):
        for lens in (None, torch.zeros(6, dtype=torch.int32)):
            want = verify_draft_ref(p, x, us, q, lens)
            same(ops.verify_draft(*(None if t is None else t.cuda() for t in (p, x, us, q, lens))), want)


@gpu
def test_weights_and_ids_that_are_none():
    p, x, u, q = data(12, 3, 200, seed=4)
    p[0] = 0
    p[1, :, ::3] = NAN
    p[2, :, 5] = INF
    p[3] = -p[3]
    q[4] = NAN
    q[5] = p[5, :3]
    u[5] = 0.999
    p[6, 0] = q[6, 0] * 0.5  # nothing left of p - q
    u[6] = 0.9
    x[7, 1] = 200
    x[8, 0] = -1
    x[9, 2] = 10 ** 12
    u[10] = NAN
    lens = torch.tensor([3, 2, 1, 0, 3, 3, 3, 3, 3, 3, -4, 99], dtype=torch.int32)
    for qq in (q, None):
        want = verify_draft_ref(p, x, u, qq, lens)
        same(ops.verify_draft(*(None if t is None else t.cuda() for t in (p, x, u, qq, lens))), want)
    assert verify_draft_ref(p, x, u, q, lens)[0][0].tolist() == [-1] * 4


@gpu
def test_strides_and_index_types():
    p, x, u, q = data(4, 3, 500, seed=5)
    want = verify_draft_ref(p, x, u, q)
    big = torch.zeros(4, 6, 517)
    big[:, 1:5, 3:503] = p
    bq = torch.zeros(3, 4, 500)
    bq[:] = q.transpose(0, 1)
    got = ops.verify_draft(big.cuda()[:, 1:5, 3:503], x.int().cuda(), u.t().contiguous().cuda().t(), bq.cuda().transpose(0, 1),
                           torch.full((4,), 2 ** 32 + 3).cuda())
    same(got, want)
    turned = p.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    same(ops.verify_draft(turned, x.cuda(), u.cuda(), q.cuda()), want)


@gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.uint16, torch.int32, torch.int64])
def test_lengths_of_any_whole_type(dtype):
    """More drafted tokens than the lengths' own type counts."""
    K = 40000 if dtype in (torch.int16, torch.uint16) else 300
    p = torch.full((3, 1, 4), 0.25, device="cuda").expand(3, K + 1, 4)
    x = torch.zeros(3, K, dtype=torch.long, device="cuda")
    u = torch.zeros(3, K + 1, device="cuda")
    lens = torch.tensor([0, 3, 100]).to(dtype)
    tokens, n = ops.verify_draft(p, x, u, None, lens.cuda())
    assert n.tolist() == [0, 3, 100] and (tokens >= 0).sum(1).tolist() == [1, 4, 101]


@gpu
def test_rows_beyond_32_bit_offsets():
    """The last sequence starts more than 2^31 values into the target's probabilities."""
    V, B = 128256, 2100
    p = torch.zeros(B, 8, V, device="cuda", dtype=torch.bfloat16)
    x = torch.full((B, 7), 3, device="cuda")
    p[-1, :, 3] = 1
    p[-1, 7, 3] = 0
    p[-1, 7, V - 2] = 1
    tokens, n = ops.verify_draft(p, x, torch.full((B, 8), 0.5, device="cuda"))
    assert tokens[-1].tolist() == [3] * 7 + [V - 2] and n[-1] == 7
    assert (tokens[:-1] == -1).all() and (n[:-1] == 0).all()


@gpu
def test_captured_graph_on_another_stream():
    p, x, u, q = (t.cuda() for t in data(20, 4, 3001, seed=6))
    first = ops.verify_draft(p, x, u, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = ops.verify_draft(p, x, u, q)
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], first[0])
    u.copy_(torch.rand(20, 5, generator=torch.Generator().manual_seed(7)))
    graph.replay()
    same(got, verify_draft_ref(p.cpu(), x.cpu(), u.cpu(), q.cpu()))

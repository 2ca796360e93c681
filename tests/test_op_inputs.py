"""What the ops' shared helpers refuse and count, whichever op calls them."""
import pytest
import torch

from brain_b200 import ops
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

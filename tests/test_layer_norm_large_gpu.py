"""Layer norm's sums over many rows, whose arrays pass the last cache, element by element against 64 bits."""
import pytest
import torch

from adhip import operators as ops
from test_operators_gpu import TYPES, here

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,size", [(16000, 4099), (32000, 4096), (200003, 130)])
def test_sums_over_many_rows(hip_device, rows, size, dtype):
    """What is summed up is taken from the statistics that the forward pass left.  A lane's product with its row's mean and root is off by
    two roundings; an addend passes the additions of the rows that one of at least 256 lanes meets, 16 in its wavefront or between
    wavefronts, two between a wavefront's groups and 32 between workgroups."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, dy = (torch.randn((rows, size), generator=g, device="cuda").to(TYPES[dtype]) for _ in range(2))
    out, dx, stats = torch.empty_like(x), torch.empty_like(x), torch.empty((rows, 2), device="cuda")
    dw, db = (torch.full((size,), 7.0, device="cuda") for _ in "wb")
    room = torch.empty(ops.layer_norm_workspace(hip_device, x), dtype=torch.uint8, device="cuda").fill_(255)
    ops.layer_norm(hip_device, x, out, stats=stats, stream=here())
    ops.layer_norm_backward(hip_device, x, stats, dy, dx, weight_grad=dw, bias_grad=db, workspace=room, stream=here())
    additions = -(-rows // 256) + 16 + 2 + 32
    n = (x.double() - stats[:, :1].double()) * stats[:, 1:].double()
    for got, addends, own in ((dw, dy.double() * n, 2), (db, dy.double(), 0)):
        bound = (additions + own) * U * addends.abs().sum(0)
        off = (got.double() - addends.sum(0)).abs()
        assert bool((off <= bound).all()), float((off / bound).max())

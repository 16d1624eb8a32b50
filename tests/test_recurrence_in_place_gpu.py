"""Recurrences whose results take the place of what they are made from, against the same calls on arrays apart: the same bits."""
import pytest
import torch

from adhip import operators as ops
from test_operators_gpu import TYPES, here, to_gpu
from test_recurrence_gpu import inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("B,L,C", [(2, 600, 300), (1, 5000, 40), (1, 9001, 930), (2, 3000, 33)])
def test_a_gradient_in_place_over_long_sequences(hip_device, B, L, C, factors, dtype):
    """The first range of positions writes the gradient that the last one begins with."""
    a = inputs(B, L, C, dtype, factors=factors, seed=4, slow=8.0)
    want = run(hip_device, a, factors=factors)
    a = {n: to_gpu(x) for n, x in a.items()}
    room = torch.empty(ops.recurrence_workspace(hip_device, a["x"], backward=True) + 16, dtype=torch.uint8, device="cuda")
    for _ in range(3):
        grad, x_grad, gates_grad = a["final_grad"].clone(), torch.empty_like(a["x"]), torch.empty_like(a["x"])
        ops.recurrence_backward(hip_device, a["x"], a["gates"], want["states"], a["out_grad"], x_grad, gates_grad, factors=factors, final_grad=grad,
                                initial_grad=grad, workspace=room, stream=here())
        assert torch.equal(x_grad, want["x_grad"]) and torch.equal(gates_grad, want["gates_grad"]) and torch.equal(grad, want["initial_grad"])


ODD = [(2, L, C) for L in (4, 600, 3000) for C in (33, 35, 65)] + [(9, 600, 1857), (9, 600, 1925), (1, 9001, 1857), (1, 9001, 1925)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("B,L,C", ODD)
def test_channels_that_fill_no_pack_in_place(hip_device, B, L, C, factors, dtype):
    """Of bf16, the last pack of a row begins before its place and two lanes own a channel (35, 1925), or the last channel is alone in its
    workgroup (33, 65, 1857), in rows of 64 and of 128 bytes, in one range and in several."""
    a = inputs(B, L, C, dtype, factors=factors, seed=9)
    want = run(hip_device, a, factors=factors)
    a = {n: to_gpu(x) for n, x in a.items()}
    room = torch.empty(ops.recurrence_workspace(hip_device, a["x"], backward=True) + 16, dtype=torch.uint8, device="cuda")
    how = dict(factors=factors, workspace=room, stream=here())
    for n in ("x", "gates"):
        g = {k: None if v is None else v.clone() for k, v in a.items()}
        ops.recurrence(hip_device, g["x"], g["gates"], g[n], initial=g["initial"], final=g["initial"], **how)
        assert torch.equal(g[n], want["out"]) and torch.equal(g["initial"], want["final"])
    for to in (("x", "gates"), ("out_grad", "x"), ("gates", "out_grad")):
        g = {k: None if v is None else v.clone() for k, v in a.items()}
        ops.recurrence_backward(hip_device, g["x"], g["gates"], want["states"], g["out_grad"], g[to[0]], g[to[1]], final_grad=g["final_grad"],
                                initial_grad=g["final_grad"], **how)
        assert torch.equal(g[to[0]], want["x_grad"]) and torch.equal(g[to[1]], want["gates_grad"]) and torch.equal(g["final_grad"], want["initial_grad"])

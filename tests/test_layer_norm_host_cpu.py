"""Layer norm's kernels on the host (host_operators.py), with workgroups in either order: a result must not depend on it."""
import os

import pytest
import torch

import host_operators as host
import training_oracle as oracle
from adhip import operators as ops

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev(tmp_path_factory):
    if not os.path.exists(host.CLANG):
        pytest.skip("no clang to build the kernels with")
    return host.build(str(tmp_path_factory.mktemp("kernels")), "layer_norm")


def inputs(rows, size, dtype):
    g = torch.Generator().manual_seed(size)
    a = {n: torch.randn((rows, size), generator=g).to(TYPES[dtype]) for n in ("x", "out_grad", "total_grad")}
    return a | {"weight": 1 + 0.3 * torch.randn(size, generator=g), "bias": torch.randn(size, generator=g)}


def run(dev, a, *, one=False):
    """Both passes; with `one` the sums over rows are asked for in one array."""
    (rows, size), new = a["x"].shape, lambda *s: torch.full(s, 7.0)
    r = {"out": torch.full_like(a["x"], 7.0), "stats": new(rows, 2), "x_grad": torch.full_like(a["x"], 7.0), "weight_grad": new(size), "bias_grad": new(size)}
    if one:
        r["weight_grad"] = r["bias_grad"]
    h = {n: host.seen(t) for n, t in {**a, **r}.items()}
    ops.layer_norm(dev, h["x"], h["out"], weight=h["weight"], bias=h["bias"], stats=h["stats"], stream=0)
    ops.layer_norm_backward(dev, h["x"], h["stats"], h["out_grad"], h["x_grad"], weight=h["weight"], weight_grad=h["weight_grad"],
                            bias_grad=h["bias_grad"], total_grad=h["total_grad"], workspace=host.room(ops.layer_norm_workspace(dev, h["x"])), stream=0)
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,size", [(5, 3), (70, 40), (9, 128), (6, 500), (3, 1025), (20, 2048)])
def test_the_host_runs_the_kernels(dev, rows, size, dtype):
    a = inputs(rows, size, dtype)
    want, bound = oracle.layer_norm(a["x"], a["weight"], a["bias"], out_grad=a["out_grad"], total_grad=a["total_grad"])
    first, last = dev.in_both_orders(lambda: run(dev, a))
    for n in first:
        off = (first[n].double() - want[n]).abs()
        assert bool((off <= bound[n]).all()), (n, float((off / bound[n]).max()))
        assert torch.equal(first[n], last[n]), n


@pytest.mark.parametrize("size", [5, 300])
def test_one_array_for_both_sums_holds_the_bias_gradient(dev, size):
    a = inputs(20, size, "f32")
    want = run(dev, a)
    for got in dev.in_both_orders(lambda: run(dev, a, one=True)):
        assert torch.equal(got["bias_grad"], want["bias_grad"]) and torch.equal(got["x_grad"], want["x_grad"])


def test_sums_that_share_memory_are_refused(dev):
    """Apart from one array for both, and from halves of one."""
    a = inputs(6, 40, "f32")
    h, both = {n: host.seen(t) for n, t in a.items()}, torch.full((100,), 7.0)
    stats, dx, room = host.seen(torch.ones(6, 2)), host.seen(torch.empty(6, 40)), host.room(ops.layer_norm_workspace(dev, h["x"]))

    def call(weight_grad, bias_grad):
        ops.layer_norm_backward(dev, h["x"], stats, h["out_grad"], dx, weight=h["weight"], weight_grad=host.seen(weight_grad),
                                bias_grad=host.seen(bias_grad), workspace=room, stream=0)

    for weight_grad, bias_grad in ((both[:40], both[39:79]), (both[39:79], both[:40]), (both[:40], both.view(torch.bfloat16)[:40]),
                                   (both.view(torch.bfloat16)[78:118], both[:40])):
        with pytest.raises(RuntimeError, match="weight_grad and bias_grad share memory"):
            call(weight_grad, bias_grad)
    assert (both == 7).all()
    call(both[:40], both[40:80])
    assert (both[:80] != 7).any() and (both[80:] == 7).all()

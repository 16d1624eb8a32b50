"""The norm over all gradients, clipping by it and AdamW behind it (adhip.operators) against a plain 64-bit restatement
(training_oracle.py).  Tolerances are the oracle's bounds."""
import math

import pytest
import torch

import training_oracle as oracle
from adhip import operators as ops
from test_operators_gpu import TYPES, assert_within, here

pytestmark = pytest.mark.gpu


def gradients(counts, dtype, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    kinds = [TYPES[dtype]] if dtype in TYPES else [torch.float32, torch.bfloat16]
    return [(torch.randn(n, generator=g) * size).to(kinds[i % len(kinds)]) for i, n in enumerate(counts)]


def run(dev, gs, limit, *, grad_scale=1.0, outs=None, clip=True):
    norm, factor = torch.full((1,), 7.0, device="cuda"), torch.full((1,), 7.0, device="cuda")
    room = torch.empty(ops.gradient_norm_workspace(dev, gs), dtype=torch.uint8, device="cuda").fill_(255)
    how = dict(limit=limit, factor=factor, grad_scale=grad_scale, workspace=room, stream=here())
    if clip:
        ops.clip_gradients(dev, gs, norm, gradients_out=outs, **how)
    else:
        ops.gradient_norm(dev, gs, norm, **how)
    torch.cuda.synchronize()
    return {"norm": norm, "factor": factor, "g": gs if outs is None else outs}


def check(dev, host, what, limit=1.0, grad_scale=1.0, in_place=False, clip=True):
    gs = [g.cuda() for g in host]
    outs = None if in_place or not clip else [torch.full_like(g, 7.0) for g in gs]
    got = run(dev, gs, limit, grad_scale=grad_scale, outs=outs, clip=clip)
    want, bound = oracle.clip(host, limit, grad_scale)
    for n in ("norm", "factor"):
        assert_within(got[n], want[n], bound[n], f"{what}: {n}")
    for i in range(len(host) if clip else 0):
        assert_within(got["g"][i], want["g"][i], bound["g"][i], f"{what}: gradient {i}")
    if not in_place:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(gs, host)), "inputs are left alone"


LISTS = {
    "one number": [1],
    "the README's perceptron": [12, 4, 8, 2],
    "ends of packs": [1, 3, 4, 5, 7, 8, 9, 15, 16, 17, 255, 256, 257, 1023, 1025, 2047],
    "ends of chunks": [16383, 16384, 16385, 32768, 50001],
    "empty ones among them": [0, 5, 0, 0, 4000, 0],
    "more than a launch holds": [1 + (37 * i) % 500 for i in range(300)],
    "one large": [3_000_001],
}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "both"])
@pytest.mark.parametrize("name", LISTS)
def test_lists(hip_device, name, dtype):
    host = gradients(LISTS[name], dtype, seed=len(name))
    check(hip_device, host, f"{name}, {dtype}")
    check(hip_device, host, f"{name}, {dtype}, below the limit", limit=1e6)
    check(hip_device, host, f"{name}, {dtype}, in place", limit=0.5, grad_scale=-0.25, in_place=True)
    check(hip_device, host, f"{name}, {dtype}, norm alone", limit=math.inf, grad_scale=3.0, clip=False)


@pytest.mark.parametrize("dtype", TYPES)
def test_arrays_that_begin_anywhere(hip_device, dtype):
    base = gradients([5000], dtype)[0]
    gs = [base.cuda()[i:i + 700 + i] for i in range(1, 6)]
    host = [g.cpu() for g in gs]
    outs = [torch.full((g.numel() + 3,), 7.0, dtype=g.dtype, device="cuda") for g in gs]
    got = run(hip_device, gs, 0.1, outs=[o[1:-2] for o in outs])
    want, bound = oracle.clip(host, 0.1)
    for i, o in enumerate(outs):
        assert_within(got["g"][i], want["g"][i], bound["g"][i], f"gradient {i}, {dtype}")
        assert (o[0] == 7).all() and (o[-2:] == 7).all()
    assert_within(got["norm"], want["norm"], bound["norm"], "norm")


def test_squares_beyond_32_bits(hip_device):
    """Numbers whose squares f32 does not hold, above and below, and their sum."""
    for size in (1e30, 1e-30, 3e38, 1e-38):
        check(hip_device, [torch.tensor([size, -size, size / 3] * 50)], f"{size}")
    check(hip_device, [torch.full((100000,), 3e38)], "a norm beyond f32", limit=1e30)


def test_no_gradients(hip_device):
    for gs in ([], [torch.empty(0, device="cuda")]):
        got = run(hip_device, gs, 1.0)
        assert float(got["norm"]) == 0.0 and float(got["factor"]) == 1.0


def test_gradients_that_are_not_finite_show(hip_device):
    gs = gradients([500, 40000], "f32")
    gs[1][39999] = float("nan")
    got = run(hip_device, [g.cuda() for g in gs], 1.0)
    assert got["norm"].isnan().all() and got["factor"].isnan().all() and all(g.isnan().all() for g in got["g"])
    gs[1][39999] = float("-inf")
    got = run(hip_device, [g.cuda() for g in gs], 1.0)
    assert got["norm"].isinf().all() and float(got["factor"]) == 0.0
    assert not got["g"][0].any() and not got["g"][1][:-1].any() and got["g"][1][-1].isnan()
    got = run(hip_device, [g.cuda() for g in gs], math.inf)
    assert got["norm"].isinf().all() and float(got["factor"]) == 1.0 and torch.equal(got["g"][1].cpu(), gs[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_factor_of_one_changes_no_bit(hip_device, dtype):
    host = gradients([10, 70000], dtype, size=1e-3)
    got = run(hip_device, [g.cuda() for g in host], 100.0)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got["g"], host))


def test_the_same_gradients_give_the_same_bits(hip_device):
    gs = [g.cuda() for g in gradients(LISTS["ends of chunks"], "both", seed=3)]
    norms = {float(run(hip_device, gs, 1.0, clip=False)["norm"]) for _ in range(4)}
    assert len(norms) == 1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", TYPES)
def test_adamw_takes_the_factor_from_the_device(hip_device, dtype, bits):
    """The same bits as with the factor given from the host, and without one as before."""
    g = torch.Generator().manual_seed(5)
    counts = [5, 1000, 256, 70001]
    gs = [x.cuda() for x in gradients(counts, dtype, seed=6)]
    factor = torch.full((1,), 7.0, device="cuda")
    room = torch.empty(ops.gradient_norm_workspace(hip_device, gs), dtype=torch.uint8, device="cuda")
    ops.gradient_norm(hip_device, gs, torch.empty(1, device="cuda"), limit=2.0, factor=factor, grad_scale=0.5, workspace=room, stream=here())
    p0 = [torch.randn(n, generator=g).to(TYPES[dtype]) for n in counts]

    def step(**how):
        p = [x.cuda() for x in p0]
        if bits == 32:
            states = {n: [torch.zeros(c, device="cuda") for c in counts] for n in ("first", "second")}
        else:
            blocks = [ops.adamw_blocks(c) for c in counts]
            states = {n: [torch.zeros((b, 256), device="cuda").to(torch.float8_e4m3fn) for b in blocks] for n in ("first", "second")}
            states |= {n: [torch.zeros(b, device="cuda") for b in blocks] for n in ("first_scales", "second_scales")}
        ops.adamw(hip_device, p, gs, step=1, rate=0.1, stream=here(), **states, **how)
        return p + [x for n in states for x in states[n]]

    half = float(factor)  # (a power of two times a 32-bit number is exact, in whatever width it is multiplied)
    assert 0.0 < half < 1.0
    for a, b in zip(step(factor=factor, grad_scale=0.5), step(grad_scale=0.5 * half)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    one = torch.ones(1, device="cuda")
    for a, b in zip(step(factor=one, grad_scale=0.3), step(grad_scale=0.3)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))

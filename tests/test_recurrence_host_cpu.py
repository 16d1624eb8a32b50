"""The recurrence's kernels on the host (host_operators.py), where workgroups run one after the other: what a call reads late, after
others of its workgroups have ended, shows every time."""
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
    return host.build(str(tmp_path_factory.mktemp("kernels")), "recurrence")


def inputs(B, L, C, dtype, *, factors=False, seed=0, slow=3.0, masked=False):
    g = torch.Generator().manual_seed(seed)
    gates = torch.randn((B, L, C), generator=g) + slow * torch.rand(C, generator=g)
    a = {"x": torch.randn((B, L, C), generator=g), "gates": torch.sigmoid(gates) if factors else gates, "out_grad": torch.randn((B, L, C), generator=g)}
    a = {n: x.to(TYPES[dtype]) for n, x in a.items()}
    a["initial"], a["final_grad"] = torch.randn((B, C), generator=g), torch.randn((B, C), generator=g)
    a["documents"] = torch.cumsum(torch.rand((B, L), generator=g) < 0.001, 1).to(torch.int32) if masked else None
    a["lengths"] = torch.tensor([L - 300] * B, dtype=torch.int32) if masked else None
    return a


def run(dev, a, *, factors=False, in_place=False):
    """Both passes; with `in_place` the state and its gradient are carried in one array each."""
    x, (B, L, C) = a["x"], a["x"].shape
    new = lambda *s: torch.full(s, 7.0)  # noqa: E731
    r = {n: torch.full_like(x, 7.0).as_strided(x.shape, x.stride()) for n in ("out", "x_grad", "gates_grad")} | {"states": new(B, ops.recurrence_blocks(L), C)}
    initial, final_grad = a["initial"].clone(), a["final_grad"].clone()
    r["final"], r["initial_grad"] = (initial, final_grad) if in_place else (new(B, C), new(B, C))
    h = {n: host.seen(t) for n, t in {**a, **r, "initial": initial, "final_grad": final_grad}.items()}
    how = dict(factors=factors, lengths=h["lengths"], documents=h["documents"], stream=0,
               workspace=host.room(ops.recurrence_workspace(dev, h["x"], backward=True)))
    ops.recurrence(dev, h["x"], h["gates"], h["out"], initial=h["initial"], final=h["final"], states=h["states"], **how)
    ops.recurrence_backward(dev, h["x"], h["gates"], h["states"], h["out_grad"], h["x_grad"], h["gates_grad"], final_grad=h["final_grad"],
                            initial_grad=h["initial_grad"], **how)
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,C,masked", [(1, 20, 33, False), (2, 700, 9, False), (1, 5000, 40, False), (1, 5000, 40, True)])
def test_the_host_runs_the_kernels(dev, B, L, C, masked, dtype):
    """(exp2 and quotients are the host's, within the oracle's bounds)"""
    a = inputs(B, L, C, dtype, masked=masked)
    got = run(dev, a)
    want, bound = oracle.recurrence(a["x"], a["gates"], initial=a["initial"], lengths=a["lengths"], documents=a["documents"], out_grad=a["out_grad"],
                                    final_grad=a["final_grad"])
    for n in got:
        off = (got[n].double() - want[n]).abs()
        assert bool((off <= bound[n]).all()), (n, float((off / bound[n]).max()))


CARRIED = [(B, L, C, masked, factors, dtype) for B, L, C, masked in ((1, 300, 40, False), (1, 5000, 40, False), (2, 3000, 33, True))
           for factors in (False, True) for dtype in TYPES] + [(1, 9001, 930, False, False, "f32")]


@pytest.mark.parametrize("B,L,C,masked,factors,dtype", CARRIED)
def test_states_and_their_gradients_are_carried_in_place(dev, B, L, C, masked, factors, dtype):
    """Over several ranges of positions the first one writes the gradient that the last one begins with (forwards, the last one the state
    that the first one begins with)."""
    a = inputs(B, L, C, dtype, factors=factors, seed=4, slow=8.0, masked=masked)
    apart = run(dev, a, factors=factors)
    for carried in dev.in_both_orders(lambda: run(dev, a, factors=factors, in_place=True)):
        for n in apart:
            assert torch.equal(apart[n], carried[n]), n


@pytest.mark.parametrize("dtype", TYPES)
def test_one_position_has_no_distance_to_speak_of(dev, dtype):
    """One token of arrays that have all sequences of a position beside one another, however many those are."""
    a = inputs(3, 1, 40, dtype)
    want = run(dev, a)
    for n in ("x", "gates", "out_grad"):
        a[n] = a[n].as_strided((3, 1, 40), (40, 1 << 40, 1))
    got = run(dev, a)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("L,C", [(L, C) for L in (4, 300, 1100) for C in (33, 35)])
def test_channels_that_fill_no_pack_in_place(dev, L, C, factors):
    """The last pack of a row that begins before its place, and a last channel alone in its workgroup."""
    a = inputs(2, L, C, "bf16", factors=factors)
    want = run(dev, a, factors=factors)

    def forward(to):
        g = {n: None if t is None else t.clone() for n, t in a.items()}
        h = {n: host.seen(t) for n, t in g.items()}
        ops.recurrence(dev, h["x"], h["gates"], h[to], factors=factors, initial=h["initial"], final=h["initial"], stream=0,
                       workspace=host.room(ops.recurrence_workspace(dev, h["x"])))
        return g[to], g["initial"]

    def backward(to):
        g = {n: None if t is None else t.clone() for n, t in a.items()}
        h = {n: host.seen(t) for n, t in g.items()}
        ops.recurrence_backward(dev, h["x"], h["gates"], host.seen(want["states"]), h["out_grad"], h[to[0]], h[to[1]], factors=factors,
                                final_grad=h["final_grad"], initial_grad=h["final_grad"], stream=0,
                                workspace=host.room(ops.recurrence_workspace(dev, h["x"], backward=True)))
        return g[to[0]], g[to[1]], g["final_grad"]

    for to in ("x", "gates"):
        for out, final in dev.in_both_orders(lambda: forward(to)):
            assert torch.equal(out, want["out"]) and torch.equal(final, want["final"])
    for to in (("x", "gates"), ("out_grad", "x"), ("gates", "out_grad")):
        for got in dev.in_both_orders(lambda: backward(to)):
            assert all(torch.equal(g, want[n]) for g, n in zip(got, ("x_grad", "gates_grad", "initial_grad")))

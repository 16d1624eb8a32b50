"""The norm over gradients and clipping on the host (host_operators.py), kernels and all: which bits an address decides."""
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
    return host.build(str(tmp_path_factory.mktemp("kernels")), "gradients")


def at(t, off):
    """A copy that begins `off` elements behind a multiple of 16 bytes, between elements that must not change."""
    room = torch.full((t.numel() + 64,), 7.0, dtype=t.dtype)
    first = -room.data_ptr() % 16 // t.element_size() + 16 + off
    copy = room[first:first + t.numel()]
    copy.copy_(t)
    assert copy.data_ptr() % 16 == off * t.element_size() % 16
    return copy


def run(dev, gradients, outs=None):
    """norm, factor and the workgroups' sums, of the norm alone or with clipped gradients written to `outs`."""
    h, norm, factor = [host.seen(g) for g in gradients], torch.full((1,), 7.0), torch.full((1,), 7.0)
    room = host.room(ops.gradient_norm_workspace(dev, h))
    how = dict(limit=1.5, factor=host.seen(factor), workspace=room, stream=0)
    if outs is None:
        ops.gradient_norm(dev, h, host.seen(norm), **how)
    else:
        ops.clip_gradients(dev, h, host.seen(norm), gradients_out=[host.seen(o) for o in outs], **how)
    return norm, factor, room.t[:-8].clone()


SIZES = [[3, 1, 900], [20000, 5, 70001], [30000]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_the_host_runs_the_kernels(dev, sizes, dtype):
    g = [torch.randn(n, generator=torch.Generator().manual_seed(n)).to(TYPES[dtype]) for n in sizes]
    outs = [torch.full_like(x, 7.0) for x in g]
    norm, factor, _ = run(dev, g, outs)
    want, bound = oracle.clip(g, 1.5)
    assert (norm.double() - want["norm"]).abs() <= bound["norm"] and (factor.double() - want["factor"]).abs() <= bound["factor"]
    for o, x in zip(outs, g):
        assert torch.equal(o, (x.float() * factor).to(x.dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_addresses_decide_over_no_bit(dev, sizes, dtype):
    """Views of odd sizes in one buffer are a usual home of gradients.  Sums, and what is made of them, are those of aligned copies,
    for the norm alone and with clipped gradients anywhere."""
    g = [torch.randn(n, generator=torch.Generator().manual_seed(n)).to(TYPES[dtype]) for n in sizes]
    plain = run(dev, [at(x, 0) for x in g])
    outs = [at(x, 0) for x in g]
    run(dev, [at(x, 0) for x in g], outs)
    for off, to in ((1, None), (3, None), (0, 1), (1, 0), (5, 2)):
        there = [at(torch.full_like(x, 7.0), to) for x in g] if to is not None else None
        got = run(dev, [at(x, off) for x in g], there)
        assert all(torch.equal(a, b) for a, b in zip(got, plain)), (off, to)
        if there is not None:
            for a, b in zip(there, outs):
                assert torch.equal(a, b)
                assert a.storage_offset() > 0 and (a._base[:a.storage_offset()] == 7).all() and (a._base[a.storage_offset() + a.numel():] == 7).all()

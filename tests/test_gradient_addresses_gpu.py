"""The norm over gradients and clipping where gradients begin at any element: views of odd sizes in one buffer, as a flat buffer of
all gradients holds them, give the bits of aligned copies."""
import pytest
import torch

from adhip import operators as ops
from test_operators_gpu import TYPES, here

pytestmark = pytest.mark.gpu


def views(xs, off):
    """Copies of all of them, one behind the other, the first one `off` elements behind an aligned address; and the whole buffer."""
    buffer = torch.full((sum(x.numel() for x in xs) + off + 9,), 7.0, dtype=xs[0].dtype, device="cuda")
    out, at = [], off
    for x in xs:
        out.append(buffer[at:at + x.numel()])
        out[-1].copy_(x)
        at += x.numel()
    return out, buffer


def clip(dev, g, outs, limit=1.5):
    norm, factor = torch.full((1,), 7.0, device="cuda"), torch.full((1,), 7.0, device="cuda")
    room = torch.empty(ops.gradient_norm_workspace(dev, g), dtype=torch.uint8, device="cuda").fill_(255)
    if outs is None:
        ops.gradient_norm(dev, g, norm, limit=limit, factor=factor, workspace=room, stream=here())
    else:
        ops.clip_gradients(dev, g, norm, limit=limit, factor=factor, gradients_out=outs, workspace=room, stream=here())
    torch.cuda.synchronize()
    return norm, factor, room[:-8]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [3, 900, 7], [8191, 5, 8192, 8193], [70001, 1, 300003, 4096], [45_000_001, 33_000_003]])
def test_addresses_decide_over_no_bit(hip_device, sizes, dtype):
    """The largest ones are written past the caches."""
    g = [torch.randn(n, device="cuda").to(TYPES[dtype]) for n in sizes]
    plain = clip(hip_device, g, None)
    outs = [torch.full_like(x, 7.0) for x in g]
    assert all(torch.equal(a, b) for a, b in zip(clip(hip_device, g, outs), plain))
    factor = float(plain[1])
    assert all(torch.equal(o, (x.float() * factor).to(x.dtype)) for o, x in zip(outs, g))
    for off, to in ((1, None), (0, 1), (3, 0), (3, 6), (1, "in place")):
        there, _ = views(g, off)
        if to == "in place":
            got, buffer = clip(hip_device, there, there), there[0]._base
            made, to = there, off
        elif to is None:
            got, made = clip(hip_device, there, None), None
        else:
            made, buffer = views([torch.full_like(x, 7.0) for x in g], to)
            got = clip(hip_device, there, made)
        assert all(torch.equal(a, b) for a, b in zip(got, plain)), (off, to)
        if made is not None:
            assert all(torch.equal(a, b) for a, b in zip(made, outs)), (off, to)
            assert (buffer[:to] == 7).all() and (buffer[to + sum(sizes):] == 7).all()

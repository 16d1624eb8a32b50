"""Layer norm on device arrays (adhip.operators) against a plain 64-bit restatement (training_oracle.py), at the sizes, layouts and
values where it can go wrong.  Tolerances are the oracle's bounds, element by element."""
import pytest
import torch

import training_oracle as oracle
from adhip import operators as ops
from test_operators_gpu import TYPES, assert_within, here, to_gpu

pytestmark = pytest.mark.gpu


def inputs(shape, dtype, weights, seed=0, level=0.5):
    g = torch.Generator().manual_seed(seed)
    size = shape[-1]
    a = {"x": torch.randn(shape, generator=g) * torch.exp(torch.randn(size, generator=g) * 0.5) + level}
    a |= {n: torch.randn(shape, generator=g) for n in ("added", "out_grad", "total_grad")}
    a = {n: x.to(TYPES[dtype]) for n, x in a.items()}
    a["weight"] = (1 + 0.3 * torch.randn(size, generator=g)).to(TYPES[weights])
    a["bias"] = torch.randn(size, generator=g).to(TYPES[weights])
    return a


def run(dev, a, *, eps=1e-5, centered=True, adds=True, affine=True, grad_type=None, backward=True, like=torch.empty_like):
    """Forward and backward; every output begins as numbers that must not survive."""
    a = {n: to_gpu(x) for n, x in a.items()}
    new = lambda x: like(x).fill_(7.0)  # noqa: E731
    weight, bias = (a["weight"], a["bias"]) if affine else (None, None)
    out, stats = new(a["x"]), torch.full((*a["x"].shape[:-1], 2), 7.0, device="cuda")
    total = new(a["x"]) if adds else None
    ops.layer_norm(dev, a["x"], out, weight=weight, bias=bias, eps=eps, centered=centered, added=a["added"] if adds else None, total=total,
                   stats=stats, stream=here())
    r = {"out": out, "stats": stats} | ({"total": total} if adds else {})
    if backward:
        x = total if adds else a["x"]
        r["x_grad"] = new(x)
        size, grad_type = x.shape[-1], grad_type or torch.float32
        r["weight_grad"], r["bias_grad"] = (torch.full((size,), 7.0, dtype=grad_type, device="cuda") for _ in "wb")
        room = torch.empty(ops.layer_norm_workspace(dev, x), dtype=torch.uint8, device="cuda").fill_(255)
        ops.layer_norm_backward(dev, x, stats, a["out_grad"], r["x_grad"], weight=weight, weight_grad=r["weight_grad"], bias_grad=r["bias_grad"],
                                centered=centered, total_grad=a["total_grad"] if adds else None, workspace=room, stream=here())
    torch.cuda.synchronize()
    return r


def check(dev, a, what, *, eps=1e-5, centered=True, adds=True, affine=True, grad_type=torch.float32, **how):
    got = run(dev, a, eps=eps, centered=centered, adds=adds, affine=affine, grad_type=grad_type, **how)
    want, bound = oracle.layer_norm(a["x"], a["weight"] if affine else None, a["bias"] if affine else None, eps=eps, centered=centered,
                                    added=a["added"] if adds else None, out_grad=a["out_grad"], total_grad=a["total_grad"] if adds else None,
                                    grad_type=grad_type)
    for n in want:
        assert_within(got[n], want[n], bound[n], f"{what}: {n}")


SIZES = [1, 2, 7, 8, 16, 33, 127, 128, 129, 255, 256, 257, 511, 1000, 1023, 1024, 1025, 2049, 4095, 4096, 4097, 8191, 16383, 16384]


@pytest.mark.parametrize("dtype,weights", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("size", SIZES)
def test_sizes(hip_device, size, dtype, weights):
    a = inputs((5, size), dtype, weights, seed=size)
    check(hip_device, a, f"5 x {size}, {dtype}", grad_type=TYPES[weights])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,size", [(1, 64), (2, 300), (17, 128), (64, 130), (65, 200), (257, 1500), (1025, 16), (4097, 24), (20001, 8), (5003, 260),
                                       (1100, 1030), (530, 2100), (301, 4100)])
def test_rows(hip_device, rows, size, dtype):
    """Rows that fill no workgroup, and more than all workgroups have at once."""
    check(hip_device, inputs((rows, size), dtype, "f32", seed=rows), f"{rows} x {size}, {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("how", [dict(centered=False), dict(adds=False), dict(affine=False), dict(centered=False, affine=False, adds=False),
                                 dict(eps=1e-9), dict(eps=3.0)])
def test_forms(hip_device, how, dtype):
    for shape in ((6, 130), (3, 1100), (2, 5000)):
        check(hip_device, inputs(shape, dtype, "f32", seed=3), f"{shape}, {how}, {dtype}", **how)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_mean_that_is_large_against_the_deviations(hip_device, dtype):
    a = inputs((4, 700), dtype, "f32", seed=9, level=3000.0 if dtype == "f32" else 30.0)
    check(hip_device, a, f"level, {dtype}", adds=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1, 2, 4, 8, 32, 64])
def test_a_mean_whose_product_with_the_root_passes_the_range(hip_device, size, dtype):
    """Rows of 2^80 alone (a sum and a mean that are exact) have no deviation, and a root of 1e15: mean times root is infinite, and lanes
    behind the end of the rows must not bring it into the sums."""
    a = inputs((5, size), dtype, "f32", seed=size)
    a["x"] = torch.full_like(a["x"], 2.0**80)
    got = run(hip_device, a, eps=1e-30, adds=False)
    assert torch.equal(got["out"].cpu(), a["bias"].expand(5, size).to(TYPES[dtype])) and got["x_grad"].isfinite().all()
    assert (got["weight_grad"] == 0).all()
    # five addends, added in some order: four roundings of sums that are at most the sum of magnitudes
    exact = a["out_grad"].double().sum(0)
    assert ((got["bias_grad"].cpu() - exact).abs() <= 4 * 2.0**-24 * a["out_grad"].double().abs().sum(0)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_equal_values(hip_device, dtype):
    """No deviation: the root is that of eps alone."""
    a = inputs((3, 64), dtype, "f32")
    a["x"] = torch.full_like(a["x"], 0.5)
    check(hip_device, a, f"equal, {dtype}", adds=False)
    a["x"] = torch.zeros_like(a["x"])
    check(hip_device, a, f"zeros, {dtype}", adds=False, centered=False)


def strided(x, layout):
    """The same values under other strides."""
    if layout == "unaligned":            # rows that begin one element in and have five behind them
        wide = torch.zeros((*x.shape[:-1], x.shape[-1] + 6), dtype=x.dtype)
        wide[..., 1:-5] = x
        return wide[..., 1:-5]
    if layout == "heads first":          # [batch, heads, length, size] memory seen as [batch, length, heads, size]
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "length first":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,layout", [((2, 5, 3, 72), "unaligned"), ((2, 5, 3, 72), "heads first"), ((3, 4, 130), "length first"),
                                          ((2, 3, 2, 1101), "unaligned"), ((2, 3, 2, 1101), "heads first"), ((1, 5, 1, 40), "heads first"),
                                          ((4, 1, 3, 50), "length first"), ((2, 2, 5001), "unaligned")])
def test_layouts(hip_device, shape, layout, dtype):
    a = inputs(shape, dtype, "f32", seed=1)
    plain = run(hip_device, a)
    a |= {n: strided(a[n], layout) for n in ("x", "added", "out_grad", "total_grad")}
    check(hip_device, a, f"{shape}, {layout}, {dtype}", like=lambda x: strided(torch.zeros(x.shape, dtype=x.dtype), layout).cuda()
          if layout == "unaligned" else torch.empty_like(x))
    again = run(hip_device, a)
    assert all(torch.equal(plain[n], again[n]) for n in plain), "strides decide over no bit"


@pytest.mark.parametrize("dtype", TYPES)
def test_arrays_of_different_layouts(hip_device, dtype):
    a = inputs((3, 4, 2, 96), dtype, "f32")
    a["x"], a["out_grad"] = strided(a["x"], "heads first"), strided(a["out_grad"], "length first")
    a["added"] = a["added"][:1, :, :1].expand(3, 4, 2, 96)  # one for all sequences and heads
    a["total_grad"] = strided(a["total_grad"], "unaligned")
    check(hip_device, a, f"mixed, {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [100, 1200, 9000])
def test_in_place(hip_device, size, dtype):
    """The residual stream is updated where it is, and the normed rows where they came from; gradients likewise."""
    a = inputs((7, size), dtype, "f32", seed=5)
    want = run(hip_device, a)
    g = {n: x.cuda() for n, x in a.items()}
    ops.layer_norm(hip_device, g["x"], g["added"], weight=g["weight"], bias=g["bias"], added=g["added"], total=g["x"], stream=here())
    room = torch.empty(ops.layer_norm_workspace(hip_device, g["x"]), dtype=torch.uint8, device="cuda")
    dw = torch.empty(size, device="cuda")
    ops.layer_norm_backward(hip_device, g["x"], want["stats"], g["out_grad"], g["out_grad"], weight=g["weight"], weight_grad=dw,
                            total_grad=g["total_grad"], workspace=room, stream=here())
    torch.cuda.synchronize()
    assert torch.equal(g["x"], want["total"]) and torch.equal(g["added"], want["out"])
    assert torch.equal(g["out_grad"], want["x_grad"]) and torch.equal(dw, want["weight_grad"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,size", [(1, 256), (3, 512), (257, 128), (16 * 256 + 1, 512), (513, 4096)])
def test_a_last_row_in_place_that_is_not_finite(hip_device, rows, size, dtype):
    """What x_grad puts in the place of the last row is not read by those that have no row."""
    a = inputs((rows, size), dtype, "f32", seed=rows)
    a["total_grad"][-1] = float("inf")
    want = run(hip_device, a)
    room = torch.empty(ops.layer_norm_workspace(hip_device, want["total"]), dtype=torch.uint8, device="cuda")
    dw, db = torch.empty(size, device="cuda"), torch.empty(size, device="cuda")
    g = {n: a[n].cuda() for n in ("weight", "out_grad", "total_grad")}
    ops.layer_norm_backward(hip_device, want["total"], want["stats"], g["out_grad"], want["total"], weight=g["weight"], weight_grad=dw, bias_grad=db,
                            total_grad=g["total_grad"], workspace=room, stream=here())
    torch.cuda.synchronize()
    assert torch.equal(want["total"], want["x_grad"]) and want["x_grad"][-1].isinf().all()
    assert dw.isfinite().all() and torch.equal(dw, want["weight_grad"]) and torch.equal(db, want["bias_grad"])


def test_gradients_that_are_not_asked_for(hip_device):
    a = inputs((9, 300), "f32", "f32")
    want = run(hip_device, a, adds=False)
    g = {n: x.cuda() for n, x in a.items()}
    dx, db = torch.empty_like(g["x"]), torch.empty(300, device="cuda", dtype=torch.bfloat16)
    how = dict(weight=g["weight"], stream=here())
    ops.layer_norm_backward(hip_device, g["x"], want["stats"], g["out_grad"], dx, **how)  # no sums, no workspace
    assert torch.equal(dx, want["x_grad"])
    room = torch.empty(ops.layer_norm_workspace(hip_device, g["x"]), dtype=torch.uint8, device="cuda")
    ops.layer_norm_backward(hip_device, g["x"], want["stats"], g["out_grad"], dx, bias_grad=db, workspace=room, **how)
    assert torch.equal(dx, want["x_grad"]) and torch.equal(db, want["bias_grad"].to(torch.bfloat16))


def test_no_rows(hip_device):
    x = torch.empty((0, 40), device="cuda")
    ops.layer_norm(hip_device, x, x, stats=torch.empty((0, 2), device="cuda"), stream=here())
    dw, db = torch.full((40,), 7.0, device="cuda"), torch.full((40,), 7.0, device="cuda")
    ops.layer_norm_backward(hip_device, x, torch.empty((0, 2), device="cuda"), x, x, weight_grad=dw, bias_grad=db,
                            workspace=torch.empty(16, dtype=torch.uint8, device="cuda"), stream=here())
    assert not dw.any() and not db.any()


def test_rows_that_are_not_finite_stay_alone(hip_device):
    a = inputs((6, 500), "f32", "f32")
    want = run(hip_device, a, adds=False)
    a["x"][2, 30], a["x"][4, 499] = float("nan"), float("inf")
    got = run(hip_device, a, adds=False)
    whole = [0, 1, 3, 5]
    assert torch.equal(got["out"][whole], want["out"][whole]) and torch.equal(got["x_grad"][whole], want["x_grad"][whole])
    assert got["out"][[2, 4]].isnan().all() and got["x_grad"][[2, 4]].isnan().all()

"""The operators on device arrays (adhip.operators) against plain 64-bit restatements (operator_oracle.py), at the sizes,
layouts and masks where they can go wrong.  Tolerances are the oracle's bounds, element by element."""
import math

import numpy as np
import pytest
import torch

import operator_oracle as oracle
from adhip import operators as ops

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
W = {"f32": 0.0, "bf16": 2.0 ** -8}  # half the spacing of eight significant bits


def here():
    return torch.cuda.current_stream().cuda_stream


def assert_within(got, want, bound, what):
    got, bound = got.double().cpu(), bound + 1e-30
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, torch.zeros_like(bound), (got - want).abs() / bound)
    worst = float(off.max()) if off.numel() else 0.0
    assert not torch.isnan(off).any(), f"{what}: NaN where there is none"
    assert worst <= 1.0, f"{what}: {worst:.3g} of the bound at {np.unravel_index(int(off.argmax()), off.shape)}"


# ---- attention ----------------------------------------------------------------------------------------------------------

# name: batch, queries, keys, heads, key heads, size, and what masks and scores
ATTENTION = {
    "one token": (1, 1, 1, 1, 1, 64, {}),
    "one token, one feature": (2, 1, 9, 2, 1, 1, dict(causal=True)),
    "tokens against a cache": (3, 1, 700, 8, 2, 128, dict(causal=True, lengths=[700, 0, 129])),
    "several tokens against a cache": (2, 5, 333, 6, 3, 80, dict(causal=True, lengths=[3, 333], window=40)),
    "33 rows": (1, 33, 65, 1, 1, 32, dict(causal=True)),
    "shared by 5, odd": (2, 37, 37, 5, 1, 33, dict(causal=True, cap=5.0)),
    "full, odd": (1, 129, 257, 2, 2, 100, {}),
    "causal over several tiles": (1, 300, 300, 4, 2, 128, dict(causal=True, cap=30.0)),
    "window both ways": (1, 200, 200, 2, 1, 64, dict(window=17)),
    "window of one": (1, 70, 70, 2, 2, 64, dict(causal=True, window=1)),
    "prefix": (3, 150, 150, 2, 2, 96, dict(causal=True, prefix=[0, 70, 1000], slopes=True)),
    "prefix and window, shorter": (2, 130, 150, 4, 2, 48, dict(causal=True, prefix=[5, 40], window=9, lengths=[150, 77])),
    "documents": (2, 260, 260, 3, 3, 64, dict(causal=True, documents=True)),
    "documents both ways, shared": (1, 190, 190, 4, 1, 72, dict(documents=True, slopes=True)),
    "more queries than keys": (2, 50, 20, 2, 1, 64, dict(causal=True, slopes=True)),
    "lengths shorter than the queries": (3, 64, 64, 2, 2, 64, dict(causal=True, lengths=[64, 0, 10])),
    "wide heads": (1, 100, 130, 2, 1, 256, dict(causal=True, cap=50.0)),
    "wide heads, not whole": (1, 40, 70, 2, 2, 200, dict(slopes=True)),
    "192 features, few rows": (1, 2, 200, 2, 2, 192, dict(causal=True)),
    "256 features, few rows": (2, 1, 300, 4, 2, 256, dict(causal=True, lengths=[300, 31])),
}

# few tiles of rows and long keys, or the other way round: walks in ranges (two to eight, and more), joined and added up
LONG = {
    "ranges, 100 features": (1, 40, 1500, 2, 1, 100, dict(causal=True, cap=20.0)),
    "ranges, 61 features": (2, 50, 1100, 2, 2, 61, dict(lengths=[1100, 301])),
    "ranges, 256 features": (1, 35, 900, 4, 2, 256, dict(causal=True, window=800)),
    "ranges, 33 features, many": (1, 64, 9001, 1, 1, 33, dict(causal=True, prefix=[4000])),
    "ranges, 128 features, many": (1, 40, 9003, 2, 1, 128, dict(slopes=True)),
    "ranges, documents": (1, 2000, 2000, 2, 2, 64, dict(causal=True, documents=True)),
    "ranges of rows": (1, 1501, 70, 4, 2, 90, {}),
}


# the same with scales that are given: below zero the largest product is the smallest score
SCALES = [("causal over several tiles", dict(scale=-0.11)), ("33 rows", dict(scale=-0.2)), ("prefix", dict(scale=-0.1, cap=2.0)),
          ("prefix and window, shorter", dict(scale=-0.3)), ("tokens against a cache", dict(scale=-0.09, cap=1.5)), ("one token", dict(scale=0.0)),
          ("full, odd", dict(scale=0.0, cap=3.0)), ("several tokens against a cache", dict(scale=3.0, cap=0.5))]


def attention_inputs(name, dtype, layout="plain", seed=0):
    B, Lq, Lk, H, Hk, D, how = {**ATTENTION, **LONG}[name]
    how = dict(how)
    g = torch.Generator().manual_seed(seed + len(name))

    def array(*shape):
        x = torch.randn(shape, generator=g)
        if layout == "heads first":      # [B, H, L, D] memory seen as [B, L, H, D]
            return x.transpose(1, 2).contiguous().to(TYPES[dtype]).transpose(1, 2)
        if layout == "unaligned":        # rows of D + 3 that begin one element in
            wide = torch.zeros(shape[0], shape[1], shape[2], shape[3] + 3)
            wide[..., 1:-2] = x
            return wide.to(TYPES[dtype])[..., 1:-2]
        return x.to(TYPES[dtype])

    a = {"q": array(B, Lq, H, D), "k": array(B, Lk, Hk, D), "v": array(B, Lk, Hk, D), "out_grad": array(B, Lq, H, D)}
    if "slopes" in how:
        how["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(H)])
    for x in ("lengths", "prefix"):
        if x in how:
            how[x] = torch.tensor(how[x], dtype=torch.int32)
    if how.pop("documents", False):
        d = torch.cumsum(torch.rand((B, Lk), generator=g) < 0.03, 1).to(torch.int32)
        d[:, Lk - 20:] = -1
        d[:, 7] = 5                      # ids need not be sorted
        how["key_documents"] = how["query_documents"] = d
    return a, how


def to_gpu(x):
    """The same values under the same strides."""
    if not isinstance(x, torch.Tensor):
        return x
    span = 1 + sum((n - 1) * s for n, s in zip(x.shape, x.stride())) if x.numel() else 0
    base = torch.as_strided(x, (x.storage_offset() + span,), (1,), 0).cuda()
    return torch.as_strided(base, x.shape, x.stride(), x.storage_offset())


def run_attention(dev, a, how, backward, strided_out=False):
    q, k, v, do = (to_gpu(a[n]) for n in ("q", "k", "v", "out_grad"))
    how = {n: to_gpu(x) for n, x in how.items()}
    like = (lambda x: torch.full_like(x, 7.0)) if not strided_out else (
        lambda x: torch.full(x.transpose(1, 2).shape, 7.0, dtype=x.dtype, device="cuda").transpose(1, 2))
    out, lse = like(q), torch.full(q.shape[:3], 7.0, device="cuda")
    room = torch.empty(ops.attention_workspace(dev, q, k, v, backward=backward), dtype=torch.uint8, device="cuda")
    room.fill_(255)  # NaN wherever it is read before it is written
    ops.attention(dev, q, k, v, out, lse, workspace=room, stream=here(), **how)
    r = {"out": out, "lse": lse}
    if backward:
        r |= {"dq": like(q), "dk": like(k), "dv": like(v)}
        room.fill_(255)
        ops.attention_backward(dev, q, k, v, out, lse, do, r["dq"], r["dk"], r["dv"], workspace=room, stream=here(), **how)
    torch.cuda.synchronize()
    return r


def check_attention(dev, name, dtype, layout="plain", strided_out=False):
    a, how = attention_inputs(name, dtype, layout)
    scale = 1.0 / math.sqrt(a["q"].shape[-1])
    want, bound = oracle.attention(a["q"], a["k"], a["v"], out_grad=a["out_grad"], rounding=W[dtype], scale=scale, **how)
    got = run_attention(dev, a, how, True, strided_out)
    for n in want:
        assert_within(got[n], want[n], bound[n], f"{name}, {dtype}, {layout}: {n}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ATTENTION)
def test_attention_and_its_gradients(hip_device, name, dtype):
    check_attention(hip_device, name, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["plain", "unaligned"])
@pytest.mark.parametrize("name", LONG)
def test_attention_in_ranges(hip_device, name, layout, dtype):
    check_attention(hip_device, name, dtype, layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["heads first", "unaligned"])
@pytest.mark.parametrize("name", ["tokens against a cache", "causal over several tiles", "shared by 5, odd", "wide heads, not whole"])
def test_attention_on_other_layouts(hip_device, name, layout, dtype):
    check_attention(hip_device, name, dtype, layout, strided_out=layout == "heads first")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name,change", SCALES)
def test_attention_with_scales_of_either_sign(hip_device, name, change, dtype):
    a, how = attention_inputs(name, dtype)
    how |= change
    want, bound = oracle.attention(a["q"], a["k"], a["v"], out_grad=a["out_grad"], rounding=W[dtype], **how)
    got = run_attention(hip_device, a, how, True)
    for n in want:
        assert_within(got[n], want[n], bound[n], f"{name}, {change}, {dtype}: {n}")


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_in_split_walks(hip_device, dtype):
    """Few heads and many positions: forward and both backward walks in parts, the keys' documents and lengths uneven."""
    g = torch.Generator().manual_seed(2)
    B, L, H, Hk, D = 1, 1900, 2, 1, 48
    a = {n: torch.randn(B, L, h, D, generator=g).to(TYPES[dtype]) for n, h in (("q", H), ("k", Hk), ("v", Hk), ("out_grad", H))}
    d = torch.cumsum(torch.rand((B, L), generator=g) < 0.002, 1).to(torch.int32)
    d[:, 1700:] = -1
    for how in (dict(causal=True), dict(causal=True, window=300, prefix=torch.tensor([100], dtype=torch.int32)),
                dict(causal=True, query_documents=d, key_documents=d), dict(lengths=torch.tensor([1234], dtype=torch.int32), cap=4.0)):
        want, bound = oracle.attention(a["q"], a["k"], a["v"], out_grad=a["out_grad"], rounding=W[dtype], scale=D ** -0.5, **how)
        got = run_attention(hip_device, a, how, True)
        for n in want:
            assert_within(got[n], want[n], bound[n], f"{list(how)}, {dtype}: {n}")


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_reads_nothing_that_no_query_may_see(hip_device, dtype):
    """NaN and infinities behind the lengths, in positions of no document, and in the gradient of rows that see nothing."""
    a, how = attention_inputs("documents", dtype)
    how["lengths"] = torch.tensor([260, 201], dtype=torch.int32)
    dirty = {n: x.clone() for n, x in a.items()}
    none = how["key_documents"] < 0
    none[1, 201:] = True
    for n, bad in (("k", math.nan), ("v", math.inf)):
        dirty[n][none] = bad
    n0 = torch.tensor([260, 201])
    at = torch.arange(260)[None, :] + n0[:, None] - 260
    empty = (how["query_documents"] < 0) | (at < 0)
    dirty["out_grad"][empty] = math.nan
    dirty["q"][empty] = math.nan
    want, bound = oracle.attention(dirty["q"], dirty["k"], dirty["v"], out_grad=dirty["out_grad"], rounding=W[dtype], scale=0.125, **how)
    got = run_attention(hip_device, dirty, dict(how, scale=0.125), True)
    assert torch.isneginf(want["lse"]).any()
    for n in want:
        assert_within(got[n], want[n], bound[n], n)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_scores_that_overflow(hip_device, dtype):
    """Scores of some thousands: the running maximum keeps the exponentials finite; one key takes all the weight."""
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, 40, 2, 64, generator=g) for _ in range(3))
    a = {"q": (q * 40).to(TYPES[dtype]), "k": (k * 40).to(TYPES[dtype]), "v": v.to(TYPES[dtype]), "out_grad": v.to(TYPES[dtype])}
    want, bound = oracle.attention(a["q"], a["k"], a["v"], scale=1.0, causal=True, rounding=W[dtype])
    got = run_attention(hip_device, a, dict(scale=1.0, causal=True), False)
    for n in want:
        assert_within(got[n], want[n], bound[n], n)


def test_attention_gradients_against_differences(hip_device):
    """The gradients along a direction against differences of the 64-bit forward."""
    a, how = attention_inputs("prefix", "f32")
    how["cap"] = 2.0
    scale = 1.0 / math.sqrt(96)
    got = run_attention(hip_device, a, how, True)
    g = torch.Generator().manual_seed(9)
    for n, d in (("q", "dq"), ("k", "dk"), ("v", "dv")):
        way = torch.randn(a[n].shape, generator=g).double()
        h = 1e-4
        ends = []
        for s in (h, -h):
            x = {m: a[m].double() for m in "qkv"}
            x[n] = x[n] + s * way
            ends.append(float((oracle.attention(x["q"], x["k"], x["v"], scale=scale, **how)[0]["out"] * a["out_grad"].double()).sum()))
        slope, mine = (ends[0] - ends[1]) / (2 * h), float((got[d].double().cpu() * way).sum())
        size = float((got[d].double().cpu() * way).norm())
        # differences: h^2 of a third derivative of order one per term; kernel: 1e-5 of each term at worst
        assert abs(slope - mine) <= 1e-4 * size, (n, slope, mine, size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["tokens against a cache", "causal over several tiles", "documents both ways, shared"])
def test_attention_gives_the_same_bits_again(hip_device, name, dtype):
    a, how = attention_inputs(name, dtype)
    one, two = (run_attention(hip_device, a, how, True) for _ in range(2))
    for n in one:
        assert torch.equal(one[n], two[n]), n


def test_attention_of_nothing(hip_device):
    e = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    # no keys: every row is empty
    q, k, out, lse = e(2, 3, 2, 64), e(2, 0, 1, 64), e(2, 3, 2, 64), e(2, 3, 2)
    dq, dk = e(2, 3, 2, 64), e(2, 0, 1, 64)
    room = torch.empty(ops.attention_workspace(hip_device, q, k, k, backward=True), dtype=torch.uint8, device="cuda")
    ops.attention(hip_device, q, k, k, out, lse, workspace=room, stream=here())
    ops.attention_backward(hip_device, q, k, k, out, lse, out, dq, dk, dk, workspace=room, stream=here())
    assert (out == 0).all() and torch.isneginf(lse).all() and (dq == 0).all()
    # no queries: nothing to write forward, gradients of keys are zero
    q, k, out, lse = e(2, 0, 2, 64), e(2, 5, 1, 64), e(2, 0, 2, 64), e(2, 0, 2)
    dk, dv = e(2, 5, 1, 64), e(2, 5, 1, 64)
    ops.attention(hip_device, q, k, k, out, lse, workspace=room, stream=here())
    ops.attention_backward(hip_device, q, k, k, out, lse, out, out, dk, dv, workspace=room, stream=here())
    assert (dk == 0).all() and (dv == 0).all()
    # no sequences
    q, k, lse = e(0, 3, 2, 64), e(0, 3, 2, 64), e(0, 3, 2)
    ops.attention(hip_device, q, k, k, q, lse, workspace=room, stream=here())
    ops.attention_backward(hip_device, q, k, k, q, lse, q, q, k, k, workspace=room, stream=here())


def test_attention_over_a_cache_that_passes_32_bits(hip_device):
    """One token against the end of a cache of more than 2^31 elements (bf16): offsets of 64 bits."""
    Lk, D = 33_600_000, 64
    k = torch.zeros((1, Lk, 1, D), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    q = torch.ones((1, 1, 1, D), dtype=torch.bfloat16, device="cuda")
    tail = 5
    k[:, -tail:], v[:, -tail:] = 1.0, torch.arange(D, device="cuda").to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((1, 1, 1), device="cuda")
    room = torch.empty(ops.attention_workspace(hip_device, q, k, v), dtype=torch.uint8, device="cuda")
    # scores: 64 for the last five, 0 for the others, which together weigh 3.4e7 e^-64 of one
    ops.attention(hip_device, q, k, v, out, lse, scale=1.0, causal=True, workspace=room, stream=here())
    assert torch.equal(out.flatten().float(), torch.arange(D, device="cuda").float())
    assert abs(float(lse) - (64 + math.log(tail))) < 1e-4
    del k, v
    torch.cuda.empty_cache()


# ---- rotary positions -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,pairs", [((1, 1, 1, 2), 1), ((2, 3, 2, 64), 32), ((1, 7, 5, 80), 20), ((2, 5, 3, 33), 11), ((1, 2, 4, 100), 50),
                                         ((3, 40, 6, 128), 64), ((1, 1, 70, 72), 36), ((1, 500, 9, 96), 36)])
def test_rotary(hip_device, shape, pairs, interleaved, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    B, L, H, D = shape
    x, y = torch.randn(shape, generator=g).to(TYPES[dtype]), torch.randn((B, L, 2, D), generator=g).to(TYPES[dtype])
    cos, sin = (torch.from_numpy(t) for t in ops.rotary_table(200, 2 * pairs))
    at = torch.randint(0, 200, (B, L), generator=g, dtype=torch.int32)
    for inverse in (False, True):
        xg, yg = x.cuda(), y.cuda()
        out = torch.empty_like(yg)
        # x in place, the second array into another
        ops.rotary(hip_device, xg, xg, cos.cuda(), sin.cuda(), at.cuda(), second=yg, second_out=out, interleaved=interleaved, inverse=inverse,
                   stream=here())
        for got, src in ((xg, x), (out, y)):
            want, bound = oracle.rotary(src, cos, sin, at, interleaved, inverse)
            assert_within(got, want, bound + (W[dtype] * want.abs()), f"{shape}, inverse {inverse}")


def test_rotary_layouts_and_positions_outside_of_the_table(hip_device):
    g = torch.Generator().manual_seed(4)
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rotary_table(50, 16))
    wide = torch.randn((2, 3, 4, 43), generator=g).cuda()
    x, out = wide[..., 1:25], torch.full((2, 4, 3, 24), 7.0, device="cuda").transpose(1, 2)
    at = torch.tensor([[0, 49, 50], [-1, 7, 2 ** 31 - 1]], dtype=torch.int32)
    ops.rotary(hip_device, x, out, cos, sin, at.cuda(), stream=here())
    want, bound = oracle.rotary(x.cpu(), cos.cpu(), sin.cpu(), at, False, False)
    assert torch.isnan(want).any()
    assert_within(out, want, bound, "strided")
    # one sequence's positions for all
    one = at[:1].cuda().expand(2, 3)
    ops.rotary(hip_device, x, out, cos, sin, one, stream=here())
    want, bound = oracle.rotary(x.cpu(), cos.cpu(), sin.cpu(), one.cpu(), False, False)
    assert_within(out, want, bound, "broadcast positions")


def test_rotary_inverse_is_the_gradient(hip_device):
    """<y, R x> = <R' y, x>, where R' is what `inverse` computes, over a whole batch."""
    g = torch.Generator().manual_seed(8)
    x, y = (torch.randn((2, 30, 3, 64), generator=g).cuda() for _ in range(2))
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rotary_table(64, 48))
    at = torch.arange(30, dtype=torch.int32).expand(2, 30).contiguous().cuda()
    rx, ry = torch.empty_like(x), torch.empty_like(x)
    ops.rotary(hip_device, x, rx, cos, sin, at, interleaved=True, stream=here())
    ops.rotary(hip_device, y, ry, cos, sin, at, interleaved=True, inverse=True, stream=here())
    left, right = (y.double() * rx.double()), (ry.double() * x.double())
    assert abs(float(left.sum() - right.sum())) <= 6 * oracle.U * float(left.abs().sum() + right.abs().sum())


# ---- AdamW --------------------------------------------------------------------------------------------------------------------

HOW = dict(step=7, rate=1e-2, beta1=0.9, beta2=0.99, eps=1e-6, decay=0.1, grad_scale=0.25)


def e4m3(t):
    return t.cpu().view(torch.float8_e4m3fn).double().numpy()


def blocks(x):
    """codes and scales of float64 values, for a start: what a program would have from the step before"""
    x = np.concatenate([x, np.zeros(-x.size % 256)]).reshape(-1, 256)
    scale = (np.maximum(np.abs(x).max(1), 2.0 ** -100) / 448).astype(np.float32)
    return torch.from_numpy((x / scale[:, None]).astype(np.float32)).to(torch.float8_e4m3fn), torch.from_numpy(scale)


@pytest.mark.parametrize("state", [32, 8])
@pytest.mark.parametrize("p_type", TYPES)
@pytest.mark.parametrize("g_type", TYPES)
@pytest.mark.parametrize("counts", [[1], [255, 256, 257, 4], [5000, 1, 4096, 16385] + [3] * 40])
def test_adamw(hip_device, counts, p_type, g_type, state):
    rng = np.random.default_rng(len(counts) + state)
    p = [torch.from_numpy(rng.normal(size=n).astype(np.float32)).to(TYPES[p_type]) for n in counts]
    g = [torch.from_numpy((rng.normal(size=n) * 10.0 ** rng.integers(-6, 1, n)).astype(np.float32)).to(TYPES[g_type]) for n in counts]
    m, v = [rng.normal(size=n) * 0.1 for n in counts], [rng.normal(size=n) ** 2 * 0.1 for n in counts]
    for x in g + m:
        x[0] = 0.0
    for x in v:
        x[:] = np.where(np.arange(x.size) % 7 == 0, 0.0, x)
    out = {}
    if state == 32:
        mt, vt = ([torch.from_numpy(x.astype(np.float32)).cuda() for x in y] for y in (m, v))
        m, v = ([x.double().cpu().numpy() for x in y] for y in (mt, vt))
        scales = {}
    else:
        mb, vb = [blocks(x) for x in m], [blocks(np.sqrt(x)) for x in v]
        m = [(e4m3(c) * s.double().numpy()[:, None]).reshape(-1)[:n] for (c, s), n in zip(mb, counts)]
        v = [((e4m3(c) * s.double().numpy()[:, None]) ** 2).reshape(-1)[:n] for (c, s), n in zip(vb, counts)]
        mt, vt = [c.cuda() for c, _ in mb], [c.cuda() for c, _ in vb]
        scales = dict(first_scales=[s.cuda() for _, s in mb], second_scales=[s.cuda() for _, s in vb])
    pt, gt = [x.cuda() for x in p], [x.cuda() for x in g]
    outs = {}
    if len(counts) > 1:  # into other arrays; the single tensor in place
        outs = dict(parameters_out=[torch.full_like(x, 7.0) for x in pt], first_out=[torch.empty_like(x) for x in mt],
                    second_out=[torch.empty_like(x) for x in vt])
        if scales:
            outs |= dict(first_scales_out=[torch.empty_like(x) for x in scales["first_scales"]],
                         second_scales_out=[torch.empty_like(x) for x in scales["second_scales"]])
    ops.adamw(hip_device, pt, gt, mt, vt, **scales, **outs, stream=here(), **HOW)
    torch.cuda.synchronize()
    out = {n: outs.get(n + "_out", x) for n, x in dict(parameters=pt, first=mt, second=vt, **scales).items()}
    for i, n in enumerate(counts):
        # the rate, betas and factors travel in 32 bits: their products with the state carry one rounding more (in the bounds)
        want, bound = oracle.adamw(p[i].double().numpy(), g[i].double().numpy(), m[i], v[i], **HOW)
        assert_within(out["parameters"][i], torch.from_numpy(want[0]), torch.from_numpy(bound[0] + W[p_type] * np.abs(want[0])), f"p[{i}]")
        if state == 32:
            assert_within(out["first"][i], torch.from_numpy(want[1]), torch.from_numpy(bound[1]), f"m[{i}]")
            assert_within(out["second"][i], torch.from_numpy(want[2]), torch.from_numpy(bound[2]), f"v[{i}]")
            continue
        for name, x, lift in (("first", want[1], False), ("second", np.sqrt(want[2]), True)):
            whole = np.concatenate([x, np.zeros(-n % 256)]).reshape(-1, 256)
            scale = out[name + "_scales"][i].double().cpu().numpy()
            exact = np.maximum(np.abs(whole).max(1), 2.0 ** -100) / 448
            assert np.all(np.abs(scale - exact) <= 8 * oracle.U * exact), f"{name}[{i}]: scales"
            held = e4m3(out[name][i]) * scale[:, None]
            # half a step of three bits of mantissa, half the smallest step below 2^-6; a root that is not zero is held as
            # one smallest step at least
            step = np.maximum(2.0 ** -4 * np.abs(whole), 2.0 ** -10 * scale[:, None])
            if lift:
                step = np.where((whole > 0) & (whole < 2.0 ** -9 * scale[:, None]), 2.0 ** -9 * scale[:, None], step)
                assert np.all(held[whole > 0] > 0), f"{name}[{i}]: a second moment was lost"
            assert np.all(np.abs(held - whole) <= step * (1 + 1e-5) + 1e-38), f"{name}[{i}]"
            assert np.all(held.reshape(-1)[n:] == 0), f"{name}[{i}]: behind the end"


def test_adamw_on_unaligned_tensors(hip_device):
    """Tensors that begin one element into an allocation take the same step, to the bit."""
    rng = np.random.default_rng(1)
    wide = [torch.from_numpy(rng.normal(size=3001).astype(np.float32)).cuda() for _ in range(4)]
    wide[3] = wide[3].square()
    views = [x[1:].clone() for x in wide], [x[1:] for x in wide]
    for p, g, m, v in views:
        ops.adamw(hip_device, [p], [g], [m], [v], stream=here(), **HOW)
    for a, b in zip(*views):
        assert torch.equal(a, b)


def test_adamw_not_finite(hip_device):
    """A NaN gradient makes its element NaN and, in 8 bits, its block's scales; other elements and blocks step as ever."""
    n = 600
    p, g = torch.ones(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    g[300] = math.nan
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    ops.adamw(hip_device, [p], [g], [m], [v], stream=here(), **HOW)
    assert torch.isnan(p).nonzero().flatten().tolist() == [300]
    p = torch.ones(n, device="cuda")
    codes = [torch.zeros((3, 256), device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.ones(3, device="cuda") for _ in range(2)]
    ops.adamw(hip_device, [p], [g], codes[:1], codes[1:], first_scales=scales[:1], second_scales=scales[1:], stream=here(), **HOW)
    assert torch.isnan(p).nonzero().flatten().tolist() == [300]
    for s in scales:
        assert torch.isnan(s).tolist() == [False, True, False]


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------------


def test_operators_follow_the_stream_they_are_given(hip_device):
    """Behind a long queue on a side stream, results are what the queue's end leaves."""
    a, how = attention_inputs("causal over several tiles", "bf16")
    want = run_attention(hip_device, a, how, False)["out"]
    q, k, v = (to_gpu(a[n]) for n in "qkv")
    side, out, lse = torch.cuda.Stream(), torch.empty_like(q), torch.empty(q.shape[:3], device="cuda")
    room = torch.empty(ops.attention_workspace(hip_device, q, k, v), dtype=torch.uint8, device="cuda")
    late = torch.zeros_like(q)
    x = torch.randn(2048, 2048, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            x = torch.mm(x, x).tanh()
        late.copy_(q)
        ops.attention(hip_device, late, k, v, out, lse, workspace=room, stream=side.cuda_stream, **how)
    side.synchronize()
    assert torch.equal(out, want)


def test_operators_in_a_graph(hip_device):
    """Captured once, replayed on other inputs with eager work between: every replay is the eager result."""
    a, how = attention_inputs("documents", "bf16")
    how = {n: to_gpu(x) for n, x in how.items()}
    q, k, v, do = (to_gpu(a[n]) for n in ("q", "k", "v", "out_grad"))
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rotary_table(300, 64))
    at = torch.arange(260, dtype=torch.int32, device="cuda").expand(2, 260).contiguous()
    p, m, s = torch.ones_like(q, dtype=torch.float32), torch.zeros_like(q, dtype=torch.float32), torch.zeros_like(q, dtype=torch.float32)
    names = ("rq", "rk", "out", "lse", "dq", "dk", "dv", "p", "m", "s")
    held = {"rq": torch.empty_like(q), "rk": torch.empty_like(k), "out": torch.empty_like(q), "lse": torch.empty(q.shape[:3], device="cuda"),
            "dq": torch.empty_like(q), "dk": torch.empty_like(k), "dv": torch.empty_like(v), "p": torch.empty_like(p), "m": torch.empty_like(m),
            "s": torch.empty_like(s)}
    room = torch.empty(ops.attention_workspace(hip_device, q, k, v, backward=True), dtype=torch.uint8, device="cuda")

    def step():
        ops.rotary(hip_device, q, held["rq"], cos, sin, at, second=k, second_out=held["rk"], stream=here())
        ops.attention(hip_device, held["rq"], held["rk"], v, held["out"], held["lse"], workspace=room, stream=here(), **how)
        ops.attention_backward(hip_device, held["rq"], held["rk"], v, held["out"], held["lse"], do, held["dq"], held["dk"], held["dv"],
                               workspace=room, stream=here(), **how)
        ops.adamw(hip_device, [p], [held["dq"]], [m], [s], parameters_out=[held["p"]], first_out=[held["m"]], second_out=[held["s"]],
                  stream=here(), **HOW)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        q.normal_()
        do.normal_()
        step()
        torch.cuda.synchronize()
        want = {n: held[n].clone() for n in names}
        for x in held.values():
            x.fill_(5.0)
        room.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        for n in names:
            assert torch.equal(held[n], want[n]), (i, n)


def test_refusals_of_attention(hip_device):
    f = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(q=f(2, 8, 4, 64), k=f(2, 9, 2, 64), v=f(2, 9, 2, 64), out=f(2, 8, 4, 64), lse=f(2, 8, 4))
    room = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")

    def refused(message, **change):
        x = {**good, "workspace": room, **change}
        with pytest.raises((RuntimeError, ValueError), match=message):
            ops.attention(hip_device, x.pop("q"), x.pop("k"), x.pop("v"), x.pop("out"), x.pop("lse"), stream=here(), **x)

    refused("q is int32", q=i(2, 8, 4, 64))
    refused("k is bf16, f32 is wanted", k=f(2, 9, 2, 64, t=torch.bfloat16))
    refused("k has 3 dims", k=f(2, 9, 64))
    refused("v is f32", v=f(2, 8, 2, 64))
    refused("k is f32", k=f(2, 9, 2, 32))
    refused("cannot share", k=f(2, 9, 3, 64), v=f(2, 9, 3, 64))
    refused("1 to 256", q=f(2, 8, 4, 257), k=f(2, 9, 2, 257), v=f(2, 9, 2, 257), out=f(2, 8, 4, 257))
    refused("last stride of q", q=f(2, 8, 4, 128)[..., ::2])
    refused("share memory", out=f(2, 8, 1, 64).expand(2, 8, 4, 64))
    refused("lse has 0 dims", lse=None)
    refused("lse is f32", lse=f(2, 4, 8))
    refused("lengths is int32 .3.", lengths=i(3))
    refused("prefix is f32", prefix=f(2))
    refused("slopes", slopes=f(2))
    refused("key_documents", query_documents=i(2, 8))
    refused("query_documents", query_documents=i(2, 9), key_documents=i(2, 9))
    refused("elements apart", query_documents=i(2, 8), key_documents=torch.as_strided(i(9 << 21), (2, 9), (1, 1 << 21)))
    refused("cap", cap=-1.0)
    refused("cap", cap=math.nan)
    refused("scale", scale=math.inf)
    refused("window", window=-1)
    need = ops.attention_workspace(hip_device, good["q"], good["k"], good["v"])
    refused(f"{need - 1} bytes is given, {need} are needed", workspace=room[:need - 1])
    refused("aligned to 256", workspace=room[1:])
    refused("not supported", q=f(2, 8, 4, 64, t=torch.float64))
    with pytest.raises(RuntimeError, match="out_grad"):
        ops.attention_backward(hip_device, good["q"], good["k"], good["v"], good["out"], good["lse"], None, good["out"], good["k"], good["v"],
                               workspace=room, stream=here())


def test_refusals_of_rotary_and_adamw(hip_device):
    f = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    good = dict(x=f(2, 3, 4, 16), out=f(2, 3, 4, 16), cos=f(9, 8), sin=f(9, 8), positions=i(2, 3))

    def refused(message, **change):
        x = {**good, **change}
        with pytest.raises((RuntimeError, ValueError), match=message):
            ops.rotary(hip_device, x.pop("x"), x.pop("out"), x.pop("cos"), x.pop("sin"), x.pop("positions"), stream=here(), **x)

    refused("x is int32", x=i(2, 3, 4, 16))
    refused("out is f32", out=f(2, 3, 5, 16))
    refused("do not fit", cos=f(9, 9), sin=f(9, 9))
    refused("sin", sin=f(8, 8))
    refused("rows of the tables", cos=f(9, 16)[:, :8])
    refused("positions is f32", positions=f(2, 3))
    refused("second is f32", second=f(2, 3, 4, 8), second_out=f(2, 3, 4, 8))
    refused("second_out", second=f(2, 3, 4, 16))
    refused("share memory", out=f(2, 3, 1, 16).expand(2, 3, 4, 16))
    refused("positions has 0 dims", positions=None)

    p, g, m, v = (f(10) for _ in range(4))
    for message, args, how in [
        ("first step is 1", ([p], [g], [m], [v]), dict(step=0)),
        ("betas", ([p], [g], [m], [v]), dict(beta1=1.0)),
        ("finite", ([p], [g], [m], [v]), dict(rate=math.inf)),
        ("eps", ([p], [g], [m], [v]), dict(eps=-1.0)),
        ("packed elements", ([p], [f(9)], [m], [v]), {}),
        ("packed elements", ([p], [f(20)[::2]], [m], [v]), {}),
        ("1 gradients for 2", ([p, p], [g], [m, m], [v, v]), {}),
        ("one supported type", ([p], [i(10)], [m], [v]), {}),
        ("first_scales", ([p], [g], [f(1, 256).to(torch.float8_e4m3fn)], [f(1, 256).to(torch.float8_e4m3fn)]), {}),
    ]:
        with pytest.raises((RuntimeError, ValueError), match=message):
            ops.adamw(hip_device, *args, stream=here(), **{**HOW, **how})
    ops.adamw(hip_device, [], [], [], [], stream=here(), **HOW)


def test_device_arrays_and_a_programs_buffers(hip_device):
    """DeviceArray copies, and a program whose kept buffers an operator reads and writes."""
    from adhip import autodiff
    x = np.arange(24, dtype=np.float32).reshape(2, 3, 4)
    a = ops.DeviceArray.of(hip_device, x)
    assert a.shape == (2, 3, 4) and a.stride() == (12, 4, 1) and np.array_equal(a.numpy(), x)
    assert np.array_equal(a.reshape(6, 4).numpy(), x.reshape(6, 4))
    with pytest.raises(ValueError):
        a.reshape(5, 4)
    with pytest.raises(ValueError):
        ops.DeviceArray.empty(hip_device, (3,), "float64")
    half = ops.DeviceArray.empty(hip_device, (4,), "bfloat16")
    assert half.nbytes == 8 and half.numpy().dtype == np.float32
    autodiff.set_device(hip_device)
    w = autodiff.tensor(np.ones(6, np.float32), [2, 3])
    y = w * 2.0
    y.forward()
    w.val().keep()
    y.val().keep()
    from adhip import ir as IR
    from adhip.core import STATE
    STATE.irb.add_cmd(IR.EX())
    program = hip_device.compile(STATE.irb.proc, set(STATE.dep_tracker))
    program.upload()
    wb, yb = (ops.program_array(program, t.val().id) for t in (w, y))
    assert wb.shape == (2, 3)
    with pytest.raises(KeyError):
        ops.program_array(program, "no such id")
    grads = [ops.DeviceArray.of(hip_device, np.full((2, 3), 0.5, np.float32))]
    moments = [ops.DeviceArray.of(hip_device, np.zeros((2, 3), np.float32)) for _ in range(2)]
    program.enqueue()
    ops.adamw(hip_device, [wb], grads, moments[:1], moments[1:], step=1, rate=0.125, eps=0.0, decay=0.0)
    program.enqueue()
    ops.synchronize(hip_device)
    # the first step of Adam is the rate in the gradient's direction
    assert np.allclose(wb.numpy(), 1.0 - 0.125, rtol=1e-6) and np.array_equal(yb.numpy(), 2.0 * wb.numpy())
    program.close()

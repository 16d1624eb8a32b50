"""Inputs at the edges of what the operators on device arrays promise, against the 64-bit restatements of operator_oracle.py
with its bounds: distances that score upwards, values that nothing may use, widths between the tested ones, numbers that fill a
launch."""
import ctypes
import math

import pytest
import torch

import operator_oracle as oracle
from adhip import operators as ops
from test_operators_gpu import TYPES, W, assert_within, here, run_attention, to_gpu

pytestmark = pytest.mark.gpu


def inputs(dtype, B, Lq, Lk, H, Hk, D, seed=0, unaligned=False):
    g = torch.Generator().manual_seed(seed)

    def array(length, heads):
        x = torch.randn((B, length, heads, D), generator=g).to(TYPES[dtype])
        if not unaligned:
            return x
        wide = torch.zeros((B, length, heads, D + 3), dtype=x.dtype)
        wide[..., 1:-2] = x
        return wide[..., 1:-2]

    return {n: array(length, heads) for n, length, heads in (("q", Lq, H), ("k", Lk, Hk), ("v", Lk, Hk), ("out_grad", Lq, H))}


def documents(B, L, rate, none, seed=0):
    """Rising numbers of documents, the last `none` positions of no document."""
    d = torch.cumsum(torch.rand((B, L), generator=torch.Generator().manual_seed(seed)) < rate, 1).to(torch.int32)
    d[:, L - none:] = -1
    return d


def check(dev, a, dtype, what, **how):
    how.setdefault("scale", 1.0 / math.sqrt(a["q"].shape[-1]))
    want, bound = oracle.attention(a["q"], a["k"], a["v"], out_grad=a["out_grad"], rounding=W[dtype], **how)
    got = run_attention(dev, a, how, True)
    for n in want:
        assert_within(got[n], want[n], bound[n], f"{what}, {dtype}: {n}")


# ---- attention: scores that rise with distance --------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,size,how", [
    (181, 64, dict(causal=True)),
    (181, 64, dict(causal=True, prefix=[130, 0])),
    (215, 128, dict(causal=True, cap=5.0, lengths=[215, 200])),
    (203, 40, dict()),
    (183, 192, dict(causal=True)),
    (181, 256, dict(causal=True)),
])
def test_attention_with_slopes_below_zero(hip_device, queries, size, how, dtype):
    """exp(0.5 x 180) passes what 32 bits hold: a row that is not there must not meet the products with it."""
    a = inputs(dtype, 2, queries, queries, 4, 2, size, seed=queries)
    how = {n: torch.tensor(x, dtype=torch.int32) if isinstance(x, list) else x for n, x in how.items()}
    check(hip_device, a, dtype, f"{queries} x {size}, {list(how)}", slopes=torch.tensor([-0.5, 0.25, -0.75, -0.6]), **how)


# ---- attention: values that nothing may use --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries,heads,size,how", [
    (1, 8, 128, dict(causal=True, window=40)),
    (1, 4, 64, dict(window=1)),
    (5, 6, 80, dict(causal=True, window=100, prefix=[0, 70, 150], cap=4.0)),
    (2, 2, 192, dict(causal=True, window=33, prefix=[3, 0, 0])),
    (70, 4, 64, dict(causal=True, window=50, lengths=[300, 91, 40])),
    (40, 2, 256, dict(window=64, prefix=[33, 0, 64])),
    (130, 2, 128, dict(causal=True, window=129, documents=True)),
])
def test_attention_reads_nothing_in_front_of_every_window(hip_device, queries, heads, size, how, dtype):
    """A cache of 300 positions whose windows have moved on: what lies between the prefix and the first query's window is NaN and
    infinite."""
    B, Lk = 3, 300
    how = dict(how)
    a = inputs(dtype, B, queries, Lk, heads, 2, size, seed=queries + size)
    n = how.get("lengths", [Lk] * B)
    first = [n[b] - queries - how["window"] + 1 for b in range(B)]
    prefix = how.get("prefix", [0] * B)
    hidden = 0
    for b in range(B):
        a["k"][b, prefix[b]:max(first[b], prefix[b])] = math.nan
        a["v"][b, prefix[b]:max(first[b], prefix[b])] = math.inf
        hidden += max(first[b] - prefix[b], 0)
    assert hidden > 50
    if how.pop("documents", False):
        d = documents(B, Lk, 0.01, 20)
        how |= dict(key_documents=d, query_documents=d[:, Lk - queries:].contiguous())
    how = {x: torch.tensor(y, dtype=torch.int32) if isinstance(y, list) else y for x, y in how.items()}
    check(hip_device, a, dtype, f"{queries} x {size}, {list(how)}", **how)


# ---- attention: widths and walks between the tested ones -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("unaligned", [False, True])
@pytest.mark.parametrize("batch,queries,keys,heads,shared,size,how", [
    (1, 300, 300, 4, 2, 192, dict(causal=True, cap=20.0)),
    (2, 170, 231, 2, 1, 150, dict(causal=True, window=60)),
    (1, 210, 210, 3, 3, 129, dict(slopes=True)),
    (1, 70, 1900, 1, 1, 192, dict(causal=True)),           # walks in ranges
    (1, 1300, 90, 2, 2, 176, dict()),                      # ranges of rows
    (2, 260, 260, 2, 2, 192, dict(causal=True, documents=True, lengths=[260, 133])),
    (2, 150, 150, 2, 1, 256, dict(documents=True, lengths=[90, 150])),
    (1, 1100, 1100, 1, 1, 240, dict(causal=True, documents=True)),
])
def test_attention_of_129_features_and_more(hip_device, batch, queries, keys, heads, shared, size, how, unaligned, dtype):
    how = dict(how)
    a = inputs(dtype, batch, queries, keys, heads, shared, size, seed=queries + size, unaligned=unaligned)
    if how.pop("slopes", False):
        how["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(heads)])
    if how.pop("documents", False):
        how["query_documents"] = how["key_documents"] = documents(batch, keys, 0.02, 20)
    if "lengths" in how:
        how["lengths"] = torch.tensor(how["lengths"], dtype=torch.int32)
    check(hip_device, a, dtype, f"{queries} x {keys} x {size}, {list(how)}, unaligned {unaligned}", **how)


# ---- what the host decides ---------------------------------------------------------------------------------------------------


class Shape:
    """An array that has a shape and a type, and memory nowhere."""

    def __init__(self, *shape, dtype="float32"):
        self.shape, self.dtype = shape, dtype

    def stride(self):
        return tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))

    def data_ptr(self):
        return 0


@pytest.mark.parametrize("backward", [False, True])
def test_attention_workspace_goes_by_shapes_alone(hip_device, backward):
    for dtype in TYPES:
        q, k = torch.empty((2, 50, 4, 64), dtype=TYPES[dtype], device="cuda"), torch.empty((2, 900, 2, 64), dtype=TYPES[dtype], device="cuda")
        need = ops.attention_workspace(hip_device, q, k, k, backward=backward)
        q, k = Shape(*q.shape, dtype=q.dtype), Shape(*k.shape, dtype=k.dtype)
        assert ops.attention_workspace(hip_device, q, k, k, backward=backward) == need > 0


def test_an_error_that_another_call_left_is_not_the_operators(hip_device):
    """A failed call of the HIP runtime stands as its last error until it is asked for: the operators neither report nor take it."""
    x = torch.randn((1, 3, 2, 8), device="cuda")
    out, at = torch.empty_like(x), torch.zeros((1, 3), dtype=torch.int32, device="cuda")
    cos, sin = (torch.from_numpy(t).cuda() for t in ops.rotary_table(8, 8))
    lse, room = torch.empty((1, 3, 2), device="cuda"), torch.empty(ops.attention_workspace(hip_device, x, x, x, backward=True), dtype=torch.uint8, device="cuda")
    grads, moments = [torch.empty_like(x) for _ in range(3)], [torch.zeros_like(x) for _ in range(2)]
    torch.cuda.synchronize()
    stream, runtime = here(), hip_device._lib
    refused = runtime.hipSetDevice(1000)
    try:
        ops.rotary(hip_device, x, out, cos, sin, at, stream=stream)
        ops.attention(hip_device, x, x, x, out, lse, workspace=room, stream=stream)
        ops.attention_backward(hip_device, x, x, x, out, lse, out, *grads, workspace=room, stream=stream)
        ops.adamw(hip_device, [x], [out], moments[:1], moments[1:], step=1, rate=0.1, stream=stream)
    finally:
        left = runtime.hipGetLastError()
    assert refused != 0 and left == refused
    torch.cuda.synchronize()


def test_attention_of_more_workgroups_than_a_launch_holds_is_refused(hip_device):
    """2^24 workgroups of 256 threads: the number of threads would begin anew at 2^32."""
    for sequences, queries, keys, backward, fits in [(2 ** 21 - 1, 1, 3, False, True), (2 ** 21, 1, 3, False, False), (2 ** 20 - 1, 1, 3, True, True),
                                                     (2 ** 20, 1, 3, True, False), (2 ** 20, 1, 3, False, True)]:
        q, k = Shape(sequences, queries, 8, 8, dtype="bfloat16"), Shape(sequences, keys, 8, 8, dtype="bfloat16")
        if fits:
            assert ops.attention_workspace(hip_device, q, k, k, backward=backward) > 0
        else:
            with pytest.raises(RuntimeError, match="too large for one call"):
                ops.attention_workspace(hip_device, q, k, k, backward=backward)


def test_rotary_of_more_tokens_than_a_row_of_a_launch_holds(hip_device):
    """2^24 tokens of a block each, 129 heads of one pair: every one of them is turned."""
    tokens = 2 ** 24 + 5
    x = torch.randn((1, 1, 129, 2), device="cuda").to(torch.bfloat16).expand(1, tokens, 129, 2)
    out = torch.zeros((1, tokens, 129, 2), dtype=torch.bfloat16, device="cuda")
    cos, sin = (torch.from_numpy(t) for t in ops.rotary_table(8, 2))
    at = torch.tensor([[3]], dtype=torch.int32)
    ops.rotary(hip_device, x, out, cos.cuda(), sin.cuda(), at.cuda().expand(1, tokens), stream=here())
    want, bound = oracle.rotary(x[:, :1].cpu(), cos, sin, at, False, False)
    assert_within(out[:, :1], want, bound + W["bf16"] * want.abs(), "the first token")
    for i in range(0, tokens, 2 ** 20):
        assert (out[:, i:i + 2 ** 20] == out[:, :1]).all(), f"from token {i}"
    del out
    torch.cuda.empty_cache()


def test_attention_in_f32_of_heads_that_pass_the_offsets_of_a_tile_is_refused(hip_device):
    """f32 in parts: 32 rows of 2^25 features and more reach 2^31 bytes from a tile's first, where its loads end."""
    for heads, shared, backward, fits in [(2 ** 18, 2 ** 18, False, True), (300_000, 300_000, False, False), (300_000, 300_000, True, False),
                                          (300_000, 100_000, False, True), (300_000, 100_000, True, False)]:
        q, k = Shape(1, 40, heads, 128), Shape(1, 3, shared, 128)
        if fits:
            assert ops.attention_workspace(hip_device, q, k, k, backward=backward) > 0
        else:
            with pytest.raises(RuntimeError, match="too large for one call"):
                ops.attention_workspace(hip_device, q, k, k, backward=backward)
    q, k = (Shape(1, n, 300_000, 128, dtype="bfloat16") for n in (40, 3))
    assert ops.attention_workspace(hip_device, q, k, k) > 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,queries,keys,heads,shared,size,how", [
    (1, 1, 9000, 2, 1, 33, dict(causal=True)),
    (2, 1, 7001, 3, 1, 61, dict(causal=True, lengths=[7001, 12])),
    (3, 2, 6000, 4, 2, 128, dict(causal=True, cap=8.0, lengths=[0, 6000, 3111])),
    (1, 4, 5003, 8, 1, 256, dict(causal=True, slopes=True)),
    (1, 3, 8000, 2, 2, 200, dict(causal=True, window=5000, prefix=[100])),
    (2, 1, 12000, 1, 1, 64, dict(causal=True, documents=True)),
])
def test_attention_of_tokens_over_many_ranges(hip_device, batch, queries, keys, heads, shared, size, how, dtype):
    """Caches long enough that the keys of a token are split into more ranges than one thread joins."""
    how = dict(how)
    a = inputs(dtype, batch, queries, keys, heads, shared, size, seed=keys)
    if how.pop("slopes", False):
        how["slopes"] = torch.tensor([2.0 ** -(h + 5) for h in range(heads)])
    if how.pop("documents", False):
        d = documents(batch, keys, 0.0003, 0)
        how |= dict(key_documents=d, query_documents=d[:, keys - queries:].contiguous())
    how = {x: torch.tensor(y, dtype=torch.int32) if isinstance(y, list) else y for x, y in how.items()}
    check(hip_device, a, dtype, f"{queries} x {keys} x {size}, {list(how)}", **how)

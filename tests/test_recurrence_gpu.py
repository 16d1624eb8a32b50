"""The gated recurrence on device arrays (adhip.operators) against a plain 64-bit restatement (training_oracle.py), at the lengths,
layouts, masks and values where it can go wrong.  Tolerances are the oracle's bounds, element by element."""
import pytest
import torch

import training_oracle as oracle
from adhip import operators as ops
from test_operators_gpu import TYPES, assert_within, here, to_gpu

pytestmark = pytest.mark.gpu


def inputs(B, L, C, dtype, *, factors=False, seed=0, initial=True, lengths=None, documents=0.0, slow=3.0):
    g = torch.Generator().manual_seed(seed)
    gates = torch.randn((B, L, C), generator=g) + slow * torch.rand(C, generator=g)
    a = {"x": torch.randn((B, L, C), generator=g), "gates": torch.sigmoid(gates) if factors else gates,
         "out_grad": torch.randn((B, L, C), generator=g)}
    a = {n: x.to(TYPES[dtype]) for n, x in a.items()}
    a["initial"] = torch.randn((B, C), generator=g) if initial else None
    a["final_grad"] = torch.randn((B, C), generator=g) if initial else None
    a["lengths"] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    a["documents"] = None
    if documents:
        d = torch.cumsum(torch.rand((B, L), generator=g) < documents, 1).to(torch.int32)
        d[torch.rand((B, L), generator=g) < documents / 3] = -1
        a["documents"] = d
    return a


def run(dev, a, *, factors=False, backward=True, like=torch.empty_like, stream=None):
    """Forward and backward; every output begins as numbers that must not survive."""
    a = {n: to_gpu(x) for n, x in a.items()}
    new = lambda x: like(x).fill_(7.0)  # noqa: E731
    (B, L, C), stream = a["x"].shape, here() if stream is None else stream
    out, final = new(a["x"]), torch.full((B, C), 7.0, device="cuda")
    states = torch.full((B, ops.recurrence_blocks(L), C), 7.0, device="cuda")
    room = torch.empty(ops.recurrence_workspace(dev, a["x"], backward=backward) + 16, dtype=torch.uint8, device="cuda").fill_(255)
    how = dict(factors=factors, lengths=a["lengths"], documents=a["documents"], workspace=room, stream=stream)
    ops.recurrence(dev, a["x"], a["gates"], out, initial=a["initial"], final=final, states=states if backward else None, **how)
    r = {"out": out, "final": final}
    if backward:
        r |= {"states": states, "x_grad": new(a["x"]), "gates_grad": new(a["x"]), "initial_grad": torch.full((B, C), 7.0, device="cuda")}
        room.fill_(255)
        ops.recurrence_backward(dev, a["x"], a["gates"], states, a["out_grad"], r["x_grad"], r["gates_grad"], final_grad=a["final_grad"],
                                initial_grad=r["initial_grad"], **how)
    torch.cuda.synchronize()
    return r


def check(dev, a, what, *, factors=False, backward=True, **how):
    got = run(dev, a, factors=factors, backward=backward, **how)
    grads = dict(out_grad=a["out_grad"], final_grad=a["final_grad"]) if backward else {}
    want, bound = oracle.recurrence(a["x"], a["gates"], factors=factors, initial=a["initial"], lengths=a["lengths"], documents=a["documents"], **grads)
    for n in got:
        assert_within(got[n], want[n], bound[n], f"{what}: {n}")
    return got


SHAPES = [(1, 1, 1), (2, 1, 5), (3, 2, 33), (2, 7, 31), (1, 8, 32), (2, 9, 17), (1, 32, 16), (3, 33, 64), (2, 64, 40), (1, 255, 48), (1, 256, 16),
          (2, 257, 33), (1, 511, 64), (1, 513, 130), (2, 700, 9), (1, 1025, 65), (300, 3, 7), (1, 5, 2000), (40, 20, 65), (5, 100, 131), (3, 8, 4097),
          (70, 17, 1025), (3, 40, 3001), (2, 300, 4097)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(hip_device, shape, factors, dtype):
    check(hip_device, inputs(*shape, dtype, factors=factors, seed=sum(shape)), f"{shape}, {dtype}", factors=factors)


LONG = [(1, 5000, 20), (2, 3333, 65), (1, 9001, 3), (3, 2048, 33)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("shape", LONG)
def test_long_sequences_of_few_channels(hip_device, shape, factors, dtype):
    check(hip_device, inputs(*shape, dtype, factors=factors, seed=2, slow=6.0), f"{shape}, {dtype}", factors=factors)


@pytest.mark.parametrize("dtype,C", [("f32", 930), ("bf16", 1857)])
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_long_ranges_of_wide_rows(hip_device, masked, factors, dtype, C):
    """Channels in rows of 128 bytes (of bf16, the last one alone in its row) and positions in ranges."""
    masks = dict(documents=0.002, lengths=[8700]) if masked else {}
    a = inputs(1, 9001, C, dtype, factors=factors, seed=3, slow=5.0, **masks)
    assert ops.recurrence_workspace(hip_device, a["x"]) > 0
    check(hip_device, a, f"9001 x {C}, {dtype}", factors=factors)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_many_sequences_of_several_tiles(hip_device, masked, dtype):
    """Rows of 128 bytes without ranges."""
    masks = dict(documents=0.01, lengths=[700, 530, 0, 1, 256, 699]) if masked else {}
    check(hip_device, inputs(6, 700, 1473, dtype, seed=3, **masks), f"many, {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,lines", [(1, 9001, 29), (9, 530, 32)])
def test_rows_of_whole_cache_lines(hip_device, B, L, lines, dtype):
    """Workgroups that share no cache lines are numbered otherwise: the same bits as in rows that begin off a line."""
    C = lines * (32 if dtype == "f32" else 64)
    a = inputs(B, L, C, dtype, seed=3, slow=5.0)
    check(hip_device, a, f"{B} x {L} x {C}, {dtype}")
    plain = run(hip_device, a)
    for n in ("x", "gates", "out_grad"):
        wide = torch.zeros((B, L, C + 3), dtype=a[n].dtype)
        wide[..., 1:-2] = a[n]
        a[n] = wide[..., 1:-2]
    got = run(hip_device, a, like=torch.empty_like)
    assert all(torch.equal(got[n], plain[n]) for n in plain)


MASKS = {
    "lengths": dict(lengths=[700, 0, 256]),
    "lengths out of range": dict(lengths=[9999, -3, 1]),
    "documents": dict(documents=0.02),
    "documents of a few positions": dict(documents=0.5),
    "documents and lengths": dict(documents=0.02, lengths=[699, 257, 512]),
    "no initial state": dict(documents=0.02, initial=False),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("mask", MASKS)
def test_masks(hip_device, mask, factors, dtype):
    for L, C in ((700, 37), (6, 20)):
        check(hip_device, inputs(3, L, C, dtype, factors=factors, seed=4, **MASKS[mask]), f"{mask}, {L} positions, {dtype}", factors=factors)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
def test_long_masks(hip_device, factors, dtype):
    a = inputs(2, 4500, 18, dtype, factors=factors, seed=6, documents=0.002, lengths=[4500, 3100])
    check(hip_device, a, f"long, {dtype}", factors=factors)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [-1, 0, 1])
@pytest.mark.parametrize("every", [64, 1024])
def test_documents_that_begin_where_ranges_do(hip_device, every, off, dtype):
    """The last and the first one of a range decide what it does to a state."""
    a = inputs(2, 4500, 18, dtype, seed=6, slow=6.0, lengths=[4500, 2305])
    a["documents"] = ((torch.arange(4500) - off) // every).to(torch.int32).expand(2, 4500).contiguous()
    a["documents"][:, 2304:2306] = -1
    check(hip_device, a, f"every {every} and {off}, {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("L", [600, 5, 4100])
def test_hidden_positions_may_hold_anything(hip_device, L, factors, dtype):
    a = inputs(2, L, 24, dtype, factors=factors, seed=5, documents=0.05, lengths=[L, L * 2 // 3])
    hidden = a["documents"] < 0
    hidden[1, L * 2 // 3:] = True
    if L == 5:
        hidden[0, 2], a["documents"][0, 2] = True, -1
    want = run(hip_device, a, factors=factors)
    for n, bad in (("x", "nan"), ("gates", "inf"), ("out_grad", "nan")):
        a[n][hidden] = float(bad)
    got = run(hip_device, a, factors=factors)
    assert hidden.any() and all(torch.equal(got[n], want[n]) for n in want)
    hidden = hidden.cuda()
    assert not any(got[n][hidden].any() for n in ("out", "x_grad", "gates_grad"))


@pytest.mark.parametrize("dtype", TYPES)
def test_states_that_are_dropped_may_be_infinite(hip_device, dtype):
    """A document that grows beyond all bounds does not reach the next one, nor does its gradient the one before."""
    for L in (40, 700, 3000):
        a = inputs(1, L, 10, dtype, factors=True, seed=3, initial=False)
        a["documents"] = torch.zeros((1, L), dtype=torch.int32)
        mid = L // 2
        a["documents"][0, mid - 10:] = 1
        a["documents"][0, mid + 3:] = 2
        a["gates"][0, mid - 10:mid + 3] = 3e38
        got = run(hip_device, a, factors=True)
        assert got["out"][0, mid - 10:mid + 3].isinf().any() or got["out"][0, mid - 10:mid + 3].isnan().any()
        for n in ("out", "x_grad", "gates_grad"):
            assert got[n][0, :mid - 10].isfinite().all() and got[n][0, mid + 3:].isfinite().all(), (n, L)
        assert got["final"].isfinite().all()


def test_states_of_zero_take_any_factor(hip_device):
    """Nothing put in stays nothing, however far factors would take it."""
    for L in (40, 700, 3000):
        a = inputs(1, L, 10, "f32", factors=True, initial=False)
        a["gates"][:] = 3.0
        a["x"][:, :L - 5] = 0.0
        got = run(hip_device, a, factors=True, backward=False)
        want, bound = oracle.recurrence(a["x"], a["gates"], factors=True)
        assert_within(got["out"], want["out"], bound["out"], f"{L}: out")


@pytest.mark.parametrize("dtype", TYPES)
def test_gates_at_their_ends(hip_device, dtype):
    """Gates that hold or forget altogether: exact states, no NaN."""
    a = inputs(1, 300, 8, dtype, seed=1)
    a["gates"][:, :, 0], a["gates"][:, :, 1] = float("inf"), float("-inf")
    a["gates"][:, :, 2], a["gates"][:, :, 3] = 200.0, -200.0
    got = run(hip_device, a)
    first, x = a["initial"].cuda(), a["x"].cuda()
    assert torch.equal(got["out"][0, :, 0], first[0, 0].to(TYPES[dtype]).expand(300)) and torch.equal(got["out"][0, :, 1], x[0, :, 1])
    assert torch.equal(got["out"][0, :, 2], got["out"][0, :1, 2].expand(300)) and torch.equal(got["out"][0, :, 3], x[0, :, 3])
    for n in ("x_grad", "gates_grad", "initial_grad"):
        assert got[n].isfinite().all()
    a["gates"][0, 100, 4] = float("nan")
    got = run(hip_device, a)
    assert got["out"][0, 100:, 4].isnan().all() and got["out"][0, :100].isfinite().all() and got["out"][0, :, 5:].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
@pytest.mark.parametrize("layout", ["unaligned", "length first", "heads of a wider array"])
def test_layouts(hip_device, layout, factors, dtype):
    a = inputs(3, 300, 45, dtype, factors=factors, seed=7, documents=0.01, lengths=[300, 280, 299])
    plain = run(hip_device, a, factors=factors)

    def strided(x):
        if layout == "length first":
            return x.transpose(0, 1).contiguous().transpose(0, 1)
        extra = 3 if layout == "unaligned" else 64
        wide = torch.zeros((*x.shape[:-1], x.shape[-1] + extra), dtype=x.dtype)
        wide[..., 1:1 + x.shape[-1]] = x
        return wide[..., 1:1 + x.shape[-1]]

    a |= {n: strided(a[n]) for n in ("x", "gates", "out_grad")}
    a["documents"] = a["documents"].T.contiguous().T
    a["lengths"] = torch.stack((a["lengths"], a["lengths"] * 0), 1)[:, 0]
    a["initial"] = torch.cat((a["initial"], a["initial"]), 1)[:, :45]
    got = run(hip_device, a, factors=factors, like=lambda x: strided(torch.zeros(x.shape, dtype=x.dtype)).cuda() if layout != "length first"
              else torch.empty_like(x))
    assert all(torch.equal(got[n], plain[n]) for n in plain), "strides decide over no bit"


def test_inputs_that_are_broadcast(hip_device):
    """One gate for all positions and sequences."""
    a = inputs(2, 270, 33, "f32", seed=7)
    a["gates"] = a["gates"][:1, :1].expand(2, 270, 33)
    check(hip_device, a, "broadcast")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factors", [False, True])
def test_tokens_one_by_one(hip_device, factors, dtype):
    """A state that is carried from call to call in one array gives what one call over all positions gives, within both bounds."""
    B, L, C = 3, 21, 70
    a = inputs(B, L, C, dtype, factors=factors, seed=8)
    want, bound = oracle.recurrence(a["x"], a["gates"], factors=factors, initial=a["initial"])
    x, gates, state = a["x"].cuda(), a["gates"].cuda(), a["initial"].cuda()
    out = torch.empty_like(x)
    for t in range(0, L, 3):
        for n in ((1, 1, 1), (3,), (2, 1))[t % 3]:
            ops.recurrence(hip_device, x[:, t:t + n], gates[:, t:t + n], out[:, t:t + n], factors=factors, initial=state, final=state, stream=here())
            t += n
    assert_within(out, want["out"], bound["out"], f"tokens, {dtype}")
    assert_within(state, want["final"], bound["final"], f"state, {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [4, 600, 3000])
def test_in_place(hip_device, L, dtype):
    a = inputs(2, L, 50, dtype, seed=9)
    want = run(hip_device, a)
    for n in ("x", "gates"):
        g = {k: to_gpu(v) for k, v in a.items()}
        room = torch.empty(ops.recurrence_workspace(hip_device, g["x"]) + 16, dtype=torch.uint8, device="cuda")
        ops.recurrence(hip_device, g["x"], g["gates"], g[n], initial=g["initial"], workspace=room, stream=here())
        assert torch.equal(g[n], want["out"])
    for to in (("x", "gates"), ("out_grad", "x"), ("gates", "out_grad")):
        g = {k: to_gpu(v) for k, v in a.items()}
        room = torch.empty(ops.recurrence_workspace(hip_device, g["x"], backward=True) + 16, dtype=torch.uint8, device="cuda")
        ops.recurrence_backward(hip_device, g["x"], g["gates"], want["states"], g["out_grad"], g[to[0]], g[to[1]], final_grad=g["final_grad"],
                                initial_grad=g["initial"], workspace=room, stream=here())
        assert torch.equal(g[to[0]], want["x_grad"]) and torch.equal(g[to[1]], want["gates_grad"]) and torch.equal(g["initial"], want["initial_grad"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L,C", [(600, 300), (5000, 40), (9001, 930)])
def test_a_state_in_place_over_long_sequences(hip_device, L, C, dtype):
    """The last range of positions writes the state that the first one begins with."""
    a = {n: to_gpu(x) for n, x in inputs(1, L, C, dtype, factors=True, seed=4, slow=8.0).items()}
    room = torch.empty(ops.recurrence_workspace(hip_device, a["x"]) + 16, dtype=torch.uint8, device="cuda")
    out, final = torch.empty_like(a["x"]), torch.empty_like(a["initial"])
    for _ in range(3):
        ops.recurrence(hip_device, a["x"], a["gates"], out, factors=True, initial=a["initial"], final=final, workspace=room, stream=here())
        state, again = a["initial"].clone(), torch.empty_like(out)
        ops.recurrence(hip_device, a["x"], a["gates"], again, factors=True, initial=state, final=state, workspace=room, stream=here())
        assert torch.equal(out, again) and torch.equal(final, state)
        a["initial"] = state


@pytest.mark.parametrize("factors", [False, True])
def test_no_positions_and_no_sequences(hip_device, factors):
    a = inputs(2, 0, 40, "f32", factors=factors)
    got = run(hip_device, a, factors=factors)
    assert torch.equal(got["final"], a["initial"].cuda()) and torch.equal(got["initial_grad"], a["final_grad"].cuda())
    run(hip_device, inputs(0, 5, 40, "f32"), factors=factors)
    run(hip_device, inputs(2, 5, 0, "f32"), factors=factors)


@pytest.mark.parametrize("L", [300, 4000])
def test_the_same_inputs_give_the_same_bits(hip_device, L):
    a = inputs(2, L, 100, "bf16", seed=11)
    first = run(hip_device, a)
    for _ in range(3):
        again = run(hip_device, a)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_long_memory(hip_device):
    """States that hardly fade over ten thousand positions."""
    a = inputs(1, 10000, 5, "f32", seed=12)
    a["gates"] = a["gates"] * 0.1 + torch.tensor([8.0, 9.0, 10.0, 11.0, 12.0])
    check(hip_device, a, "long memory")

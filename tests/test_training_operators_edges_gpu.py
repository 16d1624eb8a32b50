"""Layer norm, the recurrence, the norm over gradients and AdamW behind it together as a training step makes them, captured and
replayed, on other streams, beside one another, and at offsets that 32 bits do not hold."""
import pytest
import torch

import training_oracle as oracle
from adhip import operators as ops
from test_operators_gpu import TYPES, assert_within, here

pytestmark = pytest.mark.gpu


class Step:
    """norm -> recurrence -> norm's way back -> clipped AdamW on the norm's weights, as calls on arrays that a program keeps."""

    def __init__(self, dev, dtype, B=2, L=700, C=200, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = TYPES[dtype]
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.dev, self.dtype = dev, t
        self.x, self.branch, self.gates, self.dout = (rand(B, L, C).to(t) for _ in range(4))
        self.weight, self.bias = 1 + 0.1 * rand(C), 0.1 * rand(C)
        self.documents = torch.cumsum(torch.rand((B, L), generator=g, device="cuda") < 0.01, 1).to(torch.int32)
        self.total, self.normed, self.out, self.dnormed, self.dgates, self.dx = (torch.empty_like(self.x) for _ in range(6))
        self.stats, self.states = torch.empty((B, L, 2), device="cuda"), torch.empty((B, ops.recurrence_blocks(L), C), device="cuda")
        self.final = torch.empty((B, C), device="cuda")
        self.dweight, self.dbias = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        self.norm, self.factor = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
        self.first, self.second = [torch.zeros(C, device="cuda") for _ in "wb"], [torch.zeros(C, device="cuda") for _ in "wb"]
        self.new = [torch.empty(C, device="cuda") for _ in "wb"]
        self.first_new, self.second_new = [torch.empty(C, device="cuda") for _ in "wb"], [torch.empty(C, device="cuda") for _ in "wb"]
        need = max(ops.layer_norm_workspace(dev, self.x), ops.recurrence_workspace(dev, self.x, backward=True),
                   ops.gradient_norm_workspace(dev, [self.dweight, self.dbias, self.dgates]))
        self.room = torch.empty(need, dtype=torch.uint8, device="cuda")  # one for all: each call is done with it before the next

    def run(self, stream):
        how = dict(workspace=self.room, stream=stream)
        ops.layer_norm(self.dev, self.x, self.normed, weight=self.weight, bias=self.bias, added=self.branch, total=self.total, stats=self.stats,
                       stream=stream)
        ops.recurrence(self.dev, self.normed, self.gates, self.out, final=self.final, states=self.states, documents=self.documents, **how)
        ops.recurrence_backward(self.dev, self.normed, self.gates, self.states, self.dout, self.dnormed, self.dgates, documents=self.documents, **how)
        ops.layer_norm_backward(self.dev, self.total, self.stats, self.dnormed, self.dx, weight=self.weight, weight_grad=self.dweight,
                                bias_grad=self.dbias, total_grad=self.dout, **how)
        ops.gradient_norm(self.dev, [self.dweight, self.dbias, self.dgates], self.norm, limit=1.0, factor=self.factor, **how)
        ops.adamw(self.dev, [self.weight, self.bias], [self.dweight, self.dbias], self.first, self.second, step=1, rate=0.1, factor=self.factor,
                  parameters_out=self.new, first_out=self.first_new, second_out=self.second_new, stream=stream)

    def results(self):
        return [self.total, self.normed, self.stats, self.out, self.final, self.states, self.dnormed, self.dgates, self.dx, self.dweight, self.dbias,
                self.norm, self.factor, *self.new, *self.first_new, *self.second_new]

    def clear(self):
        for t in self.results():
            t.fill_(7.0)
        self.room.fill_(255)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_step_is_its_formulas(hip_device, dtype):
    """The calls one after the other, each against its own restatement on what the calls before it gave."""
    s = Step(hip_device, dtype)
    s.clear()
    s.run(here())
    torch.cuda.synchronize()
    c = lambda t: t.detach().cpu()  # noqa: E731
    want, bound = oracle.layer_norm(c(s.x), c(s.weight), c(s.bias), added=c(s.branch), out_grad=c(s.dnormed), total_grad=c(s.dout))
    for n, got in (("total", s.total), ("out", s.normed), ("stats", s.stats), ("x_grad", s.dx), ("weight_grad", s.dweight), ("bias_grad", s.dbias)):
        assert_within(got, want[n], bound[n], n)
    want, bound = oracle.recurrence(c(s.normed), c(s.gates), documents=c(s.documents), out_grad=c(s.dout))
    for n, got in (("out", s.out), ("final", s.final), ("states", s.states), ("x_grad", s.dnormed), ("gates_grad", s.dgates)):
        assert_within(got, want[n], bound[n], n)
    grads = [c(s.dweight), c(s.dbias), c(s.dgates)]
    want, bound = oracle.clip(grads, 1.0)
    assert_within(s.norm, want["norm"], bound["norm"], "norm")
    assert_within(s.factor, want["factor"], bound["factor"], "factor")
    f = float(s.factor)
    assert 0 < f < 1
    for p, g, new in zip((s.weight, s.bias), grads, s.new):
        m, v = 0.1 * f * g.double(), 0.001 * (f * g.double()) ** 2
        step = 0.1 * (m / 0.1) / ((v / 0.001).sqrt() + 1e-8)
        # the step is 0.1 at most, made of ten rounded operations; the parameter is rounded once, its decay once
        assert float((new.cpu().double() - (c(p).double() * (1 - 0.1 * 0.01) - step)).abs().max()) <= 0.1 * 16 * 2.0 ** -24 + 2.0 ** -22


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [5, 700, 3000])
def test_captured_steps(hip_device, L, dtype):
    """Two captured steps that share a workspace, replayed in turn with eager work and new inputs between them."""
    steps = [Step(hip_device, dtype, L=L, seed=i) for i in range(2)]
    steps[1].room = steps[0].room
    eager, graphs = [], []
    for s in steps:
        s.clear()
        s.run(here())
        torch.cuda.synchronize()
    for s in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run(here())
        graphs.append(graph)
    for turn in range(3):
        for s, graph in zip(steps, graphs):
            s.x.normal_(generator=torch.Generator(device="cuda").manual_seed(10 + turn))
            s.clear()
            s.run(here())
            torch.cuda.synchronize()
            eager = [t.clone() for t in s.results()]
            s.clear()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(s.results(), eager)), f"replay {turn}"
    for s, graph in zip(steps, graphs):
        s.clear()
    for graph in graphs:  # one right behind the other
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(steps[1].results(), eager))


@pytest.mark.parametrize("dtype", TYPES)
def test_streams_beside_one_another(hip_device, dtype):
    """Two steps at once, each on a stream and with a workspace of its own, give what they give alone."""
    steps, alone = [Step(hip_device, dtype, L=1500, seed=i) for i in range(2)], []
    for s in steps:
        s.run(here())
        torch.cuda.synchronize()
        alone.append([t.clone() for t in s.results()])
        s.clear()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        for s, stream in zip(steps, streams):
            s.run(stream.cuda_stream)
    torch.cuda.synchronize()
    for s, want in zip(steps, alone):
        assert all(torch.equal(a, b) for a, b in zip(s.results(), want))


def test_the_devices_own_stream(hip_device):
    """Without a stream the calls go to the device's own, one after the other."""
    s = Step(hip_device, "f32")
    s.run(here())
    torch.cuda.synchronize()
    want = [t.clone() for t in s.results()]
    s.clear()
    torch.cuda.synchronize()
    s.run(None)
    ops.synchronize(hip_device)
    assert all(torch.equal(a, b) for a, b in zip(s.results(), want))


def far_apart(shape, stride, dtype):
    """An array whose memory reaches past what 32 bits count, of which only its own elements are written."""
    span = 1 + sum((n - 1) * s for n, s in zip(shape, stride))
    return torch.empty(span, dtype=dtype, device="cuda").as_strided(shape, stride)


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_beyond_32_bits(hip_device, dtype):
    t = TYPES[dtype]
    # rows 2^31 elements and more apart
    shape, stride = (3, 2, 33), ((1 << 30) + 5, (1 << 29) + 3, 1)
    near = torch.randn(shape, dtype=torch.float32, device="cuda").to(t)
    x, out = far_apart(shape, stride, t), far_apart(shape, stride, t)
    x.copy_(near)
    ops.layer_norm(hip_device, x, out, stream=here())
    want = torch.empty_like(near)
    ops.layer_norm(hip_device, near, want, stream=here())
    assert torch.equal(out, want)
    del x, out
    # positions as far apart as they may be, over more than a tile
    shape = (1, 600, 6)
    x, gates = (torch.randn(shape, device="cuda").to(t) for _ in range(2))
    far = far_apart(shape, (1 << 31, 1 << 21, 1), t)
    far.copy_(x)
    room = torch.empty(ops.recurrence_workspace(hip_device, x) + 16, dtype=torch.uint8, device="cuda")
    want = torch.empty_like(x)
    ops.recurrence(hip_device, x, gates, want, workspace=room, stream=here())
    ops.recurrence(hip_device, far, gates, far, workspace=room, stream=here())
    assert torch.equal(far, want)


def test_gradients_beyond_32_bits(hip_device):
    """More than 2^32 bytes in one tensor: the last elements count."""
    n = (1 << 31) + 5
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-3:] = torch.tensor([3.0, 4.0, 12.0])
    norm, factor = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    room = torch.empty(ops.gradient_norm_workspace(hip_device, [g]), dtype=torch.uint8, device="cuda")
    ops.clip_gradients(hip_device, [g], norm, limit=6.5, factor=factor, workspace=room, stream=here())
    assert float(norm) == 13.0 and float(factor) == 0.5
    assert g[-4:].tolist() == [0.0, 1.5, 2.0, 6.0]


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_past_the_caches(hip_device, dtype):
    """A call whose arrays pass the last cache writes past it; the same rows in calls of a quarter do not, and give the same bits."""
    rows, size = (16000, 4099) if dtype == "f32" else (32000, 4096)
    t = TYPES[dtype]
    x, added, dy, dt = (torch.randn((rows, size), device="cuda").to(t) for _ in range(4))
    w = torch.randn(size, device="cuda")
    stats = torch.empty((rows, 2), device="cuda")

    def both(x, added, dy, dt, stats):
        total, out, dx, dw = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x), torch.empty(size, device="cuda")
        room = torch.empty(ops.layer_norm_workspace(hip_device, x), dtype=torch.uint8, device="cuda")
        ops.layer_norm(hip_device, x, out, weight=w, added=added, total=total, stats=stats, stream=here())
        ops.layer_norm_backward(hip_device, total, stats, dy, dx, weight=w, weight_grad=dw, total_grad=dt, workspace=room, stream=here())
        return total, out, dx, dw

    assert rows * size * x.element_size() * 4 > 1 << 28 > rows * size * x.element_size()
    whole = both(x, added, dy, dt, stats)
    parts = [both(*(a.reshape(4, rows // 4, -1)[i] for a in (x, added, dy, dt, stats))) for i in range(4)]
    for i in range(3):
        assert torch.equal(whole[i], torch.cat([part[i] for part in parts]))
    assert torch.allclose(whole[3], sum(part[3] for part in parts), rtol=1e-4, atol=1e-4 * rows ** 0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,C", [(1, 1300, 60001), (9, 700, 7000), (1, 300000, 150)])
def test_recurrences_past_the_caches(hip_device, B, L, C, dtype):
    """Channels are independent: some of a call that passes the last cache, against their restatement."""
    t = TYPES[dtype]
    L = L if dtype == "bf16" or L < 100000 else L // 2
    x, gates, dout = (torch.randn((B, L, C), device="cuda").to(t) for _ in range(3))
    assert 3 * x.numel() * x.element_size() > 1 << 28 or 5 * x.numel() * x.element_size() > 1 << 28
    out, dx, dg = (torch.empty_like(x) for _ in range(3))
    states = torch.empty((B, ops.recurrence_blocks(L), C), device="cuda")
    room = torch.empty(ops.recurrence_workspace(hip_device, x, backward=True) + 16, dtype=torch.uint8, device="cuda")
    ops.recurrence(hip_device, x, gates, out, states=states, workspace=room, stream=here())
    ops.recurrence_backward(hip_device, x, gates, states, dout, dx, dg, workspace=room, stream=here())
    some = [0, 1, C // 3, C - 2, C - 1]
    if L <= 20000:
        pick = lambda a: a[..., some].cpu()  # noqa: E731
        first = last = 0
    else:  # the beginning of the long one (its states fade within some hundred positions), and its end backwards
        first, last = 0, 3000
        pick = lambda a: a[:, :3000, some].cpu()  # noqa: E731
    want, bound = oracle.recurrence(pick(x), pick(gates), out_grad=pick(dout))
    assert_within(out[:, first:last or L, some], want["out"], bound["out"], "out")
    end = (last - 400) if last else L  # the gradient of what lies behind the part has faded 400 positions before its end: a < 0.98^400
    for n, got in (("x_grad", dx), ("gates_grad", dg)):
        assert_within(got[:, :end, some], want[n][:, :end], bound[n][:, :end] + (1e-3 * want[n].abs().max() if last else 0), n)


def test_gradients_past_the_caches(hip_device):
    g = [torch.randn(n, device="cuda") for n in (30_000_001, 8_000_000, 5)]
    out, norm, factor = [torch.full_like(x, 7.0) for x in g], torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    room = torch.empty(ops.gradient_norm_workspace(hip_device, g), dtype=torch.uint8, device="cuda")
    ops.clip_gradients(hip_device, g, norm, limit=1.0, factor=factor, gradients_out=out, workspace=room, stream=here())
    assert all(torch.equal(o, x * factor) for x, o in zip(g, out))
    want = torch.sqrt(sum((x.double() ** 2).sum() for x in g))
    assert abs(float(norm) / float(want) - 1) <= 2.0 ** -23

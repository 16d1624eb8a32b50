"""Layers that train through programs and operators together (adhip.decoder) with a norm, with clipped gradients and with the
recurrence, against the same steps in 64-bit torch with its own backward pass."""
import numpy as np
import pytest
import torch

from adhip import operators as ops
from adhip.decoder import DecoderAttention, DecoderRecurrence

pytestmark = pytest.mark.gpu


def attention(w, x, heads, key_heads, size, documents):
    B, L, _ = x.shape
    cos, sin = (torch.from_numpy(t).double()[None, :, None, :] for t in ops.rotary_table(L, size))

    def turn(t):
        a, b = t[..., :size // 2], t[..., size // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    q, k, v = (torch.matmul(x, w["W" + n]).view(B, L, -1, size) for n in "qkv")
    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(heads // key_heads, 2) for t in (k, v))
    sees = torch.tril(torch.ones(L, L, dtype=torch.bool))[None].repeat(B, 1, 1)
    if documents is not None:
        d = torch.from_numpy(documents)
        sees = sees & (d[:, :, None] == d[:, None, :])
    z = torch.einsum("bihd,bjhd->bhij", q, k) * size ** -0.5
    return torch.einsum("bhij,bjhd->bihd", torch.softmax(z.masked_fill(~sees[:, None], -np.inf), -1), v).reshape(B, L, -1)


def recurrence(w, x, documents):
    u, a = torch.matmul(x, w["Wu"]), torch.sigmoid(torch.matmul(x, w["Wg"]))
    h, rows = torch.zeros_like(u[:, 0]), []
    for t in range(x.shape[1]):
        if documents is not None and t > 0:
            h = h * torch.from_numpy((documents[:, t] == documents[:, t - 1]).astype(np.float64))[:, None]
        h = a[:, t] * h + (1 - a[:, t]) * u[:, t]
        rows.append(h)
    return torch.stack(rows, 1)


def reference(start, x, target, mix, steps, rate, clip):
    """Losses, norms of the gradients before they are clipped, and the weights at the end."""
    w = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in start.items()}
    xt, yt = torch.tensor(x, dtype=torch.float64), torch.tensor(target, dtype=torch.float64)
    optimizer = torch.optim.AdamW(w.values(), lr=rate, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    losses, norms = [], []
    for _ in range(steps):
        o = mix(w, xt)
        if "scale" in w:
            o = (o - o.mean(-1, keepdim=True)) / torch.sqrt(o.var(-1, unbiased=False, keepdim=True) + 1e-5) * w["scale"] + w["bias"]
        loss = ((o @ w["Wo"] - yt) ** 2).mean()
        optimizer.zero_grad()
        loss.backward()
        norm = torch.sqrt(sum((t.grad ** 2).sum() for t in w.values()))
        if clip:
            for t in w.values():
                t.grad *= min(1.0, clip / float(norm))
        optimizer.step()
        losses.append(float(loss.detach()))
        norms.append(float(norm))
    return losses, norms, {n: t.detach().numpy() for n, t in w.items()}


@pytest.mark.parametrize("kind", ["attention", "recurrence"])
@pytest.mark.parametrize("norm,clip,packed", [(True, 0.0, False), (False, 0.02, False), (True, 0.05, True), (False, 0.0, True), (True, 1e3, False)])
def test_steps_are_those_of_the_formulas(hip_device, kind, norm, clip, packed):
    rng = np.random.default_rng(5)
    B, L, width, steps = 2, 45, 24, 4
    x, target = (rng.standard_normal((B, L, width)).astype(np.float32) for _ in range(2))
    documents = np.sort(rng.integers(0, 3, (B, L)), 1).astype(np.int32) if packed else None
    how = dict(rate=1e-3, norm=norm, clip=clip, documents=documents)
    if kind == "attention":
        layer = DecoderAttention(hip_device, x, target, 4, 2, 32, **how)
        mix = lambda w, t: attention(w, t, 4, 2, 32, documents)  # noqa: E731
    else:
        layer = DecoderRecurrence(hip_device, x, target, 70, **how)
        mix = lambda w, t: recurrence(w, t, documents)  # noqa: E731
    start = {n: a.copy() for n, a in layer.weights.items()}
    assert ("scale" in start) == norm
    losses, norms = [], []
    for _ in range(steps):
        layer.step()
        losses.append(layer.loss())
        if clip:
            norms.append(float(layer.grad_norm.numpy()[0]))
            assert np.isclose(float(layer.factor.numpy()[0]), min(1.0, clip / norms[-1]), rtol=1e-6)
    want, want_norms, weights = reference(start, x, target, mix, steps, 1e-3, clip)
    assert np.allclose(losses, want, rtol=1e-5), (losses, want)
    if clip:
        assert np.allclose(norms, want_norms, rtol=1e-4), (norms, want_norms)
        assert clip > 1 or min(norms) > clip, "the limit takes hold"
    for n, a in weights.items():
        # four steps of 1e-3 at most; a step's direction is a gradient over its own size, whose error near zero is larger than
        # a product's: a hundredth of the way is far outside of that and far inside of a wrong gradient
        assert np.abs(layer.weight(n).reshape(a.shape) - a).max() <= 4e-5, n
        assert np.abs(layer.weight(n).reshape(a.shape) - start[n]).max() > 1e-3, n


def test_gradients_of_a_layer_against_differences(hip_device):
    """The gradients that a step leaves, along a direction, against the loss at both sides of the weights."""
    rng = np.random.default_rng(8)
    x, target = (rng.standard_normal((2, 300, 16)).astype(np.float32) for _ in range(2))
    layer = DecoderRecurrence(hip_device, x, target, 40, rate=0.0, norm=True)
    layer.step()
    for name in ("Wu", "Wg", "Wo", "scale", "bias"):
        grad, at = layer.arrays["d" + name].numpy().astype(np.float64), layer.weight(name)
        along = np.sign(grad).astype(np.float32)  # the slope is the sum of all magnitudes: nothing cancels
        step, sides = 2.0 ** -9, []
        for side in (1, -1):
            layer.arrays[name].set((at.reshape(-1) + side * step * along.reshape(-1)).reshape(at.shape))
            layer.forward()
            sides.append(layer.loss())
        layer.arrays[name].set(at)
        slope, want = (sides[0] - sides[1]) / (2 * step), float(np.abs(grad).sum())
        # a loss of about one is rounded to 2^-24 on each side, some operations deep: 2^-20 over 2^-8; curvature enters by step^2
        assert abs(slope - want) <= 2.0 ** -12 + 0.02 * want, (name, slope, want)


def test_a_state_that_is_carried_gives_the_rows_of_the_whole(hip_device):
    """Positions one by one, as they are generated, from a state in place."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 37, 16)).astype(np.float32)
    layer = DecoderRecurrence(hip_device, x, x, 48)
    layer.forward()
    whole, u, g = (layer.seen[n].numpy() for n in "mug")
    state = ops.DeviceArray.of(hip_device, np.zeros((2, 48), np.float32))
    for t in range(37):
        ut, gt = ops.DeviceArray.of(hip_device, u[:, t:t + 1]), ops.DeviceArray.of(hip_device, g[:, t:t + 1])
        out = ops.DeviceArray.empty(hip_device, (2, 1, 48))
        ops.recurrence(hip_device, ut, gt, out, initial=state, final=state)
        assert np.allclose(out.numpy()[:, 0], whole[:, t], rtol=0, atol=1e-6 * np.abs(whole).max())


def test_layers_refuse(hip_device):
    x = np.zeros((1, 4, 8), np.float32)
    with pytest.raises(ValueError, match="clip"):
        DecoderRecurrence(hip_device, x, x, 8, clip=-1.0)
    with pytest.raises(ValueError, match="target"):
        DecoderRecurrence(hip_device, x, x[:, :2], 8)

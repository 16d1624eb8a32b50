"""The decoder layer that trains through programs and operators together (adhip.decoder), against the same steps in 64-bit
torch with its own backward pass."""
import numpy as np
import pytest
import torch

from adhip import operators as ops
from adhip.decoder import DecoderAttention

pytestmark = pytest.mark.gpu


def reference(weights, x, target, heads, key_heads, size, steps, *, rate, cap, window, documents):
    B, L, width = x.shape
    w = {n: torch.tensor(a, dtype=torch.float64, requires_grad=True) for n, a in weights.items()}
    xt, yt = torch.tensor(x, dtype=torch.float64), torch.tensor(target, dtype=torch.float64)
    cos, sin = (torch.from_numpy(t).double()[None, :, None, :] for t in ops.rotary_table(L, size))

    def turn(t):
        a, b = t[..., :size // 2], t[..., size // 2:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)

    far = torch.arange(L)[:, None] - torch.arange(L)[None, :]
    sees = far >= 0
    if window:
        sees = sees & (far < window)
    sees = sees[None].repeat(B, 1, 1)
    if documents is not None:
        d = torch.from_numpy(documents)
        sees = sees & (d[:, :, None] == d[:, None, :])
    optimizer = torch.optim.AdamW(w.values(), lr=rate, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    losses = []
    for _ in range(steps):
        q, k, v = (torch.matmul(xt, w[n]).view(B, L, -1, size) for n in ("Wq", "Wk", "Wv"))
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(heads // key_heads, 2) for t in (k, v))
        z = torch.einsum("bihd,bjhd->bhij", q, k) * size ** -0.5
        z = cap * torch.tanh(z / cap) if cap else z
        o = torch.einsum("bhij,bjhd->bihd", torch.softmax(z.masked_fill(~sees[:, None], -np.inf), -1), v).reshape(B, L, -1)
        loss = ((o @ w["Wo"] - yt) ** 2).mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses, {n: t.detach().numpy() for n, t in w.items()}


@pytest.mark.parametrize("heads,key_heads,size,how", [(4, 2, 32, dict()), (3, 1, 20, dict(cap=5.0, window=11)), (2, 2, 64, dict(documents=True))])
def test_steps_are_those_of_the_formulas(hip_device, heads, key_heads, size, how):
    rng = np.random.default_rng(5)
    B, L, width = 2, 45, 24
    x, target = (rng.standard_normal((B, L, width)).astype(np.float32) for _ in range(2))
    how = {"cap": 0.0, "window": 0, **how}
    how["documents"] = np.sort(rng.integers(0, 3, (B, L)), 1).astype(np.int32) if how.pop("documents", False) else None
    layer = DecoderAttention(hip_device, x, target, heads, key_heads, size, rate=1e-3, **how)
    start = {n: a.copy() for n, a in layer.weights.items()}
    losses = []
    for _ in range(4):
        layer.step()
        losses.append(layer.loss())
    want, weights = reference(start, x, target, heads, key_heads, size, 4, rate=1e-3, **how)
    assert np.allclose(losses, want, rtol=1e-5), (losses, want)
    for n, a in weights.items():
        # four steps of 1e-3 at most; a step's direction is a gradient over its own size, whose error near zero is larger than
        # a product's: a hundredth of the way is far outside of that and far inside of a wrong gradient
        assert np.abs(layer.weight(n) - a).max() <= 4e-5, n
        assert np.abs(layer.weight(n) - start[n]).max() > 1e-3, n


def test_states_in_eight_bits_train_too(hip_device):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, 64, 32)).astype(np.float32)
    target = np.cumsum(x, 1) / np.arange(1, 65, dtype=np.float32)[None, :, None]
    ends = {}
    for eight in (False, True):
        layer = DecoderAttention(hip_device, x, target, 4, 4, 16, rate=1e-2, eight_bit_states=eight)
        layer.step()
        first = layer.loss()
        for _ in range(40):
            layer.step()
        ends[eight] = layer.loss()
        assert ends[eight] < 0.5 * first
    assert abs(ends[True] - ends[False]) < 0.25 * ends[False]


def test_a_token_against_the_cache_is_the_last_row(hip_device):
    """The last position of a sequence, computed alone against keys and values as a cache, is the last row of the whole."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 77, 32)).astype(np.float32)
    layer = DecoderAttention(hip_device, x, x, 4, 2, 16, cap=20.0)
    layer.forward()
    h = layer.heads
    whole, q = h["o"].numpy(), h["q"].numpy()
    last = ops.DeviceArray.of(hip_device, q[:, -1:])
    out, lse = ops.DeviceArray.empty(hip_device, last.shape), ops.DeviceArray.empty(hip_device, (2, 1, 4))
    room = ops.DeviceArray.empty(hip_device, (max(1, ops.attention_workspace(hip_device, last, h["k"], h["v"]) // 4),))
    ops.attention(hip_device, last, h["k"], h["v"], out, lse, causal=True, cap=20.0, workspace=room)
    assert np.allclose(out.numpy()[:, 0], whole[:, -1], rtol=0, atol=1e-5 * np.abs(whole).max())
    assert np.allclose(lse.numpy()[:, 0], layer.lse.numpy()[:, -1], rtol=1e-6)

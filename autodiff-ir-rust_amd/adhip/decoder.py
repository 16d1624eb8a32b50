"""Training of a decoder's layers that mix positions, resident on the GPU: the products run as programs of the autodiff front end,
what lies between them as operators on the programs' own buffers, and nothing passes through the host.

DecoderAttention
    q, k, v = x Wq, x Wk, x Wv          program `project`
    q, k    = rotary(q, k)              in place
    m       = attention(q, k, v)        causal, heads that share key heads, capped scores and packed documents as asked for
DecoderRecurrence
    u, g    = x Wu, x Wg                program `project`
    m       = recurrence(u, g)          m = a m + (1 - a) u with a = sigmoid(g), documents as asked for
and of both
    o       = m, or layer_norm(m)
    y = o Wo, loss, dWo, do             program `close`, with the front end's backward pass
    do -> dm -> dq, dk, dv or du, dg    the operators' backward calls
    dWq, ... = x' dq, ...               program `weigh`
    the norm over all gradients, where they are clipped
    AdamW on all weights                in the buffers that the next step's programs read

    python -m adhip.decoder [attention | recurrence]     trains one on random data and prints the loss
"""
from __future__ import annotations

import sys
from typing import Optional

import numpy as np

from . import autodiff, operators as ops
from . import ir as IR
from .core import STATE, dot


def _compile(dev):
    """What the front end has recorded since set_device, as a resident program."""
    STATE.irb.add_cmd(IR.EX())
    program = dev.compile(STATE.irb.proc, set(STATE.dep_tracker))
    program.upload()
    return program


class DecoderLayer:
    """What layers have in common.  x, target [batch, length, width] (float32); `step()` queues one training step on
    mean((y - target)^2).  `parts` names what x is projected to, and how wide; `mixed` is how wide the mixed positions are.  `norm` puts a
    layer norm behind them, `clip` limits the norm over all gradients (0: none)."""

    def __init__(self, dev, x, target, parts: dict, mixed: int, *, rate: float = 1e-2, decay: float = 0.0, norm: bool = False,
                 clip: float = 0.0, documents: Optional[np.ndarray] = None, eight_bit_states: bool = False, seed: int = 0):
        x, target = np.ascontiguousarray(x, np.float32), np.ascontiguousarray(target, np.float32)
        batch, length, width = x.shape
        if target.shape != x.shape:
            raise ValueError(f"target is {list(target.shape)}, x {list(x.shape)}")
        if not clip >= 0.0:
            raise ValueError(f"clip {clip}: a limit above zero is wanted, or 0 for none")
        if documents is not None:
            documents = ops._host_values(documents, "int32").reshape(batch, length)
        rows = batch * length
        self.dev, self.rate, self.decay, self.clip, self.steps = dev, rate, decay, clip, 0
        rng = np.random.default_rng(seed)
        self.weights = {n: (rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)
                        for n, s in [("W" + n, (width, w)) for n, w in parts.items()] + [("Wo", (mixed, width))]}
        self.names = list(self.weights)

        def tensor(values):
            return autodiff.tensor(values, list(values.shape))

        # (ids begin anew in every program: what is looked up in one belongs to it)
        autodiff.set_device(dev)
        at = {"W" + n: tensor(self.weights["W" + n]) for n in parts}
        xt = tensor(x.reshape(rows, width))
        for n in parts:
            at[n] = dot(xt, at["W" + n])
            at[n].forward()
            at[n].val().keep()
        self.project = _compile(dev)
        self.arrays = {n: ops.program_array(self.project, t.val().id) for n, t in at.items()}

        autodiff.set_device(dev)
        o, wo, yt = tensor(np.zeros((rows, mixed), np.float32)), tensor(self.weights["Wo"]), tensor(target.reshape(rows, width))
        off = dot(o, wo) - yt
        loss = (off * off).sum(0).sum(0) * (1.0 / (rows * width))
        loss.forward()
        loss.backward()
        for v in (loss.val(), o.grad(), wo.grad()):
            v.keep()
        self.close = _compile(dev)
        for n, v in (("o", o.val()), ("Wo", wo.val()), ("loss", loss.val()), ("do", o.grad()), ("dWo", wo.grad())):
            self.arrays[n] = ops.program_array(self.close, v.id)

        autodiff.set_device(dev)
        xt = tensor(x.reshape(rows, width))
        grads = {"d" + n: tensor(np.zeros((rows, w), np.float32)) for n, w in parts.items()}
        made = {}
        for n, t in grads.items():
            made["dW" + n[1:]] = dot(xt.t(), t)
            made["dW" + n[1:]].forward()
            made["dW" + n[1:]].val().keep()
        self.weigh = _compile(dev)
        for n, t in {**grads, **made}.items():
            self.arrays[n] = ops.program_array(self.weigh, t.val().id)

        a = self.arrays
        self.documents = None if documents is None else ops.DeviceArray.of(dev, documents)
        self.norm = norm
        if norm:
            # the mixed positions as they are normed, and the gradient that comes back through the norm
            a["m"], a["dm"] = (ops.DeviceArray.empty(dev, (rows, mixed)) for _ in "md")
            self.stats = ops.DeviceArray.empty(dev, (rows, 2))
            self.norm_room = ops.DeviceArray.empty(dev, (ops.layer_norm_workspace(dev, a["m"]) // 4 + 1,))
            for n, values in (("scale", np.ones(mixed, np.float32)), ("bias", np.zeros(mixed, np.float32))):
                self.weights[n], a[n], a["d" + n] = values, ops.DeviceArray.of(dev, values), ops.DeviceArray.empty(dev, (mixed,))
                self.names.append(n)
        else:
            a["m"], a["dm"] = a["o"], a["do"]
        counts = [a[n].numel() for n in self.names]
        self.grads = [a["d" + n] for n in self.names]
        if clip:
            self.grad_norm, self.factor = (ops.DeviceArray.empty(dev, (1,)) for _ in "nf")
            self.clip_room = ops.DeviceArray.empty(dev, (ops.gradient_norm_workspace(dev, self.grads) // 4 + 1,))
        if eight_bit_states:
            def zero_codes():
                return [ops.DeviceArray.empty(dev, (ops.adamw_blocks(c), ops.ADAMW_BLOCK), "float8_e4m3fn") for c in counts]

            self.states = {"first": zero_codes(), "second": zero_codes(),
                           "first_scales": [ops.DeviceArray.of(dev, np.zeros(ops.adamw_blocks(c), np.float32)) for c in counts],
                           "second_scales": [ops.DeviceArray.of(dev, np.zeros(ops.adamw_blocks(c), np.float32)) for c in counts]}
            for s in self.states["first"] + self.states["second"]:
                s.clear()
        else:
            self.states = {k: [ops.DeviceArray.of(dev, np.zeros(c, np.float32)) for c in counts] for k in ("first", "second")}

    def mix(self):
        """From the projections to `m`."""
        raise NotImplementedError

    def mix_backward(self):
        """From `dm` to the projections' gradients."""
        raise NotImplementedError

    def forward(self):
        """Queues the layer up to the loss and the gradients of o and Wo."""
        a = self.arrays
        self.project.enqueue()
        self.mix()
        if self.norm:
            ops.layer_norm(self.dev, a["m"], a["o"], weight=a["scale"], bias=a["bias"], stats=self.stats)
        self.close.enqueue()

    def step(self):
        """Queues one training step."""
        a = self.arrays
        self.forward()
        if self.norm:
            ops.layer_norm_backward(self.dev, a["m"], self.stats, a["do"], a["dm"], weight=a["scale"], weight_grad=a["dscale"], bias_grad=a["dbias"],
                                    workspace=self.norm_room)
        self.mix_backward()
        self.weigh.enqueue()
        self.steps += 1
        how = {}
        if self.clip:
            ops.gradient_norm(self.dev, self.grads, self.grad_norm, limit=self.clip, factor=self.factor, workspace=self.clip_room)
            how["factor"] = self.factor
        ops.adamw(self.dev, [a[n] for n in self.names], self.grads, step=self.steps, rate=self.rate, decay=self.decay, **how, **self.states)

    def loss(self) -> float:
        """The loss of the last step's forward pass (waits)."""
        return float(self.arrays["loss"].numpy().reshape(-1)[0])

    def weight(self, name: str) -> np.ndarray:
        return self.arrays[name].numpy()


class DecoderAttention(DecoderLayer):
    """Attention, heads that share key heads; the other arguments as `DecoderLayer`'s."""

    def __init__(self, dev, x, target, heads: int, key_heads: int, size: int, *, window: int = 0, cap: float = 0.0, **how):
        super().__init__(dev, x, target, {"q": heads * size, "k": key_heads * size, "v": key_heads * size}, heads * size, **how)
        batch, length, _ = np.shape(x)
        # heads seen apart, tables, masks and workspace
        self.heads = {n: self.arrays[n].reshape(batch, length, h, size) for n, h in
                      (("q", heads), ("k", key_heads), ("v", key_heads), ("m", heads), ("o", heads), ("do", heads), ("dm", heads), ("dq", heads),
                       ("dk", key_heads), ("dv", key_heads))}
        self.lse = ops.DeviceArray.empty(dev, (batch, length, heads))
        self.cos, self.sin = (ops.DeviceArray.of(dev, t) for t in ops.rotary_table(length, size))
        self.positions = ops.DeviceArray.of(dev, np.broadcast_to(np.arange(length, dtype=np.int32), (batch, length)))
        self.masks = dict(causal=True, window=window, cap=cap, query_documents=self.documents, key_documents=self.documents)
        h = self.heads
        room = ops.attention_workspace(dev, h["q"], h["k"], h["v"], backward=True)
        self.room = ops.DeviceArray.empty(dev, ((room + 3) // 4,))

    def mix(self):
        h = self.heads
        ops.rotary(self.dev, h["q"], h["q"], self.cos, self.sin, self.positions, second=h["k"], second_out=h["k"])
        ops.attention(self.dev, h["q"], h["k"], h["v"], h["m"], self.lse, workspace=self.room, **self.masks)

    def mix_backward(self):
        h = self.heads
        ops.attention_backward(self.dev, h["q"], h["k"], h["v"], h["m"], self.lse, h["dm"], h["dq"], h["dk"], h["dv"], workspace=self.room,
                               **self.masks)
        ops.rotary(self.dev, h["dq"], h["dq"], self.cos, self.sin, self.positions, second=h["dk"], second_out=h["dk"], inverse=True)


class DecoderRecurrence(DecoderLayer):
    """A gated recurrence of `channels`; the other arguments as `DecoderLayer`'s.  What it knows of all positions before one is a state
    of `channels` numbers, whatever their number."""

    def __init__(self, dev, x, target, channels: int, **how):
        super().__init__(dev, x, target, {"u": channels, "g": channels}, channels, **how)
        batch, length, _ = np.shape(x)
        self.seen = {n: self.arrays[n].reshape(batch, length, channels) for n in ("u", "g", "m", "dm", "du", "dg")}
        self.kept = ops.DeviceArray.empty(dev, (batch, ops.recurrence_blocks(length), channels))
        self.room = ops.DeviceArray.empty(dev, (ops.recurrence_workspace(dev, self.seen["u"], backward=True) // 4 + 1,))

    def mix(self):
        s = self.seen
        ops.recurrence(self.dev, s["u"], s["g"], s["m"], states=self.kept, documents=self.documents, workspace=self.room)

    def mix_backward(self):
        s = self.seen
        ops.recurrence_backward(self.dev, s["u"], s["g"], self.kept, s["dm"], s["du"], s["dg"], documents=self.documents, workspace=self.room)


def main(kind: str = "attention"):
    if kind not in ("attention", "recurrence"):
        raise SystemExit(f"{kind}: attention or recurrence is wanted")
    from . import HipDevice
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 512, 256)).astype(np.float32)
    target = np.cumsum(x, 1) / np.arange(1, 513, dtype=np.float32)[None, :, None]  # the mean of what each position sees
    if kind == "recurrence":
        layer = DecoderRecurrence(HipDevice(0), x, target, channels=512, rate=3e-3, norm=True, clip=1.0)
    else:
        layer = DecoderAttention(HipDevice(0), x, target, heads=8, key_heads=2, size=64, rate=3e-3, cap=30.0)
    for i in range(101):
        layer.step()
        if i % 20 == 0:
            print(f"step {i}: loss {layer.loss():.5f}")


if __name__ == "__main__":
    main(*sys.argv[1:2])

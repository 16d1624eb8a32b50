"""Training of a decoder's attention layer, resident on the GPU: the products run as programs of the autodiff front end, what
lies between them as operators on the programs' own buffers, and nothing passes through the host.

    q, k, v = x Wq, x Wk, x Wv          program `project`
    q, k    = rotary(q, k)              in place
    o       = attention(q, k, v)        causal, heads that share key heads, capped scores and packed documents as asked for
    y = o Wo, loss, dWo, do             program `close`, with the front end's backward pass
    dq, dk, dv = attention_backward(do)
    dq, dk  = inverse rotary            in place
    dWq, dWk, dWv = x' dq, x' dk, x' dv program `weigh`
    AdamW on Wq, Wk, Wv, Wo             in the buffers that the next step's programs read

    python -m adhip.decoder             trains one on random data and prints the loss
"""
from __future__ import annotations

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


class DecoderAttention:
    """x, target [batch, length, width] (float32); `step()` queues one training step on mean((y - target)^2)."""

    def __init__(self, dev, x, target, heads: int, key_heads: int, size: int, *, rate: float = 1e-2, decay: float = 0.0, window: int = 0,
                 cap: float = 0.0, documents: Optional[np.ndarray] = None, eight_bit_states: bool = False, seed: int = 0):
        x, target = np.ascontiguousarray(x, np.float32), np.ascontiguousarray(target, np.float32)
        batch, length, width = x.shape
        if target.shape != x.shape:
            raise ValueError(f"target is {list(target.shape)}, x {list(x.shape)}")
        rows, wide, narrow = batch * length, heads * size, key_heads * size
        self.dev, self.rate, self.decay, self.steps = dev, rate, decay, 0
        rng = np.random.default_rng(seed)
        self.weights = {n: (rng.standard_normal(s) / np.sqrt(s[0])).astype(np.float32)
                        for n, s in (("Wq", (width, wide)), ("Wk", (width, narrow)), ("Wv", (width, narrow)), ("Wo", (wide, width)))}
        self.programs = []

        def tensor(values):
            return autodiff.tensor(values, list(values.shape))

        # (ids begin anew in every program: what is looked up in one belongs to it)
        autodiff.set_device(dev)
        at = {n: tensor(self.weights[n]) for n in ("Wq", "Wk", "Wv")}
        xt = tensor(x.reshape(rows, width))
        for n, w in (("q", "Wq"), ("k", "Wk"), ("v", "Wv")):
            at[n] = dot(xt, at[w])
            at[n].forward()
            at[n].val().keep()
        self.project = _compile(dev)
        self.arrays = {n: ops.program_array(self.project, t.val().id) for n, t in at.items()}

        autodiff.set_device(dev)
        o, wo, yt = tensor(np.zeros((rows, wide), np.float32)), tensor(self.weights["Wo"]), tensor(target.reshape(rows, width))
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
        parts = {n: tensor(np.zeros((rows, w), np.float32)) for n, w in (("dq", wide), ("dk", narrow), ("dv", narrow))}
        made = {}
        for n, t in parts.items():
            made["dW" + n[1]] = dot(xt.t(), t)
            made["dW" + n[1]].forward()
            made["dW" + n[1]].val().keep()
        self.weigh = _compile(dev)
        for n, t in {**parts, **made}.items():
            self.arrays[n] = ops.program_array(self.weigh, t.val().id)

        # heads seen apart, tables, masks, workspace and states
        self.heads = {n: self.arrays[n].reshape(batch, length, h, size) for n, h in
                      (("q", heads), ("k", key_heads), ("v", key_heads), ("o", heads), ("do", heads), ("dq", heads), ("dk", key_heads), ("dv", key_heads))}
        self.lse = ops.DeviceArray.empty(dev, (batch, length, heads))
        self.cos, self.sin = (ops.DeviceArray.of(dev, t) for t in ops.rotary_table(length, size))
        self.positions = ops.DeviceArray.of(dev, np.broadcast_to(np.arange(length, dtype=np.int32), (batch, length)))
        docs = None if documents is None else ops.DeviceArray.of(dev, np.asarray(documents, np.int32).reshape(batch, length))
        self.masks = dict(causal=True, window=window, cap=cap, query_documents=docs, key_documents=docs)
        h = self.heads
        room = ops.attention_workspace(dev, h["q"], h["k"], h["v"], backward=True)
        self.room = ops.DeviceArray.empty(dev, ((room + 3) // 4,))
        self.names = ["Wq", "Wk", "Wv", "Wo"]
        counts = [self.arrays[n].numel() for n in self.names]
        if eight_bit_states:
            def zero_codes():
                return [ops.DeviceArray.empty(dev, (ops.adamw_blocks(c), ops.ADAMW_BLOCK), "float8_e4m3fn") for c in counts]

            self.states = {"first": zero_codes(), "second": zero_codes(),
                           "first_scales": [ops.DeviceArray.of(dev, np.zeros(ops.adamw_blocks(c), np.float32)) for c in counts],
                           "second_scales": [ops.DeviceArray.of(dev, np.zeros(ops.adamw_blocks(c), np.float32)) for c in counts]}
            for a in self.states["first"] + self.states["second"]:
                a.clear()
        else:
            self.states = {k: [ops.DeviceArray.of(dev, np.zeros(c, np.float32)) for c in counts] for k in ("first", "second")}

    def forward(self):
        """Queues the layer up to the loss and the gradients of o and Wo."""
        h = self.heads
        self.project.enqueue()
        ops.rotary(self.dev, h["q"], h["q"], self.cos, self.sin, self.positions, second=h["k"], second_out=h["k"])
        ops.attention(self.dev, h["q"], h["k"], h["v"], h["o"], self.lse, workspace=self.room, **self.masks)
        self.close.enqueue()

    def step(self):
        """Queues one training step."""
        h, a = self.heads, self.arrays
        self.forward()
        ops.attention_backward(self.dev, h["q"], h["k"], h["v"], h["o"], self.lse, h["do"], h["dq"], h["dk"], h["dv"], workspace=self.room,
                               **self.masks)
        ops.rotary(self.dev, h["dq"], h["dq"], self.cos, self.sin, self.positions, second=h["dk"], second_out=h["dk"], inverse=True)
        self.weigh.enqueue()
        self.steps += 1
        ops.adamw(self.dev, [a[n] for n in self.names], [a["d" + n] for n in self.names], step=self.steps, rate=self.rate, decay=self.decay,
                  **self.states)

    def loss(self) -> float:
        """The loss of the last step's forward pass (waits)."""
        return float(self.arrays["loss"].numpy().reshape(-1)[0])

    def weight(self, name: str) -> np.ndarray:
        return self.arrays[name].numpy()


def main():
    from . import HipDevice
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 512, 256)).astype(np.float32)
    target = np.cumsum(x, 1) / np.arange(1, 513, dtype=np.float32)[None, :, None]  # the mean of what each position sees
    layer = DecoderAttention(HipDevice(0), x, target, heads=8, key_heads=2, size=64, rate=3e-3, cap=30.0)
    for i in range(101):
        layer.step()
        if i % 20 == 0:
            print(f"step {i}: loss {layer.loss():.5f}")


if __name__ == "__main__":
    main()

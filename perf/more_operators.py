"""The operators that surround a decoder's mixing of positions while it trains: layer norm with its residual and the sums of its
weights' gradients, a gated linear recurrence (a mixer whose state does not grow with the context; forward, backward, single
tokens), and the norm over all gradients with clipping.

`run` computes them from elementary torch operations in 32 bits where `own` is false, and with the framework's kernels
(`adhip.operators`) where it is true; `exact` restates each definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
WIDE = {"f32": 4, "bf16": 2}
GPU = "cuda"
BLOCK = 256  # positions between the states that a recurrence keeps for its backward pass

# the benchmark's perceptron (4096-4096-4096-1024), its encoder layer with a table whose rows fit no block, the README's perceptron
PERCEPTRON = "4096x4096,4096,4096x4096,4096,4096x1024,1024"
ENCODER = ",".join(["1024x1024"] * 4 + ["1024x4096", "4096", "4096x1024", "1024", "1024", "1024", "5003x1023"])
README = "3x4,4,4x2,2"


def listed():
    return [
        # one new token of each of four sequences, the benchmark's encoder width: latency alone
        norm_case("norm token", "f32", "f32", "forward", 4, 1024),
        # a norm of each head's queries, as it stands before attention: many short rows, no mean
        norm_case("norm heads", "bf16", "f32", "train", 2 * 4096 * 16, 128, centered=False),
        # odd rows and sizes in the framework's own type, with the residual added on the way
        norm_case("norm odd", "f32", "f32", "train", 3001, 1023, added=True),
        # the ordinary norm of a training batch with its residual, parameters in bf16 as everything else
        norm_case("norm training", "bf16", "bf16", "train", 2 * 8192, 4096, added=True),
        # one new token of each of eight sequences: latency alone
        recurrence_case("recurrence token", "bf16", "forward", 8, 1, 1024, initial=True),
        # prompts of different lengths read into states, with factors that the program has computed by a rule of its own
        recurrence_case("recurrence prompts", "bf16", "forward", 4, 2049, 2560, factors=True, ragged=True, initial=True),
        # documents packed into one row, odd sizes, the framework's own type
        recurrence_case("recurrence documents", "f32", "train", 1, 8191, 1000, document=1200),
        # the ordinary training step of long sequences
        recurrence_case("recurrence training", "bf16", "train", 2, 8192, 4096),
        # the README's two-layer perceptron: four small tensors
        clip_case("clip small", "f32", README),
        # the benchmark's perceptron: gradients in bf16, matrices and their small companions
        clip_case("clip encoder", "bf16", ENCODER),
        clip_case("clip perceptron", "f32", PERCEPTRON),
        # the norm, and AdamW that takes the factor from where the norm left it
        clip_case("clip step", "f32", ENCODER, step=True),
    ]


def norm_case(name, dtype, weights, direction, rows, size, added=False, centered=True):
    return {"name": name, "op": "norm", "dtype": dtype, "weights": weights, "direction": direction, "rows": rows, "size": size,
            "added": added, "centered": centered}


def recurrence_case(name, dtype, direction, batch, length, channels, factors=False, ragged=False, document=0, initial=False):
    return {"name": name, "op": "recurrence", "dtype": dtype, "direction": direction, "batch": batch, "length": length,
            "channels": channels, "factors": factors, "ragged": ragged, "document": document, "initial": initial}


def clip_case(name, dtype, shapes, step=False):
    return {"name": name, "op": "clip", "dtype": dtype, "shapes": shapes, "step": step}


def draw(rng):
    def size(lo, hi):
        """Between lo and hi, evenly over the logarithm; one in three rounded to a multiple of 16, the rest as they fall."""
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(16, n // 16 * 16) if n >= 16 and rng.random() < 0.34 else n

    op = rng.choice(["norm", "norm", "recurrence", "recurrence", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "norm":
        width = size(16, 16384)
        rows = size(1, max(2, min(131072, 2 * 8192 * 4096 // (width * (2 if dtype == "f32" else 1)))))
        c = norm_case("", dtype, rng.choice(["f32", dtype]), rng.choice(["forward", "train", "train"]), rows, width,
                      rng.random() < 0.5, rng.random() < 0.7)
    elif op == "recurrence":
        kind = rng.choice(["token", "forward", "train", "train"])
        channels = size(16, 8192)
        most = 2 * 8192 * 4096 // (channels * (2 if dtype == "f32" else 1))
        length = 1 if kind == "token" else size(2, max(2, min(32768, most)))
        batch = size(1, 256) if kind == "token" else size(1, max(1, min(16, most // length)))
        c = recurrence_case("", dtype, "train" if kind == "train" else "forward", batch, length, channels, rng.random() < 0.3,
                            kind != "token" and rng.random() < 0.25, rng.choice([0, 0, size(16, 4096)]) if length > 1 else 0,
                            kind == "token" or rng.random() < 0.3)
    else:
        step = rng.random() < 0.3
        shapes, total, most = [], 0, 17_000_000 if step else 37_000_000
        for _ in range(rng.randint(1, 40)):
            shape = [size(2, 4096)] + ([size(2, 4096)] if rng.random() < 0.6 else [])
            if total + math.prod(shape) <= most:
                shapes.append("x".join(map(str, shape)))
                total += math.prod(shape)
        c = clip_case("", dtype, ",".join(shapes) or "7", step)
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=GPU).manual_seed(seed)
    return {"norm": prepare_norm, "recurrence": prepare_recurrence, "clip": prepare_clip}[case["op"]](case, g)


def normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=GPU) * scale).to(dtype)


def prepare_norm(c, g):
    t, n, d = TYPES[c["dtype"]], c["rows"], c["size"]
    s = {"case": c, "room": None}
    # a stream of activations: no zero mean, some features far larger than the others
    wide = torch.exp(normal(g, (d,), scale=0.7))
    s["x"] = (torch.randn((n, d), generator=g, device=GPU) * wide + normal(g, (d,), scale=0.5)).to(t)
    s["added"] = normal(g, (n, d), t) if c["added"] else None
    s["weight"] = (1.0 + normal(g, (d,), scale=0.2)).to(TYPES[c["weights"]])
    s["bias"] = normal(g, (d,), TYPES[c["weights"]], 0.1) if c["centered"] else None
    s["out"], s["stats"] = torch.empty_like(s["x"]), torch.empty((n, 2), device=GPU)
    s["total"] = torch.empty_like(s["x"]) if c["added"] else None
    if c["direction"] == "train":
        s["out_grad"] = normal(g, (n, d), t)
        s["total_grad"] = normal(g, (n, d), t) if c["added"] else None
        s["x_grad"], s["weight_grad"] = torch.empty_like(s["x"]), torch.empty_like(s["weight"])
        s["bias_grad"] = torch.empty_like(s["bias"]) if c["centered"] else None
    return s


def prepare_recurrence(c, g):
    t, b, n, d = TYPES[c["dtype"]], c["batch"], c["length"], c["channels"]
    s = {"case": c, "room": None, "x": normal(g, (b, n, d), t)}
    # gates that remember from a few to some hundred positions; factors of the same
    gates = torch.randn((b, n, d), generator=g, device=GPU) + (torch.rand((d,), generator=g, device=GPU) * 5.0)
    s["gates"] = (torch.sigmoid(gates) if c["factors"] else gates).to(t)
    s["initial"] = normal(g, (b, d)) if c["initial"] else None
    s["lengths"] = torch.randint(n // 2, n + 1, (b,), generator=g, device=GPU, dtype=torch.int32) if c["ragged"] else None
    s["documents"] = None
    if c["document"]:
        # ends of documents fall anywhere, one for every `document` positions; the last positions belong to none
        ends = torch.rand((b, n), generator=g, device=GPU) < 1.0 / c["document"]
        s["documents"] = torch.cumsum(ends, 1).to(torch.int32).contiguous()
        s["documents"][:, n - n // 32:] = -1
    s["out"], s["final"] = torch.empty_like(s["x"]), torch.empty((b, d), device=GPU)
    if c["direction"] == "train":
        s["out_grad"] = normal(g, (b, n, d), t)
        s["states"] = torch.empty((b, -(-n // BLOCK), d), device=GPU)
        s["x_grad"], s["gates_grad"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["initial_grad"] = torch.empty((b, d), device=GPU) if c["initial"] else None
    return s


LIMIT = 1.0
STEP = {"step": 100, "rate": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "decay": 0.1}


def prepare_clip(c, g):
    t, shapes = TYPES[c["dtype"]], [[int(n) for n in x.split("x")] for x in c["shapes"].split(",")]
    s = {"case": c, "room": None, "norm": torch.empty(1, device=GPU), "factor": torch.empty(1, device=GPU)}
    # norms from below the limit to well above it
    count = sum(math.prod(x) for x in shapes)
    size = torch.exp(torch.rand((), generator=g, device=GPU) * 3.0 - 1.0) * (LIMIT / math.sqrt(count))
    s["g"] = [(torch.randn(x, generator=g, device=GPU) * size).to(t) for x in shapes]
    if c["step"]:
        s["p"] = [normal(g, x, t, 0.02) for x in shapes]
        s["m"], s["v"] = [normal(g, x, scale=2e-4) for x in shapes], [normal(g, x, scale=5e-4).square() for x in shapes]
        for name in "pmv":
            s[name + "_out"] = [torch.empty_like(x) for x in s[name]]
    else:
        s["g_out"] = [torch.empty_like(x) for x in s["g"]]
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": own_norm, "recurrence": own_recurrence, "clip": own_clip}[op](state)
    return {"norm": plain_norm, "recurrence": plain_recurrence, "clip": plain_clip}[op](state)


EPS = 1e-5


def plain_norm(s):
    c, t = s["case"], s["x"].dtype
    answer, x = {}, s["x"]
    if c["added"]:
        # the sum is rounded where it is kept: it is the stream that the next layer and the backward pass read
        x = answer["total"] = (x.float() + s["added"].float()).to(t)
    x, w = x.float(), s["weight"].float()
    mean = x.mean(1, keepdim=True) if c["centered"] else x.new_zeros((len(x), 1))
    x = x - mean
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    x = x * r
    y = x * w
    answer |= {"out": (y + s["bias"].float() if c["centered"] else y).to(t), "stats": torch.cat((mean, r), 1)}
    if c["direction"] == "train":
        dy = s["out_grad"].float()
        u = dy * w
        dx = u - x * (u * x).mean(1, keepdim=True)
        if c["centered"]:
            dx = dx - u.mean(1, keepdim=True)
            answer["bias_grad"] = dy.sum(0).to(s["bias"].dtype)
        dx = dx * r
        if c["added"]:
            dx = dx + s["total_grad"].float()
        answer |= {"x_grad": dx.to(t), "weight_grad": (dy * x).sum(0).to(w.dtype if c["weights"] == "f32" else t)}
    return answer


def marks(s):
    """Which positions count, [batch, length, 1], and at which of them the state goes on; None where all do."""
    c = s["case"]
    live = goes_on = None
    if s["documents"] is not None:
        d = s["documents"]
        live = d >= 0
        goes_on = live.clone()
        goes_on[:, 1:] &= d[:, 1:] == d[:, :-1]
    if s["lengths"] is not None:
        within = torch.arange(c["length"], device=GPU)[None] < s["lengths"][:, None]
        live = within if live is None else live & within
        goes_on = torch.ones_like(within) if goes_on is None else goes_on | ~within
    return (None, None) if live is None else (live[..., None], goes_on[..., None])


def scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dim 1, from nothing, by doubling: products of the factors and sums over 1, 2, 4, ... positions."""
    n, step = a.shape[1], 1
    while step < n:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), 1)
        a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def plain_recurrence(s):
    c, t = s["case"], s["x"].dtype
    x, gate = s["x"].float(), s["gates"].float()
    if c["factors"]:
        a, b = gate, x
    else:
        a, rest = torch.sigmoid(gate), torch.sigmoid(-gate)
        b = rest * x
    live, goes_on = marks(s)
    m = a
    if live is not None:
        zero = torch.zeros_like(a)
        # behind the lengths the state goes on as it is; where a document begins, it goes on from nothing
        b = torch.where(live, b, zero)
        m = torch.where(goes_on, torch.where(live, a, zero + 1.0), zero)
    first = b[:, :1] if s["initial"] is None else b[:, :1] + m[:, :1] * s["initial"][:, None]
    h = scan(m, torch.cat((first, b[:, 1:]), 1))
    answer = {"out": (h if live is None else torch.where(live, h, torch.zeros_like(h))).to(t), "final": h[:, -1].contiguous()}
    if c["direction"] == "train":
        start = torch.zeros_like(h[:, :1]) if s["initial"] is None else s["initial"][:, None]
        before = torch.cat((start, h[:, :-1]), 1)
        answer["states"] = before[:, ::BLOCK].contiguous()
        dout = s["out_grad"].float()
        if live is not None:
            dout = torch.where(live, dout, torch.zeros_like(dout))
        later = torch.cat((m[:, 1:], torch.zeros_like(m[:, :1])), 1)
        l = scan(later.flip(1), dout.flip(1)).flip(1)
        if s["initial"] is not None:
            answer["initial_grad"] = (l * m)[:, 0].contiguous()
        if goes_on is not None:
            before = torch.where(goes_on, before, torch.zeros_like(before))
            l = torch.where(live, l, torch.zeros_like(l))
        if c["factors"]:
            answer |= {"x_grad": l.to(t), "gates_grad": (l * before).to(t)}
        else:
            answer |= {"x_grad": (l * rest).to(t), "gates_grad": (l * (before - x) * (a * rest)).to(t)}
    return answer


def plain_clip(s):
    c = s["case"]
    g = [x.float() for x in s["g"]]
    # (squares of small gradients and long sums: in 64 bits)
    norm = torch.stack([(x.double() * x).sum() for x in g]).sum().sqrt()
    factor = torch.where(norm <= LIMIT, torch.ones_like(norm), LIMIT / norm).float().reshape(1)
    answer = {"norm": norm.float().reshape(1), "factor": factor}
    g = [x * factor for x in g]
    if not c["step"]:
        return answer | {"g": [x.to(y.dtype) for x, y in zip(g, s["g"])]}
    b1, b2, step, rate = STEP["beta1"], STEP["beta2"], STEP["step"], STEP["rate"]
    answer |= {"p": [], "m": [], "v": []}
    for p, x, m, v in zip(s["p"], g, s["m"], s["v"]):
        m = m * b1 + x * (1.0 - b1)
        v = v * b2 + x * x * (1.0 - b2)
        under = v.sqrt() * (1.0 / math.sqrt(1.0 - b2 ** step)) + STEP["eps"]
        new = p.float() * (1.0 - rate * STEP["decay"]) - m / under * (rate / (1.0 - b1 ** step))
        for name, value in (("p", new.to(p.dtype)), ("m", m), ("v", v)):
            answer[name].append(value)
    return answer


# ---- the framework's operators --------------------------------------------------------------------------------

_device = None


def framework():
    """The operators and the device handle that a program keeps for its whole life."""
    global _device
    if _device is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "autodiff-ir-rust_amd"))
        from adhip import HipDevice, operators
        _device = (operators, HipDevice(0))
    return _device


def workspace(s, need):
    """A program keeps its workspaces for as long as its arrays."""
    if s["room"] is None:
        s["room"] = torch.empty(max(1, need()), dtype=torch.uint8, device=GPU)
    return s["room"]


def own_norm(s):
    ops, dev = framework()
    train, stream = s["case"]["direction"] == "train", torch.cuda.current_stream().cuda_stream
    ops.layer_norm(dev, s["x"], s["out"], weight=s["weight"], bias=s["bias"], eps=EPS, centered=s["case"]["centered"], added=s["added"],
                   total=s["total"], stats=s["stats"], stream=stream)
    answer = {n: s[n] for n in ("total", "out", "stats") if s[n] is not None}
    if not train:
        return answer
    x = s["x"] if s["total"] is None else s["total"]
    room = workspace(s, lambda: ops.layer_norm_workspace(dev, x))
    ops.layer_norm_backward(dev, x, s["stats"], s["out_grad"], s["x_grad"], weight=s["weight"], weight_grad=s["weight_grad"],
                            bias_grad=s["bias_grad"], centered=s["case"]["centered"], total_grad=s["total_grad"], workspace=room, stream=stream)
    return answer | {n: s[n] for n in ("x_grad", "weight_grad", "bias_grad") if s[n] is not None}


def own_recurrence(s):
    ops, dev = framework()
    train, stream = s["case"]["direction"] == "train", torch.cuda.current_stream().cuda_stream
    room = workspace(s, lambda: ops.recurrence_workspace(dev, s["x"], backward=train))
    how = dict(factors=s["case"]["factors"], lengths=s["lengths"], documents=s["documents"], workspace=room, stream=stream)
    ops.recurrence(dev, s["x"], s["gates"], s["out"], initial=s["initial"], final=s["final"], states=s["states"] if train else None, **how)
    answer = {"out": s["out"], "final": s["final"]}
    if not train:
        return answer
    ops.recurrence_backward(dev, s["x"], s["gates"], s["states"], s["out_grad"], s["x_grad"], s["gates_grad"],
                            initial_grad=s["initial_grad"], **how)
    return answer | {n: s[n] for n in ("states", "x_grad", "gates_grad", "initial_grad") if s[n] is not None}


def own_clip(s):
    ops, dev = framework()
    stream = torch.cuda.current_stream().cuda_stream
    room = workspace(s, lambda: ops.gradient_norm_workspace(dev, s["g"]))
    how = dict(limit=LIMIT, factor=s["factor"], workspace=room, stream=stream)
    answer = {"norm": s["norm"], "factor": s["factor"]}
    if not s["case"]["step"]:
        ops.clip_gradients(dev, s["g"], s["norm"], gradients_out=s["g_out"], **how)
        return answer | {"g": s["g_out"]}
    ops.gradient_norm(dev, s["g"], s["norm"], **how)
    ops.adamw(dev, s["p"], s["g"], s["m"], s["v"], factor=s["factor"], parameters_out=s["p_out"], first_out=s["m_out"], second_out=s["v_out"],
              stream=stream, **STEP)
    return answer | {n: s[n + "_out"] for n in "pmv"}


# ---- work ---------------------------------------------------------------------------------------------------------


def work(case):
    c, w = case, WIDE[case["dtype"]]
    if c["op"] == "norm":
        n = c["rows"] * c["size"]
        passes, flops = (4 if c["added"] else 2), 8
        if c["direction"] == "train":
            passes, flops = passes + (4 if c["added"] else 3), 24
        small = c["size"] * WIDE[c["weights"]] * (2 if c["centered"] else 1) * (2 if c["direction"] == "train" else 1)
        return {"bytes": passes * n * w + 8 * c["rows"] + small, "flops": flops * n}
    if c["op"] == "recurrence":
        n, ends = c["batch"] * c["length"] * c["channels"], c["batch"] * c["channels"]
        live = int(n * (0.75 if c["ragged"] else 1.0))  # inputs behind the lengths need not be read, outputs are written
        bytes_ = 2 * live * w + n * w + 4 * ends * (2 if c["initial"] else 1) + (4 * c["batch"] * c["length"] if c["document"] else 0)
        flops = 4 * live
        if c["direction"] == "train":
            bytes_ += 3 * live * w + 2 * n * w + 4 * ends * -(-c["length"] // BLOCK) + (4 * ends if c["initial"] else 0)
            flops += 8 * live
        return {"bytes": bytes_, "flops": flops}
    n = sum(math.prod(int(k) for k in x.split("x")) for x in c["shapes"].split(","))
    # the gradients once (a card's last cache may hold them for the second look), what is made of them once
    return {"bytes": n * ((3 * w + 16) if c["step"] else 2 * w) + 8, "flops": (17 if c["step"] else 3) * n}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": exact_norm, "recurrence": exact_recurrence, "clip": exact_clip}[case["op"]](case, s)


def exact_norm(c, s):
    r, x = {}, s["x"].double()
    if c["added"]:
        r["total"] = x + s["added"].double()
        x = r["total"].float().to(s["x"].dtype).double()  # the sum as it is kept
    d = c["size"]
    mean = torch.sum(x, -1) / d if c["centered"] else torch.zeros(c["rows"], dtype=torch.float64, device=GPU)
    spread = torch.sum((x - mean.unsqueeze(-1)) ** 2, -1) / d
    root = (spread + EPS) ** -0.5
    unit = (x - mean.unsqueeze(-1)) * root.unsqueeze(-1)
    out = unit * s["weight"].double()
    if c["centered"]:
        out += s["bias"].double()
    r["out"], r["stats"] = out, torch.stack((mean, root), -1)
    if c["direction"] == "train":
        dy = s["out_grad"].double()
        if c["centered"]:
            r["bias_grad"] = torch.sum(dy, 0)
        # through y = unit w, unit = (x - mean) root, root = (spread + eps)^-1/2
        d_unit = dy * s["weight"].double()
        d_spread = torch.sum(d_unit * unit, -1) / root * (-0.5 * root ** 3)
        dx = d_unit * root.unsqueeze(-1) + (2.0 / d) * d_spread.unsqueeze(-1) * (x - mean.unsqueeze(-1))
        if c["centered"]:
            dx -= torch.sum(dx, -1, keepdim=True) / d
        if c["added"]:
            dx += s["total_grad"].double()
        r["x_grad"] = dx
        r["weight_grad"] = torch.sum(dy * unit, 0)
    return {n: r[n] for n in ("total", "out", "stats", "bias_grad", "x_grad", "weight_grad") if n in r}


def exact_recurrence(c, s):
    """Position by position."""
    b, n, d = c["batch"], c["length"], c["channels"]
    like = dict(dtype=torch.float64, device=GPU)
    train = c["direction"] == "train"
    h = torch.zeros((b, d), **like) if s["initial"] is None else s["initial"].double()
    out = torch.empty((b, n, d), **like)
    before = torch.empty_like(out) if train else None
    at = torch.arange(n, device=GPU)
    counts = torch.ones((b, n), dtype=torch.bool, device=GPU)
    if s["lengths"] is not None:
        counts = at < s["lengths"].unsqueeze(1)
    begins = torch.zeros((b, n), dtype=torch.bool, device=GPU)
    none = torch.zeros_like(begins)
    if s["documents"] is not None:
        none = (s["documents"] < 0) & counts
        begins[:, 1:] = s["documents"][:, 1:] != s["documents"][:, :-1]
    a_of = (lambda t: s["gates"][:, t].double()) if c["factors"] else (lambda t: torch.sigmoid(s["gates"][:, t].double()))
    for t in range(n):
        if train:
            before[:, t] = h
        a, x = a_of(t), s["x"][:, t].double()
        if not c["factors"]:
            x = x / (1.0 + torch.exp(s["gates"][:, t].double()))
        fresh = torch.where(begins[:, t, None], torch.zeros_like(h), h)
        new = torch.where(none[:, t, None], torch.zeros_like(h), torch.addcmul(x, a, fresh))
        h = torch.where(counts[:, t, None], new, h)
        out[:, t] = torch.where(counts[:, t, None], h, torch.zeros_like(h))
    r = {"out": out, "final": h}
    if train:
        r["states"] = before[:, ::BLOCK].clone()
        r["x_grad"], r["gates_grad"] = torch.zeros_like(out), torch.zeros_like(out)
        back = torch.zeros((b, d), **like)
        for t in range(n - 1, -1, -1):
            used = (counts[:, t] & ~none[:, t])[:, None]
            l = torch.where(used, back + s["out_grad"][:, t].double(), back)
            a = a_of(t)
            carried = used & ~begins[:, t, None]
            da = torch.where(carried, l * before[:, t], torch.zeros_like(l))
            if c["factors"]:
                dx, dg = l, da
            else:
                rest = 1.0 / (1.0 + torch.exp(s["gates"][:, t].double()))
                dx, dg = l * rest, (da - l * s["x"][:, t].double()) * a * rest
            r["x_grad"][:, t] = torch.where(used, dx, torch.zeros_like(dx))
            r["gates_grad"][:, t] = torch.where(used, dg, torch.zeros_like(dg))
            back = torch.where(carried, l * a, torch.where(counts[:, t, None], torch.zeros_like(l), l))
        if c["initial"]:
            r["initial_grad"] = back
    return {k: r[k] for k in ("out", "final", "states", "initial_grad", "x_grad", "gates_grad") if k in r}


def exact_clip(c, s):
    squares = 0.0
    for x in s["g"]:
        squares = squares + torch.linalg.vector_norm(x.double()) ** 2
    norm = squares ** 0.5
    factor = torch.clamp(LIMIT / norm, max=1.0)
    r = {"norm": norm.reshape(1), "factor": factor.reshape(1)}
    if not c["step"]:
        return r | {"g": [x.double() * factor for x in s["g"]]}
    r |= {"p": [], "m": [], "v": []}
    b1, b2, t = STEP["beta1"], STEP["beta2"], STEP["step"]
    for p, x, m, v in zip(s["p"], s["g"], s["m"], s["v"]):
        x = x.double() * factor
        m, v = b1 * m.double() + (1 - b1) * x, b2 * v.double() + (1 - b2) * x ** 2
        ahead = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + STEP["eps"])
        r["p"].append((1 - STEP["rate"] * STEP["decay"]) * p.double() - STEP["rate"] * ahead)
        r["m"].append(m)
        r["v"].append(v)
    return r

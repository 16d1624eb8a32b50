"""The operators that training and running a decoder takes beside this framework's programs: rotary positions, attention
with capped scores, distance bias, masks and shared heads (forward, backward, single tokens against a cache), and AdamW
over many tensors with states in 32 or 8 bits.

`run` computes them from elementary torch operations in 32 bits where `own` is false, and with the framework's kernels
(`adhip.operators`) where it is true; `exact` restates each definition in 64 bits.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GPU = "cuda"
BLOCK = 256  # elements that share a scale where AdamW's states are held in 8 bits


def listed():
    return [
        # one token of one sequence against a short cache: latency alone
        attention_case("attention token small", "f32", "forward", 1, 1, 129, 4, 4, 64, causal=True),
        # a batch of sequences of different lengths that each take one token, a long cache, four query heads a key head
        attention_case("attention token long", "bf16", "forward", 8, 1, 16384, 32, 8, 128, causal=True, ragged=True),
        # a prompt of odd length into wide heads, with capped scores and a sliding window
        attention_case("attention window", "bf16", "forward", 1, 3001, 3001, 8, 4, 256, causal=True, window=1024, cap=30.0),
        # the benchmark's encoder layer (2048 positions, eight heads of 128) in the framework's own type, trained with a
        # prefix that all positions see and scores that fall with distance
        attention_case("attention prefix f32", "f32", "train", 1, 2048, 2048, 8, 8, 128, causal=True, prefix=True, slopes=True),
        # documents of uneven lengths packed into one row, with padding at its end
        attention_case("attention documents", "bf16", "train", 1, 8191, 8191, 8, 8, 64, causal=True, document=1200),
        # the ordinary training step of a decoder: causal, shared heads, capped scores
        attention_case("attention training", "bf16", "train", 2, 4096, 4096, 16, 4, 128, causal=True, cap=50.0),
        # queries and keys of one new token for each of four sequences: latency alone
        rotary_case("rotary token", "f32", "forward", 4, 1, 8, 8, 64, 64, False),
        # the gradient of interleaved pairs over half of each head, sizes between the tiles
        rotary_case("rotary partial", "f32", "gradient", 3, 1001, 8, 8, 80, 40, True),
        # a training batch of long sequences, shared key heads, frequencies scaled for the length
        rotary_case("rotary long", "bf16", "forward", 2, 8192, 32, 8, 128, 128, False),
        # the README's two-layer perceptron: four small tensors
        adamw_case("adamw small", "f32", "f32", 32, "3x4,4,4x2,2"),
        # the benchmark's perceptron, 4096-4096-4096-1024
        adamw_case("adamw large", "f32", "f32", 32, "4096x4096,4096,4096x4096,4096,4096x1024,1024"),
        # the benchmark's encoder layer in bf16 with states in 8 bits, and a table whose rows fit no block
        adamw_case("adamw 8 bits", "bf16", "bf16", 8,
                   ",".join(["1024x1024"] * 4 + ["1024x4096", "4096", "4096x1024", "1024", "1024", "1024", "5003x1023"])),
    ]


def attention_case(name, dtype, direction, batch, queries, keys, heads, shared, size, causal=False, window=0, cap=0.0,
                   prefix=False, slopes=False, document=0, ragged=False):
    return {"name": name, "op": "attention", "dtype": dtype, "direction": direction, "batch": batch, "queries": queries,
            "keys": keys, "heads": heads, "key_heads": shared, "size": size, "causal": causal, "window": window, "cap": cap,
            "prefix": prefix, "slopes": slopes, "document": document, "ragged": ragged}


def rotary_case(name, dtype, direction, batch, length, heads, shared, size, rotated, interleaved):
    return {"name": name, "op": "rotary", "dtype": dtype, "direction": direction, "batch": batch, "length": length,
            "heads": heads, "key_heads": shared, "size": size, "rotated": rotated, "interleaved": interleaved}


def adamw_case(name, dtype, grad, bits, shapes):
    return {"name": name, "op": "adamw", "dtype": dtype, "grad": grad, "bits": bits, "shapes": shapes}


def draw(rng):
    def size(lo, hi):
        """Between lo and hi, evenly over the logarithm; one in three rounded to a multiple of 16, the rest as they fall."""
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        n = max(16, n // 16 * 16) if n >= 16 and rng.random() < 0.34 else n
        return n + 1 if n == 3072 else n  # no configuration here has that size

    op = rng.choice(["attention", "attention", "attention", "rotary", "adamw"])
    if op == "attention":
        dtype = rng.choice(["f32", "bf16", "bf16"])
        width = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 192, 256])
        shared = rng.choice([1, 2, 4, 8])
        heads = shared * rng.choice([1, 1, 2, 3, 4])
        kind = rng.choice(["token", "forward", "train"])
        window = rng.choice([0, 0, size(16, 1024)])
        cap = rng.choice([0.0, 0.0, 30.0, 50.0])
        causal = rng.random() < 0.75
        prefix = rng.random() < 0.25
        slopes = rng.random() < 0.25
        if kind == "token":
            c = attention_case("", dtype, "forward", size(1, 16), rng.choice([1, 1, 1, 2, 5]), size(64, 16384), heads, shared, width,
                               causal, window, cap, prefix, slopes, 0, True)
        else:
            most = 8192 if dtype == "bf16" else 2048
            n = size(48, most)
            # no more scores than the largest listed case has
            room = 2 * 16 * 4096 * 4096 if dtype == "bf16" else 8 * 2048 * 2048
            batch = rng.randint(1, max(1, min(4, room // (n * n * heads))))
            while n * n * heads * batch * width > room * 128:
                n = n * 2 // 3
            c = attention_case("", dtype, kind, batch, n, n, heads, shared, width, causal, window, cap, prefix, slopes,
                               rng.choice([0, 0, size(32, 2048)]), rng.random() < 0.2)
    elif op == "rotary":
        width = rng.choice([32, 64, 72, 80, 96, 128, 192, 256])
        shared = rng.choice([1, 2, 4, 8])
        heads = shared * rng.choice([1, 2, 3, 4])
        length = size(1, 8192)
        batch = rng.randint(1, 8)
        while batch > 1 and batch * length * (heads + shared) * width > 2 * 8192 * 40 * 128:
            batch -= 1
        while length * (heads + shared) * width > 2 * 8192 * 40 * 128:
            length //= 2
        rotated = width if rng.random() < 0.6 else 2 * rng.randint(4, width // 2)
        c = rotary_case("", rng.choice(["f32", "bf16"]), rng.choice(["forward", "gradient"]), batch, length, heads, shared, width,
                        rotated, rng.random() < 0.5)
    else:
        shapes, total = [], 0
        bits = rng.choice([32, 8])
        for _ in range(rng.randint(2, 20 if bits == 32 else 12)):
            shape = [size(2, 4096)] + ([size(2, 4096)] if rng.random() < 0.6 else [])
            if total + math.prod(shape) <= 37_000_000:
                shapes.append("x".join(map(str, shape)))
                total += math.prod(shape)
        c = adamw_case("", rng.choice(["f32", "bf16"]), rng.choice(["f32", "bf16"]), bits, ",".join(shapes))
    del c["name"]
    return c


# ---- inputs -------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=GPU).manual_seed(seed)
    return {"attention": prepare_attention, "rotary": prepare_rotary, "adamw": prepare_adamw}[case["op"]](case, g)


def normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=GPU) * scale).to(dtype)


def integers(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=g, device=GPU, dtype=torch.int32)


def prepare_attention(c, g):
    t, b, lq, lk, h, hk, d = TYPES[c["dtype"]], c["batch"], c["queries"], c["keys"], c["heads"], c["key_heads"], c["size"]
    s = {"case": c}
    # capped scores are met where they grow large
    s["q"] = normal(g, (b, lq, h, d), t, 4.0 if c["cap"] else 1.0)
    s["k"], s["v"] = normal(g, (b, lk, hk, d), t), normal(g, (b, lk, hk, d), t)
    s["lengths"] = integers(g, max(0, lk // 2), lk + 1, (b,)) if c["ragged"] else None
    s["prefix"] = integers(g, 0, lk // 2 + 1, (b,)) if c["prefix"] else None
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device=GPU) if c["slopes"] else None
    s["documents"] = None
    if c["document"]:
        # ends of documents fall anywhere, one for every `document` positions; the last positions belong to none
        ends = torch.rand((b, lk), generator=g, device=GPU) < 1.0 / c["document"]
        s["documents"] = torch.cumsum(ends, 1).to(torch.int32).contiguous()
        s["documents"][:, lk - lk // 32:] = -1
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((b, lq, h), device=GPU)
    if c["direction"] == "train":
        s["dout"] = normal(g, (b, lq, h, d), t)
        s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[x]) for x in "qkv")
    return s


def prepare_rotary(c, g):
    t, b, n, r = TYPES[c["dtype"]], c["batch"], c["length"], c["rotated"]
    rows = 2 * n + 64  # the table serves positions beyond this call's
    turns = torch.arange(rows, dtype=torch.float64)[:, None] / 4.0 * 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    s = {"case": c, "cos": turns.cos().float().to(GPU), "sin": turns.sin().float().to(GPU)}
    s["positions"] = (torch.arange(n, device=GPU, dtype=torch.int32) + integers(g, 0, n + 64, (b, 1))).contiguous()
    s["q"], s["k"] = normal(g, (b, n, c["heads"], c["size"]), t), normal(g, (b, n, c["key_heads"], c["size"]), t)
    s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    return s


STEP = {"step": 100, "rate": 3e-4, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "decay": 0.1, "grad_scale": 0.5}


def prepare_adamw(c, g):
    s = {"case": c, "p": [], "g": [], "m": [], "v": [], "m_scale": [], "v_scale": []}
    for shape in ([int(n) for n in x.split("x")] for x in c["shapes"].split(",")):
        s["p"].append(normal(g, shape, TYPES[c["dtype"]], 0.02))
        s["g"].append(normal(g, shape, TYPES[c["grad"]], 0.01))
        m, v = normal(g, shape, scale=2e-3), normal(g, shape, scale=5e-3).square()
        if c["bits"] == 8:
            (m, ms), (v, vs) = to_blocks(m), to_blocks(v.sqrt())
            s["m_scale"].append(ms)
            s["v_scale"].append(vs)
        s["m"].append(m)
        s["v"].append(v)
    for name in ("p", "m", "v", "m_scale", "v_scale"):
        s[name + "_out"] = [torch.empty_like(x) for x in s[name]]
    return s


# ---- the plain forms ----------------------------------------------------------------------------------------


def run(state):
    c = state["case"]
    if c["op"] == "attention":
        return own_attention(state) if own else plain_attention(state)
    if c["op"] == "rotary":
        return own_rotary(state) if own else plain_rotary(state)
    return own_adamw(state) if own else plain_adamw(state)


def visible(s):
    """Which keys a query sees, [batch, 1, 1, queries, keys], and how far each is."""
    c, lq, lk = s["case"], s["case"]["queries"], s["case"]["keys"]
    n = torch.full((c["batch"],), lk, device=GPU) if s["lengths"] is None else s["lengths"].long()
    at = torch.arange(lq, device=GPU)[None, :, None] + (n - lq)[:, None, None]
    j = torch.arange(lk, device=GPU)[None, None, :]
    far = at - j
    sees = far >= 0 if c["causal"] else torch.ones_like(far, dtype=torch.bool)
    if c["window"]:
        sees = sees & (far.abs() < c["window"])
    if s["prefix"] is not None:
        sees = sees | (j < s["prefix"][:, None, None])
    sees = sees & (j < n[:, None, None])
    if s["documents"] is not None:
        mine, theirs = s["documents"][:, lk - lq:, None], s["documents"][:, None, :]
        sees = sees & (mine == theirs) & (mine >= 0)
    return sees[:, None, None], far.abs()[:, None, None]


def by_key_head(x, c):
    """[batch, length, heads, size] in 32 bits as [batch, key heads, heads of one key head * length, size]."""
    b, n, h, d = x.shape
    return x.float().reshape(b, n, c["key_heads"], h // c["key_heads"], d).permute(0, 2, 3, 1, 4).reshape(b, c["key_heads"], -1, d)


def from_key_head(x, like):
    b, n, h, d = like.shape
    return x.reshape(b, x.shape[1], h // x.shape[1], n, d).permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(like.dtype)


def plain_attention(s):
    c = s["case"]
    b, lq, lk, hk, group, d = c["batch"], c["queries"], c["keys"], c["key_heads"], c["heads"] // c["key_heads"], c["size"]
    scale = 1.0 / math.sqrt(d)
    q, k, v = by_key_head(s["q"], c), by_key_head(s["k"], c), by_key_head(s["v"], c)
    z = (torch.matmul(q, k.transpose(2, 3)) * scale).reshape(b, hk, group, lq, lk)
    bent = None
    if c["cap"]:
        bent = torch.tanh(z / c["cap"])
        z = bent * c["cap"]
    sees, far = visible(s)
    if s["slopes"] is not None:
        z = z - s["slopes"].reshape(1, hk, group, 1, 1) * far
    z = torch.where(sees, z, torch.full_like(z, -math.inf))
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).reshape(b, hk * group, lq).transpose(1, 2).contiguous()
    p = (e / torch.where(total > 0, total, torch.ones_like(total))).reshape(b, hk, group * lq, lk)
    o = torch.matmul(p, v)
    answer = {"out": from_key_head(o, s["q"]), "lse": lse}
    if c["direction"] == "train":
        do = by_key_head(s["dout"], c)
        dp = torch.matmul(do, v.transpose(2, 3))
        ds = p * (dp - (do * o).sum(-1, keepdim=True))
        if bent is not None:
            ds = ds * (1.0 - bent.reshape(ds.shape).square())
        ds = ds * scale
        answer |= {"dq": from_key_head(torch.matmul(ds, k), s["q"]), "dk": from_key_head(torch.matmul(ds.transpose(2, 3), q), s["k"]),
                   "dv": from_key_head(torch.matmul(p.transpose(2, 3), do), s["v"])}
    return answer


def plain_rotary(s):
    c = s["case"]
    cos, sin = (s[x][s["positions"].long()][:, :, None, :] for x in ("cos", "sin"))
    sin = -sin if c["direction"] == "gradient" else sin
    return {"q": turned(s["q"], cos, sin, c), "k": turned(s["k"], cos, sin, c)}


def turned(x, cos, sin, c):
    r, half, y = c["rotated"], c["rotated"] // 2, x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if c["interleaved"] else (y[..., :half], y[..., half:r])
    first, second = a * cos - b * sin, a * sin + b * cos
    both = torch.stack((first, second), -1).flatten(-2) if c["interleaved"] else torch.cat((first, second), -1)
    return torch.cat((both, y[..., r:]), -1).to(x.dtype)


def to_blocks(x):
    """Values in 8 bits (e4m3) with a scale for each 256: ([blocks, 256], [blocks])."""
    x = torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)).reshape(-1, BLOCK)
    scale = x.abs().amax(1).clamp(min=2.0 ** -100) / 448.0
    return (x / scale[:, None]).to(torch.float8_e4m3fn), scale


def plain_adamw(s):
    done = [plain_tensor(s, i) for i in range(len(s["p"]))]
    names = ("p", "m", "v", "m_scale", "v_scale") if s["case"]["bits"] == 8 else ("p", "m", "v")
    return {n: [d[i] for d in done] for i, n in enumerate(names)}


def plain_tensor(s, i):
    shape, n = s["p"][i].shape, s["p"][i].numel()
    m, v = s["m"][i], s["v"][i]
    if s["case"]["bits"] == 8:
        m = (m.float() * s["m_scale"][i][:, None]).reshape(-1)[:n].reshape(shape)
        v = (v.float() * s["v_scale"][i][:, None]).reshape(-1)[:n].reshape(shape).square()
    p, g = s["p"][i].float(), s["g"][i].float() * STEP["grad_scale"]
    m = m * STEP["beta1"] + g * (1.0 - STEP["beta1"])
    v = v * STEP["beta2"] + g * g * (1.0 - STEP["beta2"])
    root = v.sqrt()
    under = root * (1.0 / math.sqrt(1.0 - STEP["beta2"] ** STEP["step"])) + STEP["eps"]
    p = p * (1.0 - STEP["rate"] * STEP["decay"]) - m / under * (STEP["rate"] / (1.0 - STEP["beta1"] ** STEP["step"]))
    p = p.to(s["p"][i].dtype)
    if s["case"]["bits"] == 32:
        return p, m, v
    (m, m_scale) = to_blocks(m)
    root = torch.nn.functional.pad(root.reshape(-1), (0, -n % BLOCK)).reshape(-1, BLOCK)
    v_scale = root.amax(1).clamp(min=2.0 ** -100) / 448.0
    # a second moment that is not zero does not become zero: the step is divided by its root
    root = torch.where(root > 0, (root / v_scale[:, None]).clamp(min=2.0 ** -9), root)
    return p, m, root.to(torch.float8_e4m3fn), m_scale, v_scale


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


def own_attention(s):
    ops, dev = framework()
    c, stream = s["case"], torch.cuda.current_stream().cuda_stream
    how = dict(causal=c["causal"], window=c["window"], cap=c["cap"], slopes=s["slopes"], lengths=s["lengths"], prefix=s["prefix"],
               query_documents=s["documents"], key_documents=s["documents"])
    room = torch.empty(ops.attention_workspace(dev, s["q"], s["k"], s["v"], backward=c["direction"] == "train"), dtype=torch.uint8, device=GPU)
    ops.attention(dev, s["q"], s["k"], s["v"], s["out"], s["lse"], workspace=room, stream=stream, **how)
    if c["direction"] == "forward":
        return {"out": s["out"], "lse": s["lse"]}
    ops.attention_backward(dev, s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"], s["dv"], workspace=room,
                           stream=stream, **how)
    return {x: s[x] for x in ("out", "lse", "dq", "dk", "dv")}


def own_rotary(s):
    ops, dev = framework()
    c = s["case"]
    ops.rotary(dev, s["q"], s["q_out"], s["cos"], s["sin"], s["positions"], second=s["k"], second_out=s["k_out"],
               interleaved=c["interleaved"], inverse=c["direction"] == "gradient", stream=torch.cuda.current_stream().cuda_stream)
    return {"q": s["q_out"], "k": s["k_out"]}


def own_adamw(s):
    ops, dev = framework()
    scales = {}
    if s["case"]["bits"] == 8:
        scales = dict(first_scales=s["m_scale"], second_scales=s["v_scale"], first_scales_out=s["m_scale_out"], second_scales_out=s["v_scale_out"])
    ops.adamw(dev, s["p"], s["g"], s["m"], s["v"], parameters_out=s["p_out"], first_out=s["m_out"], second_out=s["v_out"], **scales,
              stream=torch.cuda.current_stream().cuda_stream, **STEP)
    names = ("p", "m", "v", "m_scale", "v_scale") if s["case"]["bits"] == 8 else ("p", "m", "v")
    return {n: s[n + "_out"] for n in names}


# ---- work ---------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    wide = {"f32": 4, "bf16": 2}
    if c["op"] == "rotary":
        rows = c["batch"] * c["length"]
        moved = 2 * rows * (c["heads"] + c["key_heads"]) * c["size"] * wide[c["dtype"]]
        return {"bytes": moved + 4 * rows + min(rows, 2 * c["length"] + 64) * c["rotated"] * 4,
                "flops": 3 * rows * (c["heads"] + c["key_heads"]) * c["rotated"]}
    if c["op"] == "adamw":
        n = sum(math.prod(int(k) for k in x.split("x")) for x in c["shapes"].split(","))
        held = 2 * (4 if c["bits"] == 32 else 1 + 4 / BLOCK)
        return {"bytes": n * (2 * wide[c["dtype"]] + wide[c["grad"]] + 2 * held), "flops": 14 * n}
    b, lq, h, hk, d, w = c["batch"], c["queries"], c["heads"], c["key_heads"], c["size"], wide[c["dtype"]]
    lk = int(c["keys"] * (0.75 if c["ragged"] else 1.0))
    # keys that a query sees on average; ends of documents and prefixes by their mean
    seen = lk - (lq - 1) / 2 if c["causal"] and lk >= lq else lk / 2 if c["causal"] else lk
    if c["window"]:
        seen = min(seen, c["window"] if c["causal"] else 2 * c["window"])
    if c["prefix"]:
        seen = min(lk, max(seen, c["keys"] / 4 + seen / 2))
    if c["document"]:
        seen = min(seen, c["document"] * (1 if c["causal"] else 2))
    rows = b * lq * h
    bytes_ = 2 * rows * d * w + 4 * rows + 2 * b * lk * hk * d * w
    flops = 4 * rows * seen * d
    if c["direction"] == "train":
        bytes_ += 2 * rows * d * w + 2 * b * lk * hk * d * w
        flops *= 3.5
    return {"bytes": bytes_, "flops": flops}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": exact_attention, "rotary": exact_rotary, "adamw": exact_adamw}[case["op"]](case, s)


def exact_attention(c, s):
    b, lq, lk, h, d = c["batch"], c["queries"], c["keys"], c["heads"], c["size"]
    group, train = h // c["key_heads"], c["direction"] == "train"
    like = dict(dtype=torch.float64, device=GPU)
    r = {"out": torch.zeros((b, lq, h, d), **like), "lse": torch.zeros((b, lq, h), **like)}
    if train:
        r |= {"dq": torch.zeros((b, lq, h, d), **like), "dk": torch.zeros((b, lk, c["key_heads"], d), **like)}
        r["dv"] = torch.zeros_like(r["dk"])
    for n in range(b):
        length = lk if s["lengths"] is None else int(s["lengths"][n])
        query_at = torch.arange(length - lq, length, device=GPU).unsqueeze(1)
        key_at = torch.arange(lk, device=GPU).unsqueeze(0)
        hidden = torch.zeros((lq, lk), dtype=torch.bool, device=GPU)
        if c["causal"]:
            hidden |= key_at > query_at
        if c["window"]:
            hidden |= (query_at - key_at >= c["window"]) | (key_at - query_at >= c["window"])
        if s["prefix"] is not None:
            hidden &= key_at >= int(s["prefix"][n])
        hidden |= key_at >= length
        if s["documents"] is not None:
            mine = s["documents"][n]
            hidden |= (mine[lk - lq:].unsqueeze(1) != mine.unsqueeze(0)) | (mine < 0).unsqueeze(0)
        for a in range(h):
            q, k, v = s["q"][n, :, a].double(), s["k"][n, :, a // group].double(), s["v"][n, :, a // group].double()
            raw = q @ k.T / math.sqrt(d)
            score = c["cap"] * torch.tanh(raw / c["cap"]) if c["cap"] else raw
            slope = torch.ones_like(score)
            if c["cap"] and train:
                slope = 1 - (score / c["cap"]) ** 2
            if s["slopes"] is not None:
                score = score - float(s["slopes"][a]) * (query_at - key_at).abs()
            score = score.masked_fill(hidden, -math.inf)
            lse = torch.logsumexp(score, 1)
            weight = torch.exp(score - lse.unsqueeze(1)).masked_fill(hidden, 0.0)
            r["lse"][n, :, a] = lse
            r["out"][n, :, a] = weight @ v
            if train:
                do = s["dout"][n, :, a].double()
                r["dv"][n, :, a // group] += weight.T @ do
                dw = do @ v.T
                ds = weight * (dw - (weight * dw).sum(1, keepdim=True)) * slope / math.sqrt(d)
                r["dq"][n, :, a] = ds @ k
                r["dk"][n, :, a // group] += ds.T @ q
    return r


def exact_rotary(c, s):
    """Each pair as a complex number, times exp(i angle) from the table."""
    factor = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()].unsqueeze(2)
    factor = factor.conj() if c["direction"] == "gradient" else factor
    r = {}
    for name in ("q", "k"):
        x = s[name].double()
        part = x[..., :c["rotated"]]
        if c["interleaved"]:
            z = torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous())
            y = torch.view_as_real(z * factor).flatten(-2)
        else:
            z = torch.complex(*(t.contiguous() for t in part.unflatten(-1, (2, -1)).unbind(-2))) * factor
            y = torch.cat((z.real, z.imag), -1)
        r[name] = x.clone()
        r[name][..., :c["rotated"]] = y
    return r


def exact_adamw(c, s):
    r = {n: [] for n in (("p", "m", "v", "m_scale", "v_scale") if c["bits"] == 8 else ("p", "m", "v"))}
    b1, b2, t = STEP["beta1"], STEP["beta2"], STEP["step"]
    for i, p in enumerate(s["p"]):
        n = p.numel()
        m, v = s["m"][i].double(), s["v"][i].double()
        if c["bits"] == 8:
            m = (m * s["m_scale"][i].double().unsqueeze(1)).flatten()[:n]
            v = ((v * s["v_scale"][i].double().unsqueeze(1)) ** 2).flatten()[:n]
        g = s["g"][i].double().flatten() * STEP["grad_scale"]
        m, v = b1 * m.flatten() + (1 - b1) * g, b2 * v.flatten() + (1 - b2) * g ** 2
        ahead = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + STEP["eps"])
        x = p.double().flatten()
        r["p"].append((x - STEP["rate"] * STEP["decay"] * x - STEP["rate"] * ahead).reshape(p.shape))
        if c["bits"] == 32:
            r["m"].append(m.reshape(p.shape))
            r["v"].append(v.reshape(p.shape))
            continue
        for name, x in (("m", m), ("v", v ** 0.5)):
            rows = torch.cat((x, x.new_zeros(-n % BLOCK))).view(-1, BLOCK)
            scale = rows.abs().max(1).values.clamp(min=2.0 ** -100) / 448
            held = rows / scale.unsqueeze(1)
            if name == "v":
                held = torch.where(held > 0, held.clamp(min=2.0 ** -9), held)
            r[name].append(held.to(torch.float8_e4m3fn).double())
            r[name + "_scale"].append(scale)
    return r

"""The gradients of the restatements that the kernels are held to (training_oracle.py), against automatic differentiation of the
formulas and against differences of their own results, in 64 bits."""
import pytest
import torch

import training_oracle as oracle


def differences(f, x, direction, step=1e-6):
    """Of a number, along a direction."""
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)


@pytest.mark.parametrize("centered", [True, False])
def test_layer_norm(centered):
    g = torch.Generator().manual_seed(1)
    x, dy, w, b = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((4, 9), (4, 9), (9,), (9,)))
    oracle.W[torch.float64] = 0.0
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    t = leaves[0] - leaves[0].mean(-1, keepdim=True) if centered else leaves[0]
    y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-5) * leaves[1] + leaves[2]
    grads = torch.autograd.grad((y * dy).sum(), leaves)
    r, _ = oracle.layer_norm(x, w, b, centered=centered, out_grad=dy)
    assert torch.allclose(r["out"], y, rtol=1e-12, atol=1e-12)
    for n, want in zip(("x_grad", "weight_grad", "bias_grad"), grads):
        assert torch.allclose(r[n], want, rtol=1e-10, atol=1e-12), n
    along = torch.randn(x.shape, generator=g, dtype=torch.float64)
    slope = differences(lambda v: float((oracle.layer_norm(v, w, b, centered=centered)[0]["out"] * dy).sum()), x, along)
    assert abs(slope - float((r["x_grad"] * along).sum())) <= 1e-7 * float((r["x_grad"] * along).abs().sum())


@pytest.mark.parametrize("factors", [True, False])
@pytest.mark.parametrize("masked", [True, False])
def test_recurrence(factors, masked):
    g = torch.Generator().manual_seed(2)
    B, L, C = 3, 23, 4
    oracle.W[torch.float64] = 0.0
    x, gates, dout = (torch.randn((B, L, C), generator=g, dtype=torch.float64) for _ in range(3))
    first, last = (torch.randn((B, C), generator=g, dtype=torch.float64) for _ in range(2))
    how = dict(factors=factors)
    if masked:
        d = torch.cumsum(torch.rand((B, L), generator=g) < 0.2, 1).to(torch.int32)
        d[0, 5:7] = -1
        how |= dict(documents=d, lengths=torch.tensor([23, 0, 11]))
    leaves = [t.clone().requires_grad_() for t in (x, gates, first)]
    outs, hs = [], []
    for b in range(B):
        h, n = leaves[2][b], int(how["lengths"][b]) if masked else L
        rows = []
        for t in range(L):
            if t >= n or (masked and d[b, t] < 0):
                if t < n:
                    h = torch.zeros_like(h)
                rows.append(torch.zeros_like(h))
                continue
            before = torch.zeros_like(h) if masked and t > 0 and d[b, t] != d[b, t - 1] else h
            p = leaves[1][b, t]
            h = p * before + leaves[0][b, t] if factors else torch.sigmoid(p) * before + (1 - torch.sigmoid(p)) * leaves[0][b, t]
            rows.append(h)
        outs.append(torch.stack(rows))
        hs.append(h)
    out, final = torch.stack(outs), torch.stack(hs)
    grads = torch.autograd.grad((out * dout).sum() + (final * last).sum(), leaves)
    r, _ = oracle.recurrence(x, gates, initial=first, out_grad=dout, final_grad=last, **how)
    assert torch.allclose(r["out"], out, rtol=1e-12, atol=1e-12) and torch.allclose(r["final"], final, rtol=1e-12, atol=1e-12)
    for n, want in zip(("x_grad", "gates_grad", "initial_grad"), grads):
        assert torch.allclose(r[n], want, rtol=1e-10, atol=1e-12), n
    along = torch.randn(x.shape, generator=g, dtype=torch.float64)

    def total(v):
        r, _ = oracle.recurrence(x, v, initial=first, **how)
        return float((r["out"] * dout).sum() + (r["final"] * last).sum())

    assert abs(differences(total, gates, along) - float((r["gates_grad"] * along).sum())) <= 1e-7 * float((r["gates_grad"] * along).abs().sum())

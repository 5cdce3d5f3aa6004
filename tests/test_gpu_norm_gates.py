"""norm_after's gradient of gates that are nearly open or shut, against float64. Its factor
sigmoid(-gate) is e^-gate for an open gate, and is held to its own size here: 1 - sigmoid(gate) in
float32 would be off by 2^-24, which is all of it from a gate of 17 on.

Bounds as in tests/test_gpu_norms.py, K = 256 roundings of the sum of the magnitudes, the factor among
them: with |gate| <= 30 the two sigmoids pass 2 |gate| + 6 roundings each (the exponential's argument
times log2 e, both rounded, move it by 2 |gate| u), the two norms 80, the products 16: 228."""
import pytest
import torch

import test_gpu_norms as norms

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def expect(t):
    want = norms.expect(t)
    f = {n: None if x is None else x.double() for n, x in t.items()}
    sg, shut = torch.sigmoid(f["gate"]), torch.sigmoid(-f["gate"])
    hn = f["h"] * (f["h"].square().mean(-1, keepdim=True) + norms.EPS).rsqrt()
    c = f["scale"] * f["weight"] * sg * hn * shut
    g, mag = want["resid"]   # the gradient of y
    rows = t["gate"].dim() == 2
    want["gate"] = tuple(x if rows else x.sum(0) for x in (g * c, mag * c.abs()))
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["rows", "cols"])
@pytest.mark.parametrize("following", [False, True])
@pytest.mark.parametrize("n,D", [(40, 64), (9, 121), (3, 2048)])
def test_gates_far_from_zero(n, D, following, gate, dtype, device):
    t = norms.make(n, D, dtype, device, True, gate, True, following, seed=n)
    t["gate"] = torch.linspace(-30, 30, t["gate"].numel(), device=device).view_as(
        t["gate"]).to(t["gate"].dtype)
    norms.check(norms.run(t), expect(t), n)


@pytest.mark.parametrize("gate", ["rows", "cols"])
def test_gates_past_every_exponential(gate, device):
    """Beyond float32's exponentials: zeros on the far side, no NaN or infinity anywhere."""
    t = norms.make(8, 48, torch.float32, device, True, gate, True, True)
    far = torch.tensor([-3e38, -1000.0, -89.0, 89.0, 1000.0, 3e38], device=device)
    t["gate"] = far.repeat(t["gate"].numel() // 6).view_as(t["gate"])
    got = norms.run(t)
    for n, x in got.items():
        assert torch.isfinite(x).all(), n
    assert got["gate"].abs().max() < 1e-36


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_with_a_parameters_gate(dtype, device):
    """h (D,) and a float32 gate (D,): what the same row gives as a batch of one, bit by bit."""
    from gatx import BlockNorm
    m = BlockNorm(40).to(device)
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(40, generator=g))
    h, r, gy, gn = (torch.randn(40, generator=g).to(dtype).to(device) for _ in range(4))

    def step(h, r, gy, gn):
        x = [h.clone().requires_grad_(True), r.clone().requires_grad_(True)]
        outs = m(x[0], x[1])
        return [o.detach().flatten() for o in outs] + [
            y.flatten() for y in torch.autograd.grad(outs, x + list(m.parameters()), [gy, gn])]
    one, batch = step(h, r, gy, gn), step(h[None], r[None], gy[None], gn[None])
    assert all(torch.equal(a, b) for a, b in zip(one, batch))

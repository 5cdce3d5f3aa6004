"""The graph-transformer operators where an element's offset passes 32 bits: the last rows of tensors
of more than 2^31 elements against float64 on those rows alone, with the bounds of the operators' own
tests. (Not against the bits of a small call: how many lanes share a row, and so the order of its
sums, depends on the number of rows.)"""
import math

import pytest
import torch

import attention_reference as ref
import test_gpu_distillation as distillation

pytestmark = pytest.mark.gpu


def test_attention_far_rows(device):
    from gatx import diff_attention
    from gatx.graph import Graph
    N, H, d, dv, M = 1_100_000, 8, 128, 256, 200   # keys and values: 2.25e9 elements each
    g = torch.Generator(device=device).manual_seed(1)
    e = torch.randint(0, M, (2, 4000), device=device, generator=g)
    small = {"q": (M, H, 2, d), "k": (M, H, 2, d), "v": (M, H, dv), "go": (M, H, dv)}
    small = {n: torch.randn(s, device=device, generator=g).bfloat16() for n, s in small.items()}
    lam = torch.rand(H, device=device, generator=g)

    def run(t, edges, n):
        x = {m: t[m].detach().requires_grad_(True) for m in ("q", "k", "v")}
        x["lam"] = lam.clone().requires_grad_(True)
        graph = Graph(edges, n, False)
        out = diff_attention(x["q"], x["k"], x["v"], x["lam"], graph)
        got = torch.autograd.grad(out, list(x.values()), t["go"])
        nodes = torch.tensor([n - 1, n - M], device=device)
        with torch.no_grad():
            served = diff_attention(x["q"][nodes], x["k"], x["v"], lam, graph, nodes=nodes)
        return [out.detach()[n - M:], served] + [y[n - M:] for y in got[:3]] + [got[3]]
    big = {}
    for n, x in small.items():
        big[n] = torch.zeros((N,) + x.shape[1:], dtype=x.dtype, device=device)
        big[n][N - M:] = x
    got = dict(zip(("out", "served", "q", "k", "v", "lam"), run(big, e + (N - M), N)))
    f64 = {n: x.double().cpu() for n, x in small.items()}
    want = ref.attention(f64["q"], f64["k"], f64["v"], lam.double().cpu(), e[0].cpu(), e[1].cpu(),
                         torch.arange(M), 1 / math.sqrt(d), go=f64["go"])
    want["served"] = tuple(x[[M - 1, 0]] for x in want["out"])
    for n, x in got.items():
        ref.check(x, want[n], n)


def test_norm_far_rows(device):
    from gatx import norm_after
    n, D, M = 270_000, 8192, 40
    g = torch.Generator(device=device).manual_seed(2)
    w = [1 + 0.1 * torch.randn(D, device=device, generator=g) for _ in range(3)]
    small = torch.randn(M, D, device=device, generator=g).bfloat16()

    def run(h):
        h = h.detach().requires_grad_(True)
        y, nxt = norm_after(h, w[0], scale=w[1], next_weight=w[2])
        gh, = torch.autograd.grad([y, nxt], h, [y.detach(), nxt.detach()])
        return [t.detach()[-M:] for t in (y, nxt, gh)]
    want = run(small)
    big = torch.ones(n, D, dtype=torch.bfloat16, device=device)
    big[n - M:] = small
    for i, (a, b) in enumerate(zip(want, run(big))):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("n,C", [(70_000, 32_768), (2_300_000, 1000)])
def test_distillation_far_rows(n, C, device):
    M, K = 30, 8
    g = torch.Generator(device=device).manual_seed(3)
    x = torch.randn(M, C, device=device, generator=g).bfloat16()
    t = torch.randn(M, K, device=device, generator=g)
    i = torch.randint(0, C, (M, K), device=device, generator=g)

    loss, lb, grad, gb = distillation.expect(x, t, i, 2.0)
    big = [torch.zeros((n,) + y.shape[1:], dtype=y.dtype, device=device) for y in (x, t, i)]
    big[2].fill_(-1)
    for a, b in zip(big, (x, t, i)):
        a[n - M:] = b
    got, g = distillation.run(*big, 2.0, "none", torch.ones(n, device=device))
    distillation.near(got[n - M:], loss, lb)
    distillation.near(g[n - M:], grad, gb)
    assert not bool(got[:n - M].any()) and not bool(g[:n - M].any())

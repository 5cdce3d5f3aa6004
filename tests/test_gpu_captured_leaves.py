"""A captured backward beside an eager graph that is alive on the default stream: refused where it would
go on to one of that graph's leaves (also through the cast of a 16-bit parameter, a view of the leaf or
other operations), and captured where nothing there is asked for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def calls(device):
    """{operator: (leaves, a call on what `of` makes of them, the first leaf's gradient with them)}"""
    from gatx import diff_attention, norm_after
    from gatx.graph import Graph
    from gatx.losses import topk_distillation
    N = 40
    g = torch.Generator(device=device).manual_seed(1)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=device).to(dtype)
    graph = Graph(torch.randint(0, N, (2, 300), device=device, generator=g), N, False)
    q, k, v = normal(N, 2, 2, 8), normal(N, 2, 2, 8), normal(N, 2, 16)
    pos = torch.arange(N, device=device)
    h, t = normal(N, 24), normal(N, 3)
    i = torch.randint(0, 24, (N, 3), device=device, generator=g)
    return {
        "diff_attention": ({"lam": normal(2, dtype=torch.bfloat16),
                            "bias": normal(8, 2, dtype=torch.bfloat16), "q": q},
                           lambda x: diff_attention(x["q"], k, v, x["lam"], graph, bias=x["bias"],
                                                    positions=pos, max_distance=20)),
        "norm_after": ({"weight": normal(24, dtype=torch.bfloat16),
                        "scale": normal(24, dtype=torch.float16),
                        "gate": normal(24, dtype=torch.bfloat16), "h": h},
                       lambda x: norm_after(x["h"], x["weight"], scale=x["scale"], gate=x["gate"])),
        "topk_distillation": ({"h": h.t().contiguous()},
                              lambda x: topk_distillation(x["h"].t(), t, i)),
        "projection": ({"w": normal(24, 24)},
                       lambda x: topk_distillation(norm_after(h @ x["w"] + h, h.new_ones(24)), t, i)),
    }


def warm(device):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.randn(4, device=device, requires_grad=True).sum().backward()   # the engine's thread
    torch.cuda.synchronize()
    return s


CASES = [("diff_attention", "lam"), ("diff_attention", "bias"), ("norm_after", "weight"),
         ("norm_after", "scale"), ("norm_after", "gate"), ("topk_distillation", "h"),
         ("projection", "w")]


@pytest.mark.parametrize("name,asked", CASES)
def test_leaves_behind_a_cast_or_a_view_are_seen(name, asked, device):
    leaves, call = calls(device)[name]
    x = {n: t.clone().requires_grad_(True) for n, t in leaves.items()}
    alive = call(x)
    ones = torch.ones_like(alive)
    want, = torch.autograd.grad(alive, x[asked], ones, retain_graph=True)
    s = warm(device)

    def step():
        return torch.autograd.grad(call(x), x[asked], ones)[0]
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="alive on the default stream"):
        with torch.cuda.graph(graph, stream=s):
            step()
    torch.cuda.synchronize()
    del alive
    with torch.cuda.stream(s):
        assert torch.equal(step(), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step()
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("name,asked", [("diff_attention", "q"), ("norm_after", "h")])
def test_leaves_that_nothing_asks_for_do_not_count(name, asked, device):
    """The gradient of one tensor alone, the parameters' eager graph alive on the default stream."""
    leaves, call = calls(device)[name]
    x = {n: t.clone().requires_grad_(True) for n, t in leaves.items() if n != asked}
    own = leaves[asked].clone().requires_grad_(True)
    alive = call({**x, asked: own.detach()})
    ones = torch.ones_like(alive)
    s = warm(device)

    def step():
        return torch.autograd.grad(call({**x, asked: own}), own, ones)[0]
    with torch.cuda.stream(s):
        want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step()
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert torch.isfinite(alive).all()

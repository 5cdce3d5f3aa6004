"""The graph-transformer operators called inside torch.compile: they run eagerly between the compiled
parts, with the eager call's results and gradients, graph after graph; one whole graph is refused.

The compiled parts may add in another order: a few float32 roundings of values of size 1 to 10."""
import pytest
import torch

pytestmark = pytest.mark.gpu

N = 64


def stack(device):
    from gatx import BlockNorm, DiffAttention, norm_before
    from gatx.losses import topk_distillation
    torch.manual_seed(0)
    att = DiffAttention(16, 8, 2, position_buckets=8, max_distance=20).to(device)
    block = BlockNorm(16).to(device)
    w = torch.ones(16, device=device, requires_grad=True)
    pos = torch.arange(N, device=device)
    teacher = torch.randn(N, 3, device=device)
    index = torch.randint(0, 16, (N, 3), device=device)

    def step(x, graph):
        y, n = block(att(norm_before(x * 1.5, w), positions=pos, graph=graph).sin(), x)
        return topk_distillation(y + n, teacher, index) * 3
    return step


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_steps_equal_eager_ones(backend, device):
    from gatx.graph import Graph
    torch._dynamo.reset()
    step = stack(device)
    compiled = torch.compile(step, backend=backend)
    for i in range(12):   # past the number of recompilations that torch allows
        graph = Graph(torch.randint(0, N, (2, 300 + 40 * i), device=device), N, False)
        x = torch.randn(N, 16, device=device)
        got = []
        for f in (step, compiled, compiled):
            y = x.clone().requires_grad_(True)
            loss = f(y, graph)
            got.append((loss.detach(), torch.autograd.grad(loss, y)[0]))
        for a, b in zip(got[0] * 2, got[1] + got[2]):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6), i
    torch._dynamo.reset()


def test_one_whole_graph_is_refused(device):
    from gatx.graph import Graph
    torch._dynamo.reset()
    graph = Graph(torch.randint(0, N, (2, 300), device=device), N, False)
    compiled = torch.compile(stack(device), backend="eager", fullgraph=True)
    with pytest.raises(torch._dynamo.exc.Unsupported):
        compiled(torch.randn(N, 16, device=device), graph)
    torch._dynamo.reset()

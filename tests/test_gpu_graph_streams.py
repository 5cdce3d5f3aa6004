"""One gatx.Graph used by a GAT layer on one stream and by diff_attention on another, without a wait
between them: what the first builds (the CSR, the transpose, plans, the order of rows) is behind a long
queue on its stream when the second asks for it. The same bits as alone."""
import pytest
import torch

from test_gpu_attention import graph_of, make, run

pytestmark = pytest.mark.gpu

N = 3000


def inputs(device):
    t = make(N, 30000, 3, 16, 24, torch.float32, device, seed=8, hub=2000, buckets=8)
    g = torch.Generator().manual_seed(2)
    t["x"], t["W"], t["a"] = (torch.randn(*s, generator=g).to(device) for s in
                              ((N, 12), (2 * 8, 12), (2, 2 * 2 * 8)))
    return t


def gat(t, graph):
    from gatx.functional import gat_layer_lazy
    x, W = (t[n].clone().requires_grad_(True) for n in ("x", "W"))
    out, _, _ = gat_layer_lazy(x, None, W, t["a"], None, 2, 8, True, False, graph=graph)
    gx, gW = torch.autograd.grad(out.square().sum(), [x, W])
    return {"out": out.detach(), "x": gx, "W": gW}


def attention(t, graph):
    return run(t, graph)


def queue(device):
    """Some 20 ms of work."""
    a = torch.randn(4096, 4096, device=device)
    for _ in range(20):
        a = a @ a
        a = a / a.norm()


@pytest.mark.parametrize("first,second", [(gat, attention), (attention, gat),
                                          (attention, attention)])
def test_the_second_stream_waits(first, second, device):
    t = inputs(device)
    want = [f(t, graph_of(t, N, device)) for f in (first, second)]
    edges = torch.stack([t["src"], t["dst"]]).to(device)
    queue(device)   # (the library's first calls)
    torch.cuda.synchronize()
    from gatx.graph import Graph
    for _ in range(3):
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            queue(device)
            graph = Graph(edges, N, False)
            one = first(t, graph)
        with torch.cuda.stream(b):
            two = second(t, graph)
            again = second(t, graph)
        del graph   # its memory may be handed out again once both streams are done with it
        with torch.cuda.stream(a):
            junk = [torch.full((30000,), -1, dtype=torch.int32, device=device) for _ in range(12)]
        torch.cuda.synchronize()
        for got, w in ((one, want[0]), (two, want[1]), (again, want[1])):
            for n in w:
                assert torch.equal(got[n], w[n]), n
        del junk


def test_graphs_built_on_several_streams_at_once(device):
    """Many small graphs, each with its own sizes, ids and self-loops, on four streams in turn."""
    from gatx.graph import Graph
    g = torch.Generator().manual_seed(5)
    edges = [torch.randint(0, 50 + 37 * i, (2, 3000 + 711 * i), generator=g).to(device)
             for i in range(12)]
    for e in edges[::2]:
        e[1, ::3] = e[0, ::3]   # self-loops, dropped
    want = [Graph(e, int(e.max()) + 1, True).csr_host() for e in edges]
    sizes = [int(e.max()) + 1 for e in edges]
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        torch.cuda.synchronize()
        built = []
        for i, e in enumerate(edges):
            with torch.cuda.stream(streams[i % 4]):
                built.append(Graph(e, sizes[i], True))
        torch.cuda.synchronize()
        for got, w in zip(built, want):
            assert all(torch.equal(a, b) for a, b in zip(got.csr_host(), w))


def test_the_graph_cache_hands_a_graph_to_another_stream(device):
    """DiffAttention and GATLayer find the graph of an edge_index in the cache."""
    import gatx
    from gatx import DiffAttention
    t = inputs(device)
    edges = torch.stack([t["src"], t["dst"]]).to(device)
    layer = DiffAttention(12, 8, 2).to(device)

    def step():
        x = t["x"].clone().requires_grad_(True)
        out = layer(x, edges)
        return out.detach(), torch.autograd.grad(out.square().sum(), x)[0]
    gatx.clear_graph_cache()
    want = step()
    queue(device)
    gatx.clear_graph_cache()
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        queue(device)
        one = step()
    with torch.cuda.stream(b):
        two = step()
    torch.cuda.synchronize()
    for got in (one, two):
        for x, y in zip(got, want):
            assert torch.equal(x, y)

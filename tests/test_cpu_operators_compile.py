"""torch.compile does not look into what handles streams and events: diff_attention, the building of a
gatx.Graph and the graph cache run as they are between the compiled parts. (It would keep weak references
to the graph's events and follow them after the graph is gone.)"""
import types

import pytest
import torch


@pytest.fixture
def seen(monkeypatch):
    torch._dynamo.reset()
    yield []
    torch._dynamo.reset()


def twice(f, *args):
    compiled = torch.compile(f, backend="eager")
    return [compiled(*args) for _ in range(2)]


def test_diff_attention(seen, monkeypatch):
    from gatx import attention

    def check(*args):
        seen.append(("check", torch.compiler.is_compiling()))

    class Stub:
        rowptr = col = rowidx = None
        num_nodes, edge_bound, device = 5, 9, torch.device("cpu")

        def _poll(self):
            seen.append(("poll", torch.compiler.is_compiling()))
    monkeypatch.setattr(attention, "_check", check)
    monkeypatch.setattr(attention, "_host", types.SimpleNamespace(
        diff_attention_nodes=lambda q, *a: q + 1))
    graph, nodes = Stub(), torch.arange(2)
    q = torch.zeros(2, 1, 2, 4)
    for out in twice(lambda q: attention.diff_attention(q * 2, q, q, q, graph, nodes=nodes) * 3, q):
        assert torch.equal(out, torch.full_like(q, 3))
    assert seen and not any(compiling for _, compiling in seen), seen


def test_graphs(seen, monkeypatch):
    from gatx import graph

    def build(self, edge_index, num_nodes, add_self_loops):
        seen.append(("build", torch.compiler.is_compiling()))
        self._error, self._builds, self._E2 = None, {}, 3

    class OnDevice(torch.Tensor):
        is_cuda = True
    monkeypatch.setattr(graph.Graph, "_build_csr", build)
    cache = graph.GraphCache()
    edges = torch.zeros(2, 3, dtype=torch.int64).as_subclass(OnDevice)

    def f(x):
        graph.Graph(edges, 5, False)
        cache.get(edges, 5, False)
        return x + 1
    assert all(torch.equal(y, torch.ones(2)) for y in twice(f, torch.zeros(2)))
    assert seen and not any(compiling for _, compiling in seen), seen


@pytest.mark.parametrize("name", ["poll", "ensure_transpose", "hub_plan", "node_blocks"])
def test_a_graphs_methods(name, seen, monkeypatch):
    from gatx import graph
    g = object.__new__(graph.Graph)
    g.device, g.srowptr, g._builds, g._hub_plans, g._error, g._E2 = "cpu", None, {}, {}, None, 3

    def build(self, *args):
        seen.append(torch.compiler.is_compiling())
        return torch.zeros(1), 0, 0
    for inner in ("follow", "_build_transpose", "_kept"):
        monkeypatch.setattr(graph.Graph, inner, build)
    monkeypatch.setattr(graph, "on_device", lambda device: graph._BUILDING)
    args = {"hub_plan": (512,), "node_blocks": (2304,)}.get(name, ())

    def f(x):
        getattr(g, name)(*args)
        return x + 1
    assert all(torch.equal(y, torch.ones(2)) for y in twice(f, torch.zeros(2)))
    assert seen and not any(seen), seen

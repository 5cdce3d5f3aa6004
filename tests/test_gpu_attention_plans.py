"""diff_attention's plans of long rows over many steps on one gatx.Graph: rows longer than
attn_hub_edges among the destinations alone, the sources alone, both or neither, whatever is known of
them when a step runs. Against float64 (tests/attention_reference.py), and the same bits every step."""
import pytest
import torch

from test_gpu_attention import check_all, expect, graph_of, make, run

pytestmark = pytest.mark.gpu

N, T = 2000, 512


def one_sided(kind, dtype, device, seed=0, buckets=8):
    """Random edges (15 a node or so) and 1700 more into node 3 (from different nodes) and / or out of
    node 5 (to different nodes)."""
    t = make(N, 8000, 2, 16, 24, dtype, device, seed=seed, buckets=buckets)
    g = torch.Generator().manual_seed(100 + seed)
    if kind in ("destinations", "both"):
        t["src"] = torch.cat([t["src"], torch.randperm(N, generator=g)[:1700]])
        t["dst"] = torch.cat([t["dst"], torch.full((1700,), 3)])
    if kind in ("sources", "both"):
        t["src"] = torch.cat([t["src"], torch.full((1700,), 5)])
        t["dst"] = torch.cat([t["dst"], torch.randperm(N, generator=g)[:1700]])
    longest = [int(torch.bincount(t[n], minlength=N).max()) for n in ("dst", "src")]
    assert (longest[0] > T) == (kind in ("destinations", "both"))
    assert (longest[1] > T) == (kind in ("sources", "both"))
    return t


KINDS = ["destinations", "sources", "both", "neither"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", KINDS)
def test_steps_on_one_graph(kind, dtype, device):
    t = one_sided(kind, dtype, device)
    graph, want = graph_of(t, N, device), None
    first = None
    for step in range(4):
        got = run(t, graph)
        torch.cuda.synchronize()   # what the plans hold is known to the next step
        if step == 0:
            first, want = got, expect(t, N)
        check_all(got, want)
        for n in first:
            assert torch.equal(got[n], first[n]), (step, n)
    known = [graph._hub_plans.get((T, source, "entries")) == 0 for source in (False, True)]
    assert known == [kind in ("sources", "neither"), kind in ("destinations", "neither")]


def test_pieces_of_a_long_source_alone(device):
    """In pieces of several lengths, before and after the plans are known."""
    from gatx import tuning
    t = one_sided("sources", torch.float32, device, seed=2)
    graph, want = graph_of(t, N, device), expect(t, N)
    for hub_edges in (64, 100, 512, 1699, 4000):
        with tuning.override(attn_hub_edges=hub_edges):
            for _ in range(2):
                check_all(run(t, graph), want)
                torch.cuda.synchronize()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("source", [False, True])
def test_one_direction_known_before_the_other(kind, source, device):
    """The counts arrive one after the other: steps in between, eager and captured, are whole."""
    from gatx.capture import CapturedStep
    t = one_sided(kind, torch.bfloat16, device, seed=4)
    first = run(t, graph_of(t, N, device))
    graph = graph_of(t, N, device)
    run(t, graph)
    torch.cuda.synchronize()

    class Unknown:   # a copy that has not arrived
        def query(self):
            return False

    def step():
        for s in (False, True):
            key = (T, s, "entries")
            if s == source:
                count = graph._hub_plans[(T, s)][1] if (T, s) in graph._hub_plans else None
                if count is not None and not torch.cuda.is_current_stream_capturing():
                    graph._hub_plans[key] = 0 if int(count) == 0 else (None, Unknown())
            else:
                graph._hub_plans[key] = (None, Unknown())
        return run(t, graph)
    got = step()
    for n in first:
        assert torch.equal(got[n], first[n]), n
    cap = CapturedStep(step)
    for i in range(3):
        got = {n: x.clone() for n, x in cap().items()}
        torch.cuda.synchronize()
        for n in first:
            assert torch.equal(got[n], first[n]), (i, n)
        run(t, graph)
        torch.cuda.synchronize()


def test_many_graphs_without_waiting(device):
    """A loop over batches, a new graph each, the host ahead of the GPU."""
    ts = [one_sided("neither", torch.float16, device, seed=s) for s in range(3)]
    graphs = [graph_of(t, N, device) for t in ts]
    want = [run(t, g) for t, g in zip(ts, graphs)]
    for _ in range(6):
        for t, g, w in zip(ts, graphs, want):
            got = run(t, g)
            for n in w:
                assert torch.equal(got[n], w[n]), n

"""gatx.diff_attention against float64 on the host (tests/attention_reference.py): every type, odd
and ragged sizes, rows without edges, long rows in pieces, shut buckets, strided inputs, the serving
form, and the gradients of everything learned."""
import math

import pytest
import torch

import attention_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(N, E, H, d, dv, dtype, device, seed=0, hub=0, buckets=0, bidirectional=True, shut=(),
         far=64):
    """Inputs on the device: random edges (about a tenth of the rows have none), `hub` more into
    node 0 and out of node 1."""
    g = torch.Generator().manual_seed(seed)
    dst = torch.randint(0, max(1, N - N // 10), (E,), generator=g)
    src = torch.randint(0, N, (E,), generator=g)
    if hub:
        src = torch.cat([src, torch.randint(0, N, (hub,), generator=g), torch.ones(hub).long()])
        dst = torch.cat([dst, torch.zeros(hub).long(), torch.randint(0, N, (hub,), generator=g)])
        order = torch.randperm(len(src), generator=g)
        src, dst = src[order], dst[order]
    t = {"q": torch.randn(N, H, 2, d, generator=g), "k": torch.randn(N, H, 2, d, generator=g),
         "v": torch.randn(N, H, dv, generator=g), "go": torch.randn(N, H, dv, generator=g)}
    t = {n: x.to(dtype) for n, x in t.items()}
    t["lam"] = 0.2 + 0.6 * torch.rand(H, generator=g)
    t["bias"] = t["positions"] = None
    if buckets:
        t["bias"] = torch.randn(buckets, H, generator=g)
        for b in shut:
            t["bias"][b] = -math.inf
        t["positions"] = torch.randint(-3 * far, 3 * far, (N,), generator=g)
    t = {n: None if x is None else x.to(device) for n, x in t.items()}
    t["src"], t["dst"] = src, dst
    t["kw"] = dict(max_distance=far, bidirectional=bidirectional) if buckets else {}
    return t


def graph_of(t, N, device):
    from gatx.graph import Graph
    return Graph(torch.stack([t["src"], t["dst"]]).to(device), N, False)


def expect(t, N, nodes=None, grads=True, scale=None):
    f64 = {n: t[n].double().cpu() for n in ("q", "k", "v", "go", "lam")}
    src, dst = t["src"], t["dst"]
    row_of = torch.arange(N)
    q = f64["q"]
    if nodes is not None:
        row_of = torch.full((N,), -1)
        row_of[nodes] = torch.arange(len(nodes))
        keep = row_of[dst] >= 0
        src, dst = src[keep], dst[keep]
    bias = bucket = None
    if t["bias"] is not None:
        bias = t["bias"].double().cpu()
        pos = t["positions"].cpu()
        bucket = ref.buckets(pos[src] - pos[dst], bias.size(0), t["kw"]["max_distance"],
                             t["kw"]["bidirectional"])
    scale = 1 / math.sqrt(q.size(-1)) if scale is None else scale
    return ref.attention(q, f64["k"], f64["v"], f64["lam"], src, dst, row_of, scale, bias, bucket,
                         f64["go"] if grads else None)


def run(t, graph, **kw):
    from gatx import diff_attention
    names = ["q", "k", "v", "lam"] + (["bias"] if t["bias"] is not None else [])
    x = {n: t[n].detach().requires_grad_(True) for n in names}
    kw.update(t["kw"])
    if t["bias"] is not None:
        kw.update(bias=x["bias"], positions=t["positions"])
    out = diff_attention(x["q"], x["k"], x["v"], x["lam"], graph, **kw)
    return {"out": out, **dict(zip(names, torch.autograd.grad(out, [x[n] for n in names],
                                                              t["go"])))}


def check_all(got, want):
    assert set(got) == set(want)
    for n in want:
        ref.check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,d,dv", [(1, 1, 1), (2, 8, 16), (3, 7, 5), (4, 6, 12), (2, 16, 16),
                                    (1, 33, 65), (2, 64, 128), (3, 61, 121), (2, 128, 256),
                                    (1, 256, 512), (1, 129, 40), (1, 20, 511)])
def test_widths(H, d, dv, dtype, device):
    N = 70
    t = make(N, 600, H, d, dv, dtype, device, seed=d)
    check_all(run(t, graph_of(t, N, device)), expect(t, N))


@pytest.mark.parametrize("N,E", [(1, 0), (1, 1), (2, 1), (3, 40), (65, 30), (300, 3000),
                                 (2300, 2300), (5000, 40000)])
@pytest.mark.parametrize("H", [1, 5])
def test_sizes(N, E, H, device):
    t = make(N, E, H, 16, 24, torch.float32, device, seed=N)
    check_all(run(t, graph_of(t, N, device)), expect(t, N))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hub_edges", [0, 64, 512])
@pytest.mark.parametrize("d,dv", [(8, 16), (61, 121)])
def test_long_rows(hub_edges, d, dv, dtype, device):
    """A node of 1500 in-edges, another of 1500 out-edges: in pieces or not, the same gradients."""
    from gatx import tuning
    N = 120
    t = make(N, 500, 2, d, dv, dtype, device, seed=3, hub=1500)
    with tuning.override(attn_hub_edges=hub_edges):
        check_all(run(t, graph_of(t, N, device)), expect(t, N))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("buckets,bidirectional,shut,far", [
    (8, True, (), 64), (32, True, (3, 20), 64), (32, False, (31,), 100), (5, False, (), 7),
    (256, True, (), 500), (256, False, (255, 0), 129), (4, True, (0, 1, 2, 3), 9),
    (2, False, (), 2)])
@pytest.mark.parametrize("hub", [0, 900])
def test_bias(buckets, bidirectional, shut, far, dtype, hub, device):
    """The learned bias and its gradient, shut buckets (all of them: every row is empty)."""
    N = 90
    t = make(N, 800, 3, 16, 32, dtype, device, seed=buckets, hub=hub, buckets=buckets,
             bidirectional=bidirectional, shut=shut, far=far)
    got, want = run(t, graph_of(t, N, device)), expect(t, N)
    check_all(got, want)
    if len(shut) == buckets:
        assert all(not bool(x.any()) for x in got.values())


@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_behind_a_shut_edge_counts(dtype, device):
    """NaN and inf in the keys and values that only shut edges point at leave no trace."""
    N, H, d, dv = 60, 2, 16, 32
    t = make(N, 700, H, d, dv, dtype, device, seed=5, buckets=4, bidirectional=False, shut=(3,),
             far=4)
    # sources 0..9 far behind every destination: their edges fall into the shut bucket
    t["positions"][:10] = -1000
    t["positions"][10:] = 0
    keep = t["dst"] >= 10
    t["src"], t["dst"] = t["src"][keep], t["dst"][keep]
    want = expect(t, N)
    for n in ("k", "v"):
        t[n][:10] = float("nan")
        t[n][3] = float("inf")
    got = run(t, graph_of(t, N, device))
    for n in want:
        ref.check(got[n], want[n], n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lowest_bias_is_not_a_mask(dtype, device):
    """A bias of the type's lowest value keeps a row alive where it has nothing else: the logits
    vanish beside it, so the row's edges share it evenly."""
    from gatx import diff_attention
    N, H = 12, 1
    t = make(N, 100, H, 8, 8, dtype, device, seed=6, buckets=2, bidirectional=False, far=2)
    t["positions"][:] = 0
    t["bias"][0] = torch.finfo(torch.float32).min
    t["lam"][:] = 0.25
    g = graph_of(t, N, device)
    got = diff_attention(t["q"], t["k"], t["v"], t["lam"], g, bias=t["bias"],
                         positions=t["positions"], **t["kw"]).double().cpu()
    v, n = t["v"].double().cpu(), torch.bincount(t["dst"], minlength=N).clamp(min=1).view(-1, 1, 1)
    mean = torch.zeros(N, H, 8, dtype=torch.float64).index_add_(0, t["dst"], v[t["src"]]) / n
    mag = torch.zeros(N, H, 8, dtype=torch.float64).index_add_(0, t["dst"], v[t["src"]].abs()) / n
    limit = ref.half_step(dtype) * 0.75 * mean.abs() + ref.U32 * (4 * n + 64) * 1.25 * mag
    assert ((got - 0.75 * mean).abs() <= limit * (1 + ref.half_step(dtype))).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [1, 2, 37, 64])
@pytest.mark.parametrize("d,dv,buckets", [(8, 16, 0), (7, 13, 16), (64, 128, 0)])
def test_serving_rows(M, d, dv, buckets, dtype, device):
    """nodes=: the rows asked for alone, from rows without edges to one of 3000, whichever way
    their edges are split; the same node twice is answered twice."""
    from gatx import diff_attention
    N = 64
    t = make(N, 800, 3, d, dv, dtype, device, seed=M, hub=3000, buckets=buckets)
    g = graph_of(t, N, device)
    nodes = torch.randperm(N, generator=torch.Generator().manual_seed(M))[:M]
    want = expect({**t, "q": t["q"][nodes]}, N, nodes=nodes, grads=False)["out"]
    kw = dict(t["kw"])
    if buckets:
        kw.update(bias=t["bias"], positions=t["positions"])
    with torch.no_grad():
        got = diff_attention(t["q"][nodes], t["k"], t["v"], t["lam"], g, nodes=nodes.to(device),
                             **kw)
        ref.check(got, want, "rows")
        twice = torch.cat([nodes, nodes]).to(device, torch.int32)
        again = diff_attention(t["q"][twice.long()], t["k"], t["v"], t["lam"], g, nodes=twice,
                               **kw)
    ref.check(again, tuple(torch.cat([x, x]) for x in want), "twice")


def test_serving_unknown_nodes_give_nan(device):
    """Ids outside the graph: NaN rows, and nothing is read there; their neighbours are whole."""
    from gatx import diff_attention
    N = 20
    t = make(N, 100, 2, 8, 16, torch.float32, device, buckets=4, bidirectional=False, far=9)
    g = graph_of(t, N, device)
    for M in (3, 300):
        nodes = torch.full((M,), 4)
        nodes[0], nodes[2] = -1, N
        with torch.no_grad():
            got = diff_attention(t["q"][nodes.clamp(0, N - 1)], t["k"], t["v"], t["lam"], g,
                                 nodes=nodes.to(device), bias=t["bias"],
                                 positions=t["positions"], **t["kw"])
        assert got[0].isnan().all() and got[2].isnan().all()
        want = expect({**t, "q": t["q"][[4]]}, N, nodes=torch.tensor([4]), grads=False)["out"]
        ref.check(got[1:2], want, "row 4")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,dv", [(16, 32), (7, 13)])
def test_slices_of_a_projection(d, dv, dtype, device):
    """q, k, v as column ranges of one projection's output, go expanded: the packed result's bits."""
    N, H = 50, 3
    t = make(N, 400, H, d, dv, dtype, device, seed=9)
    g = graph_of(t, N, device)
    t["go"] = torch.ones(1, 1, dv, dtype=dtype, device=device).expand(N, H, dv)
    a = run(t, g)
    wide = torch.cat([t["q"].flatten(1), t["k"].flatten(1), t["v"].flatten(1),
                      torch.ones(N, 8, dtype=dtype, device=device)], 1)
    q, k, v, _ = wide.split([2 * H * d, 2 * H * d, H * dv, 8], 1)
    s = {**t, "q": q.unflatten(1, (H, 2, d)), "k": k.unflatten(1, (H, 2, d)),
         "v": v.unflatten(1, (H, dv))}
    b = run(s, g)
    s["q"] = t["q"].transpose(1, 2).contiguous().transpose(1, 2)   # heads not packed
    c = run(s, g)
    for n in a:
        assert torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]), n


def test_same_bits_every_time(device):
    t = make(3000, 60000, 4, 32, 64, torch.bfloat16, device, hub=2000, buckets=32)
    g = graph_of(t, 3000, device)
    a, b = run(t, g), run(t, g)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_some_gradients_only(device):
    """Each gradient alone has the bits it has among the others."""
    from gatx import diff_attention
    N = 80
    t = make(N, 500, 2, 16, 32, torch.float32, device, hub=700, buckets=8)
    g = graph_of(t, N, device)
    every = run(t, g)
    for n in ("q", "k", "v", "lam", "bias"):
        x = {m: t[m].detach().requires_grad_(m == n) for m in ("q", "k", "v", "lam", "bias")}
        out = diff_attention(x["q"], x["k"], x["v"], x["lam"], g, bias=x["bias"],
                             positions=t["positions"], **t["kw"])
        got, = torch.autograd.grad(out, x[n], t["go"])
        assert torch.equal(got, every[n]), n


def test_gradients_against_differences(device):
    """Along random directions, the kernels' float32 gradients against central differences of the
    float64 definition. Step h: the difference is off by h^2 / 6 times a third derivative; at
    h = 1e-4 that and the gradients' own bounds are far below 1e-3 of the direction's length
    times the gradient's."""
    N = 40
    t = make(N, 300, 2, 8, 12, torch.float32, device, seed=11, buckets=8)
    g = graph_of(t, N, device)
    got = run(t, g)
    go = t["go"].double().cpu()
    for n in ("q", "k", "v", "lam", "bias"):
        u = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(1)).double()
        base, h = t[n].double().cpu(), 1e-4

        def f(x):
            return float((expect({**t, n: x}, N, grads=False)["out"][0] * go).sum())
        want = (f(base + h * u) - f(base - h * u)) / (2 * h)
        grad = got[n].double().cpu()
        assert abs(float((grad * u).sum()) - want) <= 1e-3 * float(grad.norm() * u.norm()), n


def test_other_stream_and_replayed_capture(device):
    """On a side stream and as a replayed hipGraph (forward and backward, new inputs between the
    replays): the eager bits."""
    from gatx import diff_attention
    N = 200
    t = make(N, 3000, 2, 16, 32, torch.bfloat16, device, hub=900, buckets=8)
    g = graph_of(t, N, device)
    want = run(t, g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(t, g)
    s.synchronize()
    for n in want:
        assert torch.equal(want[n], got[n]), n
    x = {n: t[n].clone().requires_grad_(True) for n in ("q", "k", "v", "lam", "bias")}

    def step():
        out = diff_attention(x["q"], x["k"], x["v"], x["lam"], g, bias=x["bias"],
                             positions=t["positions"], **t["kw"])
        return [out.detach()] + list(torch.autograd.grad(out, list(x.values()), t["go"]))
    from gatx.capture import CapturedStep
    cap = CapturedStep(step)
    for i in range(3):
        new = make(N, 3000, 2, 16, 32, torch.bfloat16, device, seed=20 + i, hub=900, buckets=8)
        with torch.no_grad():
            for n in x:
                x[n].copy_(new[n])
        got = [y.clone() for y in cap()]
        torch.cuda.synchronize()
        want = run({**t, **{n: x[n] for n in x}}, g)
        for a, n in zip(got, ["out"] + list(x)):
            assert torch.equal(a, want[n]), (i, n)


def test_graph_with_self_loops_and_padding(device):
    """A graph whose edge_index' is shorter than its allocation (dropped self-loops)."""
    from gatx.graph import Graph
    N = 30
    t = make(N, 200, 2, 8, 8, torch.float32, device, seed=13, buckets=8)
    t["src"][:40] = t["dst"][:40]
    g = Graph(torch.stack([t["src"], t["dst"]]).to(device), N, True)
    ei = g.edge_index.cpu()
    got = run(t, g)
    t["src"], t["dst"] = ei[0], ei[1]
    check_all(got, expect(t, N))


def test_layer(device):
    """DiffAttention: shapes, the function's own values, gradients for every parameter."""
    from gatx import DiffAttention, diff_attention
    from gatx.graph import Graph
    torch.manual_seed(0)
    N, H, F = 40, 3, 16
    layer = DiffAttention(20, F, H, add_self_loops=True, position_buckets=8).to(device)
    ei = torch.randint(0, N, (2, 200), device=device)
    pos = torch.arange(N, device=device)
    x = torch.randn(N, 20, device=device)
    out = layer(x, ei, pos)
    assert out.shape == (N, H * F)
    g = Graph(ei, N, True)
    q, k, v = layer.qkv(x).split([H * F, H * F, H * F], 1)
    same = diff_attention(q.view(N, H, 2, F // 2), k.view(N, H, 2, F // 2), v.view(N, H, F),
                          layer.lam, g, bias=layer.position_bias, positions=pos)
    assert torch.equal(out, same.reshape(N, H * F))
    out.square().sum().backward()
    for n, p in layer.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0, n
    with pytest.raises(ValueError, match="positions"):
        layer(x, ei)


def test_serving_refuses_gradients(device):
    from gatx import diff_attention
    t = make(20, 50, 1, 8, 8, torch.float32, device)
    g = graph_of(t, 20, device)
    q = t["q"][:2].requires_grad_(True)
    with pytest.raises(RuntimeError, match="no_grad"):
        diff_attention(q, t["k"], t["v"], t["lam"], g,
                       nodes=torch.tensor([0, 1], device=device))


def test_second_derivative_is_refused(device):
    t = make(20, 50, 1, 8, 8, torch.float32, device)
    g = graph_of(t, 20, device)
    from gatx import diff_attention
    q = t["q"].requires_grad_(True)
    out = diff_attention(q, t["k"], t["v"], t["lam"], g)
    gq, = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        gq.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [1, 2, 5, 70])
@pytest.mark.parametrize("H,d,dv", [(1, 1, 1), (3, 7, 5), (2, 8, 16), (1, 9, 8), (3, 61, 121),
                                    (1, 250, 3)])
def test_queries_read_where_they_are(H, d, dv, N, dtype, device):
    """Without gradients q is not repacked: rows of any width and alignment up to the last element
    of their memory, what lies between them never let in."""
    from gatx import diff_attention
    t = make(N, 9 * N, H, d, dv, dtype, device, seed=N + d)
    graph, want = graph_of(t, N, device), expect(t, N, grads=False)["out"]
    n = 2 * H * d
    fused = torch.full((N, n + 3), float("nan"), dtype=dtype, device=device)
    fused[:, 3:] = t["q"].reshape(N, n)
    nodes = torch.arange(N - 1, -1, -1, device=device)
    with torch.no_grad():
        for q in (t["q"], fused[:, 3:].unflatten(1, (H, 2, d))):
            ref.check(diff_attention(q, t["k"], t["v"], t["lam"], graph), want, "out")
            served = diff_attention(q[nodes], t["k"], t["v"], t["lam"], graph, nodes=nodes)
            ref.check(served, tuple(x[nodes.cpu()] for x in want), "served")
        q = t["q"][:1].expand(N, H, 2, d)   # one row for all of them
        same = {**t, "q": q}
        ref.check(diff_attention(q, t["k"], t["v"], t["lam"], graph),
                  expect(same, N, grads=False)["out"], "expanded")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,d,dv", [(1, 8, 8), (2, 9, 15), (3, 61, 121), (1, 250, 509), (2, 16, 17),
                                    (4, 17, 16), (2, 7, 12), (2, 12, 7)])
@pytest.mark.parametrize("hub", [0, 3000])
def test_serving_reads_keys_and_values_where_they_are(H, d, dv, hub, dtype, device):
    """Any width and alignment, NaN between the rows; one piece a row and many."""
    from gatx import diff_attention
    N = 50
    t = make(N, 300, H, d, dv, dtype, device, seed=d + hub, hub=hub)
    graph = graph_of(t, N, device)
    nodes = torch.tensor([0, N - 1, 7, 7, 1], device=device)
    want = expect(t, N, grads=False)["out"]
    want = tuple(x[nodes.cpu()] for x in want)
    nk, nv = 2 * H * d, H * dv
    fused = torch.full((N, 1 + nk + 1 + nv), float("nan"), dtype=dtype, device=device)
    fused[:, 1:1 + nk] = t["k"].reshape(N, nk)
    fused[:, 2 + nk:] = t["v"].reshape(N, nv)
    k, v = fused[:, 1:1 + nk].unflatten(1, (H, 2, d)), fused[:, 2 + nk:].unflatten(1, (H, dv))
    with torch.no_grad():
        for kk, vv in ((t["k"], t["v"]), (k, v)):
            got = diff_attention(t["q"][nodes], kk, vv, t["lam"], graph, nodes=nodes)
            ref.check(got, want, "served")


@pytest.mark.parametrize("N,E", [(1, 0), (2047, 9000), (2048, 0), (2049, 60000), (6000, 40000)])
def test_rows_by_length(N, E, device):
    """A stable sort of every 2048 rows by pairs of edges (1022 and more alike), longest first."""
    from gatx._lib import call, ptr, stream
    t = make(N, E, 1, 8, 8, torch.float32, device, seed=N, hub=1500 if N == 6000 else 0)
    graph = graph_of(t, N, device)
    order = torch.full((N, 4), -1, dtype=torch.int32, device=device)
    call("gatx_diff_attention_row_order", ptr(graph.rowptr), N, ptr(order), stream())
    rowptr = graph.rowptr.cpu().long()
    length = rowptr[1:] - rowptr[:-1]
    key = ((length + 1) // 2).clamp(max=511)
    rows = torch.cat([c[torch.sort(key[c], descending=True, stable=True).indices]
                      for c in torch.arange(N).split(2048)])
    assert torch.equal(order.cpu().long(), torch.stack(
        [rows, rowptr[:-1][rows], length[rows], torch.zeros(N, dtype=torch.int64)], 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,dv", [(16, 24), (8, 300)])
def test_row_order_changes_no_bit(d, dv, dtype, device, monkeypatch):
    from gatx import attention
    N, H = 3000, 6
    t = make(N, 30000, H, d, dv, dtype, device, seed=8, hub=2000, buckets=8)
    assert N * H >= attention._ORDER_ITEMS
    a = run(t, graph_of(t, N, device))
    monkeypatch.setattr(attention, "_ORDER_ITEMS", 1 << 40)
    b = run(t, graph_of(t, N, device))
    check_all(a, expect(t, N))
    for n in a:
        assert torch.equal(a[n], b[n]), n

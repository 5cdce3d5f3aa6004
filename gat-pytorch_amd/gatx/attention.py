"""Differential attention over a graph's in-neighbourhoods, with a learned relative position bias
(csrc/diff_attn.hip): the dot-product counterpart of gatx.functional's additive GAT attention, on
the same gatx.Graph. Each head attends with two softmax maps and subtracts one from the other, so
what both maps give to irrelevant neighbours cancels:

    x_m[e, h] = scale q[i, h, m] . k[j, h, m] + bias[bucket(positions[j] - positions[i]), h]
    out[i, h] = sum over edges e = j -> i of (p_1 - lam[h] p_2) v[j, h],   p_m = softmax over them

float32, bfloat16 and float16; sums, softmax statistics and the gradients of lam and bias are
float32. There is no CPU path."""
from __future__ import annotations

import math

import torch
from torch import nn

from . import tuning
from ._lib import DTYPES, call, host as _host, on_device, ptr, stream, untraced
from .graph import Graph, graph_cache

MAX_HEAD_WIDTH = 256    # d
MAX_VALUE_WIDTH = 512   # dv
MAX_BUCKETS = 256

# waves a call for a few nodes is split into: enough loads in flight to fill the memory system
_SERVING_WAVES = 2048


def bucket_bounds(num_buckets: int, max_distance: int, bidirectional: bool):
    """(exact, bounds) of the position buckets: `exact` distances with a bucket each, then bucket
    exact + j from the distance bounds[j - 1] on. With n buckets a side and m = n // 2 exact ones,
    that bound is the smallest distance >= m (max_distance / m)^(j / (n - m)), found in whole
    numbers, so no distance lands on the wrong side of one by a rounding."""
    if bidirectional and num_buckets % 2:
        raise ValueError("gatx: a bidirectional bias needs an even number of buckets")
    n = num_buckets // 2 if bidirectional else num_buckets
    if n < 2 or num_buckets > MAX_BUCKETS:
        raise ValueError(f"gatx: {num_buckets} position buckets (2 a side to {MAX_BUCKETS} in all)")
    m = n // 2
    if not m < max_distance < 2 ** 62:
        raise ValueError(f"gatx: max_distance must exceed the {m} exact buckets of a side, got "
                         f"{max_distance}")
    bounds = []
    for j in range(1, n - m):
        # the smallest x with x^(n-m) >= m^(n-m-j) max_distance^j
        want = m ** (n - m - j) * max_distance ** j
        lo, hi = m, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** (n - m) >= want:
                hi = mid
            else:
                lo = mid + 1
        bounds.append(lo)
    return m, bounds


_BOUNDS: dict = {}


def _bounds(num_buckets, max_distance, bidirectional):
    """bucket_bounds, kept by its three numbers (the search is in whole numbers of any size)."""
    key = (num_buckets, max_distance, bidirectional)
    hit = _BOUNDS.get(key)
    if hit is None:
        hit = _BOUNDS[key] = bucket_bounds(num_buckets, max_distance, bidirectional)
        while len(_BOUNDS) > 64:
            _BOUNDS.pop(next(iter(_BOUNDS)))
    return hit


def _needs(graph: Graph, built: bool, what: str):
    """A captured step must not be the first to build what an eager-built graph keeps: it would
    only be filled by a replay, and eager calls would read it before."""
    if not built and graph._event is not None and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"gatx: the graph's {what} must exist before a capture (run the step "
                           "once eagerly)")


def _transpose(graph: Graph):
    _needs(graph, graph.srowptr is not None, "transpose")
    graph._ensure_transpose()
    return graph.srowptr, graph.scol, graph.seid


# rows x heads from which rows share a wave
_ORDER_ITEMS = 8192


def _row_order(graph: Graph, heads: int, source: bool):
    """The rows by length (csrc/diff_attn.hip, row_order_kernel), for rows that share waves. No
    result depends on it, so a capture that finds none goes without."""
    if graph.num_nodes * heads < _ORDER_ITEMS:
        return None
    key = ("order", source)
    if (key not in graph._hub_plans and graph._event is not None
            and torch.cuda.is_current_stream_capturing()):
        return None

    def build():
        order = torch.empty((graph.num_nodes, 4), dtype=torch.int32, device=graph.device)
        call("gatx_diff_attention_row_order", ptr(graph.srowptr if source else graph.rowptr),
             graph.num_nodes, ptr(order), stream())
        return (order,)
    return graph._kept(key, build)[0]


_NO_PLAN = (0, None, None, 0)


def _plan(graph: Graph, heads: int, source: bool):
    return _hub_plan(graph, source) + (_row_order(graph, heads, source),)


def _hub_plan(graph: Graph, source: bool):
    """(edges, entries, count, bound) of the pieces of long rows; no plan once it is known that the
    graph has none (its count is copied to the host when the plan is built and looked at when it
    has arrived, so nothing waits; until then, and inside a first capture, the pieces' launches
    find nothing to do)."""
    T = tuning.get("attn_hub_edges")
    if T <= 0 or graph.edge_bound <= T:
        return _NO_PLAN
    plans, key = graph._hub_plans, (T, source, "entries")
    known = plans.get(key)
    if known == 0:
        return _NO_PLAN
    _needs(graph, (T, source) in plans, "hub plan")
    hubs, count, bound = graph.hub_plan(T, source)
    if not torch.cuda.is_current_stream_capturing():
        if known is None:
            # a graph built inside a capture has its counts only after a replay: never read
            if graph._event is not None:
                host = torch.empty(1, dtype=torch.int32, pin_memory=True)
                host.copy_(count, non_blocking=True)
                event = torch.cuda.Event()
                event.record()
                plans[key] = (host, event)
        elif not isinstance(known, int) and known[1].query():
            plans[key] = int(known[0])
            if plans[key] == 0:
                return _NO_PLAN
    return T, hubs, count, bound


def _check(q, k, v, lam, graph, bias, positions, nodes):
    if not isinstance(graph, Graph):
        raise TypeError("gatx: diff_attention needs a gatx.Graph (Graph(edge_index, num_nodes, "
                        "add_self_loops))")
    named = [("q", q), ("k", k), ("v", v), ("lam", lam), ("bias", bias),
             ("positions", positions), ("nodes", nodes)]
    for name, t in named:
        if t is not None and t.device != graph.device:
            raise RuntimeError(f"gatx: diff_attention: {name} is on {t.device}, the graph on "
                               f"{graph.device} (no CPU path)")
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("gatx: diff_attention: q, k, v must share one of float32, bfloat16, "
                           f"float16, got {q.dtype}, {k.dtype}, {v.dtype}")
    if q.dim() != 4 or q.size(2) != 2 or k.dim() != 4 or v.dim() != 3:
        raise ValueError("gatx: diff_attention: q and k are (rows, heads, 2, d), v (nodes, heads, "
                         f"dv), got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    N, H, d, dv = graph.num_nodes, q.size(1), q.size(3), v.size(2)
    rows = N if nodes is None else nodes.numel()
    if (q.size(0) != rows or tuple(k.shape) != (N, H, 2, d) or tuple(v.shape[:2]) != (N, H)):
        raise ValueError(f"gatx: diff_attention: {rows} rows of q and {N} of k and v expected, "
                         f"with the same heads and widths, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if H < 1 or not (1 <= d <= MAX_HEAD_WIDTH and 1 <= dv <= MAX_VALUE_WIDTH):
        raise ValueError(f"gatx: diff_attention: {H} heads of d = {d} (1 to {MAX_HEAD_WIDTH}) "
                         f"and dv = {dv} (1 to {MAX_VALUE_WIDTH})")
    if tuple(lam.shape) != (H,) or not lam.is_floating_point():
        raise ValueError(f"gatx: diff_attention: lam is one number a head, got {tuple(lam.shape)}")
    if (bias is None) != (positions is None):
        raise ValueError("gatx: diff_attention: bias and positions go together")
    if bias is not None:
        if bias.dim() != 2 or bias.size(1) != H or not bias.is_floating_point():
            raise ValueError(f"gatx: diff_attention: bias is (buckets, {H}), got "
                             f"{tuple(bias.shape)}")
        if tuple(positions.shape) != (N,) or positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"gatx: diff_attention: positions are {N} int32 or int64, got "
                             f"{tuple(positions.shape)} {positions.dtype}")
    if nodes is not None and (nodes.dim() != 1 or nodes.dtype not in (torch.int32, torch.int64)):
        raise ValueError("gatx: diff_attention: nodes is a 1-D int32 or int64 tensor")


@untraced
def diff_attention(q, k, v, lam, graph: Graph, *, scale=None, bias=None, positions=None,
                   max_distance: int = 128, bidirectional: bool = True, nodes=None):
    """Differential attention of every node over its in-neighbours in `graph`.

    q, k: (N, H, 2, d) (both maps' queries and keys), v: (N, H, dv), one dtype; slices of a fused
    projection are read in place where their rows are 16-byte aligned and d, dv multiples of 8, and
    packed in one launch otherwise (with nodes: read as they are, but for widths below 8).
    lam: (H,). scale: 1 / sqrt(d) unless given. Returns (N, H, dv). A node without in-edges (or with
    every one of them shut) gets zeros.

    bias (num_buckets, H) with positions (N,): a learned bias by the bucket of positions[source] -
    positions[destination]: half of a side's buckets one distance each, the others log-spaced up to
    max_distance and the last one open (bucket_bounds); bidirectional: the second half of the
    buckets for sources ahead of their destination, else those all count as distance 0. An entry
    of -inf shuts its bucket: nothing behind it is attended to.

    nodes (M,): only these nodes' rows are computed (q is (M, H, 2, d), the result (M, H, dv)), k and
    v still every node's: the serving form, where the others' keys and values are kept. Without
    gradients. Ids outside the graph give rows of NaN.

    Gradients: q, k, v, lam, bias, once differentiable, the same bits every time."""
    _check(q, k, v, lam, graph, bias, positions, nodes)
    graph._poll()
    scale = 1.0 / math.sqrt(q.size(3)) if scale is None else float(scale)
    exact, bounds = (0, []) if bias is None else _bounds(bias.size(0), int(max_distance),
                                                         bool(bidirectional))
    grad = torch.is_grad_enabled()
    args = (q, k, v, lam, bias, positions, exact, bounds, bool(bidirectional), scale, graph.rowptr,
            graph.col, graph.rowidx, graph.num_nodes, graph.edge_bound)
    if nodes is not None:
        if grad and any(t is not None and t.requires_grad for t in (q, k, v, lam, bias)):
            raise RuntimeError("gatx: diff_attention(nodes=...) has no gradients: call it under "
                               "torch.no_grad()")
        items = max(1, nodes.numel() * q.size(1))
        pieces = max(1, min(_SERVING_WAVES // items, 256, -(-graph.edge_bound // 256)))
        return _host.diff_attention_nodes(*args, nodes, pieces)
    with on_device(graph.device):   # (the graph's own launches)
        transpose, src_plan = (None, None, None), _NO_PLAN + (None,)
        if grad and (k.requires_grad or v.requires_grad):
            transpose = _transpose(graph)
            src_plan = _plan(graph, q.size(1), True)
        return _host.diff_attention(*args, _plan(graph, q.size(1), False), *transpose, src_plan)


class DiffAttention(nn.Module):
    """A differential attention layer on a graph: one projection to q, k and v, diff_attention, the
    heads side by side: (N, in_features) -> (N, num_heads * out_features). Beside GATLayer, with the
    same edge_index and self-loop handling; position_buckets > 0 adds the learned position bias
    (forward then takes the nodes' positions). lam starts at lambda_init in every head."""

    def __init__(self, in_features, out_features, num_heads, add_self_loops=False,
                 lambda_init=0.8, position_buckets=0, max_distance=128, bidirectional=True):
        super().__init__()
        self.in_features, self.out_features, self.num_heads = in_features, out_features, num_heads
        self.add_self_loops = add_self_loops
        self.lambda_init = lambda_init
        self.max_distance, self.bidirectional = max_distance, bidirectional
        # the two maps share a head's width between them
        self.map_features = max(1, out_features // 2)
        self.qkv = nn.Linear(in_features, num_heads * (4 * self.map_features + out_features),
                             bias=False)
        self.lam = nn.Parameter(torch.empty(num_heads))
        if position_buckets:
            bucket_bounds(position_buckets, max_distance, bidirectional)   # raises on bad ones
            self.position_bias = nn.Parameter(torch.empty(position_buckets, num_heads))
        else:
            self.register_parameter("position_bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.xavier_uniform_(self.qkv.weight)
        nn.init.constant_(self.lam, self.lambda_init)
        if self.position_bias is not None:
            nn.init.zeros_(self.position_bias)

    def forward(self, x, edge_index=None, positions=None, *, graph=None):
        """edge_index (2, E), or a prebuilt gatx.Graph as graph=."""
        if graph is None:
            graph = graph_cache.get(edge_index, x.size(0), self.add_self_loops)
        N, H, d = x.size(0), self.num_heads, self.map_features
        q, k, v = self.qkv(x).split([2 * H * d, 2 * H * d, H * self.out_features], dim=1)
        kw = {}
        if self.position_bias is not None:
            if positions is None:
                raise ValueError("gatx: DiffAttention with position_buckets needs positions")
            kw = dict(bias=self.position_bias, positions=positions,
                      max_distance=self.max_distance, bidirectional=self.bidirectional)
        out = diff_attention(q.unflatten(1, (H, 2, d)), k.unflatten(1, (H, 2, d)),
                             v.unflatten(1, (H, self.out_features)), self.lam, graph, **kw)
        return out.reshape(N, H * self.out_features)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"num_heads={self.num_heads}, add_self_loops={self.add_self_loops}")

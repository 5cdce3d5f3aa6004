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
from torch.autograd.function import once_differentiable

from . import tuning
from ._lib import DTYPES, call, lib, on_device, ptr, stream
from .functional import _span
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


def _bounds_array(num_buckets, max_distance, bidirectional):
    """bucket_bounds as the host array of a launch (a pure function of its three numbers)."""
    import ctypes
    key = (num_buckets, max_distance, bidirectional)
    hit = _BOUNDS.get(key)
    if hit is None:
        m, b = bucket_bounds(num_buckets, max_distance, bidirectional)
        hit = _BOUNDS[key] = (m, (ctypes.c_int64 * max(len(b), 1))(*b), len(b))
        while len(_BOUNDS) > 64:
            _BOUNDS.pop(next(iter(_BOUNDS)))
    return hit


def _buckets(graph: Graph, positions, num_buckets, max_distance, bidirectional, nodes):
    import ctypes
    m, bounds, n = _bounds_array(num_buckets, max_distance, bool(bidirectional))
    bucket = torch.empty(max(graph.edge_bound, 1), dtype=torch.uint8, device=graph.device)
    call("gatx_relative_buckets", ptr(graph.rowptr), ptr(graph.col), ptr(graph.rowidx),
         graph.edge_bound, graph.num_nodes, ptr(nodes), 0 if nodes is None else nodes.numel(),
         ptr(positions), int(positions.dtype == torch.int64), m,
         ctypes.addressof(bounds), n, int(bool(bidirectional)), ptr(bucket), stream())
    return bucket


def _rows(t: torch.Tensor):
    """(tensor, row stride) with each row's heads packed: the tensor itself where only its rows
    are strided (a slice of a fused projection's output), else a packed copy."""
    want = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != want:
            t = t.contiguous()
            return t, t.stride(0)
        want *= size
    return t, (t.stride(0) if t.size(0) > 1 else want)


def _chunked(t, ld, width) -> bool:
    """Whether the kernels read these rows as they are: 8-element chunks, 16-byte aligned."""
    return width % 8 == 0 and t.data_ptr() % 16 == 0 and ld * t.element_size() % 16 == 0


def _pack(dtype, H, d, dv, q=None, k=None, v=None):
    """[(tensor, row stride)] of q, k, v (None: absent) in the kernels' layout, one launch for those
    that are not yet."""
    given = [None if t is None else _rows(t) for t in (q, k, v)]
    out, args, any_packed = [], [], False
    rows = keys = 0
    for i, (pair, width, groups) in enumerate(zip(given, (d, d, dv), (2 * H, 2 * H, H))):
        if pair is None or _chunked(*pair, width):
            out.append(pair)
            args += [None, 0, None]
            continue
        t, ld = pair
        p = torch.empty((t.size(0), groups, -(-width // 8) * 8), dtype=t.dtype, device=t.device)
        out.append((p, p.stride(0)))
        args += [ptr(t), ld, ptr(p)]
        any_packed = True
        if i == 0:
            rows = t.size(0)
        else:
            keys = t.size(0)
    if any_packed:
        call("gatx_diff_attention_pack", dtype, rows, keys, H, d, dv, *args, stream())
    return out


def _needs(graph: Graph, built: bool, what: str):
    """A captured step must not be the first to build what an eager-built graph keeps: it would
    only be filled by a replay, and eager calls would read it before."""
    if not built and graph._event is not None and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"gatx: the graph's {what} must exist before a capture (run the step "
                           "once eagerly)")


def _hub_args(graph: Graph, source: bool):
    """(edges, plan, count, bound) of the pieces of long rows."""
    T = tuning.get("attn_hub_edges")
    if T <= 0 or graph.edge_bound <= T:
        return 0, None, None, 0
    _needs(graph, (T, source) in graph._hub_plans, "hub plan")
    hubs, count, bound = graph.hub_plan(T, source)
    return T, ptr(hubs), ptr(count), bound


class DiffAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, bias, graph: Graph, scale: float, bucket, nodes, pieces: int):
        dt, dev = DTYPES[q.dtype], q.device
        M, H, _, d = q.shape
        dv = v.size(2)
        lam = lam.contiguous()
        bias = None if bias is None else bias.contiguous()
        (qp, ldq), (kp, ldk), (vp, ldv) = _pack(dt, H, d, dv, q, k, v)
        out = torch.empty((M, H, dv), dtype=q.dtype, device=dev)
        E, N = graph.edge_bound, graph.num_nodes
        if nodes is None:
            S = torch.empty((H, max(E, 1), 2), dtype=torch.float32, device=dev)
            stat = torch.empty((H, N, 4), dtype=torch.float32, device=dev)
            hub = _hub_args(graph, False)
            slots = hub[3]
        else:
            S = stat = None
            hub = (0, None, None, 0)
            slots = M * pieces if pieces > 1 else 0
        nb = lib.gatx_diff_attention_part_bytes(slots, H, -(-dv // 8) * 8)
        part = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        with _span("diff_attention", (M, E, H, d, dv)):
            call("gatx_diff_attention", dt, ptr(qp), ldq, ptr(kp), ldk, ptr(vp), ldv, H, d, dv,
                 ptr(graph.rowptr), ptr(graph.col), E, M, N, ptr(nodes), pieces, scale, ptr(lam),
                 ptr(bias), ptr(bucket), ptr(out), ptr(S), ptr(stat), *hub, ptr(part), nb,
                 stream())
        if any(ctx.needs_input_grad[:5]):
            ctx.save_for_backward(qp, kp, vp, lam, bias, bucket, S, stat)
            ctx.graph, ctx.scale, ctx.lds, ctx.dims = graph, scale, (ldq, ldk, ldv), (H, d, dv)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        qp, kp, vp, lam, bias, bucket, S, stat = ctx.saved_tensors
        graph, (H, d, dv), (ldq, ldk, ldv) = ctx.graph, ctx.dims, ctx.lds
        N, E, dev, dtype = graph.num_nodes, graph.edge_bound, qp.device, qp.dtype
        dt = DTYPES[dtype]
        need_q, need_k, need_v, need_lam, need_bias = ctx.needs_input_grad[:5]
        with on_device(dev):
            gop, ldgo = _pack(dt, H, d, dv, v=go)[2]
            gq = torch.empty((N, H, 2, d), dtype=dtype, device=dev) if need_q else None
            gk = torch.empty((N, H, 2, d), dtype=dtype, device=dev) if need_k else None
            gv = torch.empty((N, H, dv), dtype=dtype, device=dev) if need_v else None
            glam = torch.empty(H, dtype=torch.float32, device=dev) if need_lam else None
            nb = bias.size(0) if need_bias else 0
            gbias = torch.empty((nb, H), dtype=torch.float32, device=dev) if need_bias else None
            hub = _hub_args(graph, False)
            src_hub, T = (None, None, 0), (None, None, None)
            if need_k or need_v:
                _needs(graph, graph.srowptr is not None, "transpose")
                graph.ensure_transpose()
                src_hub = _hub_args(graph, True)[1:]
                T = (ptr(graph.srowptr), ptr(graph.scol), ptr(graph.seid))
            wb = lib.gatx_diff_attention_backward_workspace_bytes(N, E, H, d, dv, nb, hub[3],
                                                                  src_hub[2])
            ws = torch.empty(wb, dtype=torch.uint8, device=dev)
            with _span("diff_attention_bwd", (N, E, H, d, dv)):
                call("gatx_diff_attention_backward", dt, ptr(qp), ldq, ptr(kp), ldk, ptr(vp), ldv,
                     ptr(gop), ldgo, H, d, dv, ptr(graph.rowptr), ptr(graph.col), *T, E, N,
                     ctx.scale, ptr(lam), ptr(bucket), nb, ptr(S), ptr(stat), ptr(gq), ptr(gk),
                     ptr(gv), ptr(glam), ptr(gbias), *hub, *src_hub, ptr(ws), wb, stream())
        return gq, gk, gv, glam, gbias, None, None, None, None, None


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


def diff_attention(q, k, v, lam, graph: Graph, *, scale=None, bias=None, positions=None,
                   max_distance: int = 128, bidirectional: bool = True, nodes=None):
    """Differential attention of every node over its in-neighbours in `graph`.

    q, k: (N, H, 2, d) (both maps' queries and keys), v: (N, H, dv), one dtype; slices of a fused
    projection are read in place where their rows are 16-byte aligned and d, dv multiples of 8.
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
    graph.poll()
    scale = 1.0 / math.sqrt(q.size(3)) if scale is None else float(scale)
    pieces = 1
    if nodes is not None:
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                           for t in (q, k, v, lam, bias)):
            raise RuntimeError("gatx: diff_attention(nodes=...) has no gradients: call it under "
                               "torch.no_grad()")
        nodes = nodes.to(torch.int64).contiguous()
        items = max(1, nodes.numel() * q.size(1))
        pieces = max(1, min(_SERVING_WAVES // items, 256, -(-graph.edge_bound // 256)))
    with on_device(graph.device):
        bucket = None
        if bias is not None:
            bucket = _buckets(graph, positions.contiguous(), bias.size(0), int(max_distance),
                              bidirectional, nodes)
        return DiffAttentionFunction.apply(
            q, k, v, lam.float(), None if bias is None else bias.float(), graph, scale, bucket,
            nodes, pieces)


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

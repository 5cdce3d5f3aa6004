"""Device-side graph preprocessing for the GAT layer: the self-loop rewrite + destination CSR
(and, for the backward, the source-ordered transpose), cached per edge_index.

The reference rewrites self-loops inside every forward of every layer
(`models/gat_layer.py:53-54` -> `models/utils.py:47-67`) and then scatters/gathers by raw edge
indices. Here the rewrite and the CSR build run once per distinct edge_index on the GPU
(`gatx_graph_meta` + `gatx_graph_build`, csrc/graph.hip) and are reused by every layer and step
that sees the same tensor.

No host sync: the reference's `int(index.max())` (`models/utils.py:70-72`) sizes edge_index' on
the host; here |edge_index'| stays on the device (meta[0]) and the host allocates for the bound
E + num_nodes. The exact count is read back only when something host-side needs it — the
returned edge_index' / attention tensors (`num_edges`, `edge_index`) — so a forward that returns
only the node outputs never waits for the device, and the whole step can be captured into a
hipGraph. Invalid ids (negative, or >= num_nodes) make the device build an empty graph (nothing
indexes out of bounds) and raise here as soon as the meta is read: at the first host-side use,
at `Graph.poll()` (non-blocking, called by every layer on a cached graph) or at
`gatx.graph.check_pending()` — asynchronous error reporting, as for a device-side assert.
"""
from __future__ import annotations

import threading
import weakref
from collections import OrderedDict

import torch

from . import _lib
from ._lib import call, on_device, ptr, stream, untraced, version

_I32_LIMIT = 2 ** 31 - 2

# one thread builds what a Graph keeps at a time
_BUILDING = threading.RLock()


def _here(device) -> int:
    """`device`'s current stream."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _status_error(meta, N):
    status, mn, mx = int(meta[2]), int(meta[3]), int(meta[4])
    if status == 1:
        return RuntimeError(f"index {mn} is out of bounds: edge_index has negative node ids")
    if status == 2:
        return IndexError(f"index {mx} is out of bounds for dimension 0 with size {N}")
    return None


class Graph:
    """CSR of edge_index' (int32), plus edge_index' itself.

    rowptr [N+1], col [Eb] (source), rowidx [Eb] (destination), perm [Eb] (CSR slot -> position
    in edge_index'); srowptr / scol / seid: the source-ordered transpose, built on first use.
    Eb = `edge_bound` >= E' is the allocation; kernels read E' from `e2_ptr` (device).

    One Graph may be used on any stream: what it holds was filled on the stream that first needed
    it, and another one waits for that before its first use (follow). It is built on its edges'
    device, whichever is current."""

    @untraced
    def __init__(self, edge_index: torch.Tensor, num_nodes, add_self_loops: bool):
        """num_nodes None: size the node range from the edges (max id + 1; one host sync)."""
        if edge_index.dim() != 2 or edge_index.size(0) != 2:
            raise RuntimeError(f"edge_index must have shape (2, E), got {tuple(edge_index.shape)}")
        if edge_index.dtype not in (torch.int64, torch.int32):
            raise RuntimeError(f"edge_index must be int64 or int32, got {edge_index.dtype}")
        if not edge_index.is_cuda:
            raise RuntimeError("gatx: edge_index must be on the HIP device (no CPU path)")
        self.device = edge_index.device
        with on_device(self.device):
            self._build_csr(edge_index, num_nodes, add_self_loops)

    def _build_csr(self, edge_index, num_nodes, add_self_loops):
        dev = self.device
        if edge_index.stride(1) != 1:
            edge_index = edge_index.contiguous()
        self.add_self_loops = add_self_loops
        self.source = edge_index
        E = edge_index.size(1)
        self.num_input_edges = E
        is64 = int(edge_index.dtype == torch.int64)
        ld = edge_index.stride(0)
        if E == 0 and add_self_loops:
            # maybe_num_nodes: int(index.max()) on an empty tensor (models/utils.py:72)
            raise RuntimeError("max(): Expected reduction dim to be specified for input.numel() == 0. "
                               "Specify the reduction dim with the 'dim' argument.")
        s = stream()
        # {E2, num_loops, status, min, max, self-loops, nb, chunk} + the compaction's block
        # offsets (GATX_META_WORDS); the host only ever reads the first 8
        self.meta = torch.empty(_lib.META_WORDS, dtype=torch.int64, device=dev)
        ws = torch.empty(_lib.lib.gatx_graph_meta_workspace_bytes(), dtype=torch.uint8, device=dev)
        if num_nodes is None:   # sized by the edges themselves: the one case that must sync
            call("gatx_graph_meta", ptr(edge_index), is64, E, ld, int(add_self_loops),
                 _I32_LIMIT, ptr(self.meta), ptr(ws), s)
            m = self.meta[:8].cpu()
            err = _status_error(m, _I32_LIMIT)
            if err is not None:
                raise err
            num_nodes = int(m[4]) + 1 if E else 0
        self.num_nodes = N = int(num_nodes)
        call("gatx_graph_meta", ptr(edge_index), is64, E, ld, int(add_self_loops), N,
             ptr(self.meta), ptr(ws), s)
        Eb = E + N if add_self_loops else E
        if Eb >= 2 ** 31 - 1 or N >= 2 ** 31 - 1:
            raise RuntimeError("gatx: graphs are limited to 2^31-1 nodes / edges")
        self.edge_bound = Eb
        i32 = dict(dtype=torch.int32, device=dev)
        self.rowptr = torch.empty(N + 1, **i32)
        self.col = torch.empty(max(Eb, 1), **i32)
        self.rowidx = torch.empty(max(Eb, 1), **i32)
        self.perm = torch.empty(max(Eb, 1), **i32)
        if add_self_loops:
            self._ei_flat = torch.empty(max(2 * Eb, 2), dtype=torch.int64, device=dev)
            ei_out = ptr(self._ei_flat)
        else:
            self._ei_flat = None   # the reference returns its input unchanged
            ei_out = None
        ws_bytes = _lib.lib.gatx_graph_build_workspace_bytes(E, Eb, N)
        bws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        call("gatx_graph_build", ptr(edge_index), is64, E, ld, int(add_self_loops), N, Eb,
             ptr(self.meta), ei_out, ptr(self.rowptr), ptr(self.col), ptr(self.rowidx),
             ptr(self.perm), ptr(bws), ws_bytes, s)
        self.srowptr = self.scol = self.seid = None
        self._hub_plans = {}
        self._builds = {}
        self._E2 = None
        # |edge_index'| promised by the caller (expect_num_edges): answers num_edges without a
        # device read (so a captured step may return edge_index' / alpha); checked against the
        # device count whenever that is read
        self._E2_hint = _hint_lookup(edge_index, N, add_self_loops)
        self._error = None
        self._edge_index = None
        # non-blocking validation: the meta lands in pinned memory behind an event
        self._meta_host = None
        self._event = None
        if not torch.cuda.is_current_stream_capturing():
            self._meta_host = torch.empty(8, dtype=torch.int64, pin_memory=True)
            self._meta_host.copy_(self.meta[:8], non_blocking=True)
            self._event = torch.cuda.Event()
            self._event.record()
            self._built("csr", (self.meta, self.rowptr, self.col, self.rowidx, self.perm,
                                self._ei_flat), self._event)
            check_pending(block=False)   # surfaces errors of earlier graphs that have landed
            _PENDING.append(weakref.ref(self))

    # ---- streams
    def _built(self, key, tensors, event=None, side=None):
        """Tensors whose filling was just launched (on the current stream, or `side`), before
        anybody else can find them. Nothing to keep inside a capture: whoever replays it orders it."""
        if event is None:
            if torch.cuda.is_current_stream_capturing():
                return
            event = torch.cuda.Event()
            event.record(*(() if side is None else (side,)))
        # the stream itself is behind its launches (and behind a side stream once it has joined it)
        self._builds[key] = (event, {_here(self.device)},
                             [t for t in tensors if isinstance(t, torch.Tensor)])

    def follow(self, key="csr"):
        """The current stream behind the build of `key`, the memory kept for it. Inside a capture
        nothing is waited for: the device has caught up when one begins."""
        build = self._builds.get(key)
        if build is None:
            return
        event, streams, tensors = build
        here = _here(self.device)
        if here in streams:
            return
        with on_device(self.device):
            if torch.cuda.is_current_stream_capturing():
                return
            current = torch.cuda.current_stream()
            current.wait_event(event)
            for t in tensors:
                t.record_stream(current)
        streams.add(here)

    def _kept(self, key, build, side=None):
        """What build() launched and returned (a tuple), once a graph and key."""
        hit = self._hub_plans.get(key)
        if hit is None:
            with _BUILDING, on_device(self.device):
                hit = self._hub_plans.get(key)
                if hit is None:
                    self.follow()
                    hit = build()
                    self._built(key, hit, side=side)
                    self._hub_plans[key] = hit
        self.follow(key)
        return hit

    # ---- device-side sizes
    @property
    def e2_ptr(self) -> int:
        """Device address of |edge_index'| (int64), for the kernels' edge-count argument."""
        return ptr(self.meta)

    @property
    def ei_args(self):
        """(pointer, is64, ld) of edge_index' for gatx_attention_alpha_ei: the flat (2, E')
        buffer (ld < 0: taken from the device count) or the untouched input."""
        if self._ei_flat is not None:
            return ptr(self._ei_flat), 1, -1
        t = self.source
        return ptr(t), int(t.dtype == torch.int64), t.stride(0)

    def _validate(self, m):
        err = _status_error(m, self.num_nodes)
        if err is not None:
            self._error = err   # every later use of this graph raises it again
            raise err
        self._E2 = int(m[0])
        if self._E2_hint is not None and self._E2 != self._E2_hint:
            self._error = RuntimeError(
                f"gatx: edge_index' has {self._E2} edges, but expect_num_edges promised "
                f"{self._E2_hint} for this edge_index (its contents changed?)")
            raise self._error

    def _poll(self):
        """Validate without blocking if the device has produced the meta (raises on bad ids); the
        current stream may use the CSR from here on."""
        if self._error is not None:
            raise self._error
        self.follow()
        if (self._E2 is None and self._event is not None
                and not torch.cuda.is_current_stream_capturing() and self._event.query()):
            self._validate(self._meta_host)

    poll = untraced(_poll)

    # ---- host-side sizes (synchronise on first use)
    @property
    def num_edges(self) -> int:
        """|edge_index'| (reads the device meta once: a sync if it is not there yet)."""
        if self._error is not None:
            raise self._error
        if self._E2 is None and self._E2_hint is not None:
            # trust the promise now; the device count is compared when it lands (poll /
            # check_pending), or never inside a captured step
            return self._E2_hint
        if self._E2 is None:
            self._read_meta()
        return self._E2

    @untraced
    def _read_meta(self):
        if self._event is not None:
            self._event.synchronize()
            self._validate(self._meta_host)
        else:
            self._validate(self.meta.cpu())

    @property
    def edge_index(self) -> torch.Tensor:
        """edge_index' as the reference returns it: a contiguous int64 (2, E') tensor (the input
        itself without the rewrite)."""
        if self._edge_index is None:
            E2 = self.num_edges
            if self._ei_flat is None:
                self._edge_index = self.source
            else:
                self._edge_index = self._ei_flat[:2 * E2].view(2, E2)
                graph_cache.alias(self._edge_index, self)
        return self._edge_index

    def _ensure_transpose(self):
        if self.srowptr is None:
            with _BUILDING, on_device(self.device):
                if self.srowptr is None:
                    self._build_transpose()
        self.follow("transpose")

    ensure_transpose = untraced(_ensure_transpose)

    def _build_transpose(self):
        self.follow()
        N, Eb, dev = self.num_nodes, self.edge_bound, self.device
        i32 = dict(dtype=torch.int32, device=dev)
        srowptr = torch.empty(N + 1, **i32)
        scol = torch.empty(max(Eb, 1), **i32)
        seid = torch.empty(max(Eb, 1), **i32)
        ws_bytes = _lib.lib.gatx_graph_transpose_workspace_bytes(Eb, N)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        call("gatx_graph_transpose", ptr(self.col), ptr(self.rowidx), N, Eb, self.e2_ptr,
             ptr(srowptr), ptr(scol), ptr(seid), ptr(ws), ws_bytes, stream())
        self._built("transpose", (srowptr, scol, seid))
        self.scol, self.seid = scol, seid
        self.srowptr = srowptr   # the last: what others look at

    @untraced
    def hub_plan(self, hub_edges: int, source: bool = False):
        """(hubs, hub_count, hub_bound) of gatx_graph_hub_plan for this CSR: destination segments
        (source=True: source segments of the transpose, for the backward's source pass) longer
        than hub_edges listed as pieces (device-side count; built once per graph)."""
        def build():
            if source:
                self._ensure_transpose()
            bound = int(_lib.lib.gatx_graph_hub_bound(self.edge_bound, hub_edges))
            hubs = torch.empty((max(bound, 1), 4), dtype=torch.int32, device=self.device)
            count = torch.empty(1, dtype=torch.int32, device=self.device)
            call("gatx_graph_hub_plan", ptr(self.srowptr if source else self.rowptr),
                 self.num_nodes, hub_edges, ptr(hubs), bound, ptr(count), stream())
            return hubs, count, bound
        return self._kept((hub_edges, source), build)

    @untraced
    def node_blocks(self, max_rows: int, side: bool = False):
        """(segs, count) of gatx_graph_segments for this CSR (device tensors, built once per graph
        and max_rows): contiguous node blocks no edge crosses, each <= max_rows nodes; count -1
        when the graph has none (a gap-free run longer than max_rows). The workspace is a
        per-device scratch that lives as long as the process, so a captured step's launches
        keep its address.
        side: launch on the per-device side stream (forked from the current stream; the caller
        joins it with join_side before reading the result), so the four small launches run
        under the projection GEMM instead of after it. The tensors are allocated on the current
        stream either way."""
        from . import tuning
        dev = self.device
        sst = side_stream(dev) if side and tuning.get("side_stream") else None

        def build():
            segs = torch.empty(_lib.lib.gatx_graph_segments_max() + 2, dtype=torch.int32,
                               device=dev)
            count = torch.empty(1, dtype=torch.int32, device=dev)
            wb = _lib.lib.gatx_graph_segments_workspace_bytes(self.num_nodes)
            ws = _seg_ws(dev, wb)
            if sst is not None:
                sst.wait_stream(torch.cuda.current_stream(dev))
                call("gatx_graph_segments", ptr(self.rowptr), ptr(self.col), self.num_nodes,
                     int(max_rows), ptr(segs), ptr(count), ptr(ws), wb, sst.cuda_stream)
                _SIDE_PENDING[dev] = True
            else:
                join_side(dev)   # (the scratch may still be in use by a side-stream build)
                call("gatx_graph_segments", ptr(self.rowptr), ptr(self.col), self.num_nodes,
                     int(max_rows), ptr(segs), ptr(count), ptr(ws), wb, stream())
            return segs, count
        return self._kept(("blocks", max_rows), build, sst)

    def lds_blocks(self, max_rows: int, side: bool = False):
        """(segs, count, n_blocks) of node_blocks(max_rows) when this edge_index is known to cut
        into such blocks, else None. Known: decided once per edge_index tensor (storage, version,
        shape, node count) by one read of the device count (outside a capture), cached across
        graph rebuilds (clear_graph_cache) — the same identity the graph cache keys on; inside a
        capture an undecided graph takes the L2-gather pass."""
        key = _hint_key(self.source, self.num_nodes, self.add_self_loops) + (
            version(self.source), max_rows)
        known = _BLOCKS.get(key)
        if known is None:
            if torch.cuda.is_current_stream_capturing():
                return None
            segs, count = self.node_blocks(max_rows)
            known = _BLOCKS[key] = int(count.item())
            while len(_BLOCKS) > 64:
                _BLOCKS.pop(next(iter(_BLOCKS)))
        if known <= 0:
            return None
        segs, count = self.node_blocks(max_rows, side)
        return segs, count, known

    def csr_host(self):
        """(rowptr, col, perm) as CPU tensors — for tests."""
        E2 = self.num_edges
        return self.rowptr.cpu(), self.col[:E2].cpu(), self.perm[:E2].cpu()


_PENDING: list = []
_HINTS: dict = {}
_BLOCKS: dict = {}   # edge_index identity -> node-block count (<= 0: no LDS-staged passes)


def _hint_key(edge_index: torch.Tensor, num_nodes, add_self_loops: bool):
    return (edge_index.data_ptr(), tuple(edge_index.shape), edge_index.dtype, edge_index.device,
            num_nodes, add_self_loops)


def expect_num_edges(edge_index: torch.Tensor, num_nodes: int, add_self_loops: bool,
                     num_edges: int | None) -> None:
    """Promise |edge_index'| for this edge_index tensor (same storage, shape and node count) for
    every later graph build from it, cached or rebuilt, so returning edge_index' / the attention
    weights needs no device read: what lets a step that rebuilds its CSR every time (the
    reference rewrites self-loops in every layer call) and returns the attention (PPI_GAT /
    PlanetoidGAT's forward_and_return_attention) be captured as a hipGraph. The device count is
    still compared with the promise whenever it is read outside a capture (a mismatch raises, as
    a device assert would). None withdraws the promise. Survives clear_graph_cache()."""
    k = _hint_key(edge_index, num_nodes, add_self_loops)
    if num_edges is None:
        _HINTS.pop(k, None)
    else:
        # the promise is bound to this tensor object at its current version: an in-place rewrite
        # of it, or another tensor the allocator later places at the same address, finds no
        # promise (and the count is read from the device as usual)
        _HINTS[k] = (int(num_edges), version(edge_index), weakref.ref(edge_index))


def _hint_lookup(edge_index: torch.Tensor, num_nodes, add_self_loops: bool):
    """The count promised by expect_num_edges for exactly this tensor, unmodified since; else
    None."""
    hit = _HINTS.get(_hint_key(edge_index, num_nodes, add_self_loops))
    if hit is None:
        return None
    n, ver, ref = hit
    if ref() is not edge_index or version(edge_index) != ver:
        return None
    return n


_SIDE: dict = {}


def side_stream(dev) -> torch.cuda.Stream:
    """A per-device second stream for short launches that can run beside the current stream's
    work (forked with wait_stream, joined with join_side; both are captured as graph edges)."""
    st = _SIDE.get(dev)
    if st is None:
        st = _SIDE[dev] = torch.cuda.Stream(device=dev)
    return st


def join_side(dev) -> None:
    """The current stream waits for what was launched on the side stream since the last join
    (nothing to wait for: no event, so a capture never waits on an uncaptured stream)."""
    st = _SIDE.get(dev)
    if st is not None and _SIDE_PENDING.pop(dev, False):
        torch.cuda.current_stream(dev).wait_stream(st)


_SIDE_PENDING: dict = {}


_SEG_WS: dict = {}
_SEG_WS_RETIRED: list = []


def _seg_ws(dev, nbytes: int):
    """Per-device scratch of gatx_graph_segments, grown to the largest graph seen and never
    freed (a captured step's launches keep its address)."""
    t = _SEG_WS.get(dev)
    if t is None or t.numel() < nbytes:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gatx: node-block scratch must be sized before a capture (run "
                               "the step once eagerly)")
        if t is not None:
            _SEG_WS_RETIRED.append(t)   # a captured graph may still launch on the old one
        t = _SEG_WS[dev] = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
    return t


def check_pending(block: bool = True):
    """Validate every live graph whose meta has not been read yet (blocking by default): raises
    the first bad-index error, like torch.cuda.synchronize() surfacing a device assert. Called
    non-blocking by every Graph construction."""
    global _PENDING
    pending, _PENDING = _PENDING, []
    for i, r in enumerate(pending):
        g = r()
        if g is None or g._E2 is not None or g._error is not None:
            continue   # gone, validated, or its error already raised
        try:
            if block:
                g._read_meta()
            else:
                g.poll()
        except Exception:
            _PENDING.extend(x for x in pending[i + 1:] if x() is not None)
            raise
        if g._E2 is None:
            _PENDING.append(r)


class GraphCache:
    """Small LRU of Graphs keyed on the edge_index tensor's identity and version. Entries hold a
    reference to their key tensor, so a cached data_ptr can never be recycled under them. A
    Graph built with add_self_loops also answers for its own output edge_index' once that is
    materialised (the rewrite is idempotent, so GATModel.forward_and_return_attention's chaining
    of layers hits the cache)."""

    def __init__(self, capacity: int = 8):
        self.capacity = capacity
        self._d: OrderedDict = OrderedDict()

    @staticmethod
    def _key(t: torch.Tensor, num_nodes, add_self_loops: bool):
        return (t.data_ptr(), version(t), tuple(t.shape), tuple(t.stride()), t.dtype,
                t.device, num_nodes, add_self_loops)

    @untraced
    def get(self, edge_index: torch.Tensor, num_nodes: int, add_self_loops: bool) -> Graph:
        k = self._key(edge_index, num_nodes, add_self_loops)
        hit = self._d.get(k)
        if hit is not None:
            self._d.move_to_end(k)
            g = hit[1]
            g._poll()
            return g
        g = Graph(edge_index, num_nodes, add_self_loops)
        self._put(k, edge_index, g)
        return g

    def alias(self, ei2: torch.Tensor, g: Graph):
        """Register a tensor holding a graph's edge_index' (its materialised buffer, or a copy of
        it such as the one the registered op gatx::layer_fwd returns) as a key of the same
        graph."""
        if g.add_self_loops:
            self._put(self._key(ei2, g.num_nodes, True), ei2, g, True)

    @staticmethod
    def _same(a: torch.Tensor, b: torch.Tensor) -> bool:
        return a is b or (a.data_ptr() == b.data_ptr() and version(a) == version(b)
                          and a.shape == b.shape and a.stride() == b.stride()
                          and a.dtype == b.dtype and a.device == b.device)

    @untraced
    def for_edges(self, edge_index: torch.Tensor) -> Graph:
        """The Graph whose edge_index' IS this tensor (what a layer returned), else a CSR of it
        as given (no rewrite), sized by its max id — for consumers of a layer's output edges
        such as the attention-norm regulariser."""
        for t, g, is_alias in reversed(self._d.values()):
            ei = g._edge_index
            if (ei is not None and self._same(ei, edge_index)) or (
                    is_alias and self._same(t, edge_index)):
                g.follow()
                return g
        k = self._key(edge_index, -1, False)
        hit = self._d.get(k)
        if hit is not None:
            hit[1].follow()
            return hit[1]
        g = Graph(edge_index, None, False)
        self._put(k, edge_index, g)
        return g

    def _put(self, k, t, g, is_alias=False):
        self._d[k] = (t, g, is_alias)
        self._d.move_to_end(k)
        while len(self._d) > self.capacity:
            self._d.popitem(last=False)

    def clear(self):
        self._d.clear()


graph_cache = GraphCache()


def clear_graph_cache():
    graph_cache.clear()

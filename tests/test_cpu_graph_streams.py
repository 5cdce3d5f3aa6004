"""Which stream a gatx.Graph's lazily built arrays wait for, on the host: streams, events and launches
are stand-ins that write down what was asked of them, in order."""
import threading

import pytest
import torch


class Recorder:
    """The device as the code under test sees it: the current stream, launches, events, waits."""

    def __init__(self, monkeypatch):
        from gatx import attention, graph
        self.log, self.now, self.capturing = [], 1, False
        rec = self

        class Event:
            def record(self, stream=None):
                self.on = rec.now if stream is None else stream.cuda_stream
                rec.log.append(("record", self.on))

            def query(self):
                return False

        class Stream:
            def __init__(self, at):
                self.cuda_stream = at

            def wait_event(self, event):
                rec.log.append(("wait", self.cuda_stream, event.on))

            def wait_stream(self, other):
                rec.log.append(("join", self.cuda_stream, other.cuda_stream))

        def call(name, *args):
            rec.log.append(("launch", name, rec.now))
        monkeypatch.setattr(torch.cuda, "Event", Event)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(rec.now))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: rec.capturing)
        monkeypatch.setattr(torch.Tensor, "record_stream",
                            lambda t, s: rec.log.append(("keep", s.cuda_stream)))
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: rec.now,
                            raising=False)
        for module in (graph, attention):
            monkeypatch.setattr(module, "call", call)
            monkeypatch.setattr(module, "stream", lambda: rec.now)

    def on(self, stream):
        self.now = stream
        self.log.clear()


@pytest.fixture
def rec(monkeypatch):
    return Recorder(monkeypatch)


def built(rec, N=40, E=3000):
    """A Graph whose CSR was filled on the current stream."""
    from gatx.graph import Graph
    g = object.__new__(Graph)
    g.device, g.num_nodes, g.edge_bound, g.num_input_edges = torch.device("cpu"), N, E, E
    g.meta = torch.zeros(8, dtype=torch.int64)
    g.rowptr, g.col = torch.zeros(N + 1).int(), torch.zeros(E).int()
    g.rowidx, g.perm, g._ei_flat = torch.zeros(E).int(), torch.zeros(E).int(), None
    g.srowptr = g.scol = g.seid = None
    g._hub_plans, g._builds, g._error, g._E2 = {}, {}, None, E
    g._event = torch.cuda.Event()
    g._event.record()
    g._built("csr", (g.meta, g.rowptr, g.col, g.rowidx, g.perm, g._ei_flat), g._event)
    return g


def launches(rec):
    return [x[1] for x in rec.log if x[0] == "launch"]


def waits(rec):
    return [x[1:] for x in rec.log if x[0] == "wait"]


USES = {"transpose": lambda g: g.ensure_transpose(), "plan": lambda g: g.hub_plan(512),
        "source plan": lambda g: g.hub_plan(512, True), "blocks": lambda g: g.node_blocks(2304)}


@pytest.mark.parametrize("what", USES)
def test_another_stream_waits_for_the_build_once(what, rec, monkeypatch):
    from gatx import graph
    monkeypatch.setattr(graph, "_seg_ws", lambda dev, n: torch.zeros(1))
    g = built(rec)
    use = USES[what]
    rec.on(1)
    use(g)
    assert launches(rec) and not waits(rec)
    assert [x[0] for x in rec.log].index("record") > [x[0] for x in rec.log].index("launch")
    rec.on(1)
    use(g)
    assert not rec.log   # its own stream: nothing
    rec.on(2)
    use(g)
    assert not launches(rec) and waits(rec) == [(2, 1)]
    assert ("keep", 2) in rec.log
    rec.on(2)
    use(g)
    assert not rec.log   # it is behind the build from then on
    rec.on(3)
    use(g)
    assert waits(rec) == [(3, 1)]


@pytest.mark.parametrize("what", USES)
def test_a_build_waits_for_what_it_reads(what, rec, monkeypatch):
    """The CSR filled on stream 1, the rest built on stream 2."""
    from gatx import graph
    monkeypatch.setattr(graph, "_seg_ws", lambda dev, n: torch.zeros(1))
    g = built(rec)
    rec.on(2)
    USES[what](g)
    assert waits(rec)[0] == (2, 1)
    assert [x[0] for x in rec.log].index("wait") < [x[0] for x in rec.log].index("launch")


def test_a_source_plan_waits_for_a_transpose_of_another_stream(rec):
    """... that a GAT layer's backward built (it calls ensure_transpose alone)."""
    g = built(rec)
    rec.on(2)
    g.ensure_transpose()
    rec.on(1)
    g.hub_plan(512, True)
    assert waits(rec) == [(1, 2)] and launches(rec) == ["gatx_graph_hub_plan"]


def test_the_attention_uses_the_graphs_own_bookkeeping(rec, monkeypatch):
    from gatx import attention
    monkeypatch.setattr(attention, "_ORDER_ITEMS", 1)
    plans = lambda: (attention._transpose(g), attention._row_order(g, 2, True),   # noqa: E731
                     attention._row_order(g, 2, False))
    g = built(rec)
    rec.on(1)
    g.ensure_transpose()   # as a GAT layer does
    rec.on(2)
    g.poll()
    plans()
    assert waits(rec) == [(2, 1), (2, 1)]   # the CSR, the transpose
    rec.on(1)
    plans()
    assert waits(rec) == [(1, 2), (1, 2)]   # both orders
    rec.on(1)
    plans()
    assert not rec.log


def test_nothing_is_waited_for_inside_a_capture(rec):
    g = built(rec)
    g.ensure_transpose()
    rec.on(2)
    rec.capturing = True
    g.ensure_transpose()
    g.poll()
    assert not rec.log
    rec.capturing = False
    g.ensure_transpose()   # an eager call there still has to wait
    assert waits(rec) == [(2, 1)]


def test_nobody_finds_what_has_no_event_yet(rec, monkeypatch):
    """Another thread that looks while a plan is launched: the plan is not there, or behind its event."""
    g = built(rec)
    seen = []
    real = g._built

    def slow(key, tensors, event=None, side=None):
        seen.append((key, g.srowptr is None, key in g._hub_plans))
        real(key, tensors, event, side)
    monkeypatch.setattr(type(g), "_built", lambda self, *a, **k: slow(*a, **k))
    g.hub_plan(512, True)
    assert [x[0] for x in seen] == ["transpose", (512, True)]
    assert seen[0][1] and not seen[1][2]
    # and two threads build it once
    g = built(rec)
    rec.on(1)
    go = threading.Barrier(4)

    def work():
        go.wait()
        g.hub_plan(64)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert launches(rec) == ["gatx_graph_hub_plan"]


class OnDevice(torch.Tensor):
    """A host tensor that says it is on the device."""
    is_cuda = True


@pytest.mark.parametrize("what", ["csr", "order"] + list(USES))
def test_everything_is_launched_on_the_graphs_own_device(what, rec, monkeypatch):
    """... whichever is current."""
    import contextlib

    from gatx import attention, graph
    inside = []

    @contextlib.contextmanager
    def on_device(device):
        inside.append(device)
        yield
        inside.pop()
    seen = []
    for module in (graph, attention):
        monkeypatch.setattr(module, "on_device", on_device)
        monkeypatch.setattr(module, "call", lambda name, *a: seen.append((name, list(inside))))
    monkeypatch.setattr(graph, "_seg_ws", lambda dev, n: torch.zeros(1))
    monkeypatch.setattr(graph, "_PENDING", [])
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, pin_memory=False, **k: empty(*a, **k))
    event, record = torch.cuda.Event, []

    class Event(event):
        def record(self, stream=None):
            record.append(list(inside))
            super().record(stream)
    if what == "csr":
        monkeypatch.setattr(torch.cuda, "Event", Event)
        graph.Graph(torch.zeros(2, 9, dtype=torch.int64).as_subclass(OnDevice), 5, True)
    else:
        g = built(rec)
        monkeypatch.setattr(torch.cuda, "Event", Event)
        if what == "order":
            monkeypatch.setattr(attention, "_ORDER_ITEMS", 1)
            attention._row_order(g, 2, False)
        else:
            USES[what](g)
    assert seen and all(x == torch.device("cpu") for _, d in seen for x in d)
    assert all(d for _, d in seen), seen
    assert record and all(record)


def test_graphs_built_at_once_share_no_workspace(rec, monkeypatch):
    """On two streams (or one of them in a replayed capture): what one writes between its launches is its
    own."""
    from gatx import graph
    alive, used = [], []
    empty = torch.empty

    def kept(*a, pin_memory=False, **k):
        alive.append(empty(*a, **k))   # nothing's memory is handed out again
        return alive[-1]
    monkeypatch.setattr(torch, "empty", kept)
    monkeypatch.setattr(graph, "_PENDING", [])
    monkeypatch.setattr(graph, "call", lambda name, *a: used.append((name, a)))
    for _ in range(2):
        graph.Graph(torch.zeros(2, 9, dtype=torch.int64).as_subclass(OnDevice), 5, True)
    meta = [a[7] for name, a in used if name == "gatx_graph_meta"]
    build = [a[13] for name, a in used if name == "gatx_graph_build"]
    assert len(set(meta)) == len(set(build)) == 2

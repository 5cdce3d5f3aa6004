"""What the graph-transformer operators refuse, on the host: argument checks of the Python entry
points and of the C-ABI (nothing is launched), and the position buckets' bounds."""
import ctypes

import pytest
import torch

import attention_reference as ref


def fake_graph(N=6, E=9):
    """A Graph that was never built: what the argument checks look at."""
    from gatx.graph import Graph
    g = object.__new__(Graph)
    g.device, g.num_nodes, g.edge_bound = torch.device("cpu"), N, E
    return g


def inputs(N=6, H=2, d=4, dv=8, dtype=torch.float32):
    return dict(q=torch.zeros(N, H, 2, d, dtype=dtype), k=torch.zeros(N, H, 2, d, dtype=dtype),
                v=torch.zeros(N, H, dv, dtype=dtype), lam=torch.zeros(H), bias=None,
                positions=None, nodes=None)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(6, 2, 4)), ValueError),
    (dict(q=torch.zeros(5, 2, 2, 4)), ValueError),
    (dict(k=torch.zeros(6, 2, 2, 5)), ValueError),
    (dict(k=torch.zeros(6, 1, 2, 4)), ValueError),
    (dict(v=torch.zeros(5, 2, 8)), ValueError),
    (dict(v=torch.zeros(6, 3, 8)), ValueError),
    (dict(q=torch.zeros(6, 2, 2, 257), k=torch.zeros(6, 2, 2, 257)), ValueError),
    (dict(v=torch.zeros(6, 2, 513)), ValueError),
    (dict(v=torch.zeros(6, 2, 8, dtype=torch.float16)), RuntimeError),
    (dict(q=torch.zeros(6, 2, 2, 4, dtype=torch.float64)), RuntimeError),
    (dict(lam=torch.zeros(3)), ValueError),
    (dict(lam=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(bias=torch.zeros(8, 2)), ValueError),
    (dict(positions=torch.zeros(6, dtype=torch.int64)), ValueError),
    (dict(bias=torch.zeros(8, 3), positions=torch.zeros(6, dtype=torch.int64)), ValueError),
    (dict(bias=torch.zeros(8, 2), positions=torch.zeros(6)), ValueError),
    (dict(bias=torch.zeros(8, 2), positions=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(nodes=torch.zeros(2, 3, dtype=torch.int64)), ValueError),
    (dict(nodes=torch.zeros(6)), ValueError),
    (dict(nodes=torch.zeros(2, dtype=torch.int64)), ValueError),
])
def test_attention_arguments(change, error):
    from gatx.attention import _check
    a = inputs()
    g = fake_graph()
    _check(a["q"], a["k"], a["v"], a["lam"], g, None, None, None)
    a.update(change)
    with pytest.raises(error, match="diff_attention"):
        _check(a["q"], a["k"], a["v"], a["lam"], g, a["bias"], a["positions"], a["nodes"])


def test_attention_needs_a_graph_and_its_device():
    from gatx import diff_attention
    a = inputs()
    with pytest.raises(TypeError, match="Graph"):
        diff_attention(a["q"], a["k"], a["v"], a["lam"], torch.zeros(2, 3, dtype=torch.int64))
    g = fake_graph()
    g.device = torch.device("cuda:0")
    with pytest.raises(RuntimeError, match="no CPU path"):
        diff_attention(a["q"], a["k"], a["v"], a["lam"], g)


@pytest.mark.parametrize("n,far,both", [(1, 9, False), (2, 9, True), (5, 9, True), (257, 999, False),
                                        (32, 8, True), (32, 16, False), (8, 2 ** 62, True)])
def test_bad_buckets(n, far, both):
    from gatx.attention import bucket_bounds
    with pytest.raises(ValueError, match="bucket"):
        bucket_bounds(n, far, both)


@pytest.mark.parametrize("n,far,both", [(2, 2, False), (4, 2, True), (4, 9, True), (32, 128, True),
                                        (32, 128, False), (33, 57, False), (256, 129, False),
                                        (256, 100000, True), (16, 2 ** 40, False)])
def test_bucket_bounds(n, far, both):
    """The bounds give every distance near one of them the bucket that whole-number powers do."""
    from gatx.attention import bucket_bounds
    m, bounds = bucket_bounds(n, far, both)
    side = n // 2 if both else n
    assert m == side // 2 and len(bounds) == side - m - 1 and bounds == sorted(bounds)
    near = sorted({max(0, x + o) for x in bounds + [m, far] for o in (-2, -1, 0, 1, 2)})
    want = ref.buckets(-torch.tensor(near), n, far, both).tolist()
    got = [x if x < m else m + sum(b <= x for b in bounds) for x in near]
    assert got == want


NORM = dict(h=torch.zeros(3, 8), weight=torch.ones(8))


@pytest.mark.parametrize("change,error", [
    (dict(h=torch.zeros(3, 8, dtype=torch.float64)), RuntimeError),
    (dict(h=torch.zeros(3, 8193), weight=torch.ones(8193)), ValueError),
    (dict(h=torch.zeros(3, 0), weight=torch.ones(0)), ValueError),
    (dict(weight=torch.ones(7)), ValueError),
    (dict(weight=torch.ones(8, dtype=torch.int32)), ValueError),
    (dict(scale=torch.ones(1)), ValueError),
    (dict(next_weight=torch.ones(9)), ValueError),
    (dict(gate=torch.ones(7)), ValueError),
    (dict(gate=torch.ones(2, 8)), ValueError),
    (dict(gate=torch.ones(3, 8, dtype=torch.bfloat16)), ValueError),
    (dict(resid=torch.ones(8)), ValueError),
    (dict(resid=torch.ones(3, 8, dtype=torch.float16)), ValueError),
    (dict(), RuntimeError),   # host tensors
])
def test_norm_arguments(change, error):
    from gatx import norm_after
    a = {**NORM, **change}
    with pytest.raises(error, match="norm_after"):
        norm_after(a.pop("h"), a.pop("weight"), **a)


def test_norm_before_arguments():
    from gatx import norm_before
    with pytest.raises(ValueError, match="norm_before"):
        norm_before(torch.zeros(3, 8), torch.ones(4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_before(torch.zeros(3, 8), torch.ones(8))


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(3)), ValueError),
    (dict(logits=torch.zeros(3, 0)), ValueError),
    (dict(logits=torch.zeros(4, 8)), ValueError),
    (dict(logits=torch.zeros(3, 8, dtype=torch.float64)), RuntimeError),
    (dict(teacher=torch.zeros(3, 3)), ValueError),
    (dict(teacher=torch.zeros(3, 2).long()), RuntimeError),
    (dict(teacher=torch.zeros(3, 2, requires_grad=True)), RuntimeError),
    (dict(teacher=torch.zeros(3, 0), index=torch.zeros(3, 0).long()), ValueError),
    (dict(teacher=torch.zeros(3, 1025), index=torch.zeros(3, 1025).long()), ValueError),
    (dict(index=torch.zeros(3, 2)), RuntimeError),
    (dict(temperature=0.0), ValueError),
    (dict(temperature=float("nan")), ValueError),
    (dict(reduction="batchmean"), ValueError),
    (dict(), RuntimeError),   # host tensors
])
def test_distillation_arguments(change, error):
    from gatx.losses import TopKDistillationLoss, topk_distillation
    a = {**dict(logits=torch.zeros(3, 8), teacher=torch.zeros(3, 2),
                index=torch.zeros(3, 2).long()), **change}
    with pytest.raises(error, match="topk_distillation"):
        topk_distillation(a.pop("logits"), a.pop("teacher"), a.pop("index"), **a)
    with pytest.raises(RuntimeError, match="no CPU path"):
        TopKDistillationLoss(2.0)(torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2).long())


@pytest.mark.parametrize("temperature", [-1.0, 1e-19, 1e19, float("inf"), 1e-60])
def test_distillation_temperatures(temperature):
    from gatx.losses import topk_distillation
    with pytest.raises(ValueError, match="temperature"):
        topk_distillation(torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2).long(),
                          temperature)


def c_call(name, *args):
    from gatx._lib import lib
    rc = getattr(lib, name)(*args)
    return rc, lib.gatx_last_error().decode()


# a 16-byte aligned host address that is never followed: the calls below are refused first
_buf = ctypes.create_string_buffer(64)
ANY = (ctypes.addressof(_buf) + 15) // 16 * 16


@pytest.mark.parametrize("args", [
    (3, 4, 8, ANY, 8, ANY, None, 0, None, 0, 0, None, None, 1e-6, ANY, None, None, None, None),
    (0, 4, 8193, ANY, 8, ANY, None, 0, None, 0, 0, None, None, 1e-6, ANY, None, None, None, None),
    (0, -1, 8, ANY, 8, ANY, None, 0, None, 0, 0, None, None, 1e-6, ANY, None, None, None, None),
    (0, 4, 8, ANY, 8, None, ANY, 8, None, 0, 0, None, ANY, 1e-6, None, ANY, None, None, None),
    (0, 4, 8, ANY, 8, None, None, 0, None, 0, 0, None, None, 1e-6, None, None, None, None, None),
    (0, 4, 8, ANY, 8, ANY, None, 0, None, 0, 0, None, ANY, 1e-6, ANY, None, None, None, None),
    (0, 4, 8, None, 8, ANY, None, 0, None, 0, 0, None, None, 1e-6, ANY, None, None, None, None),
])
def test_block_norm_c_refusals(args):
    rc, msg = c_call("gatx_block_norm", *args)
    assert rc == 1000 and "block_norm" in msg


def test_block_norm_backward_c_refusals():
    ok = [0, 4, 8, ANY, 8, ANY, None, 0, None, 0, 0, None, None, ANY, None, ANY, 8, None, 0, ANY,
          None, None, ANY, None, None, ANY, 10 ** 6, None]
    for at, value in ((0, 7), (2, 9000), (3, None), (13, None), (26, 16), (17, ANY)):
        bad = list(ok)
        bad[at] = value
        rc, msg = c_call("gatx_block_norm_backward", *bad)
        assert rc == 1000 and "block_norm_backward" in msg, at


def test_distill_c_refusals():
    ok = [0, ANY, 4, 8, 8, 0, ANY, ANY, 1, 2, 1.0, None, ANY, 1, ANY, None, ANY, 10 ** 6, None]
    for at, value in ((0, 5), (5, 9), (1, None), (2, -1), (3, 0), (9, 0), (9, 1025), (10, 0.0),
                      (10, float("nan")), (10, float("inf")), (14, None), (17, 4)):
        bad = list(ok)
        bad[at] = value
        rc, msg = c_call("gatx_topk_distill", *bad)
        assert rc == 1000 and "topk_distill" in msg, at
    ok = [0, ANY, 4, 8, 8, 0, ANY, ANY, 1, 2, 1.0, ANY, ANY, 0, None, ANY, None]
    for at, value in ((11, None), (12, None), (13, 2), (15, None)):
        bad = list(ok)
        bad[at] = value
        rc, msg = c_call("gatx_topk_distill_backward", *bad)
        assert rc == 1000 and "topk_distill_backward" in msg, at


def test_attention_c_refusals():
    #      dt q    ldq k    ldk v    ldv H  d  dv rowptr col E  M  N  nodes pieces
    ok = [0, ANY, 32, ANY, 32, ANY, 16, 2, 8, 8, ANY, ANY, 9, 6, 6, None, 1, 1.0, ANY, None, None,
          ANY, ANY, ANY, 0, None, None, 0, None, 0, None, None]
    for at, value in ((0, 4), (1, None), (2, 31), (1, ANY + 4), (4, 31), (7, 0), (8, 257), (9, 513),
                      (12, 1 << 31), (13, 5), (15, ANY), (16, 5000), (19, ANY), (20, ANY),
                      (21, None), (21, ANY + 8), (22, None), (24, 4)):
        bad = list(ok)
        bad[at] = value
        if at == 16:
            bad[15], bad[22], bad[23] = ANY, None, None
        rc, msg = c_call("gatx_diff_attention", *bad)
        assert rc == 1000 and "diff_attention" in msg, (at, msg)
    bad = list(ok)   # pieces without room for them
    bad[15], bad[16], bad[22], bad[23] = ANY, 8, None, None
    rc, msg = c_call("gatx_diff_attention", *bad)
    assert rc == 1000 and "workspace" in msg


def test_attention_backward_c_refusals():
    ok = [0, ANY, 32, ANY, 32, ANY, 16, ANY, 16, 2, 8, 8, ANY, ANY, ANY, ANY, ANY, 9, 6, 1.0, ANY,
          None, 0, ANY, ANY, ANY, ANY, ANY, ANY, None, 0, None, None, 0, None, None, 0, ANY,
          10 ** 9, None, None, None]
    for at, value in ((0, 4), (7, None), (8, 15), (14, None), (22, 257), (29, ANY), (23, None),
                      (25, ANY + 4), (30, 4), (38, 8)):
        bad = list(ok)
        bad[at] = value
        rc, msg = c_call("gatx_diff_attention_backward", *bad)
        assert rc == 1000 and "diff_attention_backward" in msg, (at, msg)


def test_row_order_c_refusals():
    for bad in ((None, 5, ANY, None), (ANY, 5, None, None), (ANY, 5, ANY + 4, None),
                (ANY, 1 << 31, ANY, None), (ANY, -1, ANY, None)):
        rc, msg = c_call("gatx_diff_attention_row_order", *bad)
        assert rc == 1000 and "row_order" in msg, bad


def test_order_c_refusals():
    ok = [0, ANY, 32, ANY, 32, ANY, 16, 2, 8, 8, ANY, ANY, 9, 6, 6, None, 1, 1.0, ANY, None, None,
          ANY, ANY, ANY, 0, None, None, 0, None, 0, ANY + 4, None]
    rc, msg = c_call("gatx_diff_attention", *ok)
    assert rc == 1000 and "order" in msg


def test_buckets_c_refusals():
    ok = [ANY, ANY, ANY, 9, 6, None, 0, ANY, 1, 4, ANY, 3, 1, ANY, None]
    for at, value in ((9, 0), (11, 127), (11, -1), (10, None), (7, None), (13, None)):
        bad = list(ok)
        bad[at] = value
        rc, msg = c_call("gatx_relative_buckets", *bad)
        assert rc == 1000 and "relative_buckets" in msg, at

"""The plans of long rows in diff_attention's backward, on the host: the destinations' and the sources'
are independent of each other in the C-ABI (nothing is launched: every call is refused at last)."""
import itertools

import pytest

from test_cpu_operator_refusals import ANY, c_call

# gatx_diff_attention_backward's arguments from hub_edges on, and a complete call around them that is
# refused for its workspace alone
HUB_EDGES, HUBS, COUNT, BOUND, SRC_HUBS, SRC_COUNT, SRC_BOUND, WORKSPACE_BYTES = (
    30, 31, 32, 33, 34, 35, 36, 38)


def refusal(gq=ANY, gk=ANY, gv=ANY, **at):
    a = [0, ANY, 32, ANY, 32, ANY, 16, ANY, 16, 2, 8, 8, ANY, ANY, ANY, ANY, ANY, 9, 6, 1.0, ANY,
         None, 0, ANY, ANY, gq, gk, gv, ANY, None, 0, None, None, 0, None, None, 0, ANY,
         8, None, None, None]
    for i, value in at.items():
        a[int(i[1:])] = value
    rc, msg = c_call("gatx_diff_attention_backward", *a)
    assert rc == 1000
    return msg


DST = {f"_{HUBS}": ANY, f"_{COUNT}": ANY, f"_{BOUND}": 3}
SRC = {f"_{SRC_HUBS}": ANY, f"_{SRC_COUNT}": ANY, f"_{SRC_BOUND}": 3}


@pytest.mark.parametrize("dst,src", itertools.product([False, True], repeat=2))
def test_either_direction_may_go_without_a_plan(dst, src):
    plans = {**(DST if dst else {}), **(SRC if src else {})}
    if plans:
        plans[f"_{HUB_EDGES}"] = 512
    assert "workspace" in refusal(**plans)
    assert "workspace" in refusal(gk=None, gv=None, **plans)
    assert "workspace" in refusal(gq=None, **plans)


@pytest.mark.parametrize("wrong", [
    {HUBS: None}, {COUNT: None}, {SRC_HUBS: None}, {SRC_COUNT: None}, {HUB_EDGES: -1},
    {BOUND: -1}, {SRC_BOUND: -1}])
def test_half_a_plan_is_refused(wrong):
    plans = {**DST, **SRC, f"_{HUB_EDGES}": 512, **{f"_{i}": x for i, x in wrong.items()}}
    assert "hub plan" in refusal(**plans)


def test_pieces_without_any_plan_are_refused():
    assert "hub plan" in refusal(**{f"_{HUB_EDGES}": 512})

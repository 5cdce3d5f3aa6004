"""The graph-transformer operators together, as they are used: a GATModel with norms around its
layers, and a student of differential attention blocks (position bias, block norms) that learns from
a teacher's top logits, each against the same stack in float64 on the host.

Tolerance: 1e-4 of max(1, the largest reference value) of every compared tensor, as for the layers'
own gradients: a step of these stacks passes each value through fewer than 100 float32 operations of
relative error 2^-24, sums of up to 400 terms, and norms and softmaxes that amplify an error at most
a few times."""
import math

import pytest
import torch
import torch.nn.functional as F

import attention_reference as ref

pytestmark = pytest.mark.gpu


def close(got, want, name):
    want = want.detach()
    err = float((got.detach().double().cpu() - want).abs().max())
    assert err <= 1e-4 * max(1.0, float(want.abs().max())), (name, err)


def rms(x, weight):
    return x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight


def block(p, h, resid):
    y = p["scale"] * torch.sigmoid(p["gate"]) * rms(h, p["weight"])
    y = y if resid is None else resid + y
    return y, rms(y, p["next_weight"])


def params(module, prefix=""):
    return {n[len(prefix):]: p.detach().double().cpu().requires_grad_(True)
            for n, p in module.named_parameters() if n.startswith(prefix)}


def sub(p, prefix):
    return {n[len(prefix):]: v for n, v in p.items() if n.startswith(prefix)}


def gat_layer64(x, ei, W, a, NH, Fo, concat):
    """models/gat_layer.py:42-140 in float64 (self-loops already added)."""
    Wh = (x @ W.t()).view(-1, NH, Fo)
    src, dst = ei
    cat = torch.cat([Wh[src], Wh[dst]], -1).flatten(1)   # (E, NH * 2F)
    raw = cat @ a.t()
    e = torch.exp(F.leaky_relu(raw - raw.max(), 0.01))
    den = torch.zeros(x.size(0), NH, dtype=x.dtype).index_add(0, dst, e)
    alpha = e / (den[dst] + 1e-8)
    out = torch.zeros(x.size(0), NH, Fo, dtype=x.dtype).index_add(0, dst, alpha.unsqueeze(-1) * Wh[src])
    return out.flatten(1) if concat else out.mean(1)


def randomise(module, seed):
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        for n, p in module.named_parameters():
            if p.dim() == 1:
                p.add_(0.3 * torch.randn(p.shape, generator=g).to(p.device))


@pytest.mark.parametrize("skip", [[False, True, True], [True, False, False]])
def test_gat_model_with_block_norms(skip, device):
    from gatx import GATModel
    torch.manual_seed(1)
    m = GATModel(num_classes=5, num_input_node_features=20, num_layers=3,
                 num_heads_per_layer=[4, 2, 3], heads_concat_per_layer=[True, True, False],
                 head_output_features_per_layer=[20, 8, 16, 5], add_skip_connection=skip,
                 dropout=0.0, block_norm=True).to(device)
    randomise(m, 2)
    N = 60
    g = torch.Generator().manual_seed(3)
    x = torch.randn(N, 20, generator=g)
    ei = torch.randint(0, N, (2, 300), generator=g)
    ei[:, 0] = N - 1
    xd = x.to(device).requires_grad_(True)
    out, ei2, att = m.forward_and_return_attention(xd, ei.to(device))
    assert len(att) == 3 and att[0].shape[1] == 4
    go = torch.randn(out.shape, generator=g)
    out.backward(go.to(device))

    p = params(m)
    x64 = x.double().requires_grad_(True)
    e = ei2.cpu()
    s, n = x64, rms(x64, p["input_norm_weight"])
    k = 0
    for i in range(3):
        NH, Fo, concat = [4, 2, 3][i], [8, 16, 5][i], i != 2
        h = gat_layer64(n, e, p[f"gat_layer_list.{i}.W.weight"], p[f"gat_layer_list.{i}.a.weight"],
                        NH, Fo, concat)
        resid = None
        if skip[i]:
            w = p.get(f"skip_layer_list.{k}.weight")
            resid = s if w is None else s @ w.t()
            resid = resid if concat else resid.view(-1, NH, Fo).mean(1)
            k += 1
        if i == 2:
            s = h if resid is None else h + resid
        else:
            s, n = block(sub(p, f"block_norm_list.{i}."), F.elu(h), resid)
    s.backward(go.double())
    close(out, s, "out")
    close(xd.grad, x64.grad, "x")
    for n_, q in m.named_parameters():
        close(q.grad, p[n_].grad, n_)


def test_block_norm_is_off_by_default(device):
    from gatx import GATModel
    from gatx.config import data_config
    m = GATModel(**data_config["PATTERN"])
    assert not any("norm" in n for n in m.state_dict())
    m = GATModel(**data_config["PATTERN"], block_norm=True).to(device)
    x = torch.randn(50, 3, device=device)
    ei = torch.randint(0, 50, (2, 200), device=device)
    m.train()
    m.dropout = 0.2
    m(x, ei).square().sum().backward()
    for n, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), n


class Student(torch.nn.Module):
    def __init__(self, fin, width, heads, classes):
        super().__init__()
        from gatx import BlockNorm, DiffAttention
        self.inp = torch.nn.Linear(fin, width)
        self.first = torch.nn.Parameter(torch.ones(width))
        self.att = torch.nn.ModuleList(DiffAttention(width, width // heads, heads,
                                                     position_buckets=8, max_distance=20)
                                       for _ in range(2))
        self.norm = torch.nn.ModuleList(BlockNorm(width) for _ in range(2))
        self.out = torch.nn.Linear(width, classes)

    def forward(self, x, graph, pos):
        from gatx import norm_before
        s = self.inp(x)
        n = norm_before(s, self.first)
        for att, norm in zip(self.att, self.norm):
            s, n = norm(att(n, positions=pos, graph=graph), s)
        return self.out(n)


def test_student_learns_from_a_teacher(device):
    from gatx.graph import Graph
    from gatx.losses import topk_distillation
    torch.manual_seed(4)
    N, fin, width, H, C, K, T = 70, 12, 32, 4, 9, 4, 2.0
    net = Student(fin, width, H, C).to(device)
    randomise(net, 5)
    with torch.no_grad():
        for a in net.att:
            a.position_bias.normal_()
    g = torch.Generator().manual_seed(6)
    x = torch.randn(N, fin, generator=g)
    src, dst = torch.randint(0, N, (400,), generator=g), torch.randint(0, N - 5, (400,), generator=g)
    pos = torch.arange(N)
    teacher = 3 * torch.randn(N, K, generator=g)
    index = (torch.randint(0, C, (N, 1), generator=g) + 2 * torch.arange(K)) % C
    index[::7] = -1
    graph = Graph(torch.stack([src, dst]).to(device), N, False)
    xd = x.to(device).requires_grad_(True)
    loss = topk_distillation(net(xd, graph, pos.to(device)), teacher.to(device), index.to(device), T)
    loss.backward()

    p = params(net)
    x64 = x.double().requires_grad_(True)
    bucket = ref.buckets(pos[src] - pos[dst], 8, 20, True)
    s = x64 @ p["inp.weight"].t() + p["inp.bias"]
    n = rms(s, p["first"])
    d = width // H // 2
    for i in range(2):
        a = sub(p, f"att.{i}.")
        q, k, v = (n @ a["qkv.weight"].t()).split([2 * H * d, 2 * H * d, width], 1)
        q, k, v = q.view(N, H, 2, d), k.view(N, H, 2, d), v.view(N, H, width // H)
        z = (q[dst] * k[src]).sum(-1) / math.sqrt(d) + a["position_bias"][bucket].unsqueeze(-1)
        e = torch.exp(z)
        den = torch.zeros(N, H, 2, dtype=e.dtype).index_add(0, dst, e)
        w = e / den[dst]
        w = w[..., 0] - a["lam"] * w[..., 1]
        h = torch.zeros(N, H, width // H, dtype=e.dtype).index_add(0, dst, w.unsqueeze(-1) * v[src])
        s, n = block(sub(p, f"norm.{i}."), h.flatten(1), s)
    z = (n @ p["out.weight"].t() + p["out.bias"]) / T
    there = index >= 0
    t = torch.where(there, teacher.double() / T, -math.inf)
    some = there.any(1)
    pt = torch.softmax(torch.where(some[:, None], t, 0.0), 1) * there
    lq = torch.log_softmax(z, 1).gather(1, index.clamp(min=0))
    terms = torch.where(there, pt * (torch.log(pt.clamp(min=1e-300)) - lq), 0.0)
    want = T * T * terms.sum() / some.sum()
    want.backward()
    close(loss, want, "loss")
    close(xd.grad, x64.grad, "x")
    for n_, q in net.named_parameters():
        close(q.grad, p[n_].grad, n_)


def test_training_step_captured_beside_an_eager_graph(device):
    """The student's whole step, optimizer included, in a hipGraph while an eager autograd graph of
    the same parameters is alive; every replay equals an eager twin's step."""
    import copy

    from gatx.capture import CapturedStep
    from gatx.graph import Graph
    from gatx.losses import topk_distillation
    torch.manual_seed(7)
    N = 64
    net = Student(10, 32, 4, 6).to(device)
    twin = copy.deepcopy(net)
    graph = Graph(torch.randint(0, N, (2, 500), device=device), N, False)
    pos = torch.arange(N, device=device)
    x = torch.randn(N, 10, device=device)
    teacher = torch.randn(N, 3, device=device)
    index = torch.stack([torch.randperm(6, device=device)[:3] for _ in range(N)])

    def stepper(m):
        opt = torch.optim.Adam(m.parameters(), lr=1e-3, capturable=True)

        def step():
            opt.zero_grad(set_to_none=True)
            loss = topk_distillation(m(x, graph, pos), teacher, index, 2.0)
            loss.backward()
            opt.step()
            return loss.detach()
        return step
    cap = CapturedStep(stepper(net), warmup=2)
    eager = stepper(twin)
    for _ in range(2):
        eager()
    alive = topk_distillation(net(x, graph, pos), teacher, index, 2.0)   # an eager graph, kept
    for i in range(3):
        x.copy_(torch.randn(N, 10, generator=torch.Generator().manual_seed(i)))
        got = cap().clone()
        torch.cuda.synchronize()
        want = eager()
        assert torch.equal(got, want), i
    for (n, a), b in zip(net.named_parameters(), twin.parameters()):
        assert torch.equal(a, b), n
    assert torch.isfinite(alive)


def leaf_calls(device):
    """{operator: (leaf, a call on it)}"""
    from gatx import diff_attention, norm_after, norm_before
    from gatx.graph import Graph
    from gatx.losses import topk_distillation
    N = 40
    graph = Graph(torch.randint(0, N, (2, 300), device=device), N, False)
    q, k = (torch.randn(N, 2, 2, 8, device=device) for _ in range(2))
    v, lam = torch.randn(N, 2, 16, device=device), torch.rand(2, device=device)
    h, w = torch.randn(N, 24, device=device), torch.ones(24, device=device)
    t = torch.randn(N, 3, device=device)
    i = torch.randint(0, 24, (N, 3), device=device)
    return {"diff_attention": (q, lambda x: diff_attention(x, k, v, lam, graph)),
            "norm_before": (h, lambda x: norm_before(x, w)),
            "norm_after": (h, lambda x: norm_after(x, w, resid=h)),
            "topk_distillation": (h, lambda x: topk_distillation(x, t, i))}


OPERATORS = ["diff_attention", "norm_before", "norm_after", "topk_distillation"]


@pytest.mark.parametrize("name", OPERATORS)
def test_captured_backward_beside_an_eager_graph_on_the_default_stream(name, device):
    """Refused while the eager graph of the same leaf lives; captured and right once it is gone."""
    leaf, call = leaf_calls(device)[name]
    x = leaf.clone().requires_grad_(True)
    alive = call(x)
    ones = torch.ones_like(alive)
    want, = torch.autograd.grad(alive, x, ones, retain_graph=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        return torch.autograd.grad(call(x), x, ones)[0]
    with torch.cuda.stream(s):
        torch.randn(4, device=device, requires_grad=True).sum().backward()   # the engine's thread
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="alive on the default stream"):
        with torch.cuda.graph(graph, stream=s):
            step()
    torch.cuda.synchronize()
    del alive
    with torch.cuda.stream(s):
        assert torch.equal(step(), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step()
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("name", OPERATORS)
def test_forward_mode_is_refused(name, device):
    import torch.autograd.forward_ad as fw
    leaf, call = leaf_calls(device)[name]
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fw.make_dual(leaf, torch.ones_like(leaf)))


@pytest.mark.parametrize("name", OPERATORS)
def test_a_second_backward_through_freed_inputs_is_refused(name, device):
    leaf, call = leaf_calls(device)[name]
    x = leaf.clone().requires_grad_(True)
    loss = call(x).sum()
    loss.backward(retain_graph=True)
    first = x.grad.clone()
    loss.backward()
    assert torch.equal(x.grad, first + first)
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()

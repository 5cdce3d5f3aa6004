"""gatx.losses.topk_distillation against float64: types, one class to many, one slot to 1024, empty
slots and rows, repeated classes, strided and unaligned logits, extremes, gradients.

Bounds (u = 2^-24): a class's probability is exp2 of a difference of at most X = (max - min) log2(e)
/ T, whose two products and subtractions are off by 4 u X, divided by a sum of at most C such terms
of which each lane adds up to C / 8 + 64 in turn and rescales as often (3 u and its share of 2 X
u each time): eps_q = u (8 X + 4 (C / 8 + 64)) relative, and the same with K for the teacher. The
loss weighs logarithms that are off by these by p; its sum over K slots, and that over the rows, adds
K + 64 and n + 64 roundings. The gradient is rounded once to its type (finfo.eps / 2). A probability
below float32's normal range is 0 (the hardware's exp2 returns no smaller numbers): p and q are off
by up to 2^-126 more, whatever they are, which reaches the gradient times T and the loss times T^2
and the logarithms it weighs."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
FLUSH = 2.0 ** -126


def make(n, C, K, dtype, device, seed=0, empty=True, repeat=False, tdtype=None):
    g = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(n, C, generator=g)).to(dtype)
    t = (3 * torch.randn(n, K, generator=g)).to(tdtype or dtype)
    if repeat or K > C:
        i = torch.randint(0, C, (n, K), generator=g)
    else:
        i = (torch.randint(0, C, (n, 1), generator=g) + torch.arange(K)) % C
    if empty:   # rows of 0 .. K slots, in no order
        i[torch.rand(n, K, generator=g) < torch.rand(n, 1, generator=g)] = -1
    return x.to(device), t.to(device), i.to(device)


def expect(x, t, i, T):
    """(row losses, their bound, gradient of their sum, its bound) in float64."""
    x, t = x.double() / T, t.double() / T
    C, K = x.size(1), t.size(1)
    there = (i >= 0) & (t > -math.inf)
    some = there.any(1, keepdim=True)
    t = torch.where(there, t, -math.inf)
    lp = torch.where(there, t - torch.logsumexp(torch.where(some, t, 0.0), 1, True), 0.0)
    p = torch.where(there, lp.exp(), 0.0)
    lq = torch.log_softmax(x, 1)
    at = i.clamp(min=0)
    d = torch.where(p > 0, lp - lq.gather(1, at), 0.0)

    def span(z):
        fine = torch.isfinite(z)
        hi = torch.where(fine, z, -math.inf).amax(1, keepdim=True)
        lo = torch.where(fine, z, math.inf).amin(1, keepdim=True)
        return (hi - lo).clamp(min=0) / math.log(2)
    eq = U * (8 * span(x) + 4 * (C / 8 + 64))
    ep = torch.where(some, U * (8 * span(t) + 4 * (K / 8 + 64)), 0.0)
    loss = T * T * (p * d).sum(1)
    bound = T * T * ((p * (eq + ep)).sum(1) + ((ep + U * (K + 64)) * p * d.abs()).sum(1))
    bound = bound + T * T * FLUSH * torch.where(there & torch.isfinite(d), d.abs() + 1, 0.0).sum(1)
    P = torch.zeros_like(x).scatter_add_(1, at, p)
    q = torch.where(some, lq.exp(), 0.0)
    return loss, bound, T * (q - P), T * (eq * q + (ep + U * K) * P + (K + 1) * FLUSH)


def near(got, value, bound):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    x = got.double()
    limit = half * (value.abs() + bound) + bound + tiny
    ok = ((x - value).abs() <= limit) | (x == value)
    assert ok.all(), (int((~ok).sum()), float(((x - value).abs() / limit)[~ok].max()))


def run(x, t, i, T, reduction="mean", weight=None):
    from gatx.losses import topk_distillation
    x = x.detach().requires_grad_(True)
    loss = topk_distillation(x, t, i, temperature=T, reduction=reduction)
    g, = torch.autograd.grad(loss, x, weight)
    return loss.detach(), g


def check(x, t, i, T):
    n = x.size(0)
    loss, lb, grad, gb = expect(x, t, i, T)
    some = int(((i >= 0) & (t > -math.inf)).any(1).sum())
    w = torch.linspace(-2, 3, n, device=x.device)
    got, g = run(x, t, i, T, "none", w)
    near(got, loss, lb)
    near(g, w.double()[:, None] * grad, w.double().abs()[:, None] * gb
         + 4 * U * (w.double()[:, None] * grad).abs())
    total = loss.sum(), lb.sum() + U * (n + 64) * loss.abs().sum()
    for reduction, over in (("sum", 1), ("mean", max(some, 1))):
        got, g = run(x, t, i, T, reduction)
        near(got, total[0] / over, (total[1] + 2 * U * total[0].abs()) / over)
        near(g, grad / over, (gb + 4 * U * grad.abs()) / over)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,C,K", [(1, 1, 1), (3, 2, 1), (50, 7, 3), (300, 121, 16), (9, 8, 8),
                                   (20, 1024, 64), (20, 1024, 65), (20, 1025, 64), (5, 4999, 5),
                                   (3, 32000, 64), (2, 65537, 200), (4, 3000, 1024), (700, 3, 2),
                                   (600, 1500, 10), (2100, 2000, 3), (1, 131072, 64),
                                   (70000, 5, 2)])
def test_sizes(n, C, K, dtype, device):
    check(*make(n, C, K, dtype, device, seed=C), 2.0)


@pytest.mark.parametrize("T", [0.5, 1.0, 7.0])
@pytest.mark.parametrize("C", [33, 2222])
def test_temperatures_and_types(T, C, device):
    """Teacher logits of another type, int32 classes."""
    x, t, i = make(40, C, 9, torch.bfloat16, device, tdtype=torch.float32)
    check(x, t, i.int(), T)
    x, t, i = make(40, C, 9, torch.float32, device, tdtype=torch.float16)
    check(x, t, i, T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,C,K", [(30, 4, 20), (20, 7, 64), (20, 300, 100), (5, 2000, 300),
                                   (3, 5, 1024)])
def test_repeated_classes(n, C, K, dtype, device):
    """Slots of one class add up."""
    check(*make(n, C, K, dtype, device, repeat=True), 1.5)


@pytest.mark.parametrize("C", [64, 1500])
def test_no_slots(C, device):
    """No row has a slot: loss 0, gradient 0, whatever the logits hold."""
    x, t, i = make(6, C, 4, torch.float32, device)
    i[:] = -1
    x[0, 0], x[1, 1], x[2] = float("nan"), float("inf"), -float("inf")
    for r in ("mean", "sum"):
        loss, g = run(x, t, i, 1.0, r)
        assert loss.item() == 0 and not g.any()
    # a teacher of -inf is an empty slot too
    t[:] = -float("inf")
    i[:] = 0
    loss, g = run(x, t, i, 1.0)
    assert loss.item() == 0 and not g.any()


@pytest.mark.parametrize("C", [64, 1500])
def test_masked_and_bad_rows(C, device):
    """Classes at -inf (untaught: no gradient; taught: an infinite loss), NaN, classes past the
    last: each row by itself."""
    x, t, i = make(8, C, 4, torch.float32, device, empty=False)
    i[:, :] = torch.arange(4, device=device)
    x[0, 10:20] = -float("inf")
    x[1, 2] = -float("inf")
    x[2, 5] = float("nan")
    t[3, 1] = float("nan")
    i[4, 3] = C
    i[5, 0] = 2 ** 40
    x[6, 9] = torch.finfo(torch.float32).min
    t[7, 2] = -float("inf")
    loss, g = run(x, t, i, 1.0, "none", torch.ones(8, device=device))
    e, eb, ge, gb = expect(x, t, i.clamp(max=C - 1), 1.0)
    for r in (0, 6, 7):
        near(loss[r], e[r], eb[r])
        near(g[r], ge[r], gb[r] + 4 * U * ge[r].abs())
    assert not g[0, 10:20].any()
    assert loss[1] == float("inf") and torch.isfinite(g[1]).all()
    near(g[1], ge[1], gb[1] + 4 * U * ge[1].abs())
    for r in (2, 3, 4, 5):
        assert loss[r].isnan() and g[r].isnan().all(), r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [120, 1601])
def test_strided_logits(C, dtype, device):
    """Logits that are a column range of a wider tensor, at any alignment: the same bounds; their
    gradient lands in the range."""
    from gatx.losses import topk_distillation
    x, t, i = make(20, C, 5, dtype, device)
    _, _, grad, gb = expect(x, t, i, 1.0)
    for off in (0, 1, 8):
        wide = torch.full((20, C + 9), float("nan"), dtype=dtype, device=device)
        wide[:, off:off + C] = x
        wide.requires_grad_(True)
        loss = topk_distillation(wide[:, off:off + C], t, i, reduction="sum")
        g, = torch.autograd.grad(loss, wide)
        near(g[:, off:off + C], grad, gb + 4 * U * grad.abs())
        assert not g[:, :off].any() and not g[:, off + C:].any()
    near(run(x.t().contiguous().t(), t, i, 1.0, "sum")[1], grad, gb + 4 * U * grad.abs())


def test_large_logits(device):
    """Logits far from zero: only their differences count."""
    for C in (50, 3000):
        x, t, i = make(10, C, 6, torch.float32, device)
        check(x * 100 + 3000, t * 20 - 5000, i, 2.0)


def test_gradient_against_differences(device):
    """Central differences of the float64 loss, step 1e-4: far below 1e-3 of the lengths."""
    x, t, i = make(9, 40, 6, torch.float32, device)
    _, g = run(x, t, i, 2.0, "sum")
    u = torch.randn(9, 40, generator=torch.Generator().manual_seed(3)).double().to(device)
    f = [float(expect(x.double() + s * 1e-4 * u, t, i, 2.0)[0].sum()) for s in (1, -1)]
    want = (f[0] - f[1]) / 2e-4
    assert abs(float((g.double() * u).sum()) - want) <= 1e-3 * float(g.norm() * u.norm())


@pytest.mark.parametrize("C", [121, 3001])
def test_same_bits_every_time_and_captured(C, device):
    from gatx.capture import CapturedStep
    x, t, i = make(900, C, 16, torch.bfloat16, device, repeat=True)
    a, b = run(x, t, i, 2.0), run(x, t, i, 2.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    cap = CapturedStep(lambda: run(x, t, i, 2.0))
    for s in range(3):
        x.copy_(make(900, C, 16, torch.bfloat16, device, seed=s)[0])
        got = [y.clone() for y in cap()]
        torch.cuda.synchronize()
        want = run(x, t, i, 2.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), s


def test_loss_scaled_in_place(device):
    """The loss may be changed in place before its backward (gradient accumulation)."""
    from gatx.losses import topk_distillation
    x, t, i = make(30, 20, 4, torch.float32, device)
    want = run(x, t, i, 1.0)[1] / 4
    x.requires_grad_(True)
    loss = topk_distillation(x, t, i)
    loss /= 4
    loss.backward()
    assert torch.equal(x.grad, want)


def test_no_rows(device):
    loss, g = run(torch.zeros(0, 9, device=device), torch.zeros(0, 2, device=device),
                  torch.zeros(0, 2, dtype=torch.int64, device=device), 1.0)
    assert loss.item() == 0 and g.shape == (0, 9)


def test_module(device):
    from gatx.losses import TopKDistillationLoss, topk_distillation
    x, t, i = make(30, 20, 4, torch.float32, device)
    assert torch.equal(TopKDistillationLoss(3.0, "sum")(x, t, i),
                       topk_distillation(x, t, i, 3.0, "sum"))

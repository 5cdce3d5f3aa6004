"""gatx.norm_before / norm_after against float64: types, odd and wide rows, every set of optional
parts, strided rows, gradients against the formula and against differences.

Bounds (u = 2^-24): a row's sum of squares is a tree of at most 40 float32 additions of positive
terms, a normalised value passes two such sums, the sigmoid 4 + |gate| roundings and at most 16
products, so each result is off by at most K u times the sum of the magnitudes of the terms it is
made of, K = 256 (the gates drawn here stay within 8); `mag` below computes that sum with every
difference taken as a sum. Column sums over n rows add n + 64 roundings. Rows and gradients of rows
are then rounded once to their type (finfo.eps / 2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U, K = 2.0 ** -24, 256
EPS = 1e-6


def make(n, D, dtype, device, resid, gate, scale, following, seed=0):
    g = torch.Generator().manual_seed(seed)

    def rows():
        return torch.randn(n, D, generator=g).to(dtype).to(device)

    def cols(about):
        return (about + 0.3 * torch.randn(D, generator=g)).to(device)
    return {"h": rows(), "weight": cols(1.0), "resid": rows() if resid else None,
            "gate": {None: None, "rows": rows(), "cols": cols(0.2)}[gate],
            "scale": cols(0.7) if scale else None, "next_weight": cols(1.0) if following else None,
            "gy": rows(), "gn": rows() if following else None}


def expect(t):
    """{name: (value, magnitude)} in float64, on the device."""
    f = {n: None if x is None else x.double() for n, x in t.items()}
    n, D = f["h"].shape
    one = torch.ones(1, dtype=torch.float64, device=f["h"].device)

    def mean(x):
        return x.mean(-1, keepdim=True)
    rh = (mean(f["h"] ** 2) + EPS).rsqrt()
    hn = f["h"] * rh
    sg = one if f["gate"] is None else torch.sigmoid(f["gate"])
    sc = one if f["scale"] is None else f["scale"]
    w = f["weight"]
    c = sc * sg * w
    y, ya = c * hn, (c * hn).abs()
    if f["resid"] is not None:
        y, ya = y + f["resid"], ya + f["resid"].abs()
    out = {"y": (y, ya)}
    g, ga = f["gy"], f["gy"].abs()
    if f["next_weight"] is not None:
        wn = f["next_weight"]
        ry = (mean(y ** 2) + EPS).rsqrt()
        R = torch.clamp(mean(ya ** 2) * ry ** 2, min=1.0)   # how far ya can outgrow y in ry
        yn, yna = y * ry, ya * ry * R
        out["next"] = (yn * wn, yna * wn.abs())
        u = f["gn"] * wn
        g = g + ry * (u - yn * mean(u * yn))
        ga = ga + ry * R * (u.abs() + yna * mean(u.abs() * yna))
        out["next_weight"] = ((f["gn"] * yn).sum(0), (f["gn"].abs() * yna).sum(0))
    if f["resid"] is not None:
        out["resid"] = (g, ga)
    a, aa = g * sg * hn, ga * sg * hn.abs()
    out["weight"] = ((a * sc).sum(0), (aa * sc.abs()).sum(0))
    if f["scale"] is not None:
        out["scale"] = ((a * w).sum(0), (aa * w.abs()).sum(0))
    if f["gate"] is not None:
        gg, gga = a * sc * w * (1 - sg), aa * (sc * w).abs()
        out["gate"] = (gg, gga) if f["gate"].dim() == 2 else (gg.sum(0), gga.sum(0))
    x, xa = g * c, ga * c.abs()
    out["h"] = (rh * (x - hn * mean(x * hn)), rh * (xa + hn.abs() * mean(xa * hn.abs())))
    return out


def run(t, f=None):
    from gatx import norm_after
    names = [n for n in ("h", "weight", "resid", "gate", "scale", "next_weight")
             if t[n] is not None]
    x = {n: t[n].detach().requires_grad_(True) for n in names}
    r = (f or norm_after)(x["h"], x["weight"], resid=x.get("resid"), gate=x.get("gate"),
                          scale=x.get("scale"), next_weight=x.get("next_weight"), eps=EPS)
    outs = list(r) if "next_weight" in x else [r]
    gos = [t["gy"], t["gn"]][:len(outs)]
    got = dict(zip(("y", "next"), (o.detach() for o in outs)))
    got.update(zip(names, torch.autograd.grad(outs, [x[n] for n in names], gos)))
    return got


def check(got, want, n):
    assert set(got) == set(want)
    for name, (value, mag) in want.items():
        x = got[name].double()
        summed = name in ("weight", "scale", "next_weight") or got[name].dim() == 1
        dt = got[name].dtype
        k = K + (n + 64 if summed else 0)
        half = torch.finfo(dt).eps / 2
        tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        limit = half * (value.abs() + k * U * mag) + k * U * mag + tiny
        bad = ~((x - value).abs() <= limit)
        assert not bad.any(), (name, int(bad.sum()), float(((x - value).abs() / limit)[bad].max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D", [(1, 1), (1, 1024), (5, 3), (3, 48), (33, 121), (7, 512),
                                 (100, 1024), (9, 1000), (3, 2049), (5, 4096), (2, 8192),
                                 (2, 8191), (3, 4100), (3000, 96), (1, 7)])
def test_all_parts(n, D, dtype, device):
    t = make(n, D, dtype, device, True, "rows", True, True, seed=D)
    check(run(t), expect(t), n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("resid", [False, True])
@pytest.mark.parametrize("gate", [None, "rows", "cols"])
@pytest.mark.parametrize("scale,following", [(False, False), (True, False), (False, True),
                                             (True, True)])
@pytest.mark.parametrize("n,D", [(70, 48), (17, 121), (9, 2048)])
def test_parts(n, D, resid, gate, scale, following, dtype, device):
    t = make(n, D, dtype, device, resid, gate, scale, following, seed=n)
    check(run(t), expect(t), n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D", [(1, 1), (40, 48), (33, 121), (2, 8191), (1500, 1024)])
def test_norm_before(n, D, dtype, device):
    from gatx import norm_before
    t = make(n, D, dtype, device, False, None, False, True)
    x, w = t["h"].detach().requires_grad_(True), t["weight"].detach().requires_grad_(True)
    out = norm_before(x, w, eps=EPS)
    gx, gw = torch.autograd.grad(out, [x, w], t["gn"])
    f, wd, g = x.detach().double(), w.detach().double(), t["gn"].double()
    r = ((f * f).mean(-1, keepdim=True) + EPS).rsqrt()
    u, yn = g * wd, f * r
    m, ma = (u * yn).mean(-1, keepdim=True), (u * yn).abs().mean(-1, keepdim=True)
    check({"next": out.detach(), "h": gx, "next_weight": gw},
          {"next": (yn * wd, (yn * wd).abs()),
           "h": (r * (u - yn * m), r * (u.abs() + yn.abs() * ma)),
           "next_weight": ((g * yn).sum(0), (g * yn).abs().sum(0))}, n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows_and_shapes(dtype, device):
    """Rows that are column ranges of a wider tensor, three dimensions, one row: the same bits."""
    t = make(60, 64, dtype, device, True, "rows", True, True)
    a = run(t)
    s = dict(t)
    for n in ("h", "resid", "gate", "gy", "gn"):
        wide = torch.full((60, 3 * 64), float("nan"), dtype=dtype, device=device)
        wide[:, 64:128] = t[n]
        s[n] = wide[:, 64:128]
    b = run(s)
    from gatx import norm_after

    def folded(h, weight, resid, gate, **kw):
        r = norm_after(h.view(5, 12, 64), weight, resid=resid.view(5, 12, 64),
                       gate=gate.view(5, 12, 64), **kw)
        assert r[0].shape == (5, 12, 64)
        return tuple(x.reshape(60, 64) for x in r)
    c = run(t, folded)
    for n in a:
        assert torch.equal(a[n], b[n]) and torch.equal(a[n], c[n]), n
    one = norm_after(t["h"][7], t["weight"], resid=t["resid"][7], gate=t["gate"][7],
                     scale=t["scale"], next_weight=t["next_weight"], eps=EPS)
    assert torch.equal(one[0], a["y"][7]) and torch.equal(one[1], a["next"][7])
    # rows of another alignment (an odd offset) take single elements: within the same bounds
    for n in ("h", "resid", "gate"):
        wide = torch.zeros((60, 65), dtype=dtype, device=device)
        wide[:, 1:] = t[n]
        s[n] = wide[:, 1:]
    check(run(s), expect(t), 60)


def test_no_rows_and_zero_rows(device):
    """No rows: empty results, zero gradients. Rows of zeros: finite, the residual alone."""
    t = make(0, 32, torch.float32, device, True, "cols", True, True)
    got = run(t)
    assert got["y"].shape == (0, 32)
    for n in ("weight", "scale", "gate", "next_weight"):
        assert got[n].shape == (32,) and not got[n].any(), n
    t = make(4, 32, torch.float32, device, True, "cols", True, True)
    t["h"].zero_()
    t["resid"][0].zero_()
    check(run(t), expect(t), 4)


def test_one_output_used(device):
    """A gradient through y alone or next alone: the other counts as zero."""
    from gatx import norm_after
    t = make(50, 96, torch.float32, device, True, "rows", True, True)
    for which, zero in ((0, "gn"), (1, "gy")):
        x = {n: t[n].detach().requires_grad_(True)
             for n in ("h", "weight", "resid", "gate", "scale", "next_weight")}
        r = norm_after(x["h"], x["weight"], resid=x["resid"], gate=x["gate"], scale=x["scale"],
                       next_weight=x["next_weight"], eps=EPS)
        g = torch.autograd.grad(r[which], list(x.values()), t[("gy", "gn")[which]],
                                allow_unused=True)
        s = dict(t)
        s[zero] = torch.zeros_like(t[zero])
        want = expect(s)
        got = dict(zip(x, g))
        if which == 0:
            assert got.pop("next_weight") is None
            want.pop("next_weight")
        want = {n: want[n] for n in got}
        check(got, want, 50)


def test_gradients_against_differences(device):
    """Central differences of the float64 definition along random directions, step 1e-4: their own
    error (h^2) and the bounds above are far below 1e-3 of the lengths involved."""
    for gate in ("rows", "cols"):
        t = make(12, 40, torch.float32, device, True, gate, True, True)
        got = run(t)
        for n in ("h", "weight", "resid", "gate", "scale", "next_weight"):
            u = torch.randn(t[n].shape, generator=torch.Generator().manual_seed(2)).double()
            u = u.to(device)
            base, h = t[n].double(), 1e-4

            def f(x):
                e = expect({**t, n: x})
                return float((e["y"][0] * t["gy"].double()).sum()
                             + (e["next"][0] * t["gn"].double()).sum())
            want = (f(base + h * u) - f(base - h * u)) / (2 * h)
            grad = got[n].double()
            assert abs(float((grad * u).sum()) - want) <= 1e-3 * float(grad.norm() * u.norm()), n


def test_same_bits_every_time_and_captured(device):
    from gatx.capture import CapturedStep
    t = make(5000, 1024, torch.bfloat16, device, True, "rows", True, True)
    a, b = run(t), run(t)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    cap = CapturedStep(lambda: run(t))
    for i in range(3):
        t["h"].copy_(make(5000, 1024, torch.bfloat16, device, False, None, False, False,
                          seed=i)["h"])
        got = {n: x.clone() for n, x in cap().items()}
        torch.cuda.synchronize()
        want = run(t)
        for n in want:
            assert torch.equal(got[n], want[n]), (i, n)


def test_module(device):
    from gatx import BlockNorm
    m = BlockNorm(48).to(device)
    h, r = (torch.randn(30, 48, device=device) for _ in range(2))
    y, n = m(h, r)
    want = r + 0.5 * h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    assert torch.allclose(y, want, atol=1e-5)
    (y.sum() + n.square().sum()).backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    assert BlockNorm(48, gate=False, following=False).to(device)(h).shape == (30, 48)

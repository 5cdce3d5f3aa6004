"""Differential neighbourhood attention in float64 on the host, edge by edge from its definition,
with the forward-error bounds the GPU tests hold the kernels to.

Bounds (u = 2^-24, one rounding in float32): a logit passes at most 8 + 5 + 2 roundings (8-element
chunk, 5 exchanges, scale and bias) of terms that add up to X = sum |q k| |scale| + |bias|; the
difference from the maximum and its product with log2 e two more of at most 2 X; the maximum itself
cancels in the softmax. A weight p is a quotient of two such exponentials, of a sum of n of them, and
is rescaled (a product of exponentials of differences that telescope to at most 2 X, each off by
3 u) at most n times: its relative error is within eps = u (40 X + 4 n + 64), sums of n weighted
values included. dw = go . v is off by 24 u W, W = sum |go v|, and so dx = p (dw - D) by 6 eps p Wmax
(Wmax over the row). Each result is then rounded once to its type (finfo.eps / 2)."""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def buckets(rel, num_buckets, max_distance, bidirectional):
    """The bucket of each relative position, from whole-number comparisons."""
    n = num_buckets // 2 if bidirectional else num_buckets
    m = n // 2
    out = []
    for r in rel.tolist():
        away = abs(r) if bidirectional else max(-r, 0)
        b = min(away, m)
        # bucket m + j holds the distances x with x^(n-m) >= m^(n-m-j) max_distance^j
        for j in range(1, n - m):
            b += away ** (n - m) >= m ** (n - m - j) * max_distance ** j
        out.append(b + (n if bidirectional and r > 0 else 0))
    return torch.tensor(out, dtype=torch.int64)


def attention(q, k, v, lam, src, dst, row_of, scale, bias=None, bucket=None, go=None):
    """{name: (value, bound without the final rounding)}. All tensors float64 on the host; dst the
    destination node of each edge, row_of[dst] its row in q."""
    M, H = q.shape[:2]
    row = row_of[dst]
    n_of = torch.bincount(row, minlength=M).double()

    def by(index, x, size):
        return torch.zeros((size,) + x.shape[1:], dtype=x.dtype).index_add_(0, index, x)

    x = (q[row] * k[src]).sum(-1) * scale
    X = (q[row] * k[src]).abs().sum(-1) * scale
    shut = torch.zeros_like(x, dtype=torch.bool)
    if bias is not None:
        b = bias[bucket].unsqueeze(-1)
        shut = (b == -float("inf")).expand_as(x)
        x = x + torch.where(shut, 0.0, b)
        X = X + torch.where(shut, 0.0, b.abs())
    # what a shut edge points at may be anything: it does not take part
    x, X = torch.where(shut, -float("inf"), x), torch.where(shut, 0.0, X)
    top = torch.full((M, H, 2), -float("inf"), dtype=x.dtype)
    top = top.scatter_reduce(0, row.view(-1, 1, 1).expand_as(x), x, "amax")
    e = torch.where(shut, 0.0, torch.exp(x - torch.where(torch.isinf(top), 0.0, top)[row]))
    total = by(row, e, M)
    p = e / torch.where(total == 0, 1.0, total)[row]
    w = p[..., 0] - lam * p[..., 1]
    A = p[..., 0] + lam.abs() * p[..., 1]
    Xm = torch.zeros((M, H), dtype=x.dtype).scatter_reduce(
        0, row.view(-1, 1).expand(-1, H), X.amax(-1), "amax") if len(row) else torch.zeros(M, H)
    eps = U32 * (40 * Xm + 4 * n_of.view(-1, 1) + 64)
    vs = torch.where(shut[..., :1], 0.0, v[src])
    out = {"out": (by(row, w.unsqueeze(-1) * vs, M),
                   eps.unsqueeze(-1) * by(row, A.unsqueeze(-1) * vs.abs(), M))}
    if go is None:
        return out
    N = k.size(0)
    gs = go[row]
    dw, W = (gs * vs).sum(-1), (gs * vs).abs().sum(-1)
    Wm = torch.zeros((M, H), dtype=x.dtype).scatter_reduce(
        0, row.view(-1, 1).expand(-1, H), W, "amax") if len(row) else torch.zeros(M, H)
    D = by(row, p * dw.unsqueeze(-1), M)
    sign = torch.stack([torch.ones_like(lam), -lam], -1)
    dx = sign * p * (dw.unsqueeze(-1) - D[row])
    ex = sign.abs() * p * (6 * eps * Wm)[row].unsqueeze(-1)   # its bound
    ks = torch.where(shut.unsqueeze(-1), 0.0, k[src])
    qs = torch.where(shut.unsqueeze(-1), 0.0, q[row])
    gs = torch.where(shut[..., :1], 0.0, gs)
    cnt = torch.bincount(src, minlength=N).double()
    row_sum = U32 * (n_of + 8).view(-1, 1, 1, 1)
    src_sum = U32 * (cnt + 8).view(-1, 1, 1, 1)
    a = dx.abs().unsqueeze(-1)
    out["q"] = (scale * by(row, dx.unsqueeze(-1) * ks, M),
                scale * (by(row, ex.unsqueeze(-1) * ks.abs(), M)
                         + row_sum * by(row, a * ks.abs(), M)))
    out["k"] = (scale * by(src, dx.unsqueeze(-1) * qs, N),
                scale * (by(src, ex.unsqueeze(-1) * qs.abs(), N)
                         + src_sum * by(src, a * qs.abs(), N)))
    ev = (eps[row] * A).unsqueeze(-1) * gs.abs()
    out["v"] = (by(src, w.unsqueeze(-1) * gs, N),
                by(src, ev, N) + src_sum[..., 0] * by(src, w.abs().unsqueeze(-1) * gs.abs(), N))
    out["lam"] = (-D[..., 1].sum(0), (2 * eps * Wm).sum(0) + U32 * (M + 8) * D[..., 1].abs().sum(0))
    if bias is not None:
        nb = bias.size(0)
        s = dx.sum(-1)
        out["bias"] = (by(bucket, s, nb),
                       by(bucket, ex.sum(-1), nb)
                       + U32 * (len(row) + 8) * by(bucket, dx.abs().sum(-1), nb))
    return out


def check(got, want, name):
    value, bound = want
    got64 = got.detach().double().cpu()
    assert got64.shape == value.shape, (name, got64.shape, value.shape)
    # results below the type's normal range are off by up to half its smallest step instead
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    limit = half_step(got.dtype) * (value.abs() + bound) + bound + tiny
    bad = ~((got64 - value).abs() <= limit)
    assert not bad.any(), (name, int(bad.sum()), bad.numel(),
                           float(((got64 - value).abs() / limit)[bad].max()))

"""Cases of the graph-transformer operators: differential neighbourhood attention (with and
without the learned relative position bias), the norms around a block, and top-k distillation.

Each case is one pass of one operator, as a training step or a server runs it. `own` False: the
plain form in elementary torch operations, in float32, rounded once at the end; True: gatx's
kernels. `exact` restates the definition in float64, a head (or a block of rows) at a time."""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def _attn(name, dtype, train, graphs, nodes, edges, heads, d, dv, buckets=0, max_distance=128,
          bidirectional=True, window=False, skew=False, serve=0):
    """graphs x (nodes, edges + one self-loop a node); serve = m > 0: m nodes of `edges` random
    in-neighbours each are asked for, out of `nodes` whose keys and values are at hand."""
    return {"name": name, "op": "attention", "dtype": dtype, "train": train, "graphs": graphs,
            "nodes": nodes, "edges": edges, "heads": heads, "d": d, "dv": dv, "buckets": buckets,
            "max_distance": max_distance, "bidirectional": bidirectional, "window": window,
            "skew": skew, "serve": serve}


def _norm(name, dtype, train, rows, cols, resid, gate, after, following):
    """gate: "none", "row" (one value an element) or "vector" (a parameter); after False: the norm
    before the block alone; following: the next block's norm in the same call."""
    return {"name": name, "op": "norm", "dtype": dtype, "train": train, "rows": rows, "cols": cols,
            "resid": resid, "gate": gate, "after": after, "following": following}


def _distill(name, dtype, train, rows, classes, k, temperature, empty):
    """empty: a share of the rows carries no teacher at all, and of the others some fewer than k."""
    return {"name": name, "op": "distill", "dtype": dtype, "train": train, "rows": rows,
            "classes": classes, "k": k, "temperature": temperature, "empty": empty}


def listed():
    return [
        # the hidden layer of the PPI stack (4 heads of 256) on the 20 training graphs: a step
        _attn("attn_ppi_train_bf16", "bf16", True, 20, 2245, 61318, 4, 128, 256),
        # its last layer (6 heads of 121) in float32 on the same batch: evaluation, odd widths
        _attn("attn_ppi_eval_fp32", "fp32", False, 20, 2245, 61318, 6, 61, 121),
        # PATTERN's batch of 8 graphs, 4 heads of 12: a small training step, latency-bound
        _attn("attn_pattern_train_fp32", "fp32", True, 8, 119, 6099, 4, 6, 12),
        # one node with 65 537 neighbours asked for, keys and values resident: serving
        _attn("attn_one_node_bf16", "bf16", False, 1, 70000, 65537, 8, 64, 128, serve=1),
        # the PPI batch with node order as positions: 32 signed log buckets, a training step
        _attn("bias_ppi_train_fp16", "fp16", True, 20, 2245, 61318, 4, 64, 128, buckets=32),
        # the Cora graph (8 heads of 8), past only, far neighbours masked out: evaluation
        _attn("bias_cora_eval_fp32", "fp32", False, 1, 2708, 10556, 8, 4, 8, buckets=16,
              max_distance=512, bidirectional=False, window=True),
        # the PPI hidden state (4 x 256 wide) between two blocks, gated by a projection: a step
        _norm("norm_ppi_train_bf16", "bf16", True, 44900, 1024, True, "row", True, True),
        # PATTERN's (4 x 12 wide), gated by a parameter: a small step
        _norm("norm_pattern_train_fp32", "fp32", True, 952, 48, True, "vector", True, True),
        # one row between two blocks: serving a single node
        _norm("norm_one_row_bf16", "bf16", False, 1, 1024, True, "row", True, True),
        # a wide classifier learning from 64 kept logits a row: a training step
        _distill("distill_wide_train_bf16", "bf16", True, 8192, 32000, 64, 2.0, False),
        # PPI's 121 outputs from a teacher's 16 best, some rows without a teacher: a step
        _distill("distill_ppi_train_fp32", "fp32", True, 44900, 121, 16, 1.0, True),
        # Cora's 7 classes from the 3 best: the smallest step
        _distill("distill_cora_train_fp32", "fp32", True, 2708, 7, 3, 4.0, False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    op = rng.choice(["attention", "bias", "norm", "distill"])
    if op in ("attention", "bias"):
        heads, d = rng.randint(1, 8), _log(rng, 1, 128)
        dv = rng.choice([2 * d, 2 * d, _log(rng, 1, 256)])
        if rng.random() < 0.3:
            heads = rng.choice([1, 2, 4, 8])
            d = rng.choice([8, 16, 32, 64, 128])
            dv = rng.choice([d, 2 * d])
        graphs = _log(rng, 1, 24)
        nodes = _log(rng, 1, 45000 // graphs)
        edges = int(nodes * math.exp(rng.uniform(math.log(0.5), math.log(60.0))))
        # no dearer than the PPI batch's step
        edges = min(edges, int(6.0e8 / (graphs * heads * (2 * d + dv))), 1200000 // graphs)
        serve = 0
        train = rng.random() < 0.6
        if rng.random() < 0.2:
            graphs, train, serve = 1, False, _log(rng, 1, 40)
            nodes, edges = _log(rng, 300, 100000), _log(rng, 1, 80000 // serve)
        buckets, far, both, window = 0, 128, True, False
        if op == "bias":
            both = rng.random() < 0.5
            buckets = rng.choice([8, 16, 32, 64, 128])
            far = _log(rng, buckets, 4 * 2245)
            window = rng.random() < 0.3
        c = _attn("", dtype, train, graphs, nodes, max(edges, 1), heads, d, dv, buckets, far,
                  both, window, rng.random() < 0.3, serve)
    elif op == "norm":
        cols = _log(rng, 3, 8192)
        rows = _log(rng, 1, min(100000, 46000000 // cols))
        after = rng.random() < 0.8
        c = _norm("", dtype, rng.random() < 0.7, rows, cols, after and rng.random() < 0.7,
                  rng.choice(["none", "row", "vector"]) if after else "none", after,
                  not after or rng.random() < 0.7)
    else:
        classes = _log(rng, 2, 131072)
        rows = _log(rng, 1, min(60000, 260000000 // classes))
        c = _distill("", dtype, rng.random() < 0.7, rows, classes,
                     _log(rng, 1, min(classes, 256)), rng.choice([1.0, 2.0, 4.0]),
                     rng.random() < 0.4)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------- inputs

def _package():
    """gatx, from the checkout this file lies in (only where own is true)."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "gat-pytorch_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def _edges(c, g):
    """(sources, destinations) of every edge, int64, in a random order."""
    dev = g.device
    if c["serve"]:
        asked = torch.randperm(c["nodes"], generator=g, device=dev)[:c["serve"]]
        dst = asked.repeat_interleave(c["edges"])
        return torch.randint(0, c["nodes"], dst.shape, generator=g, device=dev), dst, asked
    G, n, e = c["graphs"], c["nodes"], c["edges"]
    off = (torch.arange(G, device=dev) * n).repeat_interleave(e)
    u = torch.rand(2, G * e, generator=g, device=dev, dtype=torch.float64)
    if c["skew"]:   # few nodes with most of the edges, as in graphs with hubs
        u = u ** 3
    src, dst = ((u * n).long().clamp_(max=n - 1) + off)
    loops = torch.arange(G * n, device=dev)
    return torch.cat([src, loops]), torch.cat([dst, loops]), None


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(1000003 * int(seed) + 17)
    dt = _DT[c["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=dev).to(dtype)

    if c["op"] == "attention":
        H, d, dv = c["heads"], c["d"], c["dv"]
        src, dst, asked = _edges(c, g)
        N = c["graphs"] * c["nodes"]
        M = N if asked is None else c["serve"]
        s = {"case": c, "src": src, "dst": dst, "asked": asked, "q": normal(M, H, 2, d),
             "k": normal(N, H, 2, d), "v": normal(N, H, dv),
             "lam": 0.2 + 0.6 * torch.rand(H, generator=g, device=dev),
             "go": normal(M, H, dv) if c["train"] else None, "bias": None, "positions": None}
        if c["buckets"]:
            s["bias"] = normal(c["buckets"], H, dtype=torch.float32)
            if c["window"]:   # the farthest buckets are shut
                s["bias"][c["buckets"] - 1] = -math.inf
                if c["bidirectional"]:
                    s["bias"][c["buckets"] // 2 - 1] = -math.inf
            s["positions"] = torch.arange(c["nodes"], device=dev).repeat(c["graphs"])
        s["graph"] = None
        if own:   # the graph's CSR and its transpose: what a program keeps for its edges
            _package()
            from gatx.graph import Graph
            s["graph"] = Graph(torch.stack([src, dst]), N, False)
            if c["train"]:
                s["graph"].ensure_transpose()
        return s
    if c["op"] == "norm":
        n, D = c["rows"], c["cols"]

        def parameter(about):
            return about + 0.2 * torch.randn(D, generator=g, device=dev)

        return {"case": c, "h": normal(n, D), "weight": parameter(1.0) if c["after"] else None,
                "resid": normal(n, D) if c["resid"] else None,
                "gate": {"none": None, "row": normal(n, D) if c["gate"] == "row" else None,
                         "vector": parameter(0.5)}[c["gate"]],
                "scale": parameter(0.6) if c["after"] else None,
                "next_weight": parameter(1.0) if c["following"] else None,
                "gy": normal(n, D) if c["train"] and c["after"] else None,
                "gn": normal(n, D) if c["train"] and c["following"] else None}
    n, C, K = c["rows"], c["classes"], c["k"]
    logits = (2.0 * torch.randn(n, C, generator=g, device=dev)).to(dt)
    teacher = (3.0 * torch.randn(n, K, generator=g, device=dev)).to(dt)
    # a row's kept classes, all different: an offset and a stride that shares no factor with C
    stride = max(1, C // K)
    index = (torch.randint(0, C, (n, 1), generator=g, device=dev)
             + stride * torch.arange(K, device=dev)) % C
    if c["empty"]:
        kept = torch.randint(0, K + 1, (n, 1), generator=g, device=dev)
        index = torch.where(torch.arange(K, device=dev) < kept, index, -1)
    return {"case": c, "logits": logits, "teacher": teacher, "index": index}


# ---------------------------------------------------------------------------- the plain forms

_EPS = 1e-6


def _bounds(c):
    """The smallest distance that falls into each bucket past the exact ones: bucket m + j holds
    the distances from m (far / m)^(j / (n - m)) on, n buckets a side, the first m = n // 2 of
    them one distance each."""
    n = c["buckets"] // 2 if c["bidirectional"] else c["buckets"]
    m = n // 2
    at = []
    for j in range(1, n - m):
        x = max(m, int(m * (c["max_distance"] / m) ** (j / (n - m))) - 2)
        while x ** (n - m) * m ** j < m ** (n - m) * c["max_distance"] ** j:
            x += 1
        at.append(x)
    return n, m, at


def _buckets(c, relative):
    """The bucket of each relative position (source minus destination)."""
    n, m, at = _bounds(c)
    away = relative.abs() if c["bidirectional"] else (-relative).clamp(min=0)
    past = torch.bucketize(away, torch.tensor(at, device=relative.device, dtype=torch.int64),
                           right=True)
    b = torch.where(away < m, away, m + past)
    return b + n * (relative > 0) if c["bidirectional"] else b


def _plain_attention(s, q, k, v, lam, bias):
    c, src, dst = s["case"], s["src"], s["dst"]
    row = dst
    if s["asked"] is not None:
        row = torch.empty(k.size(0), dtype=torch.int64, device=k.device)
        row[s["asked"]] = torch.arange(q.size(0), device=k.device)
        row = row[dst]
    x = (q[row] * k[src]).sum(-1) / math.sqrt(c["d"])          # (E, H, 2)
    shut = torch.zeros_like(x, dtype=torch.bool)
    if bias is not None:
        b = _buckets(c, s["positions"][src] - s["positions"][dst])
        # through float64, and 1024 copies of the table in turn: its gradient sums every edge of
        # a bucket, and a scatter to a few rows alone would be most of the step
        turn = torch.arange(b.numel(), device=b.device) % 1024
        b = bias.double().repeat(1024, 1)[b + c["buckets"] * turn].float().unsqueeze(-1)
        shut = shut | (b == -math.inf)
        x = x + torch.where(b == -math.inf, 0.0, b)
    at = row.view(-1, 1, 1).expand_as(x)
    top = torch.full((q.size(0),) + x.shape[1:], -math.inf, device=x.device)
    top = top.scatter_reduce(0, at, torch.where(shut, -math.inf, x).detach(), "amax")
    e = torch.where(shut, 0.0, torch.exp(torch.where(shut, 0.0, x - top[row])))
    total = torch.zeros_like(top).index_add(0, row, e)
    p = e / torch.where(total == 0, 1.0, total)[row]
    w = p[..., 0] - lam * p[..., 1]
    out = torch.zeros(q.size(0), v.size(1), v.size(2), device=x.device)
    return out.index_add(0, row, w.unsqueeze(-1) * v[src])


def _plain_norm(h, weight, resid, gate, scale, next_weight):
    y = h
    if weight is not None:
        y = scale * (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS)) * weight
        if gate is not None:
            y = y / (1 + torch.exp(-gate))
        if resid is not None:
            y = resid + y
    n = None
    if next_weight is not None:
        n = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * next_weight
    return y, n


def _plain_distill(c, logits, teacher, index):
    T = c["temperature"]
    there = index >= 0
    at = index.clamp(min=0)
    t = torch.where(there, teacher / T, -math.inf)
    some = there.any(-1)
    t = torch.where(some.unsqueeze(-1), t, 0.0)
    t = t - t.amax(-1, keepdim=True)
    lse_t = torch.log(torch.exp(t).sum(-1, keepdim=True))
    lp = torch.where(there, t - lse_t, 0.0)
    p = torch.where(there, torch.exp(lp), 0.0)
    x = logits / T
    x = x - x.detach().amax(-1, keepdim=True)
    lq = x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    row = (T * T) * (p * (lp - lq.gather(1, at))).sum(-1)
    return row.sum() / some.sum().clamp(min=1)


def _leaf(t):
    return None if t is None else t.detach().float().requires_grad_(True)


def _grads(outs, gos, names, leaves, dtypes):
    pairs = [(o, g.float()) for o, g in zip(outs, gos) if g is not None]
    got = torch.autograd.grad([o for o, _ in pairs], leaves, [g for _, g in pairs])
    return {n: g.to(t) for n, g, t in zip(names, got, dtypes)}


def _run_plain(s):
    c = s["case"]
    dt = _DT[c["dtype"]]
    f32 = torch.float32
    if c["op"] == "attention":
        if not c["train"]:
            q, k, v = (s[n].float() for n in ("q", "k", "v"))
            return {"out": _plain_attention(s, q, k, v, s["lam"], s["bias"]).to(dt)}
        q, k, v, lam, bias = (_leaf(s[n]) for n in ("q", "k", "v", "lam", "bias"))
        out = _plain_attention(s, q, k, v, lam, bias)
        names, leaves, types = ["q", "k", "v", "lam"], [q, k, v, lam], [dt, dt, dt, f32]
        if bias is not None:
            names, leaves, types = names + ["bias"], leaves + [bias], types + [f32]
        return {"out": out.detach().to(dt), **_grads([out], [s["go"]], names, leaves, types)}
    if c["op"] == "norm":
        names = ["h", "weight", "resid", "gate", "scale", "next_weight"]
        ins = [_leaf(s[n]) for n in names]
        if not c["train"]:
            with torch.no_grad():
                y, n = _plain_norm(*ins)
        else:
            y, n = _plain_norm(*ins)
        r = {"y": y.detach().to(dt)} if c["after"] else {}
        if n is not None:
            r["next"] = n.detach().to(dt)
        if c["train"]:
            here = [(a, x, s[a].dtype) for a, x in zip(names, ins) if x is not None]
            outs = [(o, g) for o, g in ((y, s["gy"]), (n, s["gn"])) if g is not None]
            r.update(_grads([o for o, _ in outs], [g for _, g in outs], [a for a, _, _ in here],
                            [x for _, x, _ in here], [t for _, _, t in here]))
        return r
    x = _leaf(s["logits"])
    if not c["train"]:
        with torch.no_grad():
            return {"loss": _plain_distill(c, x, s["teacher"].float(), s["index"])}
    loss = _plain_distill(c, x, s["teacher"].float(), s["index"])
    return {"loss": loss.detach(), "logits": torch.autograd.grad(loss, x)[0].to(dt)}


# -------------------------------------------------------------------------- gatx's own calls

def _run_own(s):
    _package()
    c = s["case"]
    if c["op"] == "attention":
        from gatx.attention import diff_attention
        kw = {}
        if s["bias"] is not None:
            kw = {"bias": s["bias"], "positions": s["positions"],
                  "max_distance": c["max_distance"], "bidirectional": c["bidirectional"]}
        if s["asked"] is not None:
            kw["nodes"] = s["asked"]
        if not c["train"]:
            with torch.no_grad():
                return {"out": diff_attention(s["q"], s["k"], s["v"], s["lam"], s["graph"], **kw)}
        names = ["q", "k", "v", "lam"] + (["bias"] if s["bias"] is not None else [])
        x = {n: s[n].detach().requires_grad_(True) for n in names}
        kw.update({n: x[n] for n in ("bias",) if n in x})
        out = diff_attention(x["q"], x["k"], x["v"], x["lam"], s["graph"], **kw)
        got = torch.autograd.grad(out, [x[n] for n in names], s["go"])
        return {"out": out.detach(), **dict(zip(names, got))}
    if c["op"] == "norm":
        from gatx.norms import norm_after, norm_before
        names = [n for n in ("h", "weight", "resid", "gate", "scale", "next_weight")
                 if s[n] is not None]
        x = {n: s[n].detach().requires_grad_(c["train"]) for n in names}
        with torch.set_grad_enabled(c["train"]):
            if c["after"]:
                got = norm_after(x["h"], x["weight"], resid=x.get("resid"), gate=x.get("gate"),
                                 scale=x["scale"], next_weight=x.get("next_weight"), eps=_EPS)
                y, n = got if c["following"] else (got, None)
            else:
                y, n = None, norm_before(x["h"], x["next_weight"], eps=_EPS)
        outs = [(a, o, g) for a, o, g in (("y", y, s["gy"]), ("next", n, s["gn"]))
                if o is not None]
        r = {a: o.detach() for a, o, _ in outs}
        if c["train"]:
            got = torch.autograd.grad([o for _, o, _ in outs], [x[n] for n in names],
                                      [g for _, _, g in outs])
            r.update(zip(names, got))
        return r
    from gatx.losses import topk_distillation
    x = s["logits"].detach().requires_grad_(c["train"])
    loss = topk_distillation(x, s["teacher"], s["index"], temperature=c["temperature"])
    if not c["train"]:
        return {"loss": loss}
    return {"loss": loss.detach(), "logits": torch.autograd.grad(loss, x)[0]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------- work and exact

def work(case):
    """Bytes: every input and output once (of the keys and values of nodes that are asked for,
    the neighbours' alone). Operations: a multiply and an add for each term of each sum."""
    c, z = case, _SIZE[case["dtype"]]
    if c["op"] == "attention":
        H, d, dv = c["heads"], c["d"], c["dv"]
        N = c["graphs"] * c["nodes"]
        M, E = N, c["graphs"] * c["edges"] + N
        if c["serve"]:
            M, E = c["serve"], c["serve"] * c["edges"]
        rows = min(N, E)
        b = z * H * (M * 2 * d + rows * (2 * d + dv) + M * dv) + 4 * E + 4 * (M + 1)
        f = E * H * (4 * d + 2 * dv + 10)
        if c["buckets"]:
            b += 8 * N
        if c["train"]:   # the output's gradient in, those of q, k, v out; the transposed edges
            b += z * H * (M * dv + M * 2 * d + N * (2 * d + dv)) + 8 * E
            f += E * H * (8 * d + 4 * dv + 12)
        return {"bytes": float(b), "flops": float(f)}
    if c["op"] == "norm":
        n = c["rows"] * c["cols"]
        streams = 1 + c["resid"] + (c["gate"] == "row") + c["after"] + c["following"]
        f = 12.0 * n
        if c["train"]:   # the outputs' gradients in, those of h, resid and gate out
            streams += c["after"] + c["following"] + 1 + c["resid"] + (c["gate"] == "row")
            f += 30.0 * n
        return {"bytes": float(z * n * streams + 16 * c["cols"]), "flops": f}
    n = c["rows"] * c["classes"]
    b = z * n * (2 if c["train"] else 1) + c["rows"] * c["k"] * (z + 8)
    return {"bytes": float(b), "flops": float(n * (8 if c["train"] else 4))}


def _exact_attention(s):
    c, src, dst = s["case"], s["src"], s["dst"]
    H, d, M, N = c["heads"], c["d"], s["q"].size(0), s["k"].size(0)
    row = dst
    if s["asked"] is not None:
        where = torch.zeros(N, dtype=torch.int64, device=dst.device)
        where[s["asked"]] = torch.arange(M, device=dst.device)
        row = where[dst]
    order = torch.argsort(row, stable=True)
    row, src = row[order], src[order]
    count = torch.bincount(row, minlength=M)

    def segments(x):   # sums over each destination's run of edges
        return torch.segment_reduce(x, "sum", lengths=count, axis=0)

    bucket = None
    if s["bias"] is not None:
        rel = (s["positions"][s["src"]] - s["positions"][dst])[order]
        n, m, at = _bounds(c)
        away = rel.abs() if c["bidirectional"] else torch.where(rel < 0, -rel, 0)
        bucket = torch.minimum(away, torch.full_like(away, m))
        for x in at:
            bucket = bucket + (away >= x)
        if c["bidirectional"]:
            bucket = torch.where(rel > 0, bucket + n, bucket)
    r = {n: [] for n in ("out", "q", "k", "v", "lam", "bias")}
    for h in range(H):
        q, k, v = (s[n][:, h].double() for n in ("q", "k", "v"))
        lam = s["lam"][h].double()
        p = []
        for j in range(2):
            x = (q[row, j] * k[src, j]).sum(1) / math.sqrt(d)
            if bucket is not None:
                x = x + s["bias"][:, h].double()[bucket]
            top = torch.segment_reduce(x, "max", lengths=count, axis=0, initial=-1e300)
            e = torch.exp(x - top[row])
            total = segments(e)
            p.append(torch.where(total[row] > 0, e / total[row], 0.0))
        vs = v[src]
        r["out"].append(segments((p[0] - lam * p[1]).unsqueeze(1) * vs))
        if not c["train"]:
            continue
        go = s["go"][:, h].double()[row]
        dw = (go * vs).sum(1)
        del vs
        r["v"].append(torch.zeros_like(v).index_add_(
            0, src, (p[0] - lam * p[1]).unsqueeze(1) * go))
        del go
        r["lam"].append(-(p[1] * dw).sum())
        dq, dk, db = [], [], 0.0
        for j, sign in ((0, 1.0), (1, -lam)):
            dx = sign * p[j] * (dw - segments(p[j] * dw)[row])
            db = db + dx
            dx = (dx / math.sqrt(d)).unsqueeze(1)
            dq.append(segments(dx * k[src, j]))
            dk.append(torch.zeros_like(k[:, 0]).index_add_(0, src, dx * q[row, j]))
        r["q"].append(torch.stack(dq, 1))
        r["k"].append(torch.stack(dk, 1))
        if bucket is not None:
            r["bias"].append(torch.zeros_like(s["bias"][:, h].double()).index_add_(0, bucket, db))
    return {n: torch.stack(x, 0 if n == "lam" else 1) for n, x in r.items() if x}


def _exact_norm(s):
    c, D = s["case"], s["case"]["cols"]
    h = s["h"].double()
    w, sc, wn = (None if s[n] is None else s[n].double()
                 for n in ("weight", "scale", "next_weight"))
    r, y = {}, h
    if c["after"]:
        rh = 1 / torch.sqrt((h * h).sum(1, keepdim=True) / D + _EPS)
        hn = h * rh
        sg = torch.ones(1, dtype=torch.float64, device=h.device)
        if s["gate"] is not None:
            sg = torch.sigmoid(s["gate"].double())
        y = sc * sg * hn * w + (s["resid"].double() if c["resid"] else 0.0)
        r["y"] = y
    gy = 0.0 if s["gy"] is None else s["gy"].double()
    if c["following"]:
        ry = 1 / torch.sqrt((y * y).sum(1, keepdim=True) / D + _EPS)
        r["next"] = y * ry * wn
    if not c["train"]:
        return r
    if c["following"]:
        gn = s["gn"].double()
        r["next_weight"] = (gn * y * ry).sum(0)
        u = gn * wn
        gy = gy + ry * (u - y * ry * ry * (u * y).sum(1, keepdim=True) / D)
    if not c["after"]:
        r["h"] = gy
        return r
    if c["resid"]:
        r["resid"] = gy
    r["weight"] = (gy * sc * sg * hn).sum(0)
    r["scale"] = (gy * w * sg * hn).sum(0)
    if s["gate"] is not None:
        gg = gy * sc * w * hn * sg * (1 - sg)
        r["gate"] = gg if c["gate"] == "row" else gg.sum(0)
    t = gy * sc * sg * w
    r["h"] = rh * (t - hn * (t * hn).sum(1, keepdim=True) / D)
    return r


def _exact_distill(s):
    c, T = s["case"], s["case"]["temperature"]
    n, C = s["logits"].shape
    there = s["index"] >= 0
    some = there.any(1)
    t = torch.where(there, s["teacher"].double() / T, -math.inf)
    lp = torch.where(there, t - torch.logsumexp(torch.where(some[:, None], t, 0.0), 1, True), 0.0)
    p = torch.where(there, torch.exp(lp), 0.0)
    rows = max(1, 100_000_000 // C)
    loss, g = 0.0, torch.empty(n, C, dtype=torch.float64, device=p.device) if c["train"] else None
    count = max(1, int(some.sum()))
    for a in range(0, n, rows):
        x = s["logits"][a:a + rows].double() / T
        lse = torch.logsumexp(x, 1, True)
        at = s["index"][a:a + rows].clamp(min=0)
        part = p[a:a + rows] * (lp[a:a + rows] - x.gather(1, at) + lse)
        loss = loss + T * T * part.sum() / count
        if c["train"]:
            g[a:a + rows] = torch.exp(x - lse) * some[a:a + rows, None]
            g[a:a + rows].scatter_add_(1, at, -p[a:a + rows])
    if not c["train"]:
        return {"loss": loss}
    return {"loss": loss, "logits": g * (T / count)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "norm": _exact_norm,
            "distill": _exact_distill}[case["op"]](s)

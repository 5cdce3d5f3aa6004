"""The norms before and after a block, fused with the block's gate and residual scale
(csrc/block_norm.hip):

    norm_before:  next = next_weight * rms(x)
    norm_after:   y    = resid + scale * sigmoid(gate) * weight * rms(h)
                  next = next_weight * rms(y)      (the following block's norm_before, same pass)

rms(z) = z / sqrt(mean(z^2) + eps) over the last dimension. float32, bfloat16 and float16 rows; the
parameters (vectors over the columns) are used, and their gradients summed, in float32; y is
rounded where it is returned, not on the way into next. GATModel(block_norm=True) wires a layer
stack with them. There is no CPU path."""
from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from ._lib import DTYPES, call, lib, on_device, ptr, stream
from .functional import _span

MAX_COLUMNS = 8192


def _rows(t):
    """(rows x columns view, row stride): in place where only the rows are strided."""
    t = t.reshape(-1, t.size(-1)) if t.dim() != 2 else t
    if t.size(1) > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, (t.stride(0) if t.size(0) > 1 else t.size(1))


def _opt(t):
    return (None, 0) if t is None else _rows(t)


class BlockNormFunction(torch.autograd.Function):
    """(y, next) of gatx_block_norm; weight None: norm_before alone (y is None)."""

    @staticmethod
    def forward(ctx, h, weight, resid, gate, scale, next_weight, eps: float):
        shape, dt, dev = h.shape, DTYPES[h.dtype], h.device
        weight, scale, next_weight = (None if t is None else t.contiguous()
                                      for t in (weight, scale, next_weight))
        (h2, ldh), (r2, ldr) = _rows(h), _opt(resid)
        gate_rows = gate is not None and gate.dim() > 1
        g2, ldg = _rows(gate) if gate_rows else (None if gate is None else gate.contiguous(), 0)
        n, D = h2.shape
        y = torch.empty(shape, dtype=h.dtype, device=dev) if weight is not None else None
        nxt = torch.empty(shape, dtype=h.dtype, device=dev) if next_weight is not None else None
        save = any(ctx.needs_input_grad[:6])
        rstd_h = torch.empty(n, device=dev) if save and weight is not None else None
        rstd_y = torch.empty(n, device=dev) if save and next_weight is not None else None
        with _span("block_norm", (n, D)):
            call("gatx_block_norm", dt, n, D, ptr(h2), ldh, ptr(weight), ptr(r2), ldr, ptr(g2),
                 int(gate_rows), ldg, ptr(scale), ptr(next_weight), eps, ptr(y), ptr(nxt),
                 ptr(rstd_h), ptr(rstd_y), stream())
        ctx.set_materialize_grads(False)
        if save:
            ctx.save_for_backward(h2, weight, r2, g2, scale, next_weight, rstd_h, rstd_y)
            ctx.lds, ctx.gate_rows, ctx.shape = (ldh, ldr, ldg), gate_rows, shape
            ctx.gate_shape = None if gate is None else gate.shape
        return y, nxt

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gn):
        h, weight, resid, gate, scale, next_weight, rstd_h, rstd_y = ctx.saved_tensors
        if gy is None and gn is None:
            return (None,) * 7
        (ldh, ldr, ldg), dev, dt = ctx.lds, h.device, DTYPES[h.dtype]
        n, D = h.shape
        need = ctx.needs_input_grad
        with on_device(dev):
            (gy2, ldgy), (gn2, ldgn) = _opt(gy), _opt(gn)

            def rows(wanted):
                return torch.empty(ctx.shape, dtype=h.dtype, device=dev) if wanted else None

            def cols(wanted):
                return torch.empty(D, device=dev) if wanted else None

            gh, gresid = rows(need[0]), rows(need[2])
            ggate = None
            if need[3]:
                ggate = rows(True) if ctx.gate_rows else cols(True)
            gweight, gscale = cols(need[1]), cols(need[4])
            # without gn nothing reaches next_weight (its gradient is None, as for an unused output)
            gnext = cols(need[5] and gn is not None)
            wb = lib.gatx_block_norm_backward_workspace_bytes(n, D)
            ws = torch.empty(wb, dtype=torch.uint8, device=dev)
            with _span("block_norm_bwd", (n, D)):
                call("gatx_block_norm_backward", dt, n, D, ptr(h), ldh, ptr(weight), ptr(resid),
                     ldr, ptr(gate), int(ctx.gate_rows), ldg, ptr(scale), ptr(next_weight),
                     ptr(rstd_h), ptr(rstd_y), ptr(gy2), ldgy, ptr(gn2), ldgn, ptr(gh),
                     ptr(gresid), ptr(ggate), ptr(gweight), ptr(gscale), ptr(gnext), ptr(ws), wb,
                     stream())
        return gh, gweight, gresid, ggate, gscale, gnext, None


def _check(what, x, vectors, rows):
    if x.dtype not in DTYPES:
        raise RuntimeError(f"gatx: {what} takes float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or not 1 <= x.size(-1) <= MAX_COLUMNS:
        raise ValueError(f"gatx: {what}: 1 to {MAX_COLUMNS} columns, got {tuple(x.shape)}")
    for name, t in vectors:
        if t is None:
            continue
        if tuple(t.shape) != (x.size(-1),) or not t.is_floating_point():
            raise ValueError(f"gatx: {what}: {name} is a vector of {x.size(-1)}, got "
                             f"{tuple(t.shape)}")
        if t.device != x.device:
            raise RuntimeError(f"gatx: {what}: {name} is on {t.device}, the rows on {x.device}")
    for name, t in rows:
        if t is None:
            continue
        if t.shape != x.shape or t.dtype != x.dtype:
            raise ValueError(f"gatx: {what}: {name} is {tuple(x.shape)} {x.dtype}, got "
                             f"{tuple(t.shape)} {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"gatx: {what}: {name} is on {t.device}, the rows on {x.device}")
    if not x.is_cuda:
        raise RuntimeError(f"gatx: {what} needs HIP tensors (no CPU path)")


def _f32(t):
    return None if t is None else t.float()


def norm_before(x, weight, eps: float = 1e-6):
    """weight * rms(x): the norm before a block. x: (..., D), weight: (D,)."""
    _check("norm_before", x, [("weight", weight)], [])
    with on_device(x.device):
        return BlockNormFunction.apply(x, None, None, None, None, _f32(weight), float(eps))[1]


def norm_after(h, weight, *, resid=None, gate=None, scale=None, next_weight=None,
               eps: float = 1e-6):
    """y = resid + scale * sigmoid(gate) * weight * rms(h) for a block's output h (..., D): the norm
    after the block, its gate, the residual scale and the residual. weight, scale: (D,); gate: (D,),
    a parameter, or of h's shape and dtype; resid of h's. Returns y, or with next_weight (D,) the
    pair (y, next_weight * rms(y)): the norm before the next block in the same pass."""
    vector_gate = gate is not None and gate.dim() == 1 and h.dim() != 1
    _check("norm_after", h, [("weight", weight), ("scale", scale), ("next_weight", next_weight)]
           + ([("gate", gate)] if vector_gate else []),
           [("resid", resid)] + ([] if vector_gate else [("gate", gate)]))
    if h.dim() == 1:   # one row
        r = norm_after(h.unsqueeze(0), weight, scale=scale, next_weight=next_weight, eps=eps,
                       resid=None if resid is None else resid.unsqueeze(0),
                       gate=None if gate is None else gate.unsqueeze(0))
        return r.squeeze(0) if next_weight is None else tuple(t.squeeze(0) for t in r)
    with on_device(h.device):
        y, nxt = BlockNormFunction.apply(h, _f32(weight), resid,
                                         gate.float() if vector_gate else gate, _f32(scale),
                                         _f32(next_weight), float(eps))
    return y if next_weight is None else (y, nxt)


class BlockNorm(nn.Module):
    """The parameters of norm_after for one block of `features` columns: weight, a residual scale, a
    gate per column (gate=True) and the next block's norm (following=True)."""

    def __init__(self, features, gate=True, following=True, scale_init=1.0, eps=1e-6):
        super().__init__()
        self.features, self.eps, self.scale_init = features, eps, scale_init
        self.weight = nn.Parameter(torch.empty(features))
        self.scale = nn.Parameter(torch.empty(features))
        for name, wanted in (("gate", gate), ("next_weight", following)):
            self.register_parameter(name,
                                    nn.Parameter(torch.empty(features)) if wanted else None)
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.ones_(self.weight)
        nn.init.constant_(self.scale, self.scale_init)
        if self.gate is not None:
            nn.init.zeros_(self.gate)
        if self.next_weight is not None:
            nn.init.ones_(self.next_weight)

    def forward(self, h, resid=None, gate=None):
        """y, or (y, next) with following; gate: one of h's shape instead of the parameter."""
        return norm_after(h, self.weight, resid=resid, gate=self.gate if gate is None else gate,
                          scale=self.scale, next_weight=self.next_weight, eps=self.eps)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}"

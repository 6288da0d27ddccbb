"""Muon: momentum whose update is orthogonalised by Newton-Schulz products (reference:
moonlight.py, which gives it the weight matrices and AdamW the rest).

    buf = momentum buf + g;   u = g + momentum buf  (nesterov; else buf)
    W <- (1 - lr weight_decay) W - lr rms sqrt(max(R, C)) NS(u)

NS(u) has singular values near 1, so that its root mean square is about
1 / sqrt(max(R, C)): the factor makes that of every update `rms`, whatever the matrix's shape
(0.2, that of AdamW's).  On the GPU all matrices of one shape go through
sla2h_orthogonalize together; CPU tensors run the eager products.
"""

import math

import torch

from . import ops

__all__ = ["Muon", "matrix_parameters", "newton_schulz"]


def newton_schulz(g, steps=5, coeffs=ops.NS_COEFFS):
    """ops.orthogonalize; CPU and float64 tensors, and those with a gradient or a tangent to carry, run the
    products one by one, in float32 or wider."""
    if (g.is_cuda and g.dtype != torch.float64 and ops.plain_eager(g)
            and not (g.requires_grad and torch.is_grad_enabled())):
        return ops.orthogonalize(g, steps, coeffs)
    ops._ns_coeffs(steps, ops.ns_rows(steps, coeffs))  # its checks
    # (autocast would make the products 16-bit ones)
    with torch.autocast("cuda" if g.is_cuda else "cpu", enabled=False):
        return _products(g, steps, coeffs)


def _products(g, steps, coeffs):
    x = g.to(torch.promote_types(g.dtype, torch.float32))
    if g.shape[-2] > g.shape[-1]:
        x = x.transpose(-1, -2)
    norm = x.double().square().sum((-1, -2), keepdim=True).sqrt()
    x = (x / torch.where(norm > 0, norm, torch.ones_like(norm))).to(x.dtype)
    rows = ops.ns_rows(steps, coeffs)
    for a, b, c in rows if isinstance(rows[0], tuple) else [rows] * steps:
        A = x @ x.transpose(-1, -2)
        x = a * x + (b * A + c * (A @ A)) @ x
    return (x.transpose(-1, -2) if g.shape[-2] > g.shape[-1] else x).to(g.dtype)


def matrix_parameters(module, others=("alpha_logit",)):
    """(matrices, rest) of a module's parameters that take gradients: Muon's are those of two
    dimensions, but for the names in `others` (tables, not maps)."""
    mats, rest = [], []
    for name, p in module.named_parameters():
        if p.requires_grad:
            mats.append(p) if p.dim() == 2 and name.rpartition(".")[2] not in others else rest.append(p)
    return mats, rest


class Muon(torch.optim.Optimizer):
    """Muon over matrices (R, C).  The momentum is kept in fp32; ns_steps, ns_coeffs as in
    newton_schulz.  Matrices without a gradient stay as they are."""

    def __init__(self, params, lr=2e-3, momentum=0.95, nesterov=True, weight_decay=0.0, rms=0.2,
                 ns_steps=5, ns_coeffs=ops.NS_COEFFS):
        if lr < 0 or weight_decay < 0 or rms <= 0 or not 0 <= momentum < 1:
            raise ValueError("Muon: lr and weight_decay from 0, rms above 0, momentum in [0, 1), got "
                             f"{lr}, {weight_decay}, {rms}, {momentum}")
        ops._ns_coeffs(ns_steps, ops.ns_rows(ns_steps, ns_coeffs))  # its checks
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, rms=rms, ns_steps=ns_steps,
                                      ns_coeffs=ns_coeffs))

    def add_param_group(self, group):
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2 or not p.is_floating_point() or max(p.shape) > 32768:
                self.param_groups.pop()
                raise ValueError("Muon: matrices only, sides up to 32,768, got "
                                 f"{tuple(p.shape)} {p.dtype}")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class casts a state to its weight's type: the momentum stays fp32, a copy
        old = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(old, (p for g in self.param_groups for p in g["params"])):
            kept = state_dict["state"].get(i, {}).get("momentum_buffer")
            if kept is not None:
                self.state[p]["momentum_buffer"] = kept.to(
                    p.device, torch.promote_types(p.dtype, torch.float32), copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every matrix that has a gradient; the closure's loss, if given."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon: sparse gradients are not supported")
                if p.numel():
                    alike.setdefault((p.shape, p.dtype, p.grad.dtype, p.device), []).append(p)
            for ps in alike.values():
                self._update(ps, group)
        return loss

    def _update(self, ps, group):
        """The matrices `ps` of one shape, type and device."""
        wide = torch.promote_types(ps[0].dtype, torch.float32)
        for p in ps:
            if "momentum_buffer" not in self.state[p]:
                self.state[p]["momentum_buffer"] = torch.zeros_like(
                    p, dtype=wide, memory_format=torch.contiguous_format)
        bufs = [self.state[p]["momentum_buffer"] for p in ps]
        grads = [p.grad if p.grad.dtype == wide else p.grad.to(wide) for p in ps]
        mu = group["momentum"]
        torch._foreach_mul_(bufs, mu)
        torch._foreach_add_(bufs, grads)
        u = torch.stack(torch._foreach_add(grads, bufs, alpha=mu) if group["nesterov"] else bufs)
        x = newton_schulz(u, group["ns_steps"], group["ns_coeffs"])
        R, C = ps[0].shape
        lr = float(group["lr"])
        step = -lr * group["rms"] * math.sqrt(max(R, C))
        keep = 1.0 - lr * group["weight_decay"]
        if ps[0].dtype == wide:
            if keep != 1.0:
                torch._foreach_mul_(ps, keep)
            torch._foreach_add_(ps, list(x), alpha=step)
        else:  # (16-bit weights: decay and update in fp32, rounded once)
            for p, d in zip(ps, x):
                p.copy_(p.to(wide).mul_(keep).add_(d, alpha=step))

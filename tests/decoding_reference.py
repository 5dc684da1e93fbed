"""The feature decoder's operators in 64 bits, written from their formulas, with
bounds on the error of an evaluation that holds values in 32 bits and rounds to
the tensors' dtype where the operators say they do.

Every bound is first order and elementwise.  u is the unit roundoff of 32 bits
(2^-24), v that of the dtype.  A sum of n terms in any order errs by at most
n u sum |terms|; the activations and their slopes by ACT (absolute, per unit of
magnitude), their slopes change by at most CURVE per unit of argument.
"""

import math

import torch

U = 2.0 ** -24
ACT = 2.0 ** -19      # exp and erf in 32 bits with a rounded argument, per unit of max(1, |z|)
LIFT = 1.13           # largest slope of an activation (gelu: 1.1290, silu: 1.0998)
CURVE = 0.80          # largest second derivative (gelu: 2 phi(0) = 0.798)
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def activate(z, kind):
    if kind == "relu":
        return z.clamp_min(0)
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    if kind == "gelu":
        return z * 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
    return z


def slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s + z * s * (1 - s)
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def kept(x):
    """What the 8-bit form of x stands for (finite x), in 64 bits."""
    v = x.detach().double().cpu()
    out = torch.empty_like(v)
    for c in range(0, v.shape[-1], 32):
        block = v[..., c:c + 32]
        top = block.abs().amax(-1)
        step = torch.tensor([max(-126, math.ceil(math.log2(t / 127)) if t > 0 else -126) for t in top.flatten().tolist()],
                            dtype=torch.float64).reshape(top.shape)
        for _ in range(2):  # log2 may be off by its rounding
            step = torch.where(top > 127 * 2.0 ** step, step + 1, step)
            step = torch.where((top <= 127 * 2.0 ** (step - 1)) & (step > -126), step - 1, step)
        size = (2.0 ** step.clamp_max(9 if x.dtype == torch.float16 else 121))[..., None]
        out[..., c:c + 32] = torch.round(block / size).clamp(-127, 127) * size
    return out.to(x.device)


def _rounded(value, error, dtype):
    return error + UNIT[dtype] * (value.abs() + error) + TINY[dtype]


def linear(x, weight, bias, residual, activation):
    """(y, bound)."""
    dtype = x.dtype
    x, w = x.double(), weight.double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if bias is None else bias.double()
    z = x @ w.T + b
    err_z = (x.shape[-1] + 2) * U * (x.abs() @ w.abs().T + b.abs())
    y = activate(z, activation)
    err = LIFT * err_z + (ACT * z.abs().clamp_min(1) if activation in ("silu", "gelu") else 0)
    if residual is not None:
        y = y + residual.double()
        err = err + U * (y.abs() + err)
    return y, _rounded(y, err, dtype)


def linear_grads(x, weight, bias, upstream, activation):
    """{name: (gradient, bound)} with x the value that the backward pass sees
    (64 bits or the dtype)."""
    dtype = weight.dtype
    lead = x.reshape(-1, x.shape[-1]).double()
    w, dy = weight.double(), upstream.reshape(-1, weight.shape[0]).double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if bias is None else bias.double()
    z = lead @ w.T + b
    err_z = (lead.shape[-1] + 2) * U * (lead.abs() @ w.abs().T + b.abs())
    dz = dy * slope(z, activation)
    if activation == "none":
        err = torch.zeros_like(dz)  # the upstream gradient itself
    elif activation == "relu":
        err = dy.abs() * (z.abs() <= err_z)
    else:
        err = _rounded(dz, dy.abs() * (CURVE * err_z + ACT * z.abs().clamp_min(1)), dtype)
    rows, outer = dz.shape
    dx, dw, db = dz @ w, dz.T @ lead, dz.sum(0)
    bound = {
        "x": (dx, err @ w.abs() + (outer + 2) * U * (dz.abs() @ w.abs())),
        "weight": (dw, err.T @ lead.abs() + (rows + 2) * U * (dz.abs().T @ lead.abs())),
        "bias": (db, err.sum(0) + (rows + 2) * U * dz.abs().sum(0)),
    }
    return {k: (g.reshape(x.shape) if k == "x" else g, _rounded(g, e, dtype).reshape(x.shape if k == "x" else g.shape))
            for k, (g, e) in bound.items()}


class Norm:
    """Group norm of x (images, pixels, channels) and its gradients with bounds.

    Terms of a group are summed by threads (at most RUN in a row) and merged;
    RUN u bounds the relative error of the mean (over max |x|), and RUN u kappa
    that of the variance, kappa^2 = 1 + max x^2 / var: the bound of the update
    formulas of mean and squared deviation."""

    RUN = 256

    def __init__(self, x, groups, weight, bias, eps, activation):
        self.dtype, self.kind = x.dtype, activation
        n, p, c = x.shape
        self.shape, self.groups = (n, p, groups, c // groups), groups
        view = lambda t: t.double().reshape(1, 1, groups, c // groups)
        self.gamma = torch.ones_like(view(x[0, 0])) if weight is None else view(weight)
        self.beta = torch.zeros_like(self.gamma) if bias is None else view(bias)
        v = x.double().reshape(self.shape)
        self.mean = v.mean((1, 3), keepdim=True)
        var = (v - self.mean).square().mean((1, 3), keepdim=True)
        self.rstd = (var + eps).rsqrt()
        top = v.abs().amax((1, 3), keepdim=True)
        self.err_mean = self.RUN * U * top
        # d rstd = -rstd / 2 * d var / (var + eps)
        kappa = (1 + top.square() / var.clamp_min(1e-300)).sqrt()
        self.rel_rstd = 0.5 * self.RUN * U * kappa * var * self.rstd.square() + 4 * U
        self.x = v

    def _argument(self, v):
        unit = (v - self.mean) * self.rstd
        u = unit * self.gamma + self.beta
        err = self.gamma.abs() * (self.rstd * (self.err_mean + U * (v - self.mean).abs())
                                  + unit.abs() * (self.rel_rstd + 4 * U)) + 2 * U * (u.abs() + self.beta.abs())
        return unit, u, err

    def forward(self):
        _, u, err = self._argument(self.x)
        y = activate(u, self.kind)
        err = LIFT * err + (ACT * u.abs().clamp_min(1) if self.kind in ("silu", "gelu") else 0)
        n, p, g, c = self.shape
        return y.reshape(n, p, g * c), _rounded(y, err, self.dtype).reshape(n, p, g * c)

    def grads(self, seen, upstream):
        """seen: the value of x that the backward pass has (x, or the kept one)."""
        v, dy = seen.double().reshape(self.shape), upstream.double().reshape(self.shape)
        unit, u, err_u = self._argument(v)
        dz = dy * slope(u, self.kind)
        if self.kind == "none":
            err = torch.zeros_like(dz)
        elif self.kind == "relu":
            err = dy.abs() * (u.abs() <= err_u)
        else:
            err = dy.abs() * (CURVE * err_u + ACT * u.abs().clamp_min(1))
        err = err + U * dz.abs()
        err_unit = self.rstd * (self.err_mean + U * (v - self.mean).abs()) + unit.abs() * (self.rel_rstd + 2 * U)
        s1, s2 = dz, dz * unit
        err2 = err * unit.abs() + dz.abs() * err_unit
        total = lambda t, d: t.sum(d, keepdim=True)
        run = self.RUN * U
        err_s1, err_s2 = err + run * s1.abs(), err2 + run * s2.abs()
        count = self.shape[1] * self.shape[3]
        level, along = total(self.gamma * s1, (1, 3)) / count, total(self.gamma * s2, (1, 3)) / count
        err_level = total(self.gamma.abs() * (err_s1 + run * s1.abs()), (1, 3)) / count
        err_along = total(self.gamma.abs() * (err_s2 + run * s2.abs()), (1, 3)) / count
        dx = self.rstd * (self.gamma * dz - level - unit * along)
        err_dx = self.rstd * (self.gamma.abs() * err + err_level + unit.abs() * err_along + err_unit * along.abs()) \
            + (self.rel_rstd + 6 * U) * self.rstd * ((self.gamma * dz).abs() + level.abs() + 2 * (unit * along).abs())
        n, p, g, c = self.shape
        out = {"x": (dx.reshape(n, p, g * c), err_dx.reshape(n, p, g * c)),
               "weight": (s2.sum((0, 1)).reshape(-1), err_s2.sum((0, 1)).reshape(-1)),
               "bias": (s1.sum((0, 1)).reshape(-1), err_s1.sum((0, 1)).reshape(-1))}
        return {k: (v, _rounded(v, e, self.dtype)) for k, (v, e) in out.items()}


def check(name, got, want, bound):
    got = got.detach().double().reshape(want.shape)
    excess = (got - want).abs() - bound
    worst = excess.max().item() if excess.numel() else 0.0
    assert torch.isfinite(got).all(), name
    if worst > 0:
        i = int(excess.flatten().argmax())
        raise AssertionError(f"{name}: entry {i} is {got.flatten()[i].item()!r}, want {want.flatten()[i].item()!r} "
                             f"within {bound.flatten()[i].item():.3e}; {int((excess > 0).sum())} of {excess.numel()} outside")

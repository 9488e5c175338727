"""Attention of one head in 64 bits, with bounds on a kernel's rounding.

Roundings are counted in half steps: U of f32 arithmetic, and H of the type that
weights, their gradients and results are rounded to (f32: U). Sums of n terms err
by at most n U of the sum of their magnitudes. `d` bounds a weight's relative error: a
score is a sum of hd products (hd + 4 roundings, scale and exponent among them),
and its error, absolute, is passed on by exp; the log-sum-exp adds as much again.
"""
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _largest(x):
    """A row's largest value, 0 where it has none."""
    return torch.cat([x, x.new_zeros((x.shape[0], 1))], 1).amax(1, keepdim=True)


def attend(q, k, v, scale, see, half, q_half=0.0):
    """q [a, hd], k and v [b, hd] f64, see [a, b] -> (out, lse, bound of out's error).
    q_half: relative rounding of q before its product."""
    x = (q @ k.T * scale).masked_fill(~see, -torch.inf)
    lse = torch.logsumexp(x, 1)
    p = torch.where(see, torch.exp(x - lse[:, None].clamp(min=-1e300)), torch.zeros_like(x))
    out = p @ v
    mag = (q.abs() @ k.abs().T * scale).masked_fill(~see, 0.0)
    d = ((q.shape[1] + 4) * U + q_half) * _largest(mag) + 4 * U
    near = p @ v.abs()
    bound = half * out.abs() + (half + 2 * d + (k.shape[0] + 4) * U) * near
    return out, lse, bound + 1e-30


def attend_grad(q, k, v, do, scale, see, half):
    """-> (dq, dk, dv) and their bounds; `do` and the rest f64."""
    x = (q @ k.T * scale).masked_fill(~see, -torch.inf)
    lse = torch.logsumexp(x, 1)
    p = torch.where(see, torch.exp(x - lse[:, None].clamp(min=-1e300)), torch.zeros_like(x))
    out = p @ v
    dp = do @ v.T
    delta = (do * out).sum(1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = ds @ k * scale, ds.T @ q * scale, p.T @ do
    hd, n = q.shape[1], max(k.shape[0], q.shape[0])
    mag = (q.abs() @ k.abs().T * scale).masked_fill(~see, 0.0)
    d = (2 * (hd + 4) * U * _largest(mag) + 8 * U) * torch.ones_like(p)  # scores and log-sum-exp
    # delta: out is taken as rounded, its own error (attend's bound) included
    eout = attend(q, k, v, scale, see, half)[2]
    edelta = (do.abs() * (eout + hd * U * out.abs())).sum(1, keepdim=True)
    edp = hd * U * (do.abs() @ v.abs().T)
    eds = (half + d) * ds.abs() + p * (edelta + edp)
    adds = (n + 4) * U
    bdv = half * dv.abs() + ((half + d + adds) * p).T @ do.abs()
    bdq = half * dq.abs() + (eds + adds * ds.abs()) @ k.abs() * scale
    bdk = half * dk.abs() + (eds + adds * ds.abs()).T @ q.abs() * scale
    return (dq, dk, dv), (bdq + 1e-30, bdk + 1e-30, bdv + 1e-30)


def causal(a, b, device="cuda"):
    i, j = torch.arange(a, device=device)[:, None], torch.arange(b, device=device)
    return j <= i + b - a


def rope(x, pos, theta):
    """x [rows, heads, hd] f64 rotated at positions pos [rows] (NeoX half split)."""
    hd = x.shape[-1]
    f = theta ** (-2 * torch.arange(hd // 2, dtype=torch.float64, device=x.device) / hd)
    a = (pos.double()[:, None] * f)[:, None]
    lo, hi = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)

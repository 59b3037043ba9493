"""Float64 restatements of the short filter, selective scan, layer norm and distillation loss, and how results are compared.

``error`` is the norm of the difference over a scale: the expected value's
norm, or for sums over tokens that cancel the sum of their terms' magnitudes.
Tolerances.  A result rounded once to bfloat16 is off by at most 2^-9 of each
element, 2^-8 leaves room for a rounding boundary; each further rounding of an
operand to bfloat16 adds 2^-9 of the result's scale.  float32 results carry
2^-24 a term and, where a sum of a thousand terms or an exponent of magnitude
32 enters, up to a hundred times that: 1e-5.  Plain rows of a few thousand
elements, without exponents of sums: 2e-6.
"""
from __future__ import annotations

import torch

ROUNDED = 2.0 ** -8          # one rounding to bfloat16
ROUNDED_TWICE = 3 * 2.0 ** -9  # and one of an operand
SUMMED = 1e-5                # float32 sums and exponents along a sequence
ROWS = 2e-6                  # float32 rows


def error(actual, expected, scale=None):
    actual, expected = actual.detach().double().cpu(), expected.detach().double().cpu()
    assert actual.shape == expected.shape, (tuple(actual.shape), tuple(expected.shape))
    assert torch.isfinite(actual).all()
    if expected.numel() == 0:
        return 0.0
    scale = expected.norm() if scale is None else scale.detach().double().cpu().norm()
    return float((actual - expected).norm() / scale.clamp_min(1e-300)) if float(scale) else float(actual.norm())


def check(name, actual, expected, tolerance, scale=None):
    off = error(actual, expected, scale)
    assert off <= tolerance, f"{name}: off by {off:.2e}, tolerance {tolerance:.2e}"


def conv(x, weight, bias=None, silu=False, state=None, lengths=None):
    """Token by token and tap by tap."""
    b, t, c = x.shape
    w = weight.shape[1]
    outs, finals = [], []
    for i in range(b):
        n = t if lengths is None else min(max(int(lengths[i]), 0), t)
        past = [torch.zeros(c, dtype=x.dtype)] * (w - 1) if state is None else list(state[i])
        rows = past + [x[i, s] for s in range(n)]
        ys = []
        for s in range(n):
            pre = sum(rows[s + j] * weight[:, j] for j in range(w))
            pre = pre if bias is None else pre + bias
            ys.append(pre * torch.sigmoid(pre) if silu else pre)
        ys += [torch.zeros(c, dtype=x.dtype)] * (t - n)
        outs.append(torch.stack(ys) if ys else x.new_zeros(0, c))
        finals.append(torch.stack(rows[n:n + w - 1]))
    return torch.stack(outs), torch.stack(finals)


def scan(x, dt, A, B, C, D=None, dt_bias=None, softplus=True, state=None, lengths=None):
    """Token by token; A, D and dt_bias may be given for every token ([batch, time, heads])."""
    b, t, h, p = x.shape
    g, n = B.shape[2:]
    A, D, dt_bias = (z if z is None or z.ndim == 3 else z.expand(b, t, h) for z in (A, D, dt_bias))
    step = dt if dt_bias is None else dt + dt_bias
    if softplus:
        step = torch.nn.functional.softplus(step, threshold=60.0)
    group = torch.arange(h) // (h // g)
    cut = torch.full((b,), t) if lengths is None else lengths.clamp(0, t)
    h_t = torch.zeros(b, h, p, n, dtype=x.dtype) if state is None else state
    ys = []
    for i in range(t):
        live = (i < cut).view(b, 1, 1, 1)
        new = torch.exp(step[:, i] * A[:, i])[..., None, None] * h_t \
            + (step[:, i, :, None] * x[:, i])[..., None] * B[:, i][:, group][:, :, None]
        h_t = torch.where(live, new, h_t)
        y = (h_t * C[:, i][:, group][:, :, None]).sum(-1)
        y = y if D is None else y + D[:, i, :, None] * x[:, i]
        ys.append(torch.where(live[..., 0], y, torch.zeros_like(y)))
    return (torch.stack(ys, 1) if ys else torch.zeros_like(x)), h_t


def norm(x, weight=None, bias=None, eps=1e-5):
    mean = x.mean(-1, keepdim=True)
    y = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = y if weight is None else y * weight
    return y if bias is None else y + bias


def distill(logits, teacher, index, tau):
    """Losses of the rows, entry by entry of each teacher's list."""
    losses = []
    for x, t, at in zip(logits, teacher, index):
        keep = [k for k in range(len(at)) if 0 <= int(at[k]) < len(x) and float(t[k]) != float("-inf")]
        if not keep:
            losses.append(torch.zeros((), dtype=torch.float64))
            continue
        log_p = torch.log_softmax(t[keep] / tau, -1)
        log_q = torch.log_softmax(x / tau, -1)[at[keep]]
        losses.append(tau * tau * (log_p.exp() * (log_p - log_q)).sum())
    return torch.stack(losses)

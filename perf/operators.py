"""The selective state space operators, the layer norm and the distillation loss: what they are timed on.

Each case is one call, or one training step (forward and backward), of

- ``conv``: the short causal filter with bias, SiLU and carried inputs, ``bayes_ssm.conv.causal_conv``;
- ``scan``: the selective state space scan, ``bayes_ssm.selective.selective_scan``;
- ``step``: filter and scan of one token from carried states, ``bayes_ssm.selective.selective_step``;
- ``norm``: ``bayes_ssm.norm.layer_norm``;
- ``distill``: the distillation loss from a teacher's top logits, ``bayes_ssm.distill.distillation_loss``.

With ``own`` false, ``run`` computes the same in elementary torch operations in float32, rounded once at the end.
``exact`` restates each in float64, token by token where the operator is a recurrence, with gradients written out.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "bayes-ssm_amd"))

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
own = False


def listed():
    return [
        # The filter of a 32-head block (values, keys and queries of one projection) in a training step.
        {"name": "conv_train", "path": "conv", "b": 8, "t": 2048, "c": 2304, "w": 4, "dtype": "bf16", "train": True,
         "carry": False, "ragged": False},
        # Prompts of unequal lengths that go on from an earlier part, an odd number of channels.
        {"name": "conv_prompt_odd", "path": "conv", "b": 3, "t": 1037, "c": 331, "w": 3, "dtype": "f32",
         "train": False, "carry": True, "ragged": True},
        # The training step of a 32-head block at batch 8.
        {"name": "scan_train", "path": "scan", "b": 8, "t": 2048, "h": 32, "p": 64, "n": 128, "g": 1,
         "dtype": "bf16", "train": True, "carry": False, "ragged": False},
        # A training step in float32 at odd sizes, two groups.
        {"name": "scan_train_odd", "path": "scan", "b": 2, "t": 777, "h": 6, "p": 40, "n": 24, "g": 2,
         "dtype": "f32", "train": True, "carry": False, "ragged": False},
        # One long document: few heads to share out, so the time axis has to be.
        {"name": "scan_prompt_long", "path": "scan", "b": 1, "t": 16384, "h": 32, "p": 64, "n": 128, "g": 1,
         "dtype": "bf16", "train": False, "carry": True, "ragged": False},
        # A batch of prompts of unequal lengths.
        {"name": "scan_prompt_ragged", "path": "scan", "b": 16, "t": 509, "h": 24, "p": 64, "n": 64, "g": 2,
         "dtype": "bf16", "train": False, "carry": True, "ragged": True},
        # One token for one request: latency.
        {"name": "step_one", "path": "step", "b": 1, "h": 32, "p": 64, "n": 128, "g": 1, "w": 4, "dtype": "bf16"},
        # One token for a full serving batch.
        {"name": "step_batch", "path": "step", "b": 256, "h": 32, "p": 64, "n": 128, "g": 1, "w": 4,
         "dtype": "bf16"},
        # The block's norm in a training step: batch 8 of 2048 tokens.
        {"name": "norm_train", "path": "norm", "r": 16384, "d": 2048, "dtype": "bf16", "train": True},
        # The same in float32 at a width that fills no vector.
        {"name": "norm_train_odd", "path": "norm", "r": 1021, "d": 1003, "dtype": "f32", "train": True},
        # The student's loss and the logits' gradient over a vocabulary of 32000.
        {"name": "distill_train", "path": "distill", "r": 4096, "v": 32000, "k": 64, "tau": 2.0, "dtype": "bf16",
         "train": True},
        # A held-out batch over a vocabulary of odd size in float32: each row's loss.
        {"name": "distill_eval_odd", "path": "distill", "r": 301, "v": 50257, "k": 7, "tau": 1.0, "dtype": "f32",
         "train": False},
    ]


def _log_int(rng, low, high):
    high = max(low, high)
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the ranges above."""
    path = rng.choice(["conv", "scan", "scan", "scan", "step", "norm", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    train = rng.random() < 0.6
    if path == "conv":
        c, t = _log_int(rng, 64, 4096), _log_int(rng, 1, 4096)
        return {"path": path, "b": _log_int(rng, 1, 16777216 // (c * t)), "t": t, "c": c, "w": rng.choice([2, 3, 4]),
                "dtype": dtype, "train": train, "carry": rng.random() < 0.5, "ragged": rng.random() < 0.4}
    if path == "scan":
        g = rng.choice([1, 1, 2, 4])
        h = g * rng.randint(1, 32 // g)
        p, n = rng.choice([16, 32, 40, 64, 64, 72, 128]), rng.choice([8, 16, 24, 64, 100, 128, 128])
        t = _log_int(rng, 1, 4096) if train else _log_int(rng, 1, 16384)
        top = 8 * 2048 * 32 * 64 if dtype == "bf16" else 2 * 2048 * 32 * 64
        return {"path": path, "b": _log_int(rng, 1, min(16, top // (h * max(p, 64) * t))), "t": t, "h": h, "p": p,
                "n": n, "g": g, "dtype": dtype, "train": train, "carry": rng.random() < 0.5,
                "ragged": rng.random() < 0.3}
    if path == "step":
        g = rng.choice([1, 1, 2, 4])
        return {"path": path, "b": _log_int(rng, 1, 256), "h": g * rng.randint(1, 32 // g),
                "p": rng.choice([16, 32, 40, 64, 64, 128]), "n": rng.choice([8, 16, 24, 64, 100, 128]), "g": g,
                "w": rng.choice([2, 3, 4]), "dtype": dtype}
    if path == "norm":
        d = _log_int(rng, 16, 8192)
        return {"path": path, "r": _log_int(rng, 1, 33554432 // d), "d": d, "dtype": dtype, "train": train}
    v = _log_int(rng, 100, 130000)
    return {"path": path, "r": _log_int(rng, 1, 131072000 // v), "v": v, "k": _log_int(rng, 1, 100),
            "tau": rng.choice([1.0, 2.0, 0.7]), "dtype": dtype, "train": train}


# ------------------------------------------------------------------------------------------------- inputs

def _inputs(case, seed):
    """(leaves, others): named tensors that a training step differentiates, and the rest."""
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    path, dt = case["path"], DTYPES[case["dtype"]]

    def rn(*shape):
        return torch.randn(*shape, device=DEVICE, generator=gen)

    def un(*shape):
        return torch.rand(*shape, device=DEVICE, generator=gen)

    def lengths(b, t):  # every length from nothing to the whole row; the longest fills it
        cut = torch.randint(0, t + 1, (b,), device=DEVICE, generator=gen)
        cut[b - 1] = t
        return cut

    def dynamics(h):
        """Time steps between 0.001 and 0.1 before the input moves them, decay rates between 1 and 16."""
        step = torch.exp(un(h) * math.log(100.0) + math.log(0.001))
        return {"A": -(1.0 + 15.0 * un(h)), "D": 1.0 + 0.1 * rn(h), "dt_bias": step + torch.log(-torch.expm1(-step))}

    if path == "conv":
        b, t, c, w = case["b"], case["t"], case["c"], case["w"]
        leaves = {"x": rn(b, t, c).to(dt), "weight": (rn(c, w) / w ** 0.5).to(dt), "bias": (0.1 * rn(c)).to(dt)}
        if case["carry"]:
            leaves["state"] = rn(b, w - 1, c).to(dt)
        rest = {"gy": rn(b, t, c).to(dt), "lengths": lengths(b, t) if case["ragged"] else None}
    elif path == "scan":
        b, t, h, p, n, g = (case[k] for k in "bthpng")
        silu = torch.nn.functional.silu
        leaves = {"x": silu(rn(b, t, h, p)).to(dt), "dt": (0.5 * rn(b, t, h)).to(dt),
                  "B": silu(rn(b, t, g, n)).to(dt), "C": silu(rn(b, t, g, n)).to(dt), **dynamics(h)}
        if case["carry"]:
            leaves["state"] = 0.1 * rn(b, h, p, n)
        rest = {"gy": rn(b, t, h, p).to(dt), "lengths": lengths(b, t) if case["ragged"] else None}
    elif path == "step":
        b, h, p, n, g, w = (case[k] for k in "bhpngw")
        c = h * p + 2 * g * n
        # The token's row of one projection: gate, filter's channels, time steps; the states that earlier tokens left.
        projected = rn(b, h * p + c + h)
        projected[:, h * p + c:] *= 0.5
        leaves = {}
        rest = {"projected": projected.to(dt), "weight": (rn(c, w) / w ** 0.5).to(dt), "bias": (0.1 * rn(c)).to(dt),
                "conv_state": rn(b, w - 1, c).to(dt), "state": 0.3 * rn(b, h, p, n), **dynamics(h),
                "next_conv_state": torch.empty(b, w - 1, c, device=DEVICE, dtype=dt),
                "next_state": torch.empty(b, h, p, n, device=DEVICE)}
    elif path == "norm":
        r, d = case["r"], case["d"]
        leaves = {"x": (rn(r, d) * (0.5 + un(r, 1)) + rn(r, 1)).to(dt), "weight": (1.0 + 0.1 * rn(d)).to(dt),
                  "bias": (0.1 * rn(d)).to(dt)}
        rest = {"gy": rn(r, d).to(dt)}
    else:
        r, v, k = case["r"], case["v"], case["k"]
        logits = (2.0 * rn(r, v)).to(dt)
        index = torch.randint(0, v, (r, k), device=DEVICE, generator=gen)
        teacher = (3.0 * rn(r, k)).sort(-1, descending=True).values.to(dt)
        # Lists cut short, and rows that have none (prompt tokens, padding).
        keep = torch.randint(max(1, k // 2), k + 1, (r, 1), device=DEVICE, generator=gen)
        keep = keep * (un(r, 1) < 0.9)
        keep[0] = k
        index = torch.where(torch.arange(k, device=DEVICE) < keep, index, -1)
        leaves = {"logits": logits}
        rest = {"teacher": teacher, "index": index}
    return leaves, rest


def prepare(case, seed):
    import bayes_ssm  # noqa: F401  (the package that the calls belong to)

    leaves, rest = _inputs(case, seed)
    if case.get("train"):
        leaves = {k: x.requires_grad_(True) for k, x in leaves.items()}
    return {"case": case, "leaves": leaves, **rest}


# ------------------------------------------------------------------------------------- the operators' calls

def _own(state):
    """The framework's call: (outputs, the output that the upstream gradient belongs to)."""
    case, x = state["case"], state["leaves"]
    path = case["path"]
    if path == "conv":
        from bayes_ssm.conv import causal_conv

        return causal_conv(x["x"], x["weight"], x["bias"], activation="silu", initial_state=x.get("state"),
                           lengths=state["lengths"])
    if path == "scan":
        from bayes_ssm.selective import selective_scan

        return selective_scan(x["x"], x["dt"], x["A"], x["B"], x["C"], D=x["D"], dt_bias=x["dt_bias"],
                              dt_softplus=True, initial_state=x.get("state"), lengths=state["lengths"])
    if path == "step":
        from bayes_ssm.selective import selective_step

        hp, h = case["h"] * case["p"], case["h"]
        row = state["projected"]
        return selective_step(row[:, hp:-h], row[:, -h:], state["conv_state"], state["state"], state["weight"],
                              state["A"], groups=case["g"], conv_bias=state["bias"], activation="silu",
                              D=state["D"], dt_bias=state["dt_bias"], dt_softplus=True,
                              out_states=(state["next_conv_state"], state["next_state"]))
    if path == "norm":
        from bayes_ssm.norm import layer_norm

        return (layer_norm(x["x"], x["weight"], x["bias"], eps=EPS),)
    from bayes_ssm.distill import distillation_loss

    return (distillation_loss(x["logits"], state["teacher"], state["index"], temperature=case["tau"],
                              reduction="mean" if case["train"] else "none"),)


def run(state):
    case = state["case"]
    if not case.get("train"):
        with torch.no_grad():
            return list(_own(state) if own else _plain(state, state["leaves"]))
    leaves = list(state["leaves"].values())
    if own:
        out = _own(state)
        grads = torch.autograd.grad(out[0], leaves, state.get("gy"))
        return [o.detach() for o in out] + list(grads)
    wide = {k: x.detach().float().requires_grad_(True) for k, x in state["leaves"].items()}
    out = _plain(state, wide)
    gy = state.get("gy")
    grads = torch.autograd.grad(out[0], list(wide.values()), None if gy is None else gy.float())
    return [_rounded(case, k, o.detach()) for k, o in enumerate(out)] + [g.to(x.dtype) for g, x in zip(grads, leaves)]


# ------------------------------------------------------------------------------------------ plain forms, 32 bits

def _rounded(case, k, x):
    """The k-th output in its own type: scan states and losses stay float32."""
    single = case["path"] == "distill" or (case["path"] == "scan" and k == 1) or (case["path"] == "step" and k == 2)
    return x if single else x.to(DTYPES[case["dtype"]])


def _plain(state, x):
    """The operator in float32 (``x``: its differentiable inputs); rounded at the end where nothing is differentiated."""
    case = state["case"]
    x = {k: v.float() for k, v in x.items()}
    if case["path"] == "conv":
        out = _plain_conv(x["x"], x["weight"], x["bias"], x.get("state"), state["lengths"])
    elif case["path"] == "scan":
        out = _plain_scan(x["x"], x["dt"], x["A"], x["B"], x["C"], x["D"], x["dt_bias"], x.get("state"),
                          state["lengths"])
    elif case["path"] == "step":
        out = _plain_step(state)
    elif case["path"] == "norm":
        mean = x["x"].mean(-1, keepdim=True)
        var = (x["x"] - mean).square().mean(-1, keepdim=True)
        out = [(x["x"] - mean) * torch.rsqrt(var + EPS) * x["weight"] + x["bias"]]
    else:
        out = [_plain_distill(x["logits"], state["teacher"].float(), state["index"], case["tau"], case["train"])]
    return out if torch.is_grad_enabled() else [_rounded(case, k, o) for k, o in enumerate(out)]


def _plain_conv(x, weight, bias, carried, lengths):
    b, t, c = x.shape
    w = weight.shape[1]
    if carried is None:
        carried = x.new_zeros(b, w - 1, c)
    row = torch.cat((carried, x), 1)
    y = bias + sum(row[:, j:j + t] * weight[:, j] for j in range(w))
    y = y * torch.sigmoid(y)
    if lengths is None:
        return [y, row[:, t:]]
    y = y * (torch.arange(t, device=x.device)[:, None] < lengths[:, None, None])
    last = lengths[:, None] + torch.arange(w - 1, device=x.device)
    return [y, row.gather(1, last[..., None].expand(-1, -1, c))]


def _plain_scan(x, dt, A, B, C, D, dt_bias, carried, lengths):
    """Chunks of 64 tokens: products of the chunk's tokens with each other, and the state carried between chunks."""
    b, t, h, p = x.shape
    g, n = B.shape[2:]
    v = dt + dt_bias
    step = v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))
    if lengths is not None:
        live = torch.arange(t, device=x.device)[:, None] < lengths[:, None, None]
        step = step * live
    state = x.new_zeros(b, h, p, n) if carried is None else carried
    ys = []
    for at in range(0, t, 64):
        s = slice(at, min(t, at + 64))
        u = (x[:, s] * step[:, s, :, None]).transpose(1, 2)                      # [B, H, L, P]
        a = (step[:, s] * A).transpose(1, 2).cumsum(-1)                          # [B, H, L]
        k, q = (z[:, s].transpose(1, 2).repeat_interleave(h // g, 1) for z in (B, C))  # [B, H, L, N]
        below = torch.ones(u.shape[2], u.shape[2], device=x.device).tril() > 0
        decay = torch.exp(torch.where(below, a[..., :, None] - a[..., None, :], -math.inf))
        y = ((q @ k.transpose(-1, -2)) * decay) @ u + torch.exp(a)[..., None] * (q @ state.transpose(-1, -2))
        ys.append(y.transpose(1, 2))
        left = torch.exp(a[..., -1:] - a)[..., None] * u
        state = torch.exp(a[..., -1])[..., None, None] * state + left.transpose(-1, -2) @ k
    y = torch.cat(ys, 1) + D[:, None] * x
    if lengths is not None:
        y = torch.where(live[..., None], y, 0.0)
    return [y, state]


def _plain_step(s):
    case = s["case"]
    b, h, p, n, g = (case[k] for k in "bhpng")
    hp = h * p
    row = s["projected"].float()
    carried = torch.cat((s["conv_state"].float(), row[:, None, hp:-h]), 1)
    y = s["bias"].float() + (carried * s["weight"].float().t()).sum(1)
    y = y * torch.sigmoid(y)
    x = y[:, :hp].reshape(b, h, p)
    k, q = (z.reshape(b, g, n).repeat_interleave(h // g, 1) for z in (y[:, hp:hp + g * n], y[:, hp + g * n:]))
    v = row[:, -h:] + s["dt_bias"]
    step = v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))
    state = torch.exp(step * s["A"])[..., None, None] * s["state"] + (step[..., None] * x)[..., None] * k[:, :, None]
    return [(state * q[:, :, None]).sum(-1) + s["D"][:, None] * x, carried[:, 1:], state]


def _plain_distill(logits, teacher, index, tau, mean):
    there = index >= 0
    rows = there.any(-1)
    p = torch.exp((teacher - teacher.max(-1, keepdim=True).values) / tau) * there
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    log_p = torch.log(torch.where(p > 0, p, 1.0))
    z = (logits - logits.detach().max(-1, keepdim=True).values) / tau
    log_q = z.gather(-1, index.clamp_min(0)) - torch.log(torch.exp(z).sum(-1, keepdim=True))
    loss = tau * tau * (p * (log_p - log_q)).sum(-1)
    loss = torch.where(rows, loss, 0.0)
    return loss.sum() / rows.sum().clamp_min(1) if mean else loss


# --------------------------------------------------------------------------------------------- work, bounds

def work(case):
    path, size, train = case["path"], 4 if case["dtype"] == "f32" else 2, case.get("train", False)
    if path == "conv":
        # x in, y out; with gradients the upstream one in and the input's out.  Taps, bias, SiLU.
        elements, carried = case["b"] * case["t"] * case["c"], case["b"] * (case["w"] - 1) * case["c"]
        w = case["w"]
        return {"bytes": size * (elements * (4 if train else 2) + carried * (1 + case["carry"])),
                "flops": elements * ((2 * w + 6) + ((6 * w + 10) if train else 0))}
    if path == "scan":
        b, t, h, p, n, g = (case[k] for k in "bthpng")
        ins = h * p + h + 2 * g * n
        # Per token, head and state: decay, outer product, read-out; the reverse runs the adjoint's three products
        # and the state's once more.
        return {"bytes": size * b * t * ((2 * ins + 2 * h * p) if train else ins + h * p)
                + 4 * b * h * p * n * (1 + case["carry"]),
                "flops": b * t * h * p * n * (15 if train else 5)}
    if path == "step":
        b, h, p, n, g, w = (case[k] for k in "bhpngw")
        c = h * p + 2 * g * n
        return {"bytes": b * (8 * h * p * n + size * (c + h + h * p + 2 * (w - 1) * c)) + size * c * (w + 1),
                "flops": b * (5 * h * p * n + c * (2 * w + 6))}
    if path == "norm":
        elements = case["r"] * case["d"]
        return {"bytes": size * elements * (4 if train else 2), "flops": elements * (22 if train else 8)}
    # The logits once in, their gradient once out.
    elements = case["r"] * case["v"]
    return {"bytes": size * elements * (2 if train else 1) + case["r"] * case["k"] * (8 + size),
            "flops": elements * (8 if train else 4)}


# ------------------------------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    leaves, rest = _inputs(case, seed)
    leaves = {k: x.double() for k, x in leaves.items()}
    rest = {k: x.double() if torch.is_tensor(x) and x.is_floating_point() else x for k, x in rest.items()}
    if case["path"] == "conv":
        return _exact_conv(leaves, rest, case)
    if case["path"] == "scan":
        return _exact_scan(leaves, rest, case)
    if case["path"] == "step":
        return _exact_step(rest, case)
    if case["path"] == "norm":
        return _exact_norm(leaves, rest, case)
    return _exact_distill(leaves, rest, case)


def _live(case, rest):
    b, t = case["b"], case["t"]
    cut = rest["lengths"] if rest["lengths"] is not None else torch.full((b,), t, device=DEVICE)
    return cut, torch.arange(t, device=DEVICE)[None, :] < cut[:, None]


def _exact_conv(x, rest, case):
    b, t, c, w = (case[k] for k in "btcw")
    cut, live = _live(case, rest)
    row = torch.zeros(b, t + w - 1, c, device=DEVICE, dtype=torch.float64)
    row[:, w - 1:] = x["x"]
    if case["carry"]:
        row[:, :w - 1] = x["state"]
    pre = x["bias"].expand(b, t, c).clone()
    for j in range(w):
        pre += row[:, j:j + t] * x["weight"][:, j]
    gate = 1.0 / (1.0 + torch.exp(-pre))
    out = [pre * gate * live[..., None], torch.stack([row[i, int(cut[i]):int(cut[i]) + w - 1] for i in range(b)])]
    if not case["train"]:
        return out
    g = rest["gy"] * live[..., None] * gate * (1.0 + pre * (1.0 - gate))
    g_row = torch.zeros_like(row)
    g_weight = []
    for j in range(w):
        g_row[:, j:j + t] += g * x["weight"][:, j]
        g_weight.append((g * row[:, j:j + t]).sum((0, 1)))
    out += [g_row[:, w - 1:], torch.stack(g_weight, 1), g.sum((0, 1))]
    return out + ([g_row[:, :w - 1]] if case["carry"] else [])


def _exact_scan(x, rest, case):
    b, t, h, p, n, g = (case[k] for k in "bthpng")
    if b * t * h * p * n > 6e9:
        return None
    _, live = _live(case, rest)
    live = live.double()
    v = x["dt"] + x["dt_bias"]
    step = torch.nn.functional.softplus(v, threshold=40.0) * live[..., None]
    fade = torch.exp(step * x["A"])

    def wide(z, i):  # a group's row for each of its heads
        return z[:, i].unsqueeze(2).expand(b, g, h // g, n).reshape(b, h, n)

    def advance(state, i):
        return (fade[:, i, :, None, None] * state
                + (step[:, i, :, None] * x["x"][:, i]).unsqueeze(-1) * wide(x["B"], i).unsqueeze(-2))

    state = x["state"] if case["carry"] else torch.zeros(b, h, p, n, device=DEVICE, dtype=torch.float64)
    part = 64
    starts, y = [], torch.empty_like(x["x"])
    for i in range(t):
        if i % part == 0:
            starts.append(state)
        state = advance(state, i)
        y[:, i] = (state @ wide(x["C"], i).unsqueeze(-1)).squeeze(-1)
    y = (y + x["D"][:, None] * x["x"]) * live[..., None, None]
    out = [y, state]
    if not case["train"]:
        return out
    gy = rest["gy"] * live[..., None, None]
    gx, gB, gC = x["D"][:, None] * gy, torch.zeros_like(x["B"]), torch.zeros_like(x["C"])
    g_step, adjoint = torch.zeros_like(step), torch.zeros_like(state)
    gA = torch.zeros_like(x["A"])
    for first in reversed(range(0, t, part)):
        states = [starts[first // part]]
        for i in range(first, min(t, first + part)):
            states.append(advance(states[-1], i))
        for i in reversed(range(first, min(t, first + part))):
            before, after = states[i - first], states[i - first + 1]
            gC[:, i] = (gy[:, i].unsqueeze(-2) @ after).reshape(b, g, h // g, n).sum(2)
            adjoint = adjoint + gy[:, i].unsqueeze(-1) * wide(x["C"], i).unsqueeze(-2)
            g_fade = (adjoint * before).sum((-1, -2)) * fade[:, i]
            toward = (adjoint @ wide(x["B"], i).unsqueeze(-1)).squeeze(-1)
            g_step[:, i] = (toward * x["x"][:, i]).sum(-1) + g_fade * x["A"]
            gA += (g_fade * step[:, i]).sum(0)
            gx[:, i] += step[:, i, :, None] * toward
            gB[:, i] = ((step[:, i, :, None] * x["x"][:, i]).unsqueeze(-2) @ adjoint).reshape(b, g, h // g, n).sum(2)
            adjoint = fade[:, i, :, None, None] * adjoint
    g_dt = g_step * torch.sigmoid(v) * live[..., None]
    grads = {"x": gx, "dt": g_dt, "B": gB, "C": gC, "A": gA, "D": (gy * x["x"]).sum((0, 1, 3)),
             "dt_bias": g_dt.sum((0, 1)), "state": adjoint}
    return out + [grads[k] for k in x]


def _exact_step(s, case):
    b, h, p, n, g, w = (case[k] for k in "bhpngw")
    hp, c = h * p, h * p + 2 * g * n
    taps = torch.empty(b, w, c, device=DEVICE, dtype=torch.float64)
    taps[:, :w - 1] = s["conv_state"]
    taps[:, w - 1] = s["projected"][:, hp:hp + c]
    pre = s["bias"] + torch.einsum("bwc,cw->bc", taps, s["weight"])
    out = pre / (1.0 + torch.exp(-pre))
    heads = torch.arange(h, device=DEVICE) // (h // g)
    x = out[:, :hp].view(b, h, p)
    B, C = (z.reshape(b, g, n)[:, heads] for z in out[:, hp:].split(g * n, 1))
    step = torch.nn.functional.softplus(s["projected"][:, hp + c:] + s["dt_bias"], threshold=40.0)
    state = torch.exp(step * s["A"]).view(b, h, 1, 1) * s["state"] + (step.unsqueeze(-1) * x).unsqueeze(-1) * B.unsqueeze(2)
    return [(state @ C.unsqueeze(-1)).squeeze(-1) + s["D"].unsqueeze(-1) * x, taps[:, 1:], state]


def _exact_norm(x, rest, case):
    d = case["d"]
    off = x["x"] - x["x"].sum(-1, keepdim=True) / d
    scale = (off.square().sum(-1, keepdim=True) / d + EPS).rsqrt()
    unit = off * scale
    y = unit * x["weight"] + x["bias"]
    if not case["train"]:
        return [y]
    gy = rest["gy"]
    gu = gy * x["weight"]
    gx = scale * (gu - gu.sum(-1, keepdim=True) / d - unit * (gu * unit).sum(-1, keepdim=True) / d)
    return [y, gx, (gy * unit).sum(0), gy.sum(0)]


def _exact_distill(x, rest, case):
    tau, index = case["tau"], rest["index"]
    there = index >= 0
    rows = there.any(-1)
    count = max(1, int(rows.sum()))
    p = torch.softmax((rest["teacher"] / tau).masked_fill(~there, -math.inf), -1).masked_fill(~there, 0.0)
    log_q = torch.log_softmax(x["logits"] / tau, -1)
    cross = (p * log_q.gather(-1, index.clamp_min(0))).sum(-1)
    loss = tau * tau * (torch.xlogy(p, p).sum(-1) - cross)
    loss = loss.masked_fill(~rows, 0.0)
    if not case["train"]:
        return [loss]
    out = [loss.sum() / count]
    grad = torch.exp(log_q).scatter_add_(-1, index.clamp_min(0), -p)
    return out + [(tau / count * grad).masked_fill(~rows[:, None], 0.0)]

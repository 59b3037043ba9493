"""GPU parity of the short filter, selective scan and step, layer norm and distillation loss against float64 restatements.

Inputs are rounded to the stream's type first, so that both sides compute the
same thing.  Tolerances: tests/_sequence_reference.py.
"""
from __future__ import annotations

import pytest
import torch

from tests import _sequence_reference as R

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
NAN = float("nan")


class Draws:
    def __init__(self, seed, dtype, device):
        self.gen, self.dtype, self.device = torch.Generator().manual_seed(seed), dtype, device

    def normal(self, *shape, scale=1.0, dtype=None):
        return (scale * torch.randn(*shape, generator=self.gen)).to(dtype or self.dtype).to(self.device)

    def lengths(self, b, t):
        cut = torch.randint(0, t + 1, (b,), generator=self.gen)
        cut[0] = 0
        cut[-1] = t
        return cut.to(self.device)


def wide(x, grad=False):
    """The float64 twin of a tensor on the CPU."""
    if x is None:
        return None
    y = x.detach().cpu()
    y = y.double() if y.is_floating_point() else y
    return y.requires_grad_(True) if grad else y


def leaf(x):
    return None if x is None else x.detach().requires_grad_(True)


# ----------------------------------------------------------------------------------------------- filter

CONV = [  # batch, tokens, channels, taps, extra columns, carried, ragged
    (1, 1, 1, 2, 0, False, False), (2, 3, 5, 4, 0, True, False), (3, 37, 16, 3, 8, True, True),
    (2, 300, 72, 4, 0, False, False), (3, 130, 331, 4, 1, True, True), (1, 700, 64, 2, 3, False, True),
    (4, 9, 600, 4, 0, True, True),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("b,t,c,w,extra,carry,ragged", CONV)
def test_conv(cuda_device, dtype, silu, b, t, c, w, extra, carry, ragged):
    from bayes_ssm.conv import causal_conv

    print(f"conv b={b} t={t} c={c} w={w} {dtype}", flush=True)
    d = Draws(b * t + c, dtype, cuda_device)
    x = d.normal(b, t, c + extra)[..., extra:] if extra else d.normal(b, t, c)
    weight, bias = d.normal(c, w, scale=w ** -0.5), d.normal(c, scale=0.3) if silu else None
    state, cut = d.normal(b, w - 1, c) if carry else None, d.lengths(b, t) if ragged else None
    gy, gf = d.normal(b, t, c), d.normal(b, w - 1, c)
    leaves = [leaf(z) for z in (x, weight, bias, state)]
    y, final = causal_conv(leaves[0], leaves[1], leaves[2], activation="silu" if silu else None,
                           initial_state=leaves[3], lengths=cut)
    used = [z for z in leaves if z is not None]
    grads = torch.autograd.grad((y, final), used, (gy, gf))
    refs = [wide(z, True) for z in (x, weight, bias, state)]
    ey, ef = R.conv(refs[0], refs[1], refs[2], silu, refs[3], wide(cut))
    wants = torch.autograd.grad((ey, ef), [z for z in refs if z is not None], (wide(gy), wide(gf)), allow_unused=True)
    tol = R.ROWS if dtype == F32 else R.ROUNDED
    R.check("y", y, ey, tol)
    R.check("final", final, ef, 0.0)
    for name, g, e, z in zip("x weight bias state".split(), grads, wants, used):
        R.check(name, g, torch.zeros(z.shape) if e is None else e, tol)


def test_conv_masked_places_may_hold_anything(cuda_device):
    from bayes_ssm.conv import causal_conv

    d = Draws(5, BF16, cuda_device)
    x, w, gy, cut = d.normal(2, 40, 16), d.normal(16, 4), d.normal(2, 40, 16), torch.tensor([7, 0], device=cuda_device)
    out = []
    for fill in (0.0, NAN):
        xf, gf = x.clone(), gy.clone()
        for i, n in enumerate((7, 0)):
            xf[i, n:], gf[i, n:] = fill, fill
        xl, wl = leaf(xf), leaf(w)
        y, final = causal_conv(xl, wl, activation="silu", lengths=cut)
        out.append([y, final, *torch.autograd.grad(y, (xl, wl), gf)])
    for a, b in zip(*out):
        assert torch.equal(a, b) and torch.isfinite(a).all()


# ------------------------------------------------------------------------------------------------- scan

SCAN = [  # batch, tokens, heads, values, states, groups
    (1, 1, 1, 1, 1, 1), (2, 2, 4, 5, 7, 2), (1, 16, 2, 64, 32, 1), (2, 63, 2, 16, 128, 2), (1, 64, 1, 64, 64, 1),
    (2, 65, 3, 40, 24, 3), (1, 128, 2, 64, 128, 1), (3, 129, 4, 72, 100, 2), (2, 200, 6, 8, 33, 2),
    (1, 257, 2, 130, 128, 1), (1, 1100, 2, 24, 16, 1),
]


def _scan_inputs(d, b, t, h, p, n, g, carry, ragged, fast=1.0):
    dt = d.dtype
    u = torch.rand(h, generator=d.gen)
    step = torch.exp(u * 4.6 - 6.9)  # 0.001 .. 0.1
    return {
        "x": d.normal(b, t, h, p), "dt": d.normal(b, t, h, scale=0.5),
        "A": (-fast * (1 + 15 * torch.rand(h, generator=d.gen))).to(d.device), "B": d.normal(b, t, g, n, scale=0.5),
        "C": d.normal(b, t, g, n, scale=0.5), "D": d.normal(h, dtype=F32),
        "dt_bias": (step + torch.log(-torch.expm1(-step))).to(d.device),
        "state": d.normal(b, h, p, n, scale=0.2, dtype=F32) if carry else None,
        "lengths": d.lengths(b, t) if ragged else None,
    }


def _scan_call(z, softplus=True):
    from bayes_ssm.selective import selective_scan

    return selective_scan(z["x"], z["dt"], z["A"], z["B"], z["C"], D=z["D"], dt_bias=z["dt_bias"],
                          dt_softplus=softplus, initial_state=z["state"], lengths=z["lengths"])


NAMES = ("x", "dt", "A", "B", "C", "D", "dt_bias", "state")


def _scan_compare(z, gy, gs, softplus=True):
    dtype = z["x"].dtype
    own = {k: leaf(v) if k in NAMES else v for k, v in z.items()}
    y, last = _scan_call(own, softplus)
    used = [k for k in NAMES if z[k] is not None]
    up = (gy,) if gs is None else (gy, gs)
    grads = torch.autograd.grad((y, last)[:len(up)], [own[k] for k in used], up)
    ref = {k: wide(v, k in NAMES) for k, v in z.items()}
    # A, D and dt_bias for every token, so that their gradients' terms can be told from their sums.
    b, t, h = z["dt"].shape
    each = {k: None if ref[k] is None else ref[k].detach().expand(b, t, h).contiguous().requires_grad_(True)
            for k in ("A", "D", "dt_bias")}
    ey, elast = R.scan(ref["x"], ref["dt"], each["A"], ref["B"], ref["C"], each["D"], each["dt_bias"], softplus,
                       ref["state"], ref["lengths"])
    inputs = [each.get(k, ref[k]) for k in used]
    wants = torch.autograd.grad((ey, elast)[:len(up)], inputs, [wide(u) for u in up], allow_unused=True)
    bf16 = dtype == BF16
    R.check("y", y, ey, R.ROUNDED_TWICE if bf16 else R.SUMMED)
    R.check("state", last, elast, R.SUMMED)
    for k, got, want, at in zip(used, grads, wants, inputs):
        want = torch.zeros_like(at) if want is None else want
        if k in each:
            R.check(k, got, want.sum((0, 1)), R.SUMMED, scale=want.abs().sum((0, 1)))
        else:
            single = got.dtype == F32
            R.check(k, got, want, R.SUMMED if single else R.ROUNDED if k == "dt" else R.ROUNDED_TWICE)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("carry,ragged", [(False, False), (True, True)])
@pytest.mark.parametrize("b,t,h,p,n,g", SCAN)
def test_scan(cuda_device, dtype, carry, ragged, b, t, h, p, n, g):
    print(f"scan b={b} t={t} h={h} p={p} n={n} g={g} {dtype}", flush=True)
    d = Draws(t + p + n, dtype, cuda_device)
    z = _scan_inputs(d, b, t, h, p, n, g, carry, ragged)
    _scan_compare(z, d.normal(b, t, h, p), d.normal(b, h, p, n, dtype=F32) if carry else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fast", [0.0, 30.0])
def test_scan_decays_at_both_ends(cuda_device, dtype, fast):
    """No decay at all, and decays that leave float32's range within a chunk."""
    d = Draws(11, dtype, cuda_device)
    z = _scan_inputs(d, 2, 150, 2, 16, 32, 1, True, False, fast=fast)
    _scan_compare(z, d.normal(2, 150, 2, 16), d.normal(2, 2, 16, 32, dtype=F32))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_without_softplus_bias_and_skip(cuda_device, dtype):
    d = Draws(12, dtype, cuda_device)
    z = _scan_inputs(d, 2, 70, 4, 16, 16, 2, False, False)
    z.update(dt=z["dt"].abs() * 0.1, D=None, dt_bias=None)
    _scan_compare(z, d.normal(2, 70, 4, 16), None, softplus=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_float32_steps_and_strided_views(cuda_device, dtype):
    """The streams as columns of one wider row, off 16-byte boundaries, dt in float32, one B for the batch (expanded)."""
    d = Draws(13, dtype, cuda_device)
    b, t, h, p, n, g = 2, 90, 4, 16, 24, 2
    z = _scan_inputs(d, b, t, h, p, n, g, False, False)
    row = d.normal(b, t, 3 + h * p + 2 * g * n, scale=0.5)
    z["x"], z["C"] = row[..., 3:3 + h * p].unflatten(-1, (h, p)), row[..., 3 + h * p:3 + h * p + g * n].unflatten(-1, (g, n))
    z["B"] = z["B"][:1].expand(b, t, g, n)
    z["dt"] = z["dt"].float()
    _scan_compare(z, d.normal(b, h, t, p).transpose(1, 2), None)


def test_scan_masked_places_may_hold_anything(cuda_device):
    d = Draws(14, BF16, cuda_device)
    z = _scan_inputs(d, 3, 140, 2, 16, 16, 1, True, False)
    z["lengths"] = torch.tensor([0, 77, -5], device=cuda_device)
    gy, out = d.normal(3, 140, 2, 16), []
    for fill in (0.0, NAN):
        own = {k: v if v is None else v.clone() for k, v in z.items()}
        g = gy.clone()
        for i, n in enumerate((0, 77, 0)):
            for v in (own["x"], own["dt"], own["B"], own["C"], g):
                v[i, n:] = fill
        own = {k: leaf(v) if k in NAMES else v for k, v in own.items()}
        y, last = _scan_call(own)
        out.append([y, last, *torch.autograd.grad(y, [own[k] for k in NAMES], g)])
    for a, b in zip(*out):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert torch.equal(out[0][1][0], z["state"][0]) and torch.equal(out[0][1][2], z["state"][2])


def test_scan_parts_of_a_sequence(cuda_device):
    """A prompt in three calls, each from the state that the last one left, and in one; twice the same bits."""
    d = Draws(15, F32, cuda_device)
    z = _scan_inputs(d, 1, 1500, 2, 32, 64, 1, True, False)
    y, last = _scan_call(z)
    again, _ = _scan_call(z)
    assert torch.equal(y, again)
    ys, state = [], z["state"]
    for first, end in ((0, 1), (1, 700), (700, 1500)):
        part = {k: v[:, first:end] if k in ("x", "dt", "B", "C") else v for k, v in z.items()}
        yi, state = _scan_call({**part, "state": state})
        ys.append(yi)
    R.check("y", torch.cat(ys, 1), y, R.SUMMED)
    R.check("state", state, last, R.SUMMED)


def test_scan_gradient_is_the_slope(cuda_device):
    """The kernels' gradient along a direction against differences of the float64 scan."""
    d = Draws(16, F32, cuda_device)
    z = _scan_inputs(d, 1, 140, 2, 16, 16, 1, True, False)
    gy = d.normal(1, 140, 2, 16)
    own = {k: leaf(v) if k in NAMES else v for k, v in z.items()}
    grads = torch.autograd.grad(_scan_call(own)[0], [own[k] for k in NAMES], gy)
    way = {k: 0.05 * torch.randn(z[k].shape, generator=d.gen, dtype=torch.float64) for k in NAMES}
    at = {k: wide(v) for k, v in z.items()}

    def value(e):
        m = {k: at[k] + e * way[k] for k in NAMES}
        y, _ = R.scan(m["x"], m["dt"], m["A"], m["B"], m["C"], m["D"], m["dt_bias"], True, m["state"])
        return float((y * wide(gy)).sum())

    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    terms = [float((wide(g) * way[k]).sum()) for k, g in zip(NAMES, grads)]
    assert abs(sum(terms) - slope) <= 1e-5 * sum(abs(x) for x in terms) + 1e-6 * abs(slope)


def test_scan_of_nothing(cuda_device):
    d = Draws(17, BF16, cuda_device)
    for b, t in ((0, 5), (2, 0)):
        z = _scan_inputs(d, b, t, 2, 8, 8, 1, True, False)
        own = {k: leaf(v) if k in NAMES else v for k, v in z.items()}
        y, last = _scan_call(own)
        gl = d.normal(b, 2, 8, 8, dtype=F32)
        grads = torch.autograd.grad((y, last), [own[k] for k in NAMES], (torch.zeros_like(y), gl))
        assert y.shape == (b, t, 2, 8) and torch.equal(last, z["state"]) and torch.equal(grads[-1], gl)
        assert all(not g.any() for g in grads[:-1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_streams_far_apart(cuda_device, dtype):
    """Rows whose offsets pass 2^31 elements."""
    from bayes_ssm.conv import causal_conv
    from bayes_ssm.norm import layer_norm

    d = Draws(18, dtype, cuda_device)
    far = torch.empty((1 << 31) + (1 << 26), device=cuda_device, dtype=dtype)
    x = torch.as_strided(far, (1, 66, 32), (0, 1 << 25, 1))
    x.copy_(d.normal(1, 66, 32))
    near, w = x.clone(), d.normal(32, 4)
    assert torch.equal(causal_conv(x, w)[0], causal_conv(near, w)[0])
    assert torch.equal(layer_norm(x[0]), layer_norm(near[0]))
    z = _scan_inputs(d, 1, 66, 2, 16, 16, 1, False, False)
    outs = [_scan_call({**z, "x": v.unflatten(-1, (2, 16)), "B": v[..., :16].unsqueeze(2)}) for v in (x, near)]
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------- step

STEP = [  # batch, heads, values, states, groups, taps
    (1, 1, 1, 1, 1, 2), (3, 4, 5, 7, 2, 4), (2, 6, 40, 24, 3, 3), (5, 8, 64, 64, 2, 4), (70, 16, 64, 128, 1, 4),
    (2, 4, 130, 100, 4, 4),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("b,h,p,n,g,w", STEP)
def test_step(cuda_device, dtype, b, h, p, n, g, w):
    from bayes_ssm.selective import selective_step

    print(f"step b={b} h={h} p={p} n={n} g={g} w={w} {dtype}", flush=True)
    d = Draws(b + p + n, dtype, cuda_device)
    c = h * p + 2 * g * n
    row = d.normal(b, c + h + 1)
    weight, bias, conv_state = d.normal(c, w, scale=w ** -0.5), d.normal(c, scale=0.1), d.normal(b, w - 1, c)
    z = _scan_inputs(d, b, 1, h, p, n, g, True, False)
    y, nc, ns = selective_step(row[:, 1:1 + c], row[:, 1 + c:], conv_state, z["state"], weight, z["A"], groups=g,
                               conv_bias=bias, D=z["D"], dt_bias=z["dt_bias"])
    wrow = wide(row)
    f, ef = R.conv(wrow[:, None, 1:1 + c], wide(weight), wide(bias), True, wide(conv_state))
    x, B, C = f.split((h * p, g * n, g * n), -1)
    ey, es = R.scan(x.reshape(b, 1, h, p), wrow[:, None, 1 + c:], wide(z["A"]), B.reshape(b, 1, g, n),
                    C.reshape(b, 1, g, n), wide(z["D"]), wide(z["dt_bias"]), True, wide(z["state"]))
    R.check("y", y, ey[:, 0], R.ROWS if dtype == F32 else R.ROUNDED)
    R.check("conv_state", nc, ef, 0.0)
    R.check("state", ns, es, R.ROWS)
    # Into given tensors, the state in place.
    state, out = z["state"].clone(), torch.empty_like(conv_state)
    y2, nc2, ns2 = selective_step(row[:, 1:1 + c], row[:, 1 + c:], conv_state, state, weight, z["A"], groups=g,
                                  conv_bias=bias, D=z["D"], dt_bias=z["dt_bias"], out_states=(out, state))
    assert nc2 is out and ns2 is state and torch.equal(y2, y) and torch.equal(state, ns) and torch.equal(out, nc)


def test_prompt_then_steps(cuda_device):
    """A prompt and then single tokens against the whole sequence at once."""
    from bayes_ssm.conv import causal_conv
    from bayes_ssm.selective import selective_scan, selective_step

    d = Draws(20, F32, cuda_device)
    b, t, h, p, n, g, w = 2, 77, 4, 16, 32, 2, 4
    c = h * p + 2 * g * n
    rows, dt, weight, bias = d.normal(b, t, c), d.normal(b, t, h), d.normal(c, w, scale=0.5), d.normal(c)
    z = _scan_inputs(d, b, 1, h, p, n, g, False, False)
    extra = dict(D=z["D"], dt_bias=z["dt_bias"])

    def prompt(end):
        f, cs = causal_conv(rows[:, :end], weight, bias, activation="silu")
        x, B, C = f.split((h * p, g * n, g * n), -1)
        y, s = selective_scan(x.unflatten(-1, (h, p)), dt[:, :end], z["A"], B.unflatten(-1, (g, n)),
                              C.unflatten(-1, (g, n)), **extra)
        return y, cs, s

    whole, whole_cs, whole_s = prompt(t)
    _, cs, s = prompt(70)
    for i in range(70, t):
        y, cs, s = selective_step(rows[:, i], dt[:, i], cs, s, weight, z["A"], groups=g, conv_bias=bias, **extra)
        R.check("y", y, whole[:, i], R.SUMMED)
    assert torch.equal(cs, whole_cs)
    R.check("state", s, whole_s, R.SUMMED)


def test_step_in_a_graph_and_on_another_stream(cuda_device):
    from bayes_ssm.selective import selective_step

    d = Draws(21, BF16, cuda_device)
    b, h, p, n = 3, 4, 64, 128
    c = h * p + 2 * n
    row, dt, weight, cs = d.normal(b, c), d.normal(b, h), d.normal(c, 4), d.normal(b, 3, c)
    z = _scan_inputs(d, b, 1, h, p, n, 1, True, False)
    state, conv_a, conv_b = z["state"].clone(), cs.clone(), torch.empty_like(cs)

    def two_tokens():
        with torch.no_grad():
            selective_step(row, dt, conv_a, state, weight, z["A"], out_states=(conv_b, state))
            return selective_step(row, dt, conv_b, state, weight, z["A"], out_states=(conv_a, state))[0]

    want_y, want = [], []
    for _ in range(4):
        want_y.append(two_tokens().clone())
        want.append(state.clone())
    state.copy_(z["state"]), conv_a.copy_(cs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two_tokens()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = two_tokens()
    state.copy_(z["state"]), conv_a.copy_(cs)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want_y[i]) and torch.equal(state, want[i])


# ------------------------------------------------------------------------------------------------- norm

NORM = [(1, 1), (3, 7), (9, 33), (257, 64), (5, 1000), (37, 2048), (3, 2056), (4, 8192), (2, 9001), (3, 40000), (1500, 24)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("params", ["same", "float32", "weight", "none"])
@pytest.mark.parametrize("r,w", NORM)
def test_norm(cuda_device, dtype, params, r, w):
    from bayes_ssm.norm import layer_norm

    print(f"norm r={r} w={w} {dtype} {params}", flush=True)
    d = Draws(r + w, dtype, cuda_device)
    x = (d.normal(r, w, dtype=F32) + 3.0 * d.normal(r, 1, dtype=F32)).to(dtype)
    kind = dtype if params == "same" else F32
    weight = None if params == "none" else 1.0 + d.normal(w, scale=0.2, dtype=kind)
    bias = None if params in ("none", "weight") else d.normal(w, dtype=kind)
    gy = d.normal(r, w)
    leaves = [leaf(z) for z in (x, weight, bias)]
    y = layer_norm(*leaves)
    used = [z for z in leaves if z is not None]
    grads = torch.autograd.grad(y, used, gy)
    refs = [wide(z, True) for z in (x, weight, bias)]
    want = R.norm(*refs)
    wants = torch.autograd.grad(want, [z for z in refs if z is not None], wide(gy))
    R.check("y", y, want, R.ROWS if dtype == F32 else R.ROUNDED)
    if w > 1:  # one value a row: the gradient is exactly zero
        R.check("x", grads[0], wants[0], R.SUMMED if dtype == F32 else R.ROUNDED)
    for name, g, e in zip(("weight", "bias"), grads[1:], wants[1:]):
        scale = wide(gy).abs().sum(0) if w == 1 or r == 1 else None
        R.check(name, g, e, R.SUMMED if g.dtype == F32 else R.ROUNDED, scale=scale)


def test_norm_of_a_large_mean_strided_and_empty_rows(cuda_device):
    from bayes_ssm.norm import layer_norm

    d = Draws(30, F32, cuda_device)
    x = 1000.0 + d.normal(4, 513)
    # x itself is rounded in steps of 2^-14; the mean's rounding, 2^-15, is the error against values of size 1.
    R.check("mean 1000", layer_norm(x), R.norm(wide(x)), 1e-4)
    row = d.normal(6, 3, 100)
    view = row[:, 1, 7:71]
    R.check("strided", layer_norm(view), R.norm(wide(view)), R.ROWS)
    w, b = leaf(d.normal(64)), leaf(d.normal(64))
    gw, gb = torch.autograd.grad(layer_norm(x[:0, :64], w, b), (w, b), x[:0, :64])
    assert not gw.any() and not gb.any()
    same = torch.full((2, 64), 3.0, device=cuda_device)
    assert not layer_norm(same).any()


# ---------------------------------------------------------------------------------------------- distill

DISTILL = [(1, 1, 1), (3, 11, 4), (30, 101, 7), (17, 3200, 64), (5, 5001, 1024), (4, 40000, 33), (2, 130001, 2)]


def _distill_inputs(d, r, v, k):
    x, t = d.normal(r, v, scale=2.0), d.normal(r, k, scale=2.0)
    index = torch.randint(0, v, (r, k), generator=d.gen)
    index[torch.rand(r, k, generator=d.gen) < 0.2] = -1
    index[0] = torch.randint(0, v, (k,), generator=d.gen)
    if r > 2:
        index[1] = -1
        index[2, 0] = v + 3
        t[2, -1] = float("-inf")
    return x, t, index.to(d.device)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tau", [0.5, 2.0])
@pytest.mark.parametrize("r,v,k", DISTILL)
def test_distill(cuda_device, dtype, tau, r, v, k):
    from bayes_ssm.distill import distillation_loss

    print(f"distill r={r} v={v} k={k} {dtype}", flush=True)
    d = Draws(r + v, dtype, cuda_device)
    x, t, index = _distill_inputs(d, r, v, k)
    up = d.normal(r, dtype=F32)
    ref = wide(x, True)
    losses = R.distill(ref, wide(t), index.cpu(), tau)
    listed = ((index >= 0) & (index < v) & (t > float("-inf"))).any(-1)
    count = max(1, int(listed.sum()))
    # p log p and p log q cancel where the student agrees: their own size is the scale.
    scale = losses.detach().abs() + tau * tau
    for reduction, want, g in (("none", losses, up), ("sum", losses.sum(), 2.5), ("mean", losses.sum() / count, 0.5)):
        xl = leaf(x)
        loss = distillation_loss(xl, t, index, temperature=tau, reduction=reduction)
        g = g if torch.is_tensor(g) else torch.tensor(g, device=x.device)
        got, = torch.autograd.grad(loss, xl, g)
        expected, = torch.autograd.grad(want, ref, wide(g), retain_graph=True)
        R.check(reduction, loss, want, R.SUMMED, scale=scale if reduction == "none" else scale.sum())
        # One entry of the vocabulary: q - p is exactly 0.
        if v > 1:
            R.check(reduction + " gradient", got, expected, R.SUMMED if dtype == F32 else R.ROUNDED)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_masked_vocabulary(cuda_device, dtype):
    """Entries at -infinity and at the type's lowest value, a row of nothing else, NaN in rows without a teacher."""
    from bayes_ssm.distill import distillation_loss

    d = Draws(40, dtype, cuda_device)
    x, t = d.normal(5, 600), d.normal(5, 3)
    index = torch.tensor([[1, 2, 3], [4, 5, 6], [7, 8, 9], [-1, -1, -1], [0, 1, 1]], device=cuda_device)
    x[0, 100:] = float("-inf")
    x[1, 100:] = torch.finfo(dtype).min
    x[2] = torch.finfo(dtype).min
    x[3] = NAN
    ref = wide(x).clone()
    ref[3] = 0.0
    ref.requires_grad_(True)
    xl = leaf(x)
    loss = distillation_loss(xl, t, index, temperature=0.5, reduction="none")
    got, = torch.autograd.grad(loss, xl, torch.ones(5, device=cuda_device))
    # In float64 the lowest values / 0.5 are finite too.
    want = R.distill(ref, wide(t), index.cpu(), 0.5)
    expected, = torch.autograd.grad(want.sum(), ref)
    R.check("loss", loss, want, R.SUMMED)
    R.check("gradient", got, expected, R.SUMMED if dtype == F32 else R.ROUNDED)
    assert not got[3].any() and not got[0, 100:].any()


def test_distill_strided_rows_and_backward_twice(cuda_device):
    from bayes_ssm.distill import distillation_loss

    d = Draws(41, BF16, cuda_device)
    x, t, index = _distill_inputs(d, 9, 1003, 5)
    wide_rows = d.normal(9, 1100)
    wide_rows[:, 3:1006] = x
    a, b = leaf(x), leaf(wide_rows)
    la, lb = distillation_loss(a, t, index.int()), distillation_loss(b[:, 3:1006], t, index)
    assert torch.equal(la, lb)
    ga, = torch.autograd.grad(la, a, retain_graph=True)
    keep = ga.clone()
    twice, = torch.autograd.grad(la, a, torch.tensor(2.0, device=cuda_device), retain_graph=True)
    assert torch.equal(ga, keep)
    assert torch.equal(twice, 2 * ga)
    gb, = torch.autograd.grad(lb, b)
    assert torch.equal(gb[:, 3:1006], ga)


def test_distill_of_many_rows(cuda_device):
    """More than 2^31 logits: the last rows as they are by themselves."""
    from bayes_ssm.distill import distillation_loss

    d = Draws(42, BF16, cuda_device)
    r, v = 17000, 130000
    x = torch.zeros(r, v, device=cuda_device, dtype=BF16)
    x[-3:] = d.normal(3, v)
    t, index = d.normal(r, 2), torch.randint(0, v, (r, 2), generator=d.gen).to(cuda_device)
    xl = leaf(x)
    loss = distillation_loss(xl, t, index, reduction="none")
    got, = torch.autograd.grad(loss, xl, torch.ones(r, device=cuda_device))
    few = leaf(x[-3:])
    want = distillation_loss(few, t[-3:], index[-3:], reduction="none")
    expected, = torch.autograd.grad(want, few, torch.ones(3, device=cuda_device))
    assert torch.equal(loss[-3:], want) and torch.equal(got[-3:], expected)


def test_refusals_on_the_gpu(cuda_device):
    from bayes_ssm.distill import distillation_loss
    from bayes_ssm.selective import selective_scan

    z = torch.zeros(1, 1, 1, 129, device=cuda_device)
    with pytest.raises(ValueError, match="at most 128"):
        selective_scan(z[..., :8], z[..., 0], torch.zeros(1, device=cuda_device), z, z)
    many = torch.zeros(1, 1025, device=cuda_device)
    with pytest.raises(ValueError, match="at most 1024"):
        distillation_loss(many, many, many.long())
    with pytest.raises(ValueError, match="device"):
        selective_scan(z[..., :8], z[..., 0], torch.zeros(1), z, z)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("p,n,groups", [(64, 128, 1), (40, 24, 2)])
def test_scan_single_token_without_state(cuda_device, dtype, p, n, groups):
    """One token from a zero state has no decay in its output: A's gradient is 0, not the rounding of what cancels."""
    from bayes_ssm.selective import selective_scan

    torch.manual_seed(3)
    b, h = 5, 2 * groups
    x, B, C = (torch.randn(b, 1, *s, device=cuda_device).to(dtype).requires_grad_(True)
               for s in ((h, p), (groups, n), (groups, n)))
    dt = torch.randn(b, 1, h, device=cuda_device).to(dtype)
    A = (-torch.rand(h, device=cuda_device) - 0.1).requires_grad_(True)
    y, _ = selective_scan(x, dt, A, B, C)
    (gA,) = torch.autograd.grad(y, (A,), torch.randn_like(y))
    assert torch.equal(gA, torch.zeros_like(gA))

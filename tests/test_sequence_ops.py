"""The operators around a selective state space block on the CPU: formulas, gradients by differences, refusals."""
from __future__ import annotations

import pytest
import torch

from tests import _sequence_reference as R


def _rand(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("w", [2, 3, 4])
@pytest.mark.parametrize("carry,cut", [(False, None), (True, [0, 3, 9])])
def test_conv_formula(w, carry, cut):
    from bayes_ssm.conv import causal_conv

    x, weight, bias = _rand(3, 7, 5), _rand(5, w), _rand(5)
    state = _rand(3, w - 1, 5) if carry else None
    lengths = None if cut is None else torch.tensor(cut)
    out = causal_conv(x, weight, bias, activation="silu", initial_state=state, lengths=lengths)
    for got, want in zip(out, R.conv(x, weight, bias, True, state, lengths)):
        R.check("conv", got, want, 1e-12)


@pytest.mark.parametrize("softplus,extras,cut", [(True, True, None), (False, False, None), (True, True, [0, 4])])
def test_scan_formula(softplus, extras, cut):
    from bayes_ssm.selective import selective_scan

    x, dt, B, C = _rand(2, 6, 4, 3), _rand(2, 6, 4).abs() * 0.3, _rand(2, 6, 2, 5), _rand(2, 6, 2, 5, seed=1)
    A, D, bias = -_rand(4).abs(), _rand(4, seed=1), _rand(4, seed=2)
    state = _rand(2, 4, 3, 5) if extras else None
    lengths = None if cut is None else torch.tensor(cut)
    kw = dict(D=D, dt_bias=bias) if extras else {}
    out = selective_scan(x, dt, A, B, C, dt_softplus=softplus, initial_state=state, lengths=lengths, **kw)
    want = R.scan(x, dt, A, B, C, softplus=softplus, state=state, lengths=lengths, **kw)
    for got, e in zip(out, want):
        R.check("scan", got, e, 1e-12)


def test_gradients_by_differences():
    from bayes_ssm.conv import causal_conv
    from bayes_ssm.distill import distillation_loss
    from bayes_ssm.norm import layer_norm
    from bayes_ssm.selective import selective_scan

    def leaf(*shape, seed=0):
        return _rand(*shape, seed=seed).requires_grad_(True)

    cut = torch.tensor([2, 4])
    assert torch.autograd.gradcheck(
        lambda x, w, b, s: causal_conv(x, w, b, activation="silu", initial_state=s, lengths=cut),
        (leaf(2, 4, 3), leaf(3, 4), leaf(3), leaf(2, 3, 3)))
    assert torch.autograd.gradcheck(
        lambda x, dt, a, b, c, d, bias, s: selective_scan(x, dt, -a.exp(), b, c, D=d, dt_bias=bias, initial_state=s,
                                                          lengths=cut),
        (leaf(2, 4, 2, 3), leaf(2, 4, 2), leaf(2), leaf(2, 4, 1, 3), leaf(2, 4, 1, 3, seed=1), leaf(2, seed=1),
         leaf(2, seed=2), leaf(2, 2, 3, 3)))
    assert torch.autograd.gradcheck(layer_norm, (leaf(3, 7), leaf(7), leaf(7, seed=1)))
    index = torch.tensor([[0, 3, 3], [5, -1, 9], [-1, -1, -1]])
    teacher = _rand(3, 3)
    assert torch.autograd.gradcheck(lambda x: distillation_loss(x, teacher, index, temperature=1.5), (leaf(3, 6),))


def test_step_formula_is_conv_and_scan():
    from bayes_ssm.conv import causal_conv
    from bayes_ssm.selective import selective_scan, selective_step

    b, t, h, p, n, g, w = 2, 5, 4, 3, 4, 2, 4
    c = h * p + 2 * g * n
    rows, dt, weight, bias = _rand(b, t, c), _rand(b, t, h), _rand(c, w), _rand(c)
    A, D = -_rand(h).abs(), _rand(h, seed=3)
    z, conv_state = causal_conv(rows, weight, bias, activation="silu")
    x, B, C = z.split((h * p, g * n, g * n), -1)
    y, state = selective_scan(x.reshape(b, t, h, p), dt, A, B.reshape(b, t, g, n), C.reshape(b, t, g, n), D=D)
    cs, s = torch.zeros(b, w - 1, c, dtype=torch.float64), torch.zeros(b, h, p, n, dtype=torch.float64)
    for i in range(t):
        yi, cs, s = selective_step(rows[:, i], dt[:, i], cs, s, weight, A, groups=g, conv_bias=bias, D=D)
        R.check("y", yi, y[:, i], 1e-12)
    R.check("conv_state", cs, conv_state, 1e-12)
    R.check("state", s, state, 1e-12)


@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_distill_formula(tau):
    from bayes_ssm.distill import distillation_loss

    x, teacher = _rand(5, 11), _rand(5, 4)
    index = torch.tensor([[0, 1, 2, 3], [10, 10, 4, -1], [-1, -1, -1, -1], [11, 5, 6, -7], [0, 1, 2, 3]])
    teacher[4, :3] = float("-inf")
    want = R.distill(x, teacher, index, tau)
    R.check("none", distillation_loss(x, teacher, index, temperature=tau, reduction="none"), want, 1e-12)
    R.check("sum", distillation_loss(x, teacher, index, temperature=tau, reduction="sum"), want.sum(), 1e-12)
    R.check("mean", distillation_loss(x, teacher, index, temperature=tau), want.sum() / 4, 1e-12)


def test_norm_module_and_empty_rows():
    from bayes_ssm.norm import LayerNorm, layer_norm

    m = LayerNorm(6, dtype=torch.float64)
    x = _rand(2, 3, 6)
    R.check("norm", m(x), R.norm(x, m.weight, m.bias), 1e-12)
    assert layer_norm(x[:0]).shape == (0, 3, 6)
    assert LayerNorm(6, bias=False).bias is None


def _scan_args():
    return dict(x=torch.zeros(2, 3, 4, 5), dt=torch.zeros(2, 3, 4), A=torch.zeros(4), B=torch.zeros(2, 3, 2, 6),
                C=torch.zeros(2, 3, 2, 6))


@pytest.mark.parametrize("change,kind", [
    (dict(x=torch.zeros(2, 3, 4)), ValueError), (dict(dt=torch.zeros(2, 3, 5)), ValueError),
    (dict(A=torch.zeros(3)), ValueError), (dict(B=torch.zeros(2, 3, 3, 6), C=torch.zeros(2, 3, 3, 6)), ValueError),
    (dict(C=torch.zeros(2, 3, 2, 7)), ValueError), (dict(B=torch.zeros(2, 3, 2, 6).bfloat16()), TypeError),
    (dict(x=torch.zeros(2, 3, 4, 5, dtype=torch.int32)), TypeError), (dict(D=torch.zeros(5)), ValueError),
    (dict(dt_bias=torch.zeros(1)), ValueError), (dict(initial_state=torch.zeros(2, 4, 5, 7)), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError), (dict(lengths=torch.zeros(2)), TypeError),
])
def test_scan_refuses(change, kind):
    from bayes_ssm.selective import selective_scan

    kw = {**_scan_args(), **change}
    args = [kw.pop(k) for k in ("x", "dt", "A", "B", "C")]
    with pytest.raises(kind):
        selective_scan(*args, **kw)


@pytest.mark.parametrize("change,kind", [
    (dict(x=torch.zeros(2, 3)), ValueError), (dict(weight=torch.zeros(5, 5)), ValueError),
    (dict(weight=torch.zeros(4, 4)), ValueError), (dict(bias=torch.zeros(4)), ValueError),
    (dict(activation="gelu"), ValueError), (dict(initial_state=torch.zeros(2, 2, 5)), ValueError),
    (dict(initial_state=torch.zeros(2, 3, 5).bfloat16()), TypeError), (dict(lengths=torch.zeros(2)), TypeError),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), ValueError),
])
def test_conv_refuses(change, kind):
    from bayes_ssm.conv import causal_conv

    kw = {**dict(x=torch.zeros(2, 3, 5), weight=torch.zeros(5, 4)), **change}
    with pytest.raises(kind):
        causal_conv(kw.pop("x"), kw.pop("weight"), **kw)


def _step_args():
    return dict(row=torch.zeros(2, 32), dt=torch.zeros(2, 4), conv_state=torch.zeros(2, 3, 32),
                state=torch.zeros(2, 4, 5, 3), conv_weight=torch.zeros(32, 4), A=torch.zeros(4), groups=2)


@pytest.mark.parametrize("change,kind", [
    (dict(row=torch.zeros(2, 33)), ValueError), (dict(groups=3), ValueError), (dict(dt=torch.zeros(2, 3)), ValueError),
    (dict(conv_state=torch.zeros(2, 2, 32)), ValueError), (dict(conv_weight=torch.zeros(32, 5)), ValueError),
    (dict(conv_bias=torch.zeros(3)), ValueError), (dict(activation="relu"), ValueError),
    (dict(A=torch.zeros(4, requires_grad=True)), RuntimeError),
    (dict(out_states=(torch.zeros(2, 3, 32), torch.zeros(2, 4, 5, 4))), ValueError),
])
def test_step_refuses(change, kind):
    from bayes_ssm.selective import selective_step

    kw = {**_step_args(), **change}
    args = [kw.pop(k) for k in ("row", "dt", "conv_state", "state", "conv_weight", "A")]
    with pytest.raises(kind):
        selective_step(*args, **kw)


def test_step_refuses_overlapping_states():
    from bayes_ssm.selective import selective_step

    kw = _step_args()
    args = [kw.pop(k) for k in ("row", "dt", "conv_state", "state", "conv_weight", "A")]
    out = selective_step(*args, **kw, out_states=(torch.zeros(2, 3, 32), args[3]))
    assert out[2] is args[3]
    with pytest.raises(ValueError, match="overlap"):
        selective_step(*args, **kw, out_states=(args[2], args[3]))
    both = torch.zeros(2 * 4 * 5 * 3 + 4)
    state, shifted = both[:120].view(2, 4, 5, 3), both[4:].view(2, 4, 5, 3)
    args[3] = state
    with pytest.raises(ValueError, match="overlap"):
        selective_step(*args, **kw, out_states=(torch.zeros(2, 3, 32), shifted))


@pytest.mark.parametrize("call", [
    lambda m: m.layer_norm(torch.zeros(3, 4, dtype=torch.int32)), lambda m: m.layer_norm(torch.zeros(3, 0)),
    lambda m: m.layer_norm(torch.zeros(3, 4), torch.zeros(5)), lambda m: m.layer_norm(torch.zeros(3, 4), eps=-1.0),
    lambda m: m.layer_norm(torch.zeros(3, 4), None, torch.zeros(3)),
])
def test_norm_refuses(call):
    from bayes_ssm import norm

    with pytest.raises((TypeError, ValueError)):
        call(norm)


@pytest.mark.parametrize("change,kind", [
    (dict(temperature=0.0), ValueError), (dict(temperature=float("inf")), ValueError), (dict(reduction="max"), ValueError),
    (dict(index=torch.zeros(3, 2)), TypeError), (dict(index=torch.zeros(3, 3, dtype=torch.int64)), ValueError),
    (dict(logits=torch.zeros(4, 5)), ValueError), (dict(logits=torch.zeros(3, 0)), ValueError),
])
def test_distill_refuses(change, kind):
    from bayes_ssm.distill import distillation_loss

    kw = {**dict(logits=torch.zeros(3, 5), teacher=torch.zeros(3, 2), index=torch.zeros(3, 2, dtype=torch.int64)), **change}
    with pytest.raises(kind):
        distillation_loss(kw.pop("logits"), kw.pop("teacher"), kw.pop("index"), **kw)


def test_c_entry_points_refuse():
    """Argument errors come back as codes, without touching a device."""
    from bayes_ssm import _hip

    lib = _hip.load()

    def conv(w=4, b=1, t=1, c=1):
        return lib.bssm_short_conv_forward(0, 0, w, 0, None, 0, 0, None, None, None, None, None, None, b, t, c, None)

    assert conv(w=5) == 2 and conv(b=-1) == 1 and conv() == 1 and conv(b=0) == 0
    assert lib.bssm_layer_norm_forward(0, 0, None, 1, None, None, 1e-5, None, None, None, 0, 1, None) == 0
    assert lib.bssm_layer_norm_forward(0, 0, None, 1, None, None, -1.0, None, None, None, 0, 1, None) == 1
    assert lib.bssm_distill_forward(0, 0, None, 1, None, None, 1.0, None, None, None, None, 0, None, 1, 1, 2000, None) == 2
    assert lib.bssm_distill_forward(0, 0, None, 1, None, None, 0.0, None, None, None, None, 0, None, 1, 1, 1, None) == 1

    def scan(h=4, n=8, g=2, b=1):
        return lib.bssm_select_forward(0, None, 0, 0, 0, 0, None, 0, 0, None, None, 0, 0, 0, None, 0, 0, 0, None, None, 1,
                                       None, None, None, None, None, None, None, b, 4, h, 8, n, g, None)

    assert scan(n=129) == 2 and scan(g=3) == 1 and scan(b=-1) == 1 and scan() == 1 and scan(b=0) == 0
    assert b"null" in (scan(), lib.bssm_last_error())[1]
    assert lib.bssm_select_step(0, 0, 5, 0, None, 0, 0, None, 0, None, None, None, None, None, None, None, 1, None, None,
                                None, 1, 4, 8, 8, 2, None) == 2

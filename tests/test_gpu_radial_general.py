"""-m gpu: radial networks whose activation is not the shifted softplus: infinite inputs, second order, and how many products it takes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-24


def _net(device, hs=(8, 64, 64, 100), rows=300):
    g = torch.Generator(device=device).manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    return r(rows, hs[0]), [r(a, b) for a, b in zip(hs, hs[1:])]


def _plain(x, ws, act):
    f = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[act]
    for i, w in enumerate(ws):
        x = x @ w / math.sqrt(w.shape[0])
        x = 1.3 * f(x) if i < len(ws) - 1 else x
    return x


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
def test_an_infinite_input_saturates(device, act):
    """As in fp32 arithmetic: the hidden units are at their limits, and the output is the number that follows from those."""
    from matten_amd import _lib, ops

    x, ws = _net(device)
    x[3, 2], x[77, 5] = math.inf, -math.inf
    got, want = ops.radial_mlp_general(x, ws, 1.3, _lib.ACT[act]), _plain(x.double(), [w.double() for w in ws], act)
    assert torch.isfinite(want).all()
    # (three layers of sums of at most 64 products, Lipschitz activations)
    assert ((got.double() - want).abs() <= 3 * (64 + 16) * U * want.abs().max()).all()


def test_infinite_results_keep_their_sign(device):
    from matten_amd import _lib, ops

    x, ws = _net(device, hs=(8, 24, 40))
    x, ws = x.abs(), [ws[0].abs(), ws[1]]
    x[9, 1] = math.inf
    got = ops.radial_mlp_general(x, [ws[0][:, :1], ws[1][:1]], 1.3, _lib.ACT["silu"])
    assert torch.equal(got[9], math.inf * ws[1][0].sign()) and torch.isfinite(got[:9]).all() and torch.isfinite(got[10:]).all()


@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_second_order(device, act, monkeypatch):
    """The gradient of a function of the input's gradient, as under a loss on forces, against 64 bits (2-norms: 256 roundings in a row of
    sums of at most 300); every layer's backward is two products."""
    from matten_amd import _lib, ops

    x, ws = _net(device)

    def second(f, x, ws):
        x, ws = x.clone().requires_grad_(True), [w.clone().requires_grad_(True) for w in ws]
        y = f(x, ws)
        first = torch.autograd.grad(y, [x, *ws], torch.ones_like(y), create_graph=True)
        return [*first, *torch.autograd.grad((first[0] ** 2).sum(), [x, *ws])]

    products, gemm = [], ops._gemm
    monkeypatch.setattr(ops, "_gemm", lambda *a, **k: (products.append(a[:3]), gemm(*a, **k)))

    def counted(x, ws):
        y = ops.radial_mlp_general(x, ws, 1.3, _lib.ACT[act])
        assert products == [(300, 64, 8), (300, 64, 64), (300, 100, 64)]
        del products[:]
        torch.autograd.grad(y, [x, *ws], torch.ones_like(y), create_graph=True)
        assert len(products) == 6
        return y

    got = second(counted, x, ws)
    want = second(lambda x, ws: _plain(x, ws, act), x.double(), [w.double() for w in ws])
    for a, e in zip(got, want):
        assert (a.double() - e).norm() <= 256 * U * e.norm()

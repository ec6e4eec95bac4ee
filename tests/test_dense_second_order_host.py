"""CPU: the differentiable backward of the dense product, with the launch replaced by torch's product: which products it takes, in
which type, and its derivatives against the formula's in 64 bits."""
import math

import pytest
import torch

ACTS = ["identity", "ssp", "silu", "tanh", "abs", "sigmoid", "gelu"]


def _plain(x, w, b, act, alpha, cst):
    F = torch.nn.functional
    z = alpha * x @ w + (0 if b is None else b)
    f = {"identity": lambda z: z, "ssp": lambda z: F.softplus(z) - math.log(2), "silu": F.silu, "tanh": torch.tanh, "abs": torch.abs,
         "sigmoid": torch.sigmoid, "gelu": F.gelu}[act]
    return cst * f(z)


@pytest.fixture
def ops(monkeypatch):
    from matten_amd import _lib, ops

    names = {v: k for k, v in _lib.DENSE_ACT.items()}
    ops.products = []

    def run(a, b, bias=None, residual=None, act=0, alpha=1.0, cst=1.0, keep_z=False):
        ops.products.append((a.dtype, a.shape[0], a.shape[1], b.shape[1]))
        with torch.no_grad():
            y = _plain(a.double(), b.double(), None if bias is None else bias.double(), names[act], alpha, cst)
        return y.to(a.dtype), None

    monkeypatch.setattr(ops, "_floats", lambda *a, **k: None)
    monkeypatch.setattr(ops, "_dense_run", run)
    yield ops
    del ops.products


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ACTS)
def test_products_of_the_differentiable_backward(ops, act, dt):
    """Two for the identity, in its own type; with an activation one more, that of z, all three in fp32.  None for what is not wanted."""
    x, w, b = (torch.randn(*s).to(dt).requires_grad_(True) for s in ((6, 4), (4, 5), (5,)))
    g = torch.ones(6, 5, dtype=dt)
    z = [] if act == "identity" else [(torch.float32, 6, 4, 5)]
    t = dt if act == "identity" else torch.float32
    for wanted, products in (((x, w, b), [(t, 6, 5, 4), (t, 4, 6, 5)]), ((x,), [(t, 6, 5, 4)]), ((w,), [(t, 4, 6, 5)]), ((b,), [])):
        args = [p if any(p is q for q in wanted) else p.detach() for p in (x, w, b)]
        y = ops.dense(*args, act=act, alpha=0.5)
        ops.products.clear()
        got = torch.autograd.grad(y, wanted, g, create_graph=True)
        assert ops.products == z + products
        assert all(a.dtype == dt for a in got)


@pytest.mark.parametrize("act", ACTS)
def test_second_and_third_order(ops, act):
    torch.manual_seed(4)
    t32 = [torch.randn(*s) for s in ((6, 4), (4, 5), (5,), (6, 5))]

    def derivatives(f, args):
        x, w, b, g = [t.clone().requires_grad_(True) for t in args]
        one = torch.autograd.grad(f(x, w, b), [x, w, b], g, create_graph=True)
        two = torch.autograd.grad(sum((t * t).sum() for t in one), [x, w, b, g], create_graph=True, allow_unused=True)
        three = torch.autograd.grad(sum((t * t).sum() for t in two if t is not None), [x, w, b, g], allow_unused=True)
        return [*one, *two, *three]

    got = derivatives(lambda x, w, b: ops.dense(x, w, b, act=act, alpha=0.3, act_cst=1.4), t32)
    want = derivatives(lambda x, w, b: _plain(x, w, b, act, 0.3, 1.4), [t.double() for t in t32])
    for i, (a, e) in enumerate(zip(got, want)):
        assert (a is None) == (e is None)  # (the identity's bias)
        if a is None:
            continue
        # (three nested passes of a few dozen roundings each, sums of at most thirty)
        assert (a.double() - e).abs().max() <= (64, 512, 4096)[min(2, (i + 1) // 4)] * 2.0**-24 * e.abs().max() + 1e-30, i

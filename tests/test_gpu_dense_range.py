"""-m gpu: gradients of ops.dense in 16 bits over the whole range of the type: incoming gradients near the top of fp16 and among its
subnormals, constants that carry it out of range, activations that have saturated; at layers on both sides of 64 x 64, whose
backward passes are different kernels.

Tolerances as in test_gpu_dense.py (u = 2^-24, h half a step): z is kept to 2^-12 (bf16) or 2^-15 (fp16) of itself, and
dz / act_cst goes into the products in two pieces: h^2 of it, and for fp16 at least half the least step of the second piece, which
is 2^-25 of what it is multiplied with (2^11), twice that for the factor 1/2: 2^-35.  Large bf16 layers: rounded, h."""
import math

import pytest
import torch

from tests.test_gpu_dense import U, _act, _close, _sum_bound

pytestmark = pytest.mark.gpu
SIZES = [(256, 128, 128), (256, 64, 64), (256, 64, 65), (3, 200, 130), (700, 330, 150), (4100, 160, 640)]
BF, HALF = torch.bfloat16, torch.float16


def _check(x, w, b, dy, act, alpha, cst, bias=True, exact=False):
    from matten_amd import ops

    leaves = [t.requires_grad_(True) for t in ((x, w, b) if bias else (x, w))]
    grads = torch.autograd.grad(ops.dense(x, w, b, act=act, alpha=alpha, act_cst=cst, exact_grad=exact), leaves, dy)
    (m, k), n = x.shape, w.shape[1]
    h = torch.finfo(x.dtype).eps / 2
    X, W, G = x.detach().double(), w.detach().double(), dy.double()
    z = alpha * (X @ W) + b.detach().double()
    ez = alpha * _sum_bound(X, W, k) + 8 * U * (z.abs() + b.detach().double().abs())
    ez = ez + (2.0**-12 * z.abs() + 2.0**-24 if x.dtype == BF else 2.0**-15 * z.abs())
    _, da, dda = _act(act, z)
    dz = da * G
    edz = G.abs() * (dda * ez + 16 * U * (1 + z.abs()) * torch.maximum(da.abs(), dda)) + 4 * U * dz.abs()
    one = x.dtype == BF and min(m * k, k * n, m * n) >= 2**14 and max(k, n) > 64 and not exact
    edb = edz
    edz = edz + (h if one else h * h) * (dz.abs() + edz) + (2.0**-35 if x.dtype == HALF else 0)
    c = abs(alpha * cst)
    want = {"dx": alpha * cst * (dz @ W.t()), "dw": alpha * cst * (X.t() @ dz)}
    if bias:
        want["db"] = cst * dz.sum(0)
    for v in want.values():
        assert v.abs().max() < torch.finfo(x.dtype).max / 2
    bound = {"dx": c * (_sum_bound(dz.abs() + edz, W.t(), n) + edz @ W.t().abs() + 4 * U * (dz.abs() @ W.t().abs())),
             "dw": c * (_sum_bound(X.t(), dz.abs() + edz, m) + X.t().abs() @ edz + 4 * U * (X.t().abs() @ dz.abs())),
             "db": abs(cst) * (edb.sum(0) + (64 + m / 4) * U * dz.abs().sum(0))}
    for (name, v), g in zip(want.items(), grads):
        _close(name, g, v, bound[name])


def _inputs(m, k, n, dt, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + m + k + n)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    return r, r(m, k).to(dt), r(k, n).to(dt), r(n).to(dt)


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt", [BF, HALF])
def test_large_gradients(device, dt, m, k, n):
    """A few elements of dy near the top of fp16, where act_cst act' dy is beyond it; the gradients are not."""
    r, x, w, b = _inputs(m, k, n, dt, device)
    few = (torch.arange(n, device=device)[None] + 7 * torch.arange(m, device=device)[:, None]) % 41 == 0
    for act, cst, top in (("silu", 1.6791767923989418, 45000.0), ("gelu", 1.0, 65504.0), ("silu", -3.0, 65000.0), ("sigmoid", 30.0, 60000.0)):
        dy = torch.where(few, top * torch.sign(r(m, n)), 0.0).to(dt)
        _check((x / 64).to(dt), (w / 64).to(dt), b + 2 if act != "sigmoid" else b, dy, act, 4 / math.sqrt(max(m, k, n)), cst, bias=False)  # (db is beyond fp16)


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dt", [BF, HALF])
def test_small_gradients(device, dt, m, k, n):
    """dy, act_cst dy or act' dy among the subnormals of fp16; the gradients are not."""
    r, x, w, b = _inputs(m, k, n, dt, device, 1)
    one = r(m, n).to(dt)
    for cst in (2.0**-20, 2.0**-14):
        _check(x, w, b, one, "silu", 1 / math.sqrt(k), cst)
        _check((x / 256).to(dt), w, b, one, "gelu", 2.0**8, cst * 2.0**4)
    tiny = (r(m, n) * 2.0**-20).to(dt)
    _check(x, (w * 16).to(dt), b, tiny, "tanh", 2.0**4 / math.sqrt(k) / 256, 2.0**10)
    _check((x / 256).to(dt), (w * 32).to(dt), b - 12, one, "sigmoid", 1 / 8, 1.0)  # saturated: act' about 6e-6


@pytest.mark.parametrize("dt", [BF, HALF])
def test_both_sides_of_64(device, dt):
    """The same layer as 64 x 64 and, with a column of zeros, as 64 x 65: two kernels, one result to rounding."""
    from matten_amd import ops

    r, x, w, b = _inputs(500, 64, 64, dt, device, 2)
    for dy in (r(500, 64).to(dt), (r(500, 64) * 2.0**-19).to(dt), torch.where(r(500, 64) > 2.2, 60000.0, 0.0).to(dt)):
        got = []
        for pad in (0, 1):
            wide = lambda t: torch.nn.functional.pad(t, (0, pad))  # noqa: E731
            leaves = [t.clone().requires_grad_(True) for t in ((x / 64).to(dt), wide(w))]
            dx, dw = torch.autograd.grad(ops.dense(*leaves, wide(b), act="silu", alpha=0.125, act_cst=1.7), leaves, wide(dy))
            got.append((dx.double(), dw.double()[:, :64]))
        h, top = torch.finfo(dt).eps / 2, torch.finfo(dt).max
        X, W = (x / 64).to(dt).double(), w.double()
        dz = 1.7 * _act("silu", 0.125 * (X @ W) + b.double())[1] * dy.double()
        for a, e, exact in zip(*got, (0.125 * (dz @ W.t()), 0.125 * (X.t() @ dz))):
            # (60000 x 1.7 x 1.1 x 0.125 = 14000 is multiplied with weights of up to 4 and summed: some of dx is beyond fp16 itself)
            inside = exact.abs() < 0.99 * top
            beyond = exact.abs() > 1.01 * top
            assert torch.equal(a[beyond], math.inf * exact[beyond].sign()) and torch.equal(e[beyond], a[beyond])
            a, e = a[inside], e[inside]
            size = (a.abs().amax() + e.abs().amax()).item()
            assert math.isfinite(size) and size > 0
            # each is off by its own rounding (h, or half the least step), 2^-12 or 2^-15 of act'' z dy and little else: 4 h of the largest
            assert ((a - e).abs() <= 2 * h * (a.abs() + e.abs()) + 4 * h * size / 8 + torch.finfo(dt).smallest_normal * 2 * h).all()


@pytest.mark.parametrize("dt", [BF, HALF])
@pytest.mark.parametrize("act", ["identity", "ssp", "silu", "tanh", "abs", "sigmoid", "gelu"])
@pytest.mark.parametrize("m,k,n", [(300, 200, 150), (40, 64, 64), (1, 70, 9)])
def test_differentiable_backward(device, dt, act, m, k, n):
    """First-order gradients with create_graph=True: z, dz and the sums in fp32, one rounding at the end."""
    from matten_amd import ops

    r, x, w, b = _inputs(m, k, n, dt, device, 3)
    dy, alpha, cst = r(m, n).to(dt), 0.8 / math.sqrt(k), -1.6
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.dense(*leaves, act=act, alpha=alpha, act_cst=cst), leaves, dy, create_graph=True)
    assert all(g.requires_grad for g in (grads[:2] if act == "identity" else grads))
    X, W, B, G = (t.detach().double() for t in (x, w, b, dy))
    z = alpha * (X @ W) + B
    ez = alpha * _sum_bound(X, W, k) + 8 * U * (z.abs() + B.abs())
    _, da, dda = _act(act, z)
    dz = da * G
    edz = G.abs() * (dda * ez + 16 * U * (1 + z.abs())) + 4 * U * dz.abs() if act != "identity" else 0 * z
    if act == "abs":  # the sign of a z within its error of zero is either
        edz = torch.where(z.abs() <= ez, 2 * G.abs(), edz)
    c = abs(alpha * cst)
    _close("dx", grads[0], alpha * cst * (dz @ W.t()), c * (_sum_bound(dz.abs() + edz, W.t(), n) + edz @ W.t().abs() + 4 * U * (dz.abs() @ W.t().abs())))
    _close("dw", grads[1], alpha * cst * (X.t() @ dz), c * (_sum_bound(X.t(), dz.abs() + edz, m) + X.t().abs() @ edz + 4 * U * (X.t().abs() @ dz.abs())))
    _close("db", grads[2], cst * dz.sum(0), abs(cst) * (edz.sum(0) + (64 + m / 4) * U * dz.abs().sum(0)))


@pytest.mark.parametrize("create_graph", [False, True])
def test_pre_activations_beyond_fp16(device, create_graph):
    """z of 800 000 under silu: finite gradients whichever backward pass forms them."""
    from matten_amd import ops

    r, x, w, b = _inputs(20, 80, 70, HALF, device, 4)
    x, w = torch.full_like(x, 100.0), w.clone()
    w[:, 0] = 100.0
    dy = torch.full((20, 70), 2.0**-6, dtype=HALF, device=device)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    grads = torch.autograd.grad(ops.dense(*leaves, act="silu"), leaves, dy, create_graph=create_graph)
    X, W = x.detach().double(), w.detach().double()
    z = X @ W
    _, da, dda = _act("silu", z)
    dz = da * dy.double()
    # (act'' falls off as z exp(-z): at most 1/2, and below 2^-24 of act' beyond |z| = 25, however far z is off)
    edz = dy.double() * (torch.where(z.abs() > 25, 2.0**-24, dda * (2.0**-15 * z.abs() + _sum_bound(X, W, 80))) + 64 * U) + 2.0**-22 * dz.abs() + 2.0**-35
    _close("dx", grads[0], dz @ W.t(), _sum_bound(dz.abs() + edz, W.t(), 70) + edz @ W.t().abs())
    _close("dw", grads[1], X.t() @ dz, _sum_bound(X.t(), dz.abs() + edz, 20) + X.t().abs() @ edz)


@pytest.mark.parametrize("dt", [torch.float32, BF, HALF])
@pytest.mark.parametrize("m,k,n", [(256, 128, 128), (700, 330, 150), (4096, 512, 640), (64, 64, 64)])
def test_exact_grad(device, dt, m, k, n):
    """In bf16 the gradients of a large layer are then as exact as those of a small one (h^2 of dz in the bound instead of h); elsewhere
    nothing changes."""
    from matten_amd import ops

    r, x, w, b = _inputs(m, k, n, dt, device, 5)
    dy = r(m, n).to(dt)
    if dt != torch.float32:
        _check(x, w, b, dy, "silu", 1 / math.sqrt(k), 1.3, exact=True)

    def grads(**kw):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        return torch.autograd.grad(ops.dense(*leaves, act="silu", alpha=1 / math.sqrt(k), **kw), leaves, dy)

    same = [torch.equal(p, q) for p, q in zip(grads(), grads(exact_grad=True))]
    assert same == [False, False, True] if dt == BF and k > 64 else same == [True, True, True]


def test_one_row_of_2_to_22_columns(device):
    """A single row has no stride: its gradients exist at any width."""
    from matten_amd import ops

    n = (1 << 22) + 5
    r = torch.randn(n, 3, device=device)
    x, w = torch.randn(1, 3, device=device, requires_grad=True), r.t().requires_grad_(True)
    dy = torch.zeros(1, n, device=device)
    dy[0, ::4099] = torch.randn(dy[0, ::4099].numel(), device=device)  # (1024 terms that are not zero: 6 roundings each, 64 for the joins)
    dx, dw = torch.autograd.grad(ops.dense(x, w, act="tanh", alpha=0.3), [x, w], dy)
    X, W = x.detach().double(), w.detach().double()
    z = 0.3 * (X @ W)
    dz = (1 - torch.tanh(z) ** 2) * dy.double()
    edz = dy.double().abs() * (0.3 * _sum_bound(X, W, 3) + 16 * U * (1 + z.abs())) + 4 * U * dz.abs()
    size = 0.3 * dz.abs() @ W.t().abs()
    _close("dx", dx, 0.3 * dz @ W.t(), (6 * 1024 + 67) * U * size + 0.3 * edz @ W.t().abs())
    _close("dw", dw, 0.3 * X.t() @ dz, 0.3 * X.t().abs() @ edz + 73 * U * 0.3 * (X.t() @ dz).abs())

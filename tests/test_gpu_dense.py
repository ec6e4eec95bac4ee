"""-m gpu: ops.dense (tfc_dense, tfc_dense_bwd) against the formula in 64 bits.

Tolerances are bounds on the kernels' own roundings, u = 2^-24 and h half a step of the tensors' type.  A sum of k products in
fp32: fp32 operands lose at most 2^-24 |a b| of a product (the dropped pieces: three below 2^-24 each, 3 u), and every matrix
instruction rounds the running sum once, 6 for each 16 of k, with at most 1024 partial sums joined on top: (3 + 6 k / 16 + 64) u of
sum |a b| at worst.  That worst case grows with k like no random sum does, but it is proven; k stays below 5000 where it matters.
Behind the sum come alpha, bias, activation, constant and residual: under 16 roundings of the largest of them, the activation with a
few u of its own.  In the backward pass of a 16-bit call z is kept in fp16 (bf16: 2^-12, or 2^-24 absolute) or cut to 24 bits
(fp16: 2^-15), carried by act'', and dz is rounded to the type (h), or in two
pieces where x, the weight or y has less than 2^14 elements (h^2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["identity", "ssp", "silu", "tanh", "abs", "sigmoid", "gelu"]


def _act(name, z):
    """act, act', bound on |act''|, in 64 bits."""
    one = torch.ones_like(z)
    if name == "identity":
        return z, one, 0 * one
    if name == "abs":
        return z.abs(), torch.sign(z), 0 * one
    if name == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t, one
    if name == "gelu":
        cdf, phi = torch.special.ndtr(z), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * phi, one
    s = torch.sigmoid(z)
    if name == "sigmoid":
        return s, s * (1 - s), one / 8
    if name == "silu":
        return z * s, s * (1 + z * (1 - s)), one / 2
    return torch.logaddexp(z, torch.zeros_like(z)) - math.log(2), s, one / 4


def _sum_bound(a, b, k):
    return (67 + 6 * k / 16) * U * (a.abs() @ b.abs())


def _close(name, got, want, bound):
    h = torch.finfo(got.dtype).eps / 2
    tol = bound + h * (want.abs() + bound) + torch.finfo(got.dtype).smallest_normal * 2 * h
    err = (got.detach().double() - want).abs()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    assert (err <= tol).all(), f"{name}: {(err / tol).max().item():.3g} of the bound"


def _inputs(m, k, n, dt, seed, device, bias=True, residual=True, transposed=False):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    w = (r(n, k).to(dt).t() if transposed else r(k, n).to(dt))
    return r(m, k).to(dt), w, r(n).to(dt) if bias else None, r(m, n).to(dt) if residual else None, r(m, n).to(dt)


def _check(x, w, b, r, dy, act, alpha, cst=1.0):
    from matten_amd import ops

    leaves = {n: t for n, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None}
    for t in leaves.values():
        t.requires_grad_(True)
    y = ops.dense(x, w, b, r, act=act, alpha=alpha, act_cst=cst)
    assert y.dtype == x.dtype
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        assert torch.equal(ops.dense(x, w, b, r, act=act, alpha=alpha, act_cst=cst), y)
    (m, k), n = x.shape, w.shape[1]
    h = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    X, W, G = x.detach().double(), w.detach().double(), dy.double()
    z = alpha * (X @ W)
    ez = alpha * _sum_bound(X, W, k) + 4 * U * z.abs()
    if b is not None:
        z = z + b.detach().double()
        ez = ez + 2 * U * z.abs()
    a, da, dda = _act(act, z)
    # the activations are Lipschitz with constant < 1.2; their own roundings: 16 u of values up to |z| + 1
    ey = abs(cst) * (1.2 * ez + 16 * U * (z.abs() + 1))
    want = cst * a + (0 if r is None else r.detach().double())
    _close("y", y, want, ey + 4 * U * (want.abs() + (cst * a).abs()))
    dz = cst * da * G
    kept = {torch.float32: 0 * z, torch.bfloat16: 2.0**-12 * z.abs() + 2.0**-24, torch.float16: 2.0**-15 * z.abs()}[x.dtype]
    edz = abs(cst) * G.abs() * (dda * (ez + kept) + 16 * U * (1 + z.abs())) + 4 * U * dz.abs()
    if act != "identity":
        rounded = min(m * k, k * n, m * n) >= 2**14 and max(k, n) > 64
        edz = edz + (h if rounded else h * h) * (dz.abs() + edz)
        if x.dtype == torch.float16:  # (and half the least step)
            edz = edz + 2.0 ** (-25 if rounded else -36)
    if act == "abs":  # the sign of a z within its error of zero is either
        edz = torch.where(z.abs() <= ez, 2 * abs(cst) * G.abs(), edz)
    c = abs(alpha)
    _close("dx", grads["dx"], alpha * (dz @ W.t()), c * (_sum_bound(dz.abs() + edz, W.t(), n) + edz @ W.t().abs()) + 4 * U * c * (dz.abs() @ W.t().abs()))
    _close("dw", grads["dw"], alpha * (X.t() @ dz), c * (_sum_bound(X.t(), dz.abs() + edz, m) + X.t().abs() @ edz) + 4 * U * c * (X.t().abs() @ dz.abs()))
    if b is not None:  # summed before the rounding to the type: at most 2048 partial rows of at most m / 4 + 64
        _close("db", grads["db"], dz.sum(0), edz.sum(0) + (64 + m / 4) * U * dz.abs().sum(0))
    if r is not None:
        assert torch.equal(grads["dr"], dy)


SIZES = [(1, 1, 1), (1, 7, 5), (2, 64, 3), (3, 33, 65), (31, 32, 31), (64, 64, 64), (65, 63, 66), (100, 129, 130), (127, 16, 257), (128, 256, 128),
         (129, 255, 129), (300, 511, 200), (1, 4096, 1000), (17, 1000, 4096), (513, 40, 512), (4, 4100, 129), (2, 9000, 70), (1, 1, 300),
         (4, 640, 32), (3, 2047, 31)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_sizes(device, dt, m, k, n):
    for i, transposed in enumerate((False, True)):
        act = ACTS[(m + k + n + i) % len(ACTS)]
        _check(*_inputs(m, k, n, dt, m + 3 * k + 7 * n, device, transposed=transposed), act, 1 / math.sqrt(k), 1.5)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(device, dt, act):
    x, w, b, r, dy = _inputs(70, 50, 90, dt, 5, device)
    _check(x, w, b, r, dy, act, 0.2, 1.7)
    _check(x, w, b, None, dy, act, 3.0)  # large arguments
    _check(x, w, None, r, dy, act, 1e-3)  # small ones
    _check(x, w, None, None, dy, act, 0.1, -0.5)
    _check(x, w, None, None, dy, act, 2.0**-40)  # below and beyond the range of 16 bits
    _check(x, w, None, None, dy, act, 2.0**20, 2.0**-20)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("m,k,n", [(4000, 200, 1100), (5000, 64, 64), (40000, 33, 70), (2048, 700, 2048), (4100, 300, 4109), (70003, 61, 64)])
def test_large(device, dt, m, k, n):
    """Every tile, one and many parts of the contraction (the weight's gradient sums over m)."""
    _check(*_inputs(m, k, n, dt, m + n, device), "silu", 1 / math.sqrt(k))


@pytest.mark.parametrize("dt", TYPES[1:])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("m,k,n", [(4096, 1024, 4096), (4160, 832, 4416)])
def test_tiles_of_256(device, dt, transposed, m, k, n):
    """Sizes at which all three products take the kernel for large ones, whole tiles and edges."""
    _check(*_inputs(m, k, n, dt, m + k, device, transposed=transposed), "gelu", 1 / math.sqrt(k))


def test_layouts(device):
    """Row strides, odd starts, transposed and broadcast operands, more axes: the same bits as packed copies."""
    from matten_amd import ops

    for dt in TYPES:
        x, w, b, r, dy = _inputs(96, 72, 80, dt, 7, device)
        ref = ops.dense(x, w, b, r, act="silu")
        wide = torch.randn(96, 100, device=device).to(dt)
        wide[:, 11:83] = x
        wwide = torch.randn(72, 200, device=device).to(dt)
        wwide[:, 3:83] = w
        flat = torch.zeros(96 * 80 + 1, dtype=dt, device=device)
        rodd = flat[1:].view(96, 80).copy_(r)
        for args in [(wide[:, 11:83], w, b, r), (x, wwide[:, 3:83], b, r), (x, w, b, rodd), (x.t().contiguous().t(), w, b, r),
                     (x, w.t().contiguous().t(), b, r.t().contiguous().t()), (x, w, torch.stack([b, b], 1)[:, 0], r)]:
            assert torch.equal(ops.dense(*args, act="silu"), ref)
        assert torch.equal(ops.dense(x.view(4, 24, 72), w, b, r.view(4, 24, 80), act="silu"), ref.view(4, 24, 80))
        assert torch.equal(ops.dense(x[5], w, b, r[5], act="silu"), ops.dense(x[5:6], w, b, r[5:6], act="silu")[0])
        one = x[:1].expand(96, 72)
        assert torch.equal(ops.dense(one, w, b, r, act="silu"), ops.dense(one.contiguous(), w, b, r, act="silu"))
        # gradients through the views equal those of packed leaves
        def grads(x, w):
            leaves = [t.detach().requires_grad_(True) for t in (x, w)]
            return torch.autograd.grad(ops.dense(*leaves, b, act="silu"), leaves, dy)

        base = grads(x.clone(), w.clone())
        for a, c in [(wide[:, 11:83], w.t().contiguous().t()), (x.t().contiguous().t(), wwide[:, 3:83])]:
            (gx, gw), (ex, ew) = grads(a, c), base
            assert torch.equal(gx, ex)
            if c.stride(0) != 1:
                assert torch.equal(gw, ew)
            else:  # a transposed weight's gradient is the transposed product: other order of its small terms, then one rounding
                tol = 2 * _sum_bound(x.double().t(), 2 * dy.double().abs(), 96) + 4 * torch.finfo(dt).eps * ew.double().abs()
                assert ((gw.double() - ew.double()).abs() <= tol).all()
        xb = x[:1].detach().clone().requires_grad_(True)  # a broadcast input collects the sum of its rows
        y = ops.dense(xb.expand(96, 72), w, None, None)
        (g,) = torch.autograd.grad(y, xb, dy)
        want = (dy.double() @ w.double().t()).sum(0)
        h = torch.finfo(dt).eps / 2
        assert ((g[0].double() - want).abs() <= (96 + 2) * h * (dy.double().abs() @ w.double().abs().t()).sum(0)).all()


def test_a_few_rows(device):
    """One to four rows: views give the bits of packed operands, more rows the same to rounding; both sides of the longest contraction."""
    from matten_amd import ops

    for dt in TYPES:
        for m, k, n in [(1, 72, 80), (3, 1030, 33), (4, 2049, 65), (2, 20000, 40)]:
            x, w, b, r, _ = _inputs(m, k, n, dt, 17 + m, device)
            wide, wwide = torch.zeros(m, k + 28, dtype=dt, device=device), torch.zeros(k, n + 21, dtype=dt, device=device)
            wide[:, 11 : k + 11], wwide[:, 3 : n + 3] = x, w
            wt = w.t().contiguous()
            tall = torch.zeros(n, k + 9, dtype=dt, device=device)
            tall[:, 5 : k + 5] = wt
            args = dict(act="silu", alpha=1 / math.sqrt(k))
            ref, ref_t = ops.dense(x, w, b, r, **args), ops.dense(x, wt.t(), b, r, **args)
            assert torch.equal(ops.dense(wide[:, 11 : k + 11], wwide[:, 3 : n + 3], b, r, **args), ref)
            assert torch.equal(ops.dense(wide[:, 11 : k + 11], tall[:, 5 : k + 5].t(), b, r, **args), ref_t)
            assert torch.equal(ops.dense(x[:1].expand(m, k), w, b, r, **args), ops.dense(x[:1].repeat(m, 1), w, b, r, **args))
            more = ops.dense(torch.cat([x, x, x, x, x]), w, b, torch.cat([r, r, r, r, r]), **args)[:m]
            tol = 2 * (1.2 * _sum_bound(x.double(), w.double(), k) / math.sqrt(k) + 64 * U) + 2 * torch.finfo(dt).eps * more.double().abs()
            for y in (ref, ref_t):
                assert ((y.double() - more.double()).abs() <= tol + torch.finfo(dt).smallest_normal).all()


def test_empty(device):
    from matten_amd import ops

    x = torch.zeros(0, 5, device=device, requires_grad=True)
    w = torch.ones(5, 3, device=device, requires_grad=True)
    b = torch.ones(3, device=device, requires_grad=True)
    y = ops.dense(x, w, b, act="silu")
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros(0, 3, device=device))
    assert y.shape == (0, 3) and gx.shape == (0, 5) and not gw.any() and not gb.any()
    x, w = torch.zeros(4, 0, device=device, requires_grad=True), torch.zeros(0, 3, device=device, requires_grad=True)
    y = ops.dense(x, w, b, act="tanh")
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.ones(4, 3, device=device))
    t = math.tanh(1.0)
    assert gx.shape == (4, 0) and gw.shape == (0, 3)
    assert (y.double() - t).abs().max() <= 4 * U and (gb.double() - 4 * (1 - t * t)).abs().max() <= 64 * U
    assert ops.dense(torch.zeros(2, 3, 0, device=device), torch.zeros(0, 0, device=device)).shape == (2, 3, 0)


def test_values_that_are_not_finite(device):
    """A row of x that is not finite spoils its own row of the result only, and the edge of a tile brings nothing in."""
    from matten_amd import ops

    for dt in TYPES:
        x, w, b, r, _ = _inputs(70, 45, 67, dt, 9, device)
        ref = ops.dense(x, w, b, r)
        for bad in (float("nan"), float("inf")):
            z = x.clone()
            z[33, 44] = bad
            y = ops.dense(z, w, b, r)
            assert not torch.isfinite(y[33]).any()
            keep = [i for i in range(70) if i != 33]
            assert torch.equal(y[keep], ref[keep])
        buf = torch.full((80, 64), float("nan"), dtype=dt, device=device)  # what lies around the operands does not matter
        buf[:70, :45] = x
        assert torch.equal(ops.dense(buf[:70, :45], w, b, r), ref)
        big = torch.full((70, 45), torch.finfo(dt).max, dtype=dt, device=device)
        y = ops.dense(big, torch.zeros_like(w), b, r)
        assert torch.equal(y, ops.dense(torch.zeros_like(x), w, b, r))


def test_infinities_through_activations(device):
    """Sums of 16 bits that are infinite: limits where there are any."""
    from matten_amd import ops

    inf = float("inf")
    for dt in TYPES[1:]:
        x = torch.tensor([[inf], [-inf]], dtype=dt, device=device)
        w = torch.ones(1, 1, dtype=dt, device=device)
        for act, hi, lo in [("identity", inf, -inf), ("ssp", inf, -math.log(2)), ("tanh", 1, -1), ("abs", inf, inf), ("sigmoid", 1, 0),
                            ("silu", inf, None), ("gelu", inf, None)]:
            y = ops.dense(x, w, act=act)[:, 0].tolist()
            assert y[0] == hi and (lo is None or abs(y[1] - lo) <= 2.0**-8 or y[1] == lo), (act, y)


def test_smallest_and_largest_fp32(device):
    """Pieces below the least normal number may be lost: 2^-126 of what the other operand multiplies."""
    from matten_amd import ops

    x = torch.tensor([[2.0**-149], [1.5 * 2.0**-130], [2.0**-126], [1.2345678 * 2.0**-115], [2.0**-100 / 3], [3.4e38], [-3.4028234e38]], device=device)
    for scale in (1.0, 2.0**90):
        w = torch.full((1, 3), scale, device=device)
        if scale > 1:
            x = x[:5]
        y, want = ops.dense(x, w).double(), x.double() @ w.double()
        assert ((y - want).abs() <= 3 * U * want.abs() + 2.0**-126 * 3 * scale).all()


def test_offsets_beyond_32_bits(device):
    """2^32 elements and more on either side: the last rows equal the same rows alone, sums see them all."""
    from matten_amd import ops

    m, k, n = (1 << 26) + 77, 65, 66
    dt = torch.bfloat16
    x = torch.zeros(m, k, dtype=dt, device=device)
    x[-3000:], w, b, _, dy = _inputs(3000, k, n, dt, 21, device, residual=False)
    args = dict(act="silu", alpha=0.1)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = ops.dense(*leaves, **args)
    few = [t.detach().clone().requires_grad_(True) for t in (x[-3000:], w, b)]
    ref = ops.dense(*few, **args)
    assert torch.equal(y[-3000:], ref) and torch.equal(y[0], y[m // 2])
    g = torch.zeros(m, n, dtype=dt, device=device)
    g[-3000:] = dy
    got, want = torch.autograd.grad(y, leaves, g), torch.autograd.grad(ref, few, dy)
    del y, g
    assert torch.equal(got[0][-3000:], want[0]) and not got[0][: m - 3000].any()
    for p, q in zip(got[1:], want[1:]):  # (the same products, added up in other groups)
        assert (p.double() - q.double()).abs().max() <= 2.0**-7 * q.abs().max()


def test_inputs_that_depend_on_one_another(device):
    """One tensor as both operands, a bias computed from x: the differentiable backward counts every path once."""
    from matten_amd import ops

    x, w, _, _, dy = _inputs(8, 8, 8, torch.float32, 23, device, residual=False)

    def grads(f, create, args):
        args = [t.clone().requires_grad_(True) for t in args]
        return torch.autograd.grad(f(*args), args, dy.to(args[0].dtype), create_graph=create)

    def mine(x, w):
        return ops.dense(x, x, act="silu", alpha=0.3) + ops.dense(x, w, x.sum(0), act="tanh", alpha=0.3)

    def plain(x, w):
        return torch.nn.functional.silu(0.3 * x @ x) + torch.tanh(0.3 * x @ w + x.sum(0))

    want = grads(plain, False, [x.double(), w.double()])
    for create in (False, True):
        for a, e in zip(grads(mine, create, [x, w]), want):
            assert (a.double() - e).abs().max() <= 256 * U * e.abs().max()


def test_gradients_against_differences(device):
    """Differences of the forward (fp32, L = <dy, y>) along a direction in (x, w, b) against <gradient, direction>.  Allowed: what the
    same difference is off in 64 bits, and the forward's error bound over the step."""
    from matten_amd import ops

    x, w, b, _, dy = _inputs(20, 30, 25, torch.float32, 11, device, residual=False)
    vx, vw, vb, _, _ = _inputs(20, 30, 25, torch.float32, 12, device, residual=False)
    t, alpha = 2.0**-7, 0.18
    for act in ("ssp", "silu", "tanh", "sigmoid", "gelu"):
        leaves = [p.clone().requires_grad_(True) for p in (x, w, b)]
        grads = torch.autograd.grad(ops.dense(*leaves, act=act, alpha=alpha), leaves, dy)
        slope = sum((g.double() * v.double()).sum() for g, v in zip(grads, (vx, vw, vb)))
        ends = [(x + s * t * vx, w + s * t * vw, b + s * t * vb) for s in (1, -1)]
        diff = sum(s * (ops.dense(*e, act=act, alpha=alpha).double() * dy.double()).sum() for s, e in zip((1, -1), ends)) / (2 * t)

        def exact(x, w, b):
            z = alpha * (x.double() @ w.double()) + b.double()
            return _act(act, z), z

        f = [exact(*e) for e in ends]
        (_, da, _), z = exact(x, w, b)
        dz = da * dy.double()
        true = (dz * (alpha * (vx.double() @ w.double() + x.double() @ vw.double()) + vb.double())).sum()
        cut = ((f[0][0][0] - f[1][0][0]) * dy.double()).sum() / (2 * t) - true
        ey = 1.2 * alpha * _sum_bound(x.double(), w.double(), 30) * 1.1 + 24 * U * (z.abs() + 1)
        size = (dz.abs() * (alpha * (vx.abs().double() @ w.abs().double() + x.abs().double() @ vw.abs().double()) + vb.abs().double())).sum()
        assert (slope - diff).abs() <= cut.abs() + (ey * dy.abs().double()).sum() / t + 128 * U * size


@pytest.mark.parametrize("act", ["identity", "ssp", "silu", "tanh", "sigmoid", "gelu"])
def test_second_order(device, act):
    """Gradients of a function of the gradients against autograd in 64 bits, to 512 u of the largest element (two nested passes)."""
    from matten_amd import ops

    x, w, b, r, dy = _inputs(9, 12, 10, torch.float32, 13, device)

    def second(f, args):
        args = [a.clone().requires_grad_(True) for a in args]
        g = torch.autograd.grad(f(*args[:4]), args[:4], args[4], create_graph=True)
        return torch.autograd.grad(sum((t * t).sum() for t in g), [args[0], args[1], args[2], args[4]], allow_unused=True)

    F = torch.nn.functional
    torch_act = {"identity": lambda z: z, "ssp": lambda z: F.softplus(z) - math.log(2), "silu": F.silu, "tanh": torch.tanh,
                 "sigmoid": torch.sigmoid, "gelu": F.gelu}[act]
    got = second(lambda x, w, b, r: ops.dense(x, w, b, r, act=act, alpha=0.3, act_cst=1.4), [x, w, b, r, dy])
    want = second(lambda x, w, b, r: torch_act(0.3 * x @ w + b) * 1.4 + r, [t.double() for t in (x, w, b, r, dy)])
    for a, e in zip(got, want):
        assert (a is None) == (e is None)
        if e is not None:
            assert (a.double() - e).abs().max() <= 512 * U * e.abs().max() + 1e-300


def test_runs_agree_on_streams_and_in_graphs(device):
    from matten_amd import ops

    x, w, b, r, dy = _inputs(3000, 90, 70, torch.float32, 15, device)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]

    def step():
        y = ops.dense(*leaves, act="gelu", alpha=0.1)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    ref = step()
    assert all(torch.equal(p, q) for p, q in zip(step(), ref))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = step()
    other.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(step())
    for k in range(4):
        with torch.no_grad():
            x.mul_(0.9).add_(0.1 * k)
        want = step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):  # both at once: they share no scratch memory
            graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_refusals(device):
    from matten_amd import _lib, ops

    x, w = torch.zeros(3, 8, device=device), torch.zeros(8, 4, device=device)
    for args, kw, err in [((x.cpu(), w), {}, RuntimeError), ((x, w.cpu()), {}, RuntimeError), ((x.double(), w.double()), {}, TypeError),
                          ((x, w.half()), {}, TypeError), ((x, w.t()), {}, ValueError), ((x, w[0]), {}, ValueError),
                          ((x, w, torch.zeros(3, device=device)), {}, ValueError), ((x, w, torch.zeros(1, 4, device=device)), {}, ValueError),
                          ((x, w, None, torch.zeros(1, 4, device=device)), {}, ValueError),
                          ((x, w, None, torch.zeros(3, 4, device=device).half()), {}, TypeError), ((x, w), {"act": "relu6"}, ValueError),
                          ((x, w), {"alpha": float("nan")}, ValueError), ((x, w), {"act_cst": float("inf")}, ValueError)]:
        with pytest.raises(err):
            ops.dense(*args, **kw)
    L = _lib.lib()
    c = torch.zeros(3, 4, device=device)
    make = lambda **kw: _lib.DenseDesc(**{**dict(m=3, n=4, k=8, a=x.data_ptr(), lda=8, b=w.data_ptr(), ldb=4, c=c.data_ptr(), ldc=4, alpha=1.0,  # noqa: E731
                                                 act_cst=1.0, act=0, dtype=0, a_along_k=1, b_along_k=0), **kw})
    assert L.tfc_dense(make(), None, 0, None) == 0
    for bad in (dict(dtype=3), dict(act=7), dict(m=-1), dict(a=None), dict(c=None), dict(ldc=3)):
        assert L.tfc_dense(make(**bad), None, 0, None) == -1, bad
    assert L.tfc_dense(make(a_along_k=0, b_along_k=1), None, 0, None) == -2
    assert L.tfc_dense(make(m=64, n=64, k=1 << 20, ldc=64), None, 0, None) == -1 and b"workspace" in L.tfc_last_error()
    assert L.tfc_dense(None, None, 0, None) == -1
    with pytest.raises(_lib.TfcError, match="2\\^22"):
        ops.dense(torch.zeros(2, 1 << 22, device=device), torch.zeros(1 << 22, 1, device=device))
    g = torch.zeros(3, 4, device=device)
    bwd = lambda **kw: _lib.DenseBwdDesc(**{**dict(m=3, n=4, k=80, x=x.data_ptr(), ldx=0, w=w.data_ptr(), ldw=0, dy=g.data_ptr(),  # noqa: E731
                                                   db=c.data_ptr(), alpha=1.0, act_cst=1.0, act=2, dtype=0), **kw})
    ws = torch.zeros(1 << 16, device=device)
    assert L.tfc_dense_bwd(bwd(), ws.data_ptr(), ws.numel(), None) == -1 and b"needs z" in L.tfc_last_error()
    assert L.tfc_dense_bwd(bwd(z=g.data_ptr()), None, 0, None) == -1 and b"workspace" in L.tfc_last_error()
    for bad in (dict(dtype=9), dict(act=-1), dict(n=-1), dict(dy=None), dict(ldx=-1)):
        assert L.tfc_dense_bwd(bwd(z=g.data_ptr(), **bad), ws.data_ptr(), ws.numel(), None) == -1, bad
    assert L.tfc_dense_bwd(bwd(db=None), None, 0, None) == 0  # nothing asked for
    assert L.tfc_dense_keeps_z(64, 64, 2) == 0 and L.tfc_dense_keeps_z(65, 64, 2) == 1 and L.tfc_dense_keeps_z(65, 64, 0) == 0

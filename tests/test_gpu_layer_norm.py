"""-m gpu: ops.layer_norm (tfc_layer_norm_fwd/bwd) against the formulas in 64 bits.

Tolerances are bounds on the kernels' own roundings.  u = 2^-24 (fp32, half a step), h = half a step of the result's type.
A row is summed by at most 16 values in a register, 6 steps over a wave and 16 over a workgroup's waves: under 64 roundings with
the few of the formula, so  |mean error| <= 64 u mean|x|  and, relative to themselves, variance and 1 / deviation <= 64 u once
the error of the centred values is counted.  Column sums take at most 64 rows in a register and 64 in the joins."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _half(dt):
    return torch.finfo(dt).eps / 2


def _oracle(x, w, b, eps, dy):
    """y, dx, dw, db and bounds on what fp32 arithmetic may do to them, in 64 bits."""
    x, dy = x.double(), dy.double()
    d = x.shape[-1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    eh = 64 * U * (rstd * (x.abs().mean(-1, keepdim=True) + x.abs()) + h.abs() * (1 + rstd * x.abs().mean(-1, keepdim=True)))
    g = dy * w
    s, q = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - s - h * q)
    qa = (g * h).abs().mean(-1, keepdim=True)
    rel = 64 * U * (1 + rstd * x.abs().mean(-1, keepdim=True))  # of rstd, through the centred values
    edx = rstd * (128 * U * (g.abs() + g.abs().mean(-1, keepdim=True) + h.abs() * qa) + eh * q.abs()
                  + h.abs() * (g.abs() * eh).mean(-1, keepdim=True)) + rel * dx.abs()
    r = dict(y=h * w + b, dx=dx, dw=(dy * h).sum(0), db=dy.sum(0))
    e = dict(y=eh * w.abs() + 4 * U * ((h * w).abs() + b.abs()), dx=edx, dw=(dy.abs() * eh).sum(0) + 128 * U * (dy * h).abs().sum(0),
             db=128 * U * dy.abs().sum(0))
    return r, e


def _close(name, got, want, bound):
    h = _half(got.dtype)
    tiny = torch.finfo(got.dtype).smallest_normal * 2 * h  # half a step among the subnormals
    tol = bound + h * (want.abs() + bound) + tiny
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), name
    assert (err <= tol).all(), f"{name}: {(err / tol).max().item():.3g} of the bound"


def _inputs(rows, d, dt, seed, device, weight=True, bias=True):
    g = torch.Generator(device=device).manual_seed(seed)
    x = (torch.randn(rows, d, generator=g, device=device) * 2 + 0.5).to(dt)
    w = (torch.randn(d, generator=g, device=device) * 0.3 + 1).to(dt) if weight else None
    b = (torch.randn(d, generator=g, device=device) * 0.2).to(dt) if bias else None
    dy = torch.randn(rows, d, generator=g, device=device).to(dt)
    return x, w, b, dy


def _check(x, w, b, dy, eps=1e-5):
    from matten_amd import ops

    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = ops.layer_norm(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    want, bound = _oracle(x.detach(), w, b, eps, dy)
    for name, got in {"y": y.detach(), **grads}.items():
        _close(name, got, want[name], bound[name])
    with torch.no_grad():  # the call without gradients gives the same bits
        assert torch.equal(ops.layer_norm(x, w, b, eps), y)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("d", [1, 2, 7, 8, 31, 32, 33, 64, 65, 127, 129, 255, 257, 511, 513, 1000, 1024, 1025, 2049, 4096, 4097, 8193,
                               16384, 16385, 20001])
def test_widths(device, dt, d):
    for rows in (1, 2, 5, 37):
        _check(*_inputs(rows, d, dt, 1000 * rows + d, device))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,d", [(2048, 64), (4097, 33), (1000, 1001), (131, 1024), (70001, 16), (300, 5000)])
def test_many_rows(device, dt, rows, d):
    _check(*_inputs(rows, d, dt, rows + d, device))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_weight_or_bias(device, weight, bias):
    _check(*_inputs(19, 96, torch.float32, 3, device, weight, bias))


def test_layouts(device):
    """Views that start at odd elements, transposed and higher-dimensional inputs: the same bits as the packed copy."""
    from matten_amd import ops

    for dt in TYPES:
        x, w, b, dy = _inputs(24, 65, dt, 4, device)
        ref = ops.layer_norm(x, w, b)
        buf = torch.zeros(x.numel() + 3, dtype=dt, device=device)
        for shift in (1, 3):
            view = buf[shift : shift + x.numel()].view(24, 65).copy_(x)
            wv = torch.cat([w[:1], w])[1:]
            assert torch.equal(ops.layer_norm(view, wv, b), ref)
        assert torch.equal(ops.layer_norm(x.t().contiguous().t(), w, b), ref)
        assert torch.equal(ops.layer_norm(x.view(2, 3, 4, 65), w, b), ref.view(2, 3, 4, 65))
        a = x.t().contiguous().t().requires_grad_(True)  # gradients reach a leaf that is not packed
        c = x.clone().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(ops.layer_norm(a, w, b), a, dy)[0], torch.autograd.grad(ops.layer_norm(c, w, b), c, dy)[0])
        e = torch.ones((), dtype=dt, device=device)  # a broadcast incoming gradient
        assert torch.equal(torch.autograd.grad(ops.layer_norm(c, w, b), c, e.expand(24, 65))[0],
                           torch.autograd.grad(ops.layer_norm(c, w, b), c, torch.ones_like(c))[0])


def test_no_rows(device):
    from matten_amd import ops

    x = torch.empty(0, 8, device=device, requires_grad=True)
    w = torch.ones(8, device=device, requires_grad=True)
    b = torch.ones(8, device=device, requires_grad=True)
    y = ops.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.empty(0, 8, device=device))
    assert y.shape == gx.shape == (0, 8) and not gw.any() and not gb.any()


def test_values_that_are_not_finite_stay_in_their_row(device):
    from matten_amd import ops

    for d in (48, 700, 5000):
        x, w, b, _ = _inputs(9, d, torch.float32, 5, device)
        ref = ops.layer_norm(x, w, b)
        for bad in (float("nan"), float("inf"), -float("inf")):
            z = x.clone()
            z[4, 3] = bad
            y = ops.layer_norm(z, w, b)
            assert torch.isnan(y[4]).all()
            keep = [i for i in range(9) if i != 4]
            assert torch.equal(y[keep], ref[keep])
        c = torch.full((3, d), 7.0, device=device)  # rows without spread: exactly the bias
        assert torch.equal(ops.layer_norm(c, w, b), b.expand(3, d))


def test_gradient_against_differences(device):
    """(L(x + t v) - L(x - t v)) / 2t of the kernel's forward, L = <dy, y>, against <dx, v>.  Allowed: what the same
    difference is off in 64 bits, and 2^-24-sized errors of y divided by t."""
    from matten_amd import ops

    x, w, b, dy = _inputs(6, 300, torch.float32, 6, device)
    v = torch.randn(6, 300, device=device, generator=torch.Generator(device=device).manual_seed(1))
    t = 2.0**-6
    leaf = x.clone().requires_grad_(True)
    slope = (torch.autograd.grad(ops.layer_norm(leaf, w, b), leaf, dy)[0].double() * v.double()).sum()
    hi, lo = x + t * v, x - t * v
    diff = ((ops.layer_norm(hi, w, b).double() - ops.layer_norm(lo, w, b).double()) * dy.double()).sum() / (2 * t)
    (rh, eh), (rl, el), (r0, e0) = (_oracle(z, w, b, 1e-5, dy) for z in (hi, lo, x))
    exact = (r0["dx"] * v.double()).sum()
    cut = (((rh["y"] - rl["y"]) * dy.double()).sum() / (2 * t) - exact).abs()
    near = (((eh["y"] + el["y"] + 2 * U * r0["y"].abs()) * dy.abs().double()).sum() / (2 * t)) + (e0["dx"] * v.abs().double()).sum()
    near += (U * r0["dx"].abs() * v.abs().double()).sum()
    assert (slope - diff).abs() <= cut + near


def test_second_order(device):
    """Gradients of a function of the gradients, as training on forces takes them, against autograd in 64 bits.  The formula's
    terms nearly cancel in places, so the bound is 2^-24 x 512 (roundings of two nested passes) of the largest element."""
    from matten_amd import ops

    x, w, b, dy = _inputs(7, 40, torch.float32, 8, device)
    ws = [x, w, b, dy]

    def second(f, args):
        args = [a.clone().requires_grad_(True) for a in args]
        g = torch.autograd.grad(f(*args[:3]), args[:3], args[3], create_graph=True)
        return torch.autograd.grad(sum((t * t).sum() for t in g), [args[0], args[1], args[3]])

    got = second(lambda x, w, b: ops.layer_norm(x, w, b), ws)
    want = second(lambda x, w, b: torch.nn.functional.layer_norm(x, (40,), w, b, 1e-5), [a.double() for a in ws])
    for a, e in zip(got, want):
        assert (a.double() - e).abs().max() <= 512 * U * e.abs().max()


def test_one_tensor_as_weight_and_bias(device):
    """The differentiable backward counts every path once."""
    from matten_amd import ops

    g = torch.Generator(device=device).manual_seed(31)
    x, w, dy = (torch.randn(*s, generator=g, device=device) for s in ((7, 12), (12,), (7, 12)))

    def grads(f, create, args):
        args = [t.clone().requires_grad_(True) for t in args]
        return torch.autograd.grad(f(*args), args, dy.to(args[0].dtype), create_graph=create)

    want = grads(lambda x, w: torch.nn.functional.layer_norm(x, (12,), w, w * x[0]), False, [x.double(), w.double()])
    for create in (False, True):
        for a, e in zip(grads(lambda x, w: ops.layer_norm(x, w, w * x[0]), create, [x, w]), want):
            assert (a.double() - e).abs().max() <= 256 * 2.0**-24 * e.abs().max()
    want = grads(lambda x, w: torch.nn.functional.layer_norm(x, (12,), w, w), False, [x.double(), w.double()])
    for create in (False, True):
        for a, e in zip(grads(lambda x, w: ops.layer_norm(x, w, w), create, [x, w]), want):
            assert (a.double() - e).abs().max() <= 256 * 2.0**-24 * e.abs().max()


def test_offsets_beyond_32_bits(device):
    from matten_amd import ops

    for rows, d in [((1 << 26) + 77, 65), (131100, 32800)]:  # (a wave a row; rows walked again)
        g = torch.Generator(device=device).manual_seed(32)
        x = torch.zeros(rows, d, dtype=torch.bfloat16, device=device)
        x[-2000:] = torch.randn(2000, d, generator=g, device=device)
        w, b = (torch.randn(d, generator=g, device=device).bfloat16() for _ in range(2))
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        few = [t.detach().clone().requires_grad_(True) for t in (x[-2000:], w, b)]
        y, ref = ops.layer_norm(*leaves), ops.layer_norm(*few)
        assert torch.equal(y[-2000:], ref) and torch.equal(y[0], b) and torch.equal(y[rows // 2], b)
        dy = torch.zeros_like(x)
        dy[-2000:] = torch.randn(2000, d, generator=g, device=device)
        got, want = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(ref, few, dy[-2000:].clone())
        del y, dy
        assert torch.equal(got[0][-2000:], want[0]) and not got[0][: rows - 2000].any()
        for p, q in zip(got[1:], want[1:]):  # (the same terms, added up in other groups)
            assert (p.double() - q.double()).abs().max() <= 2.0**-7 * q.abs().max()


def test_runs_agree_on_streams_and_in_graphs(device):
    from matten_amd import ops

    x, w, b, dy = _inputs(3000, 200, torch.float32, 9, device)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)

    def step():
        y = ops.layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]

    ref = step()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = step()
        graph = torch.cuda.CUDAGraph()
    other.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, ref))
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.mul_(1.01).add_(0.1 * k)
        graph.replay()
        torch.cuda.synchronize()
        now = [t.clone() for t in out]
        assert all(torch.equal(a, c) for a, c in zip(now, step()))


def test_refusals(device):
    from matten_amd import _lib, ops

    x = torch.zeros(3, 8, device=device)
    for args, err in [((x.cpu(),), RuntimeError), ((x.double(),), TypeError), ((x, x.new_zeros(7)), ValueError),
                      ((x, x.new_zeros(8).bfloat16()), TypeError), ((x, x.new_zeros(8).cpu()), RuntimeError),
                      ((x, None, x.new_zeros(2, 4)), ValueError), ((x[:, :0],), ValueError), ((x.sum(),), ValueError),
                      ((x, None, None, -1.0), ValueError), ((x, None, None, float("nan")), ValueError)]:
        with pytest.raises(err):
            ops.layer_norm(*args)
    L = _lib.lib()
    p = x.data_ptr()
    assert L.tfc_layer_norm_fwd(p, None, None, 3, 8, 1e-5, 7, p, None, None, None) == -1
    assert L.tfc_layer_norm_fwd(p, None, None, 3, 0, 1e-5, 0, p, None, None, None) == -1
    assert L.tfc_layer_norm_fwd(None, None, None, 3, 8, 1e-5, 0, p, None, None, None) == -1
    assert L.tfc_layer_norm_bwd(p, p, None, p, p, 3, 8, 0, p, p, None, p, 1, None) == -1  # workspace too small
    assert b"workspace" in L.tfc_last_error()

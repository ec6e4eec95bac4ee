"""-m gpu: optim.AdamW (tfc_grad_sumsq, tfc_adamw_step) against the same step in torch operations on the host
(tests/adamw_reference.py).  Every operation of the kernel is an fp32 operation rounded once, as there, and the random bits are a
hash of integers: without a largest norm the results agree bit for bit.  With one, the two sums of squares (double) differ in
their order: the factor may differ by one step of fp32, 2^-23, which bounds the moments and moves a parameter by no more than
8 x 2^-24 of its step."""
import copy
import io
import math

import numpy as np
import pytest
import torch

from .adamw_reference import Reference, decode

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0**-24


def _tensors(sizes, dt, device, seed, scale=0.05):
    g = torch.Generator(device=device).manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(n, generator=g, device=device) * scale).to(dt)) for n in sizes]


def _grads(params, seed, spread=1.5):
    g = torch.Generator(device=params[0].device).manual_seed(seed)
    for i, p in enumerate(params):
        r = torch.randn(p.shape, generator=g, device=p.device)
        p.grad = (r * torch.exp(spread * torch.randn(p.shape, generator=g, device=p.device)) * 10.0 ** -(i % 4)).to(p.dtype)


def _bits(t):
    return t.detach().cpu().reshape(-1).view(torch.int32 if t.element_size() == 4 else torch.int16 if t.element_size() == 2 else torch.uint8)


def _same(opt, p, ref):
    st = opt.state[p]
    assert int(st["step"]) == ref.t
    assert torch.equal(_bits(p), _bits(ref.p))
    if ref.bits == 32:
        assert torch.equal(_bits(st["exp_avg"]), _bits(ref.m)) and torch.equal(_bits(st["exp_avg_sq"]), _bits(ref.v))
    else:
        for k, want in (("exp_avg", ref.mc), ("exp_avg_scale", ref.ms), ("exp_avg_sq_root", ref.vc), ("exp_avg_sq_root_scale", ref.vs)):
            assert torch.equal(_bits(st[k]), want), k


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", TYPES)
def test_steps(device, dt, bits):
    from matten_amd import optim

    params = _tensors([1, 3, 4, 255, 256, 257, 1000, 4095, 4096, 4097, 9001], dt, device, 1)
    refs = [Reference(p, i, bits, seed=5) for i, p in enumerate(params)]
    opt = optim.AdamW(params, state_bits=bits, seed=5)
    for k in range(5):
        _grads(params, 100 + k)
        if k == 3:
            for p in params:
                p.grad.zero_()
        opt.step()
        for p, r in zip(params, refs):
            r.step(p.grad)
            _same(opt, p, r)
    assert opt.grad_norm is None


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_groups(device, bits):
    """More tensors than one launch takes, empty ones among them, in groups with hyper-parameters of their own."""
    from matten_amd import optim

    params = _tensors([(37 * i) % 700 for i in range(131)], torch.float32, device, 2)
    half = _tensors([50, 5000], torch.bfloat16, device, 3)
    hp = [dict(lr=1e-2, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.0), dict(lr=1e-4, betas=(0.0, 0.5), eps=1e-3, weight_decay=0.3)]
    opt = optim.AdamW([{"params": params[:60], **hp[0]}, {"params": params[60:] + half, **hp[1]}], state_bits=bits)
    every = params + half
    refs = [Reference(p, i, bits, lr=h["lr"], betas=h["betas"], eps=h["eps"], wd=h["weight_decay"])
            for i, p in enumerate(every) for h in [hp[0] if i < 60 else hp[1]]]
    for k in range(3):
        _grads(every, 7 + k)
        skipped = {5, 77, 131} if k == 1 else set()
        for i in skipped:
            every[i].grad = None
        opt.step()
        for i, (p, r) in enumerate(zip(every, refs)):
            if i not in skipped:
                r.step(p.grad)
            if i not in skipped or r.t:
                _same(opt, p, r)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("limit", [1e-3, 1e9])
def test_largest_norm(device, dt, bits, limit):
    from matten_amd import optim

    params = _tensors([7, 16384, 16385, 70000], dt, device, 4) + _tensors([300], torch.float32, device, 5)
    before = [p.detach().double().clone() for p in params]
    opt = optim.AdamW(params, lr=1e-2, weight_decay=0.0, state_bits=bits, max_grad_norm=limit, seed=9)
    _grads(params, 21)
    kept = [p.grad.clone() for p in params]
    opt.step()
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in kept))
    assert abs(float(opt.grad_norm) - norm) <= 2 * U * norm  # rounded to fp32 once, sums in double
    clip = min(1.0, limit / (norm + 1e-6))
    for p, q, g in zip(params, before, kept):
        assert torch.equal(p.grad, g)  # left alone
        g = g.double() * clip
        st = opt.state[p]
        if bits == 32:  # factor, product with it, and product with 1 - beta, each rounded: m to 4 u, v to 8 u
            assert ((st["exp_avg"].double() - 0.1 * g).abs() <= 4 * U * (0.1 * g).abs() + 2.0**-140).all()
            assert ((st["exp_avg_sq"].double() - 0.001 * g * g).abs() <= 8 * U * 0.001 * g * g + 2.0**-140).all()
        # the first step has size lr g / (|g| + eps'): insensitive to the factor but for eps
        step = 1e-2 * (0.1 * g / (1 - 0.9)) / ((0.001 * g * g).sqrt() / math.sqrt(1 - 0.999) + 1e-8)
        h = torch.finfo(p.dtype).eps / 2
        # (sqrt(v) loses digits where v is below fp32's normal numbers, v < 2^-126: |g| < 2^-58)
        seen = g.abs() > 2.0**-50
        want = q - step
        assert ((p.detach().double() - want).abs() <= 16 * U * step.abs() + 2 * U * q.abs() + h * want.abs() + 2.0**-25)[seen].all()
    if dt == torch.float32:
        refs = [Reference(p, i, bits, seed=9, lr=1e-2, wd=0.0) for i, p in enumerate(before)]
        if limit > 1:  # nothing to scale: the factor is exactly 1
            for p, q, r, g in zip(params, before, refs, kept):
                r.p = q.float().cpu()
                r.step(g)
                _same(opt, p, r)


def test_views_of_flat_buffers_and_gradient_layouts(device):
    """Parameters and gradients as views that start at odd elements (the layout of a flat gradient buffer), a gradient that is not
    contiguous, 2-D tensors."""
    from matten_amd import optim
    from matten_amd.dp import FlatGradBucket

    for dt in TYPES:
        sizes = [5, 1023, 4096, 33]
        flat = torch.zeros(sum(sizes) + 1, dtype=dt, device=device)
        params, at = [], 1
        for n in sizes:
            params.append(torch.nn.Parameter(flat[at : at + n]))
            at += n
        with torch.no_grad():
            for p, q in zip(params, _tensors(sizes, dt, device, 6)):
                p.copy_(q)
        FlatGradBucket(params, alias=True)
        fresh = [p.detach().clone().requires_grad_(True) for p in params]
        _grads(fresh, 31)
        for p, q in zip(params, fresh):
            p.grad.copy_(q.grad)
        a, b = optim.AdamW(params, state_bits=8), optim.AdamW(fresh, state_bits=8)
        a.step(), b.step()
        assert all(torch.equal(p, q) for p, q in zip(params, fresh)) and float(flat[0]) == 0
    w = torch.nn.Parameter(torch.randn(40, 30, device=device))
    v = torch.nn.Parameter(w.detach().clone())
    g = torch.randn(30, 40, device=device)
    w.grad, v.grad = g.t(), g.t().contiguous()
    optim.AdamW([w]).step(), optim.AdamW([v]).step()
    assert torch.equal(w, v)


def test_8_bit_moments_are_kept_on_average(device):
    """With beta near 1 a step changes a moment by far less than a code: to the nearest it would stand still.  64 x 4096 equal
    blocks; the mean of what is kept must follow the exact decay.  Rounding is independent between elements with variance at most
    (spacing / 2)^2, spacing 2^-3 of the value: 5 deviations of the mean over N elements are 5 x 2^-4 / sqrt(N) of it."""
    from matten_amd import optim

    n = 64 * 4096
    p = torch.nn.Parameter(torch.zeros(n, device=device))
    opt = optim.AdamW([p], lr=0.0, betas=(0.99, 0.999), state_bits=8, seed=3)
    p.grad = torch.full((n,), 1.0, device=device)
    opt.step()
    p.grad.zero_()
    st = opt.state[p]
    value = lambda k: decode(st[k].view(torch.uint8).cpu(), st[k + "_scale"].view(torch.uint8).cpu(), n).mean().item()  # noqa: E731
    steps = 40
    for _ in range(steps):
        opt.step()
    # each step adds an independent rounding: deviations add in squares (a decay by the root of 0.999 keeps them)
    slack = 5 * 2.0**-4 * math.sqrt(steps + 1) / math.sqrt(n)
    m, r = 0.01 * 0.99**steps, math.sqrt(0.001 * 0.999**steps)
    assert abs(value("exp_avg") / m - 1) <= slack
    # sqrt(v) is what is rounded; v = r^2 decays by 0.999 and the root of a mean of squares is what the next step reads:
    # E[r] follows r sqrt(0.999) exactly, step by step
    assert abs(value("exp_avg_sq_root") / r - 1) <= slack


def test_8_bit_extremes(device):
    """Tiny second moments beside large ones stay above zero; values that are no numbers stay in their element; all-zero blocks."""
    from matten_amd import optim

    p = torch.nn.Parameter(torch.zeros(1024, device=device))
    opt = optim.AdamW([p], state_bits=8, weight_decay=0.0)
    g = torch.full((1024,), 1e-12, device=device)
    g[0], g[300], g[301], g[302] = 1.0, float("nan"), float("inf"), -float("inf")
    g[512:768] = 0
    p.grad = g
    opt.step()
    st = opt.state[p]
    codes = st["exp_avg_sq_root"].view(torch.uint8)
    assert (codes[:512] > 0).all() and (codes[512:768] == 0).all() and (codes[768:] > 0).all()
    assert (codes[300:303] == 127).all() and torch.isnan(st["exp_avg"].float()[300:303]).all()
    ok = torch.ones(1024, dtype=torch.bool, device=device)
    ok[300:303] = False
    assert torch.isfinite(p.detach()[ok]).all() and torch.isfinite(st["exp_avg"].float()[ok]).all()
    assert int(st["exp_avg_scale"].view(torch.uint8)[2]) == 1
    # |update| <= lr m^ / r^: bounded though r is 12 orders below its block's largest
    assert p.detach()[ok].abs().max() <= 1e-3 * 1.5
    p.grad = torch.zeros_like(p)
    for _ in range(3):
        opt.step()
    assert torch.isfinite(p.detach()[ok]).all()


def test_offsets_beyond_32_bits(device):
    from matten_amd import optim

    n = 2**31 + 4096 + 5
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=device), requires_grad=True)
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=device)
    tail = _tensors([4096 + 5], torch.bfloat16, device, 8)[0]
    _grads([tail], 41)
    with torch.no_grad():
        p[2**31 :] = tail
        p.grad[2**31 :] = tail.grad
    norm = tail.grad.double().norm()
    a = optim.AdamW([p], state_bits=8, max_grad_norm=1e9)
    b = optim.AdamW([tail], state_bits=8)
    a.step(), b.step()
    assert torch.equal(p[2**31 :], tail) and not p[: 2**31].any()
    assert abs(float(a.grad_norm) - float(norm)) <= 2 * U * float(norm)
    st, su = a.state[p], b.state[tail]
    for k in ("exp_avg_scale", "exp_avg_sq_root_scale"):
        assert torch.equal(st[k].view(torch.uint8)[2**31 // 256 :], su[k].view(torch.uint8))
    d = st["exp_avg"].view(torch.uint8)[2**31 :].int() - su["exp_avg"].view(torch.uint8).int()
    assert d.abs().max() <= 1 and d.any()  # other random bits for other elements


def test_state_dict(device):
    """Stopping and continuing from a saved state equals going on; the saved state is a copy; 8-bit state keeps its types through
    torch.save."""
    from matten_amd import optim

    for bits in (32, 8):
        params = _tensors([700, 31], torch.bfloat16, device, 9)
        opt = optim.AdamW(params, lr=1e-2, state_bits=bits, seed=4)
        for k in range(3):
            _grads(params, 50 + k)
            opt.step()
        buf = io.BytesIO()
        torch.save(opt.state_dict(), buf)
        buf.seek(0)
        saved = torch.load(buf, weights_only=True)
        again = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt2 = optim.AdamW(again, lr=5.0, state_bits=bits, seed=4)
        opt2.load_state_dict(saved)
        assert opt2.param_groups[0]["lr"] == 1e-2
        third = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt3 = copy.deepcopy(opt2)
        opt3.param_groups[0]["params"] = third
        opt3.state.update({q: opt3.state.pop(p) for p, q in zip(list(opt3.state), third)})
        for k in range(3, 5):
            _grads(params, 50 + k)
            for p, q, r in zip(params, again, third):
                q.grad, r.grad = p.grad.clone(), p.grad.clone()
            opt.step(), opt2.step(), opt3.step()
        for p, q, r in zip(params, again, third):
            assert torch.equal(p, q) and torch.equal(p, r)
            assert all(torch.equal(opt.state[p][k].view(torch.uint8) if bits == 8 and k != "step" else opt.state[p][k],
                                   opt2.state[q][k].view(torch.uint8) if bits == 8 and k != "step" else opt2.state[q][k]) for k in opt.state[p])
        with pytest.raises(ValueError):
            optim.AdamW(again, state_bits=40 - bits).load_state_dict(saved)
        with pytest.raises(ValueError):
            optim.AdamW(_tensors([1024, 31], torch.bfloat16, device, 9), state_bits=bits).load_state_dict(saved)


def test_state_and_storage_that_are_replaced(device):
    """State entries, parameters' storage and the set of gradients may change between steps: the next step works on what is there."""
    from matten_amd import optim

    params = _tensors([500, 40, 7], torch.float32, device, 14)
    refs = [Reference(p, i, 32) for i, p in enumerate(params)]
    opt = optim.AdamW(params)
    for k in range(6):
        _grads(params, 80 + k)
        if k == 1:
            opt.state[params[0]]["exp_avg"] = opt.state[params[0]]["exp_avg"].clone()
        if k == 2:
            params[1].data = params[1].detach().clone()
        if k == 3:
            opt.state[params[2]] = {n: t.clone() for n, t in opt.state[params[2]].items()}
        skip = {1} if k == 4 else set()
        for i in skip:
            params[i].grad = None
        junk = [torch.full((500,), 7.0, device=device) for _ in range(8)]  # whatever was let go is somebody else's now
        opt.step()
        for i, (p, r) in enumerate(zip(params, refs)):
            if i not in skip:
                r.step(p.grad)
            _same(opt, p, r)
        assert all(bool((j == 7.0).all()) for j in junk)
    swapped = _tensors([params[0].numel()], torch.float32, device, 18)[0]  # another parameter in its place
    old, opt.param_groups[0]["params"][0] = params[0].detach().clone(), swapped
    refs[0], kept = Reference(swapped, 0, 32), params[0]
    opt.param_groups[0]["lr"] = np.float32(1e-3)
    for r in refs:
        r.lr = float(np.float32(1e-3))
    params = [swapped, *params[1:]]
    _grads(params, 89)
    opt.step()
    for p, r in zip(params, refs):
        r.step(p.grad)
        _same(opt, p, r)
    assert torch.equal(kept, old)
    more = _tensors([60], torch.float32, device, 15)
    opt.add_param_group({"params": more, "lr": 0.5})
    refs.append(Reference(more[0], 3, 32, lr=0.5))
    _grads(params + more, 90)
    opt.step()
    for p, r in zip(params + more, refs):
        r.step(p.grad)
        _same(opt, p, r)


def test_state_dict_of_torch(device):
    from matten_amd import optim

    mine = _tensors([300, 33], torch.float32, device, 17)
    other = [torch.nn.Parameter(p.detach().clone()) for p in mine]
    theirs = torch.optim.AdamW(other, lr=3e-3, betas=(0.8, 0.99), weight_decay=0.1)
    for k in range(3):
        _grads(other, 110 + k)
        theirs.step()
    opt = optim.AdamW(mine)
    opt.load_state_dict(theirs.state_dict())
    assert all(int(opt.state[p]["step"]) == 3 for p in mine)
    with torch.no_grad():
        for p, q in zip(mine, other):
            p.copy_(q)
    for k in range(2):
        _grads(other, 120 + k)
        for p, q in zip(mine, other):
            p.grad = q.grad.clone()
        theirs.step(), opt.step()
    for p, q in zip(mine, other):  # the same 12 roundings of 2^-24, in another order, of values up to |p| + lr
        assert (p - q).abs().max() <= 2 * 2 * 12 * 2.0**-24 * (1 + q.abs().max())
    for key in ("amsgrad", "maximize"):
        with pytest.raises(ValueError, match="do not exist"):
            opt.load_state_dict(torch.optim.AdamW(other, **{key: True}).state_dict())
    assert opt.param_groups[0]["betas"] == (0.8, 0.99)


def test_state_storage_that_moves(device):
    """State whose storage is taken away and brought back between steps (`.data`, as programs do that keep it on the host
    meanwhile), and a state dict that went through a file that loads without executing anything."""
    import io

    from matten_amd import optim

    for bits in (32, 8):
        params = _tensors([300, 1000], torch.float32, device, 16)
        refs = [Reference(p, i, bits) for i, p in enumerate(params)]
        opt = optim.AdamW(params, lr=1e-3, state_bits=bits)
        for k in range(4):
            _grads(params, 100 + k)
            opt.step()
            for p, r in zip(params, refs):
                r.step(p.grad)
                _same(opt, p, r)
            if k < 2:
                host = [(t, t.data.cpu()) for st in opt.state.values() for t in st.values()]
                for t, h in host:
                    t.data = h
                with pytest.raises(ValueError, match="state entry"):  # (on the host still)
                    opt.step()
                junk = [torch.full((500,), 7.0, device=device) for _ in range(8)]
                for t, h in host:
                    t.data = h.to(device)
            elif k == 2:
                f = io.BytesIO()
                torch.save(opt.state_dict(), f)
                f.seek(0)
                opt = optim.AdamW(params, lr=1e-3, state_bits=bits)
                opt.load_state_dict(torch.load(f, weights_only=True))
        assert all(bool((j == 7.0).all()) for j in junk)


def test_schedulers_closures_and_versions(device):
    from matten_amd import optim

    (p,) = _tensors([100], torch.float32, device, 10)
    ref = Reference(p, 0, 32, lr=0.1)
    opt = optim.AdamW([p], lr=0.1)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    for k in range(3):
        version = p._version

        def closure():
            opt.zero_grad()
            loss = (p * p).sum()
            loss.backward()
            return loss

        loss = opt.step(closure)
        assert loss.requires_grad and p._version > version
        ref.lr = 0.1 * 0.5**k
        ref.step(2 * ref.p)
        _same(opt, p, ref)
        sched.step()
    y = (p.exp() * p).sum()  # a backward over a parameter that has been stepped meanwhile is refused
    _grads([p], 1)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_captured_step_and_lr_tensor(device):
    """A captured step replayed with new gradients, a new learning rate and eager work in between equals eager steps."""
    from matten_amd import optim

    for bits in (32, 8):
        mine = _tensors([900, 5000, 1], torch.float32, device, 11)
        other = [torch.nn.Parameter(p.detach().clone()) for p in mine]
        lr = [torch.tensor(1e-2, device=device) for _ in range(2)]
        a = optim.AdamW(mine, lr=lr[0], state_bits=bits, max_grad_norm=0.5)
        b = optim.AdamW(other, lr=lr[1], state_bits=bits, max_grad_norm=0.5)
        _grads(mine, 60)
        for p, q in zip(mine, other):
            q.grad = p.grad.clone()
        fresh = optim.AdamW(mine, state_bits=bits)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side), pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                fresh.step()
        a.step(), b.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.step()
        for k in range(4):
            _grads(other, 61 + k)
            with torch.no_grad():
                for p, q in zip(mine, other):
                    p.grad.copy_(q.grad)
                for t in lr:
                    t.mul_(0.7)
            graph.replay()
            b.step()
            torch.cuda.synchronize()
            assert torch.equal(a.grad_norm, b.grad_norm)
            for p, q in zip(mine, other):
                assert torch.equal(p, q) and int(a.state[p]["step"]) == int(b.state[q]["step"]) == k + 2


def test_on_another_stream(device):
    from matten_amd import optim

    mine, other = _tensors([300, 9999], torch.float32, device, 12), _tensors([300, 9999], torch.float32, device, 12)
    a, b = optim.AdamW(mine, max_grad_norm=1.0), optim.AdamW(other, max_grad_norm=1.0)
    _grads(mine, 70), _grads(other, 70)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.step(), a.step()
    s.synchronize()
    b.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(mine, other))


def test_refusals_on_the_device(device):
    from matten_amd import _lib, optim

    (p,) = _tensors([64], torch.float32, device, 13)
    q = torch.nn.Parameter(torch.zeros(8, 6, device=device).t())
    q.grad = torch.zeros_like(q)
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([q]).step()
    e = torch.nn.Parameter(torch.zeros(4, 3, device=device))
    e.grad = torch.sparse_coo_tensor(torch.tensor([[0]]), torch.ones(1, 3), (4, 3), device=device)
    with pytest.raises(RuntimeError, match="dense"):
        optim.AdamW([e]).step()
    square = torch.nn.Parameter(torch.zeros(8, 8, device=device))
    opt = optim.AdamW([square])
    square.grad = torch.ones_like(square)
    opt.step()
    square.data = square.data.t()  # the same address, another order
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    square.data = square.data.t()[:4]  # and fewer elements, with the gradient and the state of all
    before = square.detach().clone()
    with pytest.raises((ValueError, RuntimeError)):
        opt.step()
    assert torch.equal(square, before)
    flat = torch.zeros(100, device=device)
    shared = [torch.nn.Parameter(flat[:60]), torch.nn.Parameter(flat[59:])]
    for t in shared:
        t.grad = torch.ones_like(t)
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([{"params": shared[:1]}, {"params": shared[1:]}]).step()
    assert not flat.any()
    p.grad = torch.zeros_like(p)
    for k, bad in [("exp_avg", torch.zeros(63, device=device)), ("exp_avg", torch.zeros(64, device=device).half()), ("step", 3),
                   ("exp_avg_sq", torch.zeros(64)), ("exp_avg", torch.zeros(128, device=device)[::2]),
                   ("step", torch.zeros((), device=device)), ("more", torch.zeros(64, device=device))]:
        opt = optim.AdamW([p])
        opt.step()
        opt.state[p][k] = bad
        with pytest.raises(ValueError, match="state entr"):
            opt.step()
    with pytest.raises(RuntimeError, match="lr tensor"):
        optim.AdamW([p], lr=torch.tensor(1e-3)).step()
    L = _lib.lib()
    opt = optim.AdamW([p])
    opt.step()
    t = opt._tables[0][0]
    h = _lib.AdamwHyper(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    before = p.detach().clone()
    assert L.tfc_adamw_step(t.rows, 1, 0, 16, h, None, 0, None, None, 0, None) == -1
    assert L.tfc_adamw_step(t.rows, 1, 5, 32, h, None, 0, None, None, 0, None) == -1
    assert L.tfc_adamw_step(t.rows, 1, 0, 32, h, None, 0, None, None, 0, None) == -1 and b"workspace" in L.tfc_last_error()
    assert L.tfc_adamw_step(t.rows, 1, 0, 8, h, None, 0, None, None, 0, None) == -1  # no scales
    torch.cuda.synchronize()
    assert torch.equal(p, before)

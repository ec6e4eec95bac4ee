"""CPU: what optim.AdamW refuses before it touches a device, and the plain step the GPU tests compare with."""
from types import SimpleNamespace

import pytest
import torch

from .adamw_reference import Reference, decode, encode


def _param(*shape, dtype=torch.float32):
    return torch.nn.Parameter(torch.zeros(*shape, dtype=dtype))


@pytest.mark.parametrize("kw", [dict(state_bits=16), dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
                                dict(eps=-1e-8), dict(weight_decay=float("inf")), dict(max_grad_norm=0.0),
                                dict(max_grad_norm=float("nan")), dict(lr=torch.zeros(2)), dict(lr=torch.tensor(1e-3, dtype=torch.float64))])
def test_hyper_parameters_are_checked(kw):
    from matten_amd import optim

    with pytest.raises(ValueError):
        optim.AdamW([_param(3)], **kw)


def test_other_types_and_devices():
    from matten_amd import optim

    with pytest.raises(TypeError):
        optim.AdamW([_param(3, dtype=torch.float64)])
    p = _param(3)
    p.grad = torch.ones(3)
    opt = optim.AdamW([p])
    with pytest.raises(RuntimeError, match="ROCm device"):
        opt.step()
    assert torch.equal(p.detach(), torch.zeros(3))
    opt.param_groups[0]["betas"] = (0.9, 1.5)
    with pytest.raises(ValueError):
        opt.step()
    p.grad = None
    opt.param_groups[0]["betas"] = (0.9, 0.99)
    assert opt.step() is None  # nothing to do
    n = len(opt.param_groups)
    with pytest.raises(TypeError):
        opt.add_param_group({"params": [_param(2, dtype=torch.float64)]})
    assert len(opt.param_groups) == n


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group")
def test_a_parameter_twice():
    from matten_amd import optim

    p, q = _param(3), _param(2)
    with pytest.raises(ValueError, match="twice"):
        optim.AdamW([p, q, p])
    with pytest.raises(ValueError):
        optim.AdamW([{"params": [p]}, {"params": [q, p]}])


def test_plain_step_equals_torch_adamw():
    """The written-out step against torch.optim.AdamW in 64 bits: fp32 roundings only (12 operations, each 2^-24)."""
    g = torch.Generator().manual_seed(0)
    p = torch.randn(500, generator=g)
    q = torch.nn.Parameter(p.double())
    ref, opt = Reference(p, 0, 32, lr=0.05), torch.optim.AdamW([q], lr=0.05)
    for _ in range(6):
        grad = torch.randn(500, generator=g)
        q.grad = grad.double()
        ref.step(grad), opt.step()
    assert (ref.p.double() - q.detach()).abs().max() <= 6 * 12 * 2.0**-24 * (1 + q.detach().abs().max())


def test_codes_bracket_what_they_stand_for():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1000, generator=g) * torch.exp(4 * torch.randn(1000, generator=g))
    x[7] = 0
    lo, hi = encode(x, torch.zeros(1000, dtype=torch.int64), False), encode(x, torch.full((1000,), 65535), False)
    a, b = (decode(*c, 1000).abs() for c in (lo, hi))
    assert (a <= x.abs().double()).all() and (b >= x.abs().double() * (1 - 2.0**-20) * (a > 0)).all()
    top = x.abs().double()
    spacing = torch.maximum(a * 2.0**-3, torch.ldexp(torch.ones(4, dtype=torch.float64), lo[1].int() - 127 - 9).repeat_interleave(256)[:1000])
    assert (b - a <= spacing * (1 + 1e-12)).all() and (top - a < spacing).all()


def test_state_of_torch_adam():
    """Its weight decay is another update rule: a state dict that carries one is refused and leaves the optimizer as it was, at a later
    step too; one without is taken."""
    from matten_amd import optim

    p = _param(5)
    p.grad = torch.ones(5)
    for torch_opt, decay, fits in ((torch.optim.Adam, 0.1, False), (torch.optim.Adam, 0.0, True), (torch.optim.AdamW, 0.1, True)):
        source = torch_opt([p], lr=0.5, weight_decay=decay)
        source.step()
        q = _param(5)
        opt = optim.AdamW([q])
        if fits:
            opt.load_state_dict(source.state_dict())
            assert opt.param_groups[0]["lr"] == 0.5 and torch.equal(opt.state[q]["exp_avg"], source.state[p]["exp_avg"])
        else:
            with pytest.raises(ValueError, match="weight decay"):
                opt.load_state_dict(source.state_dict())
            assert opt.param_groups[0]["lr"] == 1e-3 and not opt.state
        if fits and decay == 0:
            opt.param_groups[0]["weight_decay"] = 0.1
            with pytest.raises(ValueError, match="weight decay"):
                opt.step()


def test_a_parameter_of_another_type_at_the_same_address():
    """Memory that one type of 16 bits gave back may be handed to the other: the table of the last step is not the parameter's any more."""
    from matten_amd import optim

    p = _param(7, dtype=torch.bfloat16)
    p.grad = torch.zeros_like(p)
    state = {"step": torch.zeros((), dtype=torch.int32), "exp_avg": torch.zeros(7), "exp_avg_sq": torch.zeros(7)}
    table = lambda: optim._Table({"lr": 1e-3}, [p], [state], [0], 32)  # noqa: E731
    old, point = table(), optim.AdamW._point_at_gradients
    old.device = SimpleNamespace(index=-1)  # (what a host tensor's get_device says)
    assert point([old]) == []
    at = p.data_ptr()
    p.grad = None
    p.data = p.data.view(torch.float16)
    p.grad = torch.zeros_like(p)
    assert p.data_ptr() == at and old.holds({p: state}) and point([old]) is None
    new = table()
    new.device = old.device
    assert point([new]) == [] and new.each[0].g == p.grad.data_ptr()

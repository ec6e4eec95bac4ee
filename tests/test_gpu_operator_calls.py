"""-m gpu: the dense product, the layer norm and the radial networks under a trace and under forward-mode differentiation."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls(device):
    from matten_amd import _lib, ops

    g = torch.Generator(device=device).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    w, v, b, s = r(130, 70), r(70, 33), r(70), r(130)
    return r, {
        "dense": lambda x: ops.dense(x, w, b, act="silu", alpha=0.1),
        "dense_row": lambda x: ops.dense(x[:1], w, b, act="silu", alpha=0.1),
        "layer_norm": lambda x: ops.layer_norm(x, s, s),
        "radial": lambda x: ops.radial_mlp_general(x, [w, v], 1.7, _lib.ACT["silu"]),
        "together": lambda x: ops.dense(ops.layer_norm(x, s), w, b, ops.dense(x, w)),
    }


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("name", ["dense", "dense_row", "layer_norm", "radial", "together"])
def test_a_trace_gives_the_bits_of_the_call(device, name):
    r, calls = _calls(device)
    f = calls[name]
    with torch.no_grad():
        traced = torch.jit.trace(f, (r(40, 130),), check_trace=False)
        for _ in range(3):
            x = r(40, 130)
            assert torch.equal(traced(x), f(x))


@pytest.mark.parametrize("name", ["dense", "layer_norm", "radial"])
def test_forward_mode_is_refused(device, name):
    r, calls = _calls(device)
    f = calls[name]
    x = r(40, 130)
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(f(x), f(x.clone()))


def test_accumulation_under_a_living_graph_is_seen(device):
    """What GraphedStep asks before it captures, in eager calls on a stream of their own."""
    from matten_amd.graphs import _Accumulated

    layer = torch.nn.Linear(5, 3).to(device)
    x = torch.randn(7, 5, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = layer(x).sum()
        kept.backward()
        for keep, want in ((True, 2), (False, 0)):
            if not keep:
                kept = None
            with _Accumulated() as a:
                layer(x).sum().backward()
            assert len(a.leaves) == 2 and len(a.held()) == want
        with _Accumulated() as a:
            layer.zero_grad()
            layer(x).sum().backward()
        assert not a.leaves
    torch.cuda.current_stream().wait_stream(side)


def test_adamw_steps_a_parameter_that_came_back_in_another_type(device):
    """bf16 memory handed to fp16 between two steps: the second step is one of fp16, with the moments of before."""
    from matten_amd import optim

    p = torch.nn.Parameter(torch.randn(300, device=device).to(torch.bfloat16))
    opt = optim.AdamW([p], lr=0.1)
    p.grad = torch.randn_like(p)
    opt.step()
    values = torch.randn(300, device=device).half()
    moments = {k: v.clone() for k, v in opt.state[p].items()}
    at, p.grad = p.data_ptr(), None
    p.data = p.data.view(torch.float16)
    p.data.copy_(values)
    assert p.data_ptr() == at
    p.grad = torch.randn_like(p)
    q = torch.nn.Parameter(values.clone())
    fresh = optim.AdamW([q], lr=0.1)
    fresh.state[q].update(moments)
    q.grad = p.grad.clone()
    opt.step(), fresh.step()
    assert p.dtype == torch.float16 and torch.equal(p, q) and all(torch.equal(opt.state[p][k], fresh.state[q][k]) for k in moments)

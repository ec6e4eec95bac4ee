"""CPU: a trace of the dense product and of the layer norm without gradients records them, and forward-mode differentiation through
them is refused.  The launches are replaced by stand-ins that write where the kernels do: through the result's address."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad


def _through_the_address(out, value):
    value = value.contiguous()
    C.memmove(out.data_ptr(), value.data_ptr(), 4 * value.numel())
    return out


@pytest.fixture
def ops(monkeypatch):
    from matten_amd import ops

    def dense_run(a, b, bias=None, residual=None, act=0, alpha=1.0, cst=1.0, keep_z=False):
        out = a.new_empty((a.shape[0], b.shape[1]))
        with torch.no_grad():
            a, b = a.detach().numpy(), b.detach().numpy()
            return _through_the_address(out, torch.from_numpy(alpha * (a @ b))), None

    def norm_run(x, w, b, eps, keep):
        v = x.detach().numpy()
        v = v - v.mean(-1, keepdims=True)
        v = v / (v.var(-1, keepdims=True) + eps) ** 0.5 * w.detach().numpy() + b.detach().numpy()
        return _through_the_address(torch.empty_like(x), torch.from_numpy(v)), torch.zeros(2, x.shape[0])

    monkeypatch.setattr(ops, "_floats", lambda *a, **k: None)
    monkeypatch.setattr(ops, "_dense_run", dense_run)
    monkeypatch.setattr(ops, "_layer_norm_run", norm_run)
    return ops


def _calls(ops):
    w, s, b = torch.randn(13, 70), torch.rand(13), torch.randn(13)
    return {"dense": lambda x: ops.dense(x, w, alpha=0.3), "layer_norm": lambda x: ops.layer_norm(x, s, b)}


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("name", ["dense", "layer_norm"])
@pytest.mark.parametrize("guard", [torch.no_grad, torch.enable_grad])
def test_traces_record_the_call(ops, name, guard):
    f = _calls(ops)[name]
    for shape in ((9, 13), (2, 3, 13), (13,)):
        with guard():
            traced = torch.jit.trace(f, (torch.randn(shape),), check_trace=False)
            for _ in range(3):
                x = torch.randn(shape)
                assert torch.equal(traced(x), f(x))


@pytest.mark.parametrize("name", ["dense", "layer_norm"])
def test_forward_mode_is_refused(ops, name):
    f = _calls(ops)[name]
    x = torch.randn(9, 13)
    with forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
        assert torch.equal(f(x), f(x.clone()))  # (no dual tensor: nothing to refuse)
    assert not f(x).requires_grad

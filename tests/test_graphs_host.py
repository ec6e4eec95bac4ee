"""CPU: GraphedStep refuses a function that accumulates into gradients whose earlier graph is alive, before it captures anything; with
the capture replaced by a plain call."""
import contextlib

import pytest
import torch


class _Stream:
    waits = 0

    def wait_stream(self, other):
        _Stream.waits += 1


@pytest.fixture
def step(monkeypatch):
    from matten_amd import graphs, ops

    captured = []

    @contextlib.contextmanager
    def capture(graph):
        captured.append(graph)
        yield

    monkeypatch.setattr(ops, "clear_caches", lambda: None)
    monkeypatch.setattr(ops, "snapshot_caches", lambda: None)
    for name, value in (("current_stream", _Stream), ("Stream", _Stream), ("stream", lambda s: contextlib.nullcontext()), ("synchronize", lambda: None),
                        ("CUDAGraph", object), ("graph", capture)):
        monkeypatch.setattr(torch.cuda, name, value)
    leaves = [torch.nn.Parameter(torch.ones(3)) for _ in range(4)]
    monkeypatch.setattr(graphs._Accumulated, "_leaves", staticmethod(lambda: [p for p in leaves if p.requires_grad]))

    def make(fn, **kw):
        del captured[:]
        try:
            return graphs.GraphedStep(fn, **kw)
        finally:
            make.captured = len(captured)

    return leaves, make


def _backward(leaves, keep=None):
    loss = sum((p * p).sum() for p in leaves)
    loss.backward()
    if keep is not None:
        keep[:] = [loss]
    return loss.detach()


def test_accumulation_under_a_living_graph_is_refused(step):
    leaves, make = step
    held = (leaves[0] ** 2).sum()  # a loss that someone kept
    _Stream.waits = 0
    with pytest.raises(RuntimeError, match="1 leaves .*shape \\(3,\\)"):
        make(lambda: _backward(leaves[:2]))
    assert make.captured == 0 and _Stream.waits == 2  # (the warm-up's stream for the caller's work before, and that for the warm-up)
    del held
    make(lambda: _backward(leaves[:2]))
    assert make.captured == 1


def test_a_graph_of_the_warm_up_counts(step):
    leaves, make = step
    keep = []
    with pytest.raises(RuntimeError, match="2 leaves"):
        make(lambda: _backward(leaves[:2], keep))
    assert make.captured == 0


@pytest.mark.parametrize("zero", ["none", "in place", "not"])
def test_what_is_sound_is_captured(step, zero):
    """None inside the function: whatever lives.  Zeroed or not: where no earlier graph does."""
    leaves, make = step
    held = (leaves[0] ** 2).sum() if zero == "none" else None  # noqa: F841

    def fn():
        for p in leaves:
            if zero == "none":
                p.grad = None
            elif zero == "in place" and p.grad is not None:
                p.grad.zero_()
        return _backward(leaves[:3])

    for warmup in (0, 1, 3):
        make(fn, warmup=warmup)
        assert make.captured == 1


def test_gradients_are_not_held():
    from matten_amd.graphs import _Accumulated

    p = torch.nn.Parameter(torch.ones(3))
    (p * p).sum().backward()

    class Leaves(_Accumulated):
        _leaves = staticmethod(lambda: [p])

    gone = []
    with Leaves() as a:
        import weakref

        ref = weakref.ref(p.grad)
        p.grad = None
        gone.append(ref() is None)
        (p * p).sum().backward()
    assert gone == [True] and a.leaves == [] and a.held() == []
    with Leaves() as a:
        (p * p).sum().backward()
    assert a.leaves == [p] and a.held() == []


def test_leaves_are_found():
    """On the host: every leaf that collects gradients is among the objects that are walked (they only have to be on a device besides)."""
    import gc

    from matten_amd.graphs import _Accumulated

    m = torch.nn.Sequential(torch.nn.Linear(3, 4), torch.nn.Linear(4, 2))
    x = torch.zeros(2, requires_grad=True)
    ids = {id(o) for o in gc.get_objects()}
    assert all(id(p) in ids for p in [*m.parameters(), x])
    assert not any(t is x for t in _Accumulated._leaves())  # (not on a device)

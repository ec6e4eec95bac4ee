"""CPU: sizes and refusals of the dense product's backward entry (addresses are made up: nothing may read them)."""
import pytest
import torch


def test_exact_dz_takes_the_workspace_of_two_pieces():
    from matten_amd import _lib

    L, here = _lib.lib(), 1 << 20

    def desc(dtype, exact, act=2):
        return _lib.DenseBwdDesc(m=4096, n=512, k=512, x=here, ldx=512, w=here, ldw=512, z=here, dy=here, dx=here, alpha=1.0, act_cst=1.0, act=act,
                                 dtype=dtype, exact_dz=exact)

    size = lambda *a: L.tfc_dense_bwd_desc_workspace_floats(desc(*a))  # noqa: E731
    rule = lambda dtype, act=2: L.tfc_dense_bwd_workspace_floats(4096, 512, 512, dtype, act)  # noqa: E731
    one = 4096 * 512 // 2  # floats of a piece of dz
    assert size(_lib.BF16, 0) == rule(_lib.BF16) and size(_lib.BF16, 1) == rule(_lib.BF16) + one
    assert size(_lib.F16, 0) == size(_lib.F16, 1) == rule(_lib.F16) == size(_lib.BF16, 1)
    for exact in (0, 1):
        assert size(_lib.F32, exact) == rule(_lib.F32) and size(_lib.BF16, exact, 0) == rule(_lib.BF16, 0)
    assert L.tfc_dense_bwd_desc_workspace_floats(None) == 0
    assert L.tfc_dense_bwd(desc(_lib.BF16, 1), here, rule(_lib.BF16), None) == -1 and b"workspace" in L.tfc_last_error()


def test_rows_of_2_to_22_are_refused_before_anything_is_launched():
    """At the entry (the refusal comes before the pass over dz: the addresses are no memory), and by ops.dense before the forward."""
    from matten_amd import _lib

    L, here, wide = _lib.lib(), 1 << 20, 1 << 22

    def bwd(**kw):
        d = _lib.DenseBwdDesc(**{**dict(m=8, n=wide, k=16, x=here, ldx=16, w=here, ldw=16, z=here, dy=here, dx=here, dw=here, db=here, alpha=1.0,
                                        act_cst=1.0, act=2, dtype=1, w_along_k=1), **kw})
        return L.tfc_dense_bwd(d, here, 1 << 40, None)

    for kw in ({}, dict(act=0), dict(dx=None), dict(dw=None, db=None), dict(n=80, k=wide, ldx=wide, ldw=80, w_along_k=0),
               dict(n=80, k=100, ldx=wide), dict(n=80, k=100, ldw=wide)):
        assert bwd(**kw) == -2 and b"2^22" in L.tfc_last_error(), kw


def test_dense_refuses_wide_results_with_gradients(monkeypatch):
    from matten_amd import ops

    calls = []
    monkeypatch.setattr(ops, "_floats", lambda *a, **k: None)
    monkeypatch.setattr(ops, "_dense_run", lambda a, b, *args, **kw: (calls.append(1), (a.new_zeros(()).expand(a.shape[0], b.shape[1]), None))[1])
    x, w = torch.zeros(3, 2), torch.zeros(()).expand(1 << 22, 2).t()
    for leaf in (x, w):
        leaf.requires_grad_(True)
        with pytest.raises(ValueError, match="2\\^22"):
            ops.dense(x, w)
        assert not calls
        assert ops.dense(x[:1], w).shape == (1, 1 << 22)
        with torch.no_grad():
            assert ops.dense(x, w).shape == (3, 1 << 22)
            with torch.autograd.forward_ad.dual_level():  # (an autograd.Function then, and still no gradient)
                assert ops.dense(x, w).shape == (3, 1 << 22)
        leaf.requires_grad_(False)
        calls.clear()

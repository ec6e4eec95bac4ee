"""CPU: what the dense product, the layer norm and the AdamW step refuse before anything is launched, through torch and at the C
entries (addresses are made up: nothing may read them)."""
import ctypes as C

import pytest
import torch

HERE = 1 << 20  # an address that is not null


def test_host_tensors_are_refused():
    from matten_amd import ops

    x, w = torch.zeros(3, 8), torch.zeros(8, 4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.dense(x, w)
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.layer_norm(x, torch.ones(8))


def test_dense_entries():
    from matten_amd import _lib

    L = _lib.lib()

    def desc(**kw):
        return _lib.DenseDesc(**{**dict(m=30, n=40, k=80, a=HERE, lda=80, b=HERE, ldb=40, c=HERE, ldc=40, alpha=1.0, act_cst=1.0, act=0, dtype=1,
                                        a_along_k=1, b_along_k=0), **kw})

    for bad in (dict(dtype=3), dict(dtype=-1), dict(act=7), dict(act=-1), dict(m=-1), dict(n=-1), dict(k=-1), dict(a=None), dict(b=None),
                dict(c=None), dict(ldc=39), dict(lda=-1), dict(ldb=-1), dict(residual=HERE, ldr=-1)):
        assert L.tfc_dense(desc(**bad), None, 0, None) == -1, bad
    assert L.tfc_dense(None, None, 0, None) == -1
    assert L.tfc_dense(desc(a_along_k=0, b_along_k=1), None, 0, None) == -2
    for ld in ("lda", "ldb"):
        assert L.tfc_dense(desc(**{ld: 1 << 22}), None, 0, None) == -2
    for empty in (dict(m=0), dict(n=0)):
        assert L.tfc_dense(desc(**empty), None, 0, None) == 0
        assert L.tfc_dense_workspace_floats(desc(**empty)) == 0
    long = desc(m=64, n=64, k=1 << 20, lda=1 << 20, ldb=64, ldc=64)
    need = L.tfc_dense_workspace_floats(long)
    assert need > 0 and need % (64 * 64) == 0
    for ws, n in ((None, need), (HERE, need - 1), (HERE, 0)):
        assert L.tfc_dense(long, ws, n, None) == -1 and b"workspace" in L.tfc_last_error()
    assert L.tfc_dense_workspace_floats(None) == 0 and L.tfc_dense_workspace_floats(desc(m=4, k=2048, dtype=0)) == 0
    assert [L.tfc_dense_z_bytes(7, 5, d) for d in range(4)] == [140, 70, 105, 0] and L.tfc_dense_z_bytes(0, 5, 0) == 0

    def back(**kw):
        return _lib.DenseBwdDesc(**{**dict(m=30, n=40, k=80, x=HERE, ldx=80, w=HERE, ldw=40, z=HERE, dy=HERE, dx=HERE, dw=HERE, db=HERE, alpha=1.0,
                                           act_cst=1.0, act=2, dtype=1), **kw})

    big = 1 << 30
    for bad in (dict(dtype=9), dict(act=-1), dict(m=-1), dict(n=-1), dict(k=-1), dict(ldx=-1), dict(ldw=-1), dict(dy=None), dict(x=None),
                dict(w=None), dict(z=None)):
        assert L.tfc_dense_bwd(back(**bad), HERE, big, None) == -1, bad
    assert L.tfc_dense_bwd(None, HERE, big, None) == -1
    need = L.tfc_dense_bwd_workspace_floats(30, 40, 80, 1, 2)
    assert need > 0
    for ws, n in ((None, need), (HERE, need - 1)):
        assert L.tfc_dense_bwd(back(), ws, n, None) == -1 and b"workspace" in L.tfc_last_error()
    assert L.tfc_dense_bwd(back(dx=None, dw=None, db=None), None, 0, None) == 0  # nothing asked for


def test_layer_norm_entries():
    from matten_amd import _lib

    L = _lib.lib()
    fwd = lambda x=HERE, rows=5, d=8, eps=1e-5, dt=0, y=HERE, mean=None, rstd=None: L.tfc_layer_norm_fwd(x, None, None, rows, d, eps, dt, y, mean, rstd, None)  # noqa: E731
    for bad in (dict(dt=3), dict(rows=-1), dict(d=0), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None), dict(mean=HERE)):
        assert fwd(**bad) == -1, bad
    assert fwd(rows=0) == 0
    bwd = lambda dy=HERE, x=HERE, mean=HERE, rows=5, d=8, dt=0, dx=HERE, dw=HERE, ws=HERE, n=1 << 30: L.tfc_layer_norm_bwd(  # noqa: E731
        dy, x, None, mean, HERE, rows, d, dt, dx, dw, None, ws, n, None)
    for bad in (dict(dt=-1), dict(rows=-1), dict(d=0), dict(dy=None), dict(x=None), dict(mean=None), dict(ws=None), dict(n=15)):
        assert bwd(**bad) == -1, bad
    assert bwd(dx=None, dw=None, ws=None, n=0) == 0


def test_adamw_entries():
    from matten_amd import _lib

    L = _lib.lib()
    h = _lib.AdamwHyper(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)

    def step(n=1, dtype=0, bits=32, hyper=h, partials=None, n_partials=0, ws=HERE, ws_bytes=1 << 20, **kw):
        t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(**{**dict(p=HERE, g=HERE, m=HERE, v=HERE, m_scale=HERE, v_scale=HERE, step=HERE, n=100), **kw}))
        return L.tfc_adamw_step(t, n, dtype, bits, C.byref(hyper) if hyper else None, partials, n_partials, None, ws, ws_bytes, None)

    for bad in (dict(n=-1), dict(dtype=3), dict(bits=16), dict(hyper=None), dict(n_partials=3), dict(n_partials=-1), dict(ws=None), dict(ws_bytes=8),
                dict(p=None), dict(g=None), dict(m=None), dict(v=None), dict(step=None), dict(bits=8, m_scale=None), dict(bits=8, v_scale=None),
                dict(bits=8, m=HERE + 2)):
        assert step(**bad) == -1, bad
    assert step(n=0) == 0
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(g=HERE, n=100))
    assert L.tfc_grad_sumsq_partials(t, 1) == 1 and L.tfc_grad_sumsq(t, 1, 0, None, None) == -1 and L.tfc_grad_sumsq(t, 1, 7, HERE, None) == -1
    assert L.tfc_grad_sumsq_partials(None, 1) == 0

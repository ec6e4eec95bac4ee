"""CPU: sizes and refusals of the dense product's backward entry (addresses are made up: nothing may read them)."""


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

"""What the operators on the text side take and refuse at the edges of their documented limits, on the CPU: their C entry points
with no rows, which check everything else and launch nothing."""


def test_strides_of_attention_over_packed_rows(pkg):
    """Rows lie less than 2^22 elements apart (24-bit and 32-bit offsets inside a tile); heads up to 2^40."""
    lib, arg = pkg._lib.load(), pkg._lib.WANMI_ERR_ARG

    def cross(ss=256, hs=64, k_hs=64):
        return lib.wanmi_packed_cross_attention(16, ss, hs, 16, ss, k_hs, 16, ss, k_hs, 16, 16, 2, 0, 4, 4, 4, 64, 0.5, 16, 256, None, 1, None)

    def bias(ss=256, hs=64):
        import ctypes

        starts = (ctypes.c_int * 4)(0, 1, 2, 5)
        return lib.wanmi_relative_bias_attention(16, ss, hs, 16, ss, hs, 16, ss, hs, 16, 2, 0, 4, 64, 1.0, 16, 0, starts, 4, 1, 16, 256, 1, None)

    for fn in (cross, bias):
        for kw in (dict(), dict(hs=1 << 22), dict(hs=75600 * 128), dict(hs=(1 << 40) - 8), dict(ss=(1 << 22) - 8)):
            assert fn(**kw) == 0, (fn.__name__, kw)
        for kw in (dict(ss=1 << 22), dict(hs=1 << 40), dict(hs=(1 << 22) + 4), dict(hs=-64), dict(ss=-256)):
            assert fn(**kw) == arg, (fn.__name__, kw)
    assert cross(k_hs=1 << 23) == 0 and cross(k_hs=1 << 40) == arg

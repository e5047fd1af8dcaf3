"""Limits of the serving operators, on the host: no GPU, nothing is launched.  Pointers are numbers that no launch sees."""


def _gemv(L, **changes):
    a = L.GemmArgs(kind=L.KIND_F16_W4G128, epilogue=L.EPI_LINEAR, m=3, n=40, k=256, a=256, lda=256, b=512, ldb=128, row_scale=1.0, alpha=1.0,
                   out=1024, ld_out=40, out_type=L.OUT_F16, b_group_scales=2048)
    for name, value in changes.items():
        setattr(a, name, value)
    return L.lib.pk100_gemv_w4g128(None, a)


def test_gemv_refuses_more_columns_than_it_counts(pk):
    # columns are numbered in whole tiles of 128: the last number of 2^31 - 1 columns does not fit 32 bits
    L = pk.lib
    for n in ((1 << 30) + 1, (1 << 31) - 100, (1 << 31) - 1):
        assert _gemv(L, m=1, n=n) == _gemv(L, m=1, n=n, k=16512) == L.ERR_LIMIT

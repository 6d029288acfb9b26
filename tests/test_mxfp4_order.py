"""MXFP4 products whose rows come in parts: order_rows gives every part the order of sums of the whole."""
import ctypes

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


def test_order_rows_is_checked():
    import omnivideo._hip as H
    L = H.lib()
    buf = (ctypes.c_ubyte * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64
    assert L.ovd_gemm_mxfp4_as_rows(p, p, p, p, None, p, 8, None, 1, 8, 32, 0, -1, None) != 0
    assert b"order_rows" in L.ovd_last_error()
    assert L.ovd_gemm_mxfp4_as_rows(p, p, p, p, None, p, 8, None, 0, 8, 32, 0, 5, None) == 0          # no rows: nothing to do


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(8000, 512, 2592), (3200, 1536, 4128)])
def test_parts_of_a_product_have_its_bits(M, N, K):
    """large terms that cancel 8 k-groups apart: the two orders of sums differ in most outputs"""
    import omnivideo._hip as H
    from omnivideo.modules import MXFP4Matrix, mxfp4_quantize
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) / K ** 0.5
    w[:, :32] *= 2.0 ** 14
    x[:, 2048:2080], w[:, 2048:2080] = x[:, :32], -w[:, :32]
    x, w = x.cuda(), mxfp4_quantize(w.cuda())
    bias, gate = torch.randn(N, generator=g).to(BF16).cuda(), torch.randn(N, generator=g).cuda()
    resid = torch.randn(M, N, generator=g).cuda()

    def product(a, b, epilogue, order_rows):
        m = mxfp4_quantize(x[a:b])
        if epilogue == H.EPI_MXFP4_GELU:
            return H.gemm_mxfp4_gelu(m, w, MXFP4Matrix.empty(b - a, N, "cuda"), bias, order_rows=order_rows).dequantize(F32)
        out = resid[a:b].clone() if epilogue == H.EPI_RESID else \
            torch.empty(b - a, N, device="cuda", dtype=BF16 if epilogue in (H.EPI_BF16, H.EPI_BF16_GELU) else F32)
        return H.gemm_mxfp4(m, w, out, bias, epilogue, gate if epilogue == H.EPI_RESID else None, order_rows=order_rows)

    for epilogue in (H.EPI_BF16, H.EPI_BF16_GELU, H.EPI_F32, H.EPI_RESID, H.EPI_MXFP4_GELU):
        whole = product(0, M, epilogue, 0)
        assert torch.equal(product(0, M, epilogue, M), whole)
        for a, b in ((0, 1), (5, 38), (31, 286), (1000, 1600), (0, M - 1)):
            assert torch.equal(product(a, b, epilogue, M), whole[a:b]), (epilogue, a, b)
        small = product(1000, 1033, epilogue, 0)             # the other order, also for many rows
        if epilogue in (H.EPI_F32, H.EPI_BF16):              # (four bits hide most of the difference)
            assert not torch.equal(small, whole[1000:1033])
        assert torch.equal(product(0, M, epilogue, 33)[1000:1033], small)

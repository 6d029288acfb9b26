"""MXFP4: layout of the operand buffers and refusals (no GPU needed)."""
import ctypes
import os

import pytest
import torch

import omnivideo._hip as H
from omnivideo.modules import MXFP4Matrix, mxfp4_linear, mxfp4_quantize

U8 = torch.uint8


def test_from_ocp_places_codes_and_scales_in_lane_order():
    rows, cols = 70, 544
    codes = torch.arange(rows * cols // 2).reshape(rows, cols // 2).remainder(251).to(U8)
    scales = torch.arange(rows * cols // 32).reshape(rows, cols // 32).remainder(241).to(U8)
    m = MXFP4Matrix.from_ocp(codes, scales)
    assert m.shape == (rows, cols)
    assert (m.data.numel(), m.scale.numel()) == H.mxfp4_bytes(rows, cols)
    kts = 4 * -(-cols // 256)
    data = m.data.view(-1, kts, 64, 16)
    scale = m.scale.view(-1, kts // 4, 64, 4)
    for r in (0, 31, 32, 69):
        for blk in range(cols // 32):
            kt, h = blk // 2, blk % 2
            lane = 32 * h + r % 32
            assert torch.equal(data[r // 32, kt, lane], codes[r, blk * 16:blk * 16 + 16])
            assert scale[r // 32, kt // 4, lane, kt % 4] == scales[r, blk]
    assert int(data[:, 9:].sum()) == 0                 # k past the row: zeros
    c, s = m.to_ocp()
    assert torch.equal(c, codes) and torch.equal(s, scales)


def test_sizes():
    assert H.mxfp4_bytes(1, 32) == (4096, 256)
    assert H.mxfp4_bytes(33, 257 * 32) == (2 * 33 * 4096, 2 * 33 * 256)
    assert H.mxfp4_bytes(0, 64) == (0, 0)
    L = H.lib()
    for rows, cols in ((1, 32), (31, 256), (32, 288), (33, 13824), (40560, 8960)):
        assert H.mxfp4_bytes(rows, cols) == (L.ovd_mxfp4_data_bytes(rows, cols), L.ovd_mxfp4_scale_bytes(rows, cols))
    for bad in ((1, 0), (1, 48), (-1, 32)):
        with pytest.raises(ValueError):
            H.mxfp4_bytes(*bad)


def test_from_ocp_refuses():
    ok = torch.zeros(4, 32, dtype=U8), torch.zeros(4, 2, dtype=U8)
    MXFP4Matrix.from_ocp(*ok)
    for codes, scales in ((ok[0], ok[1][:3]), (ok[0][:, :24], ok[1]), (ok[0], torch.zeros(4, 1, dtype=U8)),
                          (torch.zeros(0, 32, dtype=U8), torch.zeros(0, 2, dtype=U8))):
        with pytest.raises(ValueError):
            MXFP4Matrix.from_ocp(codes, scales)
    for codes, scales in ((ok[0].int(), ok[1]), (ok[0], ok[1].float()), (ok[0][0], ok[1][0])):
        with pytest.raises(TypeError):
            MXFP4Matrix.from_ocp(codes, scales)


def test_python_entries_refuse():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = MXFP4Matrix.from_ocp(torch.zeros(8, 32, dtype=U8), torch.zeros(8, 2, dtype=U8))
    with pytest.raises(ValueError, match="CPU"):
        mxfp4_quantize(x)
    with pytest.raises(TypeError):
        mxfp4_quantize(x.half())
    with pytest.raises(ValueError, match="multiple of 32"):
        mxfp4_quantize(x[:, :48])
    with pytest.raises(NotImplementedError, match="inference"):
        mxfp4_quantize(torch.zeros(4, 64, requires_grad=True))
    with pytest.raises(TypeError, match="MXFP4Matrix"):
        mxfp4_linear(x, x)
    with pytest.raises(ValueError, match="CPU"):
        w.dequantize()
    a = MXFP4Matrix.from_ocp(torch.zeros(4, 32, dtype=U8), torch.zeros(4, 2, dtype=U8))
    with pytest.raises(ValueError, match="CPU"):
        mxfp4_linear(a, w)
    with pytest.raises(ValueError, match="shape mismatch"):
        mxfp4_linear(MXFP4Matrix.from_ocp(torch.zeros(4, 48, dtype=U8), torch.zeros(4, 3, dtype=U8)), w)
    with pytest.raises(TypeError, match="gelu"):
        mxfp4_linear(a, w, gelu=True, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="residual"):
        mxfp4_linear(a, w, gelu=True, residual=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="gate"):
        mxfp4_linear(a, w, gate=torch.ones(8))
    with pytest.raises(ValueError, match="quantize_output"):
        mxfp4_linear(a, w, quantize_output=True)
    with pytest.raises(TypeError, match="MXFP4Matrix"):
        mxfp4_linear(a, w, gelu=True, quantize_output=True, out=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="no blocks"):
        mxfp4_linear(a, w, gelu=True, quantize_output=True)
    with pytest.raises(ValueError, match="shape"):
        mxfp4_linear(a, w, out=torch.zeros(4, 9))
    with pytest.raises(ValueError, match="length"):
        mxfp4_linear(a, w, bias=torch.zeros(7, dtype=torch.bfloat16))
    for buf in (w.buf[:-1], w.buf.view(torch.int8), w.buf.view(2, -1)):
        with pytest.raises(ValueError, match="does not hold"):
            MXFP4Matrix(8, 64, buf)
    assert MXFP4Matrix(8, 64, w.buf).to_ocp()[0].shape == (8, 32)


def test_c_entries_refuse_before_any_launch():
    L = H.lib()
    buf = (ctypes.c_ubyte * 4096)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def refused(fn, *args, why):
        assert getattr(L, fn)(*args) != 0 and why in L.ovd_last_error(), (fn, L.ovd_last_error())

    refused("ovd_mxfp4_quant", None, 0, 32, p, p, 1, 32, None, why=b"null")
    refused("ovd_mxfp4_quant", p, 0, 48, p, p, 1, 48, None, why=b"multiple of 32")
    refused("ovd_mxfp4_quant", p, 0, 33, p, p, 2, 32, None, why=b"alignment")
    refused("ovd_mxfp4_quant", p + 2, 0, 32, p, p, 1, 32, None, why=b"alignment")
    refused("ovd_mxfp4_quant", p, 0, 32, p, p, -1, 32, None, why=b"M=-1")
    refused("ovd_mxfp4_dequant", p, p, p, 0, 16, 1, 32, None, why=b"alignment")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 8, None, 1, 6, 32, 0, None, why=b"not supported")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 8, None, 1, 8, 40, 0, None, why=b"not supported")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 8, None, 1, 8, 32, 5, None, why=b"epilogue")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 8, p, 1, 8, 32, 4, None, why=b"MXFP4 output")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 32, None, 1, 32, 32, 4, None, why=b"MXFP4 output")
    refused("ovd_gemm_mxfp4", p, p, p + 16, p, None, p, 32, p, 1, 32, 32, 4, None, why=b"one of the operands")
    refused("ovd_linear_mxfp4", p, 0, 32, p, p, None, p, 32, p, None, 0, 2, 32, 32, 4, None, why=b"quantised x")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 8, p, 1, 8, 32, 0, None, why=b"gate")
    refused("ovd_gemm_mxfp4", p, p, p, p, None, p, 4, None, 1, 8, 32, 0, None, why=b"ldo")
    refused("ovd_gemm_mxfp4", p, p, p + 8, p, None, p, 8, None, 1, 8, 32, 0, None, why=b"16-byte")
    refused("ovd_linear_mxfp4", p, 0, 32, p, p, None, p, 8, None, None, 0, 9, 8, 32, 0, None, why=b"workspace")
    refused("ovd_linear_mxfp4", p, 0, 32, p, p, None, p, 8, None, p, 4351, 9, 8, 32, 0, None, why=b"workspace")
    refused("ovd_linear_mxfp4", p, 0, 32, p, p, None, p + 64, 8, None, None, 0, 2, 8, 32, 0, None, why=b"shares memory")
    refused("ovd_linear_mxfp4", p, 0, 33, p, p, None, p + 1024, 8, None, None, 0, 2, 8, 32, 0, None, why=b"alignment")
    refused("ovd_linear_mxfp4", p, 0, 32, p, p, None, p, 8, None, None, 0, 2, 8, 32, 5, None, why=b"epilogue")
    assert L.ovd_linear_mxfp4_workspace_bytes(H.MXFP4_FEW_ROWS, H.MXFP4_FEW_K) == 0
    assert L.ovd_linear_mxfp4_workspace_bytes(550, 8960) == sum(H.mxfp4_bytes(550, 8960))
    assert L.ovd_linear_mxfp4_workspace_bytes(8, 13824) == 0 and L.ovd_linear_mxfp4_workspace_bytes(9, 32) == 4352
    assert L.ovd_gemm_mxfp4(p, p, p, p, None, p, 8, None, 0, 8, 32, 0, None) == 0        # no rows: nothing to do


def test_matrix_bytes_are_what_the_library_says():
    assert os.path.exists(H._LIB_PATH)
    m = MXFP4Matrix.empty(5, 96, "cpu")
    assert (m.data.numel(), m.scale.numel()) == (4096, 256)

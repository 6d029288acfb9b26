"""Linear layers on MXFP4 operands (OCP microscaling: 4-bit E2M1 elements, one power-of-two scale per 32 consecutive
values of a row): an extension beside the e4m3 mode, for layers the reference runs as bf16 nn.Linear
(omnivideo/modules/model.py:125-154, :159-179, :218-258).  Backed by ovd_mxfp4_quant, ovd_mxfp4_dequant,
ovd_gemm_mxfp4_as_rows and ovd_linear_mxfp4.  Inference only: the results carry no gradient."""
import torch

from .. import _hip as H

__all__ = ["MXFP4Matrix", "mxfp4_quantize", "mxfp4_linear"]

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


class MXFP4Matrix:
    """A [rows, cols] matrix in MXFP4, its codes and scales in the order in which the matrix instructions read them
    (include/omnihip.h).  Made by `mxfp4_quantize` or `from_ocp`; a layer's weights are laid out once."""

    __slots__ = ("rows", "cols", "buf", "_data_bytes")

    def __init__(self, rows, cols, buf):
        """buf: uint8 device buffer, the codes followed by the scales (H.mxfp4_bytes of each)."""
        nd, ns = H.mxfp4_bytes(rows, cols)
        if buf.dtype != U8 or buf.dim() != 1 or not buf.is_contiguous() or buf.numel() != nd + ns or buf.data_ptr() % 16:
            raise ValueError(f"mxfp4: the buffer does not hold a [{rows}, {cols}] matrix ({nd} + {ns} bytes)")
        self.rows, self.cols, self.buf, self._data_bytes = rows, cols, buf, nd

    @classmethod
    def empty(cls, rows, cols, device):
        """Uninitialised storage for a [rows, cols] matrix (cols a multiple of 32)."""
        nd, ns = H.mxfp4_bytes(rows, cols)
        m = cls.__new__(cls)
        m.rows, m.cols, m.buf, m._data_bytes = rows, cols, torch.empty(nd + ns, dtype=U8, device=device), nd
        return m

    def pointers(self):
        """Device addresses of the codes and the scales."""
        p = self.buf.data_ptr()
        return p, p + self._data_bytes

    @property
    def data(self):
        return self.buf[:self._data_bytes]

    @property
    def scale(self):
        return self.buf[self._data_bytes:]

    @property
    def shape(self):
        return (self.rows, self.cols)

    @property
    def device(self):
        return self.buf.device

    @classmethod
    def from_ocp(cls, codes, scales):
        """From the row-major form of checkpoints: codes uint8 [rows, cols / 2] (k ascending, low nibble first) and
        E8M0 scale bytes uint8 [rows, cols / 32]."""
        if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != U8 or scales.dtype != U8:
            raise TypeError("MXFP4: codes and scales must be two-dimensional uint8 tensors")
        rows, cols = codes.shape[0], 2 * codes.shape[1]
        if rows == 0 or cols == 0 or cols % 32 or tuple(scales.shape) != (rows, cols // 32):
            raise ValueError(f"MXFP4: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not describe a "
                             "matrix with blocks of 32")
        if codes.device != scales.device:
            raise ValueError("MXFP4: codes and scales are on different devices")
        rb, kg = -(-rows // 32), -(-cols // 256)
        c = codes.new_zeros(rb * 32, kg * 128)
        c[:rows, :cols // 2] = codes
        s = scales.new_zeros(rb * 32, kg * 8)
        s[:rows, :cols // 32] = scales
        # [rb, r, kt, h, 16 bytes] -> [rb, kt, h, r, 16];  [rb, r, kg, ks, h] -> [rb, kg, h, r, ks]
        data = c.view(rb, 32, kg * 4, 2, 16).permute(0, 2, 3, 1, 4).contiguous()
        scale = s.view(rb, 32, kg, 4, 2).permute(0, 2, 4, 1, 3).contiguous()
        return cls(rows, cols, torch.cat((data.view(-1), scale.view(-1))))

    def to_ocp(self):
        """(codes [rows, cols / 2], scale bytes [rows, cols / 32]) in row-major order."""
        rb, kg = -(-self.rows // 32), -(-self.cols // 256)
        c = self.data.view(rb, kg * 4, 2, 32, 16).permute(0, 3, 1, 2, 4).reshape(rb * 32, kg * 128)
        s = self.scale.view(rb, kg, 2, 32, 4).permute(0, 3, 1, 4, 2).reshape(rb * 32, kg * 8)
        return c[:self.rows, :self.cols // 2].contiguous(), s[:self.rows, :self.cols // 32].contiguous()

    def dequantize(self, dtype=BF16, out=None):
        """The values it stands for, [rows, cols] bf16 or fp32 (exact in both)."""
        if out is None:
            out = self.buf.new_empty((self.rows, self.cols), dtype=dtype)
        return H.mxfp4_dequant(self, out)


def _no_grad(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("mxfp4: inference only; call under torch.no_grad() or detach the inputs")


def _rows2d(x):
    """x [..., K] as [M, K] with unit column stride and rows on 16-byte boundaries (a copy where it has none)."""
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    ld, step = x2.stride()
    if step != 1 or ld < x2.shape[1] or (ld * x2.element_size()) % 16 or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2


def _check_input(x):
    if x.dtype not in (BF16, F32):
        raise TypeError(f"mxfp4: expected bf16 or fp32, got {x.dtype}")
    if x.dim() == 0 or x.shape[-1] == 0 or x.shape[-1] % 32:
        raise ValueError(f"mxfp4: the last dimension must be a positive multiple of 32, got {tuple(x.shape)}")


def mxfp4_quantize(x, out=None):
    """x [..., K] bf16 or fp32 (K a multiple of 32) -> MXFP4Matrix [M, K], M the product of the leading dimensions.
    A block of 32 gets the scale 2^(floor(log2 max|x|) - 2), its values the nearest E2M1 number (ties to even,
    saturated at 6); a block that holds an infinity or a NaN becomes NaN."""
    _check_input(x)
    _no_grad(x)
    x2 = _rows2d(x)
    if out is None:
        out = MXFP4Matrix.empty(x2.shape[0], x2.shape[1], x.device)
    return H.mxfp4_quant(x2, out)


def mxfp4_linear(x, weight, bias=None, gelu=False, out_dtype=BF16, out=None, residual=None, gate=None,
                 quantize_output=False):
    """act(x @ weight.T + bias) with both operands in MXFP4 and fp32 accumulation; one rounding, of the stored value.
    x: [..., K] bf16 or fp32 (quantised here), or an MXFP4Matrix; weight: MXFP4Matrix [N, K], N a multiple of 4;
    bias bf16 [N]; gelu: tanh-GELU (bf16 output).  Returns [..., N] in out_dtype (bf16 or fp32), written to `out` if given.
    residual: fp32 [..., N], updated in place as residual += y * gate[n] (gate fp32 [N] or None) and returned; out and
    residual may be x itself.
    The sum over K is in a fixed order that depends on the sizes: the same row in a call of more rows may differ in its
    last bit.
    quantize_output (with gelu, N a multiple of 32): the result as an MXFP4Matrix [M, N] (`out` if given), quantised from
    fp32 in the product's own pass: the input of the next layer."""
    if not isinstance(weight, MXFP4Matrix):
        raise TypeError("mxfp4_linear: weight must be an MXFP4Matrix (mxfp4_quantize or MXFP4Matrix.from_ocp)")
    packed = isinstance(x, MXFP4Matrix)
    if not packed:
        _check_input(x)
    lead = (x.rows,) if packed else x.shape[:-1]
    _no_grad(None if packed else x, bias, residual, gate)
    N = weight.rows
    if quantize_output:
        if not gelu or residual is not None or gate is not None:
            raise ValueError("mxfp4_linear: quantize_output goes with gelu, and with neither residual nor gate")
        a = x if packed else mxfp4_quantize(x)
        if out is None:
            out = MXFP4Matrix.empty(a.rows, N, weight.device)
        elif not isinstance(out, MXFP4Matrix):
            raise TypeError("mxfp4_linear: quantize_output writes an MXFP4Matrix")
        return H.gemm_mxfp4_gelu(a, weight, out, bias)
    if residual is not None:
        if out is not None or gelu:
            raise ValueError("mxfp4_linear: residual goes with neither out nor gelu")
        out, epi = residual, H.EPI_RESID
    else:
        if gate is not None:
            raise ValueError("mxfp4_linear: gate goes with residual")
        if out is None:
            out = weight.buf.new_empty((*lead, N), dtype=out_dtype)
        if gelu and out.dtype != BF16:
            raise TypeError("mxfp4_linear: gelu writes bf16")
        epi = H.EPI_BF16_GELU if gelu else (H.EPI_BF16 if out.dtype == BF16 else H.EPI_F32)
    if out.shape != (*lead, N):
        raise ValueError(f"mxfp4_linear: expected an output of shape {(*lead, N)}, got {tuple(out.shape)}")
    if packed:
        return H.gemm_mxfp4(x, weight, out, bias, epi, gate)
    return H.linear_mxfp4(_rows2d(x), weight, out, bias, epi, gate)

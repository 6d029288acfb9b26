"""linear_precision="mxfp4": each of the six layers of each block gets its own operands, weight and bias, alone and under
sequence parallelism."""
import math

import pytest
import torch

from conftest import check_rel
from test_gpu_mxfp4 import close
from test_gpu_mxfp4_model import tiny_model
from test_gpu_sequence_parallel import test_sharded_forward_equals_unsharded as sharded_equals_unsharded

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def test_every_layer_is_its_own_product(monkeypatch):
    import omnivideo._hip as H
    from omnivideo.modules import mxfp4_quantize
    from omnivideo.utils import synthetic as syn
    cfg, m = tiny_model()
    wm = m.wan_model
    lat = syn.randn("in.lat", (16, 3, 8, 12), 1).to(BF16).cuda()
    ctx = [syn.randn("in.text", (10, cfg["text_dim"]), 1).to(BF16).cuda()]
    t = torch.tensor([500])
    ref = wm([lat], t, ctx, 72)[0].clone()
    wm.linear_precision = "mxfp4"
    wm([lat], t, ctx, 72)                                  # the engine of the mode is built
    calls = []                                             # (kind, input tensor or operand, operand values, output)
    quant, gemm, gelu = H.mxfp4_quant, H.gemm_mxfp4, H.gemm_mxfp4_gelu

    def on_quant(x, out):
        quant(x, out)
        calls.append(("quant", x.data_ptr(), x.clone(), out, out.dequantize(F32)))
        return out

    def on_gemm(a, w, out, bias=None, epilogue=H.EPI_BF16, gate=None, **kw):
        assert epilogue == H.EPI_BF16 and gate is None
        gemm(a, w, out, bias, epilogue, **kw)
        calls.append(("gemm", a, a.dequantize(F32), w, bias, out.clone()))
        return out

    def on_gelu(a, w, out, bias=None, **kw):
        gelu(a, w, out, bias, **kw)
        calls.append(("gelu", a, a.dequantize(F32), w, bias, out, out.dequantize(F32)))
        return out

    monkeypatch.setattr(H, "mxfp4_quant", on_quant)
    monkeypatch.setattr(H, "gemm_mxfp4", on_gemm)
    monkeypatch.setattr(H, "gemm_mxfp4_gelu", on_gelu)
    got = wm([lat], t, ctx, 72)[0].clone()
    monkeypatch.undo()                                     # what follows quantises, too
    eng = wm.engine()
    assert [c[0] for c in calls] == (["quant", "gemm"] * 4 + ["quant", "gelu", "gemm"]) * len(wm.blocks)
    h, att = eng.h.data_ptr(), eng.att.data_ptr()
    it = iter(calls)
    for blk in wm.blocks:
        sa, ca = blk.self_attn, blk.cross_attn
        stack = lambda *ls: (torch.cat([x.weight.data for x in ls]), torch.cat([x.bias.data for x in ls]))
        layers = [(h, stack(sa.q, sa.k, sa.v)), (att, stack(sa.o)), (h, stack(ca.q)), (att, stack(ca.o)), (h, stack(blk.ffn[0])),
                  (None, stack(blk.ffn[2]))]
        operand = None
        for source, (weight, bias) in layers:
            if source is not None:
                kind, ptr, x, operand, values = next(it)
                assert kind == "quant" and ptr == source
                assert torch.equal(values, mxfp4_quantize(x).dequantize(F32))
            c = next(it)
            kind, a, A, w, b = c[:5]
            assert a is operand and (source is None or torch.equal(A, values))
            W = mxfp4_quantize(weight).dequantize(F32)
            assert torch.equal(w.dequantize(F32), W) and torch.equal(b.view(-1), bias.view(-1))
            A, W = A.double(), W.double()
            K = A.shape[1]
            want, bound = A @ W.t() + bias.double(), K * 2.0 ** -23 * (A.abs() @ W.abs().t())
            bound = bound + 2.0 ** -24 * (want.abs() + bound)
            if kind == "gemm":
                close(c[5].reshape(want.shape), want, bound, BF16)
            else:
                operand, values = c[5], c[6]
                act = 0.5 * want * (1 + torch.tanh(math.sqrt(2 / math.pi) * (want + 0.044715 * want ** 3)))
                # a code is off by at most a quarter of the value (half a step, and by saturation) or of its block's
                # smallest step; 4 % of that for the fp32 sum
                top = act.abs().reshape(act.shape[0], -1, 32).amax(2, keepdim=True).expand(-1, -1, 32).reshape(act.shape)
                assert ((values.double() - act).abs() <= 0.26 * act.abs() + top / 4 * 0.26 + 1e-6).all()
    # The whole forward.  The rounding takes 0.115 of the L2 norm of a Gaussian operand, so 0.16 of a product's and, through
    # two products one behind the other, 0.23 of what a layer pair adds to the residual stream (attention's softmax and the
    # GELU between them can add to that, what the stream holds from before is exact): below a third of the result.  A layer
    # with another one's weights makes its update independent of the right one: 1.4 of it.  Observed: 1.72e-2; held to three
    # times that.
    check_rel("mxfp4 forward, tiny model, against bf16", (got.float() - ref.float()).norm() / ref.float().norm(), 5.2e-2)


@pytest.mark.parametrize("heads,sp,seq_len", [(2, 2, 72), (4, 4, 80), (4, 2, 76)])
def test_sharded_forward_in_the_mode(heads, sp, seq_len):
    """equal bits: products of so few tiles add in one order, however many rows there are"""
    sharded_equals_unsharded(heads, sp, seq_len, "mxfp4")


def forwards(precision, groups, comms=None):
    """outputs of the forwards of a 3200-token model, one for each group of contexts (and communicator, as threads)"""
    import threading
    from omnivideo.modules.engine import DiTEngine
    from omnivideo.utils import synthetic as syn
    from test_gpu_sequence_parallel import build
    cfg = syn.dit_config("tiny", dim=512, num_heads=4, ffn_dim=2560)
    sd = syn.make_unified_state_dict(cfg, 0)
    for i in range(cfg["num_layers"]):
        # large terms that cancel, 8 k-groups apart: the small ones between them are rounded at the size of the large ones in
        # one order of the sums and exact in the other
        w0, b0, w2 = (sd[f"wan_model.blocks.{i}.ffn.{n}"] for n in ("0.weight", "0.bias", "2.weight"))
        w0[2048:2080], b0[2048:2080] = w0[:32], b0[:32]
        w2[:, :32] *= 2.0 ** 14
        w2[:, 2048:2080] = -w2[:, :32]
    wm = build(cfg, sd)
    lat = syn.randn("in.lat", (16, 5, 32, 80), 1).cuda().to(BF16)
    ts = torch.tensor([640.0], dtype=torch.float64, device="cuda")
    text = [syn.randn("in.text", (10, cfg["text_dim"]), s).cuda().to(BF16) for s in (1, 2)]
    outs, errs = [None] * len(groups), []

    def run(i):
        try:
            eng = DiTEngine(wm, precision=precision)
            eng.plan((5, 16, 40), 3200, len(groups[i]), comm=None if comms is None else comms[i])
            eng.attn_ws = None                             # its split of the last query blocks goes by the launch's grid
            out = torch.empty(len(groups[i]), 16, 5, 32, 80, device="cuda")
            eng.forward(lat, ts, eng.encode_context([text[b] for b in groups[i]], wm.text_len), out)
            torch.cuda.synchronize()
            outs[i] = out
        except Exception as e:          # noqa: BLE001
            errs.append(e)
            if comms is not None:
                comms[i].sh.barrier.abort()

    if comms is None:
        for i in range(len(groups)):
            run(i)
    else:
        th = [threading.Thread(target=run, args=(i,)) for i in range(len(groups))]
        [t.start() for t in th]
        [t.join(120) for t in th]
    assert not errs, errs
    return outs


@pytest.mark.parametrize("precision", ["mxfp4", "fp8", "bf16"])
def test_rows_do_not_depend_on_how_many_a_rank_or_a_batch_has(precision):
    """one branch alone, two in a batch, and the batch over two or four ranks: equal bits, although other kernels compute
    products of 6400 rows than of 3200 or 1600"""
    from test_gpu_sequence_parallel import ThreadComm, _Shared
    both, first, second = forwards(precision, ([0, 1], [0], [1]))
    assert torch.equal(both, torch.cat((first, second)))
    for n in (2, 4):
        shared = _Shared(n)
        for out in forwards(precision, [[0, 1]] * n, [ThreadComm(shared, r) for r in range(n)]):
            assert torch.equal(out, both), f"{n} ranks: {int((out != both).sum())} of {both.numel()} differ"

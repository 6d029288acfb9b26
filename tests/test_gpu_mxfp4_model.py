"""linear_precision="mxfp4": the DiT's large linear layers on MXFP4 operands."""
import math

import pytest
import torch

from test_gpu_mxfp4 import close
from test_planned_bytes import KEYS

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def tiny_model():
    from omnivideo.modules.unified_model import UnifiedWanWithMixedConditionModel
    from omnivideo.utils import synthetic as syn
    cfg = syn.dit_config("tiny")
    m = UnifiedWanWithMixedConditionModel(
        wan_config=dict(cfg), vlm_in_dim=cfg["vlm_in_dim"], use_visual_context_adapter=True,
        visual_context_adapter_patch_size=cfg["visual_patch_size"], max_context_len=cfg["text_len"], eps=cfg["eps"],
        skip_init=True)
    m.load_state_dict(syn.make_unified_state_dict(cfg, 0), strict=True)
    return cfg, m.to(BF16).cuda().eval()


def test_forward_in_the_mxfp4_mode():
    """what the last block's operators were given and wrote is what their definitions say; the mode is deterministic and
    switching back restores the bf16 path"""
    from omnivideo.modules import mxfp4_quantize
    from omnivideo.utils import synthetic as syn
    cfg, m = tiny_model()
    wm = m.wan_model
    lat = syn.randn("in.lat", (16, 3, 8, 12), 1).to(BF16).cuda()
    ctx = [syn.randn("in.text", (10, cfg["text_dim"]), 1).to(BF16).cuda()]
    t = torch.tensor([500])
    ref = wm([lat], t, ctx, 72)[0].clone()
    wm.linear_precision = "mxfp4"
    got = wm([lat], t, ctx, 72)[0].clone()
    eng = wm.engine()
    assert eng.precision == "mxfp4" and eng.attention == "int8" and eng.layers[0]["w_qkv"] is None
    assert torch.isfinite(got).all() and not torch.equal(got, ref)
    L, C = eng.layers[-1], eng.dim
    blk = wm.blocks[-1]
    assert torch.equal(L["w4_f0"].dequantize(), mxfp4_quantize(blk.ffn[0].weight.data).dequantize())
    assert torch.equal(eng.att4.dequantize(), mxfp4_quantize(eng.att.view(-1, C)).dequantize())
    assert torch.equal(eng.h4.dequantize(), mxfp4_quantize(eng.h).dequantize())
    # feed-forward of the last block: gelu(h W0 + b0) quantised, then its product with W2
    h, w0, w2 = (x.dequantize(F32).double() for x in (eng.h4, L["w4_f0"], L["w4_f2"]))
    f = eng.ffn4.dequantize(F32).double()
    pre = h @ w0.t() + L["b_f0"].double()
    act = 0.5 * pre * (1 + torch.tanh(math.sqrt(2 / math.pi) * (pre + 0.044715 * pre ** 3)))
    # a code is off by at most half a step: 1/4 of the value, 1/4 of the smallest normal of its block, 1/4 by saturation
    top = act.abs().reshape(act.shape[0], -1, 32).amax(2, keepdim=True).expand(-1, -1, 32).reshape(act.shape)
    assert ((f - act).abs() <= 0.26 * act.abs() + top / 4 * 0.26 + 1e-6).all()
    K = f.shape[1]
    close(eng.res, f @ w2.t() + L["b_f2"].double(), K * 2.0 ** -23 * (f.abs() @ w2.abs().t()) + 2.0 ** -22, BF16)
    wm.attention_precision = "bf16"
    assert torch.isfinite(wm([lat], t, ctx, 72)[0]).all()
    wm.attention_precision = "auto"
    assert torch.equal(wm([lat], t, ctx, 72)[0], got)
    wm.linear_precision = "bf16"
    assert torch.equal(wm([lat], t, ctx, 72)[0], ref)


def test_generate_in_the_mxfp4_mode():
    """a guided sampling run (graph replay) in the mode: runs, is repeatable, and is not the bf16 run"""
    from omnivideo.configs import Config, t2v_1_3B
    from omnivideo.utils import synthetic as syn
    from omnivideo.x2x_gen_unified_1_3B import OmniVideoX2XUnified1_3B
    cfg = syn.dit_config("tiny")
    sd, sp = syn.make_unified_state_dict(cfg, 0), syn.make_special_tokens(cfg, 0)
    text = syn.randn("in.text", (10, cfg["text_dim"]), 1).to(BF16)
    text_null = syn.randn("in.text_null", (6, cfg["text_dim"]), 1).to(BF16)
    visual = syn.randn("in.visual", (1, 16, 3, 8, 12), 1).cuda()
    noise = syn.randn("gen.noise", (16, 3, 8, 12), 11).to(BF16)
    lats = []
    for prec in ("mxfp4", "mxfp4", "bf16"):
        pipe = OmniVideoX2XUnified1_3B(Config(t2v_1_3B), None, vlm_in_dim=cfg["vlm_in_dim"],
                                       use_visual_context_adapter=True,
                                       visual_context_adapter_patch_size=cfg["visual_patch_size"],
                                       max_context_len=cfg["text_len"], wan_config=dict(cfg), linear_precision=prec)
        pipe.model.load_state_dict(sd, strict=True)
        pipe.model.to(BF16)
        pipe.special_tokens = {k: v.cuda().to(BF16) for k, v in sp.items()}
        lats.append(pipe.generate("", precomputed_context=text, precomputed_context_null=text_null, visual_emb=visual,
                                  size=(96, 64), frame_num=9, shift=5.0, sampling_steps=4, guide_scale=3.0, seed=1,
                                  noise=noise, return_latents=True).float())
    assert torch.isfinite(lats[0]).all()
    assert torch.equal(lats[0], lats[1]) and not torch.equal(lats[0], lats[2])


def test_engine_allocations_match_the_plan():
    from omnivideo import _hip as H
    from omnivideo.modules.engine import DiTEngine, planned_bytes
    from omnivideo.modules.model import WanModel
    from omnivideo.utils import synthetic as syn
    cfg = syn.dit_config("1.3B", num_layers=2, text_len=512)
    grid, seq_len, nb = (5, 16, 16), 1280, 2
    with torch.device("cuda"):
        m = WanModel(**{k: cfg[k] for k in KEYS if k in cfg}, skip_init=True).to(BF16)
    plan = planned_bytes(cfg, grid, seq_len, nb, cfg["text_len"], precision="mxfp4",
                         attn_workspace=H.flash_attn_workspace_bytes(nb, seq_len, cfg["num_heads"], seq_len))
    # bytes of the storages the engine holds beside the model's own (the allocator's block rounding left out: up to
    # 1 MiB for every buffer above 1 MiB)
    from omnivideo.modules import MXFP4Matrix

    def held(objects, known):
        seen = {}
        for o in objects:
            o = o.buf if isinstance(o, MXFP4Matrix) else o
            if torch.is_tensor(o) and o.is_cuda and o.untyped_storage().data_ptr() not in known:
                seen[o.untyped_storage().data_ptr()] = o.untyped_storage().nbytes()
        return seen

    params = {p.untyped_storage().data_ptr() for p in m.parameters()}
    eng = DiTEngine(m, precision="mxfp4")
    copies = held([v for L in eng.layers for v in L.values()], params)
    assert abs(sum(copies.values()) - plan["engine_copies"]) <= 0.001 * plan["engine_copies"]
    before = held(vars(eng).values(), params)
    eng.plan(grid, seq_len, nb)
    ws = held(vars(eng).values(), params | set(before) | set(copies))
    # the plan leaves out vectors of a few rows (modulation, time embedding, the rotation table)
    assert 0 <= sum(ws.values()) - plan["workspaces"] <= 0.002 * plan["workspaces"]

"""Packed operators: plans and refusals (no GPU needed)."""
import ctypes
import math

import pytest
import torch

import omnivideo._hip as H
from omnivideo.modules import RopePlan, grid_positions, packed_attention, packed_rope

BF16 = torch.bfloat16


def test_rope_plan_tables():
    p = RopePlan(128, device="cpu")
    assert p.sections == (22, 21, 21) and p.n_axes == 3
    assert p.axis.tolist() == [0] * 22 + [1] * 21 + [2] * 21
    assert p.freq[0] == 1 / (2 * math.pi)
    for i in range(21):
        assert abs(float(p.freq[22 + i]) * 2 * math.pi / 10000.0 ** (-i / 21) - 1) < 1e-14
    part = RopePlan(32, (2, 0, 3), theta=100.0, device="cpu")
    assert part.axis.tolist() == [0, 0, 2, 2, 2] + [-1] * 11 and part.freq[5:].abs().sum() == 0
    from omnivideo.modules.engine import build_rope_table
    tab = build_rope_table(128, 50, "cpu").double()
    ang = 2 * math.pi * 37 * p.freq
    for a in range(3):
        sel = p.axis == a
        assert (tab[a, 37, sel, 0] - ang[sel].cos()).abs().max() < 1e-7
        assert (tab[a, 37, sel, 1] - ang[sel].sin()).abs().max() < 1e-7


def test_rope_plan_refuses():
    for kw in (dict(head_dim=24), dict(head_dim=0), dict(head_dim=1024), dict(head_dim=32, sections=(9, 9)),
               dict(head_dim=32, sections=()), dict(head_dim=32, sections=(-1, 4)), dict(head_dim=32, sections=(1,) * 9),
               dict(head_dim=32, theta=0.0)):
        with pytest.raises(ValueError):
            RopePlan(device="cpu", **kw)


def test_grid_positions():
    pos, cu = grid_positions([(2, 2, 3), (0, 4, 4), (1, 1, 2)], device="cpu")
    assert cu.tolist() == [0, 12, 12, 14] and pos.dtype == torch.int32
    assert pos.tolist()[:7] == [[0, 0, 0], [0, 0, 1], [0, 0, 2], [0, 1, 0], [0, 1, 1], [0, 1, 2], [1, 0, 0]]
    assert pos.tolist()[12:] == [[0, 0, 0], [0, 0, 1]]
    with pytest.raises(ValueError):
        grid_positions([(1, -1, 2)], device="cpu")


def test_rope_refuses():
    plan = RopePlan(32, (8, 8), device="cpu")
    x, pos = torch.zeros(4, 2, 32, dtype=BF16), torch.zeros(4, 2, dtype=torch.int32)
    bad = [(x, pos[:3]), (x, pos[:, :1]), (x, pos.long()), (x[..., :16], pos), (x.half(), pos), (x[:, :, ::2], pos), (x[0], pos)]
    for a, b in bad:
        with pytest.raises(ValueError):
            packed_rope(a, b, plan)
    with pytest.raises(ValueError, match="CPU"):
        packed_rope(x, pos, plan)
    with pytest.raises(ValueError, match="one shape"):
        packed_rope(x, pos, plan, out=x.float())
    with pytest.raises(NotImplementedError, match="inference"):
        packed_rope(x.float().requires_grad_(), pos, plan)


def test_attention_refuses():
    q, k = torch.zeros(6, 4, 64, dtype=BF16), torch.zeros(9, 2, 64, dtype=BF16)
    c = torch.tensor([0, 2, 6], dtype=torch.int32)
    call = lambda q=q, k=k, v=k, c=c, ck=c, **kw: packed_attention(q, k, v, c, ck, **kw)
    with pytest.raises(ValueError, match="CPU"):
        call()
    with pytest.raises(TypeError, match="bf16"):
        call(q=q.float())
    for kw in (dict(v=k[:8]), dict(k=k[:, :1].repeat(1, 3, 1), v=k[:, :1].repeat(1, 3, 1)), dict(k=k[..., :32], v=k[..., :32]),
               dict(c=c.long()), dict(ck=c[:2]), dict(c=c[:1], ck=c[:1]), dict(prefix=c), dict(prefix=c[:2].long()),
               dict(q=q[0]), dict(q=q.transpose(0, 1)), dict(out=q[:5])):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(NotImplementedError, match="inference"):
        call(q=q.clone().requires_grad_())


def test_c_entries_refuse_before_any_launch():
    L = H.lib()
    buf = (ctypes.c_ubyte * 8192)()
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def refused(fn, *args, why):
        assert getattr(L, fn)(*args) != 0 and why in L.ovd_last_error(), (fn, L.ovd_last_error())

    rope = lambda x=p, ldx=64, axes=2, ldo=64, T=4, N=2, D=32: (x, 0, ldx, p, 0, axes, p, p, p, ldo, T, N, D, 1, 0, None)
    refused("ovd_rope_positions", *rope(x=None), why=b"null")
    refused("ovd_rope_positions", *rope(D=24), why=b"head_dim")
    refused("ovd_rope_positions", *rope(D=528, ldx=2048, ldo=2048), why=b"head_dim")
    refused("ovd_rope_positions", *rope(axes=9), why=b"axes")
    refused("ovd_rope_positions", *rope(T=-1), why=b"tokens")
    refused("ovd_rope_positions", *rope(T=2 ** 40), why=b"grid too large")
    refused("ovd_rope_positions", *rope(ldx=60), why=b"alignment")
    refused("ovd_rope_positions", *rope(x=p + 2), why=b"alignment")

    def attn(q=p, k=p, Tq=4, Tk=4, docs=1, mq=4, N=2, Nk=1, D=64, q_ld=128, k_ld=64, v_ld=64, o_ld=128, causal=0, prefix=None, scale=0.1, cap=0.0):
        return (q, k, k, p, Tq, Tk, p, p, docs, mq, 4, N, Nk, D, q_ld, k_ld, v_ld, o_ld, causal, prefix, scale, cap, None, 0, None)
    refused("ovd_attn_packed_fwd_bf16", *attn(q=None), why=b"null")
    refused("ovd_attn_packed_fwd_bf16", *attn(k=None), why=b"null")
    refused("ovd_attn_packed_fwd_bf16", *attn(D=96), why=b"head_dim")
    refused("ovd_attn_packed_fwd_bf16", *attn(N=3, Nk=2), why=b"query heads")
    refused("ovd_attn_packed_fwd_bf16", *attn(docs=0), why=b"documents")
    refused("ovd_attn_packed_fwd_bf16", *attn(Tk=2 ** 31), why=b"sizes")
    refused("ovd_attn_packed_fwd_bf16", *attn(q_ld=64), why=b"stride")
    refused("ovd_attn_packed_fwd_bf16", *attn(k_ld=68), why=b"alignment")
    refused("ovd_attn_packed_fwd_bf16", *attn(scale=0.0), why=b"softmax_scale")
    refused("ovd_attn_packed_fwd_bf16", *attn(cap=-1.0), why=b"softcap")
    refused("ovd_attn_packed_fwd_bf16", *attn(cap=math.nan), why=b"softcap")
    refused("ovd_attn_packed_fwd_bf16", *attn(prefix=p), why=b"prefix")
    refused("ovd_attn_packed_fwd_bf16", *attn(mq=-1), why=b"bound")
    refused("ovd_attn_packed_fwd_bf16", *attn(docs=2 ** 26), why=b"too many query rows")
    refused("ovd_attn_packed_fwd_bf16", *attn(docs=2 ** 24, N=8, Nk=8, q_ld=512, k_ld=512, o_ld=512, v_ld=512), why=b"grid too large")
    assert L.ovd_attn_packed_fwd_bf16(*attn(Tq=0)) == 0


def test_workspace_sizes(monkeypatch):
    assert H.attn_packed_workspace_bytes(0, 5, 1, 8, 8, 128, 1, 1) == 0
    assert H.attn_packed_workspace_bytes(20280, 20280, 4, 40, 40, 128, 9000, 9000) == 0          # enough rows: not split
    assert H.attn_packed_workspace_bytes(8, 800, 8, 40, 8, 128, 1, 100) == 0                     # short documents: neither
    n = H.attn_packed_workspace_bytes(8, 80000, 8, 40, 8, 128, 1, 32760)
    assert n > 0 and n % (8 * 40 * 130 * 4) == 0

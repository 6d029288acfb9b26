"""Packed attention whose scores are capped far above or far below what they reach, against its definition in 64 bits."""
import math

import pytest
import torch

from test_gpu_packed import check, cu, inputs, P                                     # noqa: F401  (P: the module's fixture)

pytestmark = pytest.mark.gpu
F64 = torch.float64

# scores of about one, caps that leave them as they are: from the largest cap of the plain form to past every score
CAPS = (255.0, 256.0, 257.0, 1e3, 1e4, 1e5, 1e6, 1e7, 1e9, 1e20, 9e29)
FORMS = [                                             # one per launch form: one, four, eight waves, split and joined, masked
    (False, [1, 1, 1], [4097, 1, 640], 8, 1),
    (False, [130, 0, 257, 63], [130, 0, 257, 63], 3, 1),
    (False, [1300, 300], [1900, 1100], 32, 16),
    (True, [300, 17], [65, 700], 4, 2),
    (True, [1100, 1100, 1100, 1100, 600], [1100, 1100, 1200, 1000, 600], 40, 40),
]


def reference(q, k, v, Lq, Lk, causal, cap, scale):
    """(o, bound) in 64 bits.  A score's error is relative to the score, whatever the cap:
    fp32 sums of D products: D 2^-23 of their magnitudes; the cap: below a quarter of it an odd series of four terms, truncated
    below 2^-21, its roundings below 2^-22; from a quarter on 1 - 2 / (1 + e^2x), at most 3.5 x 2^-23 off and rounded once more
    (2^-23), of a tanh of at least 0.244: below 2^-18.  Up to 256 the latter everywhere: 2^-20 of the cap."""
    N, D = q.shape[1:]
    group = N // k.shape[1]
    outs, bounds = [], []
    a = b = 0
    for lq, lk in zip(Lq, Lk):
        if lk == 0:
            outs.append(torch.zeros(lq, N, D, dtype=F64, device=q.device))
            bounds.append(outs[-1])
            a += lq
            continue
        qd = q[a:a + lq].double().transpose(0, 1)
        kd = k[b:b + lk].double().repeat_interleave(group, 1).transpose(0, 1)
        vd = v[b:b + lk].double().repeat_interleave(group, 1).transpose(0, 1)
        s = torch.matmul(qd, kd.transpose(1, 2).contiguous()) * scale
        ds = D * 2.0 ** -23 * torch.matmul(qd.abs(), kd.abs().transpose(1, 2).contiguous()) * scale
        s = cap * torch.tanh(s / cap)
        ds = ds + (cap * 2.0 ** -20 if cap <= 256 else 2.0 ** -18 * s.abs()) + 2.0 ** -22 * s.abs() + 2.0 ** -22
        if causal:
            i = torch.arange(lq, device=q.device)[:, None]
            hide = torch.arange(lk, device=q.device)[None] >= (i + lk - lq + 1).clamp(0, lk)
            s, ds = s.masked_fill(hide, -math.inf), ds.masked_fill(hide, 0.0)
        m = s.amax(2, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
        l = p.sum(2, keepdim=True)
        p = p / torch.where(l > 0, l, torch.ones_like(l))
        # every probability: 2^-8 (bf16) and twice the largest score error (numerator and sum); sums of lk terms
        rel = 2.0 ** -8 + 2 * ds.amax(2, keepdim=True) + (lk + 64) * 2.0 ** -23
        outs.append(torch.matmul(p, vd).transpose(0, 1))
        bounds.append((torch.matmul(p, vd.abs()) * rel).transpose(0, 1))
        a, b = a + lq, b + lk
    return torch.cat(outs), torch.cat(bounds)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("causal,Lq,Lk,N,Nk", FORMS)
def test_caps_far_above_the_scores(P, causal, Lq, Lk, N, Nk, D):                      # noqa: F811
    q, k, v = inputs(Lq, Lk, N, Nk, D, 13 + D)
    for cap in CAPS:
        want, bound = reference(q, k, v, Lq, Lk, causal, cap, D ** -0.5)
        check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=causal, softcap=cap), want, bound)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("cap", [300.0, 1000.0])
def test_scores_on_both_sides_of_a_large_cap(P, cap, D):                              # noqa: F811
    """scores from a thousandth of the cap to four times it in one row, of both signs"""
    Lq, Lk = [70, 3], [500, 400]
    q, k, v = inputs(Lq, Lk, 2, 2, D, 17)
    k = (k.double() * torch.logspace(-3, 0.6, 900, dtype=F64, device="cuda").view(-1, 1, 1)).to(k.dtype)
    want, bound = reference(q, k, v, Lq, Lk, False, cap, cap * D ** -0.5)
    check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), softmax_scale=cap * D ** -0.5, softcap=cap), want, bound)


@pytest.mark.parametrize("D", [128, 64])
def test_infinities_under_the_mask_with_a_large_cap(P, D):                            # noqa: F811
    Lq, Lk = [300, 130], [300, 140]
    q, k, v = inputs(Lq, Lk, 4, 2, D, 19)
    want, bound = reference(q, k, v, Lq, Lk, True, 1e6, D ** -0.5)
    for value in (math.inf, -math.inf):
        vv, kk = v.clone(), k.clone()
        vv[298, 1, 5] = value                         # seen by the last two queries of the first document
        kk[439] = math.nan                            # seen by the last query of the second
        o = P.packed_attention(q, kk, vv, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=True, softcap=1e6)
        assert (o[298:300, 2:, 5].float() == value).all() and torch.isnan(o[429]).all()
        o[298:300, 2:, 5], o[429] = want[298:300, 2:, 5].to(o.dtype), want[429].to(o.dtype)
        check(o, want, bound)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("cap,scale", [(1e-20, None), (1e-37, 10.0), (1e-42, None), (1e-50, None), (1e-30, 1e20)])
def test_caps_that_make_every_score_zero(P, cap, scale, D):                           # noqa: F811
    """a cap of next to nothing leaves the mean of the values, for scores of zero, too"""
    Lq, Lk = [70, 3], [500, 400]
    q, k, v = inputs(Lq, Lk, 2, 2, D, 23)
    q[5], k[600] = 0, 0
    o = P.packed_attention(q, k, v, cu(Lq), cu(Lk), softcap=cap, softmax_scale=scale)
    for a, b, c, d in ((0, 70, 0, 500), (70, 73, 500, 900)):
        vd = v[c:d].double()
        want, size = vd.mean(0).expand(b - a, -1, -1), vd.abs().mean(0).expand(b - a, -1, -1)
        check(o[a:b], want, size * (2.0 ** -8 + (d - c + 64) * 2.0 ** -23))

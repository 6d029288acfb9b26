"""Rotary positions and attention on packed rows of documents, against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture(scope="module")
def P():
    import omnivideo.modules.packed as P
    return P


def randn(shape, seed, scale=1.0, dtype=BF16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ------------------------------------------------------------------------------------------------ rotary positions

def ref_rope(x, pos, sections, theta=10000.0, interleaved=True, inverse=False):
    T, N, D = x.shape
    xd = x.double()
    pairs = xd.reshape(T, N, D // 2, 2) if interleaved else torch.stack((xd[..., :D // 2], xd[..., D // 2:]), -1)
    pairs = pairs.clone()
    p = 0
    for a, n in enumerate(sections):
        for i in range(n):
            ang = pos[:, a].double() * theta ** (-i / n) * (-1 if inverse else 1)
            c, s = ang.cos()[:, None], ang.sin()[:, None]
            x0, x1 = pairs[:, :, p, 0].clone(), pairs[:, :, p, 1].clone()
            pairs[:, :, p, 0], pairs[:, :, p, 1] = x0 * c - x1 * s, x0 * s + x1 * c
            p += 1
    size = pairs.abs().sum(-1, keepdim=True).expand_as(pairs)
    join = (lambda t: t.reshape(T, N, D)) if interleaved else (lambda t: torch.cat((t[..., 0], t[..., 1]), -1))
    return join(pairs), join(size)


def check_rope(got, x, pos, plan, inverse=False):
    want, size = ref_rope(x, pos, plan.sections, plan.theta, plan.interleaved, inverse)
    # sine and cosine: the reduced angle's rounding (pi/4 2^-24) and at most four roundings of the polynomials; two
    # products and a sum: 2^-24 each of |x0| + |x1| (|x0|, |x1| <= sqrt 2 of the rotated pair's sum): below 2^-20
    tol = 2.0 ** -20 * size + torch.finfo(x.dtype).eps / 2 * (want.abs() + 2.0 ** -20 * size) + 1e-40
    err = (got.double() - want).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,N,D,sections", [(1, 1, 128, None), (7, 40, 128, None), (301, 12, 128, (44, 10, 10)),
                                            (33, 3, 64, (32,)), (5, 2, 32, (1, 2, 3, 4)), (19, 5, 96, None),
                                            (64, 1, 512, (0, 256)), (10, 7, 16, (3, 3, 2)), (129, 16, 80, (10, 20))])
def test_rope_equals_definition(P, T, N, D, sections, interleaved, dtype):
    plan = P.RopePlan(D, sections, interleaved=interleaved)
    A = plan.n_axes
    x = randn((T, N, D), T + D, dtype=dtype)
    g = torch.Generator().manual_seed(D)
    pos = torch.randint(-3, 90, (T, A), generator=g).to(torch.int32).cuda()
    for inverse in (False, True):
        check_rope(P.packed_rope(x, pos, plan, inverse=inverse), x, pos, plan, inverse)
    posf = (pos.float() * 0.37)
    check_rope(P.packed_rope(x, posf, plan), x, posf, plan)


def test_rope_far_positions(P):
    """angles of positions up to 2^31 keep their accuracy"""
    plan = P.RopePlan(64, (16, 16))
    pos = torch.tensor([[0, 2 ** 31 - 1], [-2 ** 31, 1], [10 ** 9 + 7, 123456789], [99991, 65536]], dtype=torch.int32).cuda()
    for dt in (BF16, F32):
        x = randn((4, 8, 64), 1, dtype=dt)
        check_rope(P.packed_rope(x, pos, plan), x, pos, plan)


def test_rope_every_quarter_turn(P):
    """theta and positions that put the angle on and around every eighth of a turn"""
    plan = P.RopePlan(16, (8,), theta=1.0)
    pos = (torch.arange(-64, 65, dtype=F32) * (math.pi / 32)).cuda()
    x = randn((129, 4, 16), 2, dtype=F32)
    check_rope(P.packed_rope(x, pos, plan), x, pos[:, None], plan)


def test_rope_pass_through_and_special_values(P):
    plan = P.RopePlan(32, (2, 3))                        # 5 of 16 pairs turn
    x = randn((6, 2, 32), 3, dtype=F32)
    x[0, 0, 10], x[1, 1, 31] = math.inf, math.nan        # in pairs that pass through
    pos = torch.ones(6, 2, dtype=torch.int32, device="cuda")
    y = P.packed_rope(x, pos, plan)
    assert torch.equal(torch.nan_to_num(y[..., 10:], 7.0), torch.nan_to_num(x[..., 10:], 7.0))
    check_rope(y[2:], x[2:], pos[2:], plan)
    zero = P.packed_rope(x[2:], torch.zeros_like(pos[2:]), plan)
    assert torch.equal(zero, x[2:])                      # position 0 changes nothing


def test_rope_equals_grid_form(P):
    """the model's rotation of one regular grid (rope_apply) is the positions form of grid_positions"""
    from omnivideo.modules.model import rope_apply
    grids = [(3, 4, 6), (1, 9, 5)]
    pos, cu = P.grid_positions(grids)
    assert cu.tolist() == [0, 72, 117] and pos[72 + 9].tolist() == [0, 1, 4]
    x = randn((117, 2, 128), 4)
    y = P.packed_rope(x, pos, P.RopePlan(128))
    for i, (a, b) in enumerate(((0, 72), (72, 117))):
        want = rope_apply(x[None, a:b], torch.tensor([grids[i]]))[0]
        # two correctly rounded-to-bf16 forms of one value may differ by a step of bf16 where it lies next to a border
        assert ((y[a:b].float() - want).abs() <= 2.0 ** -7 * want.abs() + 1e-6).all()


def test_rope_strided_in_place_and_empty(P):
    plan = P.RopePlan(128)
    qkv = randn((50, 3 * 512), 5)
    pos, _ = P.grid_positions([(2, 5, 5)])
    want = P.packed_rope(qkv[:, 512:1024].unflatten(1, (4, 128)).contiguous(), pos, plan)
    keep = qkv.clone()
    view = qkv[:, 512:1024].unflatten(1, (4, 128))
    assert P.packed_rope(view, pos, plan, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view, want)
    assert torch.equal(qkv[:, :512], keep[:, :512]) and torch.equal(qkv[:, 1024:], keep[:, 1024:])
    back = P.packed_rope(view, pos, plan, inverse=True)
    assert ((back - keep[:, 512:1024].unflatten(1, (4, 128))).abs() <= 2.0 ** -6 * 4.5).all()
    assert P.packed_rope(view[:0], pos[:0], plan).shape == (0, 4, 128)


# ------------------------------------------------------------------------------------------------ attention

def ref_attention(q, k, v, Lq, Lk, causal, prefix, cap, scale):
    """(o, bound): bound is what the bf16 rounding of the probabilities, the fp32 scores and sums may move o by"""
    N, D = q.shape[1:]
    group = N // k.shape[1]
    outs, bounds = [], []
    a = b = 0
    for d, (lq, lk) in enumerate(zip(Lq, Lk)):
        qd = q[a:a + lq].double().transpose(0, 1)
        kd = k[b:b + lk].double().repeat_interleave(group, 1).transpose(0, 1)
        vd = v[b:b + lk].double().repeat_interleave(group, 1).transpose(0, 1)
        s = torch.matmul(qd, kd.transpose(1, 2).contiguous()) * scale
        # fp32 sums of D products: D 2^-23 of their magnitudes; then the scale and exp2: 2^-22 of the score
        ds = (D * 2.0 ** -23 * torch.matmul(qd.abs(), kd.abs().transpose(1, 2).contiguous()) * scale)
        if cap:
            s = cap * torch.tanh(s / cap)
            ds = ds + cap * 2.0 ** -20                     # 1 - 2 / (1 + e): rcp, exp2 and the sum, each 2^-22 of cap
        ds = ds + 2.0 ** -22 * s.abs() + 2.0 ** -22
        if causal:
            i = torch.arange(lq, device=q.device)[:, None]
            seen = torch.clamp(i + lk - lq + 1, min=min(prefix[d], lk) if prefix else 0).clamp(0, lk)
            hide = torch.arange(lk, device=q.device)[None] >= seen
            s = s.masked_fill(hide, -math.inf)
            ds = ds.masked_fill(hide, 0.0)
        if lk == 0:
            outs.append(torch.zeros(lq, N, D, dtype=F64, device=q.device))
            bounds.append(torch.zeros(lq, N, D, dtype=F64, device=q.device))
        else:
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


def cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def check(got, want, bound):
    err = (got.double() - want).abs()
    tol = bound + 2.0 ** -8 * (want.abs() + bound) + 1e-37
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max())} of the tolerance"


def inputs(Lq, Lk, N, Nk, D, seed, scale=1.0):
    return (randn((sum(Lq), N, D), seed, scale), randn((sum(Lk), Nk, D), seed + 1, scale), randn((sum(Lk), Nk, D), seed + 2))


CASES = [
    # Lq, Lk, N, Nk
    ([1], [1], 1, 1),
    ([5, 1, 64, 33], [5, 1, 64, 33], 2, 2),
    ([130, 0, 257, 63], [130, 0, 257, 63], 3, 1),
    ([300, 17], [65, 700], 4, 2),
    ([128, 1, 2], [0, 5, 64], 2, 1),
    ([1, 1, 1], [4097, 1, 640], 8, 1),
    ([2, 0, 1, 4], [1000, 33, 128, 3], 5, 1),
    ([1] * 70 + [200], list(range(1, 71)) + [100], 2, 2),
    ([700, 1100], [700, 1100], 12, 12),
    ([3, 40], [1200, 9], 40, 8),
]


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk,N,Nk", CASES)
def test_attention_documents(P, Lq, Lk, N, Nk, D):
    q, k, v = inputs(Lq, Lk, N, Nk, D, len(Lq) + D)
    for cap in (0.0, 20.0):
        want, bound = ref_attention(q, k, v, Lq, Lk, False, None, cap, D ** -0.5)
        check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), max_q=max(Lq), max_k=max(Lk), softcap=cap), want, bound)
    want, bound = ref_attention(q, k, v, Lq, Lk, False, None, 0.0, 0.3)
    check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), softmax_scale=0.3), want, bound)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk,N,Nk", CASES)
def test_attention_causal_and_prefix(P, Lq, Lk, N, Nk, D):
    q, k, v = inputs(Lq, Lk, N, Nk, D, 50 + len(Lq) + D)
    want, bound = ref_attention(q, k, v, Lq, Lk, True, None, 0.0, D ** -0.5)
    check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=True), want, bound)
    prefix = [(7 * i + 3) % (n + 5) for i, n in enumerate(Lk)]
    pt = torch.tensor(prefix, dtype=torch.int32, device="cuda")
    for cap in (0.0, 30.0):
        want, bound = ref_attention(q, k, v, Lq, Lk, True, prefix, cap, D ** -0.5)
        check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=True, prefix=pt, softcap=cap), want, bound)


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("causal,Lq,Lk,N,Nk", [
    (False, [1300, 1500], [1300, 1500], 16, 16), (False, [1300, 300], [1900, 1100], 32, 16),
    (True, [1100, 1100, 1100, 1100, 600], [1100, 1100, 1200, 1000, 600], 40, 40)])
def test_attention_of_enough_rows_for_wide_workgroups(P, causal, Lq, Lk, N, Nk, D):
    q, k, v = inputs(Lq, Lk, N, Nk, D, 31 + D)
    prefix = [0, 300, 5, 0, 600] if causal else None
    pt = torch.tensor(prefix, dtype=torch.int32, device="cuda") if causal else None
    for cap in (0.0, 20.0):
        want, bound = ref_attention(q, k, v, Lq, Lk, causal, prefix, cap, D ** -0.5)
        check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=causal, prefix=pt, softcap=cap), want, bound)
        if causal:                                       # a hidden infinity: seen by the last two queries of the first document
            vv = v.clone()
            vv[Lk[0] - 2, 3, 7] = math.inf
            o = P.packed_attention(q, k, vv, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=True, prefix=pt, softcap=cap)
            assert (o[Lq[0] - 2:Lq[0], 3, 7] == math.inf).all()
            o[Lq[0] - 2:Lq[0], 3, 7] = want[Lq[0] - 2:Lq[0], 3, 7].to(BF16)
            check(o, want, bound)


def test_attention_large_scores(P):
    """scores of several hundred, one dominating key late in the row, and capped ones"""
    Lq, Lk = [70, 3], [500, 400]
    q, k, v = inputs(Lq, Lk, 2, 2, 128, 9, 4.0)
    k[450] = q[0, 0:2] * 3
    for cap in (0.0, 50.0, 5.0, 300.0, 0.01, 1e6):       # scores past the cap, around half of it, far below it
        want, bound = ref_attention(q, k, v, Lq, Lk, False, None, cap, 128 ** -0.5)
        check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), softcap=cap), want, bound)


def test_attention_hints_do_not_change_what_is_computed(P):
    """length bounds that are too small or too large choose another launch, not another result"""
    Lq, Lk = [300, 1, 90], [300, 1500, 90]
    q, k, v = inputs(Lq, Lk, 4, 2, 128, 3)
    want, bound = ref_attention(q, k, v, Lq, Lk, False, None, 0.0, 128 ** -0.5)
    for mq, mk in ((1, 1), (16, 64), (0, 0), (300, 1500), (10 ** 6, 10 ** 6), (1, 10 ** 6)):
        out = torch.full_like(q, math.nan)
        check(P.packed_attention(q, k, v, cu(Lq), cu(Lk), mq, mk, out=out), want, bound)


def test_attention_outside_a_document_nothing_is_read_or_written(P):
    """NaN and infinities in rows before, between and behind the documents; output rows there stay as they were"""
    for D, N, Nk in ((128, 4, 2), (64, 2, 2)):
        for Lq, Lk in (([70, 5], [100, 37]), ([1, 2], [900, 70])):
            q, k, v = inputs(Lq, Lk, N, Nk, D, 11)
            pad = lambda t, n: torch.full((n,) + t.shape[1:], math.nan, dtype=BF16, device="cuda")
            qq = torch.cat((pad(q, 3), q, pad(q, 9)))
            kk, vv = (torch.cat((pad(t, 2), t, torch.full_like(pad(t, 80), math.inf))) for t in (k, v))
            out = torch.full_like(qq, 3.0)
            P.packed_attention(qq, kk, vv, cu(Lq) + 3, cu(Lk) + 2, max(Lq), max(Lk), out=out)
            want, bound = ref_attention(q, k, v, Lq, Lk, False, None, 0.0, D ** -0.5)
            check(out[3:-9], want, bound)
            assert (out[:3] == 3).all() and (out[-9:] == 3).all()
            # a NaN inside one document stays there
            kk[2 + Lk[0]] = math.nan
            P.packed_attention(qq, kk, vv, cu(Lq) + 3, cu(Lk) + 2, max(Lq), max(Lk), out=out)
            check(out[3:3 + Lq[0]], want[:Lq[0]], bound[:Lq[0]])
            assert torch.isnan(out[3 + Lq[0]:-9]).all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk,N,Nk", [([300], [300], 2, 2), ([1, 3], [700, 900], 8, 1), ([700, 130], [720, 140], 4, 2)])
def test_attention_infinities_and_nan_under_the_causal_mask(P, Lq, Lk, N, Nk, D):
    """what a hidden key and its value hold does not enter a row; a row that sees it gets the infinity or NaN"""
    q, k, v = inputs(Lq, Lk, N, Nk, D, 77)
    want, bound = ref_attention(q, k, v, Lq, Lk, True, None, 0.0, D ** -0.5)
    bad = Lk[0] - 2                                    # seen by the last two queries of the first document
    q0 = Lq[0]
    hidden = max(q0 - 2, 0)
    for value in (math.nan, math.inf, -math.inf):
        vv = v.clone()
        vv[bad, 0, 5], vv[bad, 0, D - 1] = value, value
        o = P.packed_attention(q, k, vv, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=True)
        heads = N // Nk
        assert torch.isfinite(o[hidden:q0, :, 6:D - 1]).all()
        seen = o[hidden:q0, :heads, [5, D - 1]].float()
        assert torch.isnan(seen).all() if math.isnan(value) else bool((seen == value).all())
        o[hidden:q0, :heads, [5, D - 1]] = want[hidden:q0, :heads, [5, D - 1]].to(BF16)
        check(o, want, bound)
    kk = k.clone()
    kk[bad] = math.nan
    o = P.packed_attention(q, kk, v, cu(Lq), cu(Lk), max(Lq), max(Lk), causal=True)
    assert torch.isnan(o[hidden:q0]).all()
    o[hidden:q0] = want[hidden:q0].to(BF16)
    check(o, want, bound)


def test_attention_strided_views_of_a_fused_projection(P):
    T, N, D = 333, 4, 128
    buf = randn((T, 3 * N * D + 8), 21)
    q, k, v = (buf[:, i * N * D:(i + 1) * N * D].unflatten(1, (N, D)) for i in range(3))
    Lq = [200, 133]
    out = torch.zeros(T, 2 * N * D, dtype=BF16, device="cuda")
    o = out[:, N * D:].unflatten(1, (N, D))
    P.packed_attention(q, k, v, cu(Lq), out=o, causal=True)
    want = P.packed_attention(*(t.contiguous() for t in (q, k, v)), cu(Lq), causal=True)
    assert torch.equal(o, want) and (out[:, :N * D] == 0).all()


def test_attention_in_place_and_without_keys(P):
    for Lq, Lk, N, Nk in (([300, 70], [200, 9], 4, 2), ([1, 2, 1], [900, 0, 70], 8, 2)):
        q, k, v = inputs(Lq, Lk, N, Nk, 128, 12)
        want = P.packed_attention(q, k, v, cu(Lq), cu(Lk), max(Lq), max(Lk))
        own = q.clone()
        assert P.packed_attention(own, k, v, cu(Lq), cu(Lk), max(Lq), max(Lk), out=own) is own
        assert torch.equal(own, want)
        for causal in (False, True):
            o = P.packed_attention(q, k[:0], v[:0], cu(Lq), torch.zeros(len(Lq) + 1, dtype=torch.int32, device="cuda"), causal=causal)
            assert (o == 0).all()
    assert P.packed_attention(q[:0], k, v, cu([0, 0, 0]), cu(Lk)).shape == (0, 8, 128)


def test_attention_equals_flash_attn_on_one_document(P):
    import omnivideo._hip as H
    q, k, v = inputs([600], [600], 2, 2, 128, 5)
    ref = torch.empty_like(q)
    H.flash_attn(q[None], k[None], v[None], ref[None])
    want, bound = ref_attention(q, k, v, [600], [600], False, None, 0.0, 128 ** -0.5)
    check(ref, want, bound)
    check(P.packed_attention(q, k, v, cu([600])), want, bound)


def test_attention_bad_offsets_stay_inside_the_tensors(P):
    """offsets past the tensors and descending ones are clamped: nothing outside is touched"""
    q, k, v = inputs([40], [60], 2, 1, 64, 6)
    out = torch.full((60, 2, 64), 3.0, dtype=BF16, device="cuda")
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for cq, ck in ((t(-5, 10, 1000), t(-9, 30, 2 ** 30)), (t(0, 50, 20), t(60, 0, 70)), (t(2 ** 30, 2 ** 30, 5), t(0, 60, 60))):
        P.packed_attention(q, k, v, cq, ck, out=out[10:50])
        torch.cuda.synchronize()
        assert (out[:10] == 3).all() and (out[50:] == 3).all()
    P.packed_attention(q, k, v, t(0, 40, 1000), t(0, 60, 1000), out=out[10:50])
    want, bound = ref_attention(q, k, v, [40], [60], False, None, 0.0, 0.125)
    check(out[10:50], want, bound)


@pytest.mark.parametrize("Lq,Lk,N,Nk", [([1, 1, 1, 1], [900, 3, 2000, 64], 8, 2), ([500, 300], [500, 300], 4, 4)])
def test_attention_streams_graphs_and_changing_lengths(P, Lq, Lk, N, Nk):
    """a captured call follows lengths that change under it; two graphs and an eager call do not share a workspace"""
    D = 128
    q, k, v = inputs(Lq, Lk, N, Nk, D, 31)
    cq, ck = cu(Lq), cu(Lk)
    eager = P.packed_attention(q, k, v, cq, ck, max(Lq), max(Lk))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(P.packed_attention(q, k, v, cq, ck, max(Lq), max(Lk)), eager)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    cq2, ck2 = cq.clone(), ck.clone()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(P.packed_attention(q, k, v, cq2, ck2, max(Lq), max(Lk)))
        graphs.append(g)
    lens = ([Lk[0] - 7] + [Lk[1] + 7] + Lk[2:], Lk, [1, Lk[0] + Lk[1] - 1] + Lk[2:])
    for n in lens:
        ck2.copy_(cu(n))
        want = P.packed_attention(q, k, v, cq, cu(n), max(Lq), max(Lk))
        ref, bound = ref_attention(q, k, v, Lq, n, False, None, 0.0, D ** -0.5)
        check(want, ref, bound)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_run_of_the_operators_together(P):
    """quantised q|k|v projection, rotation by position, attention inside documents, quantised output projection of two
    grids in one packed row: equal to each grid on its own"""
    from omnivideo.modules import mxfp4_linear, mxfp4_quantize
    C, N, D = 512, 4, 128
    grids = [(3, 10, 13), (1, 7, 9)]
    pos, c = P.grid_positions(grids)
    T = int(c[-1])
    x = randn((T, C), 1)
    wqkv = mxfp4_quantize(randn((3 * C, C), 2, 1 / math.sqrt(C)))
    wo = mxfp4_quantize(randn((C, C), 3, 1 / math.sqrt(C)))
    bias = randn((3 * C,), 4, 0.1)
    plan = P.RopePlan(D)

    def block(x, pos, c):
        qkv = mxfp4_linear(x, wqkv, bias)
        qk = qkv[:, :2 * C].unflatten(1, (2 * N, D))
        P.packed_rope(qk, pos, plan, out=qk)
        o = P.packed_attention(qk[:, :N], qk[:, N:], qkv[:, 2 * C:].unflatten(1, (N, D)), c)
        return mxfp4_linear(o.flatten(1), wo, out_dtype=F32), qkv

    y, qkv = block(x, pos, c)
    assert torch.isfinite(y).all()
    n0 = int(c[1])
    for a, b, g in ((0, n0, grids[0]), (n0, T, grids[1])):
        pg, cg = P.grid_positions([g])
        yg, qkvg = block(x[a:b], pg, cg)
        # projection sums may be formed in another order for another row count: fp32 sums of C products, then the
        # bf16 rounding may fall on the other side
        assert ((qkv[a:b].float() - qkvg.float()).abs() <= 2.0 ** -6 * qkvg.float().abs() + 1e-2).all()
        rel = float((y[a:b] - yg).norm() / yg.norm())
        assert rel < 0.1, rel

"""Operators on packed rows of tokens: several documents (videos, images, prompts of different sizes) in one [tokens, ...]
tensor, without padding.  `packed_rope` and `packed_attention` stand beside `rope_apply` and `flash_attention`
(reference: omnivideo/modules/model.py:37-65, attention.py:24-133), which take one grid and one length per batch entry.
Inference only: the results carry no gradient."""
import torch

from .. import _hip as H

__all__ = ["RopePlan", "grid_positions", "packed_rope", "packed_attention"]

BF16, F32 = torch.bfloat16, torch.float32


def _no_grad(*tensors):
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("packed operators: inference only; call under torch.no_grad() or detach the inputs")


class RopePlan:
    """Which pair of a head turns with which axis, and how fast.  sections: pairs per axis, in order (default: the
    model's time / height / width split of head_dim / 2 pairs); pairs left over are passed through.  The i-th of an
    axis' n pairs turns by theta^(-i / n) radians per unit of position.  interleaved: pairs (2p, 2p + 1) as in the
    model; otherwise (p, p + head_dim / 2)."""

    def __init__(self, head_dim, sections=None, theta=10000.0, interleaved=True, device="cuda"):
        c = head_dim // 2
        if head_dim % 16 or not 0 < head_dim <= 512:
            raise ValueError(f"rope: head_dim {head_dim} must be a multiple of 16, at most 512")
        sections = (c - 2 * (c // 3), c // 3, c // 3) if sections is None else tuple(int(n) for n in sections)
        if not 1 <= len(sections) <= 8 or any(n < 0 for n in sections) or sum(sections) > c:
            raise ValueError(f"rope: sections {sections} do not fit {c} pairs on 1 to 8 axes")
        if not theta > 0:
            raise ValueError("rope: theta must be positive")
        freq, axis = torch.zeros(c, dtype=torch.float64), torch.full((c,), -1, dtype=torch.int32)
        p = 0
        for a, n in enumerate(sections):
            if n:
                turn = torch.arange(n, dtype=torch.float64) / n
                freq[p:p + n] = torch.pow(torch.tensor(float(theta), dtype=torch.float64), -turn) / (2 * torch.pi)
                axis[p:p + n] = a
                p += n
        self.head_dim, self.sections, self.theta, self.interleaved = head_dim, sections, float(theta), bool(interleaved)
        self.freq, self.axis = freq.to(device), axis.to(device)

    @property
    def n_axes(self):
        return len(self.sections)


def grid_positions(grids, device="cuda"):
    """grids: [(frames, height, width), ...] of the documents of a packed row -> (positions int32 [T, 3] in the model's
    token order, cu_seqlens int32 [documents + 1])."""
    pos, cu = [], [0]
    for f, h, w in grids:
        if min(f, h, w) < 0:
            raise ValueError(f"grid_positions: bad grid {(f, h, w)}")
        t = torch.arange(f * h * w, dtype=torch.int32)
        hw = max(h * w, 1)
        pos.append(torch.stack((t // hw, (t % hw) // max(w, 1), t % max(w, 1)), 1))
        cu.append(cu[-1] + f * h * w)
    return torch.cat(pos).to(device), torch.tensor(cu, dtype=torch.int32, device=device)


def packed_rope(x, positions, plan, out=None, inverse=False):
    """x [T, N, D] bf16 or fp32 (dense heads; the tokens may be strided), positions [T, axes] int32 or fp32 (or [T] for
    one axis), plan a RopePlan of head_dim D.  Returns the rotated heads, in `out` if given (x itself, or memory that does
    not overlap it).
    inverse: the opposite rotation.  Angles are formed in 64 bits: off by at most 2^-51 of the turns made (2e-7 turns for any
    int32 position; fp32 positions past about 1e15 mean nothing any more).  The rotation is computed in fp32 (2^-20 of
    |x0| + |x1|) and rounded to x's type."""
    _no_grad(x)
    if positions.dim() == 1:
        positions = positions[:, None]
    if positions.dim() != 2 or positions.shape[1] != plan.n_axes:
        raise ValueError(f"packed_rope: positions must be [tokens, {plan.n_axes}], got {tuple(positions.shape)}")
    if x.dim() != 3 or x.shape[2] != plan.head_dim:
        raise ValueError(f"packed_rope: x must be [tokens, heads, {plan.head_dim}], got {tuple(x.shape)}")
    if out is None:
        out = x.new_empty(x.shape)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    return H.rope_positions(x, positions, plan.freq, plan.axis, out, plan.interleaved, inverse)


def packed_attention(q, k, v, cu_q, cu_k=None, max_q=None, max_k=None, causal=False, prefix=None, softcap=0.0,
                     softmax_scale=None, out=None, workspace=None):
    """Softmax attention inside documents.  q [Tq, Nq, D], k and v [Tk, Nk, D] bf16 with D 64 or 128, dense heads and
    free token strides (views into a fused projection buffer); query head h reads key head h // (Nq / Nk).
    cu_q, cu_k: int32 [documents + 1] device tensors; document d owns query rows cu_q[d] .. cu_q[d + 1] and key rows
    cu_k[d] .. cu_k[d + 1] (cu_k None: the same).  Query i of Lq sees the Lk keys of its document, with `causal` the
    first max(i + Lk - Lq + 1, prefix[d]) of them (prefix int32 [documents] or None).  softcap > 0 caps the scores:
    softcap * tanh(s / softcap), exact to 2^-20 of a cap up to 256 and to 2^-18 of the score above.  softmax_scale defaults to
    D ** -0.5.  Softmax and sums are fp32; the probabilities are rounded to bf16 for their product with v.
    A query that sees no key gets zeros.  Rows outside every document are not written (uninitialised when `out` is not
    given).  A key that is hidden from a query does not enter its result, whatever it and its value hold.  `out` may be q
    itself, but not share memory with k or v.
    max_q, max_k: the longest document as the caller knows it (default: the totals); they size the launch, any value
    gives right results.  workspace: a byte buffer of H.attn_packed_workspace_bytes(...) (default: allocated here)."""
    _no_grad(q, k, v)
    cu_k = cu_q if cu_k is None else cu_k
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("packed_attention: q, k and v must be [tokens, heads, head_dim]")
    Tq, Nq, D = q.shape
    max_q = Tq if max_q is None else int(max_q)
    max_k = k.shape[0] if max_k is None else int(max_k)
    if out is None:
        out = q.new_empty(q.shape)
    if workspace is None and q.is_cuda and Tq:
        n = H.attn_packed_workspace_bytes(Tq, k.shape[0], cu_q.numel() - 1, Nq, k.shape[1], D, max_q, max_k)
        if n > 0:
            workspace = torch.empty(n, dtype=torch.uint8, device=q.device)
    return H.attn_packed(q, k, v, cu_q, cu_k, out, max_q, max_k, causal, prefix, softmax_scale, softcap, workspace)

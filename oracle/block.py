"""64-bit restatements of the block operators (linear with epilogue, the norms
around a branch, key-block selection and attention) — test infrastructure only.

Each returns its result in float64 and, where a kernel's result is compared with
it, the bound on a kernel that accumulates in fp32 and rounds once, from the
magnitudes of the terms: ``U`` is fp32's half step, ``H`` bf16's.
"""

from __future__ import annotations

import math

import torch

__all__ = ["H", "U", "activation_reference", "linear_reference", "sandwich_reference", "select_reference", "sparse_reference"]

U = 2.0**-24  # half a step of fp32, relative
H = 2.0**-8  # of bf16
BLOCK_Q, BLOCK_K = 256, 64


def activation_reference(z: torch.Tensor, kind: str | None) -> torch.Tensor:
    if kind is None:
        return z
    if kind == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    assert kind == "gelu_tanh"
    return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z**3))


def linear_reference(x, weight, bias=None, activation=None, gated=False, residual=None, gate=None, index=None, *, sums=0.0, rounded=True):
    """``(y, bound)``. The bound: k products summed in any order in fp32 are off by
    at most (k + 2) U times the sum of their magnitudes (``sums`` more, relative to
    it, where the products' sums are narrower); the activations' slopes are under
    1.2, and they are evaluated to 2e-5 of their value; then the steps of the
    epilogue and, unless ``rounded`` is false, the rounding to bf16."""

    x, w = x.double().reshape(-1, x.shape[-1]), weight.double()
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    off = ((x.shape[1] + 2) * U + sums) * size
    if gated:
        (v, g), (ov, og) = z.chunk(2, -1), off.chunk(2, -1)
        a = activation_reference(g, activation)
        oa = 1.2 * og + 2e-5 * a.abs()
        y, off = v * a, ov * (a.abs() + oa) + v.abs() * oa
    else:
        y = activation_reference(z, activation)
        off = 1.2 * off + 2e-5 * y.abs()
    if gate is not None:
        t = index.reshape(-1).long()[torch.arange(x.shape[0], device=x.device) % index.numel()].clamp(0, gate.shape[0] - 1)
        y, off = y * gate.double()[t], off * gate.double()[t].abs()
    if residual is not None:
        r = residual.double().reshape(y.shape)
        y, off = y + r, off + 4 * U * (y.abs() + r.abs())
    return y, off + 8 * U * y.abs() + (H * (y.abs() + off) if rounded else 0.0) + 1e-37


def _rms(x, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)


def sandwich_reference(residual, branch, branch_weight, gate, weight, scale, shift, index, eps, residual_scale=1.0):
    """``(hidden, bound, normed, bound)``. A row's sum of squares is off by at
    most cols U of itself, its rsqrt by half that; the products by a few U."""

    C = residual.shape[-1]
    r, b = residual.double().reshape(-1, C), branch.double().reshape(-1, C)
    rows = torch.arange(r.shape[0], device=r.device)
    tables = [t for t in (gate, scale, shift) if t is not None]
    if tables:
        t = index.reshape(-1).long()[rows % index.numel()].clamp(0, min(x.shape[0] for x in tables) - 1)
    n = _rms(b, eps) * branch_weight.double()
    if gate is not None:
        n = n * gate.double()[t]
    h = residual_scale * r + n
    step = (C + 16) * U
    size = (residual_scale * r).abs() + n.abs()
    h_off = 4 * U * size + step * n.abs() + 1e-37
    if weight is None:
        return h, h_off + H * (h.abs() + h_off), None, None
    inv = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
    factor = weight.double() * (1.0 + scale.double()[t])
    # the norm's factor moves with the rounding of h: by at most the mean of h_off |h|
    move = (h_off * h.abs()).mean(-1, keepdim=True) * inv**2
    y = h * inv * factor + shift.double()[t]
    y_off = (h_off + h.abs() * (step + move)) * inv * (factor.abs() + 4 * U * weight.double().abs()) + 4 * U * (
        (h * inv * factor).abs() + shift.double()[t].abs()
    )
    return h, h_off + H * (h.abs() + h_off), y, y_off + H * (y.abs() + y_off)


def _means(x, block):
    return torch.stack([part.double().mean(dim=1) for part in x.split(block, dim=1)], dim=2).float().double()


def select_reference(q, k, topk, always=None):
    """int32 (B, H, nq, min(topk, nk)), ascending."""

    score = (_means(q, BLOCK_Q) @ _means(k, BLOCK_K).transpose(-1, -2)).float().double()
    score = torch.where(score.isnan(), -math.inf, score)
    # marked blocks first, in order of their index whatever their scores
    rank = torch.zeros_like(score) if always is None else always.double().expand(score.shape)
    score = torch.where(rank > 0, 0.0, score)
    B, H, nq, nk = score.shape
    out = torch.empty((B, H, nq, min(topk, nk)), dtype=torch.int32)
    for b in range(B):
        for h in range(H):
            for i in range(nq):
                rows = zip(rank[b, h, i].tolist(), score[b, h, i].tolist(), range(nk))
                best = sorted(rows, key=lambda r: (-r[0], -r[1], r[2]))[:topk]
                out[b, h, i] = torch.tensor(sorted(r[2] for r in best), dtype=torch.int32)
    return out


def sparse_reference(q, k, v, block_index, block_count=None, softmax_scale=None):
    """``(out, bound, lse, bound)``. A score, 128 products in fp32, is off by at
    most d = 130 U scale <|q|, |k|>, so a weight by exp(2 d) (numerator and sum);
    the weights are rounded to bf16 for the product with v (H of sum p |v|), exp2
    and the sums add a few U per key, and the output is rounded to bf16."""

    B, Sq, heads, D = q.shape
    Sk = k.shape[1]
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else softmax_scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full((B, heads, Sq), -math.inf, dtype=torch.float64)
    lse_bound = torch.zeros((B, heads, Sq), dtype=torch.float64)
    nk = -(-Sk // BLOCK_K)
    for b in range(B):
        for h in range(heads):
            qd, kd, vd = q[b, :, h].double(), k[b, :, h].double(), v[b, :, h].double()
            for i in range(block_index.shape[2]):
                ids = block_index[b, h, i].tolist()
                if block_count is not None:
                    ids = ids[: max(0, int(block_count[b, h, i]))]
                keys = [j for n in ids if 0 <= n < nk for j in range(n * BLOCK_K, min((n + 1) * BLOCK_K, Sk))]
                if not keys:
                    continue
                at = slice(i * BLOCK_Q, min((i + 1) * BLOCK_Q, Sq))
                kk, vv = kd[keys], vd[keys]
                s = qd[at] @ kk.t() * scale
                l = torch.logsumexp(s, -1, keepdim=True)
                p = torch.exp(s - l)
                d = (130 * U * scale * (qd[at].abs() @ kk.abs().t())).amax(-1, keepdim=True) + 8 * U * (1 + s.abs().amax(-1, keepdim=True))
                size = p @ vv.abs()
                o = p @ vv
                off = size * (H + torch.expm1(2 * d) + (len(keys) + 64) * U)
                out[b, at, h] = o
                bound[b, at, h] = off + H * (o.abs() + off) + 1e-37
                lse[b, h, at] = l.squeeze(-1)
                lse_bound[b, h, at] = (d + (len(keys) + 64) * U + 4 * U * l.abs()).squeeze(-1)
    return out, bound, lse, lse_bound

"""Plain PyTorch statements of every op.

These are the numerical contract (reference implementation/nnfunctions.py and
implementation/layers.py) written with differentiable torch operations.  They
run the CPU/gloo plumbing tier and serve as the fp32 oracle that the sm_100a
kernels are tested against; the GPU training path does not call them.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

__all__ = [
    "softmax", "silu", "cross_entropy", "gradient_clipping", "gradient_clippling", "sample_output",
    "dot_product_att", "rmsnorm_ref", "rope_tables", "apply_rope_ref", "attention_ref",
    "router_top2_ref", "swiglu_ref", "grouped_mm_ref", "log_softmax", "clip_gradient",
    "route_topk_ref", "gated_add_rmsnorm_ref", "quantize_fp8_ref", "dequantize_fp8_ref",
]


def softmax(x: torch.Tensor, dim_sum: int = -1, mask: torch.Tensor | None = None) -> torch.Tensor:
    """Max-subtracted softmax; an optional 0/1 mask multiplies the exponentials
    (reference nnfunctions.py:37-43)."""
    shifted = torch.exp(x - x.amax(dim=dim_sum, keepdim=True))
    if mask is not None:
        shifted = shifted * mask.to(shifted.dtype)
    return shifted / shifted.sum(dim=dim_sum, keepdim=True)


def log_softmax(x: torch.Tensor, dim: int = -1) -> torch.Tensor:
    shifted = x - x.amax(dim=dim, keepdim=True)
    return shifted - torch.log(torch.exp(shifted).sum(dim=dim, keepdim=True))


def silu(x: torch.Tensor) -> torch.Tensor:
    return x * torch.sigmoid(x)


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Mean token negative log-likelihood computed in fp32 (reference
    nnfunctions.py:56-64)."""
    logits = logits.float()
    logits = logits - logits.amax(dim=-1, keepdim=True)
    lse = torch.log(torch.exp(logits).sum(-1))
    picked = logits.gather(-1, targets.unsqueeze(-1)).squeeze(-1)
    return (lse - picked).mean()


def gradient_clipping(params, max_l2: float, eps: float = 1e-6) -> torch.Tensor:
    """Scale every ``.grad`` by ``max_l2 / (norm + eps)`` when the global L2 norm
    exceeds ``max_l2`` (reference nnfunctions.py:9-17); returns the norm."""
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        return torch.zeros(())
    norm = torch.sqrt(sum(torch.sum(g.float() ** 2) for g in grads))
    if norm > max_l2:
        scale = max_l2 / (norm + eps)
        for g in grads:
            g.mul_(scale.to(g.dtype))
    return norm


gradient_clippling = gradient_clipping  # the reference's spelling
clip_gradient = gradient_clipping


def sample_output(logits: torch.Tensor, t: float = 1.0, p: float = 0.0) -> torch.Tensor:
    """Temperature + nucleus sampling over ``[batch, vocab]`` logits: the most
    likely token always stays, further tokens stay while the running mass is
    below ``p`` (reference nnfunctions.py:66-81)."""
    prob = softmax(logits / t, dim_sum=-1)
    values, indices = torch.sort(prob, dim=-1, descending=True)
    running = torch.cumsum(values, dim=-1)
    keep = (running < p).to(values.dtype)
    keep[:, 0] = 1.0
    choice = torch.multinomial(values * keep, num_samples=1)
    return torch.gather(indices, -1, choice)


def dot_product_att(k, q, v, mask=None):
    """Naive attention with the reference's argument order (k, q, v)."""
    scores = torch.einsum("...ik,...jk->...ij", q, k) / math.sqrt(k.shape[-1])
    return torch.einsum("...ki,...ij->...kj", softmax(scores, -1, mask), v)


def rmsnorm_ref(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    xf = x.float()
    normed = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (normed * weight.float()).to(x.dtype)


def rope_tables(theta: float, head_dim: int, max_seq_len: int, device=None):
    """``cos, sin`` of shape ``[seq, head_dim/2]``.  Pair ``i`` (elements ``2i``
    and ``2i+1``, adjacent) turns by ``pos · theta^(-2i/head_dim)`` (reference
    layers.py:275-279 with ``i`` counted from 1: ``theta^((2-2i)/d)``)."""
    half = torch.arange(0, head_dim // 2, dtype=torch.float32, device=device)
    inv_freq = theta ** (-2.0 * half / head_dim)
    angles = torch.arange(max_seq_len, dtype=torch.float32, device=device)[:, None] * inv_freq[None, :]
    return torch.cos(angles), torch.sin(angles)


def apply_rope_ref(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate adjacent pairs of the last dim; ``x`` is ``[..., seq, head_dim]``
    and the tables are ``[seq, head_dim/2]``.  ``(a, b) -> (a·cos − b·sin,
    a·sin + b·cos)`` in fp32."""
    pairs = x.float().unflatten(-1, (-1, 2))
    a, b = pairs[..., 0], pairs[..., 1]
    rotated = torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1)
    return rotated.flatten(-2).to(x.dtype)


def attention_ref(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos=None, sin=None,
                  causal: bool = True) -> torch.Tensor:
    """GQA attention on ``[B, S, H, hd]`` tensors with optional RoPE on q and k;
    returns ``[B, S, Hq, hd]``."""
    qh, kh, vh = (t.transpose(1, 2) for t in (q, k, v))
    if cos is not None:
        seq = qh.shape[-2]
        qh = apply_rope_ref(qh, cos[:seq], sin[:seq])
        kh = apply_rope_ref(kh, cos[:seq], sin[:seq])
    ratio = qh.shape[1] // kh.shape[1]
    if ratio > 1:
        kh = kh.repeat_interleave(ratio, dim=1)
        vh = vh.repeat_interleave(ratio, dim=1)
    out = F.scaled_dot_product_attention(qh, kh, vh, is_causal=causal)
    return out.transpose(1, 2)


def router_top2_ref(logits: torch.Tensor, k: int = 2):
    """Softmax over experts, top-k, renormalise the kept probabilities
    (reference layers.py:126-127,142).  Returns ``(weights fp32 [T,k], idx [T,k])``."""
    probs = softmax(logits.float(), dim_sum=-1)
    top, idx = probs.topk(k, dim=-1)
    return top / top.sum(dim=-1, keepdim=True), idx


FLT_MIN, FLT_MAX = 2.0 ** -126, torch.finfo(torch.float32).max       # of the numbers that kernels take in fp32


def route_topk_ref(logits: torch.Tensor, k: int, score: str = "softmax", bias: torch.Tensor | None = None, groups: int = 1,
                   top_groups: int | None = None, group_score: int = 1, renormalize: bool = True, scale: float = 1.0):
    """``(weights fp32 [T, k], idx int64 [T, k])`` of ``logits [T, E]``.  Experts are chosen by their scores plus ``bias``
    (without one: by their logits), best first, the lower index first where two are equal, after a choice of the
    ``top_groups`` best of ``groups`` runs of experts by their best key or the sum of their two best.  The weights are the
    scores without the bias.  NaN and -inf mask an expert: it is chosen after all others of its groups, with weight 0.
    What decides the choice is evaluated in fp64."""
    tokens, experts = logits.shape
    top_groups = groups if top_groups is None else top_groups
    wide = logits if logits.dtype == torch.float64 else logits.float()
    x = torch.where(torch.isnan(wide), -math.inf, wide).clamp(max=FLT_MAX)
    dead = torch.isinf(x)

    def scores(t, off):
        """Scores of ``t``, zero where ``off``; what is masked takes no part in a gradient either."""
        safe = t.masked_fill(off, 0.0)
        if score == "sigmoid":
            return torch.sigmoid(safe) * (~off).to(t.dtype)
        top = t.detach().masked_fill(off, -math.inf).amax(-1, keepdim=True)
        part = torch.exp(safe - top.masked_fill(torch.isinf(top), 0.0)).masked_fill(off, 0.0)
        total = part.sum(-1, keepdim=True)
        return part / torch.where(total == 0, torch.ones_like(total), total)

    with torch.no_grad():
        key = x.double()
        grouped = top_groups < groups
        compared = key
        if bias is not None or (grouped and group_score == 2):
            s = key
            if score == "sigmoid":
                s = 1.0 / (1.0 + torch.exp(-key))
            else:
                s = scores(key, dead)
            compared = (s if bias is None else s + bias.double()).masked_fill(dead, -math.inf)
            if bias is not None:
                key = compared
        level = torch.ones_like(key)
        if grouped:
            best = compared.view(tokens, groups, experts // groups).sort(-1, descending=True).values
            value = best[..., 0]
            if group_score == 2:
                value = value + best[..., 1].masked_fill(torch.isinf(best[..., 1]), 0.0)
            order = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :top_groups]
            chosen = torch.zeros_like(value).scatter_(1, order, 1.0)
            level = chosen.repeat_interleave(experts // groups, dim=1)
        # experts of other groups last, masked ones of the chosen groups before them
        rank = torch.sort(key, dim=-1, descending=True, stable=True).indices
        rank = rank.gather(1, torch.sort(level.gather(1, rank), dim=-1, descending=True, stable=True).indices)
        idx = rank[:, :k]
    off = dead.gather(1, idx)
    if renormalize:
        picked = x.gather(1, idx).masked_fill(off, 0.0)
        logs = F.logsigmoid(picked) if score == "sigmoid" else picked
        top = logs.detach().masked_fill(off, -math.inf).amax(-1, keepdim=True)
        part = torch.exp(logs - top.masked_fill(torch.isinf(top), 0.0)).masked_fill(off, 0.0)
        total = part.sum(-1, keepdim=True)
        weights = part / torch.where(total == 0, torch.ones_like(total), total)
    else:
        weights = scores(x, dead).gather(1, idx)
    return weights * scale, idx


def gated_add_rmsnorm_ref(x: torch.Tensor, delta: torch.Tensor, delta_weight: torch.Tensor, weight: torch.Tensor,
                          gate: torch.Tensor | None = None, residual_scale: float = 1.0, eps: float = 1e-5):
    """``s = residual_scale x + gate rmsnorm(delta) delta_weight`` and ``rmsnorm(s) weight``, in fp32 (fp64 stays); the second
    norm sees the sum before it is rounded."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32

    def norm(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps)

    branch = norm(delta.to(wide)) * delta_weight.to(wide)
    if gate is not None:
        branch = branch * gate.to(wide)
    summed = x.to(wide) * residual_scale + branch
    return summed.to(x.dtype), (norm(summed) * weight.to(wide)).to(x.dtype)


E4M3_MAX = 448.0
SMALLEST_FP8_SCALE = 2.0 ** -120


def _fp8_blocks(x: torch.Tensor, block_rows: int) -> torch.Tensor:
    x = F.pad(x.float(), (0, -x.shape[1] % 128, 0, -x.shape[0] % block_rows))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)


def quantize_fp8_ref(x: torch.Tensor, block_rows: int = 1):
    """e4m3 values of ``x [M, K]`` and one fp32 scale for each block of ``block_rows`` x 128 of them: ``max(largest / 448,
    2^-120)``, so that the largest value becomes 448, the largest number of the type."""
    rows, cols = x.shape
    blocks = _fp8_blocks(x, block_rows)
    most = torch.where(torch.isnan(blocks), 0.0, blocks.abs()).amax((1, 3))
    # by a tensor: a division by a number is a product with its rounded reciprocal on a GPU, which half of the scales differ by
    scales = (most / torch.full_like(most, E4M3_MAX)).clamp(min=SMALLEST_FP8_SCALE)
    values = (blocks / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return values.view(blocks.shape[0] * block_rows, blocks.shape[2] * 128)[:rows, :cols].contiguous(), scales


def dequantize_fp8_ref(values: torch.Tensor, scales: torch.Tensor, block_rows: int = 1) -> torch.Tensor:
    """The fp32 numbers that ``quantize_fp8`` stands for."""
    rows, cols = values.shape
    blocks = _fp8_blocks(values, block_rows) * scales[:, None, :, None]
    return blocks.view(blocks.shape[0] * block_rows, blocks.shape[2] * 128)[:rows, :cols]


def swiglu_ref(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return (silu(gate.float()) * up.float()).to(gate.dtype)


def grouped_mm_ref(x: torch.Tensor, w: torch.Tensor, offs: torch.Tensor) -> torch.Tensor:
    """``out[rows of group e] = x[rows of group e] @ w[e].T`` with ``offs`` the
    cumulative row ends; rows past ``offs[-1]`` are zero.  Loop form for tests."""
    out = x.new_zeros(x.shape[0], w.shape[1])
    start = 0
    for e, end in enumerate(offs.tolist()):
        if end > start:
            out[start:end] = x[start:end] @ w[e].to(x.dtype).T
        start = end
    return out

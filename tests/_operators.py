"""Operators of the blocks in 64 bits, written from their definitions one value at a time or one row at a time, for the tests of
the statements and of the kernels."""
import math

import torch


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=None, group_score=1, renormalize=True, scale=1.0):
    """Choice and weights row by row in Python's floats; logits of any type."""
    top_groups = groups if top_groups is None else top_groups
    bias = None if bias is None else bias.tolist()
    all_weights, all_idx = [], []
    for row in logits.double().tolist():
        x = [-math.inf if math.isnan(v) else min(v, 3.4028234663852886e38) for v in row]
        top = max(x)
        if score == "sigmoid":
            s = [0.0 if v == -math.inf else 1.0 / (1.0 + math.exp(-v)) if v > -700 else math.exp(max(v, -745.0)) for v in x]
        else:
            e = [0.0 if v == -math.inf else math.exp(v - top) for v in x]
            s = [v / sum(e) if sum(e) else 0.0 for v in e]
        scored = [-math.inf if v == -math.inf else p + (bias[i] if bias else 0.0) for i, (v, p) in enumerate(zip(x, s))]
        key = scored if bias else x
        size = len(x) // groups
        values = []
        for g in range(groups):
            best = sorted((scored if group_score == 2 else key)[g * size:(g + 1) * size], reverse=True)
            values.append(best[0] + (best[1] if group_score == 2 and best[1] > -math.inf else 0.0))
        kept = set(sorted(range(groups), key=lambda g: (-values[g], g))[:top_groups])
        idx = sorted((i for i in range(len(x)) if i // size in kept), key=lambda i: (-key[i], i))[:k]
        if renormalize:
            logs = [x[i] if score == "softmax" else -math.log1p(math.exp(-x[i])) if x[i] > -700 else x[i] for i in idx]
            most = max(logs)
            w = [0.0 if v == -math.inf else math.exp(v - most) for v in logs]
            w = [v / sum(w) if sum(w) else 0.0 for v in w]
        else:
            w = [s[i] for i in idx]
        all_weights.append([scale * v for v in w])
        all_idx.append(idx)
    return torch.tensor(all_weights, dtype=torch.float64).view(len(logits), k), torch.tensor(all_idx).view(len(logits), k)


def route_gradient(logits, idx, dweights, score, renormalize, scale):
    """Gradient of ``(weights * dweights).sum()`` for a choice, by differentiation; rows without a live expert have none."""
    x = logits.double()
    dead = torch.isnan(x) | (x == -math.inf)
    x = x.masked_fill(dead, 0.0).requires_grad_()
    live = (~dead).double()
    if score == "sigmoid":
        s = torch.sigmoid(x) * live
    else:
        e = torch.exp(x - x.detach().amax(1, keepdim=True)) * live
        total = e.sum(1, keepdim=True)
        s = e / (total + (total == 0).double())
    w = s.gather(1, idx)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = w / (total + (total == 0).double())
    return torch.autograd.grad(w * scale, x, dweights.double())[0] * live


def gated_norm(x, delta, delta_weight, weight, gate, residual_scale, eps):
    def norm(t, w):
        return t / torch.sqrt((t * t).sum(-1, keepdim=True) / t.shape[-1] + eps) * w

    branch = norm(delta, delta_weight)
    summed = x * residual_scale + (branch if gate is None else branch * gate)
    return summed, norm(summed, weight)


def quantize(x, block_rows):
    """fp32 scales by their definition, block by block, and the e4m3 values as numbers, in 64 bits."""
    rows, cols = x.shape
    scales = torch.empty((rows + block_rows - 1) // block_rows, (cols + 127) // 128)
    values = torch.empty(rows, cols, dtype=torch.float64)
    x = x.float().cpu()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            part = (slice(i * block_rows, (i + 1) * block_rows), slice(j * 128, (j + 1) * 128))
            s = torch.clamp(x[part].abs().max() / 448.0, min=2.0 ** -120)
            scales[i, j] = s
            values[part] = (x[part] / s).clamp(-448, 448).to(torch.float8_e4m3fn).double()
    return values, scales


def spread(scales, rows, cols, block_rows):
    """The factor of each value."""
    return scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]

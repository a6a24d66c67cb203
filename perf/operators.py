"""Operators around and inside the blocks of a mixture-of-experts decoder, as a program calls them:

``route``   choice of experts: softmax or sigmoid scores, a balance bias that takes part in the choice alone, a choice among
            groups of experts first, top-k, weights renormalised or not; and the gradient of the logits.
``norm``    the norm of a block's output, its gate, the residual sum with its scale, and the norm in front of the next block;
            and the gradients of all of them.
``fp8``     products of 8-bit floating point values with one scale for each block of 128: of values that are quantised
            already, of a linear layer, and of a linear layer's training step.

``listed`` are the cases, ``draw`` gives more of the same ranges.  ``run`` computes one of them in elementary operations,
or, where ``own`` is set, by the package's operators.
"""
import math

import torch

own = False

FLT_MAX = 3.4028234663852886e38
E4M3_MAX = 448.0
SMALLEST_SCALE = 2.0 ** -120
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one decoding step of eight sequences in front of 256 experts: the time of a launch counts
        dict(name="route_decode", op="route", tokens=8, experts=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4,
             group_score=2, renormalize=True, scale=2.5, masked=0.0, dtype="fp32", backward=False),
        # a training microbatch in front of many small experts: sigmoid scores, balance bias, groups
        dict(name="route_sigmoid_groups_train", op="route", tokens=32768, experts=256, k=8, score="sigmoid", bias=True, groups=8,
             top_groups=4, group_score=2, renormalize=True, scale=2.5, masked=0.0, dtype="fp32", backward=True),
        # softmax scores that are not renormalised, so that every logit has a gradient; logits as a bf16 product leaves them
        dict(name="route_softmax_train", op="route", tokens=65536, experts=64, k=6, score="softmax", bias=False, groups=1,
             top_groups=1, group_score=1, renormalize=False, scale=1.0, masked=0.0, dtype="bf16", backward=True),
        # a ragged batch, groups by their best expert, some experts masked out by an infinite logit
        dict(name="route_masked_ragged", op="route", tokens=5003, experts=160, k=6, score="softmax", bias=False, groups=8,
             top_groups=3, group_score=1, renormalize=True, scale=1.0, masked=0.1, dtype="fp32", backward=False),
        # one decoding step of four sequences at the width of the run configuration
        dict(name="norm_decode", op="norm", batch=4, seq=1, width=4096, gate="channel", residual_scale=1.0, dtype="bf16",
             backward=False),
        # a training microbatch of two sequences of 8192 tokens at that width, with a learned gate for each channel
        dict(name="norm_channel_train", op="norm", batch=2, seq=8192, width=4096, gate="channel", residual_scale=1.0,
             dtype="bf16", backward=True),
        # a gate for each sequence (modulation by a condition), a scaled residual path, odd lengths
        dict(name="norm_sequence_train", op="norm", batch=24, seq=331, width=2048, gate="sequence", residual_scale=0.7,
             dtype="bf16", backward=True),
        # inference over a long prompt with a gate for each value
        dict(name="norm_full_prefill", op="norm", batch=1, seq=20011, width=5120, gate="full", residual_scale=1.0, dtype="bf16",
             backward=False),
        # one decoding step of 16 sequences, operands quantised before
        dict(name="fp8_product_decode", op="fp8", kind="product", rows=16, outputs=4096, inputs=4096),
        # a product whose sizes fill no tile, operands quantised before
        dict(name="fp8_product_odd", op="fp8", kind="product", rows=1003, outputs=1544, inputs=2000),
        # the fused query, key and value projection of two sequences of 8192 tokens, weight quantised before
        dict(name="fp8_linear_prefill", op="fp8", kind="linear", rows=16384, outputs=6144, inputs=4096),
        # the training step of one feed-forward projection: activations, weight and gradient quantised within the step
        dict(name="fp8_linear_train", op="fp8", kind="train", rows=8192, outputs=14336, inputs=4096),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("route", "norm", "fp8"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        per_group = _log(rng, 2 if groups > 1 else 4, 512 // groups)
        experts = groups * per_group
        group_score = rng.choice((1, 2)) if groups > 1 else 1
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(16, top_groups * per_group))
        tokens = max(1, min(_log(rng, 1, 65536), 32768 * 256 // experts))
        # one expert whose weight is renormalised has weight 1 whatever its score: nothing to differentiate
        renormalize = k > 1 and rng.random() < 0.6
        return dict(op=op, tokens=tokens, experts=experts, k=k, score=rng.choice(("softmax", "sigmoid")),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, group_score=group_score,
                    renormalize=renormalize, scale=rng.choice((1.0, 2.5)), masked=rng.choice((0.0, 0.0, 0.2)),
                    dtype=rng.choice(("fp32", "bf16", "fp16")), backward=rng.random() < 0.5)
    if op == "norm":
        width = _log(rng, 64, 8192)
        if rng.random() < 0.8:
            width = (width + 7) // 8 * 8
        room = 16384 * 4096 // width
        seq = min(_log(rng, 1, 16384), room)
        batch = max(1, min(_log(rng, 1, 64), room // seq))
        return dict(op=op, batch=batch, seq=seq, width=width, gate=rng.choice(("none", "channel", "sequence", "token", "full")),
                    residual_scale=rng.choice((1.0, 0.7)), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                    backward=rng.random() < 0.5)
    kind = rng.choice(("product", "linear", "train"))
    step = 32 if kind == "train" else rng.choice((16, 64))
    rows, outputs, inputs = _log(rng, 1, 16384), _log(rng, 64, 14336), _log(rng, 64, 14336)
    outputs, inputs = (max(step, v // step * step) for v in (outputs, inputs))
    most = 8192 * 14336 * 4096
    rows = max(1, min(rows, most // (outputs * inputs)))
    return dict(op=op, kind=kind, rows=rows, outputs=outputs, inputs=inputs)


# ------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare(case, seed):
    gen = _generator(seed)

    def normal(*shape, scale=1.0, dtype="fp32"):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(TYPES[dtype])

    state = {"case": case}
    if case["op"] == "route":
        tokens, experts = case["tokens"], case["experts"]
        logits = normal(tokens, experts) + normal(experts, scale=0.5)            # some experts are liked more than others
        if case["masked"]:
            out = torch.rand(experts, device="cuda", generator=gen) < case["masked"]
            logits = logits.masked_fill(out, -math.inf)
        state["logits"] = logits.to(TYPES[case["dtype"]])
        state["bias"] = normal(experts, scale=0.05) if case["bias"] else None
        state["dweights"] = normal(tokens, case["k"])
        return state
    if case["op"] == "norm":
        batch, seq, width, dtype = case["batch"], case["seq"], case["width"], case["dtype"]
        shape = {"none": None, "channel": (width,), "sequence": (batch, 1, width), "token": (batch, seq, 1),
                 "full": (batch, seq, width)}[case["gate"]]
        # the residual stream is larger than what a block adds to it
        state["x"] = normal(batch, seq, width, scale=2.0, dtype=dtype)
        state["delta"] = normal(batch, seq, width, scale=0.5, dtype=dtype)
        state["delta_weight"] = 1.0 + normal(width, scale=0.1)
        state["weight"] = 1.0 + normal(width, scale=0.1)
        state["gate"] = None if shape is None else normal(*shape, scale=0.3, dtype=dtype)
        if case["backward"]:
            state["dsummed"] = normal(batch, seq, width, dtype=dtype)
            state["dnormed"] = normal(batch, seq, width, dtype=dtype)
        return state
    rows, outputs, inputs = case["rows"], case["outputs"], case["inputs"]
    channels = torch.exp(normal(inputs, scale=0.7))                              # some channels are much larger than others
    x = (torch.randn(rows, inputs, device="cuda", generator=gen) * channels).to(torch.bfloat16)
    weight = normal(outputs, inputs, scale=inputs ** -0.5, dtype="bf16")
    if case["kind"] == "product":
        state["a"], state["a_scales"] = _quantize(x, 1)
        state["b"], state["b_scales"] = _quantize(weight, 128)
    elif case["kind"] == "linear":
        state["x"] = x
        state["b"], state["b_scales"] = _quantize(weight, 128)
        state["weight"] = weight
    else:
        state["x"], state["weight"] = x, weight
        state["dy"] = normal(rows, outputs, scale=0.01, dtype="bf16")
    return state


# ------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"route": _run_route, "norm": _run_norm, "fp8": _run_fp8}[case["op"]](case, state)


def _run_route(case, state):
    if own:
        from b200moe import ops
        logits = state["logits"].detach().requires_grad_(case["backward"])
        weights, idx = ops.route_topk(logits, case["k"], score=case["score"], bias=state["bias"], groups=case["groups"],
                                      top_groups=case["top_groups"], group_score=case["group_score"],
                                      renormalize=case["renormalize"], scale=case["scale"])
        if not case["backward"]:
            return {"weights": weights, "idx": idx}
        (dlogits,) = torch.autograd.grad(weights, logits, state["dweights"])
        return {"weights": weights.detach(), "idx": idx, "dlogits": dlogits}
    x, idx = _route_choice(case, state["logits"], state["bias"])
    weights, dlogits = _route_weights(case, x.float(), idx, state["dweights"])
    if not case["backward"]:
        return {"weights": weights, "idx": idx}
    return {"weights": weights, "idx": idx, "dlogits": dlogits.to(state["logits"].dtype)}


def _route_choice(case, logits, bias):
    """The chosen experts, best first, the lowest index first where two are equal.  NaN counts as masked, infinity as the
    largest number.  Scores that are compared with one another are held in 64 bits."""
    x = torch.where(torch.isnan(logits), -math.inf, logits.float()).clamp(max=FLT_MAX)
    tokens, experts = x.shape
    groups, k = case["groups"], case["k"]
    key = x
    if bias is not None or (groups > 1 and case["group_score"] > 1):
        wide = x.double()
        if case["score"] == "sigmoid":
            score = 1.0 / (1.0 + torch.exp(-wide))
        else:
            top = wide.amax(1, keepdim=True)
            part = torch.exp(wide - torch.where(torch.isinf(top), 0.0, top))
            score = part / part.sum(1, keepdim=True).clamp(min=1e-300)
        compared = score if bias is None else score + bias.double()
        compared = torch.where(torch.isinf(wide), -math.inf, compared)
        if bias is not None:
            key = compared
    candidates = torch.arange(experts, device=x.device).expand(tokens, experts)
    if groups > 1 and case["top_groups"] < groups:
        size = experts // groups
        if case["group_score"] == 1:
            value = key.view(tokens, groups, size).amax(2)
        else:
            best = compared.view(tokens, groups, size).topk(2, dim=2).values
            value = torch.where(torch.isinf(best[..., 0]), -math.inf, torch.where(torch.isinf(best), 0.0, best).sum(2))
        chosen = torch.sort(value, dim=1, descending=True, stable=True).indices[:, :case["top_groups"]].sort(1).values
        candidates = (chosen.unsqueeze(2) * size + torch.arange(size, device=x.device)).view(tokens, -1)
        key = key.gather(1, candidates)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    return x, candidates.gather(1, order)


def _route_weights(case, x, idx, dweights):
    """The weights of the chosen experts and the gradient of the logits, from the formulas."""
    scale, picked = case["scale"], x.gather(1, idx)
    dead = torch.isinf(picked)
    if case["score"] == "sigmoid":
        rest = torch.sigmoid(-picked)                                            # 1 - score
        if case["renormalize"]:
            logs = torch.minimum(picked, torch.zeros_like(picked)) - torch.log1p(torch.exp(-picked.abs()))
            weights = _softmax(logs.masked_fill(dead, -math.inf))
        else:
            weights = torch.sigmoid(picked)
    elif case["renormalize"]:
        weights = _softmax(picked)
    else:
        probs = _softmax(x)
        weights = probs.gather(1, idx)
    if not case["backward"]:
        return weights * scale, None
    part = dweights * scale
    if case["renormalize"]:
        part = part - (part * weights).sum(1, keepdim=True)
    part = part * weights
    if case["score"] == "sigmoid":
        part = part * rest
    dlogits = torch.zeros_like(x).scatter(1, idx, part)
    if case["score"] == "softmax" and not case["renormalize"]:
        dlogits = dlogits - probs * part.sum(1, keepdim=True)
    return weights * scale, dlogits


def _softmax(x):
    """Along dimension 1; zeros where all of a row is masked."""
    top = x.amax(1, keepdim=True)
    part = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = part.sum(1, keepdim=True)
    return part / torch.where(total == 0, torch.ones_like(total), total)


EPS = 1e-5


def _run_norm(case, state):
    names = ("x", "delta", "delta_weight", "weight", "gate")
    if own:
        from b200moe import ops
        x, delta, delta_weight, weight, gate = (None if state[n] is None else
                                                state[n].detach().requires_grad_(case["backward"]) for n in names)
        summed, normed = ops.gated_add_rmsnorm(x, delta, delta_weight, weight, gate=gate,
                                               residual_scale=case["residual_scale"], eps=EPS)
        out = {"summed": summed.detach(), "normed": normed.detach()}
        if case["backward"]:
            leaves = [t for t in (x, delta, delta_weight, weight, gate) if t is not None]
            grads = torch.autograd.grad((summed, normed), leaves, (state["dsummed"], state["dnormed"]))
            out.update(zip(("dx", "ddelta", "ddelta_weight", "dweight", "dgate"), grads))
        return out
    dtype = TYPES[case["dtype"]]
    x, delta, delta_weight, weight, gate = (None if state[n] is None else state[n].float() for n in names)
    delta_rstd = torch.rsqrt(delta.square().mean(-1, keepdim=True) + EPS)
    branch_hat = delta * delta_rstd
    branch = branch_hat * delta_weight
    summed = x * case["residual_scale"] + (branch if gate is None else branch * gate)
    rstd = torch.rsqrt(summed.square().mean(-1, keepdim=True) + EPS)
    hat = summed * rstd                                                          # of the sum before it is rounded
    out = {"summed": summed.to(dtype), "normed": (hat * weight).to(dtype)}
    if case["backward"]:
        dnormed, dsum = state["dnormed"].float(), state["dsummed"].float()
        out["dweight"] = (dnormed * hat).sum((0, 1))
        dhat = dnormed * weight
        dsum = dsum + rstd * (dhat - hat * (dhat * hat).mean(-1, keepdim=True))
        out["dx"] = (dsum * case["residual_scale"]).to(dtype)
        dbranch = dsum
        if gate is not None:
            dgate = dsum * branch
            dims = {"channel": (0, 1), "sequence": (1,), "token": (2,), "full": ()}[case["gate"]]
            if dims:
                dgate = dgate.sum(dims, keepdim=case["gate"] != "channel")
            out["dgate"] = dgate.to(dtype)
            dbranch = dsum * gate
        out["ddelta_weight"] = (dbranch * branch_hat).sum((0, 1))
        dhat = dbranch * delta_weight
        out["ddelta"] = (delta_rstd * (dhat - branch_hat * (dhat * branch_hat).mean(-1, keepdim=True))).to(dtype)
    return out


def _blocks(x, block_rows):
    """``x`` filled up with zeros to whole blocks: ``[row blocks, block_rows, column blocks, 128]``."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % 128, 0, -rows % block_rows))
    return x.view(x.shape[0] // block_rows, block_rows, x.shape[1] // 128, 128)


def _quantize(x, block_rows):
    """e4m3 values and one fp32 scale for each block of ``block_rows`` x 128 values: the largest becomes 448."""
    rows, cols = x.shape
    blocks = _blocks(x, block_rows)
    scales = (blocks.abs().amax((1, 3)) / E4M3_MAX).clamp(min=SMALLEST_SCALE)
    values = (blocks / scales[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return values.view(blocks.shape[0] * block_rows, -1)[:rows, :cols].contiguous(), scales


def _dequantize(values, scales, block_rows):
    rows, cols = values.shape
    return (_blocks(values, block_rows) * scales.float()[:, None, :, None]).view(-1, (cols + 127) // 128 * 128)[:rows, :cols]


def _run_fp8(case, state):
    kind = case["kind"]
    if own:
        from b200moe import ops
        if kind == "product":
            return ops.matmul_fp8(state["a"], state["a_scales"], state["b"], state["b_scales"])
        if kind == "linear":
            return ops.linear_fp8(state["x"], state["weight"], weight_fp8=(state["b"], state["b_scales"]))
        x, weight = (state[n].detach().requires_grad_() for n in ("x", "weight"))
        y = ops.linear_fp8(x, weight)
        dx, dweight = torch.autograd.grad(y, (x, weight), state["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dweight}
    if kind == "product":
        return (_dequantize(state["a"], state["a_scales"], 1) @ _dequantize(state["b"], state["b_scales"], 128).t()).bfloat16()
    x = _dequantize(*_quantize(state["x"], 1), 1)
    if kind == "linear":
        return (x @ _dequantize(state["b"], state["b_scales"], 128).t()).bfloat16()
    weight = _dequantize(*_quantize(state["weight"], 128), 128)
    dy = _dequantize(*_quantize(state["dy"], 1), 1)
    return {"y": (x @ weight.t()).bfloat16(), "dx": (dy @ weight).bfloat16(),
            "dweight": (state["dy"].float().t() @ state["x"].float()).bfloat16()}


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "route":
        tokens, experts, k, size = case["tokens"], case["experts"], case["k"], SIZE[case["dtype"]]
        logits, choice = tokens * experts * size, tokens * k * (4 + 8)
        bytes_ = logits + choice + (4 * experts if case["bias"] else 0)
        flops = 4 * tokens * experts
        if case["backward"]:
            bytes_ += logits + tokens * k * 4
            flops += 4 * tokens * experts
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "norm":
        values, width, size = case["batch"] * case["seq"] * case["width"], case["width"], SIZE[case["dtype"]]
        gate = size * {"none": 0, "channel": width, "sequence": case["batch"] * width, "token": case["batch"] * case["seq"],
                       "full": values}[case["gate"]]
        bytes_ = 4 * values * size + gate + 8 * width
        if case["backward"]:
            bytes_ += 4 * values * size + gate + 8 * width                       # two gradients in, two out
        return {"bytes": bytes_, "flops": values * (35 if case["backward"] else 10)}
    rows, outputs, inputs = case["rows"], case["outputs"], case["inputs"]
    blocks = (inputs + 127) // 128
    scales = 4 * (rows * blocks + (outputs + 127) // 128 * blocks)
    product = 2 * rows * outputs * inputs
    if case["kind"] == "product":
        return {"bytes": rows * inputs + outputs * inputs + scales + 2 * rows * outputs, "flops": product}
    if case["kind"] == "linear":
        return {"bytes": 2 * rows * inputs + outputs * inputs + 4 * ((outputs + 127) // 128) * blocks + 2 * rows * outputs,
                "flops": product}
    return {"bytes": 2 * (2 * rows * inputs + 2 * outputs * inputs + 2 * rows * outputs), "flops": 3 * product}


# ------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"route": _exact_route, "norm": _exact_norm, "fp8": _exact_fp8}[case["op"]](case, state)


def _exact_route(case, state):
    """Choices by ranks: an expert's rank is the number of those in front of it.  Gradients by differentiation."""
    raw = state["logits"].double()
    dead = torch.isnan(raw) | (raw == -math.inf)
    x = raw.masked_fill(dead, 0.0).clamp(max=FLT_MAX).requires_grad_()
    live = (~dead).double()
    if case["score"] == "sigmoid":
        score = torch.sigmoid(x) * live
    else:
        part = torch.exp(x - x.detach().masked_fill(dead, -math.inf).amax(1, keepdim=True).clamp(min=-FLT_MAX)) * live
        score = part / part.sum(1, keepdim=True).clamp(min=1e-300)
    tokens, experts = x.shape
    groups, k, size = case["groups"], case["k"], experts // case["groups"]
    with torch.no_grad():
        biased = score if state["bias"] is None else score + state["bias"].double()
        # without a bias the order of the scores is that of the logits
        key = (x if state["bias"] is None else biased).masked_fill(dead, -math.inf)
        allowed = torch.ones_like(dead)
        if case["top_groups"] < groups:
            if case["group_score"] == 1:
                value = key.view(tokens, groups, size).max(2).values
            else:
                low = biased.masked_fill(dead, -math.inf).view(tokens, groups, size).sort(2, descending=True).values[..., :2]
                value = torch.nan_to_num(low[..., 1], neginf=0.0) + low[..., 0]
            first = value.unsqueeze(2) > value.unsqueeze(1)                       # [t, i, j]: i in front of j
            number = torch.arange(groups, device=x.device)
            first |= (value.unsqueeze(2) == value.unsqueeze(1)) & (number[:, None] < number[None, :])
            allowed = (first.sum(1) < case["top_groups"]).repeat_interleave(size, 1)
        level = allowed.double() * 2 - dead.double()                              # masked experts of chosen groups, then the others
        idx = torch.empty(tokens, k, dtype=torch.int64, device=x.device)
        taken = torch.zeros_like(dead)
        for j in range(k):
            best_level = level.masked_fill(taken, -9).amax(1, keepdim=True)
            here = (level == best_level) & ~taken
            value = key.masked_fill(~here, -math.inf)
            at = ((value == value.amax(1, keepdim=True)) & here).to(torch.uint8).argmax(1, keepdim=True)
            idx[:, j:j + 1] = at
            taken.scatter_(1, at, True)
    if case["renormalize"]:
        logs = torch.nn.functional.logsigmoid(x) if case["score"] == "sigmoid" else x
        logs = logs.gather(1, idx)
        off = dead.gather(1, idx)
        part = torch.exp(logs - logs.detach().masked_fill(off, -math.inf).amax(1, keepdim=True).clamp(min=-FLT_MAX)) * (~off).double()
        weights = part / part.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        weights = score.gather(1, idx)
    weights = weights * case["scale"]
    out = {"weights": weights.detach(), "idx": idx}
    if case["backward"]:
        (dx,) = torch.autograd.grad(weights, x, state["dweights"].double())
        out["dlogits"] = dx * live
    return out


def _exact_norm(case, state):
    leaves = {n: state[n].double().requires_grad_(case["backward"]) for n in ("x", "delta", "delta_weight", "weight", "gate")
              if state[n] is not None}

    def norm(t, weight):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * weight

    branch = norm(leaves["delta"], leaves["delta_weight"])
    summed = leaves["x"] * case["residual_scale"] + (branch * leaves["gate"] if "gate" in leaves else branch)
    normed = norm(summed, leaves["weight"])
    out = {"summed": summed.detach(), "normed": normed.detach()}
    if case["backward"]:
        grads = torch.autograd.grad((summed, normed), list(leaves.values()),
                                    (state["dsummed"].double(), state["dnormed"].double()))
        out.update({f"d{n}": g for n, g in zip(leaves, grads)})
    return out


def _exact_fp8(case, state):
    def spread(scales, rows, cols, block_rows):
        return scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]

    def through_8_bits(x, block_rows):
        rows, cols = x.shape
        scales = torch.empty((rows + block_rows - 1) // block_rows, (cols + 127) // 128, dtype=torch.float64, device=x.device)
        for j in range(scales.shape[1]):
            most = x[:, 128 * j:128 * j + 128].abs().amax(1).double()
            most = torch.nn.functional.pad(most, (0, -rows % block_rows)).view(-1, block_rows).amax(1)
            scales[:, j] = torch.clamp(most / E4M3_MAX, min=SMALLEST_SCALE)
        factor = spread(scales.float(), rows, cols, block_rows)
        return (x.double() / factor).to(torch.float8_e4m3fn).double() * factor

    def back(name, block_rows):
        return state[name].double() * spread(state[f"{name}_scales"], *state[name].shape, block_rows)

    if case["kind"] == "product":
        return back("a", 1) @ back("b", 128).t()
    x = through_8_bits(state["x"], 1)
    if case["kind"] == "linear":
        return x @ back("b", 128).t()
    weight, dy = through_8_bits(state["weight"], 128), through_8_bits(state["dy"], 1)
    return {"y": x @ weight.t(), "dx": dy @ weight, "dweight": state["dy"].double().t() @ state["x"].double()}

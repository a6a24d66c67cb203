"""Routing, gated residual norm and 8-bit products on the GPU where equal, close, far and empty operands meet."""
import itertools

import pytest
import torch

import _operators as want
from b200moe import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _native():
    from b200moe.ops import native
    native.require()
    torch.manual_seed(12)
    yield
    native.check_status()


# ------------------------------------------------------------------------------ choice among equal and close experts
def _close_rows(E, front, others):
    """A row for each order of the logits ``front``, next to each other and spread over the experts; the others are far behind."""
    orders = sorted(set(itertools.permutations(front))) if len(front) <= 4 else [tuple(front), tuple(reversed(front))]
    rows = []
    for order in orders:
        for step in sorted({1, max(1, (E - 1) // max(len(front) - 1, 1))}):
            row = [others - 0.25 * i / E for i in range(E)]
            for i, v in enumerate(order):
                row[i * step] = v
            rows.append(row)
    return torch.tensor(rows)


@pytest.mark.parametrize("score,front,others,bias", [
    ("sigmoid", [17.0, 17.0, 17.125], -5.0, 0.0), ("sigmoid", [18.0, 18.0, 18.125, 18.125], -5.0, 0.0),
    ("sigmoid", [17.0, 17.125, 17.25, 17.375], -5.0, 0.5), ("sigmoid", [17.0, 17.0, 17.0, 17.125], -5.0, -0.25),
    ("sigmoid", [17.0] * 7 + [17.125], -5.0, 0.0), ("sigmoid", [17.125] + [17.0] * 6 + [17.125], -5.0, 0.0),
    ("softmax", [0.0, 0.0, 0.0078125], -20.0, 1.0), ("softmax", [0.0, 0.0078125, 0.0078125, 0.0], -20.0, 1.0),
    ("softmax", [0.0] * 7 + [0.0078125], -20.0, 1.0)])
def test_close_experts_among_equal_ones(score, front, others, bias):
    for E, k in ((9, 1), (12, 2), (9, 7), (64, 3), (64, 8), (256, 1), (256, 4), (300, 31), (1000, 32)):
        logits = _close_rows(E, front, others)
        biases = torch.full((E,), bias)
        if score == "softmax":                          # one takes nearly all of the sum, so that the others' scores are close
            logits[:, E - 1] = 17.0
            biases[E - 1] = 0.0
        for dtype in (torch.float32, torch.bfloat16):
            x = logits.to(dtype)
            _, idx = ops.route_topk(x.cuda(), k, score=score, bias=biases.cuda())
            assert torch.equal(idx.cpu(), want.route(x, k, score=score, bias=biases)[1]), (E, k, dtype)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_repeated_logits_and_biases(score, groups, top_groups):
    """Few different logits, saturated or not, and few different biases: equal and close keys everywhere."""
    T, E = 400, 64
    x = torch.randint(0, 4, (T, E)) * 0.125 + torch.tensor([0.0, 4.0, 17.0, 20.0])[torch.randint(0, 4, (T, 1))]
    bias = torch.randint(0, 2, (E,)) * 2.0 ** -22
    for k in (1, 6, 9):
        how = dict(score=score, bias=bias, groups=groups, top_groups=top_groups)
        _, idx = ops.route_topk(x.bfloat16().cuda(), k, **{**how, "bias": bias.cuda()})
        assert torch.equal(idx.cpu(), want.route(x.bfloat16(), k, **how)[1])


@pytest.mark.parametrize("biases,top_groups", [([40.0, -40.0, 40.0, -40.0], 1), ([1000.0, -1000.0, 0.5, 0.5], 1),
                                               ([3000.0, -3000.0, 0.25, 0.25, 0.0, 0.0], 2)])
def test_groups_by_two_keys_of_opposite_signs(biases, top_groups):
    """The keys round to steps of their own size, which their sum hides."""
    E = len(biases)
    T = 3000
    bias = torch.tensor(biases)
    x = torch.randn(T, E)
    value = (torch.sigmoid(x.double()) + bias.double()).view(T, E // 2, 2).sum(2)
    # the last expert's score makes the sums of its group and of the one before nearly equal
    room = torch.rand(T, dtype=torch.float64) * 2e-5 - 1e-5
    score = (torch.sigmoid(x[:, -1].double()) + value[:, -2] - value[:, -1] + room).clamp(0.001, 0.999)
    x[:, -1] = torch.log(score / (1 - score)).float()
    if E == 6:                                          # and the first group's, whose keys are the large ones
        score = (torch.sigmoid(x[:, 0].double()) + value[:, -2] - value[:, 0] + room.flip(0)).clamp(0.001, 0.999)
        x[:, 0] = torch.log(score / (1 - score)).float()
    how = dict(score="sigmoid", groups=E // 2, top_groups=top_groups, group_score=2)
    _, idx = ops.route_topk(x.cuda(), 2 * top_groups, bias=bias.cuda(), **how)
    assert torch.equal(idx.cpu(), want.route(x, 2 * top_groups, bias=bias, **how)[1])


def test_renormalised_sigmoids_far_apart():
    """Scores of one row over all of fp32's range: none vanishes that its type holds."""
    rows = [[-50.0, -90.0, -55.0], [0.0, -85.0, -100.0], [-59.0, -61.0, -130.0], [-100.0, -120.0, -180.0], [30.0, -87.0, 2.0],
            [-10.0, -95.0, -30.0], [3e38, -3.0, -88.0], [-1.0, 1.0, -1.5], [-200.0, -200.0, -201.0]]
    x = torch.tensor(rows)
    leaf = x.cuda().requires_grad_()
    weights, idx = ops.route_topk(leaf, 3, score="sigmoid")
    w, i = want.route(x, 3, score="sigmoid")
    assert torch.equal(idx.cpu(), i)
    # the difference of two logits is rounded (at most 100 steps of 2^-24 of its exponential), some ten more operations; below 2^-126 steps of 2^-149
    room = 128 * 2.0 ** -24 * w + 4 * 2.0 ** -149
    assert bool(((weights.detach().double().cpu() - w).abs() <= room).all())
    g = torch.randn(len(rows), 3)
    (got,) = torch.autograd.grad(weights, leaf, g.cuda())
    exact = want.route_gradient(x, i, g, "sigmoid", True, 1.0)
    # w_i (1 - s_i) (g_i - sum g w): relative to the weight, whose own room is above
    v = torch.zeros_like(exact).scatter_(1, i, w)
    size = v * (g.abs().double().sum(1, keepdim=True) + 1)
    assert bool(((got.double().cpu() - exact).abs() <= 256 * 2.0 ** -24 * size + 2.0 ** -146).all())


# ------------------------------------------------------------------------------ differentiation forward
def test_forward_mode_is_refused_and_not_dropped():
    from torch.autograd import forward_ad
    x, w = torch.randn(4, 64, device="cuda").bfloat16(), torch.ones(64, device="cuda")
    logits = torch.randn(4, 64, device="cuda")
    with forward_ad.dual_level():
        for t in (x, logits, w):
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError):
                if t is x:
                    ops.gated_add_rmsnorm(dual, x, w, w)
                elif t is w:
                    ops.gated_add_rmsnorm(x, x, w, w, gate=dual)
                else:
                    ops.route_topk(dual, 3)
        ops.gated_add_rmsnorm(x, x, w, w)               # plain operands are taken inside of a level too
        ops.route_topk(logits, 3)


# ------------------------------------------------------------------------------ sizes
def test_gated_norm_refuses_rows_whose_counters_would_overflow():
    one, w = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16), torch.ones(1, device="cuda")
    for rows in (2 ** 31 - 2 ** 16 + 1, 2 ** 31 - 2):
        many = one.expand(rows, 1)
        with pytest.raises(ValueError, match="rows"):
            ops.gated_add_rmsnorm(many, many, w, w)
        many = torch.empty(rows, 1, device="cuda", dtype=torch.bfloat16)      # contiguous: through the C++ node
        with pytest.raises(ValueError, match="rows"):
            ops.gated_add_rmsnorm(many, many, w, w)


def test_factors_are_numbers_of_fp32():
    x, w = torch.randn(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for bad in (1e300, -1e39):
        with pytest.raises(ValueError, match="scale"):
            ops.route_topk(x, 2, scale=bad)
        with pytest.raises(ValueError, match="residual_scale"):
            ops.gated_add_rmsnorm(x, x, w, w, residual_scale=bad)
    for bad in (1e-60, 1e300):
        with pytest.raises(ValueError, match="eps"):
            ops.gated_add_rmsnorm(x, x, w, w, eps=bad)
    with pytest.raises(ValueError, match="scale"):
        ops.route_topk(x, 2, scale=1e-60)


@pytest.mark.parametrize("B,S,D", [(1500, 2, 512), (900, 3, 264), (700, 7, 128), (1300, 4, 1000), (800, 9, 512), (601, 2, 1024), (301, 5, 2048),
                                   (40, 3, 100), (6, 2, 1999), (5001, 2, 64)])
def test_gated_norm_of_short_sequences(B, S, D):
    from test_gpu_operators import _check_norm, _norm_case
    for dtype in (torch.bfloat16, torch.float32):
        _check_norm(*_norm_case(B, S, D, "sequence", dtype))


# ------------------------------------------------------------------------------ 8-bit values
def test_quantize_fp8_statement_on_the_gpu_is_that_on_the_cpu():
    from b200moe.ops import functional as Fn
    x = torch.randn(257, 1000, device="cuda").bfloat16()
    for block_rows in (1, 128):
        values, scales = Fn.quantize_fp8_ref(x, block_rows)
        v, s = Fn.quantize_fp8_ref(x.cpu(), block_rows)
        assert torch.equal(scales.cpu(), s) and torch.equal(values.cpu().view(torch.uint8), v.view(torch.uint8))
        own = ops.quantize_fp8(x, block_rows)
        assert torch.equal(own[1], scales) and torch.equal(own[0].contiguous().view(torch.uint8), values.view(torch.uint8))


# ------------------------------------------------------------------------------ no tokens
@pytest.mark.parametrize("k", [1, 2, 3])
def test_moe_ffn_of_no_tokens(k):
    E, D, F = 8, 128, 256
    x = torch.zeros(0, D, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w1, w3 = (torch.randn(E, F, D, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w2 = torch.randn(E, D, F, device="cuda").bfloat16().requires_grad_()
    weights, idx = ops.route_topk(torch.zeros(0, E, device="cuda"), k)
    weights.requires_grad_()
    y = ops.moe_ffn(x, weights, idx, w1, w2, w3)
    assert y.shape == (0, D) and y.dtype == torch.bfloat16
    grads = torch.autograd.grad(y, (x, weights, w1, w2, w3), torch.empty_like(y))
    assert grads[0].shape == (0, D) and grads[1].shape == (0, k) and all(g.shape == w.shape and not g.any() for g, w in
                                                                          zip(grads[2:], (w1, w2, w3)))


def test_moe_ffn_looks_at_its_operands():
    E, D, F, T = 8, 128, 256, 40
    x = torch.randn(T, D, device="cuda").bfloat16()
    experts = [torch.randn(E, *shape, device="cuda").bfloat16() for shape in ((F, D), (D, F), (F, D))]
    weights, idx = ops.route_topk(torch.randn(T, E, device="cuda"), 3)
    y = ops.moe_ffn(x, weights, idx, *experts)
    assert torch.equal(ops.moe_ffn(x, weights, idx.int(), *experts), y)       # the kernels read 64-bit indices
    for bad in ((x, weights[:, :1], idx), (x[:39], weights, idx), (x, weights[:39], idx[:39]), (x, weights.cpu(), idx),
                (x, weights, idx.cpu())):
        with pytest.raises(ValueError):
            ops.moe_ffn(*bad, *experts)

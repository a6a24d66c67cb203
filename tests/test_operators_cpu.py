"""Routing, gated residual norm and 8-bit products: their PyTorch statements against 64 bits, and what they refuse."""
import math

import pytest
import torch

import _operators as want
from b200moe import ops
from b200moe.models.layers import MoELayerMulti
from b200moe.ops import functional as Fn

ROUTES = [dict(k=2), dict(k=8, score="sigmoid", groups=8, top_groups=3, group_score=2, scale=2.5), dict(k=1, renormalize=False),
          dict(k=5, score="sigmoid", renormalize=False), dict(k=6, groups=4, top_groups=2, renormalize=False, scale=0.5),
          dict(k=32, score="sigmoid"), dict(k=12, groups=16, top_groups=4, group_score=2)]


@pytest.mark.parametrize("how", ROUTES)
@pytest.mark.parametrize("biased", [False, True])
def test_route_topk_chooses_and_weighs_as_defined(how, biased):
    torch.manual_seed(3)
    logits = torch.randn(37, 64)
    logits[3] = -math.inf
    logits[4, ::2] = -math.inf
    logits[5, 1:] = -math.inf
    logits[6, 7] = math.nan
    logits[7, 9] = math.inf
    logits[8] = 0.25
    bias = torch.randn(64) * 0.1 if biased else None
    weights, idx = ops.route_topk(logits, bias=bias, **how)
    w, i = want.route(logits, bias=bias, **how)
    assert torch.equal(idx, i)
    assert torch.allclose(weights.double(), w, rtol=2e-6, atol=1e-30)       # some 16 roundings of fp32


@pytest.mark.parametrize("how", ROUTES)
def test_route_topk_gradient_against_the_formula_and_differences(how):
    torch.manual_seed(4)
    logits = torch.randn(9, 64, dtype=torch.float64, requires_grad=True)
    with torch.no_grad():
        logits[2, 5:] = -math.inf
        logits[3] = -math.inf
    weights, idx = ops.route_topk(logits, **how)
    g = torch.randn(9, how["k"], dtype=torch.float64)
    (got,) = torch.autograd.grad(weights, logits, g)
    score, renormalize, scale = how.get("score", "softmax"), how.get("renormalize", True), how.get("scale", 1.0)
    assert torch.allclose(got, want.route_gradient(logits.detach(), idx, g, score, renormalize, scale), rtol=1e-9, atol=1e-12)
    step = 1e-6
    for row, col in ((0, int(idx[0, 0])), (1, int(idx[1, -1])), (4, 11)):
        moved = [logits.detach().clone() for _ in range(2)]
        moved[0][row, col] += step
        moved[1][row, col] -= step
        high, low = ((ops.route_topk(m, **how)[0] * g).sum() for m in moved)
        assert abs(float(high - low) / (2 * step) - float(got[row, col])) < 1e-6


def test_route_topk_refuses():
    x = torch.zeros(4, 12)
    for bad in (dict(k=0), dict(k=13), dict(k=2, score="relu"), dict(k=2, groups=5), dict(k=2, groups=4, top_groups=5),
                dict(k=7, groups=4, top_groups=2), dict(k=2, groups=12, top_groups=3, group_score=2), dict(k=2, group_score=3),
                dict(k=2, scale=0.0), dict(k=2, scale=math.inf), dict(k=2, bias=torch.zeros(11))):
        with pytest.raises(ValueError):
            ops.route_topk(x, **bad)
    with pytest.raises(ValueError):
        ops.route_topk(torch.zeros(12), 2)
    with pytest.raises(ValueError):
        ops.route_topk(torch.zeros(1, 1056), 2)
    with pytest.raises(ValueError):
        ops.route_topk(torch.zeros(1, 64), 33)
    with pytest.raises(TypeError):
        ops.route_topk(torch.zeros(4, 12, dtype=torch.int64), 2)
    weights, idx = ops.route_topk(torch.zeros(0, 12), 3, groups=4, top_groups=2, group_score=2)
    assert weights.shape == idx.shape == (0, 3)


def _gate(kind, B, S, D, dtype):
    shape = {"none": None, "channel": (D,), "sequence": (B, 1, D), "token": (B, S, 1), "full": (B, S, D)}[kind]
    return None if shape is None else torch.randn(*shape, dtype=dtype)


@pytest.mark.parametrize("kind", ["none", "channel", "sequence", "token", "full"])
def test_gated_add_rmsnorm_statement_and_its_gradient(kind):
    torch.manual_seed(5)
    B, S, D = 3, 4, 10
    x, delta = torch.randn(B, S, D, dtype=torch.float64), torch.randn(B, S, D, dtype=torch.float64)
    wd, w = torch.rand(D, dtype=torch.float64) + 0.5, torch.rand(D, dtype=torch.float64) + 0.5
    gate = _gate(kind, B, S, D, torch.float64)
    got = ops.gated_add_rmsnorm(x, delta, wd, w, gate=gate, residual_scale=0.7)
    for a, b in zip(got, want.gated_norm(x, delta, wd, w, gate, 0.7, 1e-5)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    leaves = [t.requires_grad_() for t in (x, delta, wd, w) + (() if gate is None else (gate,))]
    assert torch.autograd.gradcheck(
        lambda *t: ops.gated_add_rmsnorm(*t[:4], gate=t[4] if len(t) > 4 else None, residual_scale=0.7), leaves)


def test_gated_add_rmsnorm_refuses():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    for bad in (dict(gate=torch.ones(7)), dict(gate=torch.ones(3, 8)), dict(gate=torch.ones(2, 1, 1)), dict(residual_scale=math.nan),
                dict(eps=0.0), dict(gate=torch.tensor(1.0))):
        with pytest.raises(ValueError):
            ops.gated_add_rmsnorm(x, x, w, w, **bad)
    with pytest.raises(ValueError):
        ops.gated_add_rmsnorm(x, x[:1], w, w)
    with pytest.raises(ValueError):
        ops.gated_add_rmsnorm(x, x, w[:4], w)
    with pytest.raises(TypeError):
        ops.gated_add_rmsnorm(x, x.bfloat16(), w, w)
    with pytest.raises(TypeError):
        ops.gated_add_rmsnorm(x, x, w, w, gate=torch.ones(8, dtype=torch.float16))


@pytest.mark.parametrize("rows,cols", [(1, 1), (130, 300), (128, 128), (3, 513)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_fp8_statement(rows, cols, block_rows):
    torch.manual_seed(6)
    x = torch.randn(rows, cols) * torch.exp(2 * torch.randn(cols))
    x[0] = 0
    values, scales = ops.quantize_fp8(x, block_rows)
    v, s = want.quantize(x, block_rows)
    assert torch.equal(values.double(), v) and torch.equal(scales, s)
    back = Fn.dequantize_fp8_ref(values, scales, block_rows).double()
    # half a step of e4m3 relative to the value, half its smallest step (2^-10) below 2^-6
    factor = want.spread(s, rows, cols, block_rows)
    assert bool(((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, factor * 2.0 ** -10) * (1 + 1e-6)).all())


def test_linear_fp8_statement_and_gradients():
    torch.manual_seed(7)
    x, w = torch.randn(2, 5, 160, requires_grad=True), (torch.randn(24, 160) * 0.1).requires_grad_()
    y = ops.linear_fp8(x, w)
    vx, sx = want.quantize(x.detach().view(10, 160), 1)
    vw, sw = want.quantize(w.detach(), 128)
    qx, qw = vx * want.spread(sx, 10, 160, 1), vw * want.spread(sw, 24, 160, 128)
    assert torch.allclose(y.double().view(10, 24), qx @ qw.t(), rtol=1e-5, atol=1e-5)
    dy = torch.randn(2, 5, 24)
    dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    vg, sg = want.quantize(dy.view(10, 24), 1)
    assert torch.allclose(dx.double().view(10, 160), (vg * want.spread(sg, 10, 24, 1)) @ qw, rtol=1e-5, atol=1e-5)
    assert torch.allclose(dw, dy.view(10, 24).t() @ x.detach().view(10, 160), rtol=1e-5, atol=1e-5)
    w.main_grad = torch.ones(24, 160)
    y = ops.linear_fp8(x, w, weight_fp8=ops.quantize_fp8(w.detach(), 128))
    assert torch.autograd.grad(y, (x, w), dy, allow_unused=True)[1] is None
    assert torch.allclose(w.main_grad, 1 + dw, rtol=1e-5, atol=1e-5)


def test_fp8_refuses_sizes_beyond_32_bits():
    long = torch.zeros(1, 1, dtype=torch.bfloat16)
    for shape in ((2 ** 31, 1), (1, 2 ** 32 + 128)):
        with pytest.raises(ValueError, match="rows or columns"):
            ops.quantize_fp8(long.expand(shape))
        with pytest.raises(ValueError, match="rows or columns"):
            ops.matmul_fp8(long.to(torch.float8_e4m3fn).expand(shape), torch.ones(1, 1), *ops.quantize_fp8(long, 128))
    with pytest.raises(ValueError, match="rows"):
        ops.linear_fp8(long.expand(2 ** 31, 1), long)


def test_fp8_refuses():
    q, s = ops.quantize_fp8(torch.randn(5, 200), 1)
    b, t = ops.quantize_fp8(torch.randn(7, 200), 128)
    assert ops.matmul_fp8(q, s, b, t).shape == (5, 7)
    with pytest.raises(ValueError):
        ops.quantize_fp8(torch.randn(5, 200), 64)
    with pytest.raises(ValueError):
        ops.quantize_fp8(torch.randn(5), 1)
    with pytest.raises(TypeError):
        ops.quantize_fp8(torch.zeros(5, 4, dtype=torch.int32), 1)
    with pytest.raises(TypeError):
        ops.matmul_fp8(q.float(), s, b, t)
    for args in ((q, s[:, :1], b, t), (q, s.double(), b, t), (q, s, b, t.t()), (q[:, :128], s[:, :1], b, t)):
        with pytest.raises(ValueError):
            ops.matmul_fp8(*args)
    w = torch.randn(7, 200)
    for bad in (dict(x=torch.randn(3, 100)), dict(weight_fp8=(b[:3], t)), dict(weight_fp8=(b[:, :100], t[:, :1]))):
        with pytest.raises(ValueError):
            ops.linear_fp8(bad.get("x", torch.randn(3, 200)), w, weight_fp8=bad.get("weight_fp8"))


def test_routed_layer_with_another_router():
    torch.manual_seed(8)
    how = dict(score="sigmoid", groups=4, top_groups=2, group_score=2, scale=1.5)
    layer = MoELayerMulti(32, 48, k=3, num_expert_per_node=8, dtype=torch.float32, routing={**how, "balance_bias": True})
    layer.expert_bias.copy_(torch.randn(8) * 0.2)
    assert "expert_bias" in layer.state_dict()
    x = torch.randn(2, 5, 32, requires_grad=True)
    y, aux = layer(x, return_aux_loss=True)
    logits = x.view(10, 32) @ layer.router.weight.t()
    weights, idx = Fn.route_topk_ref(logits, 3, bias=layer.expert_bias, **how)
    out = torch.zeros(10, 32)
    for t in range(10):
        for j in range(3):
            e = int(idx[t, j])
            h = Fn.silu(x.view(10, 32)[t] @ layer.experts.w1[e].t()) * (x.view(10, 32)[t] @ layer.experts.w3[e].t())
            out[t] = out[t] + weights[t, j] * (h @ layer.experts.w2[e].t())
    assert torch.allclose(y.view(10, 32), out, atol=1e-5)
    g = torch.randn(2, 5, 32)
    got = torch.autograd.grad(y, (x, layer.router.weight), g, retain_graph=True)
    for a, b in zip(got, torch.autograd.grad(out.view(2, 5, 32), (x, layer.router.weight), g)):
        assert torch.allclose(a, b, atol=1e-4)
    assert float(aux) > 0
    for bad in (dict(groups=3), dict(topk=2), dict(groups=8, top_groups=1)):
        with pytest.raises(ValueError):
            MoELayerMulti(32, 48, k=3, num_expert_per_node=8, dtype=torch.float32, routing=bad)
    with pytest.raises(ValueError):
        MoELayerMulti(32, 48, k=3, num_expert_per_node=8, dtype=torch.float32)


def test_routed_layer_with_another_router_over_two_ranks(tmp_path, free_port):
    import torch.multiprocessing as mp

    import _operator_workers as workers
    mp.spawn(workers.run_routed_layer, args=(2, free_port, str(tmp_path)), nprocs=2, join=True)
    assert (tmp_path / "routed_ok_0").exists() and (tmp_path / "routed_ok_1").exists()

"""Routing, gated residual norm and 8-bit products on the GPU against 64 bits."""
import math

import pytest
import torch

import _operators as want
from b200moe import ops
from b200moe.ops import functional as Fn

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # of a value, when it is rounded
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}                  # half of the smallest step


@pytest.fixture(autouse=True)
def _native():
    from b200moe.ops import native
    native.require()
    torch.manual_seed(11)
    yield
    native.check_status()


def _within(got, exact, slack):
    """Rounded once to the type of ``got``, after fp32 arithmetic that is off by ``slack`` at most."""
    exact = exact.to(got.device)
    room = HALF[got.dtype] * (exact.abs() + slack) + TINY[got.dtype] + slack
    bad = (got.double() - exact).abs() > room
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - exact).abs() / room.clamp(min=1e-300)).max()))


# ------------------------------------------------------------------------------ routing
ROUTES = [  # experts, and how they are chosen
    (8, dict(k=2)), (1, dict(k=1)), (5, dict(k=5, score="sigmoid")), (33, dict(k=3, renormalize=False)),
    (64, dict(k=6, renormalize=False, scale=0.5)), (77, dict(k=32, score="sigmoid")),
    (96, dict(k=4, groups=32, top_groups=5, group_score=2)), (128, dict(k=16, score="sigmoid", renormalize=False)),
    (160, dict(k=6, groups=8, top_groups=3)), (256, dict(k=8, score="sigmoid", groups=8, top_groups=4, group_score=2, scale=2.5)),
    (256, dict(k=8, groups=2, top_groups=1, group_score=2, renormalize=False)), (511, dict(k=7, score="sigmoid", groups=7, top_groups=2)),
    (512, dict(k=10, groups=4, top_groups=2, group_score=2)), (768, dict(k=12, score="sigmoid", groups=3, top_groups=1)),
    (1024, dict(k=32, renormalize=False, groups=32, top_groups=31)), (1000, dict(k=4)),
]


def _logits(T, E, dtype):
    x = torch.randn(T, E, device="cuda") * 1.5
    x[:, E // 2] = x[:, 0]                              # equal logits in every row
    if T > 8:
        x[1] = -math.inf
        x[2, 1:] = -math.inf
        x[3, ::2] = math.nan
        x[4, E - 1] = math.inf
        x[5] = 0.5
        x[6] = x[6].sign() * 0.0                        # zeros of both signs
        x[7] -= 200.0                                   # sigmoids that fp32 does not hold
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E,how", ROUTES)
@pytest.mark.parametrize("biased", [False, True])
def test_route_topk(E, how, biased, dtype):
    T = 203
    logits = _logits(T, E, dtype).requires_grad_()
    bias = torch.randn(E, device="cuda") * 0.05 if biased else None
    weights, idx = ops.route_topk(logits, bias=bias, **how)
    w, i = want.route(logits.detach().cpu(), bias=None if bias is None else bias.cpu(), **how)
    assert torch.equal(idx.cpu(), i)
    # a sum of E terms, an exponential, a division, a scale: below E + 16 roundings; of exp(x - max) also 2^-24 |x - max|
    assert torch.allclose(weights.detach().double().cpu(), w, rtol=(E + 40) * 2.0 ** -24, atol=1e-37)
    g = torch.randn(T, how["k"], device="cuda")
    (got,) = torch.autograd.grad(weights, logits, g)
    clean = torch.where(torch.isinf(logits.detach()) & (logits.detach() > 0), torch.finfo(torch.float32).max, logits.detach().double())
    score, renormalize, scale = how.get("score", "softmax"), how.get("renormalize", True), how.get("scale", 1.0)
    keep = torch.ones(T, dtype=torch.bool)
    if score == "sigmoid" and renormalize:
        keep[7] = False                                 # the definition divides by what fp64 holds of exp(-200): held apart below
    exact = want.route_gradient(clean.cpu(), i, g.cpu(), score, renormalize, scale)
    slack = (E + 60) * 2.0 ** -24 * scale * g.abs().double().sum(1, keepdim=True).cpu() * torch.ones(1, E)
    _within(got.cpu()[keep], exact[keep], slack[keep])
    again = ops.route_topk(logits.detach(), bias=bias, **how)
    assert torch.equal(again[0], weights) and torch.equal(again[1], idx)


@pytest.mark.parametrize("group_score", [0, 1, 2])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_topk_decides_what_fp32_cannot(score, group_score):
    """Keys that differ by less than an fp32 step of theirs, and keys that are equal."""
    T, E, k = 400, 64, 6
    logits = torch.randn(T, E, device="cuda")
    s = torch.softmax(logits.double(), 1) if score == "softmax" else torch.sigmoid(logits.double())
    bias = torch.randn(E, device="cuda") * 0.1
    # the bias of expert 1 makes its key nearly that of expert 0 in row 0, and so on for pairs of experts and rows
    for row in range(0, 60, 2):
        a, b = row, row + 1
        bias[a] += 1.0
        bias[b] = (s[row, a] + bias[a].double() - s[row, b]).float()
    how = dict(k=k, score=score, renormalize=False)
    if group_score:
        how.update(groups=8, top_groups=3, group_score=group_score)
    weights, idx = ops.route_topk(logits, bias=bias, **how)
    w, i = want.route(logits.cpu(), bias=bias.cpu(), **how)
    assert torch.equal(idx.cpu(), i)


def test_route_topk_of_other_layouts_streams_and_captures():
    base = torch.randn(50, 2 * 96, device="cuda")
    for logits in (base[:, ::2], base.t().contiguous().t()[:, 3:99], base.flatten()[5:5 + 50 * 96].view(50, 96)):
        weights, idx = ops.route_topk(logits, 4)
        w, i = ops.route_topk(logits.clone(memory_format=torch.contiguous_format), 4)
        assert torch.equal(weights, w) and torch.equal(idx, i)
    empty = torch.zeros(0, 96, device="cuda", requires_grad=True)
    weights, idx = ops.route_topk(empty, 4)
    assert weights.shape == (0, 4) and torch.autograd.grad(weights.sum(), empty)[0].shape == (0, 96)
    static = torch.randn(300, 256, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            ops.route_topk(static, 8, score="sigmoid")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        weights, idx = ops.route_topk(static, 8, score="sigmoid")
    static.copy_(torch.randn(300, 256, device="cuda"))
    graph.replay()
    w, i = ops.route_topk(static, 8, score="sigmoid")
    assert torch.equal(weights, w) and torch.equal(idx, i)


def test_route_topk_beyond_32_bits_of_offset():
    T, E = 2 ** 21 + 5, 1024
    logits = torch.zeros(T, E, device="cuda", dtype=torch.bfloat16).requires_grad_()
    with torch.no_grad():
        logits[-3:] = torch.randn(3, E, device="cuda").bfloat16()
    weights, idx = ops.route_topk(logits, 3, renormalize=False)
    w, i = want.route(logits.detach()[-3:].cpu(), 3, renormalize=False)
    assert torch.equal(idx[-3:].cpu(), i) and torch.allclose(weights.detach()[-3:].cpu().double(), w, rtol=1e-4)
    assert bool((idx[:-3] == torch.arange(3, device="cuda")).all())
    (got,) = torch.autograd.grad(weights, logits, torch.ones_like(weights))
    exact = want.route_gradient(logits.detach()[-3:].cpu(), i, torch.ones(3, 3), "softmax", False, 1.0)
    _within(got[-3:].cpu(), exact, torch.full_like(exact, 1e-4 * 2.0 ** -8))


# ------------------------------------------------------------------------------ gated residual norm
def _norm_case(B, S, D, kind, dtype, gate_dtype=None):
    shape = {"none": None, "channel": (D,), "sequence": (B, 1, D), "token": (B, S, 1), "full": (B, S, D)}[kind]
    x, delta = (torch.randn(B, S, D, device="cuda").to(dtype) for _ in range(2))
    wd, w = (torch.rand(D, device="cuda") + 0.5 for _ in range(2))
    gate = None if shape is None else torch.randn(*shape, device="cuda").to(gate_dtype or dtype)
    return x, delta, wd, w, gate


def _check_norm(x, delta, wd, w, gate, scale=0.7, eps=1e-5, use=(True, True)):
    leaves = [t.detach().requires_grad_() for t in (x, delta, wd, w) + (() if gate is None else (gate,))]
    summed, normed = ops.gated_add_rmsnorm(*leaves[:4], gate=None if gate is None else leaves[4], residual_scale=scale, eps=eps)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    s, y = want.gated_norm(*exact[:4], None if gate is None else exact[4], scale, eps)
    D = x.shape[-1]
    # fp32: every value is a few products of values with relative errors of some roundings (the sums of squares are sums of
    # non-negative terms: below 2^-20 for 8192 of them)
    few = 2.0 ** -19
    branch = (s - exact[0] * scale).detach()
    size = (exact[0] * scale).abs().detach() + branch.abs()
    _within(summed.detach(), s.detach(), few * size)
    ratio = (y.detach() / s.detach().where(s.detach() != 0, torch.ones_like(s))).abs()
    _within(normed.detach(), y.detach(), few * (y.detach().abs() + ratio * size))
    ds, dy = torch.randn_like(summed), torch.randn_like(normed)
    outs, grads = zip(*[(a, b) for a, b, u in ((summed, ds, use[0]), (normed, dy, use[1])) if u])
    got = torch.autograd.grad(outs, leaves, grads, allow_unused=True)
    ref = torch.autograd.grad([a for a, u in ((s, use[0]), (y, use[1])) if u], exact, [g.double() for g in grads],
                              allow_unused=True)
    # What the gradients are differences and sums of, which fp32 errors are relative to (a row of one value cancels to what eps
    # leaves of it): dS = ds + r (dy w - yhat mean), ddelta = r_d (dn w_d - nhat mean), sums of dS n and of dy yhat.
    ex, ed, ewd, ew = (t.detach() for t in exact[:4])
    eg = torch.ones_like(ewd) if gate is None else exact[4].detach()
    r = 1 / torch.sqrt((s.detach() ** 2).mean(-1, keepdim=True) + eps)
    rd = 1 / torch.sqrt((ed ** 2).mean(-1, keepdim=True) + eps)
    nhat, yhat = (ed * rd).abs(), size * r               # the sum itself is off by what its two terms are relative to
    part = r * (dy.double() * ew).abs() * use[1]
    dS_size = ds.double().abs() * use[0] + part + part.amax(-1, keepdim=True) * yhat.clamp(min=1)
    dn_size = (eg * ewd).abs() * dS_size
    rows = x.numel() // D
    sums = few + rows * 2.0 ** -24
    sizes = {"dx": few * scale * dS_size, "ddelta": few * rd * (dn_size + dn_size.amax(-1, keepdim=True) * nhat.clamp(min=1)),
             "dwd": sums * (eg.abs() * dS_size * nhat).sum_to_size(D), "dw": sums * (dy.double().abs() * yhat).sum_to_size(D)}
    if gate is not None:
        sizes["dgate"] = (few + (rows + D) * 2.0 ** -24) * (dS_size * nhat * ewd.abs()).sum_to_size(gate.shape)
    for name, a, b, leaf in zip(("dx", "ddelta", "dwd", "dw", "dgate"), got, ref, leaves):
        assert a.dtype == leaf.dtype and a.shape == leaf.shape
        _within(a, torch.zeros_like(a, dtype=torch.float64) if b is None else b, sizes[name].expand(a.shape))


@pytest.mark.parametrize("kind", ["none", "channel", "sequence", "token", "full"])
@pytest.mark.parametrize("B,S,D", [(1, 1, 64), (3, 1, 4096), (2, 77, 512), (5, 33, 1000), (7, 5, 1032), (2, 19, 2048), (3, 40, 5120),
                                   (2, 9, 8192), (4, 3, 7), (3, 21, 333), (2, 5, 4099), (300, 2, 128), (1, 700, 256), (37, 13, 264)])
def test_gated_add_rmsnorm(B, S, D, kind):
    _check_norm(*_norm_case(B, S, D, kind, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["fp32", "fp16"])
@pytest.mark.parametrize("kind", ["channel", "sequence", "token", "full"])
@pytest.mark.parametrize("B,S,D", [(2, 77, 512), (5, 7, 999), (2, 9, 2560), (2, 5, 8192), (1, 3, 1)])
def test_gated_add_rmsnorm_types(B, S, D, kind, dtype):
    _check_norm(*_norm_case(B, S, D, kind, dtype))
    if dtype == torch.float16:
        _check_norm(*_norm_case(B, S, D, kind, dtype, torch.float32))


@pytest.mark.parametrize("kind", ["none", "channel", "sequence", "token", "full"])
@pytest.mark.parametrize("B,S,D,dtype", [(7, 701, 512, torch.bfloat16), (3, 1001, 776, torch.float16), (2, 701, 2048, torch.bfloat16),
                                         (601, 5, 1024, torch.bfloat16), (13, 47, 4096, torch.bfloat16), (2, 307, 5120, torch.bfloat16),
                                         (4, 601, 264, torch.float32), (5, 80, 8192, torch.float16), (1, 617, 4096, torch.float32),
                                         (1, 300, 8192, torch.float32), (2999, 3, 104, torch.bfloat16)])
def test_gated_add_rmsnorm_of_many_rows(B, S, D, dtype, kind):
    _check_norm(*_norm_case(B, S, D, kind, dtype))
    if D in (2048, 5120):
        _check_norm(*_norm_case(B, S, D, kind, dtype, torch.float32), use=(D == 2048, D != 2048))


@pytest.mark.parametrize("kind", ["none", "channel", "sequence", "token", "full"])
@pytest.mark.parametrize("B,S,D,dtype", [(2, 307, 4104, torch.bfloat16), (11, 83, 6144, torch.bfloat16), (1, 900, 4608, torch.float16),
                                         (1, 617, 4224, torch.float32), (1, 611, 6136, torch.float32), (2, 350, 6152, torch.bfloat16)])
def test_gated_add_rmsnorm_of_ten_and_twelve_warps(B, S, D, dtype, kind):
    _check_norm(*_norm_case(B, S, D, kind, dtype))
    if dtype != torch.float32:
        _check_norm(*_norm_case(B, S, D, kind, dtype, torch.float32))


def test_gated_add_rmsnorm_uses_and_layouts():
    for use in ((True, False), (False, True)):
        _check_norm(*_norm_case(2, 30, 264, "channel", torch.bfloat16), use=use)
    x, delta, wd, w, gate = _norm_case(4, 30, 256, "sequence", torch.bfloat16, torch.float32)
    _check_norm(x.transpose(0, 1).contiguous().transpose(0, 1), delta[..., :].flip(1), wd, w, gate.expand(4, 1, 256))
    wide = torch.randn(4, 30, 300, device="cuda").bfloat16()
    _check_norm(wide[..., 3:259], delta, wd, w, gate)
    flat = torch.randn(4 * 30 * 256 + 1, device="cuda").bfloat16()[1:].view(4, 30, 256)     # 2 bytes off a 16-byte boundary
    _check_norm(flat, delta, wd, w, gate)
    _check_norm(x[0], delta[0], wd, w, torch.randn(30, 1, device="cuda").bfloat16())
    _check_norm(x.view(2, 2, 30, 256), delta.view(2, 2, 30, 256), wd, w, torch.randn(2, 1, 1, 256, device="cuda").bfloat16())
    zero = torch.zeros_like(x)
    _check_norm(zero, zero, wd, w, gate)
    with pytest.raises(ValueError):
        ops.gated_add_rmsnorm(*(torch.zeros(2, 8193, device="cuda") for _ in range(2)), *(torch.ones(8193, device="cuda") for _ in range(2)))
    empty = [t.requires_grad_() for t in (x[:0].clone(), delta[:0].clone(), wd.clone(), w.clone())]
    summed, normed = ops.gated_add_rmsnorm(*empty)
    grads = torch.autograd.grad((summed.sum() + normed.sum()), empty)
    assert not grads[2].any() and not grads[3].any() and grads[0].shape == (0, 30, 256)


def test_gated_add_rmsnorm_repeats_bit_for_bit_in_a_graph():
    x, delta, wd, w, gate = _norm_case(3, 70, 1024, "sequence", torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, delta, wd, w, gate)]
    ds, dy = torch.randn_like(x), torch.randn_like(x)

    def step():
        out = ops.gated_add_rmsnorm(*leaves[:4], gate=leaves[4])
        return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, (ds, dy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(first, captured))


def test_gated_add_rmsnorm_beyond_32_bits_of_offset():
    rows, D = 2 ** 18 + 3, 8192
    x = torch.zeros(rows, D, device="cuda", dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, D, device="cuda").bfloat16()
    delta, w = torch.ones_like(x), torch.ones(D, device="cuda")
    summed, normed = ops.gated_add_rmsnorm(x, delta, w, w)
    s, y = want.gated_norm(x[-2:].double(), delta[-2:].double(), w.double(), w.double(), None, 1.0, 1e-5)
    _within(summed[-2:], s, 2.0 ** -19 * (s.abs() + 2))
    _within(normed[-2:], y, 2.0 ** -19 * (y.abs() + 2))
    assert bool((summed[:-2] == 1).all()) and bool((normed[:-2] == 1).all())


# ------------------------------------------------------------------------------ 8-bit products
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (130, 300), (257, 1024), (3, 2057), (129, 136)])
def test_quantize_fp8(rows, cols, block_rows, dtype):
    x = (torch.randn(rows, cols, device="cuda") * torch.exp(2 * torch.randn(cols, device="cuda"))).to(dtype)
    x[0] = 0
    values, scales = ops.quantize_fp8(x, block_rows)
    v, s = want.quantize(x, block_rows)
    assert torch.equal(scales.cpu(), s) and torch.equal(values.double().cpu(), v)
    assert values.stride(0) % 16 == 0 and values.data_ptr() % 16 == 0
    whole = torch.as_strided(values.view(torch.uint8), (rows, values.stride(0)), (values.stride(0), 1))
    assert not whole[:, cols:].any()
    wide = torch.zeros(rows, cols + 9, device="cuda", dtype=dtype)
    wide[:, 5:cols + 5] = x
    again = ops.quantize_fp8(wide[:, 5:cols + 5], block_rows)
    assert torch.equal(again[0].view(torch.uint8), values.view(torch.uint8)) and torch.equal(again[1], scales)
    turned = ops.quantize_fp8(x.t().contiguous().t(), block_rows)
    assert torch.equal(turned[0].view(torch.uint8), values.view(torch.uint8))


def test_quantize_fp8_of_values_that_are_not_numbers():
    x = torch.randn(4, 256, device="cuda")
    x[0, 3], x[1, 130], x[2, 7] = math.nan, math.inf, 1e-38
    x[3] = 1e-40
    values, scales = ops.quantize_fp8(x, 1)
    v, s = Fn.quantize_fp8_ref(x.cpu(), 1)
    assert torch.equal(torch.nan_to_num(values.float().cpu(), nan=999.0), torch.nan_to_num(v.float(), nan=999.0))
    assert torch.equal(scales.cpu(), s)
    assert torch.isnan(values[0, 3].float()) and torch.isnan(values[1, 130].float()) and not torch.isnan(values[2].float()).any()


def _operand(rows, cols, block_rows):
    x = torch.randn(rows, cols, device="cuda") * torch.exp(torch.randn(cols, device="cuda"))
    return ops.quantize_fp8(x, block_rows)


def _check_product(got, a, b):
    """``a @ bᵀ`` of 64-bit numbers.  Rounded once; before that the tensor cores add 32 products at a time in fp32, in which each
    addition may cut off a unit in the last place of the sum of absolute values, and blocks are scaled and added in fp32."""
    K = a.shape[1]
    slack = (a.abs() @ b.abs().t()) * (K // 32 + K // 128 + 8) * 2.0 ** -23
    _within(got, a @ b.t(), slack)


@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (1, 4096, 4096), (16, 4096, 2048), (17, 300, 1000), (128, 256, 128), (130, 129, 130),
                                   (200, 1000, 64), (257, 517, 513), (1003, 1544, 2000), (300, 8, 4096), (64, 64, 14336), (640, 4096, 384),
                                   (129, 1, 77), (2500, 2000, 257), (5000, 320, 1024), (16, 1024, 14336), (7, 520, 9000), (32, 2056, 4096),
                                   (31, 136, 1031), (33, 4096, 4096)])
def test_matmul_fp8(M, N, K):
    a, sa = _operand(M, K, 1)
    b, sb = _operand(N, K, 128)
    exact = a.double() * want.spread(sa, M, K, 1), b.double() * want.spread(sb, N, K, 128)
    _check_product(ops.matmul_fp8(a, sa, b, sb), *exact)
    _check_product(ops.matmul_fp8(a, sa.contiguous(), b, sb.t().contiguous().t()), *exact)


@pytest.mark.parametrize("M,N,K", [(1, 128, 256), (33, 264, 160), (130, 1000, 512), (700, 512, 1376), (2100, 1024, 992), (300, 4096, 2048)])
def test_linear_fp8_and_its_gradients(M, N, K):
    x = torch.randn(M, K, device="cuda").bfloat16().requires_grad_()
    weight = (torch.randn(N, K, device="cuda") * 0.05).bfloat16().requires_grad_()
    dy = (torch.randn(M, N, device="cuda") * 0.1).bfloat16()
    y = ops.linear_fp8(x, weight)
    dx, dw = torch.autograd.grad(y, (x, weight), dy)
    (vx, sx), (vw, sw), (vg, sg) = (want.quantize(t.detach(), r) for t, r in ((x, 1), (weight, 128), (dy, 1)))
    qx, qw, qg = ((v * want.spread(s, *v.shape, r)).cuda() for v, s, r in ((vx, sx, 1), (vw, sw, 128), (vg, sg, 1)))
    _check_product(y.detach(), qx, qw)
    _check_product(dx, qg, qw.t())
    g, h = dy.double(), x.detach().double()
    _within(dw, g.t() @ h, (g.abs().t() @ h.abs()) * (M // 16 + 8) * 2.0 ** -23)
    given = ops.linear_fp8(x, weight, weight_fp8=ops.quantize_fp8(weight, 128))
    assert torch.equal(given, y)
    weight.main_grad = torch.ones(N, K, device="cuda")
    dx2, none = torch.autograd.grad(ops.linear_fp8(x.view(1, M, K), weight), (x, weight), dy.view(1, M, N), allow_unused=True)
    assert none is None and torch.equal(dx2, dx)
    _within(weight.main_grad, 1 + g.t() @ h, 2.0 ** -23 + (g.abs().t() @ h.abs()) * (M // 16 + 8) * 2.0 ** -23)


def test_linear_fp8_layouts_streams_and_graphs():
    M, N, K = 300, 512, 640
    base = torch.randn(M, 2 * K + 3, device="cuda").bfloat16()
    weight = (torch.randn(N, K, device="cuda") * 0.05).bfloat16().requires_grad_()
    for x in (base[:, 1:K + 1], base[:, ::2][:, :K], base.t()[:K].t()):
        x = x.detach().requires_grad_()
        y = ops.linear_fp8(x, weight)
        same = x.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
        z = ops.linear_fp8(same, weight)
        assert torch.equal(y, z)
        dy = torch.randn(M, 2 * N, device="cuda").bfloat16()[:, 1::2]
        for p, q in zip(torch.autograd.grad(y, (x, weight), dy), torch.autograd.grad(z, (same, weight), dy.contiguous())):
            assert torch.equal(p, q)
    x = base[:, :K].contiguous()
    packed = ops.quantize_fp8(weight, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        want_y = ops.linear_fp8(x, weight, weight_fp8=packed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph), torch.no_grad():
        y = ops.linear_fp8(x, weight, weight_fp8=packed)
    graph.replay()
    assert torch.equal(y, want_y)
    none = x[:0].clone().requires_grad_()
    y = ops.linear_fp8(none, weight)
    dx, dw = torch.autograd.grad(y, (none, weight), torch.empty_like(y))
    assert y.shape == (0, N) and dx.shape == (0, K) and dw.shape == (N, K) and not dw.any()


def test_linear_fp8_training_step_in_a_graph():
    M, N, K = 130, 256, 192
    x = torch.randn(M, K, device="cuda").bfloat16().requires_grad_()
    weight = (torch.randn(N, K, device="cuda") * 0.1).bfloat16().requires_grad_()
    dy = torch.randn(M, N, device="cuda").bfloat16()

    def step():
        y = ops.linear_fp8(x, weight)
        return [y.detach(), *torch.autograd.grad(y, (x, weight), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    captured = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            captured.append(step())
    with torch.no_grad():
        x.mul_(0.5)
        dy.add_(1)
    for graph in graphs + graphs:
        graph.replay()
    exact = step()
    for results in captured:
        assert all(torch.equal(a, b) for a, b in zip(results, exact))


def test_products_beyond_32_bits_of_offset():
    rows, K, N = 2 ** 19 + 130, 4128, 16
    x = torch.zeros(rows, K, device="cuda", dtype=torch.bfloat16)
    x[-200:] = torch.randn(200, K, device="cuda").bfloat16()
    values, scales = ops.quantize_fp8(x)
    v, s = want.quantize(x[-200:], 1)
    assert torch.equal(values[-200:].double().cpu(), v) and torch.equal(scales[-200:].cpu(), s)
    b, sb = _operand(N, K, 128)
    y = ops.matmul_fp8(values, scales, b, sb)
    _check_product(y[-200:], (v * want.spread(s, 200, K, 1)).cuda(), b.double() * want.spread(sb, N, K, 128))
    assert not y[:-200].any()


def test_linear_fp8_of_widths_that_have_no_gradient_products():
    x, w = torch.randn(9, 1000, device="cuda").bfloat16(), (torch.randn(77, 1000, device="cuda") * 0.1).bfloat16()
    (vx, sx), (vw, sw) = want.quantize(x, 1), want.quantize(w, 128)
    exact = (vx * want.spread(sx, 9, 1000, 1)).cuda(), (vw * want.spread(sw, 77, 1000, 128)).cuda()
    _check_product(ops.linear_fp8(x, w), *exact)
    _check_product(ops.linear_fp8(x, w, weight_fp8=ops.quantize_fp8(w, 128)), *exact)
    dx = torch.autograd.grad(ops.linear_fp8(x.requires_grad_(), w), x, torch.ones(9, 77, device="cuda").bfloat16())[0]
    _check_product(dx, torch.ones(9, 77, device="cuda", dtype=torch.float64), exact[1].t())


def test_rows_beyond_32_bits_are_refused():
    one, w = torch.zeros(1, 1, device="cuda", dtype=torch.bfloat16), torch.ones(1, device="cuda")
    many = one.expand(2 ** 31, 1)
    with pytest.raises(ValueError, match="rows"):
        ops.gated_add_rmsnorm(many, many, w, w)
    with pytest.raises(ValueError, match="rows"):
        ops.quantize_fp8(many)
    with pytest.raises(ValueError, match="rows"):
        ops.linear_fp8(many, one)


def test_fp8_refuses_on_the_gpu():
    a, sa = _operand(5, 200, 1)
    b, sb = _operand(7, 200, 128)
    for bad in (a.contiguous(), a[:, 8:], a.t().contiguous().t()):
        scales = sa if bad.shape == a.shape else sa[:, :(bad.shape[1] + 127) // 128]
        other = b if bad.shape == a.shape else b[:, :bad.shape[1]]
        with pytest.raises(ValueError):
            ops.matmul_fp8(bad, scales, other, sb[:, :scales.shape[1]])
    with pytest.raises(ValueError):
        ops.matmul_fp8(a, sa.cpu(), b, sb)
    with pytest.raises(TypeError):
        ops.linear_fp8(torch.zeros(3, 200, device="cuda"), torch.zeros(7, 200, device="cuda"))
    w = torch.zeros(7, 200, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError):
        ops.linear_fp8(torch.zeros(3, 200, device="cuda", dtype=torch.bfloat16), w)
    assert ops.linear_fp8(torch.zeros(3, 200, device="cuda", dtype=torch.bfloat16), w.detach()).shape == (3, 7)


# ------------------------------------------------------------------------------ together
@pytest.mark.parametrize("T,E,k", [(1, 8, 1), (77, 8, 3), (300, 64, 8), (129, 320, 6), (1000, 16, 2), (40, 1024, 32)])
def test_moe_ffn_for_any_number_of_experts_per_token(T, E, k):
    D, F = 128, 256
    x = torch.randn(T, D, device="cuda").bfloat16().requires_grad_()
    w1, w3 = ((torch.randn(E, F, D, device="cuda") * 0.08).bfloat16().requires_grad_() for _ in range(2))
    w2 = (torch.randn(E, D, F, device="cuda") * 0.06).bfloat16().requires_grad_()
    weights, idx = ops.route_topk(torch.randn(T, E, device="cuda"), k, score="sigmoid")
    weights.requires_grad_()
    y = ops.moe_ffn(x, weights, idx, w1, w2, w3)
    dy = torch.randn(T, D, device="cuda").bfloat16()
    got = torch.autograd.grad(y, (x, weights, w1, w2, w3), dy)
    leaves = [t.detach().double().requires_grad_() for t in (x, weights, w1, w2, w3)]
    dx, dweights, v1, v2, v3 = leaves
    out = torch.zeros(T, D, device="cuda", dtype=torch.float64)
    for e in range(E):
        token, j = torch.nonzero(idx == e, as_tuple=True)
        if token.numel():
            h = dx[token] @ v1[e].t()
            h = h * torch.sigmoid(h) * (dx[token] @ v3[e].t())
            out = out.index_add(0, token, dweights[token, j].unsqueeze(1) * (h @ v2[e].t()))
    exact = torch.autograd.grad(out, leaves, dy.double())
    # bf16 hidden layers and outputs of the experts between products: a few roundings of 2^-8, in the 2-norm
    assert float((y.double() - out).norm() / out.norm()) < 4 * 2.0 ** -8
    for a, b in zip(got, exact):
        assert float((a.double() - b).norm() / b.norm()) < 6 * 2.0 ** -8


def test_a_block_of_all_operators_forward_and_backward():
    """Norm, gated sum and norm around a routed layer, and an 8-bit projection, as one differentiable program."""
    from b200moe.models.layers import MoELayerMulti
    T, D = 260, 256
    how = dict(score="sigmoid", groups=8, top_groups=4, group_score=2, balance_bias=True, scale=2.5)
    with pytest.raises(ValueError):             # the product of the router and its gradients do not take 32 experts
        MoELayerMulti(D, 384, k=4, num_expert_per_node=32, routing=how).cuda()(torch.zeros(T, D, device="cuda").bfloat16())
    layer = MoELayerMulti(D, 384, k=4, num_expert_per_node=64, routing=how).cuda()
    layer.router.compute_weight = layer.router.weight.detach().bfloat16().requires_grad_()
    layer.expert_bias.copy_(torch.randn(64) * 0.05)
    x = torch.randn(T, D, device="cuda").bfloat16().requires_grad_()
    wd, w, gate = (torch.rand(D, device="cuda").add_(0.5).requires_grad_() for _ in range(3))
    proj = (torch.randn(512, D, device="cuda") * 0.05).bfloat16().requires_grad_()
    leaves = (x, wd, w, gate, proj, layer.router.compute_weight, layer.experts.w1)

    def program():
        delta, aux = layer(ops.rmsnorm(x, w), return_aux_loss=True)
        summed, normed = ops.gated_add_rmsnorm(x, delta, wd, w, gate=gate, residual_scale=0.9)
        return ops.linear_fp8(normed, proj).float().square().mean() + summed.float().square().mean() + 0.01 * aux

    loss = program()
    grads = torch.autograd.grad(loss, leaves)
    assert all(bool(torch.isfinite(g).all()) and bool(g.any()) for g in grads)
    # against differences: the norms' gains move the loss by what their gradients say; the choice of experts and the 8-bit
    # grids make steps of their own, which a gain of the branch's norm and the gate (behind both) see through the last product only
    assert torch.equal(program(), loss)
    for leaf, grad in ((gate, grads[3]), (wd, grads[1])):
        direction = torch.sign(grad.detach())
        step = 0.05
        with torch.no_grad():
            leaf.add_(step * direction)
            high = float(program())
            leaf.sub_(2 * step * direction)
            low = float(program())
            leaf.add_(step * direction)
        slope = float((grad.double() * direction.double()).sum())
        assert abs((high - low) / (2 * step) - slope) < 0.05 * abs(slope), (high, low, slope)


@pytest.fixture
def in_python(monkeypatch):
    """Runs a function with the nodes in Python, which also take what the C++ nodes leave to them."""
    from b200moe.ops import dense, fp8, moe

    def run(f):
        with monkeypatch.context() as m:
            for module in (dense, fp8, moe):
                m.setattr(module, "cpp_nodes", lambda *_: None)
            return f()
    return run


def _same(a, b):
    assert len(a) == len(b) and all(x.dtype == y.dtype and torch.equal(x, y) for x, y in zip(a, b))


def test_cpp_nodes_do_what_the_python_nodes_do(in_python):
    from b200moe.ops import native
    assert native.nodes() is not None
    logits = torch.randn(130, 96, device="cuda").bfloat16().requires_grad_()
    bias, g = torch.randn(96, device="cuda") * 0.1, torch.randn(130, 5, device="cuda")
    for how in (dict(score="sigmoid", bias=bias, groups=8, top_groups=3, group_score=2, scale=2.5), dict(renormalize=False), dict()):
        def route():
            weights, idx = ops.route_topk(logits, 5, **how)
            return [weights.detach(), idx, *torch.autograd.grad(weights, logits, g)]
        before = native.nodes().launches()
        _same(route(), in_python(route))
        assert native.nodes().launches() == before + 2
    for kind in ("none", "channel", "sequence", "token", "full"):
        x, delta, wd, w, gate = _norm_case(3, 41, 264, kind, torch.bfloat16, torch.float32)
        leaves = [t.requires_grad_() for t in (x, delta, wd, w) + (() if gate is None else (gate,))]
        ds, dy = torch.randn_like(x), torch.randn_like(x)
        for use in ((0, 1), (0,), (1,)):
            def norm():
                out = ops.gated_add_rmsnorm(*leaves[:4], gate=gate, residual_scale=0.8)
                return [t.detach() for t in out] + list(torch.autograd.grad([out[i] for i in use], leaves, [(ds, dy)[i] for i in use]))
            before = native.nodes().launches()
            _same(norm(), in_python(norm))
            assert native.nodes().launches() == before + 3
    x = torch.randn(2, 65, 160, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(2, 65, 264, device="cuda").bfloat16()
    for dtype in (torch.bfloat16, torch.float32):
        weight = (torch.randn(264, 160, device="cuda") * 0.1).to(dtype).requires_grad_()
        for packed in (None, ops.quantize_fp8(weight, 128)):
            def linear():
                y = ops.linear_fp8(x, weight, weight_fp8=packed)
                return [y.detach(), *torch.autograd.grad(y, (x, weight), dy)]
            before = native.nodes().launches()
            _same(linear(), in_python(linear))
            assert native.nodes().launches() > before
    weight.main_grad = torch.ones_like(weight)
    torch.autograd.backward(ops.linear_fp8(x, weight), dy)
    first = weight.main_grad.clone()
    weight.main_grad.fill_(1)
    in_python(lambda: torch.autograd.backward(ops.linear_fp8(x, weight), dy))
    assert torch.equal(first, weight.main_grad) and weight.grad is None
    a, sa = _operand(33, 160, 1)
    b, sb = _operand(50, 160, 128)
    _same([ops.matmul_fp8(a, sa, b, sb)], [in_python(lambda: ops.matmul_fp8(a, sa, b, sb))])


def test_gradients_are_not_differentiated_twice(in_python):
    logits = torch.randn(9, 16, device="cuda", requires_grad=True)
    x = torch.randn(4, 64, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    weight = torch.randn(32, 64, device="cuda").bfloat16().requires_grad_()
    for f in (lambda: (ops.route_topk(logits, 3)[0], logits), lambda: (ops.gated_add_rmsnorm(x, x, w, w)[1], w),
              lambda: (ops.linear_fp8(x, weight), x)):
        for run in (lambda f: f(), in_python):
            out, leaf = run(f)
            (grad,) = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                grad.float().sum().backward()


def test_refusals_reach_the_caller_through_the_nodes():
    x = torch.zeros(4, 12, device="cuda")
    for bad in (dict(k=0), dict(k=13), dict(k=2, score="relu"), dict(k=2, groups=5), dict(k=7, groups=4, top_groups=2),
                dict(k=2, scale=0.0), dict(k=2, bias=torch.zeros(11, device="cuda")), dict(k=2, bias=torch.zeros(12))):
        with pytest.raises(ValueError):
            ops.route_topk(x, **bad)
    with pytest.raises(TypeError):
        ops.route_topk(x.double(), 2)
    w = torch.ones(12, device="cuda")
    for bad in (dict(gate=torch.ones(11, device="cuda")), dict(eps=0.0), dict(residual_scale=math.inf), dict(gate=torch.ones(12))):
        with pytest.raises(ValueError):
            ops.gated_add_rmsnorm(x, x, w, w, **bad)
    with pytest.raises(TypeError):
        ops.gated_add_rmsnorm(x.double(), x.double(), w, w)

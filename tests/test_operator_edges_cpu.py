"""Routing, gated residual norm and 8-bit products: sizes and operands at the edge of what they take."""
import ctypes
import math
import os

import pytest
import torch

I, L, F, P = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p
REFUSED = -10


@pytest.fixture
def library():
    """The kernels' library without a GPU, where a call that it does not refuse fails at its launch and starts nothing."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "b200moe", "_C", "libb200moe.so")
    if torch.cuda.is_available() or not os.path.exists(path):
        pytest.skip("for a machine without a GPU and with the library built")
    try:
        return ctypes.CDLL(path)
    except OSError as error:
        pytest.skip(str(error))


def test_gated_norm_refuses_rows_whose_counters_would_overflow(library):
    null = P(None)

    def forward(rows, D):
        return library.b2_gated_norm_fwd(*[null] * 9, I(rows), I(D), I(1), I(1), I(0), I(0), F(1), F(1e-5), null, null)

    def backward(rows, D):
        return library.b2_gated_norm_bwd(*[null] * 15, I(rows), I(D), I(1), I(1), I(0), I(0), F(1), null, null)

    for call in (forward, backward):
        for D in (1, 8):
            for rows in (2 ** 31 - 2 ** 16 + 1, 2 ** 31 - 2, 2 ** 31 - 1):
                assert call(rows, D) == REFUSED
            assert call(2 ** 31 - 2 ** 16, D) != REFUSED


def test_gated_norm_workspace_is_no_larger_than_the_tensor_for_short_sequences(library):
    library.b2_gated_norm_bwd_floats.restype = L
    rows = 2 ** 20 * 3
    for D in (64, 512, 1024, 4096):
        for seq in (2, 3, 4, 6, 8, 16, 512):
            per_sequence = library.b2_gated_norm_bwd_floats(I(rows), I(D), I(seq), I(2))
            assert 0 < per_sequence - library.b2_gated_norm_bwd_floats(I(rows), I(D), I(seq), I(1)) < 2 * rows * D
            if seq & (seq - 1) == 0:
                assert per_sequence <= rows * D


def test_fp8_refuses_sizes_that_whole_tiles_round_up_beyond_32_bits(library):
    null, large = P(None), 2 ** 31 - 255

    def product(M, N, K):
        return library.b2_gemm_fp8(*[null] * 5, I(M), I(N), I(K), *[L(16)] * 2, *[L(1)] * 4, I(0), null, null)

    def quantize(M, K):
        pitch = (K + 15) // 16 * 16
        return library.b2_quantize_fp8(null, I(1), null, null, L(M), I(K), L(K), L(pitch), L(M), I(1), null)

    for sizes in ((large, 1, 1), (1, large, 1), (1, 1, large), (1, 2 ** 31 - 128, 1)):
        assert product(*sizes) == REFUSED
    assert quantize(large, 1) == quantize(1, large) == REFUSED
    from b200moe import ops
    one = torch.zeros(1, 1, dtype=torch.bfloat16)
    for shape in ((large, 1), (1, 2 ** 31 - 128)):
        with pytest.raises(ValueError, match="rows or columns"):
            ops.quantize_fp8(one.expand(shape))
        with pytest.raises(ValueError, match="rows or columns"):
            ops.linear_fp8(one.expand(1, shape[1]), one.expand(shape))
    with pytest.raises(ValueError, match="rows"):
        ops.linear_fp8(one.expand(large, 1), one)


def test_moe_ffn_refuses_operands_that_do_not_belong_together():
    from b200moe import ops
    x, experts = torch.randn(5, 16), [torch.randn(4, 24, 16), torch.randn(4, 16, 24), torch.randn(4, 24, 16)]
    weights, idx = ops.route_topk(torch.randn(5, 4), 3)
    assert ops.moe_ffn(x, weights, idx, *experts).shape == (5, 16)
    for bad in ((x, weights[:, :1], idx), (x, weights, idx[:, :2]), (x[:4], weights, idx), (x, weights[:4], idx[:4]),
                (x, weights.flatten(), idx.flatten()), (x[None], weights, idx)):
        with pytest.raises(ValueError, match="belong together"):
            ops.moe_ffn(*bad, *experts)


FACTORS = [1e300, -1e39, math.inf, math.nan]             # none of them is a number of fp32


def test_factors_are_numbers_of_fp32():
    from b200moe import ops
    x, w = torch.randn(3, 8), torch.ones(8)
    for bad in FACTORS + [0.0, 1e-60]:
        with pytest.raises(ValueError, match="scale"):
            ops.route_topk(x, 2, scale=bad)
    for bad in FACTORS:
        with pytest.raises(ValueError, match="residual_scale"):
            ops.gated_add_rmsnorm(x, x, w, w, residual_scale=bad)
    for bad in FACTORS + [0.0, 1e-60, -1e-5]:
        with pytest.raises(ValueError, match="eps"):
            ops.gated_add_rmsnorm(x, x, w, w, eps=bad)
    assert ops.gated_add_rmsnorm(x, x, w, w, residual_scale=0.0)[0].shape == x.shape

"""Routing, gated residual norm and 8-bit products on the GPU where equal, close, far and empty operands meet."""
import pytest
import torch

from b200moe import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _native():
    from b200moe.ops import native
    native.require()
    torch.manual_seed(12)
    yield
    native.check_status()


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

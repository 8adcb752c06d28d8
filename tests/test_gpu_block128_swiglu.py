"""GPU: the block-128 SwiGLU quantizer at gates far below 0 and on operands off their alignment.  Tolerances as in test_gpu_block128.py."""
import pytest
import torch

from tests.test_gpu_block128 import _check_codes

pytestmark = pytest.mark.gpu


def _h(gate, up):
    """silu(gate) * up in 64 bits."""
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def _off_alignment(x):
    """The same values in rows that begin 2 bytes off a 16-byte boundary."""
    rows, cols = x.shape
    raw = torch.empty(rows, cols + 8 + (-cols) % 8, dtype=x.dtype, device=x.device)[:, 1: cols + 1]
    raw.copy_(x)
    return raw


@pytest.mark.parametrize("cols", [256, 1027])
@pytest.mark.parametrize("fmt", [0, 1])
def test_far_gates_with_large_factors(cuda, cols, fmt):
    """silu(g) below the range of f32's normal numbers, brought back by a factor: the only elements of their blocks, and beside ordinary ones."""
    from oxicuda_b200.quant import swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(cols)
    for low in (-17.0, -60.0, -86.0, -88.0, -90.0, -96.0, -104.0, -120.0):
        # |silu(low)| * size is about 1 where bf16 has such a factor
        size = min(1.0 / abs(_h(torch.tensor([low]), torch.tensor([1.0])).item()), 2.0 ** 127)
        gate, up = [torch.randn(5, cols, device=cuda, generator=g) for _ in range(2)]
        gate[1:3] = low * (1 + 0.002 * torch.rand(2, cols, device=cuda, generator=g))
        up[1:3] *= size / 4
        gate[3, ::5] = low
        up[3, ::5] = size
        gate, up = gate.to(torch.bfloat16), up.clamp(-3e38, 3e38).to(torch.bfloat16)
        for a, b in ((gate, up), (_off_alignment(gate), _off_alignment(up))):
            codes, scales = swiglu_quantize_fp8_block128(a, b, fmt=fmt)
            _check_codes(_h(gate, up), codes, scales, fmt)

"""GPU: the block-128 SwiGLU quantizer at gates far below 0 and on operands off their alignment.  Tolerances as in test_gpu_block128.py."""
import pytest
import torch

from tests.test_gpu_block128 import _check_codes

pytestmark = pytest.mark.gpu


def _h(gate, up):
    """silu(gate) * up in 64 bits."""
    g = gate.double()
    return g / (1 + torch.exp(-g)) * up.double()


def _check_scales(h, scales, fmt):
    rows, cols = h.shape
    nb = -(-cols // 128)
    want = torch.nn.functional.pad(h, (0, nb * 128 - cols)).view(rows, nb, 128).abs().amax(dim=2) / (448.0, 57344.0)[fmt]
    assert scales.shape == (rows, nb) and ((scales.double() - want).abs() <= 1e-5 * want).all()


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


@pytest.mark.parametrize("fmt,rounding", [(0, 1), (0, 0), (1, 1), (1, 0)])
@pytest.mark.parametrize("rows,cols", [(1, 128), (700, 4096), (33, 200)])
def test_the_same_values_give_the_same_bits_off_their_alignment(cuda, fmt, rounding, rows, cols):
    """Rows that the vector loads cannot take go through another kernel: codes and scales are the same bits."""
    from oxicuda_b200.quant import swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(rows + cols + 2 * fmt + rounding)
    gate, up = [(2 * torch.randn(rows, cols, device=cuda, generator=g)).to(torch.bfloat16) for _ in range(2)]
    if rows > 1:
        gate[1] *= 30                                               # far gates, alone and beside ordinary ones
        gate[2, ::7] = -90.0
        up[2, ::7] = 1e38
        gate[3] *= 2.0 ** -110                                      # blocks next to f32's smallest numbers
        gate[4, 5], up[5, 6], gate[6, 7] = float("nan"), float("inf"), -float("inf")
        gate[7] = 0
    a = swiglu_quantize_fp8_block128(gate, up, fmt=fmt, rounding=rounding)
    b = swiglu_quantize_fp8_block128(_off_alignment(gate), _off_alignment(up), fmt=fmt, rounding=rounding)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_codes_off_their_alignment_are_those_of_the_exact_quotients(cuda):
    from oxicuda_b200.quant import swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(5)
    gate, up = [_off_alignment((1.5 * torch.randn(1000, 4096, device=cuda, generator=g)).to(torch.bfloat16)) for _ in range(2)]
    codes, _ = swiglu_quantize_fp8_block128(gate, up)
    h = _h(gate, up).view(1000, 32, 128)
    q = (h * (448.0 / h.abs().amax(dim=2, keepdim=True))).view(1000, 4096)
    grid = torch.arange(127, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn).double()
    hi = torch.searchsorted(grid, q.abs()).clamp(1, 126)
    mid = (grid[hi] + grid[hi - 1]) / 2
    want = torch.where(q.abs() > mid, grid[hi], grid[hi - 1]) * torch.sign(q)
    clear = ((q.abs() - mid).abs() > 2.0 ** -24 * q.abs()) & (q.abs() >= 2.0 ** -6)     # 2^-24: the rounding to f32 in front of the encoder
    assert torch.equal(codes.view(torch.float8_e4m3fn).double()[clear], want[clear])


@pytest.mark.parametrize("fmt", [0, 1])
@pytest.mark.parametrize("cols", [384, 133])
def test_reference_rounding(cuda, fmt, cols):
    """The truncating codec gives the codes that it gives for the same quotients, off by a whole step at most where its codes stand for what they
    stand for here: below the normal range its 0 | mantissa is 2^(1 - bias) (1 + m / 2^bits), and from 2^8 on its E4M3 code is the largest.  The
    largest element of a block is left out: its quotient is the format's largest value, a boundary of the truncation, but for the roundings."""
    from oxicuda_b200.quant import Fp8Codec, swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(cols + fmt)
    gate, up = [torch.randn(40, cols, device=cuda, generator=g).to(torch.bfloat16) for _ in range(2)]
    h = _h(gate, up)
    codes, scales = swiglu_quantize_fp8_block128(gate, up, fmt=fmt, rounding=0)
    _check_scales(h, scales, fmt)
    q = h / scales.double().repeat_interleave(128, 1)[:, :cols]
    step, least = ((2.0 ** -3, 2.0 ** -6), (2.0 ** -2, 2.0 ** -14))[fmt]
    value = codes.view((torch.float8_e4m3fn, torch.float8_e5m2)[fmt]).double()
    normal = (q.abs() >= least * (1 + 1e-5)) & (q.abs() < (256.0, 57344.0)[fmt] * (1 - 1e-5))
    assert ((value - q).abs() <= (step + 1e-5) * q.abs())[normal].all() and normal.double().mean() > 0.9
    want = (Fp8Codec.e4m3("ref") if fmt == 0 else Fp8Codec.e5m2("ref")).encode(q.float().reshape(-1)).view(40, cols)
    differ = (want != codes) & (q.abs() < (448.0, 57344.0)[fmt] * (1 - 1e-5))
    assert differ.float().mean() <= 0.001                   # quotients that lie on a boundary of the truncation in one of the two

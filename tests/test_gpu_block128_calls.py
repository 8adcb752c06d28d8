"""GPU: block-128 calls with operands as programs hold them: strided weights, weights written right before the call.  Tolerances as in
test_gpu_block128.py."""
import pytest
import torch

from tests.test_gpu_block128 import _check_product, _operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 17, 60, 128, 200])
def test_strided_weights(cuda, M):
    """A transposed weight and a column shard of a wider one give the bits of their contiguous copies, with new weights in every call."""
    from oxicuda_b200.blas import gemm_fp8_block128
    N, K = 640, 2048
    for seed in range(4):
        a, w, sa, sw = _operands(cuda, M, N, K, 0, 100 * M + seed)
        want = gemm_fp8_block128(a, w, sa, sw)
        _check_product(a, w, sa, sw, want)
        torch.cuda.synchronize()
        turned = torch.empty(K, N, dtype=torch.uint8, device=cuda)
        turned.copy_(w.t())
        assert torch.equal(gemm_fp8_block128(a, turned.t(), sa, sw), want)
        wide = torch.full((N, 3 * K), 0x7F, dtype=torch.uint8, device=cuda)
        wide[:, K: 2 * K] = w
        assert torch.equal(gemm_fp8_block128(a, wide[:, K: 2 * K], sa, sw), want)


@pytest.mark.parametrize("M", [1, 40, 128])
def test_weights_written_right_before_the_product(cuda, M):
    """With static_weights off the few-token product reads nothing before the kernel that writes its weights has completed."""
    from oxicuda_b200 import _lib as L
    from oxicuda_b200.blas import gemm_fp8_block128
    h = L.default_handle()
    N, K = 8192, 2048
    sets = [_operands(cuda, M, N, K, 0, 7 * M + i) for i in range(3)]
    want = [gemm_fp8_block128(*s) for s in sets]
    for s, x in zip(sets, want):
        _check_product(*s, x)
    torch.cuda.synchronize()
    w = torch.full((N, K), 0x7F, dtype=torch.uint8, device=cuda)
    h.set_static_weights(False)
    try:
        for (a, new, sa, sw), x in zip(sets, want):
            w.copy_(new)                                            # same stream, no synchronisation
            assert torch.equal(gemm_fp8_block128(a, w, sa, sw), x)
    finally:
        h.set_static_weights(True)
    h.check()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("fmt", [0, 1])
def test_scales_of_every_block(cuda, block_rows, fmt):
    """quantize_fp8_blocks: every block's scale is its own absmax / max_val (1 for zeros), short blocks at the edges included."""
    from oxicuda_b200.quant import quantize_fp8_blocks
    g = torch.Generator(device=cuda).manual_seed(3)
    for dtype in (torch.float32, torch.bfloat16):
        for rows, cols in ((256, 384), (130, 200), (1, 1)):
            x = (torch.randn(rows, cols, device=cuda, generator=g) * torch.exp(3 * torch.randn(rows, 1, device=cuda, generator=g))).to(dtype)
            if cols > 128:
                x[:128, :128] = 0
            codes, scales = quantize_fp8_blocks(x, block_rows, fmt=fmt)
            rb, cb = -(-rows // block_rows), -(-cols // 128)
            b = torch.nn.functional.pad(x.double(), (0, cb * 128 - cols, 0, rb * block_rows - rows)).view(rb, block_rows, cb, 128)
            top = b.abs().amax(dim=(1, 3))
            want = torch.where(top > 0, top / (448.0, 57344.0)[fmt], torch.ones_like(top))
            assert scales.shape == (rb, cb) and ((scales.double() - want).abs() <= 2.0 ** -23 * want).all()   # a division in f32: half a step
            # the largest element of a block is the largest code: its quotient is max_val but for two roundings, 2^-23 of it
            full = torch.nn.functional.pad(codes, (0, cb * 128 - cols, 0, rb * block_rows - rows)).view(rb, block_rows, cb, 128) & 127
            assert (full.amax(dim=(1, 3)) == torch.where(top > 0, (126, 123)[fmt], 0)).all()


@pytest.mark.parametrize("new,old,heads", [(1, 9000, 8), (1, 50, 80), (4, 3000, 8), (150, 0, 8), (40, 9000, 8)])
def test_attention_over_its_own_queries(cuda, new, old, heads):
    """out may be q itself: every CTA of a row tile has read its rows before one of them writes."""
    from tests.test_gpu_kv8 import _pages, _q
    lens = [old + new, new + 7]
    cache, table = _pages(cuda, lens, 32, 2, 128, new)
    q = _q(cuda, 2 * new, heads, 128, new)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    starts = None if new == 1 else torch.tensor([0, new, 2 * new], dtype=torch.int32, device=cuda)
    want = cache.attend(q, seq, table, q_starts=starts)
    for _ in range(5):
        x = q.clone()
        assert cache.attend(x, seq, table, q_starts=starts, out=x) is x and torch.equal(x, want)

"""GPU: the block-128 FP8 operators (norm, SwiGLU, product) against plain statements in 64 bits.

Tolerances.  Codes: E4M3 rounds by at most half a step, 2^-4 of the value or 2^-10 below 2^-6 (E5M2: 2^-3, 2^-17 below 2^-14); the f32
arithmetic in front of it (sums of squares over at most 64 terms per lane and a tree, square root, three products) moves the value by less
than 1e-5 of itself.  Products: bf16 rounds by 2^-8 of the value, and each of the 128 + K / 128 additions of an f32 accumulator by at most
one step, 2^-23, of a partial sum that is at most sum |a w|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

MAX = {0: 448.0, 1: 57344.0}
KIND = {0: torch.float8_e4m3fn, 1: torch.float8_e5m2}


def _values(codes, fmt=0):
    return codes.view(KIND[fmt]).double()


def _spread(scales, rows_per, rows, cols):
    return scales.double().repeat_interleave(rows_per, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _check_codes(y, codes, scales, fmt=0, slack=1e-5, rounding=1):
    rows, cols = y.shape
    nb = -(-cols // 128)
    amax = torch.nn.functional.pad(y, (0, nb * 128 - cols)).view(rows, nb, 128).abs().amax(dim=2)
    want = torch.where(amax > 0, amax / MAX[fmt], torch.ones_like(amax)).clamp(min=2.0 ** -126)
    assert scales.shape == (rows, nb)
    assert ((scales.double() - want).abs() <= slack * want).all()
    q = y / _spread(scales, 1, rows, cols)
    half = {0: (2.0 ** -4, 2.0 ** -10), 1: (2.0 ** -3, 2.0 ** -17)}[fmt]
    steps = 1.0 if rounding == 1 else 2.0                  # the truncating codec is off by a whole step
    err = (_values(codes, fmt) - q).abs()
    assert (err <= steps * (half[0] * q.abs()).clamp(min=half[1]) + slack * q.abs()).all()


@pytest.mark.parametrize("rows,cols,residual,want_y", [
    (1, 128, False, True), (3, 136, True, True), (5, 8, True, False), (2, 4096, True, True), (7, 8192, False, False), (300, 1024, True, True),
    (310, 2056, True, False), (301, 8192, True, False), (2, 32768, True, False), (2, 32776, True, True), (4, 131, True, True), (3, 1, False, True)])
def test_norm_against_f64(cuda, rows, cols, residual, want_y):
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(rows * 1000 + cols)
    x = (torch.randn(rows, cols, device=cuda, generator=g) * torch.exp(torch.randn(cols, device=cuda, generator=g))).to(torch.bfloat16)
    res = torch.randn(rows, cols, device=cuda, generator=g).to(torch.bfloat16) if residual else None
    gamma = (1 + 0.2 * torch.randn(cols, device=cuda, generator=g)).to(torch.bfloat16)
    if cols > 256:
        x[:, 128:256] = 0                                  # a block of zeros
        if residual:
            res[:, 128:256] = 0
    want_res = (res.float() + x.float()).to(torch.bfloat16) if residual else None
    v = (want_res if residual else x).double()
    y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + 1e-5) * gamma.double()
    got = rms_norm_quantize_fp8_block128(x, gamma, 1e-5, residual=res, want_y=want_y)
    if residual:
        assert torch.equal(res, want_res)
    _check_codes(y, got[0], got[1])
    if cols > 256:
        assert (got[1][:, 1] == 1).all() and (got[0][:, 128:256] == 0).all()
    if want_y:
        assert ((got[2].double() - y).abs() <= (2.0 ** -8 + 1e-5) * y.abs()).all()


@pytest.mark.parametrize("fmt,rounding", [(0, 0), (1, 0), (1, 1)])
def test_norm_and_swiglu_formats(cuda, fmt, rounding):
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    from oxicuda_b200.quant import swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(5)
    for cols in (384, 133):                                # vector and plain kernels
        x = torch.randn(6, cols, device=cuda, generator=g).to(torch.bfloat16)
        gamma = torch.ones(cols, device=cuda, dtype=torch.bfloat16)
        y = x.double() / torch.sqrt((x.double() ** 2).mean(dim=1, keepdim=True) + 1e-5)
        codes, scales = rms_norm_quantize_fp8_block128(x, gamma, 1e-5, fmt=fmt, rounding=rounding)
        if rounding == 1:
            _check_codes(y, codes, scales, fmt)
        else:                                              # the reference's codec, as the per-row quantizer applies it to the same values
            from oxicuda_b200.quant import Fp8Codec
            q = (y / _spread(scales, 1, 6, cols)).float()
            want = (Fp8Codec.e4m3("ref") if fmt == 0 else Fp8Codec.e5m2("ref")).encode(q.reshape(-1)).view(6, cols)
            assert (want != codes).float().mean() <= 0.01  # values that sit on a boundary of the truncation in one of the two
        up = torch.randn(6, cols, device=cuda, generator=g).to(torch.bfloat16)
        if rounding == 1:
            h = x.double() * torch.sigmoid(x.double()) * up.double()
            _check_codes(h, *swiglu_quantize_fp8_block128(x, up, fmt=fmt), fmt)


@pytest.mark.parametrize("cols", [1024, 8192, 16384, 1031])
def test_norm_far_from_one(cuda, cols):
    """Rows and weights whose product leaves the range of f32, or comes near its ends, beside ordinary ones."""
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(cols)
    size = torch.tensor([1.0, 2.0 ** -60, 2.0 ** 50, 2.0 ** -30, 2.0 ** 30, 1.0], device=cuda)
    x = (torch.randn(6, cols, device=cuda, generator=g) * size[:, None]).to(torch.bfloat16)
    gain = torch.exp2(torch.tensor([0.0, -90.0, 100.0, -60.0, 40.0, -20.0, 20.0, 0.0], device=cuda)).repeat_interleave(-(-cols // 8))[:cols]
    gamma = (torch.randn(cols, device=cuda, generator=g).clamp(min=0.05) * gain).to(torch.bfloat16)
    for eps in (0.0, 1e-5):
        codes, scales, yy = rms_norm_quantize_fp8_block128(x, gamma, eps, want_y=True)
        v = x.double()
        y = v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps) * gamma.double()
        _check_codes(y, codes, scales)
        assert ((yy.double() - y).abs() <= (2.0 ** -8 + 1e-5) * y.abs() + 2.0 ** -126).all()


def test_norm_codes_are_those_of_the_exact_quotients(cuda):
    """The quotient is rounded once before it is encoded: a code differs from the exact quotient's only where that lies within 2^-23 of itself
    from the middle between two codes."""
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(77)
    x, gamma = torch.randn(200, 4096, device=cuda, generator=g).to(torch.bfloat16), (1 + 0.1 * torch.randn(4096, device=cuda, generator=g)).to(torch.bfloat16)
    codes, _ = rms_norm_quantize_fp8_block128(x, gamma, 1e-5)
    w = (x.double() * gamma.double()).view(200, 32, 128)
    q = (w * (448.0 / w.abs().amax(dim=2, keepdim=True))).view(200, 4096)
    grid = torch.arange(127, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn).double()
    hi = torch.searchsorted(grid, q.abs()).clamp(1, 126)
    mid = (grid[hi] + grid[hi - 1]) / 2
    clear = (q.abs() - mid).abs() > 2.0 ** -23 * q.abs()
    want = torch.where(q.abs() > mid, grid[hi], grid[hi - 1]) * torch.sign(q)
    assert torch.equal(_values(codes)[clear], want[clear]) and clear.double().mean() > 0.999


def test_swiglu_codes_are_those_of_the_exact_quotients(cuda):
    """Elements next to a border between two codes are made again in 64 bits: above 2^-6 every code is the exact quotient's."""
    from oxicuda_b200.quant import swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(5)
    gate, up = [(1.5 * torch.randn(1000, 4096, device=cuda, generator=g)).to(torch.bfloat16) for _ in range(2)]
    codes, _ = swiglu_quantize_fp8_block128(gate, up)
    h = (gate.double() * up.double() / (1 + torch.exp(-gate.double()))).view(1000, 32, 128)
    q = (h * (448.0 / h.abs().amax(dim=2, keepdim=True))).view(1000, 4096)
    grid = torch.arange(127, dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn).double()
    hi = torch.searchsorted(grid, q.abs()).clamp(1, 126)
    mid = (grid[hi] + grid[hi - 1]) / 2
    want = torch.where(q.abs() > mid, grid[hi], grid[hi - 1]) * torch.sign(q)
    clear = ((q.abs() - mid).abs() > 2.0 ** -24 * q.abs()) & (q.abs() >= 2.0 ** -6)     # 2^-24: the rounding to f32 in front of the encoder
    assert torch.equal(_values(codes)[clear], want[clear])


def test_norm_of_non_finite_rows(cuda):
    """A row with a NaN is NaN throughout, a row with an infinity zeros and NaN (x / inf); the rows beside them are untouched."""
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(9)
    for cols in (512, 131):
        x = torch.randn(4, cols, device=cuda, generator=g).to(torch.bfloat16)
        clean = rms_norm_quantize_fp8_block128(x, torch.ones(cols, device=cuda, dtype=torch.bfloat16), 1e-5)
        x[1, 3] = float("nan")
        x[2, 5] = float("inf")
        codes, scales = rms_norm_quantize_fp8_block128(x, torch.ones(cols, device=cuda, dtype=torch.bfloat16), 1e-5)
        v = _values(codes)
        assert torch.isnan(v[1]).all() and torch.isnan(v[2, 5])
        keep = torch.ones(cols, dtype=torch.bool, device=cuda)
        keep[5] = False
        assert (v[2][keep] == 0).all()
        for r in (0, 3):
            assert torch.equal(codes[r], clean[0][r]) and torch.equal(scales[r], clean[1][r])


@pytest.mark.parametrize("rows,cols", [(1, 128), (1, 14336), (3, 200), (5, 1), (17, 1032), (130, 28672), (33, 131)])
def test_swiglu_against_f64(cuda, rows, cols):
    from oxicuda_b200.quant import swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(rows + cols)
    gu = (2 * torch.randn(rows, 2 * cols, device=cuda, generator=g)).to(torch.bfloat16)
    gu[0, : min(cols, 4)] = torch.tensor([-100.0, 100.0, -3e38, 0.0], device=cuda)[: min(cols, 4)]
    gate, up = gu[:, :cols], gu[:, cols:]
    h = gate.double() * torch.sigmoid(gate.double()) * up.double()
    _check_codes(h, *swiglu_quantize_fp8_block128(gate, up))                       # halves of one tensor
    a, b = swiglu_quantize_fp8_block128(gate.contiguous(), up.contiguous()), swiglu_quantize_fp8_block128(gate, up)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_blocks(cuda, block_rows):
    from oxicuda_b200.quant import quantize_fp8_blocks
    g = torch.Generator(device=cuda).manual_seed(3)
    for rows, cols in ((256, 384), (130, 200)):
        x = torch.randn(rows, cols, device=cuda, generator=g)
        codes, scales = quantize_fp8_blocks(x, block_rows)
        assert scales.shape == (-(-rows // block_rows), -(-cols // 128))
        s = _spread(scales, block_rows, rows, cols)
        q = x.double() / s
        assert ((_values(codes) - q).abs() <= (2.0 ** -4 * q.abs()).clamp(min=2.0 ** -10) + 1e-6 * q.abs()).all()
        assert ((codes & 127) == 126).any()                # every block's largest element is at the top of the range


def _operands(cuda, M, N, K, fmt, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    a = (torch.randn(M, K, device=cuda, generator=g) * 60).clamp(-MAX[fmt], MAX[fmt]).to(KIND[fmt]).view(torch.uint8)
    w = (torch.randn(N, K, device=cuda, generator=g) * 60).clamp(-MAX[fmt], MAX[fmt]).to(KIND[fmt]).view(torch.uint8)
    kb = -(-K // 128)
    sa = torch.exp(2 * torch.randn(M, kb, device=cuda, generator=g)) * 1e-2
    sw = torch.exp(2 * torch.randn(-(-N // 128), kb, device=cuda, generator=g)) * 1e-3
    return a, w, sa, sw


def _check_product(a, w, sa, sw, out, fmt=0):
    M, K = a.shape
    N = w.shape[0]
    da, dw = _values(a, fmt) * _spread(sa, 1, M, K), _values(w, fmt) * _spread(sw, 128, N, K)
    ref, size = da @ dw.t(), da.abs() @ dw.abs().t()
    tol = (128 + -(-K // 128)) * 2.0 ** -23 * size
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    assert out.shape == (M, N)
    assert ((out.double() - ref).abs() <= tol).all()


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 130, 128), (3, 64, 16), (1, 4096, 4096), (5, 257, 1040), (16, 1024, 2048), (17, 512, 144), (31, 8192, 512),
          (33, 384, 4096), (64, 1000, 1024), (65, 129, 256), (100, 2304, 1280), (127, 127, 1152), (128, 256, 8192), (129, 256, 128), (129, 300, 400), (200, 512, 4096),
          (256, 256, 256), (257, 513, 1024), (511, 768, 640), (700, 4096, 2176), (1025, 1152, 528), (2048, 2304, 1024), (40, 72, 100), (130, 136, 129)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_against_f64(cuda, M, N, K):
    from oxicuda_b200.blas import gemm_fp8_block128
    a, w, sa, sw = _operands(cuda, M, N, K, 0, M + N + K)
    for dtype in (torch.bfloat16, torch.float32):
        _check_product(a, w, sa, sw, gemm_fp8_block128(a, w, sa, sw, out_dtype=dtype))


@pytest.mark.parametrize("M,N,K", [(4, 256, 512), (60, 640, 1024), (300, 512, 384), (9, 40, 100)])
def test_product_e5m2(cuda, M, N, K):
    from oxicuda_b200 import _lib as L
    from oxicuda_b200.blas import gemm_fp8_block128
    a, w, sa, sw = _operands(cuda, M, N, K, 1, 7)
    _check_product(a, w, sa, sw, gemm_fp8_block128(a, w, sa, sw, out_dtype=torch.float32, fmt=L.FP8_E5M2), 1)


def test_product_zero_and_extreme_scales(cuda):
    """Blocks whose scale is 0, or so far apart that one block is the whole sum."""
    from oxicuda_b200.blas import gemm_fp8_block128
    for M in (8, 200):
        a, w, sa, sw = _operands(cuda, M, 384, 1024, 0, 11)
        sa[:, 3] = 0
        sw[1] = 0
        sa[1, 2] = 1e15
        out = gemm_fp8_block128(a, w, sa, sw)
        _check_product(a, w, sa, sw, out)
        assert (out[:, 128:256] == 0).all()


def test_product_operands_off_their_alignment(cuda):
    from oxicuda_b200.blas import gemm_fp8_block128
    a, w, sa, sw = _operands(cuda, 70, 200, 256, 0, 13)
    raw = torch.empty(70 * 256 + 3, dtype=torch.uint8, device=cuda)[3:].view(70, 256)
    raw.copy_(a)
    out = torch.empty(70 * 200 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(70, 200)
    _check_product(raw, w, sa, sw, gemm_fp8_block128(raw, w, sa, sw))
    gemm_fp8_block128(a, w, sa, sw, out=out)
    _check_product(a, w, sa, sw, out)
    sub = torch.empty(sa.numel() + 1, device=cuda)[1:].view_as(sa)
    sub.copy_(sa)
    for M in (70, 3):
        _check_product(a[:M], w, sub[:M], sw, gemm_fp8_block128(a[:M], w, sub[:M], sw))
    wide = torch.zeros(300, 512, dtype=torch.uint8, device=cuda)                    # columns of a wider matrix
    wide[:70, 128:384] = a
    _check_product(a, w, sa, sw, gemm_fp8_block128(wide[:70, 128:384], w, sa, sw))


def test_product_refusals_on_the_device(cuda):
    from oxicuda_b200 import _lib as L
    h = L.default_handle()
    a, w, sa, sw = _operands(cuda, 8, 128, 128, 0, 1)
    out = torch.empty(8, 128, dtype=torch.bfloat16, device=cuda)
    p = L.ptr
    for args, err in (((p(a), p(w), 0, 128, 128, 0, p(sa), p(sw), p(out), 0), L.InvalidDimension),
                      ((p(a), p(w), 8, 128, 128, 2, p(sa), p(sw), p(out), 0), L.InvalidArgument),
                      ((p(a), p(w), 8, 128, 128, 0, None, p(sw), p(out), 0), L.InvalidArgument),
                      ((p(a), p(w), 8, 128, 128, 0, p(sa), p(sw), p(a), 0), L.InvalidArgument),
                      ((p(a), p(w), 1 << 32, 128, 128, 0, p(sa), p(sw), p(out), 0), L.InvalidDimension)):
        with pytest.raises(err):
            h.call("b2q_gemm_fp8_block128", *args)
    with pytest.raises(L.EmptyInput):
        h.call("b2q_swiglu_quantize_fp8_block128_bf16", p(out), p(out), 0, 128, 128, 0, 1, p(sa), p(a))
    with pytest.raises(L.InvalidArgument):
        h.call("b2q_swiglu_quantize_fp8_block128_bf16", p(out), p(out), 8, 128, 127, 0, 1, p(sa), p(a))


def test_chain_on_side_streams_and_in_graphs(cuda):
    """norm -> product -> SwiGLU -> product on two streams at once, and as two captured graphs replayed in turn, give the eager bits."""
    from oxicuda_b200.blas import gemm_fp8_block128
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    from oxicuda_b200.quant import quantize_fp8_blocks, swiglu_quantize_fp8_block128
    g = torch.Generator(device=cuda).manual_seed(21)
    hidden, ffn = 512, 1024
    w1 = quantize_fp8_blocks(torch.randn(2 * ffn, hidden, device=cuda, generator=g) * 0.05, 128)
    w2 = quantize_fp8_blocks(torch.randn(hidden, ffn, device=cuda, generator=g) * 0.05, 128)
    gamma = torch.ones(hidden, device=cuda, dtype=torch.bfloat16)

    def step(x):
        c, s = rms_norm_quantize_fp8_block128(x, gamma, 1e-5)
        gu = gemm_fp8_block128(c, w1[0], s, w1[1])
        c, s = swiglu_quantize_fp8_block128(gu[:, :ffn], gu[:, ffn:])
        return gemm_fp8_block128(c, w2[0], s, w2[1])

    xs = [torch.randn(n, hidden, device=cuda, generator=g).to(torch.bfloat16) for n in (5, 60, 300)]
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(step(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(x))
        graphs.append(gr)
    for o in outs:
        o.zero_()
    for st, gr in zip(streams, graphs):
        with torch.cuda.stream(st):
            gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # the chain against the same steps in 64 bits from each step's own operands is what the tests above hold; here: it is finite and not zero
    assert all(torch.isfinite(o).all() and o.abs().max() > 0 for o in outs)

"""CPU: the argument checks of the block-128 FP8 operators and of the paged E4M3 cache fail before anything touches a device."""
import pytest
import torch


def _z(*shape, dtype=torch.uint8):
    return torch.zeros(*shape, dtype=dtype)


def test_gemm_block128_refusals(libb2q):
    from oxicuda_b200 import _lib, blas
    f = torch.float32
    a, w, sa, sw = _z(4, 256), _z(130, 256), _z(4, 2, dtype=f), _z(2, 2, dtype=f)
    with pytest.raises(_lib.DimensionMismatch):
        blas.gemm_fp8_block128(a, _z(130, 255), sa, sw)
    with pytest.raises(_lib.DimensionMismatch):
        blas.gemm_fp8_block128(a, w, _z(4, 1, dtype=f), sw)
    with pytest.raises(_lib.DimensionMismatch):
        blas.gemm_fp8_block128(a, w, sa, _z(1, 2, dtype=f))
    with pytest.raises(_lib.DimensionMismatch):
        blas.gemm_fp8_block128(a, w, sa.double(), sw)
    with pytest.raises(_lib.InvalidArgument):
        blas.gemm_fp8_block128(a, w, sa, sw, out_dtype=torch.float16)
    with pytest.raises(_lib.InvalidArgument):
        blas.gemm_fp8_block128(a, w, sa, sw, out=_z(4, 131, dtype=torch.bfloat16))
    with pytest.raises(_lib.InvalidArgument):
        blas.gemm_fp8_block128(a.float(), w, sa, sw)
    with pytest.raises(_lib.InvalidArgument):                       # host tensors: there is no CPU path
        blas.gemm_fp8_block128(a, w, sa, sw)


def test_producer_refusals(libb2q):
    from oxicuda_b200 import _lib, quant
    from oxicuda_b200.kv_cache import rms_norm_quantize_fp8_block128
    bf = torch.bfloat16
    x, g = _z(3, 256, dtype=bf), _z(256, dtype=bf)
    with pytest.raises(_lib.InvalidArgument):
        rms_norm_quantize_fp8_block128(x.float(), g, 1e-5)
    with pytest.raises(_lib.DimensionMismatch):
        rms_norm_quantize_fp8_block128(x, g[:255], 1e-5)
    with pytest.raises(_lib.EmptyInput):
        rms_norm_quantize_fp8_block128(x[:0], g, 1e-5)
    with pytest.raises(_lib.InvalidArgument):
        rms_norm_quantize_fp8_block128(x, g, 1e-5, residual=_z(3, 255, dtype=bf))
    with pytest.raises(_lib.InvalidArgument):
        rms_norm_quantize_fp8_block128(x, g, 1e-5, residual=_z(256, 3, dtype=bf).t())
    with pytest.raises(_lib.InvalidArgument):                       # host tensors
        rms_norm_quantize_fp8_block128(x, g, 1e-5)
    with pytest.raises(_lib.InvalidArgument):
        quant.swiglu_quantize_fp8_block128(x, x[:, :128])
    with pytest.raises(_lib.EmptyInput):
        quant.swiglu_quantize_fp8_block128(x[:0], x[:0])
    with pytest.raises(_lib.InvalidArgument):
        quant.swiglu_quantize_fp8_block128(x, x)
    with pytest.raises(_lib.InvalidArgument):
        quant.quantize_fp8_blocks(x, 64)
    with pytest.raises(_lib.EmptyInput):
        quant.quantize_fp8_blocks(x[:0], 1)


def test_paged_fp8_cache_refusals(libb2q):
    from oxicuda_b200 import _lib
    from oxicuda_b200.kv_cache import PagedFp8KvCache
    for page, d in ((8, 128), (24, 64), (256, 64), (16, 96), (64, 256)):
        with pytest.raises(_lib.UnsupportedOperation):
            PagedFp8KvCache.empty(4, page, 2, d, "cpu")
    codes, scales = _z(4, 2, 16, 64), _z(4, 2)
    for bad in ((codes[0], codes, scales, scales), (codes, codes[:3], scales, scales), (codes, codes, scales[:3], scales), (codes, codes, scales, scales.float()),
                (codes, codes.transpose(0, 1), scales, scales)):
        with pytest.raises(_lib.InvalidArgument):
            PagedFp8KvCache(*bad)
    cache = PagedFp8KvCache(codes, codes.clone(), scales, scales.clone())
    bf, i32 = torch.bfloat16, torch.int32
    k, lens, table = _z(3, 2, 64, dtype=bf), _z(3, dtype=i32), _z(3, 2, dtype=i32)
    with pytest.raises(_lib.InvalidArgument):
        cache.append(k.float(), k, lens, table)
    with pytest.raises(_lib.InvalidArgument):
        cache.append(k[:, :1], k, lens, table)
    with pytest.raises(_lib.DimensionMismatch):
        cache.append(k, k[:2], lens, table)
    with pytest.raises(_lib.InvalidArgument):
        cache.append(k, k, lens.long(), table)
    with pytest.raises(_lib.DimensionMismatch):
        cache.append(k, k, lens, table[:2])
    with pytest.raises(_lib.DimensionMismatch):                     # one token per sequence without q_starts
        cache.append(k, k, lens[:2], table[:2])
    with pytest.raises(_lib.DimensionMismatch):
        cache.append(k, k, lens, table, q_starts=_z(3, dtype=i32))
    with pytest.raises(_lib.EmptyInput):
        cache.append(k[:0], k[:0], lens[:0], table[:0])
    with pytest.raises(_lib.InvalidArgument):                       # host tensors
        cache.append(k, k, lens, table)
    q = _z(3, 4, 64, dtype=bf)
    with pytest.raises(_lib.InvalidDimension):
        cache.attend(q[:, :3], lens, table)
    with pytest.raises(_lib.InvalidArgument):
        cache.attend(q[..., :32], lens, table)
    with pytest.raises(_lib.InvalidArgument):
        cache.attend(q, lens, table, out=_z(3, 4, 32, dtype=bf))
    with pytest.raises(_lib.InvalidArgument):                       # host tensors
        cache.attend(q, lens, table)


def test_null_handle_is_refused_by_the_block128_entry_points(libb2q):
    assert libb2q.b2q_gemm_fp8_block128(None, None, None, 1, 1, 16, 0, None, None, None, 0) == 8
    assert libb2q.b2q_rms_norm_quantize_fp8_block128_bf16(None, None, None, None, 1, 1, 1e-5, 0, 1, None, None, None) == 8
    assert libb2q.b2q_swiglu_quantize_fp8_block128_bf16(None, None, None, 1, 1, 1, 0, 1, None, None) == 8
    assert libb2q.b2q_kv8_append_bf16(None, None, None, 64, 64, 1, None, None, None, 1, 1, 1, 16, 1, 64, None, None, None, None) == 8
    assert libb2q.b2q_kv8_attention_bf16(None, None, 64, 1, 1, None, None, None, 1, 1, 1, 16, 1, 64, None, None, None, None, 1.0, 0, None, None) == 8


def test_runner_recipe_is_validated(libb2q):
    from oxicuda_b200 import _lib
    from oxicuda_b200.model_runner import LlamaConfig
    LlamaConfig().validate()
    LlamaConfig(recipe="block128").validate()
    for bad in (LlamaConfig(recipe="per_block"), LlamaConfig(recipe="block128", n_heads=3, n_kv_heads=1)):
        with pytest.raises(_lib.InvalidConfig):
            bad.validate()

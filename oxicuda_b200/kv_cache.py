"""Host-side mirror of the KV-cache quantizers either side of the quantized linear path.

`KvCacheQuantizer` / `KvCacheConfig` / `QuantizedKvCache` follow crates/oxicuda-quant/src/scheme/kv_cache.rs,
`KvQuantConfig` / `QuantizedToken(s)` / `quantize_token` follow crates/oxicuda-infer/src/cache/kv_quant.rs, and
`rms_norm_quantize_fp8` is the RMSNorm of crates/oxicuda-dnn/src/norm/rms_norm.rs fused with the per-token FP8
quantizer that feeds the next linear.  Same names, argument meaning and error behaviour as the reference; the
arithmetic runs in CUDA kernels through the C ABI.  Host tensors are uploaded and results come back on the host.
"""
from __future__ import annotations

from dataclasses import dataclass
from enum import Enum

import torch

from . import _lib as L
from ._lib import default_handle, ptr
from .quant import _back, _dev


class KvAxis(Enum):
    """crates/oxicuda-quant/src/scheme/kv_cache.rs:33-38"""
    PerToken = 0
    PerChannel = 1


@dataclass
class KvCacheConfig:
    """kv_cache.rs:43-86"""
    bits: int
    axis: KvAxis

    @staticmethod
    def new(bits: int, axis: KvAxis) -> "KvCacheConfig":
        if not 2 <= bits <= 8:
            raise L.InvalidBitWidth(L.ERR_INVALID_BIT_WIDTH, f"invalid bit-width {bits}")
        return KvCacheConfig(bits, axis)

    @staticmethod
    def keys_int8() -> "KvCacheConfig":
        return KvCacheConfig(8, KvAxis.PerChannel)

    @staticmethod
    def values_int8() -> "KvCacheConfig":
        return KvCacheConfig(8, KvAxis.PerToken)


@dataclass
class QuantizedKvCache:
    """kv_cache.rs:91-120.  `codes` u8 [n_tokens*head_dim]; `scales`, `zero_points` f32 [n_groups]."""
    codes: torch.Tensor
    scales: torch.Tensor
    zero_points: torch.Tensor
    n_tokens: int
    head_dim: int
    bits: int
    axis: KvAxis

    def n_groups(self) -> int:
        return self.n_tokens if self.axis == KvAxis.PerToken else self.head_dim

    def packed_bytes(self) -> int:
        return (self.codes.numel() * self.bits + 7) // 8


class KvCacheQuantizer:
    """KvCacheQuantizer, kv_cache.rs:125-283."""

    def __init__(self, config: KvCacheConfig):
        self.config = config

    def quantize(self, tensor: torch.Tensor, n_tokens: int, head_dim: int) -> QuantizedKvCache:
        """kv_cache.rs:146-221; bf16 input is quantized from its exact f32 values."""
        if tensor.numel() == 0 or n_tokens == 0 or head_dim == 0:
            raise L.EmptyInput(L.ERR_EMPTY_INPUT, "KvCacheQuantizer::quantize")
        if tensor.numel() != n_tokens * head_dim:
            raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {n_tokens * head_dim}, got {tensor.numel()}")
        bf16 = tensor.dtype == torch.bfloat16
        x, was_host = _dev(tensor.reshape(-1), torch.bfloat16 if bf16 else torch.float32)
        groups = n_tokens if self.config.axis == KvAxis.PerToken else head_dim
        codes = torch.empty(n_tokens * head_dim, dtype=torch.uint8, device=x.device)
        scales = torch.empty(groups, dtype=torch.float32, device=x.device)
        zps = torch.empty(groups, dtype=torch.float32, device=x.device)
        default_handle().call("b2q_kv_cache_quantize_bf16" if bf16 else "b2q_kv_cache_quantize_f32", ptr(x), n_tokens, head_dim,
                              self.config.bits, self.config.axis.value, ptr(codes), ptr(scales), ptr(zps))
        return QuantizedKvCache(_back(codes, was_host), _back(scales, was_host), _back(zps, was_host), n_tokens, head_dim,
                                self.config.bits, self.config.axis)

    @staticmethod
    def dequantize(cache: QuantizedKvCache, out_dtype=torch.float32) -> torch.Tensor:
        """kv_cache.rs:224-238"""
        codes, was_host = _dev(cache.codes.reshape(-1), torch.uint8)
        sc, _ = _dev(cache.scales, torch.float32)
        zp, _ = _dev(cache.zero_points, torch.float32)
        out = torch.empty(cache.n_tokens * cache.head_dim, dtype=out_dtype, device=codes.device)
        name = "b2q_kv_cache_dequantize_bf16" if out_dtype == torch.bfloat16 else "b2q_kv_cache_dequantize_f32"
        default_handle().call(name, ptr(codes), cache.n_tokens, cache.head_dim, cache.axis.value, ptr(sc), ptr(zp), ptr(out))
        return _back(out, was_host)

    def append_token(self, cache: QuantizedKvCache, row: torch.Tensor) -> None:
        """kv_cache.rs:254-282: the new row gets a group of its own; the cache grows by one token."""
        if cache.axis != KvAxis.PerToken:
            raise L.InvalidConfig(L.ERR_INVALID_CONFIG, "append_token requires a PerToken cache")
        if row.numel() != cache.head_dim:
            raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {cache.head_dim}, got {row.numel()}")
        one = KvCacheQuantizer(KvCacheConfig(cache.bits, KvAxis.PerToken)).quantize(row.to(cache.codes.device), 1, cache.head_dim)
        cache.codes = torch.cat([cache.codes, one.codes.to(cache.codes.device)])
        cache.scales = torch.cat([cache.scales, one.scales.to(cache.scales.device)])
        cache.zero_points = torch.cat([cache.zero_points, one.zero_points.to(cache.zero_points.device)])
        cache.n_tokens += 1


# ---- oxicuda-infer: crates/oxicuda-infer/src/cache/kv_quant.rs ----
@dataclass(frozen=True)
class KvQuantConfig:
    """kv_quant.rs:36-77"""
    bits: int
    symmetric: bool

    @staticmethod
    def new(bits: int, symmetric: bool) -> "KvQuantConfig":
        if bits not in (4, 8):
            raise L.InvalidConfig(L.ERR_INVALID_CONFIG, "KV quant bits must be 4 or 8")
        return KvQuantConfig(bits, symmetric)

    @staticmethod
    def int8() -> "KvQuantConfig":
        return KvQuantConfig(8, False)

    def q_range(self):
        if self.symmetric:
            half = 1 << (self.bits - 1)
            return (-(half - 1), half - 1)
        return (0, (1 << self.bits) - 1)


@dataclass
class QuantizedTokens:
    """A batch of QuantizedToken (kv_quant.rs:82-101): `codes` [n_tokens, d] int8 (symmetric) or uint8, one scale and
    zero point per token."""
    codes: torch.Tensor
    scale: torch.Tensor
    zero_point: torch.Tensor
    symmetric: bool

    def dequantize(self, out_dtype=torch.float32) -> torch.Tensor:
        n, d = self.codes.shape
        codes, was_host = _dev(self.codes.reshape(-1).view(torch.uint8), torch.uint8)
        sc, _ = _dev(self.scale, torch.float32)
        zp, _ = _dev(self.zero_point, torch.float32)
        out = torch.empty(n * d, dtype=out_dtype, device=codes.device)
        name = "b2q_kv_dequantize_tokens_bf16" if out_dtype == torch.bfloat16 else "b2q_kv_dequantize_tokens_f32"
        default_handle().call(name, ptr(codes), n, d, int(self.symmetric), ptr(sc), ptr(zp), ptr(out))
        return _back(out, was_host).view(n, d)


def quantize_tokens(x: torch.Tensor, config: KvQuantConfig) -> QuantizedTokens:
    """quantize_token (kv_quant.rs:112-154) for every row of x [n_tokens, d]."""
    if x.numel() == 0:
        raise L.InvalidConfig(L.ERR_INVALID_CONFIG, "quantize_token: empty vector")
    n, d = x.shape
    bf16 = x.dtype == torch.bfloat16
    xd, was_host = _dev(x.reshape(-1), torch.bfloat16 if bf16 else torch.float32)
    codes = torch.empty(n * d, dtype=torch.uint8, device=xd.device)
    scales = torch.empty(n, dtype=torch.float32, device=xd.device)
    zps = torch.empty(n, dtype=torch.float32, device=xd.device)
    default_handle().call("b2q_kv_quantize_tokens_bf16" if bf16 else "b2q_kv_quantize_tokens_f32", ptr(xd), n, d, config.bits,
                          int(config.symmetric), ptr(codes), ptr(scales), ptr(zps))
    codes = codes.view(torch.int8) if config.symmetric else codes
    return QuantizedTokens(_back(codes, was_host).view(n, d), _back(scales, was_host), _back(zps, was_host), config.symmetric)


@dataclass
class QuantizedToken:
    """kv_quant.rs:82-101 (codes as a list of ints, like the reference's Vec<i32>)."""
    codes: list
    scale: float
    zero_point: float
    _batch: QuantizedTokens = None

    def dequantize(self) -> list:
        return self._batch.dequantize()[0].tolist()


def quantize_token(x, config: KvQuantConfig) -> QuantizedToken:
    """kv_quant.rs:112-154 for one vector (a list or a 1-D tensor)."""
    t = torch.as_tensor(x, dtype=torch.float32).reshape(1, -1)
    b = quantize_tokens(t, config)
    return QuantizedToken([int(c) for c in b.codes[0].tolist()], float(b.scale[0]), float(b.zero_point[0]), b)


def quantize_dequantize_token(x, config: KvQuantConfig) -> list:
    """kv_quant.rs:161-163"""
    return quantize_token(x, config).dequantize()


def quantization_mse(x, config: KvQuantConfig) -> float:
    """kv_quant.rs:169-182 (f64 accumulation of f32 differences)."""
    t = torch.as_tensor(x, dtype=torch.float32).reshape(-1)
    recon = torch.tensor(quantize_dequantize_token(t, config), dtype=torch.float32)
    return float(((t - recon).to(torch.float64) ** 2).sum() / t.numel())


# ---- RMSNorm -> FP8 ----
def rms_norm_quantize_fp8(x: torch.Tensor, gamma: torch.Tensor, eps: float, residual: torch.Tensor = None, fmt: int = L.FP8_E4M3,
                          rounding: int = L.ROUND_RNE, want_y: bool = False):
    """rms_norm / fused_add_rms_norm (crates/oxicuda-dnn/src/norm/rms_norm.rs:49-110, :115-170) followed by the per-token FP8
    quantizer, in one kernel.  x [rows, cols] bf16 on the device; `residual` (bf16, same shape) is updated in place with
    residual + x and normalised instead of x.  Returns (codes u8 [rows, cols], scales f32 [rows]) and y (bf16) when asked."""
    if not x.is_cuda or x.dtype != torch.bfloat16 or gamma.dtype != torch.bfloat16:
        raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, "rms_norm_quantize_fp8 takes bf16 CUDA tensors")
    rows, cols = x.shape
    if gamma.numel() != cols:
        raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {cols}, got {gamma.numel()}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != torch.bfloat16 or not residual.is_contiguous()):
        raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, "residual must be a contiguous bf16 tensor of x's shape")
    x = x.contiguous()
    codes = torch.empty(rows, cols, dtype=torch.uint8, device=x.device)
    scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    y = torch.empty_like(x) if want_y else None
    default_handle().call("b2q_rms_norm_quantize_fp8_bf16", ptr(x), ptr(residual), ptr(gamma.contiguous()), rows, cols, float(eps), fmt,
                          rounding, ptr(scales), ptr(codes), ptr(y))
    return (codes, scales, y) if want_y else (codes, scales)


def rms_norm_quantize_fp8_block128(x: torch.Tensor, gamma: torch.Tensor, eps: float, residual: torch.Tensor = None, fmt: int = L.FP8_E4M3,
                                   rounding: int = L.ROUND_RNE, want_y: bool = False):
    """rms_norm_quantize_fp8 with one scale per (row, 128 columns), the operand of blas.gemm_fp8_block128.  `residual` (bf16, x's
    shape) is updated in place with residual + x and normalised instead of x.  Returns (codes u8 [rows, cols], scales f32
    [rows, ceil(cols / 128)]) and y (bf16) when asked."""
    if x.dtype != torch.bfloat16 or gamma.dtype != torch.bfloat16 or x.dim() != 2:
        raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, "rms_norm_quantize_fp8_block128 takes a bf16 matrix and a bf16 gamma")
    rows, cols = x.shape
    if rows == 0 or cols == 0:
        raise L.EmptyInput(L.ERR_EMPTY_INPUT, "rms_norm_quantize_fp8_block128")
    if gamma.numel() != cols:
        raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {cols}, got {gamma.numel()}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != torch.bfloat16 or not residual.is_contiguous()):
        raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, "residual must be a contiguous bf16 tensor of x's shape")
    L.require_cuda("rms_norm_quantize_fp8_block128", x=x, gamma=gamma, residual=residual)
    x, gamma = x.contiguous(), gamma.contiguous()
    codes = torch.empty(rows, cols, dtype=torch.uint8, device=x.device)
    scales = torch.empty(rows, -(-cols // 128), dtype=torch.float32, device=x.device)
    y = torch.empty_like(x) if want_y else None
    default_handle().call("b2q_rms_norm_quantize_fp8_block128_bf16", x.data_ptr(), L.address(residual), gamma.data_ptr(), rows, cols, float(eps), fmt, rounding,
                          scales.data_ptr(), codes.data_ptr(), L.address(y))
    return (codes, scales, y) if want_y else (codes, scales)


class PagedFp8KvCache:
    """A paged KV cache in E4M3 codes with one power-of-two scale (an E8M0 byte) per page and kv head, and the attention that reads
    it.  Codes u8 [num_pages, n_kv_heads, page_size, head_dim], scales u8 [num_pages, n_kv_heads]; head_dim 64 or 128, page_size 16,
    32, 64 or 128.  The tensors belong to the caller, who may share them with other code."""

    PAGE_SIZES = (16, 32, 64, 128)
    HEAD_DIMS = (64, 128)

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        if k_codes.dim() != 4:
            raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, "PagedFp8KvCache: codes must be [num_pages, n_kv_heads, page_size, head_dim]")
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k_codes.shape
        if self.page_size not in self.PAGE_SIZES or self.head_dim not in self.HEAD_DIMS:
            raise L.UnsupportedOperation(L.ERR_UNSUPPORTED, f"PagedFp8KvCache: page_size must be one of {list(self.PAGE_SIZES)} and head_dim one of "
                                         f"{list(self.HEAD_DIMS)}, got {self.page_size} and {self.head_dim}")
        for t, shape in ((k_codes, k_codes.shape), (v_codes, k_codes.shape), (k_scales, k_codes.shape[:2]), (v_scales, k_codes.shape[:2])):
            if t.dtype != torch.uint8 or t.shape != shape or not t.is_contiguous():
                raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, f"PagedFp8KvCache: expected a contiguous uint8 tensor {list(shape)}, got {t.dtype} {list(t.shape)}")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales

    @staticmethod
    def empty(num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device) -> "PagedFp8KvCache":
        codes = [torch.zeros(num_pages, n_kv_heads, page_size, head_dim, dtype=torch.uint8, device=device) for _ in range(2)]
        scales = [torch.full((num_pages, n_kv_heads), 127, dtype=torch.uint8, device=device) for _ in range(2)]
        return PagedFp8KvCache(*codes, *scales)

    def _rows(self, who: str, x: torch.Tensor, heads: int):
        """x as [tokens, heads, head_dim] whose heads are packed: a view of a wider GEMM result is taken as it is."""
        if x.dtype != torch.bfloat16 or x.dim() != 3 or x.shape[2] != self.head_dim or (heads and x.shape[1] != heads):
            raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, f"{who}: expected bf16 [tokens, {heads or 'heads'}, {self.head_dim}], got {x.dtype} {list(x.shape)}")
        width = x.shape[1] * self.head_dim
        ld = x.stride(0) if x.shape[0] > 1 else width
        if x.stride(2) != 1 or (x.shape[1] > 1 and x.stride(1) != self.head_dim) or ld < width or ld % 8 or x.data_ptr() % 16:
            x = x.clone(memory_format=torch.contiguous_format)
            ld = width
        return x, ld

    def _batch(self, who: str, tokens: int, seq_lens: torch.Tensor, block_tables: torch.Tensor, q_starts):
        if seq_lens.dtype != torch.int32 or seq_lens.dim() != 1 or block_tables.dtype != torch.int32 or block_tables.dim() != 2:
            raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, f"{who}: seq_lens [seqs] and block_tables [seqs, width] are int32 tensors")
        seqs = seq_lens.numel()
        if tokens == 0 or seqs == 0:
            raise L.EmptyInput(L.ERR_EMPTY_INPUT, f"{who}: empty batch")
        if block_tables.shape[0] != seqs:
            raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {seqs} block tables, got {block_tables.shape[0]}")
        if q_starts is None and tokens != seqs:
            raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {seqs} tokens (one per sequence without q_starts), got {tokens}")
        if q_starts is not None and (q_starts.dtype != torch.int32 or q_starts.dim() != 1 or q_starts.numel() != seqs + 1):
            raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected int32 q_starts [{seqs + 1}], got {q_starts.dtype} {list(q_starts.shape)}")
        return seq_lens.contiguous(), block_tables.contiguous(), None if q_starts is None else q_starts.contiguous(), seqs

    def append(self, k: torch.Tensor, v: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor, q_starts: torch.Tensor = None) -> None:
        """Writes new keys and values (bf16 [tokens, n_kv_heads, head_dim]) into their pages.  seq_lens int32 [seqs]: cached tokens with
        the new ones included; block_tables int32 [seqs, width]; q_starts int32 [seqs + 1]: row offsets, None for one row per sequence.
        All on the device and read there: what is wrong with them is recorded, and raised by the handle's check()."""
        k, ld_k = self._rows("append", k, self.n_kv_heads)
        v, ld_v = self._rows("append", v, self.n_kv_heads)
        if k.shape[0] != v.shape[0]:
            raise L.DimensionMismatch(L.ERR_DIMENSION_MISMATCH, f"expected {k.shape[0]} rows of v, got {v.shape[0]}")
        seq_lens, block_tables, q_starts, seqs = self._batch("append", k.shape[0], seq_lens, block_tables, q_starts)
        L.require_cuda("append", k=k, v=v, seq_lens=seq_lens, block_tables=block_tables, q_starts=q_starts, k_codes=self.k_codes, v_codes=self.v_codes,
                       k_scales=self.k_scales, v_scales=self.v_scales)
        default_handle().call("b2q_kv8_append_bf16", k.data_ptr(), v.data_ptr(), ld_k, ld_v, k.shape[0], L.address(q_starts), seq_lens.data_ptr(), block_tables.data_ptr(), seqs,
                              block_tables.shape[1], self.num_pages, self.page_size, self.n_kv_heads, self.head_dim, self.k_codes.data_ptr(),
                              self.v_codes.data_ptr(), self.k_scales.data_ptr(), self.v_scales.data_ptr())

    def attend(self, q: torch.Tensor, seq_lens: torch.Tensor, block_tables: torch.Tensor, q_starts: torch.Tensor = None, scale: float = None,
               window: int = 0, out: torch.Tensor = None, want_lse: bool = False):
        """Causal attention of q (bf16 [tokens, heads, head_dim], heads a multiple of n_kv_heads) over the cached tokens, the rows' own
        included; with window > 0 over the last `window` of them.  scale: 1 / sqrt(head_dim) unless given.  Returns out (bf16, q's shape)
        and, when asked, the log-sum-exp of the scores (f32 [tokens, heads]).  Rows outside every sequence are left as they were (`out`
        given) or unspecified.  `out` may be q itself, and overlaps nothing else that the call reads."""
        q, ld_q = self._rows("attend", q, 0)
        tokens, heads, d = q.shape
        if heads == 0 or heads % self.n_kv_heads != 0:
            raise L.InvalidDimension(L.ERR_INVALID_DIMENSION, f"{heads} query heads are not a multiple of {self.n_kv_heads} kv heads")
        seq_lens, block_tables, q_starts, seqs = self._batch("attend", tokens, seq_lens, block_tables, q_starts)
        if out is None:
            out = torch.empty(tokens, heads, d, dtype=torch.bfloat16, device=q.device)
        elif out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous():
            raise L.InvalidArgument(L.ERR_INVALID_ARGUMENT, "attend: out must be a contiguous bf16 tensor of q's shape")
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=q.device) if want_lse else None
        L.require_cuda("attend", q=q, seq_lens=seq_lens, block_tables=block_tables, q_starts=q_starts, out=out, k_codes=self.k_codes,
                       v_codes=self.v_codes, k_scales=self.k_scales, v_scales=self.v_scales)
        default_handle().call("b2q_kv8_attention_bf16", q.data_ptr(), ld_q, tokens, heads, L.address(q_starts), seq_lens.data_ptr(), block_tables.data_ptr(), seqs,
                              block_tables.shape[1], self.num_pages, self.page_size, self.n_kv_heads, d, self.k_codes.data_ptr(), self.v_codes.data_ptr(),
                              self.k_scales.data_ptr(), self.v_scales.data_ptr(), d ** -0.5 if scale is None else float(scale), int(window), out.data_ptr(), L.address(lse))
        return (out, lse) if want_lse else out

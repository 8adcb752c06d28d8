// The producers of block-128 FP8 operands (one scale per row and 128 columns, what b2q_gemm_fp8_block128 multiplies):
//   RMSNorm, optionally of the residual stream after adding x to it:
//     r' = bf16(r + x);  y = r' / sqrt(mean(r'^2) + eps) * gamma        (crates/oxicuda-dnn/src/norm/rms_norm.rs:29-33, :98-103)
//   SwiGLU:
//     h = gate * up / (1 + exp(-gate))                                  (crates/oxicuda-moe/src/expert/ffn.rs:208-243)
// followed, per block of 128 columns, by scale = absmax / max_val (1 for a block of zeros, never below the smallest normal
// float) and code = encode(v / scale).  Both are bound by HBM: every input is read once, every output written once.
//
// A block of 128 columns is 16 lanes of 8 elements (one 16-byte load each), so its absmax is four shuffles: no shared
// memory, and the scale is known without a second pass.  Statistics and scales are f32; v / scale is v * (1 / scale) with
// a correctly rounded reciprocal (one rounding more than a division, which shows only in codes that sit on a rounding
// boundary; a division per element would make the kernels instruction-bound).
#include "common.cuh"

namespace {

constexpr float kMinScale = 1.17549435e-38f;   // 2^-126: its reciprocal is finite

__device__ __forceinline__ void unpack8(const uint4 q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u); }
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float block_scale(float amax, float max_val) {
  return amax > 0.0f ? fmaxf(__fdiv_rn(amax, max_val), kMinScale) : 1.0f;
}
__device__ __forceinline__ uint32_t encode1(float v, float inv_scale, int fmt, int rounding, const Fp8Fmt& F) {
  float q = __fmul_rn(v, inv_scale);
  if (rounding == B2Q_ROUND_RNE) return fp8_encode_rne_dev(q, fmt);
  q = q < -F.max_val ? -F.max_val : (q > F.max_val ? F.max_val : q);
  return fp8_encode_ref_dev(q, F);
}
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float inv_scale, int fmt, int rounding, const Fp8Fmt& F) {
  if (rounding == B2Q_ROUND_RNE) {             // the conversion saturates to +-max_val by itself
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      p[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(v[2 * j], inv_scale), __fmul_rn(v[2 * j + 1], inv_scale)),
                                                __NV_SATFINITE, fmt == B2Q_FP8_E4M3 ? __NV_E4M3 : __NV_E5M2);
    return make_uint2(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410));
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j >> 2] |= encode1(v[j], inv_scale, fmt, rounding, F) << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}
// max over the 16 lanes that hold one block of 128 columns
__device__ __forceinline__ float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float absmax8(const float (&v)[8]) {
  float a = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = fmaxf(a, fabsf(v[j]));
  return a;
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = (threadIdx.x & 31) < nw ? sh[threadIdx.x & 31] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct NormArgs {
  const __nv_bfloat16* x; __nv_bfloat16* residual; const __nv_bfloat16* gamma;
  int64_t cols; float eps; int fmt, rounding;
  float* scales; uint8_t* codes; __nv_bfloat16* y;
};

// One CTA per row; thread t keeps chunks t, t + blockDim, ... (8 elements each, NCH at most) of the row in registers.
// blockDim is a multiple of 32, so 16 neighbouring lanes always hold the 16 chunks of one block of 128 columns.
template <int NCH>
__global__ void __launch_bounds__(1024) rms_norm_block128_kernel(const NormArgs p) {
  b2q_pdl_entry();
  __shared__ float sh[32];
  const int64_t r = blockIdx.x;
  const int chunks = (int)(p.cols >> 3), nb = (int)((p.cols + 127) >> 7);
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + r * p.cols);
  uint4* rr = p.residual ? reinterpret_cast<uint4*>(p.residual + r * p.cols) : nullptr;
  const uint4* gr = reinterpret_cast<const uint4*>(p.gamma);
  float v[NCH][8];
  {
    uint4 xq[NCH], rq[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {                        // all loads of the row before the first use
      const int c = (int)threadIdx.x + k * (int)blockDim.x;
      xq[k] = c < chunks ? __ldcs(xr + c) : make_uint4(0, 0, 0, 0);
      if (rr) rq[k] = c < chunks ? __ldcs(rr + c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      unpack8(xq[k], v[k]);
      if (rr) {
        float res[8];
        unpack8(rq[k], res);
        uint4 w;                                           // the norm is taken of the sum as it is stored
        w.x = bf16_pair(__fadd_rn(res[0], v[k][0]), __fadd_rn(res[1], v[k][1]));
        w.y = bf16_pair(__fadd_rn(res[2], v[k][2]), __fadd_rn(res[3], v[k][3]));
        w.z = bf16_pair(__fadd_rn(res[4], v[k][4]), __fadd_rn(res[5], v[k][5]));
        w.w = bf16_pair(__fadd_rn(res[6], v[k][6]), __fadd_rn(res[7], v[k][7]));
        const int c = (int)threadIdx.x + k * (int)blockDim.x;
        if (c < chunks) rr[c] = w;
        unpack8(w, v[k]);
      }
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[k][j], v[k][j], ss);
  ss = block_sum(ss, sh);
  const float inv_rms = __frcp_rn(sqrtf(__fadd_rn(__fdiv_rn(ss, (float)p.cols), p.eps)));
  const Fp8Fmt F = fp8_fmt(p.fmt);
  uint2* cr = reinterpret_cast<uint2*>(p.codes + r * p.cols);
  uint4* yr = p.y ? reinterpret_cast<uint4*>(p.y + r * p.cols) : nullptr;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = (int)threadIdx.x + k * (int)blockDim.x;
    float g[8];
    unpack8(c < chunks ? __ldg(gr + c) : make_uint4(0, 0, 0, 0), g);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = c < chunks ? __fmul_rn(__fmul_rn(v[k][j], inv_rms), g[j]) : 0.0f;
    const float scale = block_scale(max16(absmax8(v[k])), F.max_val);
    if (c < chunks) {
      cr[c] = encode8(v[k], __frcp_rn(scale), p.fmt, p.rounding, F);
      if ((c & 15) == 0) p.scales[r * nb + (c >> 4)] = scale;
      if (yr) yr[c] = make_uint4(bf16_pair(v[k][0], v[k][1]), bf16_pair(v[k][2], v[k][3]), bf16_pair(v[k][4], v[k][5]), bf16_pair(v[k][6], v[k][7]));
    }
  }
}

// Any row length and alignment: one warp per block of 128 columns after the sum of squares; the row is read again from L1 / L2.
__global__ void __launch_bounds__(256) rms_norm_block128_generic_kernel(const NormArgs p) {
  b2q_pdl_entry();
  __shared__ float sh[32];
  const int64_t r = blockIdx.x;
  const __nv_bfloat16* row = p.x + r * p.cols;
  __nv_bfloat16* res = p.residual ? p.residual + r * p.cols : nullptr;
  float ss = 0.0f;
  for (int64_t i = threadIdx.x; i < p.cols; i += blockDim.x) {
    float v = __bfloat162float(row[i]);
    if (res) {
      const __nv_bfloat16 s = __float2bfloat16_rn(__fadd_rn(__bfloat162float(res[i]), v));
      res[i] = s;
      v = __bfloat162float(s);
    }
    ss = fmaf(v, v, ss);
  }
  ss = block_sum(ss, sh);                                  // its barrier also makes the stored sums visible to the CTA
  const float inv_rms = __frcp_rn(sqrtf(__fadd_rn(__fdiv_rn(ss, (float)p.cols), p.eps)));
  const __nv_bfloat16* src = res ? res : row;
  const Fp8Fmt F = fp8_fmt(p.fmt);
  const int64_t nb = (p.cols + 127) >> 7;
  const int lane = threadIdx.x & 31;
  for (int64_t b = threadIdx.x >> 5; b < nb; b += blockDim.x >> 5) {
    float v[4], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = b * 128 + j * 32 + lane;
      v[j] = i < p.cols ? __fmul_rn(__fmul_rn(__bfloat162float(src[i]), inv_rms), __bfloat162float(p.gamma[i])) : 0.0f;
      amax = fmaxf(amax, fabsf(v[j]));
    }
    const float scale = block_scale(warp_max(amax), F.max_val), inv = __frcp_rn(scale);
    if (lane == 0) p.scales[r * nb + b] = scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = b * 128 + j * 32 + lane;
      if (i < p.cols) {
        p.codes[r * p.cols + i] = (uint8_t)encode1(v[j], inv, p.fmt, p.rounding, F);
        if (p.y) p.y[r * p.cols + i] = __float2bfloat16_rn(v[j]);
      }
    }
  }
}

// silu(g) = g / (1 + e^-g) with e^-|g|, which cannot overflow: g e^g / (1 + e^g) for negative g.  silu(g) before u: g * u may
// overflow where silu(g) is next to 0.
__device__ __forceinline__ float swiglu(float g, float u) {
  const float e = exp2f(-1.4426950408889634f * fabsf(g));
  return g * (g < 0.0f ? e : 1.0f) * __frcp_rn(1.0f + e) * u;
}

struct SwigluArgs {
  const __nv_bfloat16* gate; const __nv_bfloat16* up; int64_t rows, cols, ld; int fmt, rounding;
  float* scales; uint8_t* codes;
};

// 16 lanes per block of 128 columns, a warp two blocks; the blocks of all rows are one flat index space.
__global__ void __launch_bounds__(256) swiglu_block128_kernel(const SwigluArgs p) {
  b2q_pdl_entry();
  const int64_t nb = (p.cols + 127) >> 7, total = p.rows * nb;
  const int sub = threadIdx.x & 15;
  const Fp8Fmt F = fp8_fmt(p.fmt);
  const int64_t step = (int64_t)gridDim.x * 16;
  for (int64_t b0 = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); b0 - (int64_t)((threadIdx.x >> 4) & 1) < total; b0 += step) {   // whole warps leave together
    const int64_t r = b0 / nb, b = b0 - r * nb, c = b * 128 + sub * 8;
    const bool live = b0 < total && c < p.cols;
    float h[8];
    if (live) {
      float g[8], u[8];
      unpack8(__ldcs(reinterpret_cast<const uint4*>(p.gate + r * p.ld + c)), g);
      unpack8(__ldcs(reinterpret_cast<const uint4*>(p.up + r * p.ld + c)), u);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = swiglu(g[j], u[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = 0.0f;
    }
    const float scale = block_scale(max16(absmax8(h)), F.max_val);
    if (live) {
      *reinterpret_cast<uint2*>(p.codes + r * p.cols + c) = encode8(h, __frcp_rn(scale), p.fmt, p.rounding, F);
      if (sub == 0) p.scales[b0] = scale;
    }
  }
}

// Any length and alignment: one warp per block of 128 columns.
__global__ void __launch_bounds__(256) swiglu_block128_generic_kernel(const SwigluArgs p) {
  b2q_pdl_entry();
  const int64_t nb = (p.cols + 127) >> 7, total = p.rows * nb;
  const int lane = threadIdx.x & 31;
  const Fp8Fmt F = fp8_fmt(p.fmt);
  for (int64_t b0 = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); b0 < total; b0 += (int64_t)gridDim.x * 8) {
    const int64_t r = b0 / nb, b = b0 - r * nb;
    float h[4], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = b * 128 + j * 32 + lane;
      h[j] = c < p.cols ? swiglu(__bfloat162float(p.gate[r * p.ld + c]), __bfloat162float(p.up[r * p.ld + c])) : 0.0f;
      amax = fmaxf(amax, fabsf(h[j]));
    }
    const float scale = block_scale(warp_max(amax), F.max_val), inv = __frcp_rn(scale);
    if (lane == 0) p.scales[b0] = scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = b * 128 + j * 32 + lane;
      if (c < p.cols) p.codes[r * p.cols + c] = (uint8_t)encode1(h[j], inv, p.fmt, p.rounding, F);
    }
  }
}

}  // namespace

extern "C" int32_t b2q_rms_norm_quantize_fp8_block128_bf16(b2q_handle h, const void* x, void* residual, const void* gamma, int64_t rows, int64_t cols,
                                                           float eps, int fmt, int rounding, float* scales, uint8_t* codes, void* y_out) {
  B2Q_REQUIRE_HANDLE(h);
  if (rows <= 0 || cols <= 0) B2Q_FAIL(h, B2Q_ERR_EMPTY_INPUT, "rms_norm_quantize_fp8_block128: empty input");
  if (!x || !gamma || !scales || !codes) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "rms_norm_quantize_fp8_block128: null pointer");
  if (fmt < 0 || fmt > 1 || rounding < 0 || rounding > 1) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "rms_norm_quantize_fp8_block128: bad format/rounding");
  if (rows > 0x7FFFFFFF) B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "rms_norm_quantize_fp8_block128: %lld rows", (long long)rows);
  NormArgs p{static_cast<const __nv_bfloat16*>(x), static_cast<__nv_bfloat16*>(residual), static_cast<const __nv_bfloat16*>(gamma),
             cols, eps, fmt, rounding, scales, codes, static_cast<__nv_bfloat16*>(y_out)};
  const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(gamma) |
                          reinterpret_cast<uintptr_t>(y_out) | (reinterpret_cast<uintptr_t>(codes) << 1);
  const int64_t chunks = cols >> 3;
  const bool pdl = h->sw.chain_pdl != 0;
  const dim3 grid((unsigned)rows);
  if (cols % 8 == 0 && (align & 15) == 0 && chunks <= 4 * 1024) {
    // few rows: one chunk per thread, the shortest chain; many rows: several chunks per thread, so that more CTAs share an SM
    int nch = chunks <= 1024 ? 1 : (chunks <= 2048 ? 2 : 4);
    if (rows >= 2 * (int64_t)h->sm_count && chunks > 128) nch = chunks <= 256 ? 2 : 4;
    const dim3 block((unsigned)(ceil_div64(ceil_div64(chunks, nch), 32) * 32));
    if (nch == 1) B2Q_CUDA(h, b2q_pdl_launch(pdl, rms_norm_block128_kernel<1>, grid, block, 0, h->stream, p));
    else if (nch == 2) B2Q_CUDA(h, b2q_pdl_launch(pdl, rms_norm_block128_kernel<2>, grid, block, 0, h->stream, p));
    else B2Q_CUDA(h, b2q_pdl_launch(pdl, rms_norm_block128_kernel<4>, grid, block, 0, h->stream, p));
    return B2Q_OK;
  }
  B2Q_CUDA(h, b2q_pdl_launch(pdl, rms_norm_block128_generic_kernel, grid, dim3(256), 0, h->stream, p));
  return B2Q_OK;
}

extern "C" int32_t b2q_swiglu_quantize_fp8_block128_bf16(b2q_handle h, const void* gate, const void* up, int64_t rows, int64_t cols, int64_t ld, int fmt,
                                                         int rounding, float* scales, uint8_t* codes) {
  B2Q_REQUIRE_HANDLE(h);
  if (rows <= 0 || cols <= 0) B2Q_FAIL(h, B2Q_ERR_EMPTY_INPUT, "swiglu_quantize_fp8_block128: empty input");
  if (!gate || !up || !scales || !codes || ld < cols) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "swiglu_quantize_fp8_block128: null pointer, or ld < cols");
  if (fmt < 0 || fmt > 1 || rounding < 0 || rounding > 1) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "swiglu_quantize_fp8_block128: bad format/rounding");
  SwigluArgs p{static_cast<const __nv_bfloat16*>(gate), static_cast<const __nv_bfloat16*>(up), rows, cols, ld, fmt, rounding, scales, codes};
  const int64_t total = rows * ceil_div64(cols, 128);
  const bool vec = cols % 8 == 0 && ld % 8 == 0 && ((reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(up)) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  const int64_t ctas = ceil_div64(total, vec ? 16 : 8), most = (int64_t)h->sm_count * 32;
  const dim3 grid((unsigned)(ctas < most ? ctas : most));
  B2Q_CUDA(h, b2q_pdl_launch(h->sw.chain_pdl != 0, vec ? swiglu_block128_kernel : swiglu_block128_generic_kernel, grid, dim3(256), 0, h->stream, p));
  return B2Q_OK;
}

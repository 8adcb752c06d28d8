// The producers of block-128 FP8 operands (one scale per row and 128 columns, what b2q_gemm_fp8_block128 multiplies):
//   RMSNorm, optionally of the residual stream after adding x to it:
//     r' = bf16(r + x);  y = r' / sqrt(mean(r'^2) + eps) * gamma        (crates/oxicuda-dnn/src/norm/rms_norm.rs:29-33, :98-103)
//   SwiGLU:
//     h = gate * up / (1 + exp(-gate))                                  (crates/oxicuda-moe/src/expert/ffn.rs:208-243)
// followed, per block of 128 columns, by scale = absmax / max_val (1 for a block of zeros, never below the smallest normal
// float) and code = encode(v / scale).  Both are bound by HBM: every input is read once, every output written once.
//
// A block of 128 columns is 16 lanes of 8 elements (one 16-byte load each), so its absmax is four shuffles: no shared
// memory, and the scale is known without a second pass.  Statistics and scales are f32.  No element is divided (that would make the kernels
// instruction-bound).  The norm's quotient is (r' gamma) * (max_val / absmax(r' gamma)): 1 / rms cancels, r' gamma is exact in f32 (two bf16),
// and the factor is held as a sum of two floats, so that the quotient is rounded once: of 7.4 million codes none differs from the exact
// quotient's; with each step of the formula rounded 641 did.  SwiGLU multiplies by the reciprocal of the scale, and makes the few elements that
// come out next to a border between two E4M3 codes again in 64 bits: 2047 x 28672 takes 58 us instead of 50 over one set of inputs (65 a call), and
// of 7.4 million codes above 2^-6 none differs from the exact quotient's where half a code in a million did (gates of ordinary size; the window is
// no bound of the error).
#include "common.cuh"

namespace {

constexpr float kMinScale = 1.17549435e-38f;   // 2^-126: its reciprocal is finite

// Two neighbouring elements travel in one 64-bit register (low half first): the multiply-adds of sm_100a take both at once.
__device__ __forceinline__ uint64_t pair(float lo, float hi) { return (uint64_t)__float_as_uint(hi) << 32 | __float_as_uint(lo); }
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y)); return r; }
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t x, uint64_t y) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(x), "l"(y)); }
__device__ __forceinline__ void unpack8(const uint4 q, uint64_t (&v)[4]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = (uint64_t)(w[j] & 0xFFFF0000u) << 32 | (w[j] << 16);
}
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
// bf16(a + b) of two pairs: a sum of two bf16 rounded once.  Rounding it to f32 first gives the same: where f32 rounds at all, the operands
// are more than 2^16 apart and the sum is no tie of bf16.
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float block_scale(float amax, float max_val) {
  return amax > 0.0f ? fmaxf(__fdiv_rn(amax, max_val), kMinScale) : 1.0f;
}
__device__ __forceinline__ uint32_t encode1(float q, int fmt, int rounding, const Fp8Fmt& F) {
  if (rounding == B2Q_ROUND_RNE) return fp8_encode_rne_dev(q, fmt);
  q = q < -F.max_val ? -F.max_val : (q > F.max_val ? F.max_val : q);
  return fp8_encode_ref_dev(q, F);
}
// What the kernels are compiled for: E4M3 to nearest even (the production form), or anything else (format and rounding at run time).
enum Mode { kE4m3Rne, kAny };
template <int MODE>
__device__ __forceinline__ uint2 encode8(const uint64_t (&q)[4], int fmt, int rounding, const Fp8Fmt& F) {
  if (MODE == kE4m3Rne) {                      // the conversion saturates to +-448 by itself
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo(q[j]), hi(q[j])), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410));
  }
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j >> 1] |= (encode1(lo(q[j]), fmt, rounding, F) | encode1(hi(q[j]), fmt, rounding, F) << 8) << (16 * (j & 1));
  return make_uint2(w[0], w[1]);
}
// v (hi + lo), rounded once
__device__ __forceinline__ void scale8(const uint64_t (&v)[4], float hi, float lo, uint64_t (&q)[4]) {
  const uint64_t h2 = pair(hi, hi), l2 = pair(lo, lo);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    q[j] = mul2(v[j], l2);
    fma2(q[j], v[j], h2);
  }
}
template <int MODE>
__device__ __forceinline__ uint2 encode8(const uint64_t (&v)[4], float inv_scale, int fmt, int rounding, const Fp8Fmt& F) {
  const uint64_t inv = pair(inv_scale, inv_scale), q[4] = {mul2(v[0], inv), mul2(v[1], inv), mul2(v[2], inv), mul2(v[3], inv)};
  return encode8<MODE>(q, fmt, rounding, F);
}
// max over the 16 lanes that hold one block of 128 columns
__device__ __forceinline__ float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float absmax8(const uint64_t (&v)[4]) {
  float a = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) a = fmaxf(a, fmaxf(fabsf(lo(v[j])), fabsf(hi(v[j]))));
  return a;
}
// The norm's scale of a block whose largest |r' gamma| is amax, and the factor hi + lo that takes r' gamma to codes; hi = 0: the block is outside
// the range in which no step over- or underflows, and is done by the formula's own steps.
struct NormScale { float scale, hi, lo; };
// max_val / amax as a sum of two floats (amax from 2^-100 to 2^100)
__device__ __forceinline__ void quotient(float max_val, float amax, float& hi, float& lo) {
  float inv;                                               // any quotient will do: the remainder is exact
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(amax));
  hi = __fmul_rn(max_val, inv);
  lo = __fmul_rn(fmaf(-hi, amax, max_val), inv);
}
__device__ __forceinline__ NormScale norm_scale(float amax, float inv_rms, float max_val) {
  NormScale n{block_scale(__fmul_rn(amax, inv_rms), max_val), 0.0f, 0.0f};
  if (inv_rms >= 0x1p-60f && inv_rms <= 0x1p60f) {
    if (amax == 0.0f) n.hi = 1.0f;
    else if (amax >= 0x1p-60f && amax <= 0x1p100f && n.scale > kMinScale) quotient(max_val, amax, n.hi, n.lo);
  }
  return n;
}
// The scales of the N blocks that a group of 16 lanes holds: lane k of the group makes the k'th (a division and a reciprocal are some
// twenty instructions each), the others get its reciprocal.  `mine` is the scale that this lane made (k < N).
template <int N>
__device__ __forceinline__ void block_scales(const float (&amax)[N], float max_val, float& mine, float (&inv)[N]) {
  const int lane = threadIdx.x & 31, sub = lane & 15;
  float a = amax[0];
#pragma unroll
  for (int k = 1; k < N; ++k) a = sub == k ? amax[k] : a;
  mine = block_scale(a, max_val);
  const float r = __frcp_rn(mine);
#pragma unroll
  for (int k = 0; k < N; ++k) inv[k] = __shfl_sync(0xffffffffu, r, (lane & 16) | k);
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
template <int NCH, int MODE>
__global__ void __launch_bounds__(1024) rms_norm_block128_kernel(const NormArgs p) {
  b2q_pdl_entry();
  __shared__ float sh[32];
  const int64_t r = blockIdx.x;
  const int chunks = (int)(p.cols >> 3), nb = (int)((p.cols + 127) >> 7);
  const uint4* xr = reinterpret_cast<const uint4*>(p.x + r * p.cols);
  uint4* rr = p.residual ? reinterpret_cast<uint4*>(p.residual + r * p.cols) : nullptr;
  const uint4* gr = reinterpret_cast<const uint4*>(p.gamma);
  uint4 xq[NCH];
  {
    uint4 rq[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) {                        // all loads of the row before the first use
      const int c = (int)threadIdx.x + k * (int)blockDim.x;
      xq[k] = c < chunks ? __ldcs(xr + c) : make_uint4(0, 0, 0, 0);
      if (rr) rq[k] = c < chunks ? __ldcs(rr + c) : make_uint4(0, 0, 0, 0);
    }
    if (rr) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {                      // the norm is taken of the sum as it is stored
        const int c = (int)threadIdx.x + k * (int)blockDim.x;
        xq[k] = make_uint4(add_bf16x2(rq[k].x, xq[k].x), add_bf16x2(rq[k].y, xq[k].y), add_bf16x2(rq[k].z, xq[k].z), add_bf16x2(rq[k].w, xq[k].w));
        if (c < chunks) rr[c] = xq[k];
      }
    }
  }
  uint64_t s2 = 0;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    uint64_t v[4];
    unpack8(xq[k], v);
#pragma unroll
    for (int j = 0; j < 4; ++j) fma2(s2, v[j], v[j]);
  }
  const float ss = block_sum(lo(s2) + hi(s2), sh);
  const float inv_rms = __frcp_rn(sqrtf(__fadd_rn(__fdiv_rn(ss, (float)p.cols), p.eps)));
  const uint64_t inv2 = pair(inv_rms, inv_rms);
  const Fp8Fmt F = fp8_fmt(p.fmt);
  uint2* cr = reinterpret_cast<uint2*>(p.codes + r * p.cols);
  uint4* yr = p.y ? reinterpret_cast<uint4*>(p.y + r * p.cols) : nullptr;
  uint64_t v[NCH][4];                                      // r' gamma
  float amax[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = (int)threadIdx.x + k * (int)blockDim.x;
    uint64_t g[4];
    unpack8(c < chunks ? __ldg(gr + c) : make_uint4(0, 0, 0, 0), g);
    unpack8(xq[k], v[k]);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[k][j] = mul2(v[k][j], g[j]);
    amax[k] = max16(absmax8(v[k]));
  }
  // lane k of a group of 16 makes the scale of the group's k'th block
  const int lane = threadIdx.x & 31, sub = lane & 15;
  float a = amax[0];
#pragma unroll
  for (int k = 1; k < NCH; ++k) a = sub == k ? amax[k] : a;
  const NormScale mine = norm_scale(a, inv_rms, F.max_val);
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = (int)threadIdx.x + k * (int)blockDim.x;
    const float fh = NCH == 1 ? mine.hi : __shfl_sync(0xffffffffu, mine.hi, (lane & 16) | k), fl = NCH == 1 ? mine.lo : __shfl_sync(0xffffffffu, mine.lo, (lane & 16) | k);
    float scale = mine.scale;                              // of lane k alone
    if (fh != 0.0f) {
      if (yr && c < chunks) {                              // by the formula's steps: r' gamma of an element far below its block's largest may be subnormal
        uint64_t g[4], y[4];
        unpack8(__ldg(gr + c), g);
        unpack8(rr ? rr[c] : xr[c], y);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = mul2(mul2(y[j], inv2), g[j]);
        yr[c] = make_uint4(bf16_pair(lo(y[0]), hi(y[0])), bf16_pair(lo(y[1]), hi(y[1])), bf16_pair(lo(y[2]), hi(y[2])), bf16_pair(lo(y[3]), hi(y[3])));
      }
      uint64_t q[4];
      scale8(v[k], fh, fl, q);
      if (c < chunks) cr[c] = encode8<MODE>(q, p.fmt, p.rounding, F);
    } else {                                               // all 16 lanes of the block
      uint64_t g[4], y[4];
      unpack8(c < chunks ? gr[c] : make_uint4(0, 0, 0, 0), g);
      unpack8(c < chunks ? (rr ? rr[c] : xr[c]) : make_uint4(0, 0, 0, 0), y);
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = mul2(mul2(y[j], inv2), g[j]);
      if (c < chunks) top = absmax8(y);                    // (0 * inf behind the row's end would be a NaN, which the maximum passes over)
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFu << (lane & 16), top, o));
      scale = block_scale(top, F.max_val);
      if (c < chunks) {
        cr[c] = encode8<MODE>(y, __frcp_rn(scale), p.fmt, p.rounding, F);
        if (yr) yr[c] = make_uint4(bf16_pair(lo(y[0]), hi(y[0])), bf16_pair(lo(y[1]), hi(y[1])), bf16_pair(lo(y[2]), hi(y[2])), bf16_pair(lo(y[3]), hi(y[3])));
      }
    }
    if (sub == k && (c & ~15) < chunks) p.scales[r * nb + (c >> 4)] = scale;
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
    float w[4], g[4], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = b * 128 + j * 32 + lane;
      w[j] = i < p.cols ? __bfloat162float(src[i]) : 0.0f;
      g[j] = i < p.cols ? __bfloat162float(p.gamma[i]) : 0.0f;
      amax = fmaxf(amax, fabsf(__fmul_rn(w[j], g[j])));
    }
    const NormScale n = norm_scale(warp_max(amax), inv_rms, F.max_val);
    float scale = n.scale, q[4], y[4];
    if (n.hi != 0.0f) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = __fmul_rn(w[j], g[j]);
        y[j] = __fmul_rn(__fmul_rn(w[j], inv_rms), g[j]);
        q[j] = fmaf(v, n.hi, __fmul_rn(v, n.lo));
      }
    } else {
      amax = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = __fmul_rn(__fmul_rn(w[j], inv_rms), g[j]);
        if (b * 128 + j * 32 + lane < p.cols) amax = fmaxf(amax, fabsf(y[j]));
      }
      scale = block_scale(warp_max(amax), F.max_val);
      const float inv = __frcp_rn(scale);
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = __fmul_rn(y[j], inv);
    }
    if (lane == 0) p.scales[r * nb + b] = scale;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = b * 128 + j * 32 + lane;
      if (i < p.cols) {
        p.codes[r * p.cols + i] = (uint8_t)encode1(q[j], p.fmt, p.rounding, F);
        if (p.y) p.y[r * p.cols + i] = __float2bfloat16_rn(y[j]);
      }
    }
  }
}

// silu(g) = g / (1 + e^-g), two at a time, by the hardware's exponential and reciprocal (2^-22 and 1 ulp; neither needs the handling of
// subnormals that makes their exact forms several instructions each: with those the kernel was instruction-bound, 84 us for 2047 x 28672).
// For gates down to kFarGate: g log2(e) is rounded, which moves e^-g by |g| 2^-24 of itself, and below -87.3 the reciprocal would be 0.
// silu(g) before u: g * u may overflow where silu(g) is next to 0.
__device__ __forceinline__ uint64_t silu2(uint64_t g) {
  const uint64_t t = mul2(g, pair(-1.4426950408889634f, -1.4426950408889634f));
  float ea, eb, ra, rb;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ea) : "f"(lo(t)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(eb) : "f"(hi(t)));
  const uint64_t d = add2(pair(ea, eb), pair(1.0f, 1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(ra) : "f"(lo(d)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rb) : "f"(hi(d)));
  return mul2(g, pair(ra, rb));
}
// one element by the same steps
__device__ __forceinline__ float silu1(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(__fmul_rn(g, -1.4426950408889634f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(e, 1.0f)));
  return __fmul_rn(g, r);
}
// Elements whose gate lies below this are made by silu_far: silu(g) u = (g e) (e u), e = e^(g/2) (1 + e^g is 1 here), so that what u is large enough to
// bring back into range has not been lost before; 0 where e is below 2^-126 (a number below 2^-116 whatever u is).  e = 2^t (1 + l ln 2), t + l =
// g log2(e) / 2 with t rounded.  Gates of sizes of 1.5, 10, 40 and 1000 (2047 x 28672): 61, 61, 101 and 115 us (66 and 82 for the last two without this).
constexpr float kFarGate = -80.0f;
__device__ __forceinline__ float silu_far(float g, float u) {
  constexpr float c = 0x1.715476p-1f, c_lo = 9.629815e-9f;   // log2(e) / 2
  const float t = __fmul_rn(g, c), l = fmaf(g, c_lo, fmaf(g, c, -t));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, l * 0.69314718f, e);
  return (g * e) * (e * u);
}
// whether one of eight gates lies below kFarGate (or a pair of them is NaN)
__device__ __forceinline__ bool far8(const uint4 q) {
  const __nv_bfloat162* const p = reinterpret_cast<const __nv_bfloat162*>(&q);
  return !__hbge2(__hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3])), __float2bfloat162_rn(kFarGate));
}

// A quotient this near to the middle between two E4M3 codes may lie on its other side by the f32 arithmetic in front of it (2^-21 to 2^-20 of
// itself; the hardware's exponential and reciprocal, and some roundings, are off by about 2^-22 for gates of ordinary size).  Above 2^-6 the middles are
// the floats whose 20 lowest bits are 0x80000, so the test is one multiply-add and a minimum.
constexpr uint32_t kNear = 8u << 12;
__device__ __forceinline__ uint32_t to_middle(float q) { return __float_as_uint(q) * 4096u + (0x80000000u + kNear); }   // below 2 kNear: near
// The largest of a block between these: its sums have neither over- nor underflowed.
__device__ __forceinline__ bool in_range(float amax) { return amax >= 0x1p-100f && amax <= 0x1p100f; }
__device__ __forceinline__ double swiglu64(float g, float u) { return (double)g * (double)u / (1.0 + exp(-(double)g)); }
__device__ __forceinline__ float quotient64(double h, double top) { return (float)(h * (top > 0.0 ? 448.0 / top : 1.0)); }
// The codes of a lane's 8 elements by the formula in 64 bits, for a whole warp (blocks of 16 lanes).
__device__ __noinline__ uint2 swiglu_exact8(const __nv_bfloat16* gp, const __nv_bfloat16* up, bool live) {
  double h[8], top = 0.0;
#pragma unroll 1
  for (int j = 0; j < 8; ++j) {
    h[j] = live ? swiglu64(__bfloat162float(gp[j]), __bfloat162float(up[j])) : 0.0;
    top = fmax(top, fabs(h[j]));
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(quotient64(h[2 * j], top), quotient64(h[2 * j + 1], top)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}
// 0xFF in the bytes of those of four quotients that lie near a middle
__device__ __forceinline__ uint32_t near4(uint64_t a, uint64_t b) {
  const float q[4] = {lo(a), hi(a), lo(b), hi(b)};
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) m |= to_middle(q[j]) < 2 * kNear ? 0xFFu << (8 * j) : 0u;
  return m;
}

struct SwigluArgs {
  const __nv_bfloat16* gate; const __nv_bfloat16* up; int64_t rows, cols, ld; int fmt, rounding;
  float* scales; uint8_t* codes;
  uint32_t per_row, magic;                       // blocks of a row, floor((2^32 - 1) / per_row)
};

// 16 lanes per block of 128 columns, a warp two blocks; the blocks of all rows are one flat index space (below 2^31, so that its
// division by the blocks of a row is a multiplication), two steps of it in flight per thread.
template <int MODE>
__global__ void __launch_bounds__(256, 5) swiglu_block128_kernel(const SwigluArgs p) {
  b2q_pdl_entry();
  const uint32_t total = (uint32_t)p.rows * p.per_row, step = gridDim.x * 16;
  const int sub = threadIdx.x & 15;
  const Fp8Fmt F = fp8_fmt(p.fmt);
  for (uint32_t first = blockIdx.x * 16; first < total; first += 2 * step) {       // the whole CTA leaves together
    uint4 gq[2], uq[2];
    uint32_t at[2], row[2], col[2];
    bool live[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      at[k] = first + k * step + (threadIdx.x >> 4);
      row[k] = __umulhi(at[k], p.magic);
      uint32_t b = at[k] - row[k] * p.per_row;
      if (b >= p.per_row) { b -= p.per_row; ++row[k]; }                            // the product is at most one short
      col[k] = b * 128 + sub * 8;
      live[k] = at[k] < total && col[k] < p.cols;
      gq[k] = uq[k] = make_uint4(0, 0, 0, 0);
      if (live[k]) {
        gq[k] = __ldcs(reinterpret_cast<const uint4*>(p.gate + row[k] * p.ld + col[k]));
        uq[k] = __ldcs(reinterpret_cast<const uint4*>(p.up + row[k] * p.ld + col[k]));
      }
    }
    uint64_t h[2][4];
    float amax[2], inv[2], mine;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint64_t g[4], u[4];
      unpack8(gq[k], g);
      unpack8(uq[k], u);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[k][j] = mul2(silu2(g[j]), u[j]);               // zeros where nothing was loaded
    }
    const bool far[2] = {far8(gq[0]), far8(gq[1])};
    if (__any_sync(0xffffffffu, far[0] || far[1])) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (far[k]) {
          const __nv_bfloat16 *gp = p.gate + row[k] * p.ld + col[k], *up = p.up + row[k] * p.ld + col[k];   // read again: nothing is held for this path
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float ga = __bfloat162float(gp[2 * j]), gb = __bfloat162float(gp[2 * j + 1]);
            h[k][j] = pair(ga < kFarGate ? silu_far(ga, __bfloat162float(up[2 * j])) : lo(h[k][j]),
                           gb < kFarGate ? silu_far(gb, __bfloat162float(up[2 * j + 1])) : hi(h[k][j]));
          }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) amax[k] = max16(absmax8(h[k]));
    block_scales<2>(amax, F.max_val, mine, inv);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (sub == k && at[k] < total) p.scales[at[k]] = mine;
      const uint64_t inv2 = pair(inv[k], inv[k]), q[4] = {mul2(h[k][0], inv2), mul2(h[k][1], inv2), mul2(h[k][2], inv2), mul2(h[k][3], inv2)};
      uint2 codes = encode8<MODE>(q, p.fmt, p.rounding, F);
      if (MODE == kE4m3Rne) {
        uint32_t near = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < 4; ++j) near = __vimin3_u32(near, to_middle(lo(q[j])), to_middle(hi(q[j])));
        const bool mine = live[k] && in_range(amax[k]) && near < 2 * kNear;
        if (__any_sync(0xffffffffu, mine)) {                                       // one warp in some two hundred
          const uint2 m = mine ? make_uint2(near4(q[0], q[1]), near4(q[2], q[3])) : make_uint2(0, 0);
          const uint2 exact = swiglu_exact8(p.gate + row[k] * p.ld + col[k], p.up + row[k] * p.ld + col[k], live[k]);
          codes = make_uint2((exact.x & m.x) | (codes.x & ~m.x), (exact.y & m.y) | (codes.y & ~m.y));
        }
      }
      if (live[k]) *reinterpret_cast<uint2*>(p.codes + row[k] * p.cols + col[k]) = codes;
    }
  }
}

// Any length and alignment: one warp per block of 128 columns, every element by the steps of the kernel above, so that codes and scales do not
// depend on where the operands lie.
__global__ void __launch_bounds__(256) swiglu_block128_generic_kernel(const SwigluArgs p) {
  b2q_pdl_entry();
  const int64_t nb = (p.cols + 127) >> 7, total = p.rows * nb;
  const int lane = threadIdx.x & 31;
  const Fp8Fmt F = fp8_fmt(p.fmt);
  const bool e4m3_rne = p.fmt == B2Q_FP8_E4M3 && p.rounding == B2Q_ROUND_RNE;
  for (int64_t b0 = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); b0 < total; b0 += (int64_t)gridDim.x * 8) {
    const int64_t r = b0 / nb, b = b0 - r * nb;
    float g[4], u[4], h[4], amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = b * 128 + j * 32 + lane;
      g[j] = c < p.cols ? __bfloat162float(p.gate[r * p.ld + c]) : 0.0f;
      u[j] = c < p.cols ? __bfloat162float(p.up[r * p.ld + c]) : 0.0f;
      h[j] = g[j] < kFarGate ? silu_far(g[j], u[j]) : __fmul_rn(silu1(g[j]), u[j]);
      amax = fmaxf(amax, fabsf(h[j]));
    }
    amax = warp_max(amax);
    const float scale = block_scale(amax, F.max_val), inv = __frcp_rn(scale);
    if (lane == 0) p.scales[b0] = scale;
    uint32_t code[4];
    bool near[4], any = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float q = __fmul_rn(h[j], inv);
      code[j] = encode1(q, p.fmt, p.rounding, F);
      near[j] = e4m3_rne && in_range(amax) && b * 128 + j * 32 + lane < p.cols && to_middle(q) < 2 * kNear;
      any |= near[j];
    }
    if (__any_sync(0xffffffffu, any)) {
      double x[4], top = 0.0;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        x[j] = swiglu64(g[j], u[j]);
        top = fmax(top, fabs(x[j]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
      for (int j = 0; j < 4; ++j) if (near[j]) code[j] = encode1(quotient64(x[j], top), p.fmt, p.rounding, F);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = b * 128 + j * 32 + lane;
      if (c < p.cols) p.codes[r * p.cols + c] = (uint8_t)code[j];
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
    // Few rows: one chunk per thread, the shortest chain; many rows: several chunks per thread, so that more CTAs share an SM.  Measured with 1, 2
    // and 4 chunks, us (taken: *): 7 x 4096 2.1*, 2.1, 2.9;  64 x 8192 2.8*, 2.6, 3.4;  512 x 8192 7.6, 6.6, 6.6*;  4096 x 8192 53, 45, 40*;
    // 4096 x 4096 24, 22, 20*;  4096 x 2048 12.2, 10.3*, 11.1.
    int nch = chunks <= 1024 ? 1 : (chunks <= 2048 ? 2 : 4);
    if (rows >= 2 * (int64_t)h->sm_count && chunks > 128) nch = chunks <= 256 ? 2 : 4;
    const dim3 block((unsigned)(ceil_div64(ceil_div64(chunks, nch), 32) * 32));
    const bool main = fmt == B2Q_FP8_E4M3 && rounding == B2Q_ROUND_RNE;
    auto kernel = nch == 1 ? (main ? rms_norm_block128_kernel<1, kE4m3Rne> : rms_norm_block128_kernel<1, kAny>)
                : nch == 2 ? (main ? rms_norm_block128_kernel<2, kE4m3Rne> : rms_norm_block128_kernel<2, kAny>)
                           : (main ? rms_norm_block128_kernel<4, kE4m3Rne> : rms_norm_block128_kernel<4, kAny>);
    B2Q_CUDA(h, b2q_pdl_launch(pdl, kernel, grid, block, 0, h->stream, p));
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
  const int64_t per_row = ceil_div64(cols, 128), total = rows * per_row;
  SwigluArgs p{static_cast<const __nv_bfloat16*>(gate), static_cast<const __nv_bfloat16*>(up), rows, cols, ld, fmt, rounding, scales, codes,
               (uint32_t)per_row, 0xFFFFFFFFu / (uint32_t)(per_row > 0xFFFFFFFFll ? 1 : per_row)};
  const bool vec = total < (1ll << 31) && cols < (1ll << 31) && cols % 8 == 0 && ld % 8 == 0 && ((reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(up)) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  const int64_t ctas = ceil_div64(total, vec ? 16 : 8), most = (int64_t)h->sm_count * (vec ? 24 : 32);
  const dim3 grid((unsigned)(ctas < most ? ctas : most));
  auto kernel = !vec ? swiglu_block128_generic_kernel
                     : fmt == B2Q_FP8_E4M3 && rounding == B2Q_ROUND_RNE ? swiglu_block128_kernel<kE4m3Rne> : swiglu_block128_kernel<kAny>;
  B2Q_CUDA(h, b2q_pdl_launch(h->sw.chain_pdl != 0, kernel, grid, dim3(256), 0, h->stream, p));
  return B2Q_OK;
}

// FP8 GEMM whose scales go per block of 128 along K:
//   out[m, n] = sum_b sa[m, b] * sw[n / 128, b] * sum_{k in block b} A[m, k] * W[n, k]
// A [M x K] and W [N x K] E4M3 / E5M2 codes, both K-major; sa [M x ceil(K / 128)], sw [ceil(N / 128) x ceil(K / 128)] f32.
#include "tc_common.cuh"

namespace b128 {

constexpr int T = 16;   // 16 x 16 outputs per CTA

// Any shape and alignment: codes decoded through a table, f32 FMA over k ascending, one block of K after the other.
__global__ void __launch_bounds__(T * T) gemm_fp8_block128_simt_kernel(const uint8_t* __restrict__ a, const uint8_t* __restrict__ w, int64_t M, int64_t N,
                                                                       int64_t K, int fmt, const float* __restrict__ sa, const float* __restrict__ sw,
                                                                       void* out, int out_type) {
  __shared__ float lut[256];
  __shared__ float As[T][65];
  __shared__ float Ws[T][65];
  const int tid = threadIdx.y * T + threadIdx.x;
  lut[tid] = fp8_decode_ieee_dev((uint32_t)tid, fp8_fmt(fmt));
  __syncthreads();
  const int64_t kb = (K + 127) >> 7;
  for (int64_t m0 = (int64_t)blockIdx.y * T; m0 < M; m0 += (int64_t)gridDim.y * T) {
    const int64_t m = m0 + threadIdx.y, n = (int64_t)blockIdx.x * T + threadIdx.x;
    float acc = 0.0f, part = 0.0f;
    for (int64_t k0 = 0; k0 < K; k0 += 64) {
      for (int i = tid; i < T * 64; i += T * T) {
        const int r = i >> 6, kk = i & 63;
        const int64_t k = k0 + kk, am = m0 + r, wn = (int64_t)blockIdx.x * T + r;
        As[r][kk] = (am < M && k < K) ? lut[a[am * K + k]] : 0.0f;
        Ws[r][kk] = (wn < N && k < K) ? lut[w[wn * K + k]] : 0.0f;
      }
      __syncthreads();
#pragma unroll 16
      for (int kk = 0; kk < 64; ++kk) part = fmaf(As[threadIdx.y][kk], Ws[threadIdx.x][kk], part);
      __syncthreads();
      if ((k0 & 64) || k0 + 64 >= K) {
        if (m < M && n < N) acc = fmaf(part, sa[m * kb + (k0 >> 7)] * sw[(n >> 7) * kb + (k0 >> 7)], acc);
        part = 0.0f;
      }
    }
    if (m < M && n < N) {
      if (out_type == B2Q_OUT_BF16) reinterpret_cast<__nv_bfloat16*>(out)[m * N + n] = __float2bfloat16_rn(acc);
      else reinterpret_cast<float*>(out)[m * N + n] = acc;
    }
  }
}

}  // namespace b128

extern "C" int32_t b2q_gemm_fp8_block128(b2q_handle h, const uint8_t* a, const uint8_t* w, int64_t M, int64_t N, int64_t K, int fmt,
                                         const float* scale_a, const float* scale_w, void* out, int out_type) {
  B2Q_REQUIRE_HANDLE(h);
  if (M <= 0 || N <= 0 || K <= 0)
    B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "gemm_fp8_block128: dimensions must be non-zero: m=%lld, n=%lld, k=%lld", (long long)M, (long long)N, (long long)K);
  if (M > 0x7FFFFFFF || N > 0x7FFFFFFF || K > 0x7FFFFFFF)
    B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "gemm_fp8_block128: dimensions above 2^31 - 1: m=%lld, n=%lld, k=%lld", (long long)M, (long long)N, (long long)K);
  if (!a || !w || !scale_a || !scale_w || !out) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "gemm_fp8_block128: null pointer");
  if (fmt < 0 || fmt > 1 || out_type < 0 || out_type > 1) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "gemm_fp8_block128: bad enum value");
  const uintptr_t c0 = reinterpret_cast<uintptr_t>(out), c1 = c0 + (size_t)(M * N) * (out_type == B2Q_OUT_BF16 ? 2 : 4);
  auto overlaps = [&](const void* p, size_t bytes) { const uintptr_t b = reinterpret_cast<uintptr_t>(p); return c0 < b + bytes && b < c1; };
  const int64_t kb = ceil_div64(K, 128);
  if (overlaps(a, (size_t)(M * K)) || overlaps(w, (size_t)(N * K)) || overlaps(scale_a, (size_t)(M * kb) * 4) || overlaps(scale_w, (size_t)(ceil_div64(N, 128) * kb) * 4))
    B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "gemm_fp8_block128: output buffer overlaps an input");
  const int64_t gy = ceil_div64(M, b128::T);
  dim3 grid((unsigned)ceil_div64(N, b128::T), (unsigned)(gy < 32768 ? gy : 32768));
  b128::gemm_fp8_block128_simt_kernel<<<grid, dim3(b128::T, b128::T), 0, h->stream>>>(a, w, M, N, K, fmt, scale_a, scale_w, out, out_type);
  B2Q_LAUNCH_CHECK(h, "gemm_fp8_block128_simt_kernel");
  return B2Q_OK;
}

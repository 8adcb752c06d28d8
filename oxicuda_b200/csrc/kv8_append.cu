// New keys and values into the paged 8-bit cache (layout: kv8.cuh).
//
// The scale of a page and head is 2^e with the smallest e for which absmax <= 448 * 2^e over the tokens the page holds
// (clamped to [-50, 119]): a power of two costs an E4M3 code no precision but where it falls below the normal range, and
// lets a page's scale grow later by re-encoding its codes exactly (again but for subnormals).  Page and head belong to
// one warp or one CTA: it takes the absmax of the new tokens that fall into the page, raises the page's scale if it must (a page that
// held tokens before never shrinks its scale), re-encodes the tokens already there, and writes the new ones.  No atomics:
// the result does not depend on the order in which pages are written.
// A NaN is stored as 0 and an infinity as the largest code, and B2Q_ERR_NON_FINITE_FP8 is recorded.
// Bound by latency for single tokens (two dependent reads), else by HBM: 2 bytes read and 1 written per channel.
#include "kv8.cuh"
#include <type_traits>

namespace kv8 {

constexpr int kMinExp = -50, kMaxExp = 119;

struct AppendArgs {
  Batch t;
  const __nv_bfloat16* x[2]; int64_t ld[2];      // keys, values: [tokens][n_kv_heads][head_dim], ld elements from token to token
  uint8_t* codes[2]; uint8_t* scales[2];
  int units;                                     // upper bound of (sequence, page) pairs that receive tokens
};

// smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8)
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(kMaxExp, max(kMinExp, e));          // a subnormal or zero amax ends at kMinExp
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // e in [-126, 127]

// Eight bf16 -> the largest finite size among them, and whether one is not finite.
__device__ __forceinline__ void scan8(const uint4 q, float& amax, bool& bad) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const float v = fabsf(__uint_as_float(s ? (w[j] & 0xFFFF0000u) : (w[j] << 16)));
      const bool fin = v < INFINITY;
      bad |= !fin;
      amax = fmaxf(amax, fin ? v : 0.0f);
    }
}
__device__ __forceinline__ uint2 encode8(const uint4 q, float inv) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a = __uint_as_float(w[j] << 16) * inv, b = __uint_as_float(w[j] & 0xFFFF0000u) * inv;
    a = a == a ? a : 0.0f;
    b = b == b ? b : 0.0f;
    o[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(o[0] | (o[1] << 16), o[2] | (o[3] << 16));
}
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  uint32_t half[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * s)), __NV_E4M3)));
    half[s] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v.x * f, v.y * f), __NV_SATFINITE, __NV_E4M3);
  }
  return half[0] | (half[1] << 16);
}

// W warps to each (page, head, keys or values), ROWS new tokens at most: they are read once, into registers, and encoded from there.
// ROWS = 1: one token per sequence.  Pages of 16 and 32 take a warp (four pages to a CTA), larger ones a CTA: with a CTA to a page of 16 a
// prompt of 1500 tokens took 44 us instead of 22, with a warp to a page of 128 it took 50 instead of 20.
template <int D, int ROWS>
__global__ void __launch_bounds__(128) kv8_append_kernel(const AppendArgs p) {
  constexpr bool SINGLE = ROWS == 1;
  constexpr int W = ROWS > 32 ? 4 : 1;
  constexpr int LPR = D / 8, RPW = 32 / LPR;     // lanes per token row (16-byte loads), rows a warp takes at once
  constexpr int STEP = W * RPW, NI = (ROWS + STEP - 1) / STEP;
  b2q_pdl_entry();
  const Batch& t = p.t;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % LPR, row = (W == 1 ? 0 : warp * RPW) + lane / LPR;
  const int ps = 1 << t.page_shift;
  const int64_t item = W == 1 ? (int64_t)blockIdx.x * 4 + warp : blockIdx.x;
  const int per = 2 * t.n_kv_heads;
  if (item >= (int64_t)p.units * per) return;
  const int unit = (int)(item / per), head = (int)(item % per) >> 1, kv = (int)(item & 1);
  const bool tell = head == 0 && kv == 0 && (W == 1 || warp == 0);
  Found f;
  if (SINGLE) f = Found{unit, 0, 1};
  else {
    if (unit == 0 && tell) for (int b = lane; b < t.seqs; b += 32) rows_of(t, b, true);
    f = find_unit(t.seqs, unit, [&](int b) {
      const Rows r = rows_of(t, b, false);
      return r.n > 0 ? ((r.len - 1) >> t.page_shift) - ((r.len - r.n) >> t.page_shift) + 1 : 0;
    });
    if (f.b < 0) return;
  }
  const Rows r = rows_of(t, f.b, SINGLE && tell && lane == 0);
  if (r.n == 0) return;
  const int first = r.len - r.n;                                        // position of the first new token
  const int index = (first >> t.page_shift) + f.index;
  const int pg = page_of(t, f.b, index, tell && lane == 0);
  if (pg < 0) return;
  const int base = index << t.page_shift;
  const int lo = max(first, base), n = min(r.len, base + ps) - lo;      // first position and number of rows that this page receives
  const int held = lo - base;                                           // tokens it holds already
  const __nv_bfloat16* x = p.x[kv] + (int64_t)(r.r0 + lo - first) * p.ld[kv] + (int64_t)head * D + sub * 8;
  const int64_t tile = (int64_t)pg * t.n_kv_heads + head;
  uint8_t* codes = p.codes[kv] + (tile << t.page_shift) * D + sub * 8;
  const int old = held > 0 ? (int)p.scales[kv][tile] - 127 : kMinExp;

  uint4 q[NI];
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int i = k * STEP + row;
    q[k] = i < n ? __ldg(reinterpret_cast<const uint4*>(x + (int64_t)i * p.ld[kv])) : make_uint4(0, 0, 0, 0);
  }
  float amax = 0.0f;
  bool bad = false;
#pragma unroll
  for (int k = 0; k < NI; ++k) if (k * STEP < n) scan8(q[k], amax, bad);
  amax = warp_max(amax);
  if (__any_sync(0xffffffffu, bad) && lane == 0) report(t.status, B2Q_ERR_NON_FINITE_FP8);
  if (W > 1) {
    __shared__ float sh[4];
    if (lane == 0) sh[warp] = amax;
    __syncthreads();                                                    // also: every warp has read the page's scale
    amax = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
  }
  const int e = max(old, scale_exp(amax));
  if (held > 0 && e > old) {                                            // the tokens already there move to the larger scale
    const float f2 = pow2f(max(old - e, -126));
    for (int i = row; i < held; i += STEP) {
      uint2* c = reinterpret_cast<uint2*>(codes + (int64_t)i * D);
      const uint2 was = *c;
      *c = make_uint2(rescale4(was.x, f2), rescale4(was.y, f2));
    }
  }
  const float inv = pow2f(-e);
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const int i = k * STEP + row;
    if (i < n) *reinterpret_cast<uint2*>(codes + (int64_t)(held + i) * D) = encode8(q[k], inv);
  }
  if (lane == 0 && (W == 1 || warp == 0)) p.scales[kv][tile] = (uint8_t)(e + 127);
}

}  // namespace kv8

extern "C" int32_t b2q_kv8_append_bf16(b2q_handle h, const void* k, const void* v, int64_t ld_k, int64_t ld_v, int64_t tokens, const int32_t* q_starts,
                                       const int32_t* seq_lens, const int32_t* block_tables, int64_t seqs, int64_t table_width, int64_t num_pages,
                                       int64_t page_size, int64_t n_kv_heads, int64_t head_dim, uint8_t* k_codes, uint8_t* v_codes, uint8_t* k_scales,
                                       uint8_t* v_scales) {
  B2Q_REQUIRE_HANDLE(h);
  kv8::AppendArgs p{};
  int32_t st = b2q_kv8_batch(h, "kv8_append", tokens, q_starts, seq_lens, block_tables, seqs, table_width, num_pages, page_size, n_kv_heads, head_dim, &p.t);
  if (st != B2Q_OK) return st;
  if (!k || !v || !k_codes || !v_codes || !k_scales || !v_scales) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "kv8_append: null pointer");
  if (ld_k < n_kv_heads * head_dim || ld_v < n_kv_heads * head_dim || ld_k % 8 != 0 || ld_v % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15) != 0)
    B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "kv8_append: tensors must be 16-byte aligned, token strides multiples of 8 elements and at least n_kv_heads * head_dim");
  p.x[0] = static_cast<const __nv_bfloat16*>(k); p.x[1] = static_cast<const __nv_bfloat16*>(v);
  p.ld[0] = ld_k; p.ld[1] = ld_v;
  p.codes[0] = k_codes; p.codes[1] = v_codes; p.scales[0] = k_scales; p.scales[1] = v_scales;
  // a sequence with n new tokens touches at most (n - 1) / page_size + 2 pages, and never more than n
  int64_t units = tokens;
  if (q_starts && tokens / page_size + 2 * seqs < units) units = tokens / page_size + 2 * seqs;
  p.units = (int)units;
  const int64_t items = units * 2 * n_kv_heads, ctas = q_starts && page_size > 32 ? items : ceil_div64(items, 4);
  if (ctas > 0x7FFFFFFF) B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_append: %lld tokens are too many", (long long)tokens);
  auto pick = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    return !q_starts ? kv8::kv8_append_kernel<D, 1> : page_size == 16 ? kv8::kv8_append_kernel<D, 16> : page_size == 32 ? kv8::kv8_append_kernel<D, 32>
                                                  : page_size == 64 ? kv8::kv8_append_kernel<D, 64> : kv8::kv8_append_kernel<D, 128>;
  };
  auto kernel = head_dim == 64 ? pick(std::integral_constant<int, 64>()) : pick(std::integral_constant<int, 128>());
  B2Q_CUDA(h, b2q_pdl_launch(h->sw.chain_pdl != 0, kernel, dim3((unsigned)ctas), dim3(128), 0, h->stream, p));
  return B2Q_OK;
}

// The checks of a batch that append and attention share.
int32_t b2q_kv8_batch(b2q_handle h, const char* who, int64_t tokens, const int32_t* q_starts, const int32_t* seq_lens, const int32_t* block_tables,
                      int64_t seqs, int64_t table_width, int64_t num_pages, int64_t page_size, int64_t n_kv_heads, int64_t head_dim, kv8::Batch* out) {
  if (tokens <= 0 || seqs <= 0) B2Q_FAIL(h, B2Q_ERR_EMPTY_INPUT, "%s: empty batch (%lld tokens, %lld sequences)", who, (long long)tokens, (long long)seqs);
  if (table_width <= 0 || num_pages <= 0 || n_kv_heads <= 0)
    B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "%s: dimensions must be non-zero: table_width=%lld, num_pages=%lld, n_kv_heads=%lld", who, (long long)table_width,
             (long long)num_pages, (long long)n_kv_heads);
  if (!seq_lens || !block_tables) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!q_starts && tokens != seqs)
    B2Q_FAIL(h, B2Q_ERR_DIMENSION_MISMATCH, "%s: without q_starts every sequence has one token: expected %lld tokens, got %lld", who, (long long)seqs, (long long)tokens);
  if (head_dim != 64 && head_dim != 128) B2Q_FAIL(h, B2Q_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128, got %lld", who, (long long)head_dim);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    B2Q_FAIL(h, B2Q_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64 or 128, got %lld", who, (long long)page_size);
  if (tokens > (1 << 30) || seqs > (1 << 24) || n_kv_heads > 4096 || table_width > (1 << 24) || (table_width * page_size) > 0x7FFFFFFF ||
      num_pages > 0x7FFFFFFF / (n_kv_heads * page_size))
    B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "%s: too large: tokens=%lld, sequences=%lld, table_width=%lld, num_pages=%lld", who, (long long)tokens,
             (long long)seqs, (long long)table_width, (long long)num_pages);
  out->q_starts = q_starts; out->seq_lens = seq_lens; out->table = block_tables;
  out->seqs = (int)seqs; out->table_width = (int)table_width; out->tokens = (int)tokens;
  out->num_pages = num_pages; out->page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  out->n_kv_heads = (int)n_kv_heads;
  out->status = h->d_status;
  return B2Q_OK;
}

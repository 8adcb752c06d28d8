// Attention of few query rows over the paged 8-bit cache (layout: kv8.cuh):
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  keys j <= pos_i (pos_i = len - n + i), with a window also j > pos_i - window.
// Bound by HBM: the codes of the visible keys and values are read once; everything else is small.
//
// A row is one (new token, query head) pair; the rows of one sequence and kv head that share keys are taken 8 at a time.  The
// codes feed mma.sync.m16n8k32 (E4M3 x E4M3, f32 sums) as they are stored:
//   scores   A = the 8 query rows twice: rows 0..7 the E4M3 rounding of q / 2^e, rows 8..15 the E4M3 rounding of what that
//            leaves, 2^e the power of two that brings the row's largest element into (224, 448].  A bf16 has 8 significant
//            bits and an E4M3 code 4, so the two terms add up to q exactly but for elements below 2^-9 of the row's largest
//            (absolute error at most 2^-10 * 2^e, 2^-17 of that element).  B = K as loaded, 4 channels per register.
//   outputs  A = the weights p = exp2(s - m) * 2^8, split the same way (relative error 2^-9 where a bf16 weight would have
//            2^-9 too); B = V, whose 4 x 4 byte tiles are transposed in registers (two byte permutations per register).
// One warp takes 32 keys at a time with its own running maximum and sum, so the main loop has no barrier; warps and the CTAs
// of a cluster (keys dealt round in tiles of 32) are joined once at the end, through shared and distributed shared memory:
// no workspace, one launch, and a result that does not depend on timing.
// The value scale is a power of two 2^lv per page: weights enter as p * 2^(8 + lv - R) and the outputs are kept in units of
// 2^(R - 8), R following the pages' scales, so the split keeps its precision whatever the pages' sizes are; pages of one tile
// whose scales lie more than 2^4 apart are multiplied one after the other.
// Keys behind the last visible one are never read (their codes count as zeros), so stale pages cannot reach a result.
#include "kv8.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace kv8 {

constexpr int kWarps = 4, kRows = 8, kTile = 32;
constexpr int kNone = -1000;                     // R of a warp that has seen no page

struct AttendArgs {
  Batch t;
  const __nv_bfloat16* q; int64_t ld_q;
  const uint8_t* k; const uint8_t* v; const uint8_t* ks; const uint8_t* vs;
  int group;                                     // query heads per kv head
  int window;                                    // 0: none
  float scale;                                   // softmax scale * log2(e)
  __nv_bfloat16* out; float* lse;                // [tokens][heads][head_dim], [tokens][heads]
};

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// two values -> two E4M3 codes (low half) and the codes of what the first rounding left
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __nv_fp8x2_storage_t h = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
  const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(h, __NV_E4M3)));
  hi = h;
  lo = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x - b.x, y - b.y), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(min(127, max(-126, e)) + 127) << 23); }
__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) { return __ldcs(reinterpret_cast<const uint4*>(p)); }

template <int D>
__global__ void __launch_bounds__(32 * kWarps, 3) kv8_decode_kernel(const AttendArgs p) {
  constexpr int KC = D / 64;                     // 16-byte chunks of a key row per lane
  constexpr int NT = D / 8;                      // n-tiles of the outputs
  constexpr int VB = D / 8;                      // bytes of a value row per lane (columns c * VB ..)
  __shared__ __align__(16) float s_o[kWarps][kRows][D];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ int s_r[kWarps];
  __shared__ float s_cm[kRows], s_cl[kRows];     // this CTA's join
  __shared__ int s_cr;

  b2q_pdl_entry();
  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const Batch& t = p.t;
  const int head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, tq = lane & 3;
  const int unit = (int)(blockIdx.x / split);
  const bool tell = head == 0 && part == 0 && warp == 0;

  int2 f;
  if (t.q_starts == nullptr) {
    const int per = (p.group + kRows - 1) / kRows;
    f = make_int2(unit / per, unit % per);
  } else {
    if (unit == 0 && tell) for (int b = lane; b < t.seqs; b += 32) rows_of(t, b, true);
    f = find_unit(t.seqs, unit, [&](int b) { return (int)(((int64_t)rows_of(t, b, false).n * p.group + kRows - 1) / kRows); });
    if (f.x < 0) return;                          // the whole cluster leaves: every CTA of it has the same unit
  }
  const Rows r = rows_of(t, f.x, tell && t.q_starts == nullptr && lane == 0);
  const int64_t rows = (int64_t)r.n * p.group, row0 = (int64_t)f.y * kRows;
  const int valid = (int)min((int64_t)kRows, rows - row0);            // <= 0: an impossible sequence, its rows stay as they are
  if (valid <= 0) return;
  const bool live = row < valid;
  const int token = live ? (int)((row0 + row) / p.group) : 0;
  const int qhead = head * p.group + (live ? (int)((row0 + row) % p.group) : 0);
  const int pos = live ? r.len - r.n + token : -1;
  const int first_pos = r.len - r.n + (int)(row0 / p.group), last_pos = r.len - r.n + (int)((row0 + valid - 1) / p.group);
  const int key_end = last_pos + 1;
  const int key_begin = p.window > 0 ? max(0, first_pos - p.window + 1) & ~(kTile - 1) : 0;

  // ---- the query rows as two E4M3 terms ----
  uint32_t qa[2 * KC][4];
  float qf;
  {
    const __nv_bfloat16* qp = p.q + (int64_t)(r.r0 + token) * p.ld_q + (int64_t)qhead * D + tq * 16;
    uint4 w[KC][2];
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        w[c][s] = live ? *reinterpret_cast<const uint4*>(qp + c * 64 + s * 8) : make_uint4(0, 0, 0, 0);
        const uint32_t u[4] = {w[c][s].x, w[c][s].y, w[c][s].z, w[c][s].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = fabsf(__uint_as_float(u[j] << 16)), b = fabsf(__uint_as_float(u[j] & 0xFFFF0000u));
          bad |= !(a < INFINITY) || !(b < INFINITY);
          amax = fmaxf(amax, fmaxf(a, b));
        }
      }
    amax = quad_max(amax);
    bad = (__ballot_sync(0xffffffffu, bad) >> (lane & 28)) & 0xF;
    const uint32_t u = __float_as_uint(amax);
    const int e = max(-119, (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0));
    const float inv = pow2i(-e);
    qf = bad ? __uint_as_float(0x7FC00000u) : p.scale * pow2i(e);
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t uw[4] = {w[c][s].x, w[c][s].y, w[c][s].z, w[c][s].w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) split2(__uint_as_float(uw[j] << 16) * inv, __uint_as_float(uw[j] & 0xFFFF0000u) * inv, hi[j], lo[j]);
        qa[2 * c + s][0] = hi[0] | (hi[1] << 16); qa[2 * c + s][1] = lo[0] | (lo[1] << 16);
        qa[2 * c + s][2] = hi[2] | (hi[3] << 16); qa[2 * c + s][3] = lo[2] | (lo[3] << 16);
      }
  }

  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[j][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  int R = kNone;

  const int step = kTile * kWarps * split;
  // page and scales of the 8-key group lane & 3 of a tile (a group never crosses a page)
  auto fetch = [&](int j0, int& pg, uint32_t& sc) {
    pg = -1; sc = 0;
    const int j = j0 + 8 * tq;
    if (j < key_end) {
      pg = page_of(t, f.x, j >> t.page_shift, head == 0);
      if (pg >= 0) sc = (uint32_t)p.ks[(int64_t)pg * t.n_kv_heads + head] | ((uint32_t)p.vs[(int64_t)pg * t.n_kv_heads + head] << 8);
    }
  };
  int j0 = key_begin + kTile * (part * kWarps + warp);
  int npg; uint32_t nsc;
  fetch(j0, npg, nsc);
  for (; j0 < key_end; j0 += step) {
    int pg[4]; uint32_t sc[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) { pg[g] = __shfl_sync(0xffffffffu, npg, g); sc[g] = __shfl_sync(0xffffffffu, nsc, g); }
    uint4 kr[4][KC];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int j = j0 + 8 * g + row;
      const bool in = pg[g] >= 0 && j < key_end;
      const uint8_t* kp = p.k + (((((int64_t)pg[g] * t.n_kv_heads + head) << t.page_shift) + (j & ((1 << t.page_shift) - 1))) * D) + tq * 16;
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[g][c] = in ? ld_stream(kp + c * 64) : make_uint4(0, 0, 0, 0);
    }
    uint32_t vr[4][2][VB / 4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + 8 * g + 2 * tq + e;
        const bool in = pg[g] >= 0 && j < key_end;
        const uint8_t* vp = p.v + (((((int64_t)pg[g] * t.n_kv_heads + head) << t.page_shift) + (j & ((1 << t.page_shift) - 1))) * D) + row * VB;
        if constexpr (D == 128) {
          const uint4 x = in ? ld_stream(vp) : make_uint4(0, 0, 0, 0);
          vr[g][e][0] = x.x; vr[g][e][1] = x.y; vr[g][e][2] = x.z; vr[g][e][3] = x.w;
        } else {
          const uint2 x = in ? __ldcs(reinterpret_cast<const uint2*>(vp)) : make_uint2(0, 0);
          vr[g][e][0] = x.x; vr[g][e][1] = x.y;
        }
      }
    fetch(j0 + step, npg, nsc);

    // ---- scores of 8 rows x 32 keys: this lane has keys j0 + 8 g + 2 tq + {0, 1} of its row ----
    float s[4][2], mt = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < KC; ++x) {
        mma_e4m3(c, qa[2 * x][0], qa[2 * x][1], qa[2 * x][2], qa[2 * x][3], kr[g][x].x, kr[g][x].y);
        mma_e4m3(c, qa[2 * x + 1][0], qa[2 * x + 1][1], qa[2 * x + 1][2], qa[2 * x + 1][3], kr[g][x].z, kr[g][x].w);
      }
      const float kf = qf * pow2_byte(sc[g] & 0xFF);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + 8 * g + 2 * tq + e;
        const bool see = j <= pos && (p.window <= 0 || j > pos - p.window) && pg[g] >= 0;
        s[g][e] = see ? (c[e] + c[2 + e]) * kf : -INFINITY;
        mt = fmaxf(mt, s[g][e]);
      }
    }
    const float mn = fmaxf(m, quad_max(mt));
    const float base = mn == -INFINITY ? 0.0f : mn;                   // a row that has seen nothing yet: exp2(-inf - 0) = 0
    float alpha = exp2f(m - base);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) { s[g][e] = exp2f(s[g][e] - base); l += s[g][e]; }

    // ---- outputs: the groups whose value scales lie within 2^4 of the largest at a time (nearly always all of them) ----
    unsigned rem = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) rem |= (pg[g] >= 0 && j0 + 8 * g < key_end) ? 1u << g : 0u;
    while (rem) {
      int lead = kNone;
#pragma unroll
      for (int g = 0; g < 4; ++g) if (rem >> g & 1) lead = max(lead, (int)(sc[g] >> 8) - 127);
      unsigned take = 0;
      if (R == kNone) R = lead;
      const int was = R;
      R = lead > R || lead < R - 4 ? lead : R;
      alpha *= pow2i(was - R);
      float w[4][2];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int lv = (int)(sc[g] >> 8) - 127;
        const bool on = (rem >> g & 1) && lv >= lead - 4;
        take |= on ? 1u << g : 0u;
        const float up = on ? pow2i(8 + lv - R) : 0.0f;
        w[g][0] = s[g][0] * up; w[g][1] = s[g][1] * up;
      }
      rem &= ~take;
      if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] *= alpha;
        alpha = 1.0f;
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) split2(w[g][0], w[g][1], hi[g], lo[g]);
      const uint32_t a0 = hi[0] | (hi[1] << 16), a1 = lo[0] | (lo[1] << 16), a2 = hi[2] | (hi[3] << 16), a3 = lo[2] | (lo[3] << 16);
#pragma unroll
      for (int x = 0; x < VB / 4; ++x) {                              // 4 columns at a time: 4 x 4 byte transposes
        uint32_t b[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t r0 = vr[2 * h][0][x], r1 = vr[2 * h][1][x], r2 = vr[2 * h + 1][0][x], r3 = vr[2 * h + 1][1][x];
          const uint32_t t0 = __byte_perm(r0, r1, 0x5140), t1 = __byte_perm(r0, r1, 0x7362), t2 = __byte_perm(r2, r3, 0x5140), t3 = __byte_perm(r2, r3, 0x7362);
          b[h][0] = __byte_perm(t0, t2, 0x5410); b[h][1] = __byte_perm(t0, t2, 0x7632);
          b[h][2] = __byte_perm(t1, t3, 0x5410); b[h][3] = __byte_perm(t1, t3, 0x7632);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) mma_e4m3(o[4 * x + i], a0, a1, a2, a3, b[0][i], b[1][i]);
      }
    }
  }

  // ---- join the warps of this CTA, then the CTAs of the cluster ----
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  if (tq == 0) { s_m[warp][row] = m; s_l[warp][row] = l; }
  if (lane == 0) s_r[warp] = R;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int j = 0; j < NT; j += 4)                                   // columns (2 tq + e) * VB + j ..
      *reinterpret_cast<float4*>(&s_o[warp][row][(2 * tq + e) * VB + j]) =
          make_float4(o[j][e] + o[j][2 + e], o[j + 1][e] + o[j + 1][2 + e], o[j + 2][e] + o[j + 2][2 + e], o[j + 3][e] + o[j + 3][2 + e]);
  __syncthreads();
  int cr = kNone;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) cr = max(cr, s_r[w]);
  for (int i = threadIdx.x; i < kRows * D / 4; i += 32 * kWarps) {
    const int rr = i / (D / 4), cc = (i % (D / 4)) * 4;
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][rr]);
    const float b = mm == -INFINITY ? 0.0f : mm;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = exp2f(s_m[w][rr] - b), fo = a * (s_r[w] == kNone ? 0.0f : pow2i(s_r[w] - cr));
      ll += a * s_l[w][rr];
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][rr][cc]);
      acc.x += fo * x.x; acc.y += fo * x.y; acc.z += fo * x.z; acc.w += fo * x.w;
    }
    *reinterpret_cast<float4*>(&s_o[0][rr][cc]) = acc;                // read and written by this thread alone
    if (cc == 0) { s_cm[rr] = mm; s_cl[rr] = ll; }
  }
  if (threadIdx.x == 0) s_cr = cr;
  if (split > 1) cluster.sync(); else __syncthreads();
  int tr = kNone;
  for (int c = 0; c < split; ++c) tr = max(tr, split > 1 ? *cluster.map_shared_rank(&s_cr, c) : s_cr);
  const int cols = D / split;                                         // this CTA finishes columns part * cols ..
  for (int i = threadIdx.x; i < kRows * cols / 4; i += 32 * kWarps) {
    const int rr = i / (cols / 4), cc = part * cols + (i % (cols / 4)) * 4;
    if (rr >= valid) continue;
    float mm = -INFINITY, ll = 0.0f;
    for (int c = 0; c < split; ++c) mm = fmaxf(mm, split > 1 ? *cluster.map_shared_rank(&s_cm[rr], c) : s_cm[rr]);
    const float b = mm == -INFINITY ? 0.0f : mm;
    float4 acc = make_float4(0, 0, 0, 0);
    for (int c = 0; c < split; ++c) {
      const float a = exp2f((split > 1 ? *cluster.map_shared_rank(&s_cm[rr], c) : s_cm[rr]) - b);
      const int rc = split > 1 ? *cluster.map_shared_rank(&s_cr, c) : s_cr;
      const float fo = a * (rc == kNone ? 0.0f : pow2i(rc - tr));
      ll += a * (split > 1 ? *cluster.map_shared_rank(&s_cl[rr], c) : s_cl[rr]);
      const float4 x = *reinterpret_cast<const float4*>(split > 1 ? cluster.map_shared_rank(&s_o[0][rr][cc], c) : &s_o[0][rr][cc]);
      acc.x += fo * x.x; acc.y += fo * x.y; acc.z += fo * x.z; acc.w += fo * x.w;
    }
    const int tk = (int)((row0 + rr) / p.group), hd = head * p.group + (int)((row0 + rr) % p.group);
    const int64_t orow2 = (int64_t)(r.r0 + tk) * (t.n_kv_heads * p.group) + hd;
    // a row that sees no key has ll = 0: zeros and -inf.  A query that holds an infinity or a NaN has ll = NaN and stays NaN.
    const float inv = ll == 0.0f ? 0.0f : __frcp_rn(ll), up = tr == kNone ? 0.0f : pow2i(tr - 8);
    const __nv_bfloat162 y0 = __floats2bfloat162_rn(acc.x * inv * up, acc.y * inv * up), y1 = __floats2bfloat162_rn(acc.z * inv * up, acc.w * inv * up);
    uint2 pk;
    pk.x = *reinterpret_cast<const uint32_t*>(&y0); pk.y = *reinterpret_cast<const uint32_t*>(&y1);
    *reinterpret_cast<uint2*>(p.out + orow2 * D + cc) = pk;
    if (p.lse && cc == 0) p.lse[orow2] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
  }
  if (split > 1) cluster.sync();                                      // the others may still be reading this CTA's shared memory
}

}  // namespace kv8

template <int D>
static int32_t kv8_decode_launch(b2q_handle h, const kv8::AttendArgs& p, int64_t units, int split) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * split), (unsigned)p.t.n_kv_heads);
  cfg.blockDim = dim3(32 * kv8::kWarps);
  cfg.stream = h->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = h->sw.chain_pdl != 0 ? 2 : 1;
  B2Q_CUDA(h, cudaLaunchKernelEx(&cfg, kv8::kv8_decode_kernel<D>, p));
  return B2Q_OK;
}

extern "C" int32_t b2q_kv8_attention_bf16(b2q_handle h, const void* q, int64_t ld_q, int64_t tokens, int64_t n_heads, const int32_t* q_starts,
                                          const int32_t* seq_lens, const int32_t* block_tables, int64_t seqs, int64_t table_width, int64_t num_pages,
                                          int64_t page_size, int64_t n_kv_heads, int64_t head_dim, const uint8_t* k_codes, const uint8_t* v_codes,
                                          const uint8_t* k_scales, const uint8_t* v_scales, float scale, int64_t window, void* out, float* lse) {
  B2Q_REQUIRE_HANDLE(h);
  kv8::AttendArgs p{};
  int32_t st = b2q_kv8_batch(h, "kv8_attention", tokens, q_starts, seq_lens, block_tables, seqs, table_width, num_pages, page_size, n_kv_heads, head_dim, &p.t);
  if (st != B2Q_OK) return st;
  if (n_heads <= 0 || n_heads % n_kv_heads != 0)
    B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_attention: %lld query heads are not a multiple of %lld kv heads", (long long)n_heads, (long long)n_kv_heads);
  if (!q || !out || !k_codes || !v_codes || !k_scales || !v_scales) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "kv8_attention: null pointer");
  if (ld_q < n_heads * head_dim || ld_q % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15) != 0)
    B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "kv8_attention: tensors must be 16-byte aligned, ld_q a multiple of 8 and at least n_heads * head_dim");
  if (!(scale > -INFINITY && scale < INFINITY)) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "kv8_attention: scale %f is not finite", (double)scale);
  if (window < 0) B2Q_FAIL(h, B2Q_ERR_INVALID_ARGUMENT, "kv8_attention: window %lld is negative", (long long)window);
  p.q = static_cast<const __nv_bfloat16*>(q); p.ld_q = ld_q;
  p.k = k_codes; p.v = v_codes; p.ks = k_scales; p.vs = v_scales;
  p.group = (int)(n_heads / n_kv_heads);
  const int64_t most = table_width * page_size;                        // keys that a sequence can have
  p.window = window > 0 && window < most ? (int)window : 0;
  p.scale = scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out); p.lse = lse;
  const int64_t units = q_starts ? tokens * p.group / kv8::kRows + seqs : seqs * ceil_div64(p.group, kv8::kRows);
  const int64_t keys = p.window ? p.window + kv8::kTile : most;
  int split = 1;
  while (split < 8 && units * n_kv_heads * split * 2 <= 3 * (int64_t)h->sm_count && keys > split * kv8::kTile * kv8::kWarps) split *= 2;
  if (units * split > 0x7FFFFFFF) B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_attention: %lld tokens of %lld heads are too many", (long long)tokens, (long long)n_heads);
  return head_dim == 64 ? kv8_decode_launch<64>(h, p, units, split) : kv8_decode_launch<128>(h, p, units, split);
}

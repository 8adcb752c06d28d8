// Attention of many query rows over the paged 8-bit cache (layout: kv8.cuh), on tcgen05:
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  keys j <= pos_i, with a window also j > pos_i - window.
// A CTA takes 128 rows ((new token, query head) pairs of one sequence and kv head) and walks the keys 64 at a time:
//   S [128 x 64] = Q K^T,   P = exp2(S - m),   O [128 x D] += P V,   S (two of them) and O in TMEM, f32.
// The cache is multiplied as it is stored (tcgen05.mma.kind::f8f6f4, K and V straight from TMA): Q and P enter as two E4M3 terms each,
// the rounding of x and the rounding of what that leaves.  A bf16 has 8 significant bits and an E4M3 code 4, so q / 2^e (2^e brings the
// row's largest element into (224, 448]) is exact but for elements below 2^-9 of the largest, which keep an absolute error of 2^-10 (2^-17
// of it); a weight, held as p * 2^8, is off by 2^-9 of itself, or by 2^-10 absolute below the normal range.  Two FP8 products cost what
// one bf16 product costs, and no code is converted.
// Work per 64 keys and CTA: 640 clocks of tensor core (4 D K-steps of Q K^T at N = 64 read 1.5 x the shared memory that their rate
// allows, P V at N = D runs at rate) against about 700 issue slots of softmax in four warps: two CTAs share an SM, so that one
// multiplies while the other exponentiates.
// The running maximum is followed lazily: it moves only when a score exceeds it by more than 0.75 (p * 2^8 still fits an E4M3), so O is
// rescaled (a round trip through registers) a few times per row and not per tile.  The value scale of a page is a power of two 2^lv:
// weights enter as p * 2^(8 + lv - R) and O is in units of 2^(R - 8); a tile whose pages differ by more than 2^kSpan is walked once per
// group of alike pages, the others masked.
// Warp 0 walks the block table and issues the copies, warp 1 the products, warps 2..5 are the softmax (a thread to a row).
// Keys behind the last visible one are masked and their value rows zeroed before they are multiplied; a page that the table does not
// name is neither read nor counted.  Every mbarrier wait is bounded; on expiry the kernel records B2Q_ERR_TIMEOUT and leaves.
#include "kv8.cuh"
#include "tc_common.cuh"

namespace kv8 {

using namespace tcx;

namespace pre {

constexpr int kRows = 128, kTile = 64;
constexpr int kThreads = 192;
constexpr int kStages = 3, kInfo = 8;            // K and V tiles in flight; tile descriptions (a tile is read at most 5 behind the newest)
constexpr int kSpan = 4;                         // value scales that share a tile differ by at most 2^kSpan
constexpr int kNone = -1000;
constexpr float kSlack = 0.75f;                  // 2^(8 + 0.75) = 430 < 448
constexpr uint64_t kWaitLimitNs = 2000000000ull;

template <int D> struct Cfg {
  static constexpr int kQ = 2 * kRows * D;       // both terms
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kP = kRows * 128;         // hi | lo, 64 keys each
  static constexpr int kSmem = kQ + kP + 2 * kStages * kTileBytes + 1024 + kInfo * 32 + 256;
  static constexpr int kTmemCols = D == 128 ? 256 : 256;   // S: 2 x 64, O: D
};
constexpr uint32_t kThere = 0x80000000u, kTaken = 0x40000000u;

__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// two f16 -> two E4M3 codes, and the codes of what that leaves (exact in f16)
__device__ __forceinline__ void split_f16(uint32_t x, uint16_t& hi, uint16_t& lo) {
  asm("{\n\t.reg .b16 h;\n\t.reg .b32 b, r;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 h, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 b, h;\n\t"
      "sub.rn.f16x2 r, %2, b;\n\t"
      "mov.b16 %0, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f16x2 %1, r;\n\t}" : "=h"(hi), "=h"(lo) : "r"(x));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack16(uint16_t lo, uint16_t hi) { return (uint32_t)lo | ((uint32_t)hi << 16); }

struct Info { uint32_t w[4]; int j0, last; };    // per 16 keys: scales and flags; first key; 1 for the last tile

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
kv8_prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttendArgs p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_at = base, p_at = base + C::kQ, k_at = p_at + C::kP, v_at = k_at + kStages * C::kTileBytes, bar_at = v_at + kStages * C::kTileBytes;
  auto kfull = [&](int s) { return bar_at + 8u * s; };
  auto kempty = [&](int s) { return bar_at + 8u * (kStages + s); };
  auto vfull = [&](int s) { return bar_at + 8u * (2 * kStages + s); };
  auto vempty = [&](int s) { return bar_at + 8u * (3 * kStages + s); };
  auto sfull = [&](int b) { return bar_at + 8u * (4 * kStages + b); };
  auto sempty = [&](int b) { return bar_at + 8u * (4 * kStages + 2 + b); };
  const uint32_t qready = bar_at + 8u * (4 * kStages + 4), pfull = qready + 8, pvdone = qready + 16, drain = qready + 24;
  Info* const s_info = reinterpret_cast<Info*>(smem + (bar_at - base) + 8 * (4 * kStages + 8));
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) { mbar_init(kfull(s), 1); mbar_init(kempty(s), 1); mbar_init(vfull(s), 1); mbar_init(vempty(s), 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(sfull(b), 1); mbar_init(sempty(b), 4); }
    mbar_init(qready, 4); mbar_init(pfull, 4); mbar_init(pvdone, 1); mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- which rows: the longest tiles of a sequence first ----
  const Batch& t = p.t;
  const int head = blockIdx.y;
  const bool tell = head == 0 && warp == 0;
  if (blockIdx.x == 0 && tell) for (int b = lane; b < t.seqs; b += 32) rows_of(t, b, true);
  auto count = [&](int b) { return (int)(((int64_t)rows_of(t, b, false).n * p.group + kRows - 1) / kRows); };
  const int2 f = find_unit(t.seqs, blockIdx.x, count);
  if (f.x < 0) return;                            // the whole CTA leaves, before it holds TMEM
  const Rows r = rows_of(t, f.x, false);
  const int64_t row0 = (int64_t)(count(f.x) - 1 - f.y) * kRows;
  const int valid = (int)min((int64_t)kRows, (int64_t)r.n * p.group - row0);
  const int first_pos = r.len - r.n + (int)(row0 / p.group), last_pos = r.len - r.n + (int)((row0 + valid - 1) / p.group);
  const int key_end = last_pos + 1;
  const int key_begin = p.window > 0 ? max(0, first_pos - p.window + 1) & ~(kTile - 1) : 0;

  if (warp == 1) tmem_alloc(smem_u32(&s_tmem_base), C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now may the next kernel start launching: it may take TMEM of its own before it waits for this one
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = s_tmem_base, tmem_o = tmem + 2 * kTile;
  volatile int* abort_flag = &s_abort;
  auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, abort_flag, kWaitLimitNs, 1); };

  if (warp == 0) {
    // ---------------- producer: pages and scales of 32 tiles at a time (a tile to a lane), fetched while the 32 before are issued ----------------
    const int tiles = (key_end - key_begin + kTile - 1) / kTile;
    const int subs = t.page_shift >= 6 ? 1 : kTile >> t.page_shift, rows_each = kTile / subs;
    int pg[4];
    uint32_t info[4];
    auto fetch = [&](int i0) {
      const int j0 = key_begin + kTile * (i0 + lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pg[e] = -1; info[e] = 0;
        const int j = j0 + rows_each * e;
        if (e < subs && i0 + lane < tiles && j < key_end) {
          pg[e] = page_of(t, f.x, j >> t.page_shift, head == 0);
          if (pg[e] >= 0)
            info[e] = kThere | (uint32_t)p.ks[(int64_t)pg[e] * t.n_kv_heads + head] | ((uint32_t)p.vs[(int64_t)pg[e] * t.n_kv_heads + head] << 8);
        }
      }
    };
    bool ok = true;
    int it = 0;                                   // tiles issued: a tile is walked once per group of pages whose value scales are alike
    fetch(0);
    for (int i0 = 0; i0 < tiles && ok; i0 += 32) {
      int cp[4];
      uint32_t ci[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) { cp[e] = pg[e]; ci[e] = info[e]; }
      if (i0 + 32 < tiles) fetch(i0 + 32);
      const int n = min(32, tiles - i0);
      for (int i = 0; i < n && ok; ++i) {
        const int j = key_begin + kTile * (i0 + i);
        int p4[4];
        uint32_t f4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e >= subs) { p4[e] = -1; f4[e] = 0; continue; }
          p4[e] = __shfl_sync(0xffffffffu, cp[e], i); f4[e] = __shfl_sync(0xffffffffu, ci[e], i);
        }
        unsigned rem = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) rem |= p4[e] >= 0 ? 1u << e : 0u;
        bool once = true;                         // a tile without any page is walked too: its rows see none of it
        while ((rem || once) && ok) {
          once = false;
          int lead = kNone;
#pragma unroll
          for (int e = 0; e < 4; ++e) if (rem >> e & 1) lead = max(lead, (int)(f4[e] >> 8 & 0xFF) - 127);
          unsigned take = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) take |= (rem >> e & 1) && (int)(f4[e] >> 8 & 0xFF) - 127 >= lead - kSpan ? 1u << e : 0u;
          rem &= ~take;
          const int s = it % kStages;
          if (lane == 0) {
            ok = wait(kempty(s), ((it / kStages) & 1) ^ 1);
            if (ok) {
              Info d;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int src = e / (4 / subs);
                d.w[e] = f4[src] | (take >> src & 1 ? kTaken : 0u);
              }
              d.j0 = j; d.last = i0 + i == tiles - 1 && !rem;
              s_info[it % kInfo] = d;
              int there = 0;
#pragma unroll
              for (int e = 0; e < 4; ++e) there += p4[e] >= 0;
              const int in_page = j & ((1 << t.page_shift) - 1);          // 0 but for pages of 128
              mbar_expect_tx(kfull(s), (uint32_t)(there * rows_each * D));
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (p4[e] >= 0)
                  tma_load_2d(k_at + s * C::kTileBytes + e * rows_each * D, &map_k, kfull(s), 0, ((p4[e] * t.n_kv_heads + head) << t.page_shift) + in_page);
              ok = wait(vempty(s), ((it / kStages) & 1) ^ 1);
              if (ok) {
                mbar_expect_tx(vfull(s), (uint32_t)(there * rows_each * D));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (p4[e] >= 0)
                    tma_load_2d(v_at + s * C::kTileBytes + e * rows_each * D, &map_v, vfull(s), 0, ((p4[e] * t.n_kv_heads + head) << t.page_shift) + in_page);
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          ++it;
        }
      }
    }
    if (!ok && lane == 0) {                       // give copies in flight time to land before shared memory is released
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {}
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer: S of the next tile goes out before O of this one ----------------
    if (lane == 0) {
      const uint32_t fmt = 1u << 4;               // f32 sums, E4M3 x E4M3
      const uint32_t id_s = fmt | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
      const uint32_t id_o = fmt | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);   // V: channels contiguous
      bool ok = wait(qready, 0);
      auto scores = [&](int it) {
        const int s = it % kStages, b = it & 1;
        if (!wait(kfull(s), (it / kStages) & 1) || !wait(sempty(b), ((it >> 1) & 1) ^ 1)) return false;
        tc_fence_after();
        const uint32_t kt = k_at + s * C::kTileBytes;
#pragma unroll
        for (int term = 0; term < 2; ++term) {
          const uint64_t a = make_desc_sw128(q_at + (D == 128 ? term * kRows * 128 : 0)) + (D == 128 ? 0 : term * 4);
          const uint64_t bd = D == 128 ? make_desc_sw128(kt) : make_desc_sw64(kt);
#pragma unroll
          for (int k = 0; k < D / 32; ++k) umma(tmem + b * kTile, a + 2 * k, bd + 2 * k, id_s, (uint32_t)((term | k) != 0));
        }
        tc_commit(kempty(s));
        tc_commit(sfull(b));
        return true;
      };
      ok = ok && scores(0);
      for (int it = 0; ok; ++it) {
        const int last = s_info[it % kInfo].last;   // written before the tile's copies were issued, which scores(it) waited for
        if (!last && !(ok = scores(it + 1))) break;
        const int s = it % kStages;
        if (!wait(vfull(s), (it / kStages) & 1) || !wait(pfull, it & 1)) { ok = false; break; }
        tc_fence_after();
        const uint32_t vt = v_at + s * C::kTileBytes;
#pragma unroll
        for (int k = 0; k < 4; ++k) {               // keys 0..31, 32..63 against hi, then lo
          const uint64_t a = make_desc_sw128(p_at) + 2 * k;
          const uint32_t vk = vt + (k & 1) * 32 * D;
          umma(tmem_o, a, D == 128 ? make_desc_sw128(vk) : make_desc_sw64(vk), id_o, (uint32_t)((it | k) != 0));
        }
        tc_commit(vempty(s));
        tc_commit(pvdone);
        if (last) break;
      }
      if (!ok) {
        tc_commit(drain);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0))
          if (globaltimer_ns() - t0 > 100000000ull) break;
      }
    }
  } else {
    // ---------------- softmax: this thread's row is TMEM lane 32 (warp & 3) + lane ----------------
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const bool live = row < valid;
    const int token = live ? (int)((row0 + row) / p.group) : 0, qhead = head * p.group + (live ? (int)((row0 + row) % p.group) : 0);
    const int pos = live ? r.len - r.n + token : -1;
    float qf;
    {
      const uint4* qp = reinterpret_cast<const uint4*>(p.q + (int64_t)(r.r0 + token) * p.ld_q + (int64_t)qhead * D);
      float amax = 0.0f;
      bool bad = false;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 w = live ? __ldg(qp + c) : make_uint4(0, 0, 0, 0);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = fabsf(__uint_as_float(u[j] << 16)), b = fabsf(__uint_as_float(u[j] & 0xFFFF0000u));
          bad |= !(a < INFINITY) || !(b < INFINITY);
          amax = fmaxf(amax, fmaxf(a, b));
        }
      }
      const uint32_t u = __float_as_uint(amax);
      const int e = max(-119, (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0));
      const float inv = p.scale < 0.0f ? -pow2i(-e) : pow2i(-e);
      qf = bad ? __uint_as_float(0x7FC00000u) : fabsf(p.scale) * pow2i(e);   // a query with an infinity or a NaN: NaN throughout
      uint8_t* const hi_row = smem + row * 128;
#pragma unroll 2
      for (int c = 0; c < D / 16; ++c) {                                     // 16 channels: one 16-byte unit of each term
        uint32_t h4[4], l4[4];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint4 w = live ? __ldg(qp + 2 * c + s) : make_uint4(0, 0, 0, 0);
          const uint32_t uw[4] = {w.x, w.y, w.z, w.w};
          uint16_t h2[4], l2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = __uint_as_float(uw[j] << 16) * inv, y = __uint_as_float(uw[j] & 0xFFFF0000u) * inv;
            const __nv_fp8x2_storage_t hh = __nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
            const float2 b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(hh, __NV_E4M3)));
            h2[j] = hh;
            l2[j] = __nv_cvt_float2_to_fp8x2(make_float2(x - b.x, y - b.y), __NV_SATFINITE, __NV_E4M3);
          }
          h4[2 * s] = pack16(h2[0], h2[1]); h4[2 * s + 1] = pack16(h2[2], h2[3]);
          l4[2 * s] = pack16(l2[0], l2[1]); l4[2 * s + 1] = pack16(l2[2], l2[3]);
        }
        // rows of 128 bytes, 128-byte swizzle; 64 channels: both terms share a row
        *reinterpret_cast<uint4*>(hi_row + ((c ^ (row & 7)) << 4)) = make_uint4(h4[0], h4[1], h4[2], h4[3]);
        if (D == 128) *reinterpret_cast<uint4*>(hi_row + kRows * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(l4[0], l4[1], l4[2], l4[3]);
        else *reinterpret_cast<uint4*>(hi_row + (((c + 4) ^ (row & 7)) << 4)) = make_uint4(l4[0], l4[1], l4[2], l4[3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(qready);
    }

    float m = -INFINITY, l = 0.0f;
    int R = kNone;
    uint8_t* const p_row = smem + (p_at - base) + row * 128;
    bool ok = true;
    int it = 0;
    for (;; ++it) {
      const int b = it & 1;
      if (!wait(sfull(b), (it >> 1) & 1)) { ok = false; break; }
      __syncwarp();
      tc_fence_after();
      const Info d = s_info[it % kInfo];
      uint32_t sr[64];
      tmem_ld32(tmem + b * kTile + lanes, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
      tmem_ld32(tmem + b * kTile + 32 + lanes, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sempty(b));

      const bool whole = (d.w[0] & d.w[1] & d.w[2] & d.w[3]) >> 31 && d.j0 + kTile <= key_end;   // every key is there
      // and every row sees every key, under one pair of scales
      const bool clear = whole && d.w[0] == d.w[1] && d.w[0] == d.w[2] && d.w[0] == d.w[3] && d.w[0] & kTaken && d.j0 + kTile - 1 <= first_pos &&
                         (p.window <= 0 || d.j0 > last_pos - p.window);
      int lead = kNone;
#pragma unroll
      for (int g = 0; g < 4; ++g) if (d.w[g] & kTaken) lead = max(lead, (int)(d.w[g] >> 8 & 0xFF) - 127);
      const int was = R == kNone ? lead : R;
      R = lead == kNone ? R : lead > was || lead < was - kSpan ? lead : was;
      float mt = -INFINITY;
      if (clear) {
        const float fs = qf * pow2_byte(d.w[0] & 0xFF);                        // not negative: the sign of the scale is in the query
#pragma unroll
        for (int j = 0; j < 64; ++j) mt = fmaxf(mt, __uint_as_float(sr[j]));
        mt *= fs;
      } else {
#pragma unroll
        for (int j = 0; j < 64; ++j) {
          const int key = d.j0 + j;
          const bool see = key <= pos && (p.window <= 0 || key > pos - p.window) && d.w[j >> 4] & kTaken;
          const float v = see ? __uint_as_float(sr[j]) * (qf * pow2_byte(d.w[j >> 4] & 0xFF)) : -INFINITY;
          sr[j] = __float_as_uint(v);
          mt = fmaxf(mt, v);
        }
      }
      float alpha = 1.0f;
      if (mt > m + kSlack || (m == -INFINITY && mt > -INFINITY)) { alpha = ex2(m - mt); m = mt; }
      l *= alpha;
      const float back = m == -INFINITY ? 0.0f : m;
      uint16_t hi[32], lo[32];
      if (clear) {
        const int lv = (int)(d.w[0] >> 8 & 0xFF) - 127;
        const float fs = qf * pow2_byte(d.w[0] & 0xFF), add = (float)(8 + lv - R) - back;
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 64; j += 2) {
          const float x = ex2(fmaf(__uint_as_float(sr[j]), fs, add)), y = ex2(fmaf(__uint_as_float(sr[j + 1]), fs, add));
          sum[(j >> 1) & 3] += x + y;
          split_f16(pack_f16(x, y), hi[j >> 1], lo[j >> 1]);
        }
        l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), pow2i(R - lv - 8), l);   // the sum is of the weights without the values' scale
      } else {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int lv = (int)(d.w[g] >> 8 & 0xFF) - 127;
          const float up = d.w[g] & kTaken ? pow2i(8 + lv - R) : 0.0f;
#pragma unroll
          for (int j = 16 * g; j < 16 * g + 16; j += 2) {
            const float x = ex2(__uint_as_float(sr[j]) - back), y = ex2(__uint_as_float(sr[j + 1]) - back);
            l += x + y;
            split_f16(pack_f16(x * up, y * up), hi[j >> 1], lo[j >> 1]);
          }
        }
      }
      if (it > 0 && !wait(pvdone, (it - 1) & 1)) { ok = false; break; }         // P has been read, O is up to date
      __syncwarp();
      tc_fence_after();
      alpha *= R == kNone ? 1.0f : pow2i(was - R);
      if (it > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o + c + lanes, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
          tmem_st32(tmem_o + c + lanes, o);
        }
        tmem_st_wait();
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        *reinterpret_cast<uint4*>(p_row + ((u ^ (row & 7)) << 4)) =
            make_uint4(pack16(hi[8 * u], hi[8 * u + 1]), pack16(hi[8 * u + 2], hi[8 * u + 3]), pack16(hi[8 * u + 4], hi[8 * u + 5]), pack16(hi[8 * u + 6], hi[8 * u + 7]));
        *reinterpret_cast<uint4*>(p_row + (((u + 4) ^ (row & 7)) << 4)) =
            make_uint4(pack16(lo[8 * u], lo[8 * u + 1]), pack16(lo[8 * u + 2], lo[8 * u + 3]), pack16(lo[8 * u + 4], lo[8 * u + 5]), pack16(lo[8 * u + 6], lo[8 * u + 7]));
      }
      if (!whole) {                                // value rows without a visible key: whatever they hold becomes 0
        const int s = it % kStages;
        if (!wait(vfull(s), (it / kStages) & 1)) { ok = false; break; }
        __syncwarp();
        // two threads to a row of D bytes (a whole row: the order of its 16-byte units does not matter, but 64-byte rows share a line)
        const int key = row >> 1;
        if (!(d.w[key >> 4] & kThere) || d.j0 + key >= key_end) {
          uint8_t* const vrow = smem + (v_at - base) + s * C::kTileBytes + key * D + (row & 1) * (D / 2);
#pragma unroll
          for (int u = 0; u < D / 32; ++u) *reinterpret_cast<uint4*>(vrow + 16 * u) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull);
      if (d.last) break;
    }
    if (ok) ok = wait(pvdone, it & 1);
    if (ok) {
      __syncwarp();
      tc_fence_after();
      const int64_t orow = (int64_t)(r.r0 + token) * (t.n_kv_heads * p.group) + qhead;
      // a row that sees no key has l = 0: zeros and -inf.  A query that holds an infinity or a NaN has l = NaN and stays NaN.
      const float inv = l == 0.0f ? 0.0f : __frcp_rn(l), up = R == kNone ? 0.0f : pow2i(R - 8);
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld32(tmem_o + c + lanes, o);
        tmem_ld_wait();
        if (live) {
          uint4* const y = reinterpret_cast<uint4*>(p.out + orow * D + c);
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * i]) * inv * up, __uint_as_float(o[j + 2 * i + 1]) * inv * up);
              w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            y[j / 8] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (live && p.lse) p.lse[orow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
  if (threadIdx.x == 0 && s_abort) report(t.status, B2Q_ERR_TIMEOUT);
}

template <int D>
int32_t launch(b2q_handle h, const AttendArgs& p) {
  using C = Cfg<D>;
  CUtensorMap map_k, map_v;
  const uint64_t rows = (uint64_t)p.t.num_pages * p.t.n_kv_heads << p.t.page_shift;
  const uint32_t box = p.t.page_shift < 6 ? 1 << p.t.page_shift : kTile;
  int32_t st = D == 128 ? b2q_tensor_map_2d(h, &map_k, p.k, 1, D, rows, D, box) : b2q_tensor_map_2d_sw64(h, &map_k, p.k, D, rows, box);
  if (st != B2Q_OK) return st;
  st = D == 128 ? b2q_tensor_map_2d(h, &map_v, p.v, 1, D, rows, D, box) : b2q_tensor_map_2d_sw64(h, &map_v, p.v, D, rows, box);
  if (st != B2Q_OK) return st;
  const int64_t units = (int64_t)p.t.tokens * p.group / kRows + p.t.seqs;
  if (units > 0x7FFFFFFF) B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_attention: too many rows");
  B2Q_SMEM_ATTR(h, kv8_prefill_kernel<D>, C::kSmem);
  B2Q_CUDA(h, b2q_pdl_launch(h->sw.chain_pdl != 0, kv8_prefill_kernel<D>, dim3((unsigned)units, (unsigned)p.t.n_kv_heads), dim3(kThreads), C::kSmem, h->stream,
                             map_k, map_v, p));
  return B2Q_OK;
}

}  // namespace pre
}  // namespace kv8

// The caller has checked the arguments; q_starts is not null.
int32_t b2q_kv8_prefill(b2q_handle h, const kv8::AttendArgs& p, int64_t head_dim) {
  return head_dim == 64 ? kv8::pre::launch<64>(h, p) : kv8::pre::launch<128>(h, p);
}

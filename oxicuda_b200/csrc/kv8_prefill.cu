// Attention of many query rows over the paged 8-bit cache (layout: kv8.cuh), on tcgen05:
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  keys j <= pos_i, with a window also j > pos_i - window.
// A CTA takes 128 rows ((new token, query head) pairs of one sequence and kv head) and walks the keys 64 at a time:
//   S [128 x 64] = Q K^T,   P = exp2(S - m),   O [128 x D] += P V,   S (two of them) and O in TMEM, f32.
// Q K^T multiplies the key codes as they are stored (kind::f8f6f4, straight from TMA): Q enters as two E4M3 terms, the rounding of q and
// the rounding of what that leaves.  A bf16 has 8 significant bits and an E4M3 code 4, so q / 2^e (2^e brings the row's largest element
// into (224, 448]) is exact but for elements below 2^-9 of the largest, which keep an absolute error of 2^-10 (2^-17 of it); two FP8 products
// cost what one bf16 product costs, and the split is made once per row.
// P V multiplies in f16 (kind::f16): two warps turn each value tile into f16 (exact, one conversion for 128 rows of P, where
// splitting P into E4M3 terms costs every row four instructions per pair of weights), P goes back into the TMEM columns of its S as the
// A operand.  A weight is held as p * 2^x, x from 0 to 8 (6 for most pages), and is off by 2^-11 of itself, or by 2^-25 of the row's largest (2^-31).
// Work per 64 keys and CTA: 640 clocks of tensor core (Q K^T at N = 64 reads 1.5 x the shared memory that its rate allows, P V at N = D
// runs at rate), 512 of exponentials and 120 KB of shared memory traffic (48 for Q K^T, 16 for P V, 40 to convert the values, 16 to bring the
// tiles in), 940 clocks: two CTAs share an SM, so that one multiplies while the other exponentiates.
// Measured in a graph of eight: 2 x 3900 tokens behind 150 (32 heads of 128 channels over 8 kv heads) 277 us, 780 TFLOP/s (a call among others 308;
// pages of 16 292 to 319); 1 x 8000 tokens 522 us, 1000 TFLOP/s, where a tile takes about 1100 clocks.  Leaving out the exponentials changes nothing there, leaving out the conversion of the values saves 6 %,
// three quarters of Q K^T 10 %: shared memory bounds it, with the products' latency on top in short rows.
// The running maximum is followed lazily: it moves only when a score exceeds it by more than 2^kSlack (f16 has the range), so O is rescaled
// (a round trip through registers) once or twice per row and not per tile.  The value scale of a page is a power of two 2^lv: weights
// enter as p * 2^(8 + lv - R) and O is in units of 2^(R - 8), R following the pages (next_unit in kv8.cuh); a tile whose pages differ by more
// than 2^(kSpan - kRoom) is walked once per group of alike pages, the others masked.
// Few row tiles: `split` CTAs of a cluster take every split'th key tile of the same rows and are joined through distributed shared memory.
// Warps 1 to 7 turn the query rows into E4M3 terms; then warp 0 walks the block table, issues the copies and describes each tile to the others,
// warp 1 issues the products, warps 2 and 3 convert values, warps 4 to 7 are the softmax (a thread to a row).
// Keys behind the last visible one are masked and their value rows become zeros in the conversion; a page that the table does not
// name is neither read nor counted.  Every mbarrier wait is bounded; on expiry the kernel records B2Q_ERR_TIMEOUT and leaves.
#include "kv8.cuh"
#include "tc_common.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace kv8 {

using namespace tcx;

namespace pre {

constexpr int kRows = 128, kTile = 64;
constexpr int kThreads = 256;
constexpr int kRegsFirst = 80, kRegsSoft = 176;  // of 128 a thread at launch: 128 * 80 + 128 * 176 = 256 * 128
constexpr int kKStages = 3, kVStages = 2, kInfo = 8;   // tiles in flight; tile descriptions (a tile is read at most 5 behind the newest)
constexpr int kRoom = 2;                         // R is set that far above a scale, so that pages a little larger do not move it again
constexpr float kSlack = 6.0f;                   // 2^(8 + 6) is well inside f16
constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr int kGridY = 32768;                    // row tiles: blockIdx.y, and z beyond that

template <int D> struct Cfg {
  static constexpr int kQ = 2 * kRows * D;       // both terms
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kV16 = 2 * kTileBytes;    // a value tile in f16: D / 64 blocks of 64 keys x 128 bytes
  static constexpr int kData = kQ + (kKStages + kVStages) * kTileBytes + 2 * kV16;
  static constexpr int kSmem = kData + 1024 + kInfo * 80 + 256;
  static constexpr int kTmemCols = 256;          // S: 2 x 64, O: D
  static_assert(kRows * D * 4 <= kData, "the join reuses the tiles");
};
constexpr uint32_t kThere = 0x80000000u, kTaken = 0x40000000u;

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// A in TMEM: two f16 to a column, a row to a lane
__device__ __forceinline__ void umma_f16_ta(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// four E4M3 codes -> two registers of two f16
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
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

__device__ __forceinline__ uint32_t cluster_id_x() { uint32_t r; asm("mov.u32 %0, %clusterid.x;" : "=r"(r)); return r; }

constexpr uint64_t kOne2 = 0x3F8000003F800000ull;   // 1.0f twice
__device__ __forceinline__ uint64_t dup(float x) { return (uint64_t)__float_as_uint(x) << 32 | __float_as_uint(x); }

// A tile, as the producer describes it to the others; per 16 keys and of the tile.  R follows the pages' value scales 2^lv: weights enter
// as p * 2^up, a sum of them counts 2^down, O is in units of 2^(R - 8) and moves by the factor `move` to this tile's.
struct __align__(16) Info {
  uint32_t flags[4];
  float kf[4], up[4], down[4];                   // the keys' scale, 8 + lv - R, 2^(R - lv - 8)
  int j0, last, R;                               // first key; 1 for the last tile
  float move;
};
// three at a time
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// what the last tmem_ld32 into r waits for, and no use of r before it
__device__ __forceinline__ void landed(uint32_t (&r)[64]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 64; i += 8)
    asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// SUBS: pages that a tile of keys spans (1: pages of 64 and 128), known at compile time: the producer is on the critical path, and its share of a tile
// is then shorter (2 x 3900 tokens 289 us, with the general loop 308)
template <int D, int SUBS>
__global__ void __launch_bounds__(kThreads, 2)
kv8_prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttendArgs p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_at = base, k_at = base + C::kQ, v_at = k_at + kKStages * C::kTileBytes, w_at = v_at + kVStages * C::kTileBytes, bar_at = base + C::kData;
  auto kfull = [&](int s) { return bar_at + 8u * s; };
  auto kempty = [&](int s) { return bar_at + 8u * (kKStages + s); };
  auto vfull = [&](int s) { return bar_at + 8u * (2 * kKStages + s); };
  auto vempty = [&](int s) { return bar_at + 8u * (2 * kKStages + kVStages + s); };
  const uint32_t more = bar_at + 8u * (2 * kKStages + 2 * kVStages);
  auto wfull = [&](int b) { return more + 8u * b; };          // f16 value tiles
  auto wempty = [&](int b) { return more + 8u * (2 + b); };
  auto sfull = [&](int b) { return more + 8u * (4 + b); };
  auto pfull = [&](int b) { return more + 8u * (6 + b); };    // the softmax may be a tile ahead of the products: a barrier for each S
  const uint32_t qready = more + 64, pvdone = more + 72, drain = more + 80, odone = more + 88;
  Info* const s_info = reinterpret_cast<Info*>(smem + (bar_at - base) + 8 * (2 * kKStages + 2 * kVStages + 12));   // 22 barriers in front
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;
  __shared__ float s_m[kRows], s_l[kRows];        // score factors of the rows; for the join this CTA's maxima, sums and units
  __shared__ int s_r[kRows];

  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < kKStages; ++s) { mbar_init(kfull(s), 1); mbar_init(kempty(s), 1); }
    for (int s = 0; s < kVStages; ++s) { mbar_init(vfull(s), 1); mbar_init(vempty(s), 2); }
    for (int b = 0; b < 2; ++b) { mbar_init(wfull(b), 2); mbar_init(wempty(b), 1); mbar_init(sfull(b), 1); }
    mbar_init(qready, 7); mbar_init(pfull(0), 4); mbar_init(pfull(1), 4); mbar_init(pvdone, 1); mbar_init(drain, 1); mbar_init(odone, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- which rows: the longest tiles of a sequence first, for all heads ----
  const Batch& t = p.t;
  const int head = (int)cluster_id_x(), unit = (int)(blockIdx.y + kGridY * blockIdx.z);
  const bool tell = head == 0 && part == 0 && warp == 0;
  if (unit == 0 && tell) for (int b = lane; b < t.seqs; b += 32) rows_of(t, b, true);
  const Found f = find_unit(t.seqs, unit, [&](int b) { return (rows_of(t, b, false).n * p.group + kRows - 1) / kRows; });
  if (f.b < 0) return;                            // the whole cluster leaves, before it holds TMEM
  const Rows r = rows_of(t, f.b, false);          // rows of all sequences fit 31 bits
  const int row0 = (f.count - 1 - f.index) * kRows, valid = min(kRows, r.n * p.group - row0);
  const int token0 = row0 / p.group, head0 = row0 - token0 * p.group;        // of the tile's first row, within the sequence and the group
  const int first_pos = r.len - r.n + token0, last_pos = first_pos + div_group(p, head0 + valid - 1);
  const int key_end = last_pos + 1;
  // the first key that a row sees; the first tile may begin before it, with pages that its owner has given up and that are not looked up
  const int key_low = p.window > 0 ? max(0, first_pos - p.window + 1) : 0, key_begin = key_low & ~(kTile - 1);
  const int all = (key_end - key_begin + kTile - 1) / kTile;
  int tiles = (all - part + split - 1) / split;   // tiles part, part + split, ..

  // ---------------- the query rows, by warps 1 .. 7: D / 16 lanes to a row, 16 channels (16 bytes of codes) each ----------------
  // They come in through the space of the f16 value tiles (free until the first of those is made), and a short loop turns them: five turns
  // unrolled cost every CTA more in instruction fetches than they saved (340 against 352 us at the time for 2 x 3900 tokens).
  constexpr int LPR = D / 16, RPW = 32 / LPR, QI = (kRows / RPW + 6) / 7;     // lanes to a row, rows at once, turns of a warp
  static_assert(QI * RPW <= 32, "a lane holds the address of each row");
  const int qc = lane % LPR;
  uint8_t* const raw = smem + (w_at - base);
  auto qrow_of = [&](int i, int j) { return RPW * (warp - 1 + 7 * i) + j; };  // row j of turn i
  if (warp > 0) {
    const int mine = qrow_of(lane / RPW, lane % RPW);
    const int hr = head0 + (mine < valid ? mine : 0), tk = div_group(p, hr);   // rows behind the last one: the first row's
    const __nv_bfloat16* const at = p.q + (int64_t)(r.r0 + token0 + tk) * p.ld_q + (int64_t)(head * p.group + hr - tk * p.group) * D;
#pragma unroll 1
    for (int i = 0; i < QI; ++i) {
      const int rr = qrow_of(i, lane / LPR);
      const unsigned long long from = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(at), i * RPW + lane / LPR) + 32 * qc;
      const uint32_t to = smem_u32(raw + rr * (2 * D) + 32 * qc);
      if (rr < kRows) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16), "l"(from + 16) : "memory");
      }
    }
  }

  if (warp == 1) tmem_alloc(smem_u32(&s_tmem_base), C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now may the next kernel start launching: it may take TMEM of its own before it waits for this one
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem_base, 0), tmem_o = tmem + 2 * kTile;
  volatile int* abort_flag = &s_abort;
  // by whole warps, which leave together if one lane gives up
  auto wait = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, kWaitLimitNs, 1)); };

  if (warp > 0) {
    const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < QI; ++i) {
      const int rr = qrow_of(i, lane / LPR);
      const uint4* const from = reinterpret_cast<const uint4*>(raw + min(rr, kRows - 1) * (2 * D) + 32 * qc);
      const uint4 w[2] = {from[0], from[1]};
      const __nv_bfloat162* const q2 = reinterpret_cast<const __nv_bfloat162*>(w);
      // the largest of the row, a NaN if it holds one
      __nv_bfloat162 top = __habs2(q2[0]);
#pragma unroll
      for (int j = 1; j < 8; ++j) top = __hmax2_nan(top, __habs2(q2[j]));
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) top = __hmax2_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float amax = __bfloat162float(__hmax_nan(top.x, top.y));
      const uint32_t u = __float_as_uint(amax);
      const int e = max(-119, (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0));
      const float inv = sign * pow2i(-e);
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {                                            // exact in f16 down to 2^-24
        uint16_t ha, la, hb, lb;
        const float2 x = __bfloat1622float2(q2[2 * j]), y = __bfloat1622float2(q2[2 * j + 1]);
        split_f16(pack_f16(x.x * inv, x.y * inv), ha, la);
        split_f16(pack_f16(y.x * inv, y.y * inv), hb, lb);
        h[j] = pack16(ha, hb);
        l[j] = pack16(la, lb);
      }
      if (rr < kRows) {
        // rows of 128 bytes, 128-byte swizzle; 64 channels: both terms share a row
        uint8_t* const qrow = smem + rr * 128;
        *reinterpret_cast<uint4*>(qrow + ((qc ^ (rr & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(qrow + (D == 128 ? kRows * 128 + ((qc ^ (rr & 7)) << 4) : ((qc + 4) ^ (rr & 7)) << 4)) = make_uint4(l[0], l[1], l[2], l[3]);
        // a query with an infinity or a NaN: NaN throughout
        if (qc == 0) s_m[rr] = amax < INFINITY ? fabsf(p.scale) * pow2i(e) : __uint_as_float(0x7FC00000u);
      }
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(qready);
  }

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFirst));
    if (tiles == 0) {
      // a CTA of the cluster beyond the last tile: it only joins
    } else if (warp == 0) {
      // ---------------- producer: pages and scales of 32 tiles at a time (a tile to a lane), fetched while the 32 before are issued ----------------
      constexpr int rows_each = kTile / SUBS;
      int pg[SUBS];
      uint32_t info[SUBS];
      auto fetch = [&](int i0) {
        const int j0 = key_begin + kTile * (part + split * (i0 + lane));
#pragma unroll
        for (int e = 0; e < SUBS; ++e) {
          pg[e] = -1; info[e] = 0;
          const int j = j0 + rows_each * e;
          if (i0 + lane < tiles && j < key_end && (j | (rows_each - 1)) >= key_low) {
            pg[e] = page_of(t, f.b, j >> t.page_shift, head == 0);
            if (pg[e] >= 0)
              info[e] = kThere | (uint32_t)p.ks[(int64_t)pg[e] * t.n_kv_heads + head] | ((uint32_t)p.vs[(int64_t)pg[e] * t.n_kv_heads + head] << 8);
          }
        }
      };
      bool ok = true;
      int R = kNone, top = kNone, it = 0;           // it: tiles issued: a tile is walked once per group of pages whose value scales are alike
      fetch(0);
      for (int i0 = 0; i0 < tiles && ok; i0 += 32) {
        int cp[SUBS];
        uint32_t ci[SUBS];
#pragma unroll
        for (int e = 0; e < SUBS; ++e) { cp[e] = pg[e]; ci[e] = info[e]; }
        if (i0 + 32 < tiles) fetch(i0 + 32);
        const int n = min(32, tiles - i0);
        for (int i = 0; i < n && ok; ++i) {
          const int j = key_begin + kTile * (part + split * (i0 + i)), in_page = j & ((1 << t.page_shift) - 1);   // in_page: 0 but for pages of 128
          int line[SUBS], there = 0;                // first row of the page in the map, or -1
          uint32_t fl[SUBS];
          unsigned rem = 0;
#pragma unroll
          for (int e = 0; e < SUBS; ++e) {
            const int pe = __shfl_sync(0xffffffffu, cp[e], i);
            fl[e] = __shfl_sync(0xffffffffu, ci[e], i);
            line[e] = pe >= 0 ? ((pe * t.n_kv_heads + head) << t.page_shift) + in_page : -1;
            there += pe >= 0;
            rem |= pe >= 0 ? 1u << e : 0u;
          }
          bool once = true;                         // a tile without any page is walked too: its rows see none of it
          while ((rem || once) && ok) {
            once = false;
            int lead = kNone, least = 1000;
            unsigned take = 0;
#pragma unroll
            for (int e = 0; e < SUBS; ++e) if (rem >> e & 1) lead = max(lead, (int)(fl[e] >> 8 & 0xFF) - 127);
#pragma unroll
            for (int e = 0; e < SUBS; ++e) {
              const int lv = (int)(fl[e] >> 8 & 0xFF) - 127;
              if ((rem >> e & 1) && lv >= lead + kRoom - kSpan) { take |= 1u << e; least = min(least, lv); }
            }
            rem &= ~take;
            const float move = lead == kNone ? 1.0f : next_unit(R, top, lead, least, kRoom);
            float kf[SUBS], up[SUBS], down[SUBS];
            uint32_t flag[SUBS];
#pragma unroll
            for (int e = 0; e < SUBS; ++e) {
              const int lv = (int)(fl[e] >> 8 & 0xFF) - 127;
              flag[e] = (fl[e] & kThere) | (take >> e & 1 ? kTaken : 0u);
              kf[e] = pow2_byte(fl[e] & 0xFF);
              const int x = max(8 + lv - R, kLeast);
              up[e] = (float)x;
              down[e] = pow2i(-x);
            }
            constexpr int A2 = SUBS == 4 ? 1 : 0, C2 = SUBS / 2, D2 = SUBS - 1;   // the pages of keys 16 .. 31, 32 .. 47, 48 .. 63
            const int s = it % kKStages, v = it % kVStages;
            ok = wait(kempty(s), ((it / kKStages) & 1) ^ 1);
            if (!ok) break;
            if (elect_one()) {
              Info* const d = &s_info[it % kInfo];
              *reinterpret_cast<uint4*>(d->flags) = make_uint4(flag[0], flag[A2], flag[C2], flag[D2]);
              *reinterpret_cast<float4*>(d->kf) = make_float4(kf[0], kf[A2], kf[C2], kf[D2]);
              *reinterpret_cast<float4*>(d->up) = make_float4(up[0], up[A2], up[C2], up[D2]);
              *reinterpret_cast<float4*>(d->down) = make_float4(down[0], down[A2], down[C2], down[D2]);
              *reinterpret_cast<int4*>(&d->j0) = make_int4(j, i0 + i == tiles - 1 && !rem, R, __float_as_int(move));
              mbar_expect_tx(kfull(s), (uint32_t)(there * rows_each * D));
#pragma unroll
              for (int e = 0; e < SUBS; ++e)
                if (line[e] >= 0) tma_load_2d(k_at + s * C::kTileBytes + e * rows_each * D, &map_k, kfull(s), 0, line[e]);
            }
            __syncwarp();
            ok = wait(vempty(v), ((it / kVStages) & 1) ^ 1);
            if (!ok) break;
            if (elect_one()) {
              mbar_expect_tx(vfull(v), (uint32_t)(there * rows_each * D));
#pragma unroll
              for (int e = 0; e < SUBS; ++e)
                if (line[e] >= 0) tma_load_2d(v_at + v * C::kTileBytes + e * rows_each * D, &map_v, vfull(v), 0, line[e]);
            }
            __syncwarp();
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
      // The warp stays together and elects a lane for each group of products: descriptors then live in uniform registers.  One lane alone
      // in its branch moved each operand there, product by product: 320 against 304 us at the time for 2 x 3900 tokens.
      const uint32_t id_s = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);                // E4M3 x E4M3, f32 sums
      const uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);      // f16 x f16; V: channels contiguous
      bool ok = wait(qready, 0);
      auto scores = [&](int it) {
        const int s = it % kKStages, b = it & 1;
        if (!wait(kfull(s), (it / kKStages) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t kt = k_at + s * C::kTileBytes;
#pragma unroll
          for (int term = 0; term < 2; ++term) {
            const uint64_t a = make_desc_sw128(q_at + (D == 128 ? term * kRows * 128 : 0)) + (D == 128 ? 0 : term * 4);
            const uint64_t bd = D == 128 ? make_desc_sw128(kt) : make_desc_sw64(kt);
#pragma unroll
            for (int k = 0; k < D / 32; ++k) umma_f8(tmem + b * kTile, a + 2 * k, bd + 2 * k, id_s, (uint32_t)((term | k) != 0));
          }
          tc_commit(kempty(s));
          tc_commit(sfull(b));
        }
        __syncwarp();
        return true;
      };
      ok = ok && scores(0);
      for (int it = 0; ok; ++it) {
        const int last = __shfl_sync(0xffffffffu, s_info[it % kInfo].last, 0);   // written before the tile's copies were issued, which scores(it) waited for
        // S of tile it + 1 overwrites S and P of tile it - 1: their product has to be done
        if (!last && !(ok = (it == 0 || wait(pvdone, (it - 1) & 1)) && scores(it + 1))) break;
        const int b = it & 1;
        if (!wait(wfull(b), (it >> 1) & 1) || !wait(pfull(b), (it >> 1) & 1)) { ok = false; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t vt = w_at + b * C::kV16;
          // 16 keys a step: two groups of 8 rows of 128 bytes; blocks of 64 channels lie 64 rows apart (leading byte offset)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t bd = (make_desc_sw128(vt + k * 2048) & ~(0x3FFFull << 16)) | ((uint64_t)(kTile * 128 >> 4) << 16);
            umma_f16_ta(tmem_o, tmem + b * kTile + 8 * k, bd, id_o, (uint32_t)((it | k) != 0));
          }
          tc_commit(wempty(b));
          tc_commit(pvdone);
          if (last) tc_commit(odone);
        }
        __syncwarp();
        if (last) break;
      }
      if (!ok && elect_one()) {
        tc_commit(drain);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0))
          if (globaltimer_ns() - t0 > 100000000ull) break;
      }
      __syncwarp();
    } else {
      // ---------------- values to f16, 64 threads: 16 channels of a key at a time ----------------
      // a thread keeps its unit u of 16 channels and its key modulo KEYS (a multiple of 8), so the swizzles are fixed
      constexpr int UNITS = D / 16, KEYS = 64 / UNITS;
      const int th = (int)threadIdx.x - 64, u = th % UNITS, key0 = th / UNITS, u2 = 2 * (u & 3);
      // the threads of the upper channels write their second 16 bytes first: eight threads then meet no bank twice
      const bool swap = u >= 4;
      const int src0 = key0 * D + ((D == 128 ? u ^ (key0 & 7) : u ^ ((key0 >> 1) & 3)) << 4);              // as TMA left it
      const int dst0 = (u >> 2) * (kTile * 128) + key0 * 128 + (((u2 + swap) ^ (key0 & 7)) << 4);          // block u / 4, units 2 (u & 3) and the next
      const int step = (((u2 + !swap) ^ (key0 & 7)) - ((u2 + swap) ^ (key0 & 7))) * 16;
      const bool free_now = wait(qready, 0);        // the query rows have passed through the tiles that are written here
      for (int it = 0; free_now; ++it) {
        const int v = it % kVStages, b = it & 1;
        if (!wait(vfull(v), (it / kVStages) & 1) || !wait(wempty(b), ((it >> 1) & 1) ^ 1)) break;
        const Info& d = s_info[it % kInfo];
        const uint32_t flags[4] = {d.flags[0], d.flags[1], d.flags[2], d.flags[3]};
        const int j0 = d.j0, last = d.last;
        const uint8_t* const src = smem + (v_at - base) + v * C::kTileBytes + src0;
        uint8_t* const dst = smem + (w_at - base) + b * C::kV16 + dst0;
        const bool whole = (flags[0] & flags[1] & flags[2] & flags[3]) >> 31 && j0 + kTile <= key_end;
#pragma unroll
        for (int k = 0; k < kTile; k += KEYS) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + k * D);
          uint32_t o[8];
          to_f16(swap ? x.z : x.x, o[0], o[1]); to_f16(swap ? x.w : x.y, o[2], o[3]);
          to_f16(swap ? x.x : x.z, o[4], o[5]); to_f16(swap ? x.y : x.w, o[6], o[7]);
          if (!whole && (!(d.flags[(key0 + k) >> 4] & kThere) || j0 + key0 + k >= key_end))   // no visible key here: whatever the row holds becomes 0
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = 0;
          *reinterpret_cast<uint4*>(dst + k * 128) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(dst + k * 128 + step) = make_uint4(o[4], o[5], o[6], o[7]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) { mbar_arrive(vempty(v)); mbar_arrive(wfull(b)); }
        if (last) break;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoft));
    // ---------------- softmax: this thread's row is TMEM lane 32 (warp & 3) + lane ----------------
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const bool live = row < valid;
    const int tk = live ? div_group(p, head0 + row) : 0, token = live ? token0 + tk : 0, qhead = head * p.group + (live ? head0 + row - tk * p.group : 0);
    const int pos = live ? r.len - r.n + token : -1;
    if (!wait(qready, 0)) tiles = -1;               // only if another warp has given up
    const float qf = s_m[row];

    float m = -INFINITY, l = 0.0f;
    int R = kNone;
    bool ok = tiles >= 0;
    for (int it = 0; ok && tiles > 0; ++it) {
      const int b = it & 1;
      const Info* const d = &s_info[it % kInfo];
      if (!wait(sfull(b), (it >> 1) & 1)) { ok = false; break; }
      tc_fence_after();
      uint32_t sr[64];
      tmem_ld32(tmem + b * kTile + lanes, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
      tmem_ld32(tmem + b * kTile + 32 + lanes, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
      float fs[4], mt = -INFINITY;
      const float4 kf = *reinterpret_cast<const float4*>(d->kf), up = *reinterpret_cast<const float4*>(d->up), down = *reinterpret_cast<const float4*>(d->down);
      const int4 rest = *reinterpret_cast<const int4*>(&d->j0);
      // not negative: the sign of the scale is in the query; not zero: -inf * 0 would be a NaN
      fs[0] = qf * kf.x; fs[1] = qf * kf.y; fs[2] = qf * kf.z; fs[3] = qf * kf.w;
      // clear: every row sees every key (tile edges, windows and tiles walked in parts are masked)
      const uint32_t both = d->flags[0] & d->flags[1] & d->flags[2] & d->flags[3];
      const bool clear = (both & (kThere | kTaken)) == (kThere | kTaken) && rest.x + kTile - 1 <= first_pos && (p.window <= 0 || rest.x > last_pos - p.window);
      landed(sr);
      // Masking rewrites S in TMEM, 16 columns at a time in a loop that stays rolled, and loads it again: it runs once or twice per CTA, and as
      // straight code between the load and its use it made the kernel slower by its instruction fetches.
      if (!clear) {
        const int top = pos - rest.x, low = p.window > 0 ? top - p.window : -1;      // columns low < j <= top
#pragma unroll 1
        for (int c = 0; c < kTile; c += 16) {
          uint32_t x[16];
          tmem_ld16(tmem + b * kTile + c + lanes, x);
          tmem_ld_wait();
          const int t2 = (d->flags[c >> 4] & kTaken ? top : -1) - c, l2 = low - c;
#pragma unroll
          for (int j = 0; j < 16; ++j) if (j > t2 || j <= l2) x[j] = 0xFF800000u;
          tmem_st16(tmem + b * kTile + c + lanes, x);
        }
        tmem_st_wait();
        tmem_ld32(tmem + b * kTile + lanes, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
        tmem_ld32(tmem + b * kTile + 32 + lanes, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
        landed(sr);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        fs[g] = fs[g] == 0.0f ? 1.17549435e-38f : fs[g];
        float x[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t* const y = sr + 16 * g + 8 * k;
          x[k] = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
          x[k] = max3(x[k], __uint_as_float(y[3]), __uint_as_float(y[4]));
          x[k] = max3(x[k], __uint_as_float(y[5]), __uint_as_float(y[6]));
          x[k] = fmaxf(x[k], __uint_as_float(y[7]));
        }
        mt = fmaxf(mt, fmaxf(x[0], x[1]) * fs[g]);
      }
      float alpha = 1.0f;
      if (mt > m + kSlack || (m == -INFINITY && mt > -INFINITY)) { alpha = ex2(m - mt); m = mt; }
      l *= alpha;
      const float back = m == -INFINITY ? 0.0f : m;   // a row that has seen nothing yet: exp2(-inf - 0) = 0
      uint32_t pw[32];
      const float ups[4] = {up.x, up.y, up.z, up.w}, downs[4] = {down.x, down.y, down.z, down.w};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint64_t f2 = dup(fs[g]), add2 = dup(ups[g] - back);
        uint64_t sum = 0;
#pragma unroll
        for (int j = 16 * g; j < 16 * g + 16; j += 2) {
          uint64_t e = add2;
          fma2(e, (uint64_t)sr[j + 1] << 32 | sr[j], f2);
          const float x = ex2(__uint_as_float((uint32_t)e)), y = ex2(__uint_as_float((uint32_t)(e >> 32)));
          fma2(sum, (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), kOne2);
          pw[j >> 1] = pack_f16(x, y);
        }
        l = fmaf(__uint_as_float((uint32_t)sum) + __uint_as_float((uint32_t)(sum >> 32)), downs[g], l);   // the weights without the values' scale
      }
      tmem_st32(tmem + b * kTile + lanes, pw);       // over the S that this warp has just read
      alpha *= __int_as_float(rest.w);
      R = rest.z;
      // Where the unit of O moves, O of the tile in front has to be done.  (S of this tile came after O of tile it - 2: the parity can only be
      // that of it - 2 or it - 1.)
      if (it > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
        if (!wait(pvdone, (it - 1) & 1)) { ok = false; break; }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(tmem_o + c + lanes, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
          tmem_st32(tmem_o + c + lanes, o);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull(b));
      if (rest.y) break;
    }
    if (ok && tiles > 0) ok = wait(odone, 0);
    __syncwarp();
    tc_fence_after();
    // a row that sees no key has l = 0: zeros and -inf.  A query that holds an infinity or a NaN has l = NaN and stays NaN.
    if (split == 1) {
      const int64_t orow = (int64_t)(r.r0 + token) * (t.n_kv_heads * p.group) + qhead;
      const float inv = (l == 0.0f ? 0.0f : __frcp_rn(l)) * (R == kNone ? 0.0f : pow2i(R - 8));
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld32(tmem_o + c + lanes, o);
        tmem_ld_wait();
        if (live && ok) {
          uint4* const y = reinterpret_cast<uint4*>(p.out + orow * D + c);
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * i]) * inv, __uint_as_float(o[j + 2 * i + 1]) * inv);
              w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            y[j / 8] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (live && ok && p.lse) p.lse[orow] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
    } else {
      // every product of this CTA is done, so its tiles are free: rows of D floats, 16-byte units in an order that meets no bank twice
      s_m[row] = m; s_l[row] = l; s_r[row] = R;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (tiles > 0) {
          tmem_ld32(tmem_o + c + lanes, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<uint4*>(smem + row * (D * 4) + ((((c + j) >> 2) ^ (row & 7)) << 4)) =
              tiles > 0 ? make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]) : make_uint4(0, 0, 0, 0);
      }
    }
  }
  if (split > 1) {
    cluster.sync();
    // this CTA finishes rows part * 128 / split ..
    const int mine = kRows / split;
    for (int i = threadIdx.x; i < mine * (D / 4); i += kThreads) {
      const int row = part * mine + i / (D / 4), u = i % (D / 4);
      if (row >= valid) continue;
      float mm = -INFINITY, ll = 0.0f;
      int rr = kNone;
      for (int c = 0; c < split; ++c) { mm = fmaxf(mm, *cluster.map_shared_rank(&s_m[row], c)); rr = max(rr, *cluster.map_shared_rank(&s_r[row], c)); }
      const float back = mm == -INFINITY ? 0.0f : mm;
      float4 acc = make_float4(0, 0, 0, 0);
      for (int c = 0; c < split; ++c) {
        const float a = ex2(*cluster.map_shared_rank(&s_m[row], c) - back);
        const int rc = *cluster.map_shared_rank(&s_r[row], c);
        const float fo = a * (rc == kNone ? 0.0f : move_unit(rc, rr));
        ll += a * *cluster.map_shared_rank(&s_l[row], c);
        const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(smem + row * (D * 4) + ((u ^ (row & 7)) << 4), c));
        acc.x += fo * x.x; acc.y += fo * x.y; acc.z += fo * x.z; acc.w += fo * x.w;
      }
      const int tk = div_group(p, head0 + row), hd = head * p.group + head0 + row - tk * p.group;
      const int64_t orow = (int64_t)(r.r0 + token0 + tk) * (t.n_kv_heads * p.group) + hd;
      const float inv = (ll == 0.0f ? 0.0f : __frcp_rn(ll)) * (rr == kNone ? 0.0f : pow2i(rr - 8));
      const __nv_bfloat162 y0 = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), y1 = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
      uint2 pk;
      pk.x = *reinterpret_cast<const uint32_t*>(&y0); pk.y = *reinterpret_cast<const uint32_t*>(&y1);
      *reinterpret_cast<uint2*>(p.out + orow * D + 4 * u) = pk;
      if (p.lse && u == 0) p.lse[orow] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
    }
    cluster.sync();                               // the others may still be reading this CTA's shared memory
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

template <int D, int SUBS>
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
  B2Q_SMEM_ATTR(h, (kv8_prefill_kernel<D, SUBS>), C::kSmem);
  // Few row tiles against many keys: as many CTAs to a row tile as still find a place at once, each with eight key tiles at least.  Measured, us
  // by the number of CTAs (taken: *): 1 x 512 tokens behind 15000 1: 221, 2: 154*, 4: 163;  1 x 130 behind 8000 1: 118, 2: 70, 4: 52*, 8: 53;
  // 2 x 256 behind 4000 1: 66, 2: 55*, 4: 64;  4 x 300 behind 2000 1: 47*, 2: 65.
  const int64_t most = (int64_t)p.t.table_width << p.t.page_shift, keys = p.window ? p.window + kTile : most;
  int split = 1;
  while (split < 8 && units * p.t.n_kv_heads * split * 2 <= 2 * (int64_t)h->sm_count && keys >= (int64_t)split * 16 * kTile) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.t.n_kv_heads * split), (unsigned)(units < kGridY ? units : kGridY), (unsigned)ceil_div64(units, kGridY));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
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
  B2Q_CUDA(h, cudaLaunchKernelEx(&cfg, (kv8_prefill_kernel<D, SUBS>), map_k, map_v, p));
  return B2Q_OK;
}

}  // namespace pre
}  // namespace kv8

// The caller has checked the arguments.
int32_t b2q_kv8_prefill(b2q_handle h, const kv8::AttendArgs& p, int64_t head_dim) {
  using namespace kv8::pre;
  if (head_dim == 64) return p.t.page_shift >= 6 ? launch<64, 1>(h, p) : p.t.page_shift == 5 ? launch<64, 2>(h, p) : launch<64, 4>(h, p);
  return p.t.page_shift >= 6 ? launch<128, 1>(h, p) : p.t.page_shift == 5 ? launch<128, 2>(h, p) : launch<128, 4>(h, p);
}

// Attention of few query rows over the paged 8-bit cache (layout: kv8.cuh):
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  keys j <= pos_i (pos_i = len - n + i), with a window also j > pos_i - window.
// Bound by HBM: the codes of the visible keys and values are read once; everything else is small.
//
// A row is one (new token, query head) pair; the rows of one sequence and kv head that share keys are taken 8 * RB at a time.
// Both products run on mma.sync.m16n8k16 (f16 x f16, f32 sums) with the cache as the 16-row operand and the query rows as the 8
// columns, so that none of the tensor work is padding for groups of up to 8 heads and an output takes D / 4 registers:
//   scores^T  [16 keys x 8 rows] = K [16 x D] . Q^T;      outputs^T [16 channels x 8 rows] = V^T [16 x keys] . P^T.
// An E4M3 code is exact in f16 (one conversion instruction for two).  Q enters as f16 after a power of two has brought its row's
// largest element into [2^14, 2^15): a bf16 has 8 significant bits and f16 has 11, so it is exact but for elements below 2^-28 of that
// largest.  The weights enter as p * 2^7 to p * 2^15 rounded to f16: off by 2^-11 of themselves, or by 2^-32 of the row's largest.
// Channels are dealt to lanes so that a lane's operands are 16 neighbouring bytes of a row (both products sum over, or are independent
// of, the order of channels); 8 x 8 tiles of P are transposed between lanes by movmatrix, pairs of keys of V by byte permutations.
// One warp brings tiles of 64 keys into a ring of shared memory by TMA (it alone walks the block table, a batch of tiles ahead); three
// pairs of warps take the tiles in turn, 32 keys to a warp, each with its own running maximum and sum, so the main loop has no
// barrier between them.  Warps and the CTAs of a cluster (tiles dealt round) are joined once at the end, through shared and distributed
// shared memory: no workspace, one launch, and a result that does not depend on timing.
// The value scale is a power of two 2^lv per page: weights enter as p * 2^(15 + lv - R) and the outputs are kept in units of
// 2^(R - 15), R following the pages' scales (next_unit in kv8.cuh); pages of one tile whose scales lie more than 2^8 apart are multiplied
// one after the other.
// Keys behind the last visible one are masked and their value rows zeroed before they are multiplied, so stale codes cannot reach a
// result; a page that the table does not name is neither read nor counted.
// Measured: 32 sequences x 8200 keys (32 heads of 128 channels over 8 kv heads) 88 us, 4.6 TB/s of cache (pages of 16: 94 us); the same copies
// without the arithmetic 74 us.  256 equal CTAs share 148 SMs there, so the SMs that hold two set the time.
// Every mbarrier wait is bounded; on expiry the kernel records B2Q_ERR_TIMEOUT and leaves.
#include "kv8.cuh"
#include "tc_common.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace kv8 {

using namespace tcx;

constexpr int kWarps = 6, kTile = 64;            // consumer warps (pairs); keys of one tile
constexpr int kThreads = 32 * (kWarps + 1);
constexpr uint64_t kWaitLimitNs = 500000000ull;
template <int D> struct Ring {
  static constexpr int kHalf = kTile * D, kStage = 2 * kHalf;          // keys, then values
  static constexpr int kStages = D == 128 ? 6 : 9;                     // 96 KiB / 72 KiB, two CTAs to an SM
  static_assert(kStages % (kWarps / 2) == 0, "a stage belongs to one pair of warps, which cannot run a phase ahead of its own");
  static constexpr int kSmem = kStages * kStage + kStages * 32 + 1024;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// four E4M3 codes -> two registers of two f16 (codes 0 and 1, codes 2 and 3)
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// over the 8 lanes that share lane & 3
__device__ __forceinline__ float column_max(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float column_sum(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// byte offset of 16-byte unit u of row r in a tile of D-byte rows whose 128-byte lines TMA has swizzled
template <int D> __device__ __forceinline__ uint32_t swz(int r, int u) {
  const uint32_t at = (uint32_t)(r * D + u * 16);
  return at ^ (((at >> 7) & 7) << 4);
}
// The key (within its group of 8) that row lr of an operand stands for: an order in which the 16-byte reads of both products meet no
// bank twice (keys 2 i, 2 i + 1 of the order lie in different halves of the swizzled lines, keys 2 i + e over i in different units).
template <int D> __device__ __forceinline__ int key_of(int lr) { return (D == 128 ? 0x37156240u : 0x65742130u) >> (4 * lr) & 7; }

template <int D, int RB>
__global__ void __launch_bounds__(kThreads, RB == 1 ? 2 : 1)
kv8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttendArgs p) {
  constexpr int kRows = 8 * RB;
  constexpr int KC = D / 64;                     // 16-byte chunks of a key row per lane
  constexpr int MT = D / 16;                     // 16-channel tiles of the outputs
  constexpr int VB = D / 8;                      // bytes of a value row per lane (channels lr * VB ..)
  using G = Ring<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const ring = smem_raw + (base - smem_u32(smem_raw));
  auto full_bar = [&](int i) { return base + G::kStages * G::kStage + 8u * i; };
  auto empty_bar = [&](int i) { return base + G::kStages * G::kStage + 8u * (G::kStages + i); };
  uint4* const s_info = reinterpret_cast<uint4*>(ring + G::kStages * G::kStage + 16 * G::kStages);   // [stage], one word per 16 keys
  float (*const s_o)[kRows][D] = reinterpret_cast<float (*)[kRows][D]>(ring);                       // [kWarps], when the ring is done with
  static_assert(kWarps * kRows * D * 4 <= G::kStages * G::kStage, "the join reuses the ring");
  __shared__ int4 s_line[32];                    // the producer's next tiles: lines of their pages, scales
  __shared__ uint4 s_words[32];
  __shared__ int s_abort;
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ int s_r[kWarps];
  __shared__ float s_cm[kRows], s_cl[kRows];     // this CTA's join
  __shared__ int s_cr;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int i = 0; i < G::kStages; ++i) { mbar_init(full_bar(i), 2); mbar_init(empty_bar(i), 2); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  __syncthreads();
  volatile int* abort_flag = &s_abort;
  b2q_pdl_entry();
  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const Batch& t = p.t;
  const int head = blockIdx.y, warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, lr = lane >> 2, tq = lane & 3;
  const int unit = (int)(blockIdx.x / split);
  const bool tell = head == 0 && part == 0 && warp == 0;

  Found f;
  if (t.q_starts == nullptr) {
    const int per = (p.group + kRows - 1) / kRows;
    f = Found{unit / per, unit % per, per};
  } else {
    if (unit == 0 && tell) for (int b = lane; b < t.seqs; b += 32) rows_of(t, b, true);
    f = find_unit(t.seqs, unit, [&](int b) { return (rows_of(t, b, false).n * p.group + kRows - 1) / kRows; });
    if (f.b < 0) return;                          // the whole cluster leaves: every CTA of it has the same unit
  }
  const Rows r = rows_of(t, f.b, tell && t.q_starts == nullptr && lane == 0);
  const int row0 = f.index * kRows, valid = min(kRows, r.n * p.group - row0);   // rows of all sequences fit 31 bits; <= 0: an impossible sequence
  if (valid <= 0) return;                         // its rows stay as they are
  const int token0 = row0 / p.group, head0 = row0 - token0 * p.group;       // of the first row, within the sequence and the group
  const int first_pos = r.len - r.n + token0, last_pos = first_pos + (head0 + valid - 1) / p.group;
  const int key_end = last_pos + 1;
  // the first key that a row sees; the first tile may begin before it, with pages that its owner has given up and that are not looked up
  const int key_low = p.window > 0 ? max(0, first_pos - p.window + 1) : 0, key_begin = key_low & ~(kTile - 1);

  const int tiles = (key_end - key_begin + kTile - 1) / kTile, mine = (tiles - part + split - 1) / split;   // tiles part, part + split, ..

  float o[RB][MT][4];
  float m[RB][2], l[RB][2];
  int R = kNone, top = kNone;                    // unit of o, the largest so far
#pragma unroll
  for (int x = 0; x < RB; ++x) {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[x][j][i] = 0.0f;
    m[x][0] = m[x][1] = -INFINITY;
    l[x][0] = l[x][1] = 0.0f;
  }

  if (warp == kWarps) {
    // ---------------- producer: the pages and scales of 32 tiles at a time, a tile to a lane, fetched while the copies of the 32 before
    // them are issued ----------------
    const int subs = t.page_shift >= 6 ? 1 : 64 >> t.page_shift, rows_each = kTile / subs;   // pages that a tile spans, their keys
    int pg[4];
    uint32_t info[4];
    auto pages = [&](int i0) {
      const int j0 = key_begin + kTile * (part + split * (i0 + lane));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + rows_each * e;
        pg[e] = e < subs && i0 + lane < mine && j < key_end && (j | (rows_each - 1)) >= key_low ? page_of(t, f.b, j >> t.page_shift, head == 0) : -1;
      }
    };
    auto scales = [&] {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        info[e] = pg[e] < 0 ? 0u : 0x80000000u | (uint32_t)p.ks[(int64_t)pg[e] * t.n_kv_heads + head] | ((uint32_t)p.vs[(int64_t)pg[e] * t.n_kv_heads + head] << 8);
    };
    // A lane leaves the lines of its tile's pages (the maps see lines of 128 bytes: one token of 128 channels, or two of 64; -1: no page) and
    // the scales in shared memory.  The warp stays together and elects a lane to issue, so that a copy's operands live in uniform registers: with
    // lane 0 alone in a branch, 32 x 8200 keys in pages of 16 (eight copies to a tile) took 113 us instead of 94.
    auto leave = [&](int i0) {
      const int in_page = (key_begin + kTile * (part + split * (i0 + lane))) & ((1 << t.page_shift) - 1);   // 0 but for pages of 128
      int line[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) line[e] = pg[e] < 0 ? -1 : (((pg[e] * t.n_kv_heads + head) << t.page_shift) + in_page) / (128 / D);
      s_line[lane] = make_int4(line[0], line[1], line[2], line[3]);
    };
    auto words = [&] {
      return subs == 1 ? make_uint4(info[0], info[0], info[0], info[0]) : subs == 2 ? make_uint4(info[0], info[0], info[1], info[1])
                                                                                     : make_uint4(info[0], info[1], info[2], info[3]);
    };
    const uint32_t bytes = (uint32_t)rows_each * D;
    auto copy = [&](int st, const int4 ln) {
      const uint32_t dk = base + st * G::kStage, dv = dk + G::kHalf, bar = full_bar(st);
      const int there = (ln.x >= 0) + (ln.y >= 0) + (ln.z >= 0) + (ln.w >= 0);
      mbar_expect_tx(bar, there * 2 * bytes);
      if (ln.x >= 0) { tma_load_2d(dk, &map_k, bar, 0, ln.x); tma_load_2d(dv, &map_v, bar, 0, ln.x); }
      if (subs > 1) {
        if (ln.y >= 0) { tma_load_2d(dk + bytes, &map_k, bar, 0, ln.y); tma_load_2d(dv + bytes, &map_v, bar, 0, ln.y); }
        if (ln.z >= 0) { tma_load_2d(dk + 2 * bytes, &map_k, bar, 0, ln.z); tma_load_2d(dv + 2 * bytes, &map_v, bar, 0, ln.z); }
        if (ln.w >= 0) { tma_load_2d(dk + 3 * bytes, &map_k, bar, 0, ln.w); tma_load_2d(dv + 3 * bytes, &map_v, bar, 0, ln.w); }
      }
    };
    // the first copies go out before the scales are known, and the scales arrive while they fly
    bool ok = true;
    const int lead_in = min(mine, G::kStages);
    pages(0);
    leave(0);
    __syncwarp();
    if (lane == 0) for (int i = 0; i < lead_in; ++i) copy(i, s_line[i]);
    scales();
    if (lane < lead_in) {
      s_info[lane] = words();
      mbar_arrive(full_bar(lane));                // the second of a stage's two arrivals
    }
    for (int i0 = 0; i0 < mine && ok; i0 += 32) {
      s_words[lane] = words();
      __syncwarp();
      if (i0 + 32 < mine) { pages(i0 + 32); scales(); }                // in flight while the copies are issued
      const int n = min(32, mine - i0);
      for (int i = i0 ? 0 : lead_in; i < n; ++i) {
        const int st = (i0 + i) % G::kStages;
        const int4 ln = s_line[i];
        const uint4 w = s_words[i];
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(empty_bar(st), (((i0 + i) / G::kStages) & 1) ^ 1, abort_flag, kWaitLimitNs, 1));
        if (!ok) break;
        const int4 same = make_int4(__shfl_sync(0xffffffffu, ln.x, 0), __shfl_sync(0xffffffffu, ln.y, 0), __shfl_sync(0xffffffffu, ln.z, 0), __shfl_sync(0xffffffffu, ln.w, 0));
        if (elect_one()) {
          copy(st, same);
          s_info[st] = w;
          mbar_arrive(full_bar(st));
        }
        __syncwarp();
      }
      leave(i0 + 32);
    }
    if (!ok && lane == 0) {                      // give copies in flight time to land before shared memory is released
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 2000000ull) {}
    }
  } else {
    // ---- the query rows: this lane holds channels 64 c + 16 tq .. of rows lr, lr + 8, .. as the 8-column operand ----
    uint32_t qb[RB][4 * KC][2];
    float qf[RB][2];                               // score factors of rows 8 x + 2 tq + {0, 1}, the rows of this lane's scores
    int pos[RB][2];
#pragma unroll
    for (int x = 0; x < RB; ++x) {
      const int row = 8 * x + lr;
      const bool live = row < valid;
      const int token = live ? token0 + (head0 + row) / p.group : token0, g = live ? (head0 + row) % p.group : 0;
      const __nv_bfloat16* qp = p.q + (int64_t)(r.r0 + token) * p.ld_q + (int64_t)(head * p.group + g) * D + tq * 16;
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
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      bad = (__ballot_sync(0xffffffffu, bad) >> (lane & 28)) & 0xF;
      const int e = max(-126, (int)(__float_as_uint(amax) >> 23) - 127 - 14);
      const float inv = p.scale < 0.0f ? -pow2i(-e) : pow2i(-e);        // a negative scale enters with the query
      const float factor = bad ? __uint_as_float(0x7FC00000u) : fabsf(p.scale) * pow2i(e);   // a query with an infinity or a NaN: NaN throughout
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t u[4] = {w[c][s].x, w[c][s].y, w[c][s].z, w[c][s].w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            qb[x][4 * c + 2 * s + (j >> 1)][j & 1] = pack_f16(__uint_as_float(u[j] << 16) * inv, __uint_as_float(u[j] & 0xFFFF0000u) * inv);
        }
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        qf[x][e2] = __shfl_sync(0xffffffffu, factor, 8 * tq + 4 * e2);
        const int rr = 8 * x + 2 * tq + e2;
        pos[x][e2] = rr < valid ? first_pos + (head0 + rr) / p.group : -1;
      }
    }

    const int mk = key_of<D>(lr), ve[2] = {key_of<D>(2 * tq), key_of<D>(2 * tq + 1)};   // this lane's key row, its two value rows (mod 8)
    for (int it = warp >> 1; it < mine; it += kWarps / 2) {
      const int st = it % G::kStages, j0 = key_begin + kTile * (part + split * it) + 32 * (warp & 1);   // this warp's 32 keys
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(full_bar(st), (it / G::kStages) & 1, abort_flag, kWaitLimitNs, 1))) break;
      const uint8_t* const ks = ring + st * G::kStage + 32 * (warp & 1) * D;
      uint8_t* const vs = ring + st * G::kStage + G::kHalf + 32 * (warp & 1) * D;
      const uint2 info = reinterpret_cast<const uint2*>(s_info + st)[warp & 1];
      const uint32_t sc[2] = {info.x, info.y};     // of keys 0..15 and 16..31
      if (j0 < key_end) {
        const int lv[2] = {(int)(sc[0] >> 8 & 0xFF) - 127, (int)(sc[1] >> 8 & 0xFF) - 127};
        // whole: every key is there; clear: and every row sees every key, and the value scales go together
        const bool whole = (sc[0] & sc[1]) >> 31 && j0 + 32 <= key_end;
        const bool clear = whole && abs(lv[0] - lv[1]) <= kSpan && j0 + 31 <= first_pos && (p.window <= 0 || j0 > last_pos - p.window);
        if (!whole) {                              // value rows without a visible key: whatever they hold becomes 0
          if (!(sc[lane >> 4] >> 31) || j0 + lane >= key_end)
#pragma unroll
            for (int u = 0; u < D / 16; ++u) *reinterpret_cast<uint4*>(vs + swz<D>(lane, u)) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }

        // ---- products with the keys: this lane has keys j0 + 8 g + mk of rows 8 x + 2 tq + {0, 1} ----
        float s[RB][4][2];
        float c[2][RB][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int x = 0; x < RB; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) c[mt][x][i] = 0.0f;
#pragma unroll
        for (int ch = 0; ch < KC; ++ch) {
          uint4 kk[2][2];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) kk[mt][e] = *reinterpret_cast<const uint4*>(ks + swz<D>(16 * mt + 8 * e + mk, 4 * ch + tq));
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {                          // two independent chains of products
              const uint32_t ka = k == 0 ? kk[mt][0].x : k == 1 ? kk[mt][0].y : k == 2 ? kk[mt][0].z : kk[mt][0].w;
              const uint32_t kb = k == 0 ? kk[mt][1].x : k == 1 ? kk[mt][1].y : k == 2 ? kk[mt][1].z : kk[mt][1].w;
              uint32_t a0, a1, a2, a3;
              to_f16(ka, a0, a2);
              to_f16(kb, a1, a3);
#pragma unroll
              for (int x = 0; x < RB; ++x) mma_f16(c[mt][x], a0, a1, a2, a3, qb[x][4 * ch + k][0], qb[x][4 * ch + k][1]);
            }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int x = 0; x < RB; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) s[x][2 * mt + h][e] = c[mt][x][2 * h + e];
        // o = a * o + P^T V with pb: keys 8 g + ve[e] of row 8 x + lr
        auto accumulate = [&](const float (&a)[RB][2], const uint32_t (&pb)[RB][4]) {
          uint32_t vr[4][2][VB / 4];                 // values of keys 8 g + ve[e], channels VB lr ..
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(vs + swz<D>(8 * g + ve[e], lr));
                vr[g][e][0] = x.x; vr[g][e][1] = x.y; vr[g][e][2] = x.z; vr[g][e][3] = x.w;
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(vs + swz<D>(8 * g + ve[e], lr >> 1) + 8 * (lr & 1));
                vr[g][e][0] = x.x; vr[g][e][1] = x.y;
              }
            }
          bool moved = false;
#pragma unroll
          for (int x = 0; x < RB; ++x) moved |= a[x][0] != 1.0f || a[x][1] != 1.0f;
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int x = 0; x < RB; ++x)
#pragma unroll
              for (int j = 0; j < MT; ++j) { o[x][j][0] *= a[x][0]; o[x][j][1] *= a[x][1]; o[x][j][2] *= a[x][0]; o[x][j][3] *= a[x][1]; }
          }
#pragma unroll
          for (int w = 0; w < VB / 4; ++w) {                            // channels VB lr + 4 w .. + 3: two tiles of 16
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int sel = hf ? 0x7362 : 0x5140;                     // channel pairs of two keys: k0 c0, k1 c0, k0 c1, k1 c1
#pragma unroll
              for (int k2 = 0; k2 < 2; ++k2) {
                uint32_t a0, a1, a2, a3;
                to_f16(__byte_perm(vr[2 * k2][0][w], vr[2 * k2][1][w], sel), a0, a1);
                to_f16(__byte_perm(vr[2 * k2 + 1][0][w], vr[2 * k2 + 1][1][w], sel), a2, a3);
#pragma unroll
                for (int x = 0; x < RB; ++x) mma_f16(o[x][2 * w + hf], a0, a1, a2, a3, pb[x][2 * k2], pb[x][2 * k2 + 1]);
              }
            }
          }
        };
        float alpha[RB][2];
        uint32_t pb[RB][4];
        if (clear) {
          const float move = next_unit(R, top, max(lv[0], lv[1]), min(lv[0], lv[1]), 0), kf[2] = {pow2_byte(sc[0] & 0xFF), pow2_byte(sc[1] & 0xFF)};
          const int up[2] = {max(15 + lv[0] - R, kLeast), max(15 + lv[1] - R, kLeast)};
          const float down[2] = {pow2i(-up[0]), pow2i(-up[1])}, shift[2] = {(float)up[0], (float)up[1]};
#pragma unroll
          for (int x = 0; x < RB; ++x) {
            float w[4][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float fs[2] = {qf[x][e] * kf[0], qf[x][e] * kf[1]};   // not negative: the sign of the scale is in the query
              const float mn = fmaxf(m[x][e], column_max(fmaxf(fmaxf(s[x][0][e], s[x][1][e]) * fs[0], fmaxf(s[x][2][e], s[x][3][e]) * fs[1])));
              const float a = ex2(m[x][e] - mn), base[2] = {shift[0] - mn, shift[1] - mn};
              alpha[x][e] = a * move;
              m[x][e] = mn;
#pragma unroll
              for (int g = 0; g < 4; ++g) w[g][e] = ex2(fmaf(s[x][g][e], fs[g >> 1], base[g >> 1]));
              // the sum is of the weights without the values' scale
              l[x][e] = fmaf(l[x][e], a, fmaf(w[0][e] + w[1][e], down[0], (w[2][e] + w[3][e]) * down[1]));
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) pb[x][g] = transpose8x8(pack_f16(w[g][0], w[g][1]));
          }
          accumulate(alpha, pb);
        } else {
#pragma unroll
          for (int x = 0; x < RB; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mt = -INFINITY;
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const int j = j0 + 8 * g + mk;
                const bool see = j <= pos[x][e] && (p.window <= 0 || j > pos[x][e] - p.window) && sc[g >> 1] >> 31;
                s[x][g][e] = see ? s[x][g][e] * (qf[x][e] * pow2_byte(sc[g >> 1] & 0xFF)) : -INFINITY;
                mt = fmaxf(mt, s[x][g][e]);
              }
              const float mn = fmaxf(m[x][e], column_max(mt)), base = mn == -INFINITY ? 0.0f : mn;   // nothing seen yet: exp2(-inf - 0) = 0
              alpha[x][e] = ex2(m[x][e] - base);
              m[x][e] = mn;
              l[x][e] *= alpha[x][e];
#pragma unroll
              for (int g = 0; g < 4; ++g) { s[x][g][e] = ex2(s[x][g][e] - base); l[x][e] += s[x][g][e]; }
            }
          // the halves whose value scales lie within 2^kSpan of the larger together, else one after the other
          unsigned rem = (sc[0] >> 31) | (sc[1] >> 31 && j0 + 16 < key_end ? 2u : 0u);
          while (rem) {
            const int lead = rem == 3 ? max(lv[0], lv[1]) : rem == 1 ? lv[0] : lv[1];
            const unsigned take = rem & ((lv[0] >= lead - kSpan ? 1u : 0u) | (lv[1] >= lead - kSpan ? 2u : 0u));
            const float move = next_unit(R, top, lead, take == 3 ? min(lv[0], lv[1]) : take == 1 ? lv[0] : lv[1], 0), up[2] = {take & 1 ? pow2i(15 + lv[0] - R) : 0.0f, take & 2 ? pow2i(15 + lv[1] - R) : 0.0f};
#pragma unroll
            for (int x = 0; x < RB; ++x) {
              alpha[x][0] *= move; alpha[x][1] *= move;
#pragma unroll
              for (int g = 0; g < 4; ++g) pb[x][g] = transpose8x8(pack_f16(s[x][g][0] * up[g >> 1], s[x][g][1] * up[g >> 1]));
            }
            accumulate(alpha, pb);
#pragma unroll
            for (int x = 0; x < RB; ++x) alpha[x][0] = alpha[x][1] = 1.0f;
            rem &= ~take;
          }
        }
        if (!whole) fence_async_smem();            // the zeros, before the next copy into this stage
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(st));
    }
  }

  // ---- join the warps of this CTA, then the CTAs of the cluster ----
  __syncthreads();                               // every tile has been multiplied: the ring is free
  if (warp < kWarps) {
#pragma unroll
    for (int x = 0; x < RB; ++x)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ll = column_sum(l[x][e]);
        const int rr = 8 * x + 2 * tq + e;
        if (lr == 0) { s_m[warp][rr] = m[x][e]; s_l[warp][rr] = ll; }
#pragma unroll
        for (int j = 0; j < MT; j += 2)                                 // tile j: channels VB lr + 2 j + {0, 1} (registers e and 2 + e)
          *reinterpret_cast<float4*>(&s_o[warp][rr][lr * VB + 2 * j]) = make_float4(o[x][j][e], o[x][j][2 + e], o[x][j + 1][e], o[x][j + 1][2 + e]);
      }
    if (lane == 0) s_r[warp] = R;
  }
  __syncthreads();
  // row rr, channels cc .. of the outputs: a row that sees no key has ll = 0, zeros and -inf; a query that holds an infinity or a NaN has
  // ll = NaN and stays NaN
  auto finish = [&](int rr, int cc, const float4 acc, float mm, float ll, int unit_exp) {
    const int hd = head0 + rr, tk = hd / p.group;
    const int64_t orow = (int64_t)(r.r0 + token0 + tk) * (t.n_kv_heads * p.group) + head * p.group + (hd - tk * p.group);
    const float k = (ll == 0.0f ? 0.0f : __frcp_rn(ll)) * (unit_exp == kNone ? 0.0f : pow2i(unit_exp - 15));
    const __nv_bfloat162 y0 = __floats2bfloat162_rn(acc.x * k, acc.y * k), y1 = __floats2bfloat162_rn(acc.z * k, acc.w * k);
    uint2 pk;
    pk.x = *reinterpret_cast<const uint32_t*>(&y0); pk.y = *reinterpret_cast<const uint32_t*>(&y1);
    *reinterpret_cast<uint2*>(p.out + orow * D + cc) = pk;
    if (p.lse && cc == 0) p.lse[orow] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * 0.69314718055994531f;
  };
  int cr = kNone;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) cr = max(cr, s_r[w]);
  for (int i = threadIdx.x; i < kRows * D / 4; i += kThreads) {
    const int rr = i / (D / 4), cc = (i % (D / 4)) * 4;
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][rr]);
    const float b = mm == -INFINITY ? 0.0f : mm;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float a = ex2(s_m[w][rr] - b), fo = a * (s_r[w] == kNone ? 0.0f : move_unit(s_r[w], cr));
      ll += a * s_l[w][rr];
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][rr][cc]);
      acc.x += fo * x.x; acc.y += fo * x.y; acc.z += fo * x.z; acc.w += fo * x.w;
    }
    if (split == 1) {
      if (rr < valid) finish(rr, cc, acc, mm, ll, cr);
      continue;
    }
    *reinterpret_cast<float4*>(&s_o[0][rr][cc]) = acc;                // read and written by this thread alone
    if (cc == 0) { s_cm[rr] = mm; s_cl[rr] = ll; }
  }
  if (split > 1) {
    if (threadIdx.x == 0) s_cr = cr;
    cluster.sync();
    int tr = kNone;
    for (int c = 0; c < split; ++c) tr = max(tr, *cluster.map_shared_rank(&s_cr, c));
    for (int i = part * kThreads + threadIdx.x; i < kRows * D / 4; i += split * kThreads) {   // every CTA finishes a part of the rows
      const int rr = i / (D / 4), cc = (i % (D / 4)) * 4;
      if (rr >= valid) continue;
      float mm = -INFINITY, ll = 0.0f;
      for (int c = 0; c < split; ++c) mm = fmaxf(mm, *cluster.map_shared_rank(&s_cm[rr], c));
      const float b = mm == -INFINITY ? 0.0f : mm;
      float4 acc = make_float4(0, 0, 0, 0);
      for (int c = 0; c < split; ++c) {
        const float a = ex2(*cluster.map_shared_rank(&s_cm[rr], c) - b);
        const int rc = *cluster.map_shared_rank(&s_cr, c);
        const float fo = a * (rc == kNone ? 0.0f : move_unit(rc, tr));
        ll += a * *cluster.map_shared_rank(&s_cl[rr], c);
        const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(&s_o[0][rr][cc], c));
        acc.x += fo * x.x; acc.y += fo * x.y; acc.z += fo * x.z; acc.w += fo * x.w;
      }
      finish(rr, cc, acc, mm, ll, tr);
    }
    cluster.sync();                                                   // the others may still be reading this CTA's shared memory
  }
  if (threadIdx.x == 0 && s_abort) report(t.status, B2Q_ERR_TIMEOUT);
}

}  // namespace kv8

template <int D, int RB>
static int32_t kv8_decode_launch(b2q_handle h, const kv8::AttendArgs& p, int64_t units, int split) {
  using G = kv8::Ring<D>;
  CUtensorMap map_k, map_v;
  const uint64_t lines = ((uint64_t)p.t.num_pages * p.t.n_kv_heads << p.t.page_shift) / (128 / D);
  const uint32_t box = (p.t.page_shift < 6 ? 1 << p.t.page_shift : kv8::kTile) / (128 / D);
  int32_t st = b2q_tensor_map_2d(h, &map_k, p.k, 1, 128, lines, 128, box);
  if (st != B2Q_OK) return st;
  st = b2q_tensor_map_2d(h, &map_v, p.v, 1, 128, lines, 128, box);
  if (st != B2Q_OK) return st;
  B2Q_SMEM_ATTR(h, (kv8::kv8_decode_kernel<D, RB>), G::kSmem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * split), (unsigned)p.t.n_kv_heads);
  cfg.blockDim = dim3(kv8::kThreads);
  cfg.dynamicSmemBytes = G::kSmem;
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
  B2Q_CUDA(h, cudaLaunchKernelEx(&cfg, (kv8::kv8_decode_kernel<D, RB>), map_k, map_v, p));
  return B2Q_OK;
}

// CTAs that share the keys of the same rows: the number for which the busiest SM is done first, by its CTAs times the tiles of each plus
// kFixed for what every CTA costs besides.  A CTA alone on an SM that has room for two leaves some of it idle (kAlone).  Measured with 8
// query rows to a kv head of 128 channels and 8 kv heads, by the number of CTAs to the same rows, in us:
//   sequences x keys     1     2     3     4     6     8        sequences x keys     1     2     3     4     6     8
//          1 x 32000   187    99    69    54    40    32              16 x 8200    60    52    61    54    62    68
//           4 x 8200    53    32    25    27    24    21              20 x 8200    88    70    68    71    80    87
//           8 x 8200    57    35    39    33    42    40              32 x 8200    93    92   100   102   118   130
//          12 x 8200    58    51    49    51    52    54              32 x 1000    20    25    32    37    53    65
static int kv8_decode_split(int64_t units, int64_t tiles, int rb, int sms) {
  constexpr double kFixed = 12, kAlone = 1.3;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 8; ++s) {
    const double ctas = (double)ceil_div64(units * s, sms), cost = (rb == 1 && ctas < kAlone ? kAlone : ctas) * ((double)ceil_div64(tiles, s) + kFixed);
    if (s == 1 || cost < least) { best = s; least = cost; }
  }
  return best;
}

int32_t b2q_kv8_prefill(b2q_handle h, const kv8::AttendArgs& p, int64_t head_dim);   // kv8_prefill.cu

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
  if (n_heads / n_kv_heads > 1 << 20) B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_attention: %lld query heads are too many", (long long)n_heads);
  p.group = (int)(n_heads / n_kv_heads);
  p.per_group = 1.0f / (float)p.group;
  const int64_t most = table_width * page_size;                        // keys that a sequence can have
  p.window = window > 0 && window < most ? (int)window : 0;
  p.scale = scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(out); p.lse = lse;
  if (tokens * p.group > 0x7FFFFFFF - 128)
    B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_attention: %lld tokens of %lld heads are too many", (long long)tokens, (long long)n_heads);
  // More than 16 rows to a sequence and kv head on average: the prefill kernel.  Measured there and here, us: 16 rows, 8 sequences x 4000 keys
  // 30.6 and 26.0; 32 rows, 8 x 4000 33.2 and 36.2, 32 x 2000 46 and 71, 1 x 8000 24.9 and 33.0; 64 rows, 8 x 4000 40.6 and 58.9.
  if (tokens * p.group > 16 * seqs) return b2q_kv8_prefill(h, p, head_dim);
  // Rows that share keys: up to 8 a CTA, 16 where a sequence has more than 8 on average (one conversion of the codes serves both halves).
  // 16 rows with 16 and with 8 to a CTA, us: 8 sequences x 4000 keys 25.2 and 29.9, 1 x 8000 17.9 and 20.9, 16 x 4000 36.4 and 48.0.
  const int rb = tokens * p.group > 8 * seqs ? 2 : 1, per = 8 * rb;
  const int64_t units = q_starts ? tokens * p.group / per + seqs : seqs * ceil_div64(p.group, per);   // at most
  const int64_t tiles = ceil_div64(p.window ? p.window + kv8::kTile : most, kv8::kTile);
  const int split = kv8_decode_split(seqs * ceil_div64(ceil_div64(tokens * p.group, seqs), per) * n_kv_heads, tiles, rb, h->sm_count);
  if (units * split > 0x7FFFFFFF) B2Q_FAIL(h, B2Q_ERR_INVALID_DIMENSION, "kv8_attention: %lld tokens of %lld heads are too many", (long long)tokens, (long long)n_heads);
  if (head_dim == 64) return rb == 1 ? kv8_decode_launch<64, 1>(h, p, units, split) : kv8_decode_launch<64, 2>(h, p, units, split);
  return rb == 1 ? kv8_decode_launch<128, 1>(h, p, units, split) : kv8_decode_launch<128, 2>(h, p, units, split);
}

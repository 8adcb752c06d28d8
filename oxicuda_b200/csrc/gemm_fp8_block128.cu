// FP8 GEMM whose scales go per block of 128 along K:
//   out[m, n] = sum_b sa[m, b] * sw[n / 128, b] * sum_{k in block b} A[m, k] * W[n, k]
// A [M x K] and W [N x K] E4M3 / E5M2 codes, both K-major; sa [M x ceil(K / 128)], sw [ceil(N / 128) x ceil(K / 128)] f32.
//
// Prefill kernel (gemm_block128_pair_kernel): clusters of two CTAs on 256 x BN tiles of the output, tcgen05.mma.cta_group::2 over
// 128-byte-swizzled stages that TMA fills, as in the GEMM with per-row scales (gemm_tc.cu).  What differs is the accumulator: a
// scale changes with every block of 128 along K, so each block's product is a fresh TMEM accumulator (512 / BN of them in
// flight), and eight epilogue warps per CTA add scale * product to sums that they hold in registers (BN / 2 columns of one row
// per thread) while the tensor core works on the next blocks.  Per block and CTA the tensor core needs 128 x BN x 128 / 8192 =
// 2 BN clocks; the epilogue reads BN columns of TMEM and issues BN / 2 two-wide FMAs per warp scheduler, which fits beside it in issue slots, but not in
// time: a thread reads 16 columns, waits for them, adds, and reads the next.
// Measured: 4096 x 8192 x 28672 835 to 845 us in a graph of eight (2.3 PFLOP/s), 950 in runs long enough for the power cap (2.0; a call among others
// 986), 2048 x 8192 x 8192 130 us (2.1), 512 x 8192 x 8192 36 us (1.9).  The read-out bounds it: the product with a scale per row, whose accumulators
// are read once a tile, takes 670 us (745) at the first shape; at 4096 x 8192 x 8192 the tensor pipe is active 61 % of the time here and 88 % there.
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

// ---- prefill: two-CTA tcgen05 kernel ----
constexpr int BM = 128, BK = 128;                       // accumulator rows of one CTA, K bytes per stage
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;          // warp 0 TMA, warp 1 MMA, warps 2 and 3 scales, warps 4.. epilogue
// The launch gives every thread 168 registers (64512 / 384); an epilogue thread holds BN / 2 sums and 32 columns in flight and needs
// more, the first warpgroup needs few: 128 * 88 + 256 * 208 = 64512.
constexpr int kRegsFirst = 88, kRegsEpi = 208;
constexpr int kTmemCols = 512;
constexpr int kStageOut = kEpiWarps * 4096;             // per warp 32 rows x 128 bytes, the source of its TMA stores
constexpr uint64_t kWaitLimitNs = 2000000000ull;

template <int BN> struct Cfg {
  static constexpr int kBuf = kTmemCols / BN;           // accumulators in flight
  static constexpr int kBytesA = BM * BK;               // this CTA's 128 rows of A
  static constexpr int kBytesB = BN / 2 * BK;           // this CTA's half of the BN rows of W
  static constexpr int kStageBytes = kBytesA + kBytesB;
  static constexpr int kStages = BN == 256 ? 5 : 7;
  // scales: slots of four blocks of K, the product of both scales for each of the 128 rows and each 128 columns of the tile
  static constexpr int kColBlocks = BN / 128, kSlots = 3, kSlotBytes = 4 * kColBlocks * BM * 4;
  static constexpr int kSmem = kStages * kStageBytes + kStageOut + kSlots * kSlotBytes + 1024 + 256;
  static_assert(kSmem <= 232448, "shared memory of one SM");
};

struct Params {
  int64_t M, N, K;
  int kb;                                               // blocks of 128 along K
  int tiles_m, tiles_n, group_m, col_blocks;
  uint32_t idesc;
  const float* sa; const float* sw; int vec;            // vec: both can be read four scales at a time
  void* out; int out_type, tma_store;
  int32_t* status;
};

using namespace tcx;
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return mbar_wait_bounded(bar, parity, abort_flag, kWaitLimitNs, 1);
}
// By a whole warp, whose lanes leave together if one gives up.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
__device__ __forceinline__ void umma_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ float lo32(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi32(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// scales [k0, k0 + 4) of a row of n; what lies behind the last one is 0.  vec: 16-byte aligned and n % 4 == 0
__device__ __forceinline__ float4 load4(const float* row, int k0, int n, int vec) {
  if (vec) return k0 < n ? __ldg(reinterpret_cast<const float4*>(row + k0)) : make_float4(0, 0, 0, 0);
  return make_float4(k0 < n ? __ldg(row + k0) : 0.0f, k0 + 1 < n ? __ldg(row + k0 + 1) : 0.0f, k0 + 2 < n ? __ldg(row + k0 + 2) : 0.0f,
                     k0 + 3 < n ? __ldg(row + k0 + 3) : 0.0f);
}
// groups of group_m row tiles sweep the column tiles, so that a group's rows of A stay in L2 while W streams past
__device__ __forceinline__ void tile_coords(int tile, const Params& p, int& mb, int& nb) {
  const int per = p.group_m * p.tiles_n, first = tile / per * p.group_m, gm = min(p.tiles_m - first, p.group_m), in = tile % per;
  mb = first + in % gm;
  nb = in / gm;
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
gemm_block128_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out,
                          const Params p) {
  using C = Cfg<BN>;
  constexpr int kStages = C::kStages, kBuf = C::kBuf;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t out_base = base + kStages * C::kStageBytes;
  const uint32_t scale_base = out_base + kStageOut;
  const uint32_t bar_base = scale_base + C::kSlots * C::kSlotBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * kStages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * kStages + kBuf + b); };
  auto sfull_bar = [&](int s) { return bar_base + 8u * (2 * kStages + 2 * kBuf + s); };
  auto sempty_bar = [&](int s) { return bar_base + 8u * (2 * kStages + 2 * kBuf + C::kSlots + s); };
  const uint32_t drain_bar = bar_base + 8u * (2 * kStages + 2 * kBuf + 2 * C::kSlots);
  float* const s_scale = reinterpret_cast<float*>(smem_raw + (scale_base - smem_u32(smem_raw)));   // [slot][4][kColBlocks][128]
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // the same in all lanes, and known to be
  const uint32_t rank = cluster_ctarank();              // 0 = leader (issues the MMAs), 1 = peer
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int total = p.tiles_m * p.tiles_n, num_kb = p.kb;

  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < kBuf; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), 2 * kEpiWarps); }
    for (int s = 0; s < C::kSlots; ++s) { mbar_init(sfull_bar(s), 2); mbar_init(sempty_bar(s), kEpiWarps); }
    mbar_init(drain_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    if (p.tma_store) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_out)) : "memory");
  }
  if (warp == 1) tmem_alloc2(smem_u32(&s_tmem_base), kTmemCols);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                   // both CTAs' barriers exist before anyone signals across
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, s_tmem_base, 0);
  volatile int* abort_flag = &s_abort;
  b2q_pdl_entry();                                      // everything above may overlap the previous kernel of the stream

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsFirst));
    if (warp == 0) {
      // ---------------- TMA producer (both CTAs): own rows of A, own half of W; all bytes land on the leader's barrier ----------------
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int u = pair; u < total && ok; u += num_pairs) {
          int mb, nb;
          tile_coords(u, p, mb, nb);
          for (int kb = 0; kb < num_kb; ++kb, ++it) {
            const int s = it % kStages;
            if (!mbar_wait(empty_bar(s), ((it / kStages) & 1) ^ 1, abort_flag)) { ok = false; break; }
            const uint32_t sa = base + s * C::kStageBytes, sb = sa + C::kBytesA;
            const uint32_t leader_full = mapa_u32(full_bar(s), 0);
            if (rank == 0) mbar_expect_tx(full_bar(s), 2u * C::kStageBytes);
            tma_load_2d_pair(sa, &map_a, leader_full, kb * BK, mb * 256 + (int)rank * BM);
            tma_load_2d_pair(sb, &map_w, leader_full, kb * BK, nb * BN + (int)rank * (BN / 2));
          }
        }
        if (!ok) {   // give copies already issued time to land before shared memory is released
          const uint64_t t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 1000000ull) {}
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer (leader CTA only): one accumulator per block of K ----------------
      // The warp stays together and elects a lane for the products of a block: descriptors then live in uniform registers.
      if (rank == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int u = pair; u < total && ok; u += num_pairs) {
          for (int kb = 0; kb < num_kb; ++kb, ++it) {
            const int s = it % kStages, b = it % kBuf;
            ok = warp_wait(tempty_bar(b), ((it / kBuf) & 1) ^ 1, abort_flag) && warp_wait(full_bar(s), (it / kStages) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t sa = base + s * C::kStageBytes;
              const uint64_t adesc = make_desc_sw128(sa), bdesc = make_desc_sw128(sa + C::kBytesA);
#pragma unroll
              for (int k = 0; k < 4; ++k)                   // K advance inside the swizzle atom: +32 bytes
                umma_pair(tmem_base + b * BN, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), p.idesc, (uint32_t)(k != 0));
              tc_commit_pair(empty_bar(s));
              tc_commit_pair(tfull_bar(b));
            }
            __syncwarp();
          }
        }
        if (!ok && elect_one()) {
          tc_commit(drain_bar);
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(drain_bar, 0))
            if (globaltimer_ns() - t0 > 100000000ull) break;
        }
      }
    } else {
      // ---------------- scales: a row's scales lie far from the next row's, so each read takes an L2 round trip per row; these two
      // warps run up to three slots ahead of the epilogue and hand it one product per (row, 128 columns, block) ----------------
      const int r0 = (int)threadIdx.x - 64;               // this thread's rows: r0 and r0 + 64
      uint32_t it = 0;
      bool ok = true;
      for (int u = pair; u < total && ok; u += num_pairs) {
        int mb, nb;
        tile_coords(u, p, mb, nb);
        const int64_t m0 = (int64_t)mb * 256 + rank * BM + r0;
        const float* sa0 = p.sa + (m0 < p.M ? m0 : 0) * num_kb;          // rows and columns outside: their products are zeros
        const float* sa1 = p.sa + (m0 + 64 < p.M ? m0 + 64 : 0) * num_kb;
        const float* sw[C::kColBlocks];
#pragma unroll
        for (int c = 0; c < C::kColBlocks; ++c) sw[c] = p.sw + (int64_t)min(nb * C::kColBlocks + c, p.col_blocks - 1) * num_kb;
        for (int k0 = 0; k0 < num_kb; k0 += 4, ++it) {
          const float4 a0 = load4(sa0, k0, num_kb, p.vec), a1 = load4(sa1, k0, num_kb, p.vec);
          const int s = it % C::kSlots;
          float4 w4[C::kColBlocks];
#pragma unroll
          for (int c = 0; c < C::kColBlocks; ++c) w4[c] = load4(sw[c], k0, num_kb, p.vec);
          if (!warp_wait(sempty_bar(s), ((it / C::kSlots) & 1) ^ 1, abort_flag)) { ok = false; break; }
          float* d = s_scale + s * (C::kSlotBytes / 4) + r0;
#pragma unroll
          for (int c = 0; c < C::kColBlocks; ++c) {
            constexpr int kStep = C::kColBlocks * BM;     // from one block of K to the next
            d[0 * kStep + c * BM] = a0.x * w4[c].x; d[0 * kStep + c * BM + 64] = a1.x * w4[c].x;
            d[1 * kStep + c * BM] = a0.y * w4[c].y; d[1 * kStep + c * BM + 64] = a1.y * w4[c].y;
            d[2 * kStep + c * BM] = a0.z * w4[c].z; d[2 * kStep + c * BM + 64] = a1.z * w4[c].z;
            d[3 * kStep + c * BM] = a0.w * w4[c].w; d[3 * kStep + c * BM + 64] = a1.w * w4[c].w;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sfull_bar(s));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    // ---------------- epilogue (8 warps in each CTA): warp w has TMEM lane quarter w & 3, column half w / 4 - 1 ----------------
    constexpr int HALF = BN / 2, NACC = HALF / 2;
    const int q = warp & 3, half = (warp >> 2) - 1;
    const uint32_t stage = out_base + (uint32_t)(warp - 4) * 4096u;
    uint8_t* stage_p = smem_raw + (stage - smem_u32(smem_raw));
    uint32_t it = 0, sit = 0;
    bool ok = true;
    for (int u = pair; u < total && ok; u += num_pairs) {
      int mb, nb;
      tile_coords(u, p, mb, nb);
      const int64_t m_warp0 = (int64_t)mb * 256 + rank * BM + q * 32;
      const int64_t n0 = (int64_t)nb * BN + half * HALF;
      uint64_t acc[NACC];
#pragma unroll
      for (int j = 0; j < NACC; ++j) acc[j] = 0;
      const float* my_scale = s_scale + (BN == 256 ? half * BM : 0) + q * 32 + lane;
      for (int kb = 0; kb < num_kb; ++kb, ++it) {
        const int b = it % kBuf, slot = sit % C::kSlots;
        if ((kb & 3) == 0 && !warp_wait(sfull_bar(slot), (sit / C::kSlots) & 1, abort_flag)) { ok = false; break; }
        if (!warp_wait(tfull_bar(b), (it / kBuf) & 1, abort_flag)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        const uint32_t t = tmem_base + b * BN + half * HALF + ((uint32_t)(q * 32) << 16);
        const uint32_t c = __float_as_uint(my_scale[slot * (C::kSlotBytes / 4) + (kb & 3) * C::kColBlocks * BM]);
        const uint64_t cc = pack2(c, c);
#pragma unroll
        for (int x = 0; x < HALF; x += 16) {
          uint32_t r[16];
          tmem_ld16(t + x, r);
          tmem_ld_wait();
          if (x + 16 == HALF) {                           // the accumulator has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(mapa_u32(tempty_bar(b), 0));
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) fma2(acc[x / 2 + j], pack2(r[2 * j], r[2 * j + 1]), cc);
        }
        if ((kb & 3) == 3 || kb + 1 == num_kb) {
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty_bar(slot));
          ++sit;
        }
      }
      if (!ok || m_warp0 >= p.M || n0 >= p.N) continue;                // nothing of this warp's block lies inside the output
      if (p.tma_store) {
        const bool bf16 = p.out_type == B2Q_OUT_BF16;
        uint8_t* row = stage_p + lane * 128;
        if (bf16) {
#pragma unroll
          for (int x = 0; x < HALF; x += 64) {
            if (lane == 0) tma_store_wait_read<0>();                   // the store that last read this buffer has read it
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 64; j += 8) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint64_t v = acc[(x + j) / 2 + i];
                const __nv_bfloat162 h = __floats2bfloat162_rn(lo32(v), hi32(v));
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
              }
              *reinterpret_cast<uint4*>(row + (((j >> 3) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && n0 + x < p.N) { tma_store_2d(&map_out, stage, (int)(n0 + x), (int)m_warp0); tma_store_commit(); }
          }
        } else {
#pragma unroll
          for (int x = 0; x < HALF; x += 32) {
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const uint64_t v0 = acc[(x + j) / 2], v1 = acc[(x + j) / 2 + 1];
              *reinterpret_cast<float4*>(row + (((j >> 2) ^ (lane & 7)) << 4)) = make_float4(lo32(v0), hi32(v0), lo32(v1), hi32(v1));
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && n0 + x < p.N) { tma_store_2d(&map_out, stage, (int)(n0 + x), (int)m_warp0); tma_store_commit(); }
          }
        }
      } else {
        // Pitches that TMA cannot take: 32 x 32 results through the same buffer, then row by row, a column to a lane.  (2973 x 13158 x 608 in f32
        // takes 58 us; with a row to a lane, its stores scattered over 32 rows, it took 300.)
        uint8_t* const row = stage_p + lane * 128;
        const int rows = (int)(p.M - m_warp0 < 32 ? p.M - m_warp0 : 32);
#pragma unroll
        for (int x = 0; x < HALF; x += 32) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const uint64_t v0 = acc[(x + j) / 2], v1 = acc[(x + j) / 2 + 1];
            *reinterpret_cast<float4*>(row + (((j >> 2) ^ (lane & 7)) << 4)) = make_float4(lo32(v0), hi32(v0), lo32(v1), hi32(v1));
          }
          __syncwarp();
          const int64_t n = n0 + x + lane;
          if (n < p.N) {
#pragma unroll 4
            for (int i = 0; i < rows; ++i) {
              const float v = *reinterpret_cast<const float*>(stage_p + i * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4);
              const int64_t at = (m_warp0 + i) * p.N + n;
              if (p.out_type == B2Q_OUT_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
              else reinterpret_cast<float*>(p.out)[at] = v;
            }
          }
        }
      }
    }
    if (lane == 0) tma_store_wait<0>();                                // shared memory stays valid until the last store has read it
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                   // the peer's TMEM and barriers stay valid until both CTAs are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, kTmemCols);
  }
  if (threadIdx.x == 0 && s_abort) atomicCAS(p.status, 0, (int)B2Q_ERR_TIMEOUT);
}

template <int BN>
int32_t launch_pair(b2q_handle h, const uint8_t* a, const uint8_t* w, Params p, int fmt) {
  using C = Cfg<BN>;
  CUtensorMap map_a, map_w, map_out;
  int32_t st = b2q_tensor_map_2d(h, &map_a, a, 1, (uint64_t)p.K, (uint64_t)p.M, BK, BM);
  if (st != B2Q_OK) return st;
  st = b2q_tensor_map_2d(h, &map_w, w, 1, (uint64_t)p.K, (uint64_t)p.N, BK, BN / 2);
  if (st != B2Q_OK) return st;
  memset(&map_out, 0, sizeof(map_out));
  const int es = p.out_type == B2Q_OUT_BF16 ? 2 : 4;
  p.tma_store = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && (p.N * es) % 16 == 0;
  if (p.tma_store) {
    st = b2q_tensor_map_2d(h, &map_out, p.out, es, (uint64_t)p.N, (uint64_t)p.M, (uint32_t)(128 / es), 32u);
    if (st != B2Q_OK) return st;
  }
  p.tiles_m = (int)ceil_div64(p.M, 256);
  p.tiles_n = (int)ceil_div64(p.N, BN);
  p.col_blocks = (int)ceil_div64(p.N, 128);
  // a group's panel of A (group_m x 256 rows of K bytes) within about 48 MB of the 126 MB L2, at least 8 row tiles
  const int64_t fit = (48ll << 20) / (256 * p.K);
  p.group_m = (int)(fit < 8 ? 8 : fit > 64 ? 64 : fit);
  if (p.group_m > p.tiles_m) p.group_m = p.tiles_m;
  p.idesc = (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
  B2Q_SMEM_ATTR(h, gemm_block128_pair_kernel<BN>, C::kSmem);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  const int pairs = (int)(tiles < h->sm_count / 2 ? tiles : h->sm_count / 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = h->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = h->sw.chain_pdl != 0 ? 2 : 1;
  B2Q_CUDA(h, cudaLaunchKernelEx(&cfg, gemm_block128_pair_kernel<BN>, map_a, map_w, map_out, p));
  return B2Q_OK;
}

}  // namespace b128

int32_t b2q_gemm_fp8_block128_few(b2q_handle h, const uint8_t* a, const uint8_t* w, int64_t M, int64_t N, int64_t K, int fmt, const float* scale_a,
                                  const float* scale_w, void* out, int out_type);

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
  const int64_t tiles256 = ceil_div64(M, 256) * ceil_div64(N, 256);
  if (K % 16 == 0 && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(w)) & 15) == 0 && tiles256 < (1 << 29)) {
    b128::Params p{};
    p.M = M; p.N = N; p.K = K; p.kb = (int)kb;
    p.sa = scale_a; p.sw = scale_w; p.out = out;
    p.vec = kb % 4 == 0 && ((reinterpret_cast<uintptr_t>(scale_a) | reinterpret_cast<uintptr_t>(scale_w)) & 15) == 0;
    p.out_type = out_type; p.status = h->d_status;
    // up to 128 tokens W is what has to move: 65 x 4096 x 4096 11.1 us there against 14.4 here, 100 x 10240 x 8192 32 against 38
    if (M <= 128) return b2q_gemm_fp8_block128_few(h, a, w, M, N, K, fmt, scale_a, scale_w, out, out_type);
    // The tile width that needs less time for its waves over the CTA pairs, a wave of 128-wide tiles taking 0.62 of a wave of 256-wide ones.
    // Measured, 128-wide against 256-wide: 256 x 4096 x 4096 12.7 and 18.2 us (1 wave each), 512 x 8192 x 8192 40.1 and 35.3 (2 and 1),
    // 2048 x 8192 x 8192 139.1 and 127.8 (7 and 4), 700 x 4096 x 14336 63.5 and 54.0 (2 and 1).
    const int64_t pairs = h->sm_count / 2, tiles128 = ceil_div64(M, 256) * ceil_div64(N, 128);
    const bool wide = ceil_div64(tiles256, pairs) * 100 <= ceil_div64(tiles128, pairs) * 62;
    return wide ? b128::launch_pair<256>(h, a, w, p, fmt) : b128::launch_pair<128>(h, a, w, p, fmt);
  }
  const int64_t gy = ceil_div64(M, b128::T);
  dim3 grid((unsigned)ceil_div64(N, b128::T), (unsigned)(gy < 32768 ? gy : 32768));
  b128::gemm_fp8_block128_simt_kernel<<<grid, dim3(b128::T, b128::T), 0, h->stream>>>(a, w, M, N, K, fmt, scale_a, scale_w, out, out_type);
  B2Q_LAUNCH_CHECK(h, "gemm_fp8_block128_simt_kernel");
  return B2Q_OK;
}

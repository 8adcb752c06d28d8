// The block-128 FP8 product for few tokens (M <= 128): out[m, n] = sum_b sa[m, b] * sw[n / 128, b] * sum_{k in block b} A[m, k] * W[n, k].
// The work is reading W once, so W is the M = 128 operand of tcgen05.mma.kind::f8f6f4 (a tile of 128 weight rows is exactly one row of
// scale blocks: one sw per block of K) and the tokens, padded to NB columns, are the N operand.
//   * A CTA takes one weight tile and a range of K; `split` CTAs of a cluster share a tile and are joined through distributed shared
//     memory in rank order: no workspace, no counters, deterministic, and independent of what other streams run.
//   * Each block of 128 along K is a fresh TMEM accumulator; a thread owns one weight row and adds scale * product for its NB tokens
//     to sums in registers.
//   * Two CTAs share an SM up to 64 tokens, so that one streams weights while the other starts or ends (a ring of about 100 KiB each).
//   * Programmatic dependent launch: with static weights the weight copies start before the previous kernel of the stream has ended.
// Bound by HBM.  Measured back to back over rotating weights: 16 x 8192 x 28672 38 us (6.1 TB/s), 64 x 8192 x 28672 42 us (5.7), 53 x 10240 x 8192
// 20.4 us (4.2: 240 CTAs on 148 SMs, some with one of them and some with two), 1 x 14336 x 4096 13.1 us (4.5: 224 CTAs, launch and ramp).
// Every mbarrier wait is bounded; on expiry the kernel records B2Q_ERR_TIMEOUT and leaves.
#include "tc_common.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace b128few {

constexpr int ROWS = 128, BK = 128;
constexpr uint64_t kWaitLimitNs = 500000000ull;      // counted from the previous kernel's end

template <int NB> struct Cfg {           // NB: accumulator columns = padded tokens
  static constexpr int kBytesW = ROWS * BK, kBytesX = NB * BK, kStageBytes = kBytesW + kBytesX;
  // warp 0 TMA, warp 1 MMA, warps 2 and 3 scales, warps 4.. epilogue: four per kCols columns
  static constexpr int kCols = NB >= 64 ? NB / 2 : NB, kEpiWarps = 4 * NB / kCols, kThreads = 128 + 32 * kEpiWarps;
  static constexpr int kCtas = NB == 128 ? 1 : 2;                       // per SM
  static constexpr int kStages = NB <= 32 ? 5 : NB == 64 ? 4 : 6;
  static constexpr int kBuf = 4;                       // accumulators in flight
  static constexpr int kTmemCols = kBuf * NB;
  static constexpr int kSlots = 3, kSlotBytes = 4 * NB * 4;             // scales: slots of four blocks of K
  static constexpr int kSmem = kStages * kStageBytes + kSlots * kSlotBytes + 1024 + 256;
  static_assert(ROWS * NB * 4 <= kStages * kStageBytes, "the join reuses the stages");
};

struct Params {
  int64_t N;
  int tokens, kb;
  uint32_t idesc;
  const float* sa; const float* sw;
  void* out; int out_type;
  int wait_first;
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
__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

template <int NB>
__global__ void __launch_bounds__(Cfg<NB>::kThreads, Cfg<NB>::kCtas)
gemm_block128_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const Params p) {
  using C = Cfg<NB>;
  constexpr int kStages = C::kStages, kBuf = C::kBuf;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t scale_base = base + kStages * C::kStageBytes;
  const uint32_t bar_base = scale_base + C::kSlots * C::kSlotBytes;
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto tfull_bar = [&](int b) { return bar_base + 8u * (2 * kStages + b); };
  auto tempty_bar = [&](int b) { return bar_base + 8u * (2 * kStages + kBuf + b); };
  auto sfull_bar = [&](int s) { return bar_base + 8u * (2 * kStages + 2 * kBuf + s); };
  auto sempty_bar = [&](int s) { return bar_base + 8u * (2 * kStages + 2 * kBuf + C::kSlots + s); };
  const uint32_t drain_bar = bar_base + 8u * (2 * kStages + 2 * kBuf + 2 * C::kSlots);
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  float* const s_scale = reinterpret_cast<float*>(smem + kStages * C::kStageBytes);      // [slot][4][NB]
  __shared__ uint32_t s_tmem_base;
  __shared__ int s_abort;

  cg::cluster_group cluster = cg::this_cluster();
  const int split = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;   // the same in all lanes, and known to be
  const int tile = (int)(blockIdx.x / split);
  const int k_begin = (int)((int64_t)p.kb * part / split), k_end = (int)((int64_t)p.kb * (part + 1) / split), total = k_end - k_begin;

  if (p.wait_first) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (threadIdx.x == 0) {
    s_abort = 0;
    for (int s = 0; s < kStages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
    for (int b = 0; b < kBuf; ++b) { mbar_init(tfull_bar(b), 1); mbar_init(tempty_bar(b), C::kEpiWarps); }
    for (int s = 0; s < C::kSlots; ++s) { mbar_init(sfull_bar(s), 2); mbar_init(sempty_bar(s), C::kEpiWarps); }
    mbar_init(drain_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
    for (int it = 0; it < kStages && it < total; ++it) {                // the first round of weights needs nothing but the barriers
      mbar_expect_tx(full_bar(it), C::kStageBytes);
      tma_load_2d(base + it * C::kStageBytes, &map_w, full_bar(it), (k_begin + it) * BK, tile * ROWS);
    }
  }
  if (warp == 1) tmem_alloc(smem_u32(&s_tmem_base), C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, s_tmem_base, 0);
  volatile int* abort_flag = &s_abort;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // Every thread waits for the previous kernel here: it may still be reading what this one stores, and no bounded wait counts its time.
  asm volatile("griddepcontrol.wait;" ::: "memory");

  constexpr int COLS = C::kCols, NACC = COLS / 2;
  const int col0 = warp >= 4 ? ((warp >> 2) - 1) * COLS : 0;           // the epilogue thread's tokens
  uint64_t acc[NACC];
#pragma unroll
  for (int j = 0; j < NACC; ++j) acc[j] = 0;
  bool ok = true;                                      // false: this warp has given up a wait

  if (warp == 0) {
    // ---------------- TMA: weights and activations (rows past the last token are zero-filled) ----------------
    if (lane == 0) {
      for (int it = 0; it < total; ++it) {
        const int s = it % kStages, x = (k_begin + it) * BK;
        const uint32_t at = base + s * C::kStageBytes;
        if (it >= kStages) {
          if (!mbar_wait(empty_bar(s), ((it / kStages) & 1) ^ 1, abort_flag)) { ok = false; break; }
          mbar_expect_tx(full_bar(s), C::kStageBytes);
          tma_load_2d(at, &map_w, full_bar(s), x, tile * ROWS);
        }
        tma_load_2d(at + C::kBytesW, &map_a, full_bar(s), x, 0);
      }
      if (!ok || *abort_flag) {   // give copies in flight time to land before shared memory is released
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {}
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer: one accumulator per block of K; the warp stays together and elects a lane (descriptors in uniform registers) ----------------
    for (int it = 0; it < total; ++it) {
      const int s = it % kStages, b = it % kBuf;
      ok = warp_wait(tempty_bar(b), ((it / kBuf) & 1) ^ 1, abort_flag) && warp_wait(full_bar(s), (it / kStages) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t sw = base + s * C::kStageBytes;
        const uint64_t adesc = make_desc_sw128(sw), bdesc = make_desc_sw128(sw + C::kBytesW);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f8(tmem_base + b * NB, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), p.idesc, (uint32_t)(k != 0));
        tc_commit(empty_bar(s));
        tc_commit(tfull_bar(b));
      }
      __syncwarp();
    }
    if (!ok && elect_one()) {
      tc_commit(drain_bar);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain_bar, 0))
        if (globaltimer_ns() - t0 > 100000000ull) break;
    }
  } else if (warp < 4) {
    // ---------------- scales: scale_a * scale_w of each token, four blocks of K at a time ----------------
    constexpr int PER = NB > 64 ? 2 : 1;
    const int t0 = (int)threadIdx.x - 64;
    const float* sw = p.sw + (int64_t)tile * p.kb;
    for (int k0 = 0, i = 0; k0 < total; k0 += 4, ++i) {
      const int s = i % C::kSlots;
      float v[PER][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k_begin + k0 + j;
        const float w = k < k_end ? __ldg(sw + k) : 0.0f;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          const int t = t0 + 64 * e;
          v[e][j] = k < k_end && t < p.tokens ? __ldg(p.sa + (int64_t)t * p.kb + k) * w : 0.0f;
        }
      }
      if (!warp_wait(sempty_bar(s), ((i / C::kSlots) & 1) ^ 1, abort_flag)) break;
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int t = t0 + 64 * e;
        if (t < NB)
#pragma unroll
          for (int j = 0; j < 4; ++j) s_scale[(s * 4 + j) * NB + t] = v[e][j];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull_bar(s));
    }
  } else {
    // ---------------- epilogue: this thread's weight row is TMEM lane 32 (warp & 3) + lane ----------------
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    for (int it = 0, i = 0; it < total; ++it) {
      const int b = it % kBuf, slot = i % C::kSlots;
      ok = ((it & 3) != 0 || warp_wait(sfull_bar(slot), (i / C::kSlots) & 1, abort_flag)) && warp_wait(tfull_bar(b), (it / kBuf) & 1, abort_flag);
      if (!ok) break;
      __syncwarp();
      tc_fence_after();
      const ulonglong2* c = reinterpret_cast<const ulonglong2*>(s_scale + (slot * 4 + (it & 3)) * NB + col0);   // every lane reads the same
#pragma unroll
      for (int x = 0; x < COLS; x += 16) {
        uint32_t r[16];
        tmem_ld16(tmem_base + b * NB + col0 + x + lanes, r);
        tmem_ld_wait();
        if (x + 16 == COLS) {                                            // the accumulator has been read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(tempty_bar(b));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const ulonglong2 cc = c[x / 4 + j];
          fma2(acc[x / 2 + 2 * j], (uint64_t)r[4 * j + 1] << 32 | r[4 * j], cc.x);
          fma2(acc[x / 2 + 2 * j + 1], (uint64_t)r[4 * j + 3] << 32 | r[4 * j + 2], cc.y);
        }
      }
      if ((it & 3) == 3 || it + 1 == total) {
        __syncwarp();
        if (lane == 0) mbar_arrive(sempty_bar(slot));
        ++i;
      }
    }
  }

  // ---------------- results ----------------
  const int row = warp >= 4 ? (warp & 3) * 32 + lane : -1;
  const int64_t n = (int64_t)tile * ROWS + row;
  auto store = [&](int t, int64_t at, float v) {
    if (p.out_type == B2Q_OUT_BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[(int64_t)t * p.N + at] = __float2bfloat16_rn(v);
    else reinterpret_cast<float*>(p.out)[(int64_t)t * p.N + at] = v;
  };
  if (split == 1) {
    if (row >= 0 && n < p.N && ok) {
#pragma unroll
      for (int t = 0; t < COLS; ++t)
        if (col0 + t < p.tokens) store(col0 + t, n, __uint_as_float((uint32_t)(acc[t / 2] >> (32 * (t & 1)))));
    }
  } else {
    __syncthreads();                                                     // every copy of this CTA has landed and been multiplied: the stages are free
    float* const mine = reinterpret_cast<float*>(smem);                  // [NB][128]
    if (row >= 0) {
#pragma unroll
      for (int t = 0; t < COLS; ++t)
        if (col0 + t < p.tokens) mine[(col0 + t) * ROWS + row] = __uint_as_float((uint32_t)(acc[t / 2] >> (32 * (t & 1))));
    }
    cluster.sync();
    // this CTA joins tokens part, part + split, ...: 128 threads to a token
    const int64_t n2 = (int64_t)tile * ROWS + (threadIdx.x & 127);
    for (int t = part + split * (int)(threadIdx.x >> 7); t < p.tokens; t += split * (C::kThreads / 128)) {
      float v = 0.0f;
      for (int c = 0; c < split; ++c) v += *cluster.map_shared_rank(mine + t * ROWS + (threadIdx.x & 127), c);
      if (n2 < p.N) store(t, n2, v);
    }
    cluster.sync();                                                      // the others may still be reading this CTA's sums
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
  if (threadIdx.x == 0 && s_abort) atomicCAS(p.status, 0, (int)B2Q_ERR_TIMEOUT);
}

template <int NB>
int32_t launch(b2q_handle h, const uint8_t* a, const uint8_t* w, int64_t K, Params p, int fmt) {
  using C = Cfg<NB>;
  CUtensorMap map_w, map_a;
  int32_t st = b2q_tensor_map_2d(h, &map_w, w, 1, (uint64_t)K, (uint64_t)p.N, BK, ROWS);
  if (st != B2Q_OK) return st;
  st = b2q_tensor_map_2d(h, &map_a, a, 1, (uint64_t)K, (uint64_t)p.tokens, BK, NB);
  if (st != B2Q_OK) return st;
  p.idesc = (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)(NB >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
  const int64_t tiles = ceil_div64(p.N, ROWS);
  // As many CTAs per tile as still find a place at once, each with four blocks of K at least.  Measured, us by the number of CTAs (taken: *):
  // 1 x 14336 x 4096 1: 13.3, 2: 12.6*, 3: 16.3;  53 x 10240 x 8192 2: 23.1, 3: 19.6*, 4: 25.8;  64 x 8192 x 28672 1: 79, 3: 46, 4: 41*, 5: 56;
  // 1 x 4096 x 14336 1: 29, 4: 13.4, 8: 11.9*;  128 x 10240 x 8192 1: 29.4*, 2: 42.4.
  int64_t split = C::kCtas * (int64_t)h->sm_count / tiles;
  if (split > p.kb / 4) split = p.kb / 4;
  split = split < 1 ? 1 : split > 8 ? 8 : split;
  B2Q_SMEM_ATTR(h, gemm_block128_few_kernel<NB>, C::kSmem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(C::kThreads);
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
  B2Q_CUDA(h, cudaLaunchKernelEx(&cfg, gemm_block128_few_kernel<NB>, map_w, map_a, p));
  return B2Q_OK;
}

}  // namespace b128few

// M <= 128 tokens; the caller has checked the arguments, K % 16 == 0 and the operands' alignment.
int32_t b2q_gemm_fp8_block128_few(b2q_handle h, const uint8_t* a, const uint8_t* w, int64_t M, int64_t N, int64_t K, int fmt, const float* scale_a,
                                  const float* scale_w, void* out, int out_type) {
  b128few::Params p{};
  p.N = N; p.tokens = (int)M; p.kb = (int)ceil_div64(K, 128);
  p.sa = scale_a; p.sw = scale_w; p.out = out; p.out_type = out_type;
  p.wait_first = h->dynamic_weights;
  p.status = h->d_status;
  if (M <= 16) return b128few::launch<16>(h, a, w, K, p, fmt);
  if (M <= 32) return b128few::launch<32>(h, a, w, K, p, fmt);
  if (M <= 64) return b128few::launch<64>(h, a, w, K, p, fmt);
  return b128few::launch<128>(h, a, w, K, p, fmt);
}

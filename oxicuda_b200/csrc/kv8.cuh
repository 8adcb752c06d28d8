// The paged 8-bit KV cache shared by its append and attention kernels.
//   codes  E4M3, [num_pages][n_kv_heads][page_size][head_dim]: the tokens of one page and head are one contiguous tile
//   scales E8M0 bytes, [num_pages][n_kv_heads]: value = code * 2^(byte - 127), one scale for the page_size x head_dim tile
// A sequence's token at position p lies in page table[p / page_size], slot p % page_size.
#pragma once

#include "common.cuh"

namespace kv8 {

struct Batch {                      // which rows and which cached tokens belong to which sequence
  const int32_t* q_starts;          // [seqs + 1] row offsets of the new tokens, or null: sequence b has row b and no other
  const int32_t* seq_lens;          // [seqs] cached tokens, the new ones included
  const int32_t* table;             // [seqs][table_width]
  int seqs, table_width, tokens;
  int64_t num_pages;
  int page_shift, n_kv_heads;
  int32_t* status;
};

__device__ __forceinline__ void report(int32_t* status, int code) { atomicCAS(status, 0, code); }

struct Rows { int r0, n, len; };    // first row, new tokens, cached tokens
// The rows of sequence b; an impossible entry (offsets that run backwards or out of the rows, fewer cached tokens than new
// ones, more than the table holds) counts as no rows, and is reported.
__device__ __forceinline__ Rows rows_of(const Batch& t, int b, bool tell) {
  Rows r;
  r.r0 = t.q_starts ? t.q_starts[b] : b;
  r.n = t.q_starts ? t.q_starts[b + 1] - r.r0 : 1;
  r.len = t.seq_lens[b];
  const bool ok = r.r0 >= 0 && r.n >= 0 && r.n <= t.tokens && r.r0 <= t.tokens - r.n && r.len >= r.n &&
                  (int64_t)r.len <= ((int64_t)t.table_width << t.page_shift);
  if (!ok) {
    if (tell) report(t.status, B2Q_ERR_INVALID_DIMENSION);
    r.n = 0; r.len = 0;
  }
  return r;
}
// page of the given index of a sequence, or -1 (reported) when the table names none
__device__ __forceinline__ int page_of(const Batch& t, int b, int index, bool tell) {
  const int pg = t.table[(int64_t)b * t.table_width + index];
  if (pg < 0 || pg >= t.num_pages) {
    if (tell) report(t.status, B2Q_ERR_INVALID_ARGUMENT);
    return -1;
  }
  return pg;
}

// Finds the unit'th item of a list in which sequence b has count(b) items, by a whole warp: {b, index within b, count(b)}, b = -1 past the
// end.  All counts of a possible batch fit 31 bits together; those of an impossible one may wrap, so the index is checked against its count.
struct Found { int b, index, count; };
template <typename F>
__device__ __forceinline__ Found find_unit(int seqs, int unit, F count) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < seqs; b0 += 32) {
    const int c = b0 + lane < seqs ? count(b0 + lane) : 0;
    int s = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, s > unit);
    if (hit) {
      const int src = __ffs(hit) - 1, at = __shfl_sync(0xffffffffu, unit - (s - c), src), n = __shfl_sync(0xffffffffu, c, src);
      return (unsigned)at < (unsigned)n ? Found{b0 + src, at, n} : Found{-1, 0, 0};
    }
    unit -= __shfl_sync(0xffffffffu, s, 31);
  }
  return Found{-1, 0, 0};
}

struct AttendArgs {
  Batch t;
  const __nv_bfloat16* q; int64_t ld_q;
  const uint8_t* k; const uint8_t* v; const uint8_t* ks; const uint8_t* vs;
  int group;                                     // query heads per kv head, at most 2^20
  float per_group;                               // 1 / group
  int window;                                    // 0: none
  float scale;                                   // softmax scale * log2(e)
  __nv_bfloat16* out; float* lse;                // [tokens][heads][head_dim], [tokens][heads]
};

// x / group and x % group for 0 <= x < 2^21: (x + 1/2) / group lies 1 / (2 group) off an integer at least, which the roundings do not reach
__device__ __forceinline__ int div_group(const AttendArgs& p, int x) { return (int)(((float)x + 0.5f) * p.per_group); }

__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(min(127, max(-126, e)) + 127) << 23); }
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// The unit of the outputs, 2^R.  Value codes are multiplied as they are stored, so a page's scale 2^lv enters with the f16 weights: a weight is
// p * 2^x, x = X + lv - R (X is the attention kernel's own), and outputs are summed in units of 2^(R - X).  R follows the pages: up when one lies above
// it (f16 must hold the weight), down when one lies more than 2^kSpan below it (x is X - kSpan at least: a weight is off by 2^-11 of itself or by
// 2^-(25 + x)), but by 2^kDrop at most below the largest unit so far.  What was summed in that unit is below 2^15 * 448 * 2^31 keys < 2^55 of it,
// so it stays below 2^119 in the smaller one.
constexpr int kNone = -1000;                     // R before the first page
constexpr int kSpan = 8, kDrop = 64;
// The weights of a page so far below R that f16 holds none of them: x is not less than this, so that their sum in f32 still counts them.
constexpr int kLeast = -40;
// what outputs are multiplied by when R moves: 2^(from - to), exact down to 2^-149 and 0 below (R may rise by 2^171)
__device__ __forceinline__ float move_unit(int from, int to) {
  const int d = max(from - to, -150);              // at most kDrop
  return __uint_as_float(d >= -126 ? (uint32_t)(d + 127) << 23 : (1u << (d + 150)) >> 1);
}
// R for pages whose value scales lie from 2^least to 2^lead, lead + room - least at most kSpan; `top` is the largest R so far.  Returns what outputs are
// to be multiplied by.
__device__ __forceinline__ float next_unit(int& R, int& top, int lead, int least, int room) {
  if (lead <= R && least >= R - kSpan) return 1.0f;
  const int was = R;
  R = lead > R ? lead + room : max(lead + room, top - kDrop);
  top = max(top, R);
  return was == kNone ? 1.0f : move_unit(was, R);
}
__device__ __forceinline__ float pow2_byte(uint32_t e8m0) { return e8m0_to_f32_dev(e8m0); }

}  // namespace kv8

// The checks of a batch that append and attention share (kv8_append.cu).
int32_t b2q_kv8_batch(b2q_handle h, const char* who, int64_t tokens, const int32_t* q_starts, const int32_t* seq_lens, const int32_t* block_tables,
                      int64_t seqs, int64_t table_width, int64_t num_pages, int64_t page_size, int64_t n_kv_heads, int64_t head_dim, kv8::Batch* out);

// Paged KV cache: what the append and attention kernels share.
//
// A sequence's cache is a list of page ids (a row of the page table) into one
// pool; position i is slot i % page_size of page i / page_size.  One key (or
// value) of one kv head is head_dim contiguous elements; pages, slots and kv
// heads have strides of their own.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include <float.h>

#include "async.cuh"
#include "common.cuh"
#include "share.cuh"

namespace q6w {
namespace paged {

constexpr int32_t kErrInput = 1;    // status bit 0: rejected input (a length, a page id, a position)
constexpr int32_t kErrTimeout = 4;  // status bit 2: a bounded wait ran out

struct Batch {
  void* k;
  void* v;
  int64_t page_stride, slot_stride, head_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* starts;
  int32_t* status;
  int32_t n, T, n_pages, shift, max_len, kv_heads, rep;
};

__device__ __forceinline__ void flag(int32_t* status, int32_t bit) {
  if (status) atomicOr(status, bit);
}

// Tokens that sequence s claims (the step's own included), never negative.  A
// length that its page-table row cannot hold is flagged; positions from
// max_len on do not exist.
__device__ __forceinline__ int seq_length(const Batch& b, int s) {
  const int len = __ldg(b.lengths + s);
  if (len > b.max_len) flag(b.status, kErrInput);
  return max(len, 0);
}

// First and one-past-last query token of sequence s, kept inside [0, T].
__device__ __forceinline__ void seq_tokens(const Batch& b, int s, int& t0, int& t1) {
  if (!b.starts) {
    t0 = s;
    t1 = s + 1;
    return;
  }
  t0 = min(max(__ldg(b.starts + s), 0), b.T);
  t1 = min(max(__ldg(b.starts + s + 1), t0), b.T);
}

// Flags starts of sequence s that descend or leave [0, T].
__device__ __forceinline__ void check_tokens(const Batch& b, int s) {
  const int t0 = __ldg(b.starts + s), t1 = __ldg(b.starts + s + 1);
  if (t0 < 0 || t1 < t0 || t1 > b.T) flag(b.status, kErrInput);
}

// Sequence of query token t, by the whole warp (all lanes the same t): the
// last s with starts[s] <= t, found 32-fold a round.  -1 or n: no sequence.
__device__ __forceinline__ int token_seq(const Batch& b, int t, int lane) {
  if (!b.starts) return t;
  int lo = 0, hi = b.n + 1;  // starts[i] <= t for i < lo; starts[i] > t for i >= hi
  while (lo < hi) {
    const int step = (hi - lo + 31) >> 5;
    const int i = lo + lane * step;
    const bool le = i < hi && __ldg(b.starts + i) <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    if (c == 0) {
      hi = lo;
    } else {
      hi = min(hi, lo + c * step);
      lo += (c - 1) * step + 1;
    }
  }
  return lo - 1;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The FP16 parts of a row x of queries (FP16 pages) are those of x 2^e with the
// largest element in [2^14, 2^15): elements down to 2^-17 of it keep 22 bits, as
// their low parts are then normal FP16 numbers; smaller ones err by 2^-39 of the
// largest.  Returns 2^e; back becomes 2^-e.
__device__ __forceinline__ float half_scale(float largest, float& back) {
  const int ex = min(max((int)(__float_as_uint(largest) >> 23), 15), 254);
  back = __uint_as_float((uint32_t)(ex - 14) << 23);
  return __uint_as_float((uint32_t)(268 - ex) << 23);
}
// Weights are 2^(s - m), m a reference that starts kFirst below the first maximum
// and moves when a score passes it by more than kLimit, so that the largest weight
// lies in [2^kFirst, 2^kLimit].  FP16 parts: close under FP16's largest number
// (65504 > 2^15.9), so that weights down to 2^-(kFirst + 3) of the largest keep 22
// bits (their low parts are normal numbers) and smaller ones err by 2^-(kFirst + 25)
// of it at most -- many small weights may outweigh a sink whose value is 0.  FIRST
// nearer to kLimit moves the reference more often.  FP32 pages: weights of at most 1,
// so that values up to FP32's largest do not overflow where their mean does not.  The
// exponent s - m is rounded to 24 bits of its own size, so a kFirst far from 0 costs the
// largest weights precision: errors of 8192 short FP32 requests 2.5e-7 with 0, 2.6e-7
// with -4, 2.8e-7 with -8.
template <bool HALF, int FIRST>
struct Weights {
  static constexpr float kFirst = HALF ? FIRST : -4;
  static constexpr float kLimit = HALF ? 15.9f : 0.f;
};
// A row's reference while it has seen no score.  (Weights behind it are 0: their
// scores are -inf.)
constexpr float kUnseen = -FLT_MAX;
// A maximum to subtract: nothing seen yet counts as 0, so that the weights are 2^-inf = 0.
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

// The state of one query row over keys [key0, key1) of kv head kv in FP32, one product
// after the other, by a warp (lane: dims lane, lane + 32, ..): for rows whose sum of weights
// is not a number.  In the MMAs that may be the doing of the operands' parts (inf - inf),
// of another kv head's key (times zeros) or of a key marked for its value; here a
// score is its own, and one of -inf is a weight of 0.  Ends where nothing but NaN can follow,
// a page out of range among it.
template <typename KT>
__device__ __forceinline__ void plain_row(const Batch& b, const int32_t* table, const float* q, int hd, int kv, int key0,
                                          int key1, float scale, float& m, float& l, float (&o)[4]) {
  const int lane = threadIdx.x & 31;
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = 0.f;
#pragma unroll 1
  for (int key = key0; key < key1; ++key) {
    const int id = __ldg(table + (key >> b.shift));
    if ((unsigned)id >= (unsigned)b.n_pages) {
      l = NAN;
      return;
    }
    const int64_t at = id * b.page_stride + (key & ((1 << b.shift) - 1)) * b.slot_stride + kv * b.head_stride + lane;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < hd) x = fmaf(__ldg(q + lane + 32 * e), (float)static_cast<const KT*>(b.k)[at + 32 * e], x);
#pragma unroll
    for (int i = 16; i; i >>= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
    x *= scale;
    const bool up = x > m;
    const float f = up ? ex2(m - x) : 1.f;
    if (up) m = x;
    const float p = ex2(x - ref_of(m));
    l = fmaf(l, f, p);
    bool nan = true;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < hd) {
        o[e] = fmaf(p, (float)static_cast<const KT*>(b.v)[at + 32 * e], o[e] * f);
        nan = nan && o[e] != o[e];
      }
    if (l != l || __all_sync(0xffffffffu, nan)) {
      l = NAN;
      return;
    }
  }
}

// The pool's tensor map (paged_decode.cu).
int32_t pool_map(const Batch& b, void* pool, int hd, int es, int F, int rows, int segments, CUtensorMap* map,
                 bool* swap);

// ---- decode attention (paged_decode.cu) -------------------------------------

struct DecodeArgs {
  Batch b;
  const float* q;
  int64_t ldq;
  float* out;
  float* state;     // [row][m, l], or null; with it `out` takes the unnormalised outputs
  float* wpart;     // [warp of the grid][2][state]: pieces of items
  float* part;      // [CTA][2][state]: pieces joined inside a CTA
  int4* desc;       // [CTA]: item that starts in the CTA and goes on: {s, block, CTAs, 0}
  int32_t H, HB, per;  // query heads, head blocks of a kv head, heads of a block
  int32_t hd, F;       // head_dim, kv heads side by side
  int32_t swap;        // the pool's map holds slots in front of kv heads
  float scale;         // log2(e) / sqrt(head_dim)
  int32_t stall;       // the first CTA's first tiles never arrive (q6w_selftest_paged_stall)
  int64_t wait_cycles; // bound of a wait
};

// One query token a sequence; workspace (desc): decode_workspace bytes.
int32_t decode_attention(const DecodeArgs& a, bool half, cudaStream_t st);
size_t decode_workspace(int head_dim);

// ---- many rows over the same keys (paged_tc.cu) --------------------------------

struct TcArgs {
  Batch b;
  const float* q;
  int64_t ldq;
  float* out;
  float* state;      // [row][m, l], or null; with it `out` takes the unnormalised outputs
  float* part;       // pieces: outputs [..][head_dim]; own rows [CTA][2][block row], prefix [piece][item][block row]
  float* part_ml;    // pieces: [..][m, l]
  int4* desc;        // [CTA][2]: block that starts in the CTA and goes on: {first token, kv head, block, CTAs}, {rows}
  int64_t* line;     // [n + 1]: units of the sequences in front, one kv head's
  const int32_t* own_rows;  // the ragged batch's query_starts (prefix join), or null
  int32_t H, swap;
  int32_t prefix, prefix_len, items;  // over the prefix (its pages in b.table), blocks of all kv heads
  float scale;       // log2(e) / sqrt(head_dim)
  int32_t stall;     // as DecodeArgs
  int64_t wait_cycles;
};

struct TcMaps {
  CUtensorMap k, v;
};

int32_t rows_own(const TcArgs& a, int hd, bool half, cudaStream_t st);
int32_t rows_prefix(const TcArgs& a, int hd, bool half, cudaStream_t st);
int32_t rows_join(const TcArgs& a, int hd, bool half, cudaStream_t st);
size_t rows_own_rows(int hd, bool half);  // piece rows that rows_own / rows_prefix need
size_t rows_prefix_rows(const Batch& b, int prefix_len, int hd, bool half);
int32_t zero_padding_rows(const Batch& b, float* out, int row, cudaStream_t st);

}  // namespace paged
}  // namespace q6w

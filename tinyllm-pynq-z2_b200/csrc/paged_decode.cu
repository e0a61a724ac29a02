// Decode attention over paged caches: one query token a sequence.
//
// Mathematics.  One pass over the keys with a reference exponent m, a sum l and
// an output o per query head: p = 2^(s - m), l += p, o += p v; m follows the
// largest score so far (it moves only when a score passes it by a bound, Weights;
// then l and o are scaled by 2^(m_old - m_new)).  States of disjoint key
// ranges join as m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m).
//
// Bound.  Every key and value is read once from HBM and used by the query heads
// of its kv head.  FP32 lanes alone cannot keep up with that: dot products
// of keys spread over lanes cost a shuffle network a key (measured first: 35
// us for 67 MB, 231 us for 542 MB of FP16).  So the products run on the tensor
// cores as
//   S^T[16 keys, 8 heads] = K q^T   and   O^T[dims, 8 heads] += V^T P^T
// (m16n8): keys fill the M side, so eight query heads waste nothing, S and O
// have the same heads in a lane's registers (rescaling needs no exchange),
// and a lane can load its part of K and V straight from the cache.
//
// Precision.  FP16 keys and values are exact operands; queries (scaled by a
// power of two per head, half_scale) and weights enter as two FP16 parts, hi + lo,
// 22 bits.  FP32 keys, values, queries and weights enter as two TF32 parts and
// the products hi hi + hi lo + lo hi, dropping terms of 2^-22; the first part of a
// number above 2^128 (1 - 2^-12) rounds to infinity.  The MMA adds in FP32; a unit's
// output (16 or 32 keys) is added to o in registers, rounded to nearest, so no long
// sum lives in the MMA's accumulator.
//
// Narrow heads.  While heads of head_dim <= 32 lie side by side in a slot, F kv
// heads are treated as one of F head_dim dims: their queries stand block-
// diagonally, zero elsewhere, and of the F blocks of O each head keeps its own.
// A key's bytes of all F heads are then one contiguous read and the MMAs run
// at full width.
//
// Layout of the work.  An item is (sequence, F kv heads, block of up to eight
// query heads), cut into units of 16 keys (32 where rows have up to 128 bytes).  More
// than eight heads a kv head are items of their own that read the keys again (64
// requests of 128-8192 FP16 keys, heads of 64: 117 us with 8 a kv head, 197 with 16).
// The units of all items lie on one line (a prefix sum of the lengths, taken by every CTA for itself), and every
// warp takes an equal stretch of it: ragged lengths and few long sequences
// balance alike.  A warp that holds an item whole writes its output; pieces
// of an item go through the workspace, joined by their CTA when it holds them
// all, else by merge_kernel.
//
// Measured (joins included; ten calls in a graph, a call among others): 64 requests of
// 128-16384 keys, FP16, 8 heads a group of 64: 102-106 us for 542 MB, 5.1-5.3 TB/s; 37
// requests, FP32, 5 heads a group of 128: 82-85 us for 380 MB; 8192 requests of 20-147
// keys, FP32, heads of 16: 95-98 us for 357 MB, bound by instruction issue; one request of
// 32768 keys, FP32: 27-29 us for 67 MB, of which start-up and joins are about 15.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "paged.cuh"

namespace q6w {
namespace paged {

constexpr int kTile = 16;  // keys of an MMA's M side

// A partial state: o[8][head_dim], m[8], l[8].
__host__ __device__ constexpr int state_floats(int hd) { return 8 * hd + 16; }

// First query head and heads of an item's block.
__device__ __forceinline__ void block_heads(const DecodeArgs& a, int block, int& h0, int& nr) {
  const int kb = a.HB == 1 ? block : block / a.HB, hb = block - kb * a.HB;
  h0 = kb * a.F * a.b.rep + hb * a.per;
  nr = a.F > 1 ? a.F * a.b.rep : min(a.per, a.b.rep - hb * a.per);
}

// Shapes by the width HDF = F head_dim and the element size.
//
// Loads.  A tile (16 keys of one item: 16 rows of RB bytes) is one TMA box, or
// 16 / page_size boxes of smaller pages, into a ring that the warp owns,
// half units (keys, values, keys, ...) STG - 1 ahead of the arithmetic and
// over the ends of items.  Lane-wise 16-byte copies of the same rows stopped at
// 3.5 TB/s whatever the arithmetic (64- and 128-byte requests: the L1's
// outstanding requests run out); one bulk copy a row at one row in 9 cycles
// (4 TB/s at 128 bytes).
// Rows arrive swizzled in 16-byte units by min(RB, 128) bytes; kappa(g) is the
// key that stands in row g (g + 8: kappa(g) + 8) of the MMA's M side, chosen
// for each RB so that neither the reads of K (rows g by quarter-warps) nor
// those of V (rows of four lane columns) meet in a bank (RB 512: V two-way).
template <int HDF, typename KT>
struct DecodeShape {
  static constexpr int ES = (int)sizeof(KT);
  static constexpr int RB = HDF * ES;                               // bytes of a key's row
  static constexpr int IB = RB < 128 ? RB : 128;                    // inner box bytes = swizzle span
  static constexpr int CK = RB / 4 < 16 ? RB / 4 : 16;  // bytes of a lane's K chunk
  static constexpr int CV = RB / 8 < 16 ? RB / 8 : 16;
  static constexpr int NK = RB / 4 / CK;   // K chunks of a key that a lane holds (4 lanes a key)
  static constexpr int NVC = RB / 8 / CV;  // V chunks of a key that a lane holds (8 lanes a key)
  static constexpr int EK = CK / ES, EV = CV / ES;
  // Tiles of a unit: two where the registers allow it, so that the checks, the
  // joining of a tile's output and the loop itself are paid half as often.
  static constexpr int NT = RB <= 128 ? 2 : 1;
  static constexpr int KU = NT * kTile;  // keys of a unit
  static constexpr int TILE = kTile * RB;
  static constexpr int HALF = NT * TILE;  // bytes of a unit's keys (or values)
  // CTAs of four warps an SM, by registers (255, 168, 128 a thread); 192 KB of rings an SM
  static constexpr int CTAS = HDF >= 128 ? 2 : HDF >= 64 ? 3 : 4;
  static constexpr int kMost = 48 / CTAS * 1024 / HALF;
  static constexpr int STG = kMost < 8 ? kMost : 8;
  static constexpr int RING = STG * HALF;
  __device__ static __forceinline__ int kappa(int g) {
    if (ES == 2) {
      if (RB == 128) return g ^ ((g & 1) << 2);
      if (RB == 64) return ((g & 4) | ((g >> 1) & 1)) ^ ((g & 1) * 3);
      return (g >> 1) ^ ((g & 1) * 6);
    }
    if (RB == 64) return (g & 1) | ((g & 2) << 1) | ((g & 4) >> 1);
    if (RB == 128) return ((g & 1) << 2) | (g & 2) | ((g & 4) >> 2);
    if (RB == 256) return (g & 4) | ((g & 1) << 1) | ((g >> 1) & 1);
    return g;
  }
  // Byte place of byte `at` of row `row` of a tile.
  __device__ static __forceinline__ int place(int row, int at) {
    const int x = row * RB + at;
    return IB == 128 ? x ^ ((x >> 3) & 0x70) : IB == 64 ? x ^ ((x >> 3) & 0x30) : x ^ ((x >> 3) & 0x10);
  }
};

struct DecodeMaps {
  CUtensorMap k, v;
};

constexpr int kDecodeWarps = 4;
constexpr int kDecodeThreads = 32 * kDecodeWarps;

// The line of units: prefix sums over 128 stretches of sequences.
struct Line {
  int64_t pref[kDecodeThreads];
  int64_t total;
  int64_t warp_sum[kDecodeWarps];
};

// Sequences of a stretch.
__device__ __forceinline__ int stretch(int n) {
  return n <= kDecodeThreads ? 1 : ((n + kDecodeThreads - 1) / kDecodeThreads + 31) & ~31;
}

// Keys that sequence s's token sees.
__device__ __forceinline__ int keys_of(const Batch& b, int s) { return min(max(__ldg(b.lengths + s), 0), b.max_len); }

template <int KU>
__device__ __forceinline__ int units_of(int keys) {
  return max(1, (keys + KU - 1) / KU);
}

template <int KU>
__device__ __forceinline__ void build_line(const Batch& b, Line& line) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seg = stretch(b.n);
  int64_t sum = 0;
  bool over = false;
  auto units_at = [&](int len) {
    over |= len > b.max_len;
    return units_of<KU>(min(max(len, 0), b.max_len));
  };
  if (seg == 1) {
    if (tid < b.n) sum = units_at(__ldg(b.lengths + tid));
  } else {
    // a stretch is a number of 32-sequence rows: a coalesced load and a warp-wide
    // addition each (a sequence has fewer than 2^27 units), eight loads in flight
    const int per = seg >> 5;
    const int64_t first = (int64_t)warp * 32 * seg;
    for (int g = 0; g < 32 * per && first + g * 32 < b.n; g += 8) {
      int len[8];
      bool in[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t s = first + (g + k) * 32 + lane;
        in[k] = g + k < 32 * per && s < b.n;
        len[k] = in[k] ? __ldg(b.lengths + s) : 0;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned u = __reduce_add_sync(0xffffffffu, in[k] ? (unsigned)units_at(len[k]) : 0u);
        if ((g + k) / per == lane) sum += u;
      }
    }
  }
  if (over) flag(b.status, kErrInput);
  int64_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) line.warp_sum[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kDecodeWarps; ++w) {
    if (w < warp) before += line.warp_sum[w];
    total += line.warp_sum[w];
  }
  line.pref[tid] = before + incl - sum;
  if (tid == 0) line.total = total;
  __syncthreads();
}

// Sequence that holds unit z (counted without head blocks), and its first unit.
template <int KU>
__device__ __forceinline__ void find_seq(const Batch& b, const Line& line, int64_t z, int lane, int& s, int64_t& first) {
  int c = 0;
#pragma unroll
  for (int i = 0; i < kDecodeThreads / 32; ++i) c += line.pref[i * 32 + lane] <= z;
#pragma unroll
  for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  const int seg = stretch(b.n);
  s = (c - 1) * seg;
  first = line.pref[c - 1];
  for (;;) {
    const int i = s + lane;
    const int u = i < b.n ? units_of<KU>(keys_of(b, i)) : 0;
    int64_t incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned le = __ballot_sync(0xffffffffu, first + incl <= z);  // a prefix of the lanes
    const int k = __popc(le);
    if (k) first += __shfl_sync(0xffffffffu, incl, k - 1);
    s += k;
    if (k < 32 || s >= b.n) return;
  }
}

// A piece of an item that its warp could not finish; first: the line's unit
// (counted without head blocks) at which the item's sequence starts.
struct Seg {
  int64_t first;
  int s, block, valid, begin, end;
};

// A warp's place on the line: the piece [u0, u1) of an item.
template <int KU>
struct Cursor {
  int64_t x, x1, first;
  int s, block, keys, us, u0, u1, key0, key1;
  // At unit x_ of the line, up to x1_.
  __device__ __forceinline__ void begin(const Batch& b, const Line& line, int64_t x_, int64_t x1_, int KVB, int lane) {
    x = x_;
    x1 = x1_;
    find_seq<KU>(b, line, muldiv(x, 1, KVB), lane, s, first);
    keys = keys_of(b, s);
    us = units_of<KU>(keys);
    block = (int)muldiv(x - first * KVB, 1, us);
    u0 = (int)(x - first * KVB - (int64_t)block * us);
    piece();
  }
  __device__ __forceinline__ void piece() {
    u1 = (int)min((int64_t)us, u0 + (x1 - x));
    key0 = u0 * KU;
    key1 = min(u1 * KU, keys);
  }
  __device__ __forceinline__ void next(const Batch& b, int KVB) {
    x += u1 - u0;
    u0 = 0;
    if (u1 == us && ++block == KVB) {
      block = 0;
      first += us;
      ++s;
      if (x < x1) {
        keys = keys_of(b, s);
        us = units_of<KU>(keys);
      }
    }
    piece();
  }
};

// A box of the pool: coordinates (element, segment, then kv-head block and slot in the map's order, page).
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int c2, int c3, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(0), "r"(c2), "r"(c3), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// N bytes of shared memory as 32-bit words.
template <int N>
__device__ __forceinline__ void read_words(const uint8_t* p, uint32_t (&w)[N / 4]) {
  if constexpr (N == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (N == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// d = a b + c; `first` (a constant): c is zero.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  const float c0 = first ? 0.f : d[0], c1 = first ? 0.f : d[1], c2 = first ? 0.f : d[2], c3 = first ? 0.f : d[3];
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  const float c0 = first ? 0.f : d[0], c1 = first ? 0.f : d[1], c2 = first ? 0.f : d[2], c3 = first ? 0.f : d[3];
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// Transpose of an 8 x 8 matrix of 16-bit values held as MMA fragments.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// x = hi + lo as TF32 operands: hi rounded to nearest (11 bits), lo the exact
// rest, of which the MMA takes the upper 11 bits.  A NaN stays one in lo.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi));
}
// (x, y) -> their FP16 parts hi and lo, packed.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The line's units and the warps that share them: few units are spread over the
// CTAs first, over a CTA's warps second.
struct Workers {
  int64_t units, count, me;
  int aw;  // warps of a CTA that take part
  __device__ __forceinline__ explicit Workers(int64_t n) : units(n) {
    const int warp = threadIdx.x >> 5;
    aw = units >= (int64_t)gridDim.x * kDecodeWarps ? kDecodeWarps : (int)(((uint32_t)units + gridDim.x - 1) / gridDim.x);
    count = min((int64_t)gridDim.x * aw, units);
    me = warp < aw ? (int64_t)blockIdx.x * aw + warp : count;
  }
  __device__ __forceinline__ bool active() const { return me < count; }
  __device__ __forceinline__ int64_t begin() const { return muldiv(me, units, count); }
  __device__ __forceinline__ int64_t end() const { return muldiv(me + 1, units, count); }
};

// The state of a piece by plain_row.
template <typename KT>
__device__ void plain_piece(const DecodeArgs& a, int s, int h0, int nr, int key0, int key1, bool whole, float* slot) {
  const int lane = threadIdx.x & 31;
  for (int n = 0; n < nr; ++n) {
    const int h = h0 + n;
    float m, l, o[4];
    plain_row<KT>(a.b, a.b.table + s * a.b.table_stride, a.q + s * a.ldq + (int64_t)h * a.hd, a.hd, h / a.b.rep, key0, key1,
                  a.scale, m, l, o);
    const int64_t row = (int64_t)s * a.H + h;
    const float inv = !whole || a.state ? 1.f : (l == 0.f ? 0.f : 1.f / l);
    float* dst = whole ? a.out + row * a.hd : slot + n * a.hd;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane + 32 * e < a.hd) dst[lane + 32 * e] = o[e] * inv;
    if (lane == 0 && !whole) {
      slot[8 * a.hd + n] = m;
      slot[8 * a.hd + 8 + n] = l;
    } else if (lane == 0 && a.state) {
      *reinterpret_cast<float2*>(a.state + row * 2) = make_float2(m, l);
    }
  }
}

// Goes over a warp's stretch once more and makes the pieces anew whose sum of weights
// is not a number.
template <int HDF, typename KT>
__device__ __noinline__ void plain_pieces(const DecodeArgs& a, const Line& line) {
  const Batch& b = a.b;
  const int lane = threadIdx.x & 31, KVB = b.kv_heads / a.F * a.HB, STATE = state_floats(a.hd);
  const Workers k(line.total * KVB);
  if (!k.active()) return;
  float* slots = a.wpart + ((size_t)blockIdx.x * kDecodeWarps + (threadIdx.x >> 5)) * 2 * STATE;
  Cursor<DecodeShape<HDF, KT>::KU> cur;
  cur.begin(b, line, k.begin(), k.end(), KVB, lane);
  const int64_t x = cur.x;
  while (cur.x < cur.x1) {
    int h0, nr;
    block_heads(a, cur.block, h0, nr);
    const bool whole = cur.u0 == 0 && cur.u1 == cur.us;
    float* slot = slots + (cur.x == x ? 0 : 1) * STATE;
    const int64_t row = (int64_t)cur.s * a.H + h0 + lane;
    float l = 0.f;
    if (lane < nr) l = !whole ? slot[8 * a.hd + 8 + lane] : a.state ? a.state[row * 2 + 1] : a.out[row * a.hd];
    if (__any_sync(0xffffffffu, l != l)) plain_piece<KT>(a, cur.s, h0, nr, cur.key0, cur.key1, whole, slot);
    cur.next(b, KVB);
  }
}

template <int HDF, typename KT>
__global__ void __launch_bounds__(kDecodeThreads, DecodeShape<HDF, KT>::CTAS)
    decode_kernel(const __grid_constant__ DecodeArgs a, const __grid_constant__ DecodeMaps maps) {
  using S = DecodeShape<HDF, KT>;
  constexpr bool kHalf = std::is_same<KT, __half>::value;
  constexpr int NK = S::NK, NVC = S::NVC, EK = S::EK, EV = S::EV, CK = S::CK, CV = S::CV, STG = S::STG;
  constexpr int NT = S::NT;                  // tiles of a unit
  constexpr int MT = HDF / 16;               // M tiles of O^T
  constexpr int QS = kHalf ? HDF / 16 : HDF / 8;  // K steps of S
  using Wt = Weights<kHalf, 14>;  // (moving the reference is a few instructions here)
  constexpr float kFirst = Wt::kFirst, kLimit = Wt::kLimit;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ uint8_t smem_raw[];  // [warp][RING], 1024-byte aligned
  __shared__ uint64_t bars[kDecodeWarps * STG];
  __shared__ Line line;
  __shared__ Seg segs[2 * kDecodeWarps];
  __shared__ int odd;  // a sum of weights was not a number
  const Batch& b = a.b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;  // the MMA fragments' row group and column group
  const int STATE = state_floats(a.hd);
  // of the F kv heads side by side: head g's, heads 2 c and 2 c + 1's
  const int fg = a.F > 1 ? g / b.rep : 0, fc[2] = {a.F > 1 ? 2 * c / b.rep : 0, a.F > 1 ? (2 * c + 1) / b.rep : 0};
  const int hd_shift = 31 - __clz(a.hd);
  uint64_t* bar = bars + warp * STG;
  if (threadIdx.x == 0) {
    odd = 0;
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  if (lane < STG) mbar_init(bar + lane, a.stall && blockIdx.x == 0 && lane == 0 ? 2 : 1);
  fence_mbar_init();
  build_line<S::KU>(b, line);
  const int KVB = b.kv_heads / a.F * a.HB;
  const Workers work(line.total * KVB);
  if (lane < 2) segs[2 * warp + lane].valid = 0;
  float* slots = a.wpart + ((size_t)blockIdx.x * kDecodeWarps + warp) * 2 * STATE;
  if (work.active()) {
    Cursor<S::KU> cur;
    cur.begin(b, line, work.begin(), work.end(), KVB, lane);
    const int64_t xb = cur.x;

    // ---- loads
    const uint32_t ring = ((smem_u32(smem_raw) + 1023) & ~1023u) + warp * S::RING;
    const uint8_t* ring_g = smem_raw + (ring - smem_u32(smem_raw));
    Cursor<S::KU> p = cur;
    const int bshift = b.shift >= 4 ? 0 : 4 - b.shift;  // 2^bshift boxes of a tile
    const uint32_t box_bytes = S::TILE >> bshift;
    const int bt = lane >> bshift, bi = lane & ((1 << bshift) - 1);  // this lane starts box bi of tile bt
    const int bkey = bt * kTile + (bi << b.shift);
    const int slot_mask = (1 << b.shift) - 1;
    const int32_t* row = b.table;
    int pblk = 0;
    int pt = 0, pbase = 0, plast = -1, ids = -1;  // page ids: lane i holds the id of page pbase + i
    int istage = 0;
    uint32_t bad = 0;    // bits 2 stage + tile: the tile has a page id out of range
    uint32_t armed = 0;  // bit stage: copies were started into it
    auto enter = [&]() {  // the first piece from p on that has keys
      while (p.x < p.x1 && p.key0 >= p.key1) p.next(b, KVB);
      if (p.x >= p.x1) return;
      pt = p.key0;
      pblk = a.HB == 1 ? p.block : p.block / a.HB;
      row = b.table + p.s * b.table_stride;
      pbase = p.key0 >> b.shift;
      plast = (p.key1 - 1) >> b.shift;
      ids = pbase + lane <= plast ? __ldg(row + pbase + lane) : -1;
    };
    // Start the next half unit's copies.
    auto issue = [&](bool values) {
      if (p.x < p.x1) {
        const int first = pt + bkey;  // the box's first key
        // (a unit's pages are among the lanes' or the next 32: both are aligned to the unit)
        if (!values && ((min(pt + S::KU, p.key1) - 1) >> b.shift) >= pbase + 32) {
          pbase = pt >> b.shift;
          ids = pbase + lane <= plast ? __ldg(row + pbase + lane) : -1;
        }
        const int id = __shfl_sync(kAll, ids, ((first >> b.shift) - pbase) & 31);
        const bool in = bt < NT && first < p.key1, ok = in && (unsigned)id < (unsigned)b.n_pages;
        const unsigned good = __ballot_sync(kAll, ok);
        if (!values) {
          const unsigned wrong = __ballot_sync(kAll, in) & ~good;
          bad &= ~(3u << (2 * istage));
          if (wrong) {
            const uint32_t one = (1u << (1 << bshift)) - 1u;
            bad |= ((wrong & one ? 1u : 0u) | (NT == 2 && (wrong >> (1 << bshift)) & one ? 2u : 0u)) << (2 * istage);
            if (lane == 0) flag(b.status, kErrInput);
          }
        }
        armed |= 1u << istage;
        if (lane == 0) mbar_expect_tx(bar + istage, __popc(good) * box_bytes);
        __syncwarp();
        if (ok) {
          const int slot = first & slot_mask;
          load_box(ring + istage * S::HALF + bt * S::TILE + bi * box_bytes, values ? &maps.v : &maps.k,
                   a.swap ? slot : pblk, a.swap ? pblk : slot, id, bar + istage);
        }
        if (values) {
          pt += S::KU;
          if (pt >= p.key1) {
            p.next(b, KVB);
            enter();
          }
        }
      } else {
        armed &= ~(1u << istage);
      }
      istage = istage + 1 == STG ? 0 : istage + 1;
    };
    enter();
#pragma unroll 1
    for (int i = 0; i < STG - 1; ++i) issue(i & 1);
    int stage = 0;
    uint32_t phase = 0;
    // A wait ran out: nothing more is waited for or started, and the outputs of
    // the rest of the warp's stretch become NaN.
    bool late = false;
    // Wait for the oldest half unit, and start the load that takes the place of
    // the one before it (which every lane has read), STG - 1 halves ahead.
    auto advance = [&](bool values) {
      if (!mbar_try_wait(bar + stage, phase) && !mbar_wait_for(bar + stage, phase, a.wait_cycles)) late = true;
      late = __any_sync(kAll, late);
      __syncwarp();
      const uint8_t* at = ring_g + stage * S::HALF;
      if (late) return at;
      issue(values != ((STG - 1) % 2 != 0));
      if (++stage == STG) {
        stage = 0;
        phase ^= 1;
      }
      return at;
    };
    // the lane's places in a tile: K chunk j of row kappa(g) + 8 r, V chunk j of
    // its value key i (the rows that P^T's fragments hold)
    const int krow = S::kappa(g);
    int vrow[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vrow[i] = S::kappa(kHalf ? 2 * c + (i & 1) : c + 4 * (i & 1)) + 8 * (i >> 1);

    while (cur.x < cur.x1) {
      const int key0 = cur.key0, key1 = cur.key1, s = cur.s;
      int h0, nr;
      block_heads(a, cur.block, h0, nr);
      // ---- queries: head g of the block, dims as the lane's key chunks hold them
      uint32_t qhi[2 * QS], qlo[2 * QS];       // step s: words 2 s, 2 s + 1
      float sc0 = a.scale, sc1 = a.scale;      // score scales of heads 2 c, 2 c + 1
      {
        const float* qp = a.q + s * a.ldq + (int64_t)(h0 + g) * a.hd;
        float qv[HDF / 4];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const int D = j * 4 * EK + c * EK;
          const bool in = g < nr && (a.F == 1 || D >> hd_shift == fg);
#pragma unroll
          for (int e = 0; e < EK; e += 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (in) v = __ldg(reinterpret_cast<const float4*>(qp + (D - fg * a.hd) + e));
            qv[j * EK + e] = v.x;
            qv[j * EK + e + 1] = v.y;
            qv[j * EK + e + 2] = v.z;
            qv[j * EK + e + 3] = v.w;
          }
        }
        if constexpr (kHalf) {
          float mx = 0.f;
#pragma unroll
          for (int i = 0; i < HDF / 4; ++i) mx = fmaxf(mx, fabsf(qv[i]));
          mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(kAll, mx, 2));
          float back;
          const float scale = half_scale(mx, back), us = a.scale * back;
          sc0 = __shfl_sync(kAll, us, 8 * c);
          sc1 = __shfl_sync(kAll, us, 8 * c + 4);
#pragma unroll
          for (int i = 0; i < 2 * QS; ++i) split_f16(qv[2 * i] * scale, qv[2 * i + 1] * scale, qhi[i], qlo[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 2 * QS; ++i) split_tf32(__float_as_uint(qv[i]), qhi[i], qlo[i]);
        }
      }
      float acc[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      // heads 2 c and 2 c + 1: reference, sum of weights
      float ref0 = kUnseen, ref1 = kUnseen, l0 = 0.f, l1 = 0.f;
      for (int t0 = key0; t0 < key1 && !late; t0 += S::KU) {
        // ---- S^T = K q^T: key g heads 2 c, 2 c + 1, then key g + 8
        float x[NT][4];
        {
          const uint32_t nans = bad >> (2 * stage);
          const uint8_t* kr = advance(false);
          if (late) break;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float s0[4], s1[4], s2[4];
#pragma unroll
            for (int j = 0; j < NK; ++j) {
              uint32_t w0[CK / 4], w1[CK / 4];  // keys g and g + 8
              read_words<CK>(kr + t * S::TILE + S::place(krow, j * 4 * CK + c * CK), w0);
              read_words<CK>(kr + t * S::TILE + S::place(krow + 8, j * 4 * CK + c * CK), w1);
#pragma unroll
              for (int h = 0; h < CK / 8; ++h) {
                const int st = j * (CK / 8) + h;
                if constexpr (kHalf) {
                  const uint32_t ka[4] = {w0[2 * h], w1[2 * h], w0[2 * h + 1], w1[2 * h + 1]};
                  mma_f16(s0, ka, qhi[2 * st], qhi[2 * st + 1], st == 0);
                  mma_f16(s1, ka, qlo[2 * st], qlo[2 * st + 1], st == 0);
                } else {
                  uint32_t kh[4], kl[4];
                  split_tf32(w0[2 * h], kh[0], kl[0]);
                  split_tf32(w1[2 * h], kh[1], kl[1]);
                  split_tf32(w0[2 * h + 1], kh[2], kl[2]);
                  split_tf32(w1[2 * h + 1], kh[3], kl[3]);
                  mma_tf32(s0, kh, qhi[2 * st], qhi[2 * st + 1], st == 0);
                  mma_tf32(s1, kh, qlo[2 * st], qlo[2 * st + 1], st == 0);
                  mma_tf32(s2, kl, qhi[2 * st], qhi[2 * st + 1], st == 0);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][i] = kHalf ? s0[i] + s1[i] : s0[i] + (s1[i] + s2[i]);
            if (nans >> t & 1) x[t][0] = x[t][1] = x[t][2] = x[t][3] = NAN;  // never loaded: NaN rows
          }
        }
        if (t0 + S::KU > key1) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (t0 + t * kTile + krow >= key1) x[t][0] = x[t][1] = -INFINITY;
            if (t0 + t * kTile + krow + 8 >= key1) x[t][2] = x[t][3] = -INFINITY;
          }
        }
        // ---- the references, when a score passes them by too much
        float m0 = fmaxf(x[0][0], x[0][2]), m1 = fmaxf(x[0][1], x[0][3]);
        if constexpr (NT == 2) {
          m0 = fmaxf(m0, fmaxf(x[1][0], x[1][2]));
          m1 = fmaxf(m1, fmaxf(x[1][1], x[1][3]));
        }
        m0 *= sc0;
        m1 *= sc1;
        if (__any_sync(kAll, m0 - ref0 > kLimit || m1 - ref1 > kLimit)) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(kAll, m0, o));
            m1 = fmaxf(m1, __shfl_xor_sync(kAll, m1, o));
          }
          // (a head that has seen nothing has l = o = 0: the factor 0 keeps them)
          const float n0 = fmaxf(m0 - kFirst, ref0), n1 = fmaxf(m1 - kFirst, ref1);
          const float f0 = ex2(ref0 - n0), f1 = ex2(ref1 - n1);
          ref0 = n0;
          ref1 = n1;
          l0 *= f0;
          l1 *= f1;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            acc[i][0] *= f0;
            acc[i][1] *= f1;
            acc[i][2] *= f0;
            acc[i][3] *= f1;
          }
        }
        // ---- weights, and P^T as the MMA's B side: head g, the lane's four value keys
        uint32_t phi[NT][4], plo[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float x0 = ex2(fmaf(x[t][0], sc0, -ref0)), x1 = ex2(fmaf(x[t][1], sc1, -ref1));
          const float x2 = ex2(fmaf(x[t][2], sc0, -ref0)), x3 = ex2(fmaf(x[t][3], sc1, -ref1));
          l0 += x0 + x2;
          l1 += x1 + x3;
          if constexpr (kHalf) {
            split_f16(x0, x1, phi[t][0], plo[t][0]);
            split_f16(x2, x3, phi[t][1], plo[t][1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              phi[t][i] = transpose8(phi[t][i]);
              plo[t][i] = transpose8(plo[t][i]);
            }
          } else {
            const bool odd = g & 1;
            const int sa = 4 * c + (g >> 1), sb = sa + 16;  // lanes that hold rows c (c + 8), c + 4 (c + 12)
            const float a0 = __shfl_sync(kAll, x0, sa), a1 = __shfl_sync(kAll, x1, sa);
            const float b0 = __shfl_sync(kAll, x0, sb), b1 = __shfl_sync(kAll, x1, sb);
            const float c0 = __shfl_sync(kAll, x2, sa), c1 = __shfl_sync(kAll, x3, sa);
            const float d0 = __shfl_sync(kAll, x2, sb), d1 = __shfl_sync(kAll, x3, sb);
            split_tf32(__float_as_uint(odd ? a1 : a0), phi[t][0], plo[t][0]);
            split_tf32(__float_as_uint(odd ? b1 : b0), phi[t][1], plo[t][1]);
            split_tf32(__float_as_uint(odd ? c1 : c0), phi[t][2], plo[t][2]);
            split_tf32(__float_as_uint(odd ? d1 : d0), phi[t][3], plo[t][3]);
          }
        }
        // ---- O^T += V^T P^T; M row g of tile i is the lane's dim 2 i, row g + 8 its dim 2 i + 1
        {
          const uint8_t* vr = advance(true);
          if (late) break;
          const bool tail = t0 + S::KU > key1;  // slots behind the last key may hold anything
#pragma unroll
          for (int j = 0; j < NVC; ++j) {
            float o[CV / S::ES / 2][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              uint32_t w[4][CV / 4];
#pragma unroll
              for (int i = 0; i < 4; ++i) read_words<CV>(vr + t * S::TILE + S::place(vrow[i], j * 8 * CV + g * CV), w[i]);
              if (tail) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                  for (int k = 0; k < CV / 4; ++k)
                    if (t0 + t * kTile + vrow[i] >= key1) w[i][k] = 0u;
              }
#pragma unroll
              for (int k = 0; k < EV / 2; ++k) {
                if constexpr (kHalf) {
                  const uint32_t va[4] = {__byte_perm(w[0][k], w[1][k], 0x5410), __byte_perm(w[0][k], w[1][k], 0x7632),
                                          __byte_perm(w[2][k], w[3][k], 0x5410), __byte_perm(w[2][k], w[3][k], 0x7632)};
                  mma_f16(o[k], va, plo[t][0], plo[t][1], t == 0);
                  mma_f16(o[k], va, phi[t][0], phi[t][1], false);
                } else {
#pragma unroll
                  for (int kk = 0; kk < 2; ++kk) {
                    // K slots c, c + 4 of step kk: rows c + 8 kk, c + 8 kk + 4
                    uint32_t vh[4], vl[4];
                    split_tf32(w[2 * kk][2 * k], vh[0], vl[0]);
                    split_tf32(w[2 * kk][2 * k + 1], vh[1], vl[1]);
                    split_tf32(w[2 * kk + 1][2 * k], vh[2], vl[2]);
                    split_tf32(w[2 * kk + 1][2 * k + 1], vh[3], vl[3]);
                    mma_tf32(o[k], vl, phi[t][2 * kk], phi[t][2 * kk + 1], t == 0 && kk == 0);
                    mma_tf32(o[k], vh, plo[t][2 * kk], plo[t][2 * kk + 1], false);
                    mma_tf32(o[k], vh, phi[t][2 * kk], phi[t][2 * kk + 1], false);
                  }
                }
              }
            }
#pragma unroll
            for (int k = 0; k < EV / 2; ++k)
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[j * (EV / 2) + k][i] += o[k][i];
          }
        }
      }
      // ---- the piece's state: sums over the key groups g
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(kAll, l0, o);
        l1 += __shfl_xor_sync(kAll, l1, o);
      }
      if (l0 != l0 || l1 != l1) odd = 1;
      if (late) l0 = l1 = NAN;
      const bool begin = cur.u0 == 0, end = cur.u1 == cur.us, whole = begin && end;
      const int which = cur.x == xb ? 0 : 1;
      float* slot = slots + which * STATE;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int n = 2 * c + hh;
        const float l = hh ? l1 : l0;
        const float inv = !whole || a.state ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        const int f = fc[hh];
        float* dst = whole ? a.out + ((int64_t)s * a.H + h0 + n) * a.hd : slot + n * a.hd;
        if (n < nr) {
#pragma unroll
          for (int j = 0; j < NVC; ++j) {
            const int D = j * 8 * EV + g * EV - f * a.hd;  // dims of the head's own kv head
            if (D < 0 || D >= a.hd) continue;
#pragma unroll
            for (int e = 0; e < EV; e += 2) {
              const int i = (j * EV + e) >> 1;
              *reinterpret_cast<float2*>(dst + D + e) = make_float2(acc[i][hh] * inv, acc[i][2 + hh] * inv);
            }
          }
        }
        if ((!whole || a.state) && g == 0) {
          const float ref = hh ? ref1 : ref0, m = ref == kUnseen ? -INFINITY : ref;
          if (!whole) {
            slot[8 * a.hd + n] = m;
            slot[8 * a.hd + 8 + n] = l;
          } else if (n < nr) {
            *reinterpret_cast<float2*>(a.state + ((int64_t)s * a.H + h0 + n) * 2) = make_float2(m, l);
          }
        }
      }
      if (lane == 0 && !whole) segs[2 * warp + which] = {cur.first, s, cur.block, 1, begin, end};
      cur.next(b, KVB);
    }
    if (late) {
      if (lane == 0) flag(b.status, kErrTimeout);
      // the copies that are still on their way, from the stage that was waited for
      // on, land before the CTA ends (or one more wait runs out)
      for (uint64_t left = a.wait_cycles; stage != istage;) {
        if ((armed >> stage & 1) && !mbar_wait_for(bar + stage, phase, left)) left = 0;
        if (++stage == STG) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  }
  grid_dep_launch();
  __syncthreads();
  if (odd) {
    plain_pieces<HDF, KT>(a, line);
    __syncthreads();
  }
  // ---- pieces of items inside this CTA, in order
  if (threadIdx.x == 0) a.desc[blockIdx.x].z = 0;
  const float* pieces = a.wpart + (size_t)blockIdx.x * kDecodeWarps * 2 * STATE;
  const int hd = a.hd, M0 = 8 * hd, L0 = 8 * hd + 8;
  __shared__ float pm[2 * kDecodeWarps][8], pl[2 * kDecodeWarps][8];
  if (threadIdx.x < 16 * kDecodeWarps) {
    const int k = threadIdx.x >> 3, r = threadIdx.x & 7;
    pm[k][r] = segs[k].valid ? pieces[k * STATE + M0 + r] : -INFINITY;
    pl[k][r] = segs[k].valid ? pieces[k * STATE + L0 + r] : 0.f;
  }
  __syncthreads();
  for (int i = 0; i < 2 * kDecodeWarps;) {
    if (!segs[i].valid) {
      ++i;
      continue;
    }
    int j = i + 1, last = i;
    for (; j < 2 * kDecodeWarps; ++j) {
      if (!segs[j].valid) continue;
      if (segs[j].s != segs[i].s || segs[j].block != segs[i].block) break;
      last = j;
    }
    const Seg f = segs[i];
    const bool end = segs[last].end;
    int h0, nr;
    block_heads(a, f.block, h0, nr);
    float* dst = a.part + ((size_t)blockIdx.x * 2 + (f.begin ? 1 : 0)) * STATE;
    for (int x = threadIdx.x * 4; x < nr * hd; x += kDecodeThreads * 4) {
      const int r = x / hd;
      float M = -INFINITY;
      for (int k = i; k <= last; ++k) M = fmaxf(M, pm[k][r]);
      const float ref = ref_of(M);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int n = 0; n < 2 * kDecodeWarps; ++n) {
        if (n < i || n > last || !segs[n].valid) continue;
        const float w = ex2(pm[n][r] - ref);
        const float4 v = *reinterpret_cast<const float4*>(pieces + n * STATE + x);
        o.x = fmaf(w, v.x, o.x);
        o.y = fmaf(w, v.y, o.y);
        o.z = fmaf(w, v.z, o.z);
        o.w = fmaf(w, v.w, o.w);
        l = fmaf(w, pl[n][r], l);
      }
      const bool head = x == r * hd;
      if (f.begin && end) {
        const int64_t row = (int64_t)f.s * a.H + h0;
        const float inv = a.state ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        *reinterpret_cast<float4*>(a.out + row * hd + x) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        if (a.state && head) *reinterpret_cast<float2*>(a.state + (row + r) * 2) = make_float2(M, l);
      } else {
        *reinterpret_cast<float4*>(dst + x) = o;
        if (head) {
          dst[M0 + r] = M;
          dst[L0 + r] = l;
        }
      }
    }
    if (threadIdx.x == 0 && f.begin && !end) {
      // the CTA that holds the item's last unit
      const int us = units_of<S::KU>(keys_of(b, f.s));
      const int64_t lastu = f.first * KVB + (int64_t)(f.block + 1) * us - 1;
      const int c1 = (int)(owner_of(lastu, work.units, work.count) / work.aw);
      a.desc[blockIdx.x] = make_int4(f.s, f.block, c1 - (int)blockIdx.x + 1, 0);
    }
    i = j;
  }
}

// Joins the pieces of the items that several CTAs hold: block (c, 0) all heads of
// the item that starts in CTA c when it has few pieces (8192 short requests: 11.7 us
// with a block a head, 5.9 so), block (c, y) head y when it has many (one long request:
// a block for all would walk over 111 pieces of 512 floats).  A warp a head finds the
// pieces' weights, then groups of heads head_dim / 4 threads share the pieces out.
constexpr int kMergeThreads = 256;
constexpr int kMergeMost = 1024;  // pieces of an item: the CTAs of a grid
constexpr int kFewPieces = 8;
// (kMergeMost floats would do.  With 4 KB instead of 32 more of these blocks wait beside
// the decode kernel's last CTAs: 256 requests of up to 512 keys, hd 64, 51.2 us against 50.0.)
constexpr int kMergeWeights = 8 * kMergeMost;

__global__ void __launch_bounds__(kMergeThreads) merge_kernel(DecodeArgs a) {
  grid_dep_wait();  // (launched as the decode kernel drains)
  const int4 d = a.desc[blockIdx.x];
  if (d.z == 0) return;
  int h0, nr;
  block_heads(a, d.y, h0, nr);
  const int r0 = blockIdx.y, heads = d.z <= kFewPieces ? nr : 1;
  if (r0 >= nr || (heads > 1 && r0 > 0)) return;
  __shared__ float w[kMergeWeights], total[8], top[8];
  __shared__ float4 so[kMergeThreads];
  const int STATE = state_floats(a.hd), hd = a.hd, M0 = 8 * hd + r0, L0 = 8 * hd + 8 + r0;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // (the first CTA's piece is its second slot)
  const float* base = a.part + (size_t)blockIdx.x * 2 * STATE;
  auto piece = [&](int k) { return base + ((size_t)k * 2 + (k == 0 ? 1 : 0)) * STATE; };
  // warp r: the pieces' weights of head r0 + r
  if (warp < heads) {
    float M = -INFINITY;
    for (int k = lane; k < d.z; k += 32) {
      const float m = piece(k)[M0 + warp];
      w[k * heads + warp] = m;
      M = fmaxf(M, m);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = ref_of(M);
    float l = 0.f;
    for (int k = lane; k < d.z; k += 32) {
      const float x = ex2(w[k * heads + warp] - ref);
      w[k * heads + warp] = x;
      l = fmaf(x, piece(k)[L0 + warp], l);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      total[warp] = l;
      top[warp] = M;
    }
  }
  __syncthreads();
  const int per = heads * hd / 4, groups = kMergeThreads / per;  // 4 to 256 threads a group
  const int64_t row = (int64_t)d.x * a.H + h0 + r0;
  const int x = tid % per, grp = tid / per, r = 4 * x / hd;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < groups) {
#pragma unroll 4
    for (int k = grp; k < d.z; k += groups) {
      const float4 v = *reinterpret_cast<const float4*>(piece(k) + r0 * hd + 4 * x);
      const float p = w[k * heads + r];
      o.x = fmaf(p, v.x, o.x);
      o.y = fmaf(p, v.y, o.y);
      o.z = fmaf(p, v.z, o.z);
      o.w = fmaf(p, v.w, o.w);
    }
  }
  so[tid] = o;
  __syncthreads();
  if (grp > 0) return;
  for (int k = 1; k < groups; ++k) {
    const float4 v = so[k * per + tid];
    o.x += v.x;
    o.y += v.y;
    o.z += v.z;
    o.w += v.w;
  }
  const float l = total[r], inv = a.state ? 1.f : (l == 0.f ? 0.f : 1.f / l);
  *reinterpret_cast<float4*>(a.out + row * hd + 4 * x) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  if (a.state && 4 * x == r * hd) *reinterpret_cast<float2*>(a.state + (row + r) * 2) = make_float2(top[r], l);
}

// ---- host ---------------------------------------------------------------------

constexpr int kMaxPerSm = 4;  // CTAs an SM at most (DecodeShape::CTAS)

// desc | CTA pieces | warp pieces
size_t decode_workspace(int hd) {
  const size_t ctas = (size_t)sm_count() * kMaxPerSm;
  return ctas * (sizeof(int4) + (2 + 2 * kDecodeWarps) * state_floats(hd) * sizeof(float));
}

static PFN_cuTensorMapEncodeTiled_v12000 map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// The pool as (ib bytes, segments, kv-head blocks, slots, pages) -- blocks and
// slots in ascending order of their strides -- with a box of `rows` slots and
// `segments` segments of one block.
int32_t pool_map(const Batch& b, void* pool, int hd, int es, int F, int rows, int segments, CUtensorMap* map,
                 bool* swap) {
  auto encode = map_encoder();
  if (!encode) return fail(Q6W_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const int rb = F * hd * es, ib = rb < 128 ? rb : 128;
  const int page = 1 << b.shift;
  cuuint64_t dim[5] = {(cuuint64_t)(ib / es), (cuuint64_t)(rb / ib), (cuuint64_t)(b.kv_heads / F), (cuuint64_t)page,
                       (cuuint64_t)std::max(b.n_pages, 1)};
  // (a dimension of one has no stride of its own)
  const cuuint64_t ss = page > 1 ? (cuuint64_t)b.slot_stride * es : rb;
  const cuuint64_t hs = b.kv_heads / F > 1 ? (cuuint64_t)F * b.head_stride * es : rb;
  const cuuint64_t ps = b.n_pages > 1 ? (cuuint64_t)b.page_stride * es : rb;
  cuuint64_t stride[4] = {128, hs, ss, ps};
  cuuint32_t box[5] = {(cuuint32_t)(ib / es), (cuuint32_t)segments, 1, (cuuint32_t)rows, 1};
  cuuint32_t step[5] = {1, 1, 1, 1, 1};
  *swap = hs > ss;
  if (*swap) {
    std::swap(dim[2], dim[3]);
    std::swap(stride[1], stride[2]);
    std::swap(box[2], box[3]);
  }
  const CUresult r =
      encode(map, es == 2 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 5, pool, dim, stride, box,
             step, CU_TENSOR_MAP_INTERLEAVE_NONE,
             ib == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : ib == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(Q6W_ERR_ARG, "the pages' strides cannot be described to the copy engine (%d)", (int)r);
  return Q6W_OK;
}

template <int HDF, typename KT>
static int32_t launch(DecodeArgs a, cudaStream_t st) {
  using S = DecodeShape<HDF, KT>;
  auto kern = decode_kernel<HDF, KT>;
  constexpr int smem = 1024 + kDecodeWarps * S::RING;
  static std::mutex mu;
  static bool granted[64] = {false};  // per device
  int dev = 0;
  Q6W_CUDA_TRY(cudaGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!granted[dev & 63]) {
      Q6W_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      granted[dev & 63] = true;
    }
  }
  DecodeMaps maps;
  const int rows = std::min(kTile, 1 << a.b.shift);
  bool swap = false;
  int32_t rc = pool_map(a.b, a.b.k, a.hd, S::ES, a.F, rows, S::RB / S::IB, &maps.k, &swap);
  if (!rc) rc = pool_map(a.b, a.b.v, a.hd, S::ES, a.F, rows, S::RB / S::IB, &maps.v, &swap);
  if (rc) return rc;
  a.swap = swap;
  const int64_t most = (int64_t)a.b.n * (a.b.kv_heads / a.F) * a.HB *
                       std::max<int64_t>(1, ((int64_t)a.b.max_len + S::KU - 1) / S::KU);
  const int grid = (int)std::min<int64_t>(std::min(sm_count() * S::CTAS, kMergeMost), most);
  kern<<<grid, kDecodeThreads, smem, st>>>(a, maps);
  Q6W_LAUNCH_CHECK("decode_kernel");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, (unsigned)(a.F > 1 ? a.F * a.b.rep : a.per));
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  Q6W_CUDA_TRY(cudaLaunchKernelEx(&cfg, merge_kernel, a));
  return Q6W_OK;
}

int32_t decode_attention(const DecodeArgs& args, bool half, cudaStream_t st) {
  DecodeArgs a = args;
  const size_t ctas = (size_t)sm_count() * kMaxPerSm;
  char* ws = reinterpret_cast<char*>(a.desc);
  a.part = reinterpret_cast<float*>(ws + ctas * sizeof(int4));
  a.wpart = a.part + ctas * 2 * state_floats(a.hd);
  a.HB = (a.b.rep + 7) / 8;
  a.per = (a.b.rep + a.HB - 1) / a.HB;
  // narrow heads side by side: while F head_dim <= 64 and F rep <= 8 heads
  a.F = 1;
  if (a.b.head_stride == a.hd || a.b.kv_heads == 1)
    while (2 * a.F * a.hd <= 64 && 2 * a.F * a.b.rep <= 8 && a.b.kv_heads % (2 * a.F) == 0) a.F *= 2;
  switch (a.F * a.hd) {
    case 16: return half ? launch<16, __half>(a, st) : launch<16, float>(a, st);
    case 32: return half ? launch<32, __half>(a, st) : launch<32, float>(a, st);
    case 64: return half ? launch<64, __half>(a, st) : launch<64, float>(a, st);
    default: return half ? launch<128, __half>(a, st) : launch<128, float>(a, st);
  }
}

}  // namespace paged
}  // namespace q6w

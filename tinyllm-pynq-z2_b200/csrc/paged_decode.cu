// Decode attention over paged caches: one query token a sequence.
//
// Mathematics.  One pass over the keys with a reference exponent m, a sum l and
// an output o per query head: p = 2^(s - m), l += p, o += p v; m follows the
// largest score so far (it moves only when a score passes it by more than 8,
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
// power of two per head) and weights enter as two FP16 parts, hi + lo, 22
// bits.  FP32 keys, values, queries and weights enter as two TF32 parts and
// the products hi hi + hi lo + lo hi, dropping terms of 2^-22.  The MMA adds
// in FP32; a tile's output is added to o in registers, rounded to nearest, so
// no long sum lives in the MMA's accumulator.
//
// Narrow heads.  While heads of head_dim <= 32 lie side by side in a slot, F kv
// heads are treated as one of F head_dim dims: their queries stand block-
// diagonally, zero elsewhere, and of the F blocks of O each head keeps its own.
// A key's bytes of all F heads are then one contiguous read and the MMAs run
// at full width.
//
// Layout of the work.  An item is (sequence, F kv heads, block of up to eight
// query heads), cut into units of 16 keys.  The units of all items lie on one
// line (a prefix sum of the lengths, taken by every CTA for itself), and every
// warp takes an equal stretch of it: ragged lengths and few long sequences
// balance alike.  A warp that holds an item whole writes its output; pieces
// of an item go through the workspace, joined by their CTA when it holds them
// all, else by merge_kernel.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "paged.cuh"

namespace q6w {
namespace paged {

constexpr int kTile = 16;  // keys of a unit: one MMA's M side

// A partial state: o[8][head_dim], m[8], l[8].
__host__ __device__ constexpr int state_floats(int hd) { return 8 * hd + 16; }

// First query head and heads of an item's block.
__device__ __forceinline__ void block_heads(const DecodeArgs& a, int block, int& h0, int& nr) {
  const int kb = block / a.HB, hb = block - kb * a.HB;
  h0 = kb * a.F * a.b.rep + hb * a.per;
  nr = a.F > 1 ? a.F * a.b.rep : min(a.per, a.b.rep - hb * a.per);
}

// Warps, shared-memory ring and CTAs an SM by the width HDF = F head_dim.
template <int HDF, typename KT>
struct DecodeShape {
  static constexpr int ES = (int)sizeof(KT);
  static constexpr int CK = HDF / 4 * ES < 16 ? HDF / 4 * ES : 16;  // bytes of a lane's K chunk
  static constexpr int CV = HDF / 8 * ES < 16 ? HDF / 8 * ES : 16;
  static constexpr int NK = HDF / 4 * ES / CK;  // K chunks of a key that a lane holds (4 lanes a key)
  static constexpr int NVC = HDF / 8 * ES / CV; // V chunks of a key that a lane holds (8 lanes a key)
  static constexpr int EK = CK / ES, EV = CV / ES;
  static constexpr int HALF = kTile * HDF * ES;  // bytes of a unit's keys (or values)
  // The loads run ahead in a ring of half units (K and V alternate).  HDF 128
  // FP32 needs 64 + 32 registers for q and o: one CTA an SM; else two.
  static constexpr int CTAS = HDF >= 128 ? 1 : 2;
  static constexpr int kMost = (CTAS == 1 ? 24 : 12) * 1024 / HALF;
  static constexpr int STG = kMost < 8 ? kMost : 8;
  static constexpr int RING = STG * HALF;
};

constexpr int kDecodeWarps = 8;
constexpr int kDecodeThreads = 32 * kDecodeWarps;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A maximum to subtract: nothing seen yet counts as 0, so that the weights are 2^-inf = 0.
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ int64_t owner_of(int64_t unit, int64_t units, int64_t workers) {
  // worker w holds units [w units / workers, (w + 1) units / workers)
  return ((unit + 1) * workers + units - 1) / units - 1;
}

// The line of units: prefix sums over 256 stretches of sequences.
struct Line {
  int64_t pref[kDecodeThreads];
  int64_t total;
  int64_t warp_sum[kDecodeWarps];
};

// Keys that sequence s's token sees.
__device__ __forceinline__ int keys_of(const Batch& b, int s) { return min(max(__ldg(b.lengths + s), 0), b.max_len); }

__device__ __forceinline__ int units_of(int keys) { return max(1, (keys + kTile - 1) / kTile); }

__device__ __forceinline__ void build_line(const Batch& b, Line& line) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seg = (b.n + kDecodeThreads - 1) / kDecodeThreads;
  int64_t sum = 0;
  for (int s = tid * seg; s < min((tid + 1) * seg, b.n); ++s) {
    const int len = __ldg(b.lengths + s);
    if (len > b.max_len) flag(b.status, kErrInput);
    sum += units_of(min(max(len, 0), b.max_len));
  }
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
__device__ __forceinline__ void find_seq(const Batch& b, const Line& line, int64_t z, int lane, int& s, int64_t& first) {
  int c = 0;
#pragma unroll
  for (int i = 0; i < kDecodeThreads / 32; ++i) c += line.pref[i * 32 + lane] <= z;
#pragma unroll
  for (int o = 16; o; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
  const int seg = (b.n + kDecodeThreads - 1) / kDecodeThreads;
  s = (c - 1) * seg;
  first = line.pref[c - 1];
  for (;;) {
    const int i = s + lane;
    const int u = i < b.n ? units_of(keys_of(b, i)) : 0;
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
struct Cursor {
  int64_t x, x1, first;
  int s, block, keys, us, u0, u1, key0, key1;
  __device__ __forceinline__ void piece() {
    u1 = (int)min((int64_t)us, u0 + (x1 - x));
    key0 = u0 * kTile;
    key1 = min(u1 * kTile, keys);
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
        us = units_of(keys);
      }
    }
    piece();
  }
};

// Bytes from global to shared memory, zeros instead when `in` is false.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool in) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(in ? N : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo, two TF32 values: hi rounded to nearest (11 bits), lo the rest cut
// to 11 bits.  A NaN stays one in lo.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t& hi, uint32_t& lo) {
  hi = (x + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(hi)) & 0xffffe000u;
}
// (x, y) -> their FP16 parts hi and lo, packed.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

template <int HDF, typename KT>
__global__ void __launch_bounds__(kDecodeThreads, DecodeShape<HDF, KT>::CTAS) decode_kernel(DecodeArgs a) {
  using S = DecodeShape<HDF, KT>;
  constexpr bool kHalf = std::is_same<KT, __half>::value;
  constexpr int NK = S::NK, NVC = S::NVC, EK = S::EK, EV = S::EV, CK = S::CK, CV = S::CV, STG = S::STG;
  constexpr int MT = HDF / 16;               // M tiles of O^T
  constexpr int QS = kHalf ? HDF / 16 : HDF / 8;  // K steps of S
  constexpr float kOff = kHalf ? 4.f : 0.f;  // FP16 weights reach 2^(kOff + 8): their low parts stay normal
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(16) uint8_t smem[];  // [warp][RING]
  __shared__ Line line;
  __shared__ Seg segs[2 * kDecodeWarps];
  const Batch& b = a.b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;  // the MMA fragments' row group and column group
  const int STATE = state_floats(a.hd);
  build_line(b, line);
  const int KVB = b.kv_heads / a.F * a.HB;
  const int64_t units = line.total * KVB;
  // few units: spread them over the CTAs first, over a CTA's warps second
  const int aw = (int)min((int64_t)kDecodeWarps, (units + gridDim.x - 1) / gridDim.x);
  const int64_t workers = min((int64_t)gridDim.x * aw, units);
  const int64_t wi = (int64_t)blockIdx.x * aw + warp;
  const bool active = warp < aw && wi < workers;
  if (lane < 2) segs[2 * warp + lane].valid = 0;
  float* slots = a.wpart + ((size_t)blockIdx.x * kDecodeWarps + warp) * 2 * STATE;
  if (active) {
    Cursor cur;
    cur.x = wi * units / workers;
    cur.x1 = (wi + 1) * units / workers;
    const int64_t xb = cur.x;
    find_seq(b, line, cur.x / KVB, lane, cur.s, cur.first);
    cur.keys = keys_of(b, cur.s);
    cur.us = units_of(cur.keys);
    cur.block = (int)((cur.x - cur.first * KVB) / cur.us);
    cur.u0 = (int)((cur.x - cur.first * KVB) % cur.us);
    cur.piece();

    // ---- loads: half units in consumption order (keys, values, keys, ...),
    // over the ends of items, into a ring that is private to each lane (a lane
    // reads the bytes that it copied itself: waiting for its own copies is
    // enough).  Lane (g, c) takes of keys g and g + 8 dims j 4 EK + c EK + e
    // (j < NK, e < EK), of the values of its four keys dims j 8 EV + g EV + e.
    const uint8_t* ring_g = smem + warp * S::RING;
    const uint32_t ring = smem_u32(ring_g);
    Cursor p = cur;
    const KT* kbase = static_cast<const KT*>(b.k);
    const KT* vbase = static_cast<const KT*>(b.v);
    const bool one_page = b.shift >= 4;  // a unit lies inside a page
    const int32_t* row = b.table;
    int pt = 0, pbase = 0, plast = -1, ids = -1;  // page ids: lane i holds the id of page pbase + i
    int64_t hoff = 0;
    int istage = 0;
    uint32_t bad = 0;  // bits 2 stage, 2 stage + 1: key g, key g + 8 has a page id out of range
    auto value_key = [&](int i) { return kHalf ? 2 * c + (i & 1) + 8 * (i >> 1) : c + 4 * i; };
    auto enter = [&]() {  // the first piece from p on that has keys
      while (p.x < p.x1 && p.key0 >= p.key1) p.next(b, KVB);
      if (p.x >= p.x1) return;
      pt = p.key0;
      row = b.table + p.s * b.table_stride;
      pbase = p.key0 >> b.shift;
      plast = (p.key1 - 1) >> b.shift;
      ids = pbase + lane <= plast ? __ldg(row + pbase + lane) : -1;
      hoff = (int64_t)(p.block / a.HB) * a.F * b.head_stride;
    };
    // offset of key t (any lane's), by the whole warp; -1: a bad page id
    auto offset = [&](int t) -> int64_t {
      const int id = __shfl_sync(kAll, ids, ((t >> b.shift) - pbase) & 31);
      if ((unsigned)id >= (unsigned)b.n_pages) return -1;
      return id * b.page_stride + (int64_t)(t & ((1 << b.shift) - 1)) * b.slot_stride + hoff;
    };
    auto issue = [&](bool values) {
      if (p.x < p.x1) {
        const uint32_t dst = ring + istage * S::HALF;
        if (((min(pt + kTile, p.key1) - 1) >> b.shift) >= pbase + 32) {  // warp-uniform
          pbase = pt >> b.shift;
          ids = pbase + lane <= plast ? __ldg(row + pbase + lane) : -1;
        }
        const int64_t base = one_page ? offset(pt) : 0;
        if (!values) {
          bad &= ~(3u << (2 * istage));
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int k = g + 8 * r;
            int64_t off = one_page ? (base < 0 ? base : base + k * b.slot_stride) : offset(pt + k);
            const bool in = pt + k < p.key1;
            if (in && off < 0) {
              bad |= 1u << (2 * istage + r);
              flag(b.status, kErrInput);
            }
            const bool ok = in && off >= 0;
            if (!ok) off = 0;
#pragma unroll
            for (int j = 0; j < NK; ++j)
              copy_async<CK>(dst + ((r * NK + j) * 32 + lane) * CK, kbase + off + j * 4 * EK + c * EK, ok);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = value_key(i);
            int64_t off = one_page ? (base < 0 ? base : base + k * b.slot_stride) : offset(pt + k);
            const bool ok = pt + k < p.key1 && off >= 0;
            if (!ok) off = 0;
#pragma unroll
            for (int j = 0; j < NVC; ++j)
              copy_async<CV>(dst + ((i * NVC + j) * 32 + lane) * CV, vbase + off + j * 8 * EV + g * EV, ok);
          }
          pt += kTile;
          if (pt >= p.key1) {
            p.next(b, KVB);
            enter();
          }
        }
      }
      istage = istage + 1 == STG ? 0 : istage + 1;
      copy_commit();
    };
    enter();
    bool next_values = false;
#pragma unroll
    for (int i = 0; i < STG - 1; ++i) {
      issue(next_values);
      next_values = !next_values;
    }
    int stage = 0;
    auto advance = [&]() {  // the oldest half unit is here; start the load that takes the place of the one before it
      copy_wait<STG - 2>();
      issue(next_values);
      next_values = !next_values;
      const uint8_t* at = ring_g + stage * S::HALF;
      stage = stage + 1 == STG ? 0 : stage + 1;
      return at;
    };

    while (cur.x < cur.x1) {
      const int key0 = cur.key0, key1 = cur.key1, s = cur.s;
      int h0, nr;
      block_heads(a, cur.block, h0, nr);
      // ---- queries: head g of the block, dims as the lane's key chunks hold them
      const int fg = a.F > 1 ? g / b.rep : 0;  // its kv head among the F
      uint32_t qhi[2 * QS], qlo[2 * QS];       // step s: words 2 s, 2 s + 1
      float sc0 = a.scale, sc1 = a.scale;      // score scales of heads 2 c, 2 c + 1
      {
        const float* qp = a.q + s * a.ldq + (int64_t)(h0 + g) * a.hd;
        float qv[HDF / 4];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const int D = j * 4 * EK + c * EK;
          const bool in = g < nr && (a.F == 1 || D / a.hd == fg);
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
          // 2^-e with 2^e the power of two at or below the head's largest element
          const int ex = min(max((int)(__float_as_uint(mx) >> 23), 1), 253);
          const float down = __uint_as_float((uint32_t)(254 - ex) << 23), up = __uint_as_float((uint32_t)ex << 23);
          const float us = a.scale * up;
          sc0 = __shfl_sync(kAll, us, 8 * c);
          sc1 = __shfl_sync(kAll, us, 8 * c + 4);
#pragma unroll
          for (int i = 0; i < 2 * QS; ++i) split_f16(qv[2 * i] * down, qv[2 * i + 1] * down, qhi[i], qlo[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 2 * QS; ++i) split_tf32(__float_as_uint(qv[i]), qhi[i], qlo[i]);
        }
      }
      float acc[MT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      // heads 2 c and 2 c + 1: reference (0 until a score was seen), the score that moves it, sum
      float ref0 = 0.f, ref1 = 0.f, top0 = -INFINITY, top1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      for (int t0 = key0; t0 < key1; t0 += kTile) {
        // ---- S^T = K q^T
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
        {
          const uint32_t nan2 = bad >> (2 * stage);
          const uint8_t* kr = advance() + lane * CK;
#pragma unroll
          for (int j = 0; j < NK; ++j) {
            uint32_t w0[CK / 4], w1[CK / 4];  // keys g and g + 8
            read_words<CK>(kr + j * 32 * CK, w0);
            read_words<CK>(kr + (NK + j) * 32 * CK, w1);
            if (j == 0) {
              if (nan2 & 1) w0[0] = ~0u;
              if (nan2 & 2) w1[0] = ~0u;
            }
#pragma unroll
            for (int h = 0; h < CK / 8; ++h) {
              const int st = j * (CK / 8) + h;
              if constexpr (kHalf) {
                const uint32_t ka[4] = {w0[2 * h], w1[2 * h], w0[2 * h + 1], w1[2 * h + 1]};
                mma_f16(s0, ka, qhi[2 * st], qhi[2 * st + 1]);
                mma_f16(s1, ka, qlo[2 * st], qlo[2 * st + 1]);
              } else {
                uint32_t kh[4], kl[4];
                split_tf32(w0[2 * h], kh[0], kl[0]);
                split_tf32(w1[2 * h], kh[1], kl[1]);
                split_tf32(w0[2 * h + 1], kh[2], kl[2]);
                split_tf32(w1[2 * h + 1], kh[3], kl[3]);
                mma_tf32(s0, kh, qhi[2 * st], qhi[2 * st + 1]);
                mma_tf32(s1, kh, qlo[2 * st], qlo[2 * st + 1]);
                mma_tf32(s2, kl, qhi[2 * st], qhi[2 * st + 1]);
              }
            }
          }
        }
        // ---- weights: x0, x1 of key g (heads 2 c, 2 c + 1), x2, x3 of key g + 8
        float x0 = (s0[0] + (s1[0] + s2[0])) * sc0, x1 = (s0[1] + (s1[1] + s2[1])) * sc1;
        float x2 = (s0[2] + (s1[2] + s2[2])) * sc0, x3 = (s0[3] + (s1[3] + s2[3])) * sc1;
        if (t0 + kTile > key1) {
          if (t0 + g >= key1) x0 = x1 = -INFINITY;
          if (t0 + g + 8 >= key1) x2 = x3 = -INFINITY;
        }
        if (__any_sync(kAll, fmaxf(x0, x2) > top0 || fmaxf(x1, x3) > top1)) {
          float m0 = fmaxf(x0, x2), m1 = fmaxf(x1, x3);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(kAll, m0, o));
            m1 = fmaxf(m1, __shfl_xor_sync(kAll, m1, o));
          }
          // a head that has seen nothing yet has l = o = 0: any factor will do
          m0 = fmaxf(m0, top0 == -INFINITY ? -INFINITY : ref0 + kOff);
          m1 = fmaxf(m1, top1 == -INFINITY ? -INFINITY : ref1 + kOff);
          const float n0 = m0 == -INFINITY ? 0.f : m0 - kOff, n1 = m1 == -INFINITY ? 0.f : m1 - kOff;
          const float f0 = top0 == -INFINITY ? 1.f : ex2(ref0 - n0), f1 = top1 == -INFINITY ? 1.f : ex2(ref1 - n1);
          ref0 = n0;
          ref1 = n1;
          top0 = m0 + 8.f;
          top1 = m1 + 8.f;
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
        x0 = ex2(x0 - ref0);
        x1 = ex2(x1 - ref1);
        x2 = ex2(x2 - ref0);
        x3 = ex2(x3 - ref1);
        l0 += x0 + x2;
        l1 += x1 + x3;
        // ---- P^T as the MMA's B side: head g, the lane's four keys
        float pv[4];
        {
          const bool odd = g & 1;
          if constexpr (kHalf) {
            const int sa = 8 * c + (g >> 1), sb = sa + 4;  // lanes that hold keys 2 c (2 c + 8), 2 c + 1 (2 c + 9)
            const float a0 = __shfl_sync(kAll, x0, sa), a1 = __shfl_sync(kAll, x1, sa);
            const float b0 = __shfl_sync(kAll, x0, sb), b1 = __shfl_sync(kAll, x1, sb);
            const float c0 = __shfl_sync(kAll, x2, sa), c1 = __shfl_sync(kAll, x3, sa);
            const float d0 = __shfl_sync(kAll, x2, sb), d1 = __shfl_sync(kAll, x3, sb);
            pv[0] = odd ? a1 : a0;
            pv[1] = odd ? b1 : b0;
            pv[2] = odd ? c1 : c0;
            pv[3] = odd ? d1 : d0;
          } else {
            const int sa = 4 * c + (g >> 1), sb = sa + 16;  // keys c (c + 8), c + 4 (c + 12)
            const float a0 = __shfl_sync(kAll, x0, sa), a1 = __shfl_sync(kAll, x1, sa);
            const float b0 = __shfl_sync(kAll, x0, sb), b1 = __shfl_sync(kAll, x1, sb);
            const float c0 = __shfl_sync(kAll, x2, sa), c1 = __shfl_sync(kAll, x3, sa);
            const float d0 = __shfl_sync(kAll, x2, sb), d1 = __shfl_sync(kAll, x3, sb);
            pv[0] = odd ? a1 : a0;
            pv[1] = odd ? b1 : b0;
            pv[2] = odd ? c1 : c0;
            pv[3] = odd ? d1 : d0;
          }
        }
        // ---- O^T += V^T P^T; M row g of tile i is the lane's dim 2 i, row g + 8 its dim 2 i + 1
        {
          const uint8_t* vr = advance() + lane * CV;
          uint32_t phi[4], plo[4];
          if constexpr (kHalf) {
            split_f16(pv[0], pv[1], phi[0], plo[0]);
            split_f16(pv[2], pv[3], phi[1], plo[1]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) split_tf32(__float_as_uint(pv[i]), phi[i], plo[i]);
          }
#pragma unroll
          for (int j = 0; j < NVC; ++j) {
            uint32_t w[4][CV / 4];
#pragma unroll
            for (int i = 0; i < 4; ++i) read_words<CV>(vr + (i * NVC + j) * 32 * CV, w[i]);
            if constexpr (kHalf) {
#pragma unroll
              for (int k = 0; k < CV / 4; ++k) {
                const uint32_t va[4] = {__byte_perm(w[0][k], w[1][k], 0x5410), __byte_perm(w[0][k], w[1][k], 0x7632),
                                        __byte_perm(w[2][k], w[3][k], 0x5410), __byte_perm(w[2][k], w[3][k], 0x7632)};
                float o[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(o, va, plo[0], plo[1]);
                mma_f16(o, va, phi[0], phi[1]);
                const int i = j * (CV / 4) + k;
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[i][x] += o[x];
              }
            } else {
#pragma unroll
              for (int k = 0; k < CV / 8; ++k) {
                float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                  // K slots c, c + 4 of step kk: keys c + 8 kk, c + 8 kk + 4
                  uint32_t vh[4], vl[4];
                  split_tf32(w[2 * kk][2 * k], vh[0], vl[0]);
                  split_tf32(w[2 * kk][2 * k + 1], vh[1], vl[1]);
                  split_tf32(w[2 * kk + 1][2 * k], vh[2], vl[2]);
                  split_tf32(w[2 * kk + 1][2 * k + 1], vh[3], vl[3]);
                  mma_tf32(o, vl, phi[2 * kk], phi[2 * kk + 1]);
                  mma_tf32(o, vh, plo[2 * kk], plo[2 * kk + 1]);
                  mma_tf32(o, vh, phi[2 * kk], phi[2 * kk + 1]);
                }
                const int i = j * (CV / 8) + k;
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[i][x] += o[x];
              }
            }
          }
        }
      }
      // ---- the piece's state: sums over the key groups g
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l0 += __shfl_xor_sync(kAll, l0, o);
        l1 += __shfl_xor_sync(kAll, l1, o);
      }
      const bool begin = cur.u0 == 0, end = cur.u1 == cur.us, whole = begin && end;
      const int which = cur.x == xb ? 0 : 1;
      float* slot = slots + which * STATE;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int n = 2 * c + hh;
        const float l = hh ? l1 : l0;
        const float inv = !whole ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        const int f = a.F > 1 ? n / b.rep : 0;
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
        if (!whole && g == 0) {
          slot[8 * a.hd + n] = (hh ? top1 : top0) == -INFINITY ? -INFINITY : (hh ? ref1 : ref0);
          slot[8 * a.hd + 8 + n] = l;
        }
      }
      if (lane == 0 && !whole) segs[2 * warp + which] = {cur.first, s, cur.block, 1, begin, end};
      cur.next(b, KVB);
    }
  }
  __syncthreads();
  // ---- pieces of items inside this CTA, in order
  if (threadIdx.x == 0) a.desc[blockIdx.x].z = 0;
  const float* pieces = a.wpart + (size_t)blockIdx.x * kDecodeWarps * 2 * STATE;
  const int hd = a.hd, M0 = 8 * hd, L0 = 8 * hd + 8;
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
    for (int x = threadIdx.x; x < nr * hd; x += kDecodeThreads) {
      const int r = x / hd;
      float M = -INFINITY;
      for (int k = i; k <= last; ++k)
        if (segs[k].valid) M = fmaxf(M, pieces[k * STATE + M0 + r]);
      const float ref = ref_of(M);
      float o = 0.f, l = 0.f;
      for (int k = i; k <= last; ++k)
        if (segs[k].valid) {
          const float* p = pieces + k * STATE;
          const float w = ex2(p[M0 + r] - ref);
          o += w * p[x];
          l += w * p[L0 + r];
        }
      if (f.begin && end) {
        a.out[((int64_t)f.s * a.H + h0) * hd + x] = l == 0.f ? 0.f : o / l;
      } else {
        dst[x] = o;
        if (x % hd == 0) {
          dst[M0 + r] = M;
          dst[L0 + r] = l;
        }
      }
    }
    if (threadIdx.x == 0 && f.begin && !end) {
      // the CTA that holds the item's last unit
      const int us = units_of(keys_of(b, f.s));
      const int64_t lastu = f.first * KVB + (int64_t)(f.block + 1) * us - 1;
      const int c1 = (int)(owner_of(lastu, units, workers) / aw);
      a.desc[blockIdx.x] = make_int4(f.s, f.block, c1 - (int)blockIdx.x + 1, 0);
    }
    i = j;
  }
}

// Joins the pieces of the items that several CTAs hold: block (c, r) takes
// head r of the item that starts in CTA c.  The weights of the pieces are
// found by all threads, then the threads share the pieces out: 128 / head_dim
// (at least one) groups of a head's dims.
__global__ void __launch_bounds__(128) merge_kernel(DecodeArgs a) {
  const int4 d = a.desc[blockIdx.x];
  if (d.z == 0) return;
  int h0, nr;
  block_heads(a, d.y, h0, nr);
  const int r = blockIdx.y;
  if (r >= nr) return;
  __shared__ float red[4], so[128];
  const int STATE = state_floats(a.hd), hd = a.hd, M0 = 8 * hd + r, L0 = 8 * hd + 8 + r;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto piece = [&](int k) { return a.part + ((size_t)(blockIdx.x + k) * 2 + (k == 0 ? 1 : 0)) * STATE; };
  float M = -INFINITY;
  for (int k = tid; k < d.z; k += 128) M = fmaxf(M, piece(k)[M0]);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) red[warp] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = ref_of(M);
  const int groups = 128 / hd, x = tid % hd, grp = tid / hd;
  float o = 0.f, l = 0.f;
#pragma unroll 8
  for (int k = grp; k < d.z; k += groups) {
    const float* p = piece(k);
    const float w = ex2(p[M0] - ref);
    o += w * p[r * hd + x];
    l += w * p[L0];
  }
  so[tid] = o;
  __syncthreads();
  if (tid < hd) {
    for (int k = 1; k < groups; ++k) o += so[tid + k * hd];
  }
  __syncthreads();
  so[tid] = l;
  __syncthreads();
  if (tid < hd) {
    for (int k = 1; k < groups; ++k) l += so[tid + k * hd];
    a.out[((int64_t)d.x * a.H + h0 + r) * hd + x] = l == 0.f ? 0.f : o / l;
  }
}

// ---- host ---------------------------------------------------------------------

constexpr int kMaxPerSm = 2;  // CTAs an SM at most (DecodeShape::CTAS)

// desc | CTA pieces | warp pieces
size_t decode_workspace(int hd) {
  const size_t ctas = (size_t)sm_count() * kMaxPerSm;
  return ctas * (sizeof(int4) + (2 + 2 * kDecodeWarps) * state_floats(hd) * sizeof(float));
}

template <int HDF, typename KT>
static int32_t launch(const DecodeArgs& a, cudaStream_t st) {
  using S = DecodeShape<HDF, KT>;
  auto kern = decode_kernel<HDF, KT>;
  constexpr int smem = kDecodeWarps * S::RING;
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
  const int64_t most = (int64_t)a.b.n * (a.b.kv_heads / a.F) * a.HB *
                       std::max<int64_t>(1, (a.b.max_len + kTile - 1) / kTile);
  const int grid = (int)std::min<int64_t>((int64_t)sm_count() * S::CTAS, most);
  kern<<<grid, kDecodeThreads, smem, st>>>(a);
  Q6W_LAUNCH_CHECK("decode_kernel");
  merge_kernel<<<dim3(grid, std::min(8, a.F > 1 ? a.F * a.b.rep : a.per)), 128, 0, st>>>(a);
  Q6W_LAUNCH_CHECK("merge_kernel");
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
  if (a.b.head_stride == a.hd)
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

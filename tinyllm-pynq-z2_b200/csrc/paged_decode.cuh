// Decode attention over paged caches: one query token a sequence.
//
// Mathematics.  One pass over the keys with a running maximum m, sum l and
// output o per query head: p = 2^(s - m), l += p, o += p v, everything scaled
// by 2^(m_old - m_new) when the maximum grows; partial states of disjoint key
// ranges join as m = max m_i, l = sum l_i 2^(m_i - m), o = sum o_i 2^(m_i - m).
// All of it in FP32, FP16 keys and values widened exactly.
//
// Bound.  Every key and value is read once from HBM and used by the `rep`
// query heads of its kv head: 2 rep FMA per element, 4 to 8 flop a byte at
// rep 8, so the memory rate bounds it while the issue slots keep up.
//
// Layout of the work.  An item is (sequence, kv head, block of up to eight
// query heads), cut into units of CH keys.  The units of all items lie on one
// line (a prefix sum of the lengths, taken by every CTA for itself), and every
// warp takes an equal stretch of it: ragged lengths and few long sequences
// balance alike.  A warp that holds an item whole writes its output; pieces
// of an item are joined in shared memory when one CTA holds them all, else
// by merge_kernel.
//
// Inside a warp, L lanes share a key (16 bytes each), G = 32 / L keys side by
// side, U steps of them in registers while the next U are on their way.  A
// lane's partial dot products of U keys with R heads are summed over the L
// lanes by halving exchanges, after which each lane owns NS finished scores:
// U R - 1 shuffles instead of U R log2(L).  The weights go back to the lanes
// by one shuffle each.
#pragma once

#include "paged.cuh"

namespace q6w {
namespace paged {

constexpr int kDecodeWarps = 8;
constexpr int kDecodeThreads = 32 * kDecodeWarps;

// A partial state: o[R][HD], m[R], l[R], in a whole number of 16-byte units.
__host__ __device__ constexpr int state_floats(int hd, int r) { return r * hd + (r > 1 ? 2 * r : 4); }

template <int HD, typename KT, int R>
struct DecodeShape {
  static constexpr int EPL = 16 / (int)sizeof(KT);  // elements of a key that a lane holds
  static constexpr int L = HD / EPL;                // lanes of a key
  static constexpr int G = 32 / L;                  // keys side by side
  static constexpr int U = R * EPL > 16 ? 2 : 4;    // steps of an iteration
  static constexpr int CTAS = R * EPL > 32 ? 1 : 2; // CTAs an SM: 64 + 64 registers of q and o leave room for one
  static constexpr int STG = CTAS == 1 ? 8 : (U == 4 ? 3 : 4);  // iterations in the ring: 8 to 16 KB a warp
  static constexpr int KPI = G * U;                 // keys of an iteration
  static constexpr int CH = KPI > 16 ? KPI : 16;    // keys of a unit
  static constexpr int NV = U * R;
  static constexpr int NS = NV > L ? NV / L : 1;    // scores that a lane owns
  static constexpr int DUP = NV < L ? L / NV : 1;   // lanes that own the same score
  static constexpr int RL = NS < R ? NS : R;        // query heads among them
  static constexpr int STATE = state_floats(HD, R);
  // a warp's shared memory: the state of its first piece, the ring (and in it, once
  // it has been consumed, the state of its last piece)
  static constexpr int RING = STG * U * 2 * 512;
  static constexpr int WARP = STATE * 4 + (RING > STATE * 4 ? RING : STATE * 4);
};

struct DecodeArgs {
  Batch b;
  const float* q;
  int64_t ldq;
  float* out;
  float* part;      // [CTA][2][STATE]
  int4* desc;       // [CTA]: item that starts in the CTA and goes on: {s, block, CTAs, 0}
  int32_t H, HB, per;  // query heads, head blocks of a kv head, heads of a block
  float scale;      // log2(e) / sqrt(head_dim)
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A maximum to subtract: nothing seen yet counts as 0, so that the weights are 2^-inf = 0.
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ void widen16(const uint4& w, float2 (&x)[2]) {
  x[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
  x[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ void widen16(const uint4& w, float2 (&x)[4]) {
  const __half2* h = reinterpret_cast<const __half2*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __half22float2(h[i]);
}

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

template <int CH>
__device__ __forceinline__ int units_of(int keys) {
  return max(1, (keys + CH - 1) / CH);
}

template <int CH>
__device__ void build_line(const Batch& b, Line& line) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seg = (b.n + kDecodeThreads - 1) / kDecodeThreads;
  int64_t sum = 0;
  for (int s = tid * seg; s < min((tid + 1) * seg, b.n); ++s) {
    const int len = __ldg(b.lengths + s);
    if (len > b.max_len) flag(b.status, kErrInput);
    sum += units_of<CH>(min(max(len, 0), b.max_len));
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
template <int CH>
__device__ void find_seq(const Batch& b, const Line& line, int64_t z, int lane, int& s, int64_t& first) {
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
    const int u = i < b.n ? units_of<CH>(keys_of(b, i)) : 0;
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
template <int CH>
struct Cursor {
  int64_t x, x1, first;
  int s, block, keys, us, u0, u1, key0, key1;
  __device__ __forceinline__ void piece() {
    u1 = (int)min((int64_t)us, u0 + (x1 - x));
    key0 = u0 * CH;
    key1 = min(u1 * CH, keys);
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
        us = units_of<CH>(keys);
      }
    }
    piece();
  }
};

// 16 bytes from global to shared memory, or 16 zero bytes.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int HD, typename KT, int R>
__global__ void __launch_bounds__(kDecodeThreads, DecodeShape<HD, KT, R>::CTAS) decode_kernel(DecodeArgs a) {
  using S = DecodeShape<HD, KT, R>;
  constexpr int EPL = S::EPL, L = S::L, G = S::G, U = S::U, NS = S::NS, RL = S::RL, DUP = S::DUP, CH = S::CH;
  constexpr int E2 = EPL / 2;
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int STG = S::STG;
  extern __shared__ __align__(16) uint8_t smem[];  // [warp][WARP]
  __shared__ Line line;
  __shared__ Seg segs[2 * kDecodeWarps];
  const Batch& b = a.b;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int li = lane & (L - 1), g = lane / L, gbase = lane & ~(L - 1);
  build_line<CH>(b, line);
  const int KVB = b.kv_heads * a.HB;
  const int64_t units = line.total * KVB;
  // few units: spread them over the CTAs first, over a CTA's warps second
  const int aw = (int)min((int64_t)kDecodeWarps, (units + gridDim.x - 1) / gridDim.x);
  const int64_t workers = min((int64_t)gridDim.x * aw, units);
  const int64_t wi = (int64_t)blockIdx.x * aw + warp;
  const bool active = warp < aw && wi < workers;
  if (lane < 2) segs[2 * warp + lane].valid = 0;
  uint8_t* mine = smem + warp * S::WARP;
  if (active) {
    Cursor<CH> c;
    c.x = wi * units / workers;
    c.x1 = (wi + 1) * units / workers;
    const int64_t xb = c.x;
    find_seq<CH>(b, line, c.x / KVB, lane, c.s, c.first);
    c.keys = keys_of(b, c.s);
    c.us = units_of<CH>(c.keys);
    c.block = (int)((c.x - c.first * KVB) / c.us);
    c.u0 = (int)((c.x - c.first * KVB) % c.us);
    c.piece();
    // The loads run STG - 1 iterations ahead of the arithmetic, over the ends
    // of items, into a ring that is private to each lane (a lane reads the 16
    // bytes that it copied itself, so waiting for its own copies is enough).
    const uint32_t ring = smem_u32(mine) + S::STATE * 4 + lane * 16;
    const uint4* ring_g = reinterpret_cast<const uint4*>(mine + S::STATE * 4) + lane;
    Cursor<CH> p = c;
    const KT* kb = static_cast<const KT*>(b.k) + li * EPL;
    const KT* vb = static_cast<const KT*>(b.v) + li * EPL;
    const int32_t* row = b.table;
    int pt = 0, pbase = 0, plast = -1, ids = -1;  // page ids: lane i holds the id of page pbase + i
    int64_t hoff = 0;
    uint32_t bad = 0;  // bit stage * U + u: the key's page id is out of range
    auto enter = [&]() {  // the first piece from p on that has keys
      while (p.x < p.x1 && p.key0 >= p.key1) p.next(b, KVB);
      if (p.x >= p.x1) return;
      pt = p.key0;
      row = b.table + p.s * b.table_stride;
      pbase = p.key0 >> b.shift;
      plast = (p.key1 - 1) >> b.shift;
      ids = pbase + lane <= plast ? __ldg(row + pbase + lane) : -1;
      hoff = (p.block / a.HB) * b.head_stride;
    };
    auto issue = [&](int stage) {
      if (p.x < p.x1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int tl = pt + u * G;  // first key of the step
          if (tl < p.key1 && ((min(tl + G, p.key1) - 1) >> b.shift) >= pbase + 32) {  // warp-uniform
            pbase = tl >> b.shift;
            ids = pbase + lane <= plast ? __ldg(row + pbase + lane) : -1;
          }
          const int t = tl + g;
          const int id = __shfl_sync(kAll, ids, ((t >> b.shift) - pbase) & 31);
          const bool in = t < p.key1, ok = (unsigned)id < (unsigned)b.n_pages;
          const int64_t off =
              in && ok ? id * b.page_stride + (int64_t)(t & ((1 << b.shift) - 1)) * b.slot_stride + hoff : 0;
          const uint32_t dst = ring + (stage * U + u) * 1024;
          copy16(dst, kb + off, in && ok);
          copy16(dst + 512, vb + off, in && ok);
          const uint32_t bit = 1u << (stage * U + u);
          bad &= ~bit;
          if (in && !ok) {
            bad |= bit;
            flag(b.status, kErrInput);
          }
        }
        pt += S::KPI;
        if (pt >= p.key1) {
          p.next(b, KVB);
          enter();
        }
      }
      copy_commit();
    };
    enter();
#pragma unroll
    for (int i = 0; i < STG - 1; ++i) issue(i);
    int stage = 0;
    while (c.x < c.x1) {
      const int key0 = c.key0, key1 = c.key1, s = c.s, block = c.block;
      const int kvh = block / a.HB, hb = block - kvh * a.HB;
      const int h0 = kvh * b.rep + hb * a.per;  // first query head of the block
      const int nr = min(a.per, b.rep - hb * a.per);
      float2 q2[R][E2], acc[R][E2];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float* qp = a.q + s * a.ldq + (int64_t)(h0 + r) * HD + li * EPL;
#pragma unroll
        for (int e = 0; e < E2; e += 2) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < nr) v = __ldg(reinterpret_cast<const float4*>(qp + 2 * e));
          q2[r][e] = make_float2(v.x, v.y);
          q2[r][e + 1] = make_float2(v.z, v.w);
          acc[r][e] = acc[r][e + 1] = make_float2(0.f, 0.f);
        }
      }
      float m[RL], l[RL];
#pragma unroll
      for (int i = 0; i < RL; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      for (int t0 = key0; t0 < key1; t0 += S::KPI) {
        copy_wait<STG - 2>();
        issue(stage == 0 ? STG - 1 : stage - 1);
        const uint4* rg = ring_g + stage * U * 64;
        float sc[S::NV];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float2 kx[E2];
          uint4 kw = rg[u * 64];
          if (bad >> (stage * U + u) & 1) kw = make_uint4(~0u, ~0u, ~0u, ~0u);  // NaN score, NaN row
          widen16(kw, kx);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            float2 d = make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < E2; ++e) d = __ffma2_rn(q2[r][e], kx[e], d);
            sc[u * R + r] = d.x + d.y;
          }
        }
        // halving exchange over the key's lanes
        int cnt = S::NV;
#pragma unroll
        for (int o = L / 2; o >= 1; o >>= 1) {
          if (cnt > 1) {
            cnt >>= 1;
            const bool up = (lane & o) != 0;
#pragma unroll
            for (int i = 0; i < S::NV / 2; ++i)
              if (i < cnt) {
                const float send = up ? sc[i] : sc[i + cnt], keep = up ? sc[i + cnt] : sc[i];
                sc[i] = keep + __shfl_xor_sync(kAll, send, o);
              }
          } else {
            sc[0] += __shfl_xor_sync(kAll, sc[0], o);
          }
        }
        // this lane's scores: index (li / DUP) NS + j = u R + r
        const int idx0 = (li / DUP) * NS;
        float mx[RL];
#pragma unroll
        for (int i = 0; i < RL; ++i) mx[i] = m[i];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int u = (idx0 + j) / R;
          const bool in = t0 + u * G + g < key1;
          sc[j] = in ? sc[j] * a.scale : -INFINITY;
          mx[j % RL] = fmaxf(mx[j % RL], sc[j]);
        }
        bool grew = false;
#pragma unroll
        for (int i = 0; i < RL; ++i) {
#pragma unroll
          for (int o = (R / RL) * DUP; o < L; o <<= 1) mx[i] = fmaxf(mx[i], __shfl_xor_sync(kAll, mx[i], o));
          grew |= mx[i] != m[i];
        }
        if (__any_sync(kAll, grew)) {
          float al[RL];
#pragma unroll
          for (int i = 0; i < RL; ++i) {
            al[i] = ex2(m[i] - ref_of(mx[i]));
            l[i] *= al[i];
            m[i] = mx[i];
          }
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float f = __shfl_sync(kAll, al[r % RL], gbase + (r / RL) * DUP);
            const float2 f2 = make_float2(f, f);
#pragma unroll
            for (int e = 0; e < E2; ++e) acc[r][e] = __fmul2_rn(acc[r][e], f2);
          }
        }
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          sc[j] = ex2(sc[j] - ref_of(m[j % RL]));
          l[j % RL] += sc[j];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float2 vx[E2];
          widen16(rg[u * 64 + 32], vx);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            constexpr int kDiv = NS;
            const int idx = u * R + r;
            const float p = __shfl_sync(kAll, sc[idx % NS], gbase + (DUP > 1 ? idx * DUP : idx / kDiv));
            const float2 p2 = make_float2(p, p);
#pragma unroll
            for (int e = 0; e < E2; ++e) acc[r][e] = __ffma2_rn(p2, vx[e], acc[r][e]);
          }
        }
        stage = stage + 1 == STG ? 0 : stage + 1;
      }
      // join the G groups: every lane ends with the item's m, l of its own heads
      float w[RL];
#pragma unroll
      for (int i = 0; i < RL; ++i) {
#pragma unroll
        for (int o = (R / RL) * DUP; o < L; o <<= 1) l[i] += __shfl_xor_sync(kAll, l[i], o);
        float M = m[i];
#pragma unroll
        for (int o = L; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(kAll, M, o));
        w[i] = ex2(m[i] - ref_of(M));
        m[i] = M;
        l[i] *= w[i];
#pragma unroll
        for (int o = L; o < 32; o <<= 1) l[i] += __shfl_xor_sync(kAll, l[i], o);
      }
      const bool begin = c.u0 == 0, end = c.u1 == c.us;
      // (a last piece's slot lies in the ring: its loads have been consumed, but
      // every lane has to be past its own)
      const int which = c.x == xb ? 0 : 1;
      float* slot = reinterpret_cast<float*>(mine + which * S::STATE * 4);
      if (which) {
        copy_wait<0>();
        __syncwarp();
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int src = gbase + (r / RL) * DUP;
        const float f = __shfl_sync(kAll, w[r % RL], src);
        const float lr = __shfl_sync(kAll, l[r % RL], src);
        const float mr = __shfl_sync(kAll, m[r % RL], src);
        float o2[EPL];
#pragma unroll
        for (int e = 0; e < E2; ++e) {
          float2 v = __fmul2_rn(acc[r][e], make_float2(f, f));
#pragma unroll
          for (int o = L; o < 32; o <<= 1) {
            v.x += __shfl_xor_sync(kAll, v.x, o);
            v.y += __shfl_xor_sync(kAll, v.y, o);
          }
          o2[2 * e] = v.x;
          o2[2 * e + 1] = v.y;
        }
        if (r % G == g) {  // the groups share the stores
          if (begin && end) {
            const float inv = lr == 0.f ? 0.f : 1.f / lr;
            if (r < nr) {
              float* op = a.out + ((int64_t)s * a.H + h0 + r) * HD + li * EPL;
#pragma unroll
              for (int e = 0; e < EPL; e += 4)
                *reinterpret_cast<float4*>(op + e) =
                    make_float4(o2[e] * inv, o2[e + 1] * inv, o2[e + 2] * inv, o2[e + 3] * inv);
            }
          } else {
            if (li == 0) {
              slot[R * HD + r] = mr;
              slot[R * HD + R + r] = lr;
            }
#pragma unroll
            for (int e = 0; e < EPL; e += 4)
              *reinterpret_cast<float4*>(slot + r * HD + li * EPL + e) =
                  make_float4(o2[e], o2[e + 1], o2[e + 2], o2[e + 3]);
          }
        }
      }
      if (lane == 0 && !(begin && end)) segs[2 * warp + which] = {c.first, s, block, 1, begin, end};
      c.next(b, KVB);
    }
  }
  __syncthreads();
  // ---- pieces of items inside this CTA, in order
  auto state_of = [&](int k) {
    return reinterpret_cast<const float*>(smem + (k >> 1) * S::WARP + (k & 1) * S::STATE * 4);
  };
  if (threadIdx.x == 0) a.desc[blockIdx.x].z = 0;
  for (int i = 0; i < 2 * kDecodeWarps;) {
    if (!segs[i].valid) {
      ++i;
      continue;
    }
    int j = i, last = i;
    for (++j; j < 2 * kDecodeWarps; ++j) {
      if (!segs[j].valid) continue;
      if (segs[j].s != segs[i].s || segs[j].block != segs[i].block) break;
      last = j;
    }
    const Seg f = segs[i];
    const bool end = segs[last].end;
    const int kvh = f.block / a.HB, hb = f.block - kvh * a.HB;
    const int nr = min(a.per, b.rep - hb * a.per);
    float* dst = a.part + ((size_t)blockIdx.x * 2 + (f.begin ? 1 : 0)) * S::STATE;
    for (int x = threadIdx.x; x < R * HD; x += kDecodeThreads) {
      const int r = x / HD;
      float M = -INFINITY;
      for (int k = i; k <= last; ++k)
        if (segs[k].valid) M = fmaxf(M, state_of(k)[R * HD + r]);
      const float ref = ref_of(M);
      float o = 0.f, lsum = 0.f;
      for (int k = i; k <= last; ++k)
        if (segs[k].valid) {
          const float* p = state_of(k);
          const float w = ex2(p[R * HD + r] - ref);
          o += w * p[x];
          lsum += w * p[R * HD + R + r];
        }
      if (f.begin && end) {
        if (r < nr)
          a.out[((int64_t)f.s * a.H + kvh * b.rep + hb * a.per) * HD + x] = lsum == 0.f ? 0.f : o / lsum;
      } else {
        dst[x] = o;
        if (x % HD == 0) {
          dst[R * HD + r] = M;
          dst[R * HD + R + r] = lsum;
        }
      }
    }
    if (threadIdx.x == 0 && f.begin && !end) {
      // the CTA that holds the item's last unit
      const int us = units_of<CH>(keys_of(b, f.s));
      const int64_t lastu = f.first * KVB + (int64_t)(f.block + 1) * us - 1;
      const int c1 = (int)(owner_of(lastu, units, workers) / aw);
      a.desc[blockIdx.x] = make_int4(f.s, f.block, c1 - (int)blockIdx.x + 1, 0);
    }
    i = j;
  }
}

// Joins the pieces of the items that several CTAs hold: block (c, y) takes
// its share of the outputs of the item that starts in CTA c.
template <int HD, int R>
__global__ void __launch_bounds__(128) merge_kernel(DecodeArgs a) {
  constexpr int STATE = state_floats(HD, R), M0 = R * HD, L0 = R * HD + R;
  const int4 d = a.desc[blockIdx.x];
  if (d.z == 0) return;
  const int kvh = d.y / a.HB, hb = d.y - kvh * a.HB;
  const int nr = min(a.per, a.b.rep - hb * a.per);
  const int x = blockIdx.y * 128 + threadIdx.x;
  if (x >= nr * HD) return;
  const int r = x / HD;
  const float* p0 = a.part + ((size_t)blockIdx.x * 2 + 1) * STATE;
  float M = p0[M0 + r];
  for (int k = 1; k < d.z; ++k) M = fmaxf(M, a.part[(size_t)(blockIdx.x + k) * 2 * STATE + M0 + r]);
  const float ref = ref_of(M);
  float w = ex2(p0[M0 + r] - ref);
  float o = w * p0[x], l = w * p0[L0 + r];
#pragma unroll 8
  for (int k = 1; k < d.z; ++k) {
    const float* p = a.part + (size_t)(blockIdx.x + k) * 2 * STATE;
    w = ex2(p[M0 + r] - ref);
    o += w * p[x];
    l += w * p[L0 + r];
  }
  a.out[((int64_t)d.x * a.H + kvh * a.b.rep + hb * a.per) * HD + x] = l == 0.f ? 0.f : o / l;
}

int32_t decode_attention(const DecodeArgs& a, int hd, bool half, cudaStream_t st);
size_t decode_workspace(int hd);

}  // namespace paged
}  // namespace q6w

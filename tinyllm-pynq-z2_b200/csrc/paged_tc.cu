// Attention of many query rows over the same paged keys, on tcgen05: prompts
// and chunks of prompts (causal), and a batch over its shared prefix.
//
// Mathematics.  The rows that share a kv head's keys are the query tokens times
// the `rep` heads of the group: row = token rep + r.  A CTA holds a block of
// 128 (256) rows and walks over its keys in units of 128 (FP16 pages) or 64
// (FP32): S = Q K^T, p = 2^(c s - m) with a reference m a row that moves only
// when a score passes it by a bound (Weights), l += p, O += P V.  Pieces of a
// block's keys join as in the decode kernel.
//
// Operands.  FP16 pages: K and V enter as they are, Q (scaled by a power of
// two a row, half_scale) and P as FP16 hi + lo, 22 bits: 2 + 2 MMAs.  FP32 pages: every
// operand enters as three BF16 parts (24 bits) and the products down to
// 2^-16 are kept, 6 + 6 MMAs, the small ones first.  Q and P are the MMA's A
// operand and live in tensor memory, where the softmax threads (one row each:
// TMEM lane = row) write them; P overlays the S that it was made from.  K is
// the K-major and V the MN-major B operand, both rows of keys as they lie in
// the pages, so nothing is transposed.
//
// Sums.  The MMA's FP32 accumulator loses up to a unit in the last place with
// every added product (the sum is cut, not rounded), so O stays in it for kFlush
// units only and is then added to the row's registers, rounded to nearest.
//
// Bound.  Per unit and 128 rows: 2 (12) x 128 x keys x head_dim x 2 MMA flop, 128
// x keys exponentials and about ten FP32 instructions a score; with two row
// tiles in a CTA (head_dim <= 64) the softmax of one runs under the MMAs of the
// other, with one tile (head_dim 128) S has two buffers.  An MMA takes about 60
// cycles whether N is 64 or 128, so O is one MMA wide where head_dim is 128.
// Measured (ten calls in a graph, a call among others): 2 x 2048 tokens behind up to 6144,
// FP16, 32 heads over 8 kv heads of 128: 840-890 us for 344 GFLOP, 385-410 TFLOP/s; 1024
// tokens of 32 heads over 4 kv heads of 64 and 4096 FP32 keys, with their own 20-148
// keys: 340-350 us for 35 GFLOP, of which this kernel about 265, each tile behind its
// chain softmax -> PV -> QK (tensor pipe 23% busy).  Blocks of few rows cost as
// much as full ones: 64 requests with one token each, behind 128-16384 FP16 keys, take
// 434 us here and 103 in the decode kernel.
//
// Roles: eight softmax warps (four a tile; with one tile two threads a row, each
// half of the keys and of O), four load warps, one MMA warp.
// Load warps fetch FP16 units by TMA boxes; FP32 units, units with a bad page
// id and units that some row does not see whole go through registers: keys no
// row sees become zeros, and a key whose value is not finite becomes a NaN key
// with zero values, so that only the rows that see it become NaN.  The softmax
// warps make rows whose sum of weights is not a number anew at their end (plain_row).
//
// Blocks' units lie on one line; every CTA takes an equal stretch (as the
// decode kernel's warps do).  Every wait is bounded; a timeout sets the status
// bit, makes the CTA stop and its rows NaN.
#include <cuda.h>
#include <cuda_bf16.h>

#include <string.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "paged.cuh"
#include "tc.cuh"

namespace q6w {
namespace paged {

constexpr int kTcMaxStages = 4;

template <int HD, typename KT>
struct TcShape {
  static constexpr bool kHalf = std::is_same<KT, __half>::value;
  static constexpr int TILES = HD <= 64 ? 2 : 1;   // row tiles of a CTA
  static constexpr int BUFS = 3 - TILES;           // S buffers of a tile
  static constexpr int ROWS = 128 * TILES;
  static constexpr int KEYS = kHalf ? 128 : 64;
  static constexpr int QP = kHalf ? 2 : 3;         // parts of Q and P
  static constexpr int KP = kHalf ? 1 : 3;         // parts of K and V
  // product x takes part pa(x) of A and pb(x) of B
  static constexpr int pa(int x) { return kHalf ? 1 - x : (0x046 >> 2 * x) & 3; }
  static constexpr int pb(int x) { return kHalf ? 0 : (0x124 >> 2 * x) & 3; }
  static constexpr int RB = HD * 2 < 128 ? HD * 2 : 128;  // bytes of a panel row = swizzle span
  static constexpr int PANELS = HD * 2 / RB;
  static constexpr int PANEL = KEYS * RB;
  static constexpr int PART = PANEL * PANELS;      // bytes of a unit's keys (or values), one part
  static constexpr int HALF = KP * PART;
  static constexpr int STG = 192 * 1024 / (2 * HALF) < kTcMaxStages ? 192 * 1024 / (2 * HALF) : kTcMaxStages;
  // tensor memory columns of a tile: Q parts, S / P buffers, O
  static constexpr int QC = (QP * HD / 2 + 31) / 32 * 32;
  static constexpr int SC = kHalf ? KEYS : 96;     // P: QP x KEYS / 2 columns over S
  static constexpr int S0 = kHalf ? 0 : 32;        // S inside its buffer (P's first chunk stays in front of unread S)
  static constexpr int TC = QC + BUFS * SC + (HD < 32 ? 32 : HD);
  static_assert(TC * TILES <= 512, "tensor memory columns");
  static constexpr int HALVES = 3 - TILES;         // threads of a row: each takes half of the keys and of O
  static constexpr int SOFT = 8;                   // softmax warps
  // Softmax, load and MMA warps in groups of four with registers of their own
  // (what the block was launched with, 64 K / THREADS a thread, divided anew).
  static constexpr int THREADS = 32 * (SOFT + 8);
  static constexpr int REGS = 128;
  static constexpr int SOFT_REGS = 160, LOAD_REGS = 96, MMA_REGS = 96;
  static_assert(SOFT * SOFT_REGS + 4 * LOAD_REGS + 4 * MMA_REGS <= (SOFT + 8) * REGS, "register split");
  // Units between additions of O to registers.  FP32, chunks of 201-597 tokens: errors of
  // 3.4e-7 with every unit, 6.3e-7 with every second (406 against 387 us when it was
  // chosen), the plain FP32 form 6.2e-7.
  static constexpr int kFlush = kHalf ? 4 : 2;
  static constexpr size_t SMEM = 1024 + (size_t)STG * 2 * HALF;
};

// One MMA shared-memory descriptor: rows of RB bytes swizzled over RB, eight-row
// groups RB * 8 bytes apart -- along the MMA's N for the K-major operand (which
// uses no other offset), along its K for the MN-major one, whose panels (spans of
// N) stand `panel` bytes apart.  The upper word is a constant, the lower word
// grows by bytes / 16 with the address.
template <int RB>
struct TileDesc {
  static constexpr uint32_t group = RB * 8 / 16;
  static constexpr uint32_t hi = group | (1u << 14) | ((RB == 128 ? 2u : RB == 64 ? 4u : 6u) << 29);
  __device__ static __forceinline__ uint32_t lo(uint32_t addr, int panel = 0) {
    return (addr >> 4) | ((panel ? panel / 16 : group) << 16);
  }
};

// D (tensor memory) += A (tensor memory, a + ADD) B (shared memory, b + BDD);
// `add` false: D = A B.  The constants are added inside, not held in registers.
template <int ADD, int BDD, uint32_t HI>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 bd;\n\t.reg .b32 al, bl;\n\t"
      "add.u32 al, %1, %5;\n\tadd.u32 bl, %2, %6;\n\t"
      "mov.b64 bd, {bl, %7};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [al], bd, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "n"(ADD), "n"(BDD), "n"(HI)
      : "memory");
}
// True in one lane of the (converged) warp, the same one each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

// f(0), f(1), .. f(N - 1) with the index a constant.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(const F& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    unrolled<N, I + 1>(f);
  }
}

// Byte place of byte `at` of row `row` in a swizzled panel.
template <int RB>
__device__ __forceinline__ int panel_place(int row, int at) {
  const int x = row * RB + at;
  return RB == 128 ? x ^ ((x >> 3) & 0x70) : RB == 64 ? x ^ ((x >> 3) & 0x30) : x ^ ((x >> 3) & 0x10);
}

// 32 (16) consecutive FP32 columns of this thread's TMEM lane.  The wait names the
// destination registers, so no use of them is scheduled before it.
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t at, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}

// A thread's registers from here on, `FROM` before (a whole group of four warps calls it).
template <int FROM, int TO>
__device__ __forceinline__ void set_registers() {
  if constexpr (TO > FROM)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TO));
  else if constexpr (TO < FROM)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TO));
}

// The AND of `ok` over the four load warps (all of them call it).
__device__ __forceinline__ bool load_warps_agree(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.aligned.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// (x, y) -> BF16, rounded to nearest; what would round to infinity becomes the
// largest number (infinity too).
__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
  uint32_t w;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(y), "f"(x));
  return w;
}

// Two values -> packed parts, first value in the low half.  BF16: the first part of
// a value close to FP32's largest must not round to infinity (a hidden key's weight of
// 0 would make it NaN); of an infinity the second part is one.
template <bool HALF_PARTS, int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (HALF_PARTS) {
      const __half2 h = __floats2half2_rn(x, y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
      if (i + 1 < N) {
        const float2 f = __half22float2(h);
        x -= f.x;
        y -= f.y;
      }
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      w[i] = i == 0 ? bf16_pair(x, y) : *reinterpret_cast<const uint32_t*>(&h);
      if (i + 1 < N) {
        x -= __uint_as_float(w[i] << 16);
        y -= __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}

// ---- the line of units -----------------------------------------------------------

// A block of rows of one (sequence, kv head) and a stretch [u0, u1) of its units.
struct Piece {
  int64_t x;              // the line's unit at u0
  int s, kv, j;           // sequence, kv head, row block
  int tok0, count, past;  // first query token and tokens of the sequence, cached tokens in front of them
  int keys, units;        // keys that the block's last row sees, units of the block
  int u0, u1;
};

template <int ROWS, int KEYS>
struct Walk {
  const TcArgs& a;
  Piece p;
  int64_t end;
  __device__ Walk(const TcArgs& args) : a(args) {}
  __device__ __forceinline__ int rep() const { return a.b.rep; }
  __device__ __forceinline__ int seen(int tok) const {  // keys that token tok (0 .. count-1) sees
    return a.prefix ? a.prefix_len : min(max(p.past + tok + 1, 0), a.b.max_len);
  }
  __device__ __forceinline__ int rows() const { return min(ROWS, p.count * rep() - p.j * ROWS); }
  __device__ void sequence() {
    if (a.prefix) {
      p.tok0 = 0;
      p.count = a.b.T;
      p.past = 0;
    } else {
      int t1;
      seq_tokens(a.b, p.s, p.tok0, t1);
      p.count = t1 - p.tok0;
      p.past = max(__ldg(a.b.lengths + p.s), 0) - p.count;
    }
  }
  __device__ void block() {
    p.keys = seen((p.j * ROWS + rows() - 1) / rep());
    p.units = max(1, (p.keys + KEYS - 1) / KEYS);
  }
  __device__ int blocks() const { return (p.count * rep() + ROWS - 1) / ROWS; }
  __device__ void begin(int64_t x, int64_t x1) {
    p.x = x;
    end = x1;
    if (x >= x1) return;
    int64_t rem = x;
    p.s = 0;
    if (a.prefix) {
      sequence();
      const int per = max(1, (a.prefix_len + KEYS - 1) / KEYS), nb = blocks();
      p.kv = (int)muldiv(rem, 1, (int64_t)per * nb);
      rem -= (int64_t)p.kv * per * nb;
      p.j = (int)muldiv(rem, 1, per);
      rem -= (int64_t)p.j * per;
      block();
    } else {
      int lo = 0, hi = a.b.n;  // line[lo] kv_heads <= x < line[hi] kv_heads
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.line[mid] * a.b.kv_heads <= x) lo = mid; else hi = mid;
      }
      p.s = lo;
      rem -= a.line[lo] * a.b.kv_heads;
      sequence();
      const int64_t per = a.line[lo + 1] - a.line[lo];
      p.kv = (int)muldiv(rem, 1, per);
      rem -= p.kv * per;
      for (p.j = 0;; ++p.j) {
        block();
        if (rem < p.units) break;
        rem -= p.units;
      }
    }
    p.u0 = (int)rem;
    p.u1 = (int)min((int64_t)p.units, rem + (x1 - x));
  }
  __device__ __forceinline__ bool more() const { return p.x < end; }
  __device__ void next() {
    p.x += p.u1 - p.u0;
    if (p.x >= end) return;
    if (++p.j >= blocks()) {
      p.j = 0;
      if (++p.kv == a.b.kv_heads) {
        p.kv = 0;
        do {
          ++p.s;
          sequence();
        } while (p.count == 0);
      }
    }
    block();
    p.u0 = 0;
    p.u1 = (int)min((int64_t)p.units, end - p.x);
  }
};

// Prefix sums of the sequences' units of one kv head, line[0 .. n].
template <int ROWS, int KEYS>
__global__ void __launch_bounds__(1024) line_kernel(TcArgs a, int64_t* line) {
  __shared__ int64_t part[32];
  __shared__ int64_t carry;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    carry = 0;
    line[0] = 0;
  }
  Walk<ROWS, KEYS> w(a);
  for (int base = 0; base < a.b.n; base += 1024) {
    __syncthreads();
    const int s = base + tid;
    int64_t u = 0;
    if (s < a.b.n) {
      if (__ldg(a.b.lengths + s) > a.b.max_len) flag(a.b.status, kErrInput);
      check_tokens(a.b, s);
      w.p.s = s;
      w.sequence();
      const int nb = w.blocks();
      for (w.p.j = 0; w.p.j < nb; ++w.p.j) {
        w.block();
        u += w.p.units;
      }
    }
    int64_t incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    int64_t before = carry, total = 0;
    for (int i = 0; i < 32; ++i) {
      if (i < warp) before += part[i];
      total += part[i];
    }
    if (s < a.b.n) line[s + 1] = before + incl;
    __syncthreads();
    if (tid == 0) carry += total;
  }
}

// ---- the kernel ----------------------------------------------------------------------

template <int HD, typename KT>
__global__ void __launch_bounds__(TcShape<HD, KT>::THREADS, 1)
    rows_kernel(const TcArgs a, const __grid_constant__ TcMaps maps) {
  using S = TcShape<HD, KT>;
  constexpr bool kHalf = S::kHalf;
  constexpr int KEYS = S::KEYS, STG = S::STG, TILES = S::TILES, BUFS = S::BUFS, QP = S::QP, RB = S::RB;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t k_full[STG], k_empty[STG], v_full[STG], v_empty[STG];
  __shared__ uint64_t q_full[TILES], s_full[2], p_full[2], pv_done[TILES], drain;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int stop;
  __shared__ float row_max[S::HALVES][2][128], row_sum[S::HALVES][128];  // what a row's two threads tell one another
  __shared__ uint32_t odd_keys[4];  // keys of the unit whose values are not finite
  __shared__ int odd[S::SOFT];      // a row of the softmax warp's has a sum of weights that is not a number
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  if (warp == S::SOFT + 4) {
    tc::tmem_alloc(&tmem_base, 512);
    tc::tmem_relinquish();
  }
  if (tid == 0) {
    if (!a.prefix) a.desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
    for (int i = 0; i < STG; ++i) {
      mbar_init(k_full + i, a.stall && blockIdx.x == 0 && i == 0 ? 5 : 4);
      mbar_init(v_full + i, 4);
      mbar_init(k_empty + i, 1);
      mbar_init(v_empty + i, 1);
    }
    for (int i = 0; i < TILES; ++i) {
      mbar_init(q_full + i, 4 * S::HALVES);
      mbar_init(pv_done + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 4 * S::HALVES);
    }
    mbar_init(&drain, 1);
    stop = 0;
    for (int i = 0; i < S::SOFT; ++i) odd[i] = 0;
    fence_mbar_init();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_base;

  const int64_t units = a.prefix
                            ? (int64_t)a.b.kv_heads * ((a.b.T * a.b.rep + S::ROWS - 1) / S::ROWS) *
                                  max(1, (a.prefix_len + KEYS - 1) / KEYS)
                            : a.line[a.b.n] * a.b.kv_heads;
  const int64_t workers = min((int64_t)gridDim.x, units);
  const int64_t c = blockIdx.x;
  Walk<S::ROWS, KEYS> w(a);
  if (c < workers)
    w.begin(muldiv(c, units, workers), muldiv(c + 1, units, workers));
  else
    w.begin(0, 0);
  const int64_t x0 = w.p.x;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (stop) return false;
    if (mbar_try_wait(bar, parity) || mbar_wait_for(bar, parity, a.wait_cycles)) return true;
    stop = 1;
    flag(a.b.status, kErrTimeout);
    return false;
  };
  auto tile_col = [&](int t) { return tmem + t * S::TC; };
  // Where a walk's piece leaves the state of a row of its block (`orow`: the output's):
  // the outputs' place, and that of (m, l) or null.
  auto place = [&](const Walk<S::ROWS, KEYS>& v, int row, int64_t orow, float*& ml) {
    const bool begin = v.p.u0 == 0;
    if (!a.prefix && begin && v.p.u1 == v.p.units) {
      ml = a.state ? a.state + orow * 2 : nullptr;
      return a.out + orow * HD;
    }
    int64_t at;
    if (a.prefix) {
      // piece k of item (kv, j): the CTA's number among the item's
      const int k = (int)(c - owner_of(v.p.x - v.p.u0, units, workers));
      at = ((int64_t)k * a.items + (int64_t)v.p.kv * v.blocks() + v.p.j) * S::ROWS + row;
    } else {
      at = (c * 2 + (v.p.x == x0 && !begin ? 0 : 1)) * S::ROWS + row;
    }
    ml = a.part_ml + at * 2;
    return a.part + at * HD;
  };
  int loaded = 0;  // units that this (load) warp put into shared memory

  if (warp >= S::SOFT && warp < S::SOFT + 4) {
    // ---- loads
    set_registers<S::REGS, S::LOAD_REGS>();
    const int lt = tid - 32 * S::SOFT, lw = warp - S::SOFT;  // 0..127, 0..3
    const int32_t* row = a.b.table;
    const KT* kpool = static_cast<const KT*>(a.b.k);
    const KT* vpool = static_cast<const KT*>(a.b.v);
    constexpr int EL = 16 / (int)sizeof(KT);             // elements of a 16-byte load
    constexpr int PER = HD / EL;                         // loads of a key
    constexpr int NL = KEYS * PER / 128;                 // loads of a thread for a unit's keys
    const int slot_mask = (1 << a.b.shift) - 1, slot_stride = (int)a.b.slot_stride, head_stride = (int)a.b.head_stride;
    int i = 0;
    bool ok = true;
    // Units through registers, BATCH loads of keys and values a thread at a time.
    constexpr int MOST = kHalf ? 4 : 2, BATCH = NL < MOST ? NL : MOST;
    uint4 rv[BATCH], rk[BATCH];
    int ids[BATCH];  // page ids of the batch to fetch
    auto pages = [&](const Piece& p, int u, int n0) {
#pragma unroll
      for (int n = 0; n < BATCH; ++n) {
        const int key = u * KEYS + ((n0 + n) * 128 + lt) / PER;
        ids[n] = key < p.keys ? __ldg((a.prefix ? a.b.table : a.b.table + p.s * a.b.table_stride) + (key >> a.b.shift)) : -1;
      }
    };
    auto fetch = [&](const Piece& p, int u, int n0, int n) {
      const int idx = (n0 + n) * 128 + lt, k = idx / PER, e = (idx - k * PER) * EL, key = u * KEYS + k;
      rk[n] = rv[n] = make_uint4(0u, 0u, 0u, 0u);
      if (key < p.keys) {
        if ((unsigned)ids[n] < (unsigned)a.b.n_pages) {
          const int64_t at = ids[n] * a.b.page_stride + ((key & slot_mask) * slot_stride + p.kv * head_stride + e);
          rv[n] = __ldcg(reinterpret_cast<const uint4*>(vpool + at));
          rk[n] = __ldcg(reinterpret_cast<const uint4*>(kpool + at));
        } else {
          rk[n] = make_uint4(~0u, ~0u, ~0u, ~0u);
          flag(a.b.status, kErrInput);
        }
      }
    };
    auto store = [&](uint8_t* kd, uint8_t* vd, bool whole, int n0, int n) {
      const int idx = (n0 + n) * 128 + lt, k = idx / PER, e = (idx - k * PER) * EL;
      if (!whole && (odd_keys[k >> 5] >> (k & 31) & 1)) {
        rv[n] = make_uint4(0u, 0u, 0u, 0u);
        rk[n] = make_uint4(~0u, ~0u, ~0u, ~0u);
      }
      const int col = e * 2, pn = col / RB, at = panel_place<RB>(k, col - pn * RB) + pn * S::PANEL;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint8_t* dst = (h ? kd : vd) + at;
        const uint4 r = h ? rk[n] : rv[n];
        if constexpr (kHalf) {
          *reinterpret_cast<uint4*>(dst) = r;
        } else {
          uint32_t lo[3], hi[3];
          split_pair<false, 3>(__uint_as_float(r.x), __uint_as_float(r.y), lo);
          split_pair<false, 3>(__uint_as_float(r.z), __uint_as_float(r.w), hi);
#pragma unroll
          for (int q = 0; q < 3; ++q) *reinterpret_cast<uint2*>(dst + q * S::PART) = make_uint2(lo[q], hi[q]);
        }
      }
    };
    // keys of the batch whose values are not finite
    auto mark = [&](int n0) {
#pragma unroll
      for (int n = 0; n < BATCH; ++n) {
        const uint32_t* x = reinterpret_cast<const uint32_t*>(&rv[n]);
        bool odd = false;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          odd |= kHalf ? (x[q] & 0x7C00u) == 0x7C00u || (x[q] & 0x7C000000u) == 0x7C000000u
                       : (x[q] & 0x7F800000u) == 0x7F800000u;
        if (odd) {
          const int k = ((n0 + n) * 128 + lt) / PER;
          atomicOr(&odd_keys[k >> 5], 1u << (k & 31));
        }
      }
      load_warps_agree(true);
    };
    // FP32 units all go this way: a batch's registers are loaded again, with the
    // batch behind it (the next unit's, over the ends of pieces), as they are stored.
    Walk<S::ROWS, KEYS> ahead(a);
    ahead.p = w.p;
    ahead.end = w.end;
    int au = w.p.u0, an = 0;
    auto ahead_next = [&]() {
      if ((an += BATCH) < NL) return;
      an = 0;
      if (++au < ahead.p.u1) return;
      ahead.next();
      au = ahead.p.u0;
    };
    if (!kHalf && ahead.more()) {
      pages(ahead.p, au, an);
#pragma unroll
      for (int n = 0; n < BATCH; ++n) fetch(ahead.p, au, an, n);
      ahead_next();
      if (ahead.more()) pages(ahead.p, au, an);
    }
    for (; ok && w.more(); w.next()) {
      if (!a.prefix) row = a.b.table + w.p.s * a.b.table_stride;
      const int all_see = w.seen(w.p.j * S::ROWS / a.b.rep);  // keys that the block's first row sees
      for (int u = w.p.u0; ok && u < w.p.u1; ++u, ++i) {
        const int st = i % STG, k0 = u * KEYS;
        const uint32_t par = ((i / STG) & 1) ^ 1;
        uint8_t* kd = smem + (size_t)st * 2 * S::HALF;
        uint8_t* vd = kd + S::HALF;
        // a unit that every row sees whole, of good pages?
        const bool whole = k0 + KEYS <= all_see;
        bool plain = kHalf && whole;
        if (kHalf) {
          bool good = true;
          for (int k = lane << a.b.shift; k < KEYS; k += 32 << a.b.shift)
            if (k0 + k < w.p.keys) good &= (unsigned)__ldg(row + ((k0 + k) >> a.b.shift)) < (unsigned)a.b.n_pages;
          plain = __all_sync(0xffffffffu, good) && plain;
        }
        ok = load_warps_agree(wait(k_empty + st, par) && wait(v_empty + st, par));
        if (!ok) break;
        if (plain) {
          if (lane == 0 && lw > 0) {
            mbar_arrive(k_full + st);
            mbar_arrive(v_full + st);
          }
          if (lw == 0) {
            const int rows = min(KEYS, 1 << a.b.shift), boxes = KEYS / rows;
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
              uint64_t* bar = h ? v_full + st : k_full + st;
              if (lane == 0) mbar_expect_tx(bar, S::PART);
              __syncwarp();
              for (int x = lane; x < boxes * S::PANELS; x += 32) {
                const int bx = x / S::PANELS, pn = x - bx * S::PANELS, key = k0 + bx * rows;
                const int id = __ldg(row + (key >> a.b.shift)), slot = key & slot_mask;
                const uint32_t dst = smem_u32(h ? vd : kd) + pn * S::PANEL + bx * rows * RB;
                asm volatile(
                    "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
                    "%5, %6}], [%7];" ::"r"(dst),
                    "l"(h ? &maps.v : &maps.k), "r"(0), "r"(pn), "r"(a.swap ? slot : w.p.kv),
                    "r"(a.swap ? w.p.kv : slot), "r"(id), "r"(smem_u32(bar))
                    : "memory");
              }
            }
          }
          continue;
        }
        // through registers
        if (!whole) {
          if (lt < 4) odd_keys[lt] = 0u;
          load_warps_agree(true);
        }
#pragma unroll 1
        for (int n0 = 0; n0 < NL; n0 += BATCH) {
          if (kHalf) {
            pages(w.p, u, n0);
#pragma unroll
            for (int n = 0; n < BATCH; ++n) fetch(w.p, u, n0, n);
          }
          if (!whole) mark(n0);
#pragma unroll
          for (int n = 0; n < BATCH; ++n) {
            store(kd, vd, whole, n0, n);
            if (!kHalf && ahead.more()) fetch(ahead.p, au, an, n);
          }
          if (!kHalf && ahead.more()) {
            ahead_next();
            if (ahead.more()) pages(ahead.p, au, an);
          }
        }
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(k_full + st);
          mbar_arrive(v_full + st);
        }
      }
    }
    loaded = i;
  } else if (warp >= S::SOFT + 4) {
    // ---- MMAs
    set_registers<S::REGS, S::MMA_REGS>();
    if (warp == S::SOFT + 4) {
      // The whole warp walks and waits, one elected lane issues: inside its branch
      // the MMA's operands stay in uniform registers (issued by a lone lane of a
      // diverged warp, every MMA took 100 cycles whatever its size).
      constexpr uint32_t kFmt = kHalf ? 0u : 1u;
      const uint32_t idesc_s = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(KEYS >> 3) << 17) | (8u << 24);
      const uint32_t idesc_o = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
      const uint32_t base = smem_u32(smem);
      // products (A part, B part), small ones first
      constexpr int NPROD = kHalf ? 2 : 6;
      using Desc = TileDesc<RB>;
      int i = 0, sn = 0;                 // units; S buffers written
      uint32_t qn[2] = {0, 0}, pn[2] = {0, 0}, dn[2] = {0, 0};  // waits done on q_full, p_full, pv_done
      bool ok = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, wait(bar, parity)); };
      auto qk = [&](int t, int buf, int st) {
        const uint32_t d = tile_col(t) + S::QC + (BUFS == 2 ? buf * S::SC : 0) + S::S0;
        const uint32_t lo = Desc::lo(base + st * 2 * S::HALF), q = tile_col(t);
        unrolled<NPROD * (HD / 16)>([&](auto ic) {
          constexpr int x = ic.value / (HD / 16), k = ic.value % (HD / 16);
          constexpr int panel = k * 32 / RB, at = k * 32 - panel * RB;
          mma_ts<S::pa(x) * (HD / 2) + 8 * k, (S::pb(x) * S::PART + panel * S::PANEL + at) / 16, Desc::hi>(d, q, lo, idesc_s,
                                                                                                  (x | k) != 0);
        });
      };
      auto pv = [&](int t, int buf, int st, bool add) {
        const uint32_t o = tile_col(t) + S::QC + BUFS * S::SC;
        const uint32_t p = tile_col(t) + S::QC + (BUFS == 2 ? buf * S::SC : 0);
        const uint32_t lo = Desc::lo(base + st * 2 * S::HALF + S::HALF, S::PANELS > 1 ? S::PANEL : 0);
        unrolled<NPROD * (KEYS / 16)>([&](auto ic) {
          constexpr int x = ic.value / (KEYS / 16), k = ic.value % (KEYS / 16);
          // P: chunks of 32 keys, the parts of a chunk side by side (16 columns each)
          mma_ts<(k >> 1) * 16 * QP + S::pa(x) * 16 + (k & 1) * 8, (S::pb(x) * S::PART + k * 16 * RB) / 16, Desc::hi>(
              o, p, lo, idesc_o, add || (x | k) != 0);
        });
      };
      for (; ok && w.more(); w.next()) {
        const int nt = TILES == 2 && w.rows() > 128 ? 2 : 1;
        for (int t = 0; ok && t < nt; ++t) ok = wait_all(q_full + t, qn[t]++ & 1);
        ok = ok && wait_all(k_full + i % STG, (i / STG) & 1);
        if (!ok) break;
        tc::tc_fence_after();
        // (every earlier PV has been waited for by the softmax, which then gave the new Q)
        if (elect_one()) {
          for (int t = 0; t < nt; ++t) {
            qk(t, sn & 1, i % STG);
            tc::umma_commit(s_full + (TILES == 2 ? t : sn & 1));
          }
          tc::umma_commit(k_empty + i % STG);
        }
        __syncwarp();
        for (int u = w.p.u0; ok && u < w.p.u1; ++u, ++i) {
          const int st = i % STG, nst = (i + 1) % STG;
          const bool add = (u - w.p.u0) % S::kFlush != 0, last = u + 1 == w.p.u1;
          if (TILES == 1) {
            // the next unit's S goes to the other buffer, whose P the last PV has read
            if (!last) {
              ok = wait_all(k_full + nst, ((i + 1) / STG) & 1);
              if (ok && u > w.p.u0) ok = wait_all(pv_done, dn[0]++ & 1);
              if (!ok) break;
              tc::tc_fence_after();
              if (elect_one()) {
                qk(0, (sn + 1) & 1, nst);
                tc::umma_commit(s_full + ((sn + 1) & 1));
                tc::umma_commit(k_empty + nst);
              }
              __syncwarp();
            }
            ok = wait_all(v_full + st, (i / STG) & 1) && wait_all(p_full + (sn & 1), pn[sn & 1]++ & 1);
            if (!ok) break;
            tc::tc_fence_after();
            if (elect_one()) {
              pv(0, sn & 1, st, add);
              tc::umma_commit(pv_done);
              tc::umma_commit(v_empty + st);
            }
            __syncwarp();
            ++sn;
          } else {
            ok = wait_all(v_full + st, (i / STG) & 1);
            if (ok && !last) ok = wait_all(k_full + nst, ((i + 1) / STG) & 1);
            for (int t = 0; ok && t < nt; ++t) {
              ok = wait_all(p_full + t, pn[t]++ & 1);
              if (!ok) break;
              tc::tc_fence_after();
              if (elect_one()) {
                pv(t, 0, st, add);
                tc::umma_commit(pv_done + t);
                if (t + 1 == nt) tc::umma_commit(v_empty + st);
              }
              __syncwarp();
              if (!last) {  // S overlays the P that this PV reads
                ok = wait_all(pv_done + t, dn[t]++ & 1);
                if (!ok) break;
                tc::tc_fence_after();
                if (elect_one()) {
                  qk(t, 0, nst);
                  tc::umma_commit(s_full + t);
                  if (t + 1 == nt) tc::umma_commit(k_empty + nst);
                }
                __syncwarp();
              }
            }
          }
        }
        // the PVs that this warp has not waited for are the softmax's to wait for
        if (TILES == 1)
          dn[0] += w.p.u1 - w.p.u0 > 1 ? 2 : 1;
        else
          for (int t = 0; t < nt; ++t) ++dn[t];
      }
      if (elect_one()) tc::umma_commit(&drain);
      __syncwarp();
      if (!mbar_wait(&drain, 0)) flag(a.b.status, kErrTimeout);
    }
  } else {
    // ---- softmax: one row a thread
    set_registers<S::REGS, S::SOFT_REGS>();
    constexpr int HALVES = S::HALVES;
    const int t = TILES == 2 ? warp >> 2 : 0, hf = HALVES == 2 ? warp >> 2 : 0, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t qcol = tile_col(t) + lanes, scol = qcol + S::QC, ocol = scol + BUFS * S::SC + hf * (HD / HALVES);
    // Moving the reference waits for the last PV and rewrites O: 2 x 2048 tokens behind up
    // to 6144, some heads sharp, take 870 us with 14, 836 with 12 (825 with 4, where a weight 2^-14 of the largest
    // keeps 15 bits).
    using Wt = Weights<kHalf, 12>;
    constexpr float kFirst = Wt::kFirst, kLimit = Wt::kLimit;
    constexpr int NCH = KEYS / 32 / HALVES;    // 32-key chunks of a unit that this thread takes
    constexpr int MYD = HD / HALVES;           // dims of O that this thread takes
    const int ch0 = hf * NCH;
    constexpr int DW = MYD < 32 ? 16 : 32;     // dims of O read at a time
    // With two threads a row, a warp and its partner (the same rows' other half)
    // pass the same barriers: both see the same verdict and stop together.
    auto agree = [&](bool mine) -> bool {
      mine = __all_sync(0xffffffffu, mine);
      if constexpr (HALVES == 2) {
        uint32_t v;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.aligned.pred q, %2, 64, p;\n\t"
            "selp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(v)
            : "r"((uint32_t)mine), "r"(2 + (warp & 3))
            : "memory");
        return v != 0;
      }
      return mine;
    };
    uint32_t sn = 0, s_seen[2] = {0, 0}, done = 0;
    // (false: a wait ran out.  Later ones return at once, and the rows of this and all
    // later pieces become NaN.)
    bool ok = true;
    for (; w.more(); w.next()) {
      if (TILES == 2 && t == 1 && w.rows() <= 128) continue;
      const int ri = w.p.j * S::ROWS + t * 128 + r;  // row of the (sequence, kv head)
      const bool in = t * 128 + r < w.rows();
      const int tok = ri / a.b.rep, h = w.p.kv * a.b.rep + (ri - tok * a.b.rep);
      const int64_t token = w.p.tok0 + tok;
      const int vis = in ? w.seen(tok) : 0;
      float sc = a.scale;
      {
        // Q's parts into tensor memory, two elements a column
        const float* qp = a.q + token * a.ldq + (int64_t)h * HD;
        float scale = 1.f;
        if (kHalf) {
          float mx = 0.f;
          if (in)
            for (int e = 0; e < HD; e += 4) {
              const float4 v = __ldg(reinterpret_cast<const float4*>(qp + e));
              mx = fmaxf(fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y))), fmaxf(fabsf(v.z), fabsf(v.w)));
            }
          float back;
          scale = half_scale(mx, back);
          sc *= back;
        }
#pragma unroll 2
        for (int e0 = hf * MYD; e0 < (hf + 1) * MYD; e0 += 16) {
          uint32_t part[QP][8];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (in) v = __ldg(reinterpret_cast<const float4*>(qp + e0 + e));
            uint32_t x[QP], y[QP];
            split_pair<kHalf, QP>(v.x * scale, v.y * scale, x);
            split_pair<kHalf, QP>(v.z * scale, v.w * scale, y);
#pragma unroll
            for (int q = 0; q < QP; ++q) {
              part[q][e / 2] = x[q];
              part[q][e / 2 + 1] = y[q];
            }
          }
#pragma unroll
          for (int q = 0; q < QP; ++q)
            asm volatile(
                "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(qcol + q * (HD / 2) + e0 / 2),
                "r"(part[q][0]), "r"(part[q][1]), "r"(part[q][2]), "r"(part[q][3]), "r"(part[q][4]), "r"(part[q][5]),
                "r"(part[q][6]), "r"(part[q][7])
                : "memory");
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full + t);
      }
      float acc[MYD];
#pragma unroll
      for (int d = 0; d < MYD; ++d) acc[d] = 0.f;
      float ref = kUnseen, l = 0.f;
      for (int u = w.p.u0; u < w.p.u1; ++u) {
        const int buf = TILES == 2 ? t : (int)(sn & 1);
        ok = wait(s_full + buf, s_seen[buf]++ & 1) && ok;
        if (HALVES == 1) {
          ok = agree(ok);
          if (!ok) break;
        }
        tc::tc_fence_after();
        const uint32_t pcol = scol + (BUFS == 2 ? (sn & 1) * S::SC : 0);
        const int left = vis - u * KEYS;  // keys of the unit that the row sees
        const bool masked = !__all_sync(0xffffffffu, left >= KEYS);
        // Scores are read twice; FP32 rows of two threads keep them, as P overlaps the
        // scores of the other half.
        constexpr bool kKeep = HALVES == 2 && !kHalf;
        float keep[kKeep ? NCH : 1][32];
        float mx = -INFINITY;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          float(&v)[32] = keep[kKeep ? ch : 0];
          tmem_load(pcol + S::S0 + 32 * (ch0 + ch), v);
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * (ch0 + ch) + e >= left) v[e] = -INFINITY;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) mx = fmaxf(mx, v[e]);
        }
        if constexpr (HALVES == 2) {
          row_max[hf][sn & 1][r] = mx;
          ok = agree(ok);
          if (!ok) break;
          mx = fmaxf(mx, row_max[hf ^ 1][sn & 1][r]);
        }
        ++sn;
        mx *= sc;
        const int uu = u - w.p.u0;
        const bool flush = uu > 0 && uu % S::kFlush == 0;
        const bool grow = __any_sync(0xffffffffu, mx - ref > kLimit);
        // Every PV is waited for, in order and before the weights that let the next
        // one start are handed over: a parity tells a phase from its neighbours only.
        // Here when O is needed, else behind the arithmetic.
        auto before = [&]() {
          ok = __all_sync(0xffffffffu, wait(pv_done + (TILES == 2 ? t : 0), done++ & 1)) && ok;
          tc::tc_fence_after();
        };
        if (uu > 0 && (flush || grow)) before();
        if (flush) {
#pragma unroll
          for (int d = 0; d < MYD; d += DW) {
            float v[DW];
            tmem_load(ocol + d, v);
#pragma unroll
            for (int e = 0; e < DW; ++e) acc[d + e] += v[e];
          }
        }
        if (grow) {
          const float m = fmaxf(mx - kFirst, ref), f = ex2(ref - m);
          ref = m;
          l *= f;
          if (uu > 0 && !flush) {
#pragma unroll
            for (int d = 0; d < MYD; d += 16) {
              float v[16];
              uint32_t x[16];
              tmem_load(ocol + d, v);
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(v[e] * f);
              tc::tmem_st16(ocol + d, x);
            }
          }
#pragma unroll
          for (int d = 0; d < MYD; ++d) acc[d] *= f;
        }
        float l2 = 0.f;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          float(&v)[32] = keep[kKeep ? ch : 0];
          if (!kKeep) tmem_load(pcol + S::S0 + 32 * (ch0 + ch), v);
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = ex2(fmaf(v[e], sc, -ref));
          if (masked) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * (ch0 + ch) + e >= left) v[e] = 0.f;
          }
          uint32_t part[QP][16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            uint32_t x[QP];
            l += v[2 * e];
            l2 += v[2 * e + 1];
            split_pair<kHalf, QP>(v[2 * e], v[2 * e + 1], x);
#pragma unroll
            for (int q = 0; q < QP; ++q) part[q][e] = x[q];
          }
#pragma unroll
          for (int q = 0; q < QP; ++q) tc::tmem_st16(pcol + (ch0 + ch) * 16 * QP + q * 16, part[q]);
        }
        l += l2;
        if (uu > 0 && !(flush || grow)) before();
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + buf);
      }
      if (ok) ok = wait(pv_done + (TILES == 2 ? t : 0), done++ & 1);
      if constexpr (HALVES == 2) row_sum[hf][r] = l;
      ok = agree(ok);
      if constexpr (HALVES == 2) l += row_sum[hf ^ 1][r];
      if (!ok) {
        l = NAN;
      } else {
        tc::tc_fence_after();
#pragma unroll
        for (int d = 0; d < MYD; d += 16) {
          float v[16];
          tmem_load(ocol + d, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[d + e] += v[e];
        }
        tc::tc_fence_before();
      }
      if (ok && l != l) odd[warp] = 1;
      if (in) {
        const bool begin = w.p.u0 == 0, whole = begin && w.p.u1 == w.p.units;
        const float m = ref == kUnseen ? -INFINITY : ref;
        float* ml;
        float* dst = place(w, t * 128 + r, token * a.H + h, ml);
        const float inv = ml ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int d = 0; d < MYD; d += 4)
          *reinterpret_cast<float4*>(dst + hf * MYD + d) =
              make_float4(acc[d] * inv, acc[d + 1] * inv, acc[d + 2] * inv, acc[d + 3] * inv);
        if (ml && hf == 0) {
          ml[0] = m;
          ml[1] = l;
        }
        if (!a.prefix && r == 0 && t == 0 && hf == 0 && begin && !whole) {
          const int64_t lastu = w.p.x - w.p.u0 + w.p.units - 1;
          a.desc[c * 2] = make_int4(w.p.tok0, w.p.kv, w.p.j, (int)(owner_of(lastu, units, workers) - c) + 1);
          a.desc[c * 2 + 1] = make_int4(w.rows(), 0, 0, 0);
        }
      }
    }
    // ---- rows whose sum of weights is not a number, anew (a warp its own, all dims)
    ok = agree(ok);
    __syncwarp();
    if (ok && hf == 0 && odd[warp]) {
      Walk<S::ROWS, KEYS> v(a);
      v.begin(muldiv(c, units, workers), muldiv(c + 1, units, workers));
      for (; v.more(); v.next()) {
        const int n = v.rows() - t * 128;
        float* ml;
        for (int i = 0; i < 32; ++i) {
          const int row = (warp & 3) * 32 + i, ri = v.p.j * S::ROWS + t * 128 + row;
          if (row >= n) break;
          const int tok = ri / a.b.rep, h = v.p.kv * a.b.rep + (ri - tok * a.b.rep);
          float* dst = place(v, t * 128 + row, (int64_t)(v.p.tok0 + tok) * a.H + h, ml);
          const float was = ml ? ml[1] : dst[0];
          if (was == was) continue;
          float m, l, o[4];
          plain_row<KT>(a.b, a.prefix ? a.b.table : a.b.table + v.p.s * a.b.table_stride,
                        a.q + (v.p.tok0 + tok) * a.ldq + (int64_t)h * HD, HD, v.p.kv, v.p.u0 * KEYS,
                        min(v.p.u1 * KEYS, v.seen(tok)), a.scale, m, l, o);
          const float inv = ml ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (lane + 32 * e < HD) dst[lane + 32 * e] = o[e] * inv;
          if (ml && lane == 0) {
            ml[0] = m;
            ml[1] = l;
          }
        }
      }
    }
  }
  __syncthreads();
  if (kHalf && warp == S::SOFT && stop) {
    // copies that are still on their way land before the CTA ends (or one more wait runs out)
    uint64_t left = a.wait_cycles;
    for (int st = 0; st < STG && st < loaded; ++st) {
      const uint32_t par = ((loaded - 1 - st) / STG) & 1;
      if (!mbar_wait_for(k_full + st, par, left)) left = 0;
      if (!mbar_wait_for(v_full + st, par, left)) left = 0;
    }
  }
  if (warp == S::SOFT + 4) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Sum of `pieces` partial states of a row and, with `own`, the state that its
// place in `out` holds; by one warp: groups of HD / 4 lanes take every
// 32 / (HD / 4)-th piece, four dims a lane.  at(k): the row's index in part.
template <int HD, typename At>
__device__ __forceinline__ void join_row(const TcArgs& a, int64_t row, int pieces, bool own, const At& at, int lane) {
  constexpr int W = HD / 4, G = 32 / W;
  const int x = lane % W, g = lane / W;
  const float m0 = own ? a.state[row * 2] : -INFINITY;
  float M = m0;
  for (int k = lane; k < pieces; k += 32) M = fmaxf(M, a.part_ml[at(k) * 2]);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float ref = ref_of(M);
  float l = 0.f;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float m, float li, const float* o) {
    const float w = ex2(m - ref);
    const float4 v = *reinterpret_cast<const float4*>(o + 4 * x);
    l = fmaf(w, li, l);
    s.x = fmaf(w, v.x, s.x);
    s.y = fmaf(w, v.y, s.y);
    s.z = fmaf(w, v.z, s.z);
    s.w = fmaf(w, v.w, s.w);
  };
  if (own && g == 0) add(m0, a.state[row * 2 + 1], a.out + row * HD);
#pragma unroll 4
  for (int k = g; k < pieces; k += G) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at(k) * 2);
    add(ml.x, ml.y, a.part + at(k) * HD);
  }
#pragma unroll
  for (int o = W; o < 32; o <<= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
    s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
    s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
  }
  const bool state = a.state && !own;  // the state itself, to be joined with the prefix's
  const float inv = state ? 1.f : (l == 0.f ? 0.f : 1.f / l);
  if (g == 0) *reinterpret_cast<float4*>(a.out + row * HD + 4 * x) = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
  if (state && lane == 0) *reinterpret_cast<float2*>(a.state + row * 2) = make_float2(M, l);
}

// Joins the pieces of blocks that several CTAs hold: block (c, y) takes 8 rows
// of the item that starts in CTA c, a warp a row.
template <int HD, int ROWS>
__global__ void __launch_bounds__(256) rows_merge_kernel(TcArgs a) {
  const int c = blockIdx.x;
  const int4 d = a.desc[2 * c];
  if (d.w == 0) return;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
  if (r >= a.desc[2 * c + 1].x) return;
  const int ri = d.z * ROWS + r, tok = ri / a.b.rep, h = d.y * a.b.rep + ri - tok * a.b.rep;
  join_row<HD>(a, (int64_t)(d.x + tok) * a.H + h, d.w, false,
               [&](int k) { return (int64_t)((c + k) * 2 + (k == 0 ? 1 : 0)) * ROWS + r; }, threadIdx.x & 31);
}

// Zeros the rows of tokens that no sequence holds.
__global__ void zero_rows_kernel(Batch b, float* out, int row) {
  const int lo = b.n > 0 ? min(max(__ldg(b.starts), 0), b.T) : b.T;
  const int hi = b.n > 0 ? min(max(__ldg(b.starts + b.n), lo), b.T) : b.T;
  const int64_t per = row / 4, total = (int64_t)(lo + b.T - hi) * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t t = i / per, tok = t < lo ? t : hi + (t - lo);
    reinterpret_cast<float4*>(out)[tok * per + (i - t * per)] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// Joins a token's own state (output unnormalised, (m, l) in `state`) with the
// prefix's pieces: one warp a (token, head) row.
template <int HD, int ROWS>
__global__ void __launch_bounds__(256) prefix_join_kernel(TcArgs a, int64_t units, int workers, int per) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.b.T * a.H) return;
  const int tok = (int)(row / a.H), h = (int)(row - (int64_t)tok * a.H), kv = h / a.b.rep;
  if (a.own_rows) {  // ragged: padding rows are not the batch's
    const int lo = a.b.n > 0 ? __ldg(a.own_rows) : 0, hi = a.b.n > 0 ? __ldg(a.own_rows + a.b.n) : 0;
    if (tok < lo || tok >= hi) return;
  }
  const int ri = tok * a.b.rep + h - kv * a.b.rep, j = ri / ROWS;
  const int64_t item = (int64_t)kv * (a.items / a.b.kv_heads) + j;
  const int64_t c0 = owner_of(item * per, units, workers);
  const int pieces = (int)(owner_of(item * per + per - 1, units, workers) - c0) + 1;
  join_row<HD>(a, row, pieces, true, [&](int k) { return ((int64_t)k * a.items + item) * ROWS + (ri - j * ROWS); }, lane);
}

// ---- host ---------------------------------------------------------------------------

template <int HD, typename KT>
struct TcLaunch {
  using S = TcShape<HD, KT>;

  static int32_t rows(TcArgs a, cudaStream_t st) {
    auto kern = rows_kernel<HD, KT>;
    static std::mutex mu;
    static bool granted[64] = {false};  // per device
    int dev = 0;
    Q6W_CUDA_TRY(cudaGetDevice(&dev));
    {
      std::lock_guard<std::mutex> lock(mu);
      if (!granted[dev & 63]) {
        // the register split needs all that it divides (build.py checks it too)
        cudaFuncAttributes attr;
        Q6W_CUDA_TRY(cudaFuncGetAttributes(&attr, kern));
        if (attr.numRegs != S::REGS)
          return fail(Q6W_ERR_CUDA, "rows_kernel was built for %d registers a thread, not %d", attr.numRegs, S::REGS);
        Q6W_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
        granted[dev & 63] = true;
      }
    }
    TcMaps maps;
    memset(&maps, 0, sizeof(maps));
    if (S::kHalf) {
      const int box = std::min(S::KEYS, 1 << a.b.shift);
      bool swap = false;
      int32_t rc = pool_map(a.b, a.b.k, HD, 2, 1, box, 1, &maps.k, &swap);
      if (!rc) rc = pool_map(a.b, a.b.v, HD, 2, 1, box, 1, &maps.v, &swap);
      if (rc) return rc;
      a.swap = swap;
    }
    kern<<<sm_count(), S::THREADS, S::SMEM, st>>>(a, maps);
    Q6W_LAUNCH_CHECK("rows_kernel");
    return Q6W_OK;
  }

  static int32_t own(TcArgs a, cudaStream_t st) {
    a.prefix = 0;
    line_kernel<S::ROWS, S::KEYS><<<1, 1024, 0, st>>>(a, a.line);
    Q6W_LAUNCH_CHECK("line_kernel");
    int32_t rc = rows(a, st);
    if (rc) return rc;
    rows_merge_kernel<HD, S::ROWS><<<dim3(sm_count(), S::ROWS / 8), 256, 0, st>>>(a);
    Q6W_LAUNCH_CHECK("rows_merge_kernel");
    return Q6W_OK;
  }

  static int per(const TcArgs& a) { return std::max(1, (a.prefix_len + S::KEYS - 1) / S::KEYS); }
  static int64_t items(const Batch& b) { return (int64_t)b.kv_heads * (((int64_t)b.T * b.rep + S::ROWS - 1) / S::ROWS); }
  // pieces of an item at most: CTAs that its units can reach
  static int64_t pieces(const Batch& b, int prefix_len) {
    const int64_t p = std::max(1, (prefix_len + S::KEYS - 1) / S::KEYS), units = items(b) * p;
    const int64_t g = std::min<int64_t>(sm_count(), units);
    return std::min<int64_t>(p, (p * g + units - 1) / units + 1);
  }
  static int32_t prefix(TcArgs a, cudaStream_t st) {
    a.prefix = 1;
    a.items = (int)items(a.b);
    return rows(a, st);
  }
  static int32_t join(TcArgs a, cudaStream_t st) {
    a.items = (int)items(a.b);
    const int64_t units = (int64_t)a.items * per(a);
    const int64_t total = (int64_t)a.b.T * a.H;
    prefix_join_kernel<HD, S::ROWS><<<(unsigned)((total + 7) / 8), 256, 0, st>>>(
        a, units, (int)std::min<int64_t>(sm_count(), units), per(a));
    Q6W_LAUNCH_CHECK("prefix_join_kernel");
    return Q6W_OK;
  }
  static size_t own_rows() { return (size_t)sm_count() * 2 * S::ROWS; }
  static size_t prefix_rows(const Batch& b, int prefix_len) { return (size_t)(pieces(b, prefix_len) * items(b)) * S::ROWS; }
};

#define Q6W_TC_DISPATCH(hd, half, call)                                             \
  switch (hd) {                                                                     \
    case 16: return half ? TcLaunch<16, __half>::call : TcLaunch<16, float>::call;  \
    case 32: return half ? TcLaunch<32, __half>::call : TcLaunch<32, float>::call;  \
    case 64: return half ? TcLaunch<64, __half>::call : TcLaunch<64, float>::call;  \
    default: return half ? TcLaunch<128, __half>::call : TcLaunch<128, float>::call; \
  }

int32_t rows_own(const TcArgs& a, int hd, bool half, cudaStream_t st) { Q6W_TC_DISPATCH(hd, half, own(a, st)) }
int32_t rows_prefix(const TcArgs& a, int hd, bool half, cudaStream_t st) { Q6W_TC_DISPATCH(hd, half, prefix(a, st)) }
int32_t rows_join(const TcArgs& a, int hd, bool half, cudaStream_t st) { Q6W_TC_DISPATCH(hd, half, join(a, st)) }
size_t rows_own_rows(int hd, bool half) { Q6W_TC_DISPATCH(hd, half, own_rows()) }
size_t rows_prefix_rows(const Batch& b, int prefix_len, int hd, bool half) {
  Q6W_TC_DISPATCH(hd, half, prefix_rows(b, prefix_len))
}

int32_t zero_padding_rows(const Batch& b, float* out, int row, cudaStream_t st) {
  const int64_t vecs = (int64_t)b.T * row / 4;
  zero_rows_kernel<<<(unsigned)std::min<int64_t>((vecs + 255) / 256, (int64_t)sm_count() * 4), 256, 0, st>>>(b, out, row);
  Q6W_LAUNCH_CHECK("zero_rows_kernel");
  return Q6W_OK;
}

}  // namespace paged
}  // namespace q6w

// Serving from a paged KV cache: append with rotation, causal attention over
// pages, and attention of a batch behind a shared prefix.
#include <math.h>

#include <atomic>

#include "paged.cuh"

namespace q6w {
namespace paged {

// ---- append ------------------------------------------------------------------
//
// One pass: (a, b) -> (a cos - b sin, a sin + b cos) on pairs (2j, 2j+1) of
// every query and key head at the token's position, the value rows copied.
// Bound by memory: per token 4 (2 H + 2 KV) head_dim bytes of activations and
// the page rows.  64 chunks of 1-511 tokens with 48 heads of 128, FP16 pages: 737 MB in
// 127-134 us, 5.5-5.8 TB/s; 2048 prompts of the tiny model (16 heads of 16): 552 MB
// in 113-116 us, 4.8-4.9 TB/s, the chain search -> length -> page behind it (ranges: ten
// calls in a graph, a call among others).  `tpt` threads take one token (a whole warp
// at least, so that the search for the token's sequence is a warp's), eight
// consecutive elements a thread and step: two 16-byte loads, one or two 16-byte stores.

constexpr int kGroup = 4;  // tokens of a thread, narrow tokens

struct AppendArgs {
  Batch b;
  const float* q;
  const float* k;
  const float* v;
  int64_t ldq, ldk, ldv;
  const float* cs;
  const float* sn;
  float* out;
  int32_t hd, H, rope_len, first, zero, tpt_shift;
};

__device__ __forceinline__ void store8(void* pool, int64_t off, int half, const float (&x)[8]) {
  if (half) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(static_cast<__half*>(pool) + off) = *reinterpret_cast<const uint4*>(h);
  } else {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(pool) + off);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// A token's place: its sequence's index of it, position, page slot.
struct Place {
  int at;         // index among the sequence's own tokens; out of range: nothing is written
  int64_t pos;    // position of the rotation
  int64_t slot;   // element offset of the slot, -1: a bad page id
  bool in;
};

// Sequence s holds tokens [t0, t1); moves on to the one that holds t.
__device__ __forceinline__ void follow(const Batch& b, int t, int& s, int& t0, int& t1) {
  while (s < b.n && t >= t1) {
    if (++s < b.n) seq_tokens(b, s, t0, t1);
  }
}

__device__ __forceinline__ Place place_of(const AppendArgs& a, int t, int s, int t0, int t1) {
  const Batch& b = a.b;
  Place p;
  p.at = s >= 0 && s < b.n && t >= t0 && t < t1 ? seq_length(b, s) - (t1 - t) : -1;
  p.pos = (int64_t)a.first + p.at;
  p.in = p.at >= 0 && p.at < b.max_len && p.pos < a.rope_len;
  p.slot = -1;
  if (p.in) {
    const int page = __ldg(b.table + s * b.table_stride + (p.at >> b.shift));
    if ((unsigned)page < (unsigned)b.n_pages)
      p.slot = page * b.page_stride + (int64_t)(p.at & ((1 << b.shift) - 1)) * b.slot_stride;
  }
  if (p.at >= 0 && p.slot < 0) flag(b.status, kErrInput);
  return p;
}

struct Unit {
  float x[8];
};

__device__ __forceinline__ Unit load_unit(const AppendArgs& a, int t, int i, int nq, int nk) {
  const float* src = i < nq        ? a.q + t * a.ldq + 8 * i
                     : i < nq + nk ? a.k + t * a.ldk + 8 * (i - nq)
                                   : a.v + t * a.ldv + 8 * (i - nq - nk);
  const float4 lo = __ldcs(reinterpret_cast<const float4*>(src));
  const float4 hi = __ldcs(reinterpret_cast<const float4*>(src) + 1);
  return {{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}};
}

// Rotates (queries, keys) and stores unit i of token t.
template <bool HALF>
__device__ __forceinline__ void finish_unit(const AppendArgs& a, int t, int i, int nq, int nk, const Place& p, Unit& v) {
  const int units = a.hd >> 3;
  const int j = i < nq ? i : (i < nq + nk ? i - nq : i - nq - nk);
  const int u = j & (units - 1);
  float(&x)[8] = v.x;
  if (!p.in) {
    if (i >= nq || !a.zero) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
  } else if (i < nq + nk) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(a.cs + p.pos * (a.hd >> 1) + 4 * u));
    const float4 d = __ldg(reinterpret_cast<const float4*>(a.sn + p.pos * (a.hd >> 1) + 4 * u));
    const float cc[4] = {c.x, c.y, c.z, c.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x0 = x[2 * e], x1 = x[2 * e + 1];
      x[2 * e] = __fsub_rn(__fmul_rn(x0, cc[e]), __fmul_rn(x1, dd[e]));
      x[2 * e + 1] = __fadd_rn(__fmul_rn(x0, dd[e]), __fmul_rn(x1, cc[e]));
    }
  }
  if (i < nq)
    store8(a.out, ((int64_t)t * a.H) * a.hd + 8 * j, 0, x);
  else if (p.slot >= 0)
    store8(i < nq + nk ? a.b.k : a.b.v, p.slot + (int64_t)(j / units) * a.b.head_stride + 8 * u, HALF, x);
}

// GROUP tokens a thread: where one step of tpt threads covers a token, several
// (their loads go first, in flight together, and one search serves them); wide
// tokens one, its units one ahead.
template <bool HALF, int GROUP>
__global__ void __launch_bounds__(256, 4) append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int tpt = 1 << a.tpt_shift, me = threadIdx.x & (tpt - 1);
  const int t = (blockIdx.x * (256 >> a.tpt_shift) + (threadIdx.x >> a.tpt_shift)) * GROUP;
  if (t < a.b.T) {  // warp-uniform: tpt >= 32
    const int units = a.hd >> 3;  // eight-element units of a head
    const int nq = a.H * units, nk = a.b.kv_heads * units, all = nq + 2 * nk;
    Unit x[GROUP];
#pragma unroll
    for (int g = 0; g < GROUP; ++g)
      if (me < all && t + g < a.b.T) x[g] = load_unit(a, t + g, me, nq, nk);
    int s = token_seq(a.b, t, lane), t0 = 0, t1 = 0;
    if (s >= 0 && s < a.b.n) seq_tokens(a.b, s, t0, t1);
    if (GROUP > 1) {
#pragma unroll
      for (int g = 0; g < GROUP; ++g) {
        if (t + g >= a.b.T) break;
        if (g > 0) follow(a.b, t + g, s, t0, t1);
        const Place p = place_of(a, t + g, s, t0, t1);
        if (me < all) finish_unit<HALF>(a, t + g, me, nq, nk, p, x[g]);
      }
    } else {
      const Place p = place_of(a, t, s, t0, t1);
      for (int i = me; i < all;) {
        Unit v = x[0];
        const int cur = i;
        i += tpt;
        if (i < all) x[0] = load_unit(a, t, i, nq, nk);
        finish_unit<HALF>(a, t, cur, nq, nk, p, v);
      }
    }
  }
  if (a.b.starts && a.b.status)
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.b.n; i += (int64_t)gridDim.x * 256)
      check_tokens(a.b, (int)i);
}

// ---- host ------------------------------------------------------------------------

static int32_t check_batch(const char* who, const q6w_paged_batch* p, int32_t n_tokens, Batch* b) {
  if (!p) return fail(Q6W_ERR_ARG, "%s: null batch", who);
  if (p->kv_dtype != Q6W_KV_F32 && p->kv_dtype != Q6W_KV_F16) return fail(Q6W_ERR_ARG, "%s: unknown kv_dtype", who);
  const int hd = p->head_dim;
  if (hd != 16 && hd != 32 && hd != 64 && hd != 128)
    return fail(Q6W_ERR_ARG, "%s: head_dim %d unsupported (16, 32, 64 or 128)", who, hd);
  if (p->page_size < 1 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return fail(Q6W_ERR_ARG, "%s: page_size %d is not a power of two up to 1024", who, p->page_size);
  if (p->kv_heads < 1 || p->kv_heads > 1024 || p->n_pages < 0 || p->n_seqs < 0 || p->max_pages < 0 || n_tokens < 0)
    return fail(Q6W_ERR_ARG, "%s: bad shape", who);
  if ((int64_t)p->max_pages * p->page_size > (1 << 30))
    return fail(Q6W_ERR_ARG, "%s: a sequence of up to %lld tokens is too long", who,
                (long long)p->max_pages * p->page_size);
  if (n_tokens > (1 << 24) || p->n_seqs > (1 << 24)) return fail(Q6W_ERR_ARG, "%s: more than 2^24 tokens", who);
  if (!p->query_starts && n_tokens != p->n_seqs)
    return fail(Q6W_ERR_ARG, "%s: %d tokens for %d sequences need query_starts", who, n_tokens, p->n_seqs);
  const int64_t unit = p->kv_dtype == Q6W_KV_F16 ? 8 : 4;  // elements of 16 bytes
  if (p->page_stride % unit || p->slot_stride % unit || p->head_stride % unit || p->page_stride < 0 ||
      p->slot_stride < 0 || p->head_stride < 0)
    return fail(Q6W_ERR_ALIGN, "%s: page, slot and head strides must be multiples of 16 bytes", who);
  // offsets inside a page are 32-bit in the kernels
  const int64_t span = (p->page_size - 1) * p->slot_stride + (p->kv_heads - 1) * p->head_stride + hd;
  if (p->slot_stride > (1 << 28) || p->head_stride > (1 << 28) || span > (1 << 28))
    return fail(Q6W_ERR_ARG, "%s: a page spans more than 2^28 elements", who);
  if (n_tokens > 0 && p->n_seqs > 0) {
    if (!p->k_pages || !p->v_pages || !p->lengths || (p->max_pages > 0 && !p->page_table))
      return fail(Q6W_ERR_ARG, "%s: null pointer", who);
    if (!aligned(p->k_pages, 16) || !aligned(p->v_pages, 16))
      return fail(Q6W_ERR_ALIGN, "%s: pages must be 16-byte aligned", who);
  }
  b->k = p->k_pages;
  b->v = p->v_pages;
  b->page_stride = p->page_stride;
  b->slot_stride = p->slot_stride;
  b->head_stride = p->head_stride;
  b->table = p->page_table;
  b->table_stride = p->table_stride;
  b->lengths = p->lengths;
  b->starts = p->query_starts;
  b->status = p->status;
  b->n = p->n_seqs;
  b->T = n_tokens;
  b->n_pages = p->n_pages;
  b->shift = __builtin_ctz((unsigned)p->page_size);
  b->max_len = p->max_pages * p->page_size;
  b->kv_heads = p->kv_heads;
  b->rep = 1;
  return Q6W_OK;
}

// The batch and what else the attention calls are given beside their tensors.
static int32_t check_attention(const char* who, const q6w_paged_batch* p, int32_t n_tokens, int32_t n_heads,
                               int32_t prefix_length, Batch* b) {
  const int32_t st = check_batch(who, p, n_tokens, b);
  if (st) return st;
  if (n_heads < 1 || n_heads > (1 << 14) || n_heads % p->kv_heads)
    return fail(Q6W_ERR_ARG, "%s: %d query heads are not a multiple of %d kv heads", who, n_heads, p->kv_heads);
  b->rep = n_heads / p->kv_heads;
  if (prefix_length < 0 || prefix_length > (1 << 30)) return fail(Q6W_ERR_ARG, "%s: bad prefix_length", who);
  if (p->page_size * p->head_dim * (p->kv_dtype == Q6W_KV_F16 ? 2 : 4) < 128)
    return fail(Q6W_ERR_ARG, "%s: a kv head's part of a page must be at least 128 bytes", who);
  // row numbers, rounded up to whole tiles, are 32-bit in the kernels
  if ((int64_t)n_tokens * n_heads > INT32_MAX - 512)
    return fail(Q6W_ERR_ARG, "%s: %d tokens of %d heads are more rows than 32 bits count", who, n_tokens, n_heads);
  return Q6W_OK;
}

// The workspace: a call's regions in order, each 256-byte aligned.  Base null: sizes only.
struct Space {
  char* at;
  size_t used = 0;
  explicit Space(void* base) : at(static_cast<char*>(base)) {}
  template <typename T>
  T* take(size_t count) {
    T* p = at ? reinterpret_cast<T*>(at + used) : nullptr;
    used += (count * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

struct Regions {
  char* decode = nullptr;
  float *own = nullptr, *own_ml = nullptr, *prefix = nullptr, *prefix_ml = nullptr, *state = nullptr;
  int4* desc = nullptr;
  int64_t* line = nullptr;
};

static size_t layout(const Batch& b, int hd, int H, bool half, int prefix_length, void* base, Regions* r) {
  Space s(base);
  if (b.starts) {
    const size_t rows = rows_own_rows(hd, half);
    r->own = s.take<float>(rows * hd);
    r->own_ml = s.take<float>(rows * 2);
    r->desc = s.take<int4>((size_t)sm_count() * 2);
    r->line = s.take<int64_t>((size_t)b.n + 1);
  } else {
    r->decode = s.take<char>(decode_workspace(hd));
  }
  if (prefix_length > 0) {
    const size_t rows = rows_prefix_rows(b, prefix_length, hd, half);
    r->prefix = s.take<float>(rows * hd);
    r->prefix_ml = s.take<float>(rows * 2);
    r->state = s.take<float>((size_t)b.T * H * 2);
  }
  return s.used;
}

// Bound of the attention kernels' waits while q6w_selftest_paged_stall is on; 0: off.
static std::atomic<int64_t> g_stall_cycles{0};

static int32_t attention(const char* who, const q6w_paged_batch* p, const int32_t* prefix_pages, int32_t prefix_length,
                         int32_t n_tokens, int32_t n_heads, const float* queries, int64_t query_stride, float* output,
                         int32_t zero_padding, void* workspace, size_t workspace_bytes, q6w_stream_t stream) {
  clear_error();
  Batch b;
  int32_t st = check_attention(who, p, n_tokens, n_heads, prefix_length, &b);
  if (st) return st;
  if (n_tokens == 0) return Q6W_OK;
  if (!queries || !output || (prefix_length > 0 && !prefix_pages)) return fail(Q6W_ERR_ARG, "%s: null pointer", who);
  if (!aligned(queries, 16) || !aligned(output, 16) || query_stride % 4)
    return fail(Q6W_ERR_ALIGN, "%s: queries (and their stride) and output must be 16-byte aligned", who);
  if (query_stride < (int64_t)n_heads * p->head_dim)
    return fail(Q6W_ERR_ARG, "%s: query_stride is shorter than a token's heads", who);
  const int hd = p->head_dim;
  const bool half = p->kv_dtype == Q6W_KV_F16;
  Regions r;
  const size_t need = layout(b, hd, n_heads, half, prefix_length, workspace, &r);
  if (!workspace || workspace_bytes < need)
    return fail(Q6W_ERR_ARG, "%s: the workspace needs %zu bytes", who, need);
  if (!aligned(workspace, 256)) return fail(Q6W_ERR_ALIGN, "%s: the workspace must be 256-byte aligned", who);
  cudaStream_t s = (cudaStream_t)stream;
  const int64_t stall = g_stall_cycles.load(std::memory_order_relaxed);
  const float scale = (float)(1.4426950408889634 / sqrt((double)hd));
  if (b.starts && zero_padding) {
    st = zero_padding_rows(b, output, n_heads * hd, s);
    if (st) return st;
  }
  if (b.n == 0) return Q6W_OK;
  TcArgs t = {};
  t.b = b;
  t.q = queries;
  t.ldq = query_stride;
  t.out = output;
  t.state = r.state;
  t.desc = r.desc;
  t.line = r.line;
  t.H = n_heads;
  t.scale = scale;
  t.prefix_len = prefix_length;
  t.stall = stall != 0;
  t.wait_cycles = stall ? stall : (int64_t)kWaitCycles;
  TcArgs pre = t;
  pre.part = r.prefix;
  pre.part_ml = r.prefix_ml;
  pre.b.table = prefix_pages;
  pre.b.starts = nullptr;
  if (prefix_length > 0) {
    st = rows_prefix(pre, hd, half, s);
    if (st) return st;
  }
  if (b.starts) {
    t.part = r.own;
    t.part_ml = r.own_ml;
    st = rows_own(t, hd, half, s);
  } else {
    DecodeArgs d = {};
    d.b = b;
    d.q = queries;
    d.ldq = query_stride;
    d.out = output;
    d.state = r.state;
    d.H = n_heads;
    d.hd = hd;
    d.scale = scale;
    d.desc = reinterpret_cast<int4*>(r.decode);
    d.stall = t.stall;
    d.wait_cycles = t.wait_cycles;
    st = decode_attention(d, half, s);
  }
  if (st || prefix_length == 0) return st;
  pre.own_rows = b.starts;
  return rows_join(pre, hd, half, s);
}

}  // namespace paged
}  // namespace q6w

using namespace q6w;

extern "C" int32_t q6w_paged_append(const q6w_paged_batch* batch, int32_t n_tokens, int32_t n_heads,
                                    const float* queries, int64_t query_stride, const float* keys,
                                    int64_t key_stride, const float* values, int64_t value_stride,
                                    const float* rope_cos, const float* rope_sin, int32_t rope_len,
                                    int32_t first_position, float* rotated, int32_t zero_padding,
                                    q6w_stream_t stream) {
  const char* who = "q6w_paged_append";
  clear_error();
  paged::AppendArgs a;
  int32_t st = paged::check_batch(who, batch, n_tokens, &a.b);
  if (st) return st;
  if (n_heads < 0 || n_heads > (1 << 14)) return fail(Q6W_ERR_ARG, "%s: bad n_heads", who);
  if (rope_len < 0 || first_position < 0) return fail(Q6W_ERR_ARG, "%s: negative rope_len or first_position", who);
  if (n_tokens == 0) return Q6W_OK;
  if (!keys || !values || !rope_cos || !rope_sin || (n_heads > 0 && (!queries || !rotated)))
    return fail(Q6W_ERR_ARG, "%s: null pointer", who);
  if (!aligned(keys, 16) || !aligned(values, 16) || !aligned(queries, 16) || !aligned(rotated, 16) ||
      !aligned(rope_cos, 16) || !aligned(rope_sin, 16) || query_stride % 4 || key_stride % 4 || value_stride % 4)
    return fail(Q6W_ERR_ALIGN, "%s: tensors and token strides must be 16-byte aligned", who);
  const int64_t kv_row = (int64_t)batch->kv_heads * batch->head_dim;
  if (key_stride < kv_row || value_stride < kv_row || (n_heads > 0 && query_stride < (int64_t)n_heads * batch->head_dim))
    return fail(Q6W_ERR_ARG, "%s: a token stride is shorter than a token's heads", who);
  if (rotated == queries && n_heads > 0 && query_stride != (int64_t)n_heads * batch->head_dim)
    return fail(Q6W_ERR_ARG, "%s: queries rotated in place must be contiguous", who);
  a.q = queries;
  a.k = keys;
  a.v = values;
  a.ldq = query_stride;
  a.ldk = key_stride;
  a.ldv = value_stride;
  a.cs = rope_cos;
  a.sn = rope_sin;
  a.out = rotated;
  a.hd = batch->head_dim;
  a.H = n_heads;
  a.rope_len = rope_len;
  a.first = first_position;
  a.zero = zero_padding;
  const int units = (n_heads + 2 * batch->kv_heads) * (batch->head_dim >> 3);
  a.tpt_shift = 5;
  while (a.tpt_shift < 8 && (1 << a.tpt_shift) < units) ++a.tpt_shift;
  // kGroup tokens a thread where a token is one step of its threads and the GPU
  // stays full; else one.
  const bool many = units <= 256 && (int64_t)n_tokens << a.tpt_shift >= (int64_t)sm_count() * 2048;
  const int per = (256 >> a.tpt_shift) * (many ? paged::kGroup : 1);
  const unsigned grid = (unsigned)((n_tokens + per - 1) / per);
  const bool half = batch->kv_dtype == Q6W_KV_F16;
  auto kern = many ? (half ? paged::append_kernel<true, paged::kGroup> : paged::append_kernel<false, paged::kGroup>)
                   : (half ? paged::append_kernel<true, 1> : paged::append_kernel<false, 1>);
  kern<<<grid, 256, 0, (cudaStream_t)stream>>>(a);
  Q6W_LAUNCH_CHECK("append_kernel");
  return Q6W_OK;
}

extern "C" size_t q6w_paged_workspace_bytes(const q6w_paged_batch* batch, int32_t n_tokens, int32_t n_heads,
                                            int32_t prefix_length) {
  paged::Batch b;
  if (paged::check_attention("q6w_paged_workspace_bytes", batch, n_tokens, n_heads, prefix_length, &b)) return 0;
  paged::Regions r;
  return paged::layout(b, batch->head_dim, n_heads, batch->kv_dtype == Q6W_KV_F16, prefix_length, nullptr, &r);
}

extern "C" int32_t q6w_paged_attention(const q6w_paged_batch* batch, int32_t n_tokens, int32_t n_heads,
                                       const float* queries, int64_t query_stride, float* output, int32_t zero_padding,
                                       void* workspace, size_t workspace_bytes, q6w_stream_t stream) {
  return paged::attention("q6w_paged_attention", batch, nullptr, 0, n_tokens, n_heads, queries, query_stride, output,
                          zero_padding, workspace, workspace_bytes, stream);
}

extern "C" int32_t q6w_shared_prefix_attention(const q6w_paged_batch* batch, const int32_t* prefix_pages,
                                               int32_t prefix_length, int32_t n_tokens, int32_t n_heads,
                                               const float* queries, int64_t query_stride, float* output,
                                               int32_t zero_padding, void* workspace, size_t workspace_bytes,
                                               q6w_stream_t stream) {
  return paged::attention("q6w_shared_prefix_attention", batch, prefix_pages, prefix_length, n_tokens, n_heads, queries,
                          query_stride, output, zero_padding, workspace, workspace_bytes, stream);
}

extern "C" int32_t q6w_selftest_paged_stall(int64_t wait_cycles) {
  clear_error();
  if (wait_cycles < 0 || wait_cycles > (int64_t(1) << 31))
    return fail(Q6W_ERR_ARG, "q6w_selftest_paged_stall: wait_cycles must be in [0, 2^31]");
  paged::g_stall_cycles.store(wait_cycles, std::memory_order_relaxed);
  return Q6W_OK;
}

// Paged KV cache: the batch descriptor, the division of attention work over the CTAs, the write of new tokens into
// pages and the copy of pages.
//
// Token p of sequence b lives in page table[b][p / ps], slot p % ps.  A batch is ragged: the new tokens of sequence
// b are rows q_off[b] .. q_off[b + 1] of a flat token axis, at positions len_b - n_b + i of its len_b cached tokens
// (the new ones included).  Lengths and tables live on the device, so one captured graph serves changing batches.
// Whatever the device reads there is bounded before it is used: offsets to [0, T], lengths to [0, max_pages * ps],
// and a page outside [0, num_pages) is neither read nor written but reported (CEA_DEV_BAD_PAGE).
#pragma once

#include "cea_common.cuh"
#include "kv_cache.cuh"

// First bad page or batch descriptor seen by a paged kernel; unlike g_cea_status it stops no later kernel.
__device__ int g_cea_paged_status;

namespace cea {
namespace paged {

__device__ __forceinline__ void report(int code) { atomicCAS(&g_cea_paged_status, 0, code); }

struct Batch {
  const int32_t* q_off;
  const int32_t* lens;
  const int32_t* table;
  int64_t table_sb;
  int B, T, max_pages, num_pages, ps;
};

struct Seq {
  int row0, n, len;
  int ctx;  // position of row0's token; may be negative: the first tokens then see nothing
};

constexpr int64_t kMaxLen = 0x7fffff00;  // key indices, rounded up to a tile, stay in 32 bits (places on the axis: 64)

__device__ __forceinline__ Seq load_seq(const Batch& bt, int b) {
  Seq s;
  const int64_t cap = min(static_cast<int64_t>(bt.max_pages) * bt.ps, kMaxLen);
  s.row0 = min(max(bt.q_off[b], 0), bt.T);
  s.n = min(max(bt.q_off[b + 1], s.row0), bt.T) - s.row0;
  s.len = static_cast<int>(min(static_cast<int64_t>(max(bt.lens[b], 0)), cap));
  // counted back from the sequence's end, which may lie behind T: the rows that are there keep their positions
  s.ctx = s.n > 0 ? s.len - (bt.q_off[b + 1] - s.row0) : s.len;
  return s;
}

// Two numbers with infinities and NaN replaced by zeros (of either sign).  A number times 0 is 0, an infinity or NaN the
// NaN 0x7fff, so the product's bits are those to clear: one multiply-add and one logic operation.
template <bool kBF16>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t x) {
  uint32_t bad;
  if constexpr (kBF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %2;" : "=r"(bad) : "r"(x), "r"(0u));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %2;" : "=r"(bad) : "r"(x), "r"(0u));
  return x & ~bad;
}

// `sum`, which starts at 0, stays 0 as long as both numbers of every x are finite
template <bool kBF16>
__device__ __forceinline__ void note_other(uint32_t x, uint32_t& sum) {
  if constexpr (kBF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
}

// one 16-bit number
template <bool kBF16>
__device__ __forceinline__ float widen16(uint32_t bits) {
  return kBF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

// ------------------------------------------------------------------ division of the attention work
// A unit of work is one block of `tb` new tokens of one sequence for one KV head (or, in the generic kernel, for a
// group of its query heads), over the keys its last token sees.  The units are laid end to end on one axis, each as
// long as the keys it reads (at least 1) and `cost` more, and CTA c of n takes the tiles that start in its share of
// the axis: every CTA gets the same work whatever the lengths are, with nothing known on the host.  `cost` is what a
// unit takes besides its tiles (loading its queries, filling the pipeline, writing its result), in keys: without it
// the CTAs that got many short units ended last (2048 tokens alone: 83 us, against 58 us with
// it; 192 keys in the decode kernel and 384 in the chunk kernel were the best of 64 to 512).  A unit split
// over CTAs leaves partial results, at most two a CTA (one that began before it, one that goes on behind it), which
// combine_kernel joins; so the workspace depends on the grid alone.  A sequence's units form an arithmetic series
// (block i of a causal chunk reads tb more keys than block i - 1), so its length and the block at a coordinate have
// closed forms and no work list is written or read.
struct Division {
  int B, units_h, tb;   // units_h: units per block of tokens (KV heads x head groups)
  int group;            // query rows per token and unit
  int64_t max_rows, min_rows;  // sequences with n * group outside [min_rows, max_rows] belong to another kernel
  int min_n, max_n;  // what the caller promised of sequences with n > 0
  int causal;
  int cost;             // of a unit besides its keys
  int min_share_log2;   // smallest share of the axis worth a CTA of its own; at least a tile
};

struct SeqUnits {
  int n, len, row0, nb, n0, ctx;
  int64_t S;  // length on the axis of one head's units
};

__device__ __forceinline__ int64_t units_before(const SeqUnits& s, int i, const Division& dv) {
  const int64_t cost = static_cast<int64_t>(i) * dv.cost;
  if (!dv.causal) return static_cast<int64_t>(i) * max(1, s.len) + cost;
  if (i <= s.n0) return i + cost;
  const int64_t m = i - s.n0;
  return s.n0 + m * s.ctx + static_cast<int64_t>(dv.tb) * (m * (2ll * s.n0 + m + 1) / 2) + cost;
}

// A unit's length on the axis.  In 64 bits: the keys alone may fill 31, and a length that came out negative would send
// the walk back without end.
__device__ __forceinline__ int64_t unit_span(int keys, const Division& dv) {
  return static_cast<int64_t>(max(1, keys)) + dv.cost;
}

// keys that block i reads (its last token's view)
__device__ __forceinline__ int unit_keys(const SeqUnits& s, int i, int tb, bool causal) {
  if (!causal) return s.len;
  const int64_t last = min(static_cast<int64_t>(i + 1) * tb, static_cast<int64_t>(s.n));
  return static_cast<int>(min(max(s.ctx + last, int64_t(0)), static_cast<int64_t>(s.len)));
}

// kOne: every sequence served is one block of tokens (tb >= its n), whose last token sees all its keys
template <bool kOne>
__device__ __forceinline__ SeqUnits seq_units(const Division& dv, const Seq& q) {
  SeqUnits s;
  s.n = q.n;
  s.len = q.len;
  s.row0 = q.row0;
  if constexpr (kOne) {
    s.nb = q.n > 0 && q.n <= dv.tb ? 1 : 0;
    s.n0 = 0;
    s.ctx = q.ctx;
    s.S = s.nb * unit_span(q.len, dv);
    return s;
  }
  const int64_t rows = static_cast<int64_t>(q.n) * dv.group;
  s.nb = q.n > 0 && rows >= dv.min_rows && rows <= dv.max_rows ? (q.n + dv.tb - 1) / dv.tb : 0;
  s.ctx = q.ctx;
  s.n0 = s.ctx < 0 ? min(static_cast<int>((-static_cast<int64_t>(s.ctx)) / dv.tb), max(s.nb - 1, 0)) : 0;
  s.S = s.nb == 0 ? 0
                  : units_before(s, s.nb - 1, dv) + unit_span(unit_keys(s, s.nb - 1, dv.tb, dv.causal), dv);
  return s;
}

// 64-bit division costs several hundred cycles, most axes fit 32 bits
__device__ __forceinline__ int64_t div64(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// CTA c's share of an axis of length W: [base c + min(c, rem), base (c + 1) + min(c + 1, rem)), W = base n + rem.
struct Share {
  int64_t base;
  int n, rem;  // CTAs that take part

  __device__ __forceinline__ int64_t start(int c) const { return base * c + min(c, rem); }
  // the CTA whose share holds x
  __device__ __forceinline__ int cta_of(int64_t x) const {
    const int64_t wide = (base + 1) * rem;  // the first rem shares are one longer
    return x < wide ? static_cast<int>(div64(x, base + 1)) : rem + static_cast<int>(div64(x - wide, base));
  }
};

// The last block that starts at or before r on a head's part of the axis: r = n0 + (tb m^2 + a m) / 2 + cost (n0 + m)
// with a = 2 (ctx + tb n0) + tb solved for m (in the form without a difference of large numbers), then put right where
// the float was off.
__device__ __forceinline__ int block_at(const SeqUnits& s, int64_t r, const Division& dv) {
  int i;
  if (!dv.causal) {
    i = static_cast<int>(div64(r, unit_span(s.len, dv)));
  } else {
    const int64_t r0 = static_cast<int64_t>(s.n0) * (1 + dv.cost);
    if (r < r0) {
      i = static_cast<int>(div64(r, 1 + dv.cost));
    } else {
      const float tb = dv.tb, a = 2.f * (s.ctx + dv.tb * s.n0) + tb + 2.f * dv.cost, x = static_cast<float>(r - r0);
      const float d = sqrtf(a * a + 8.f * tb * x);
      i = s.n0 + static_cast<int>(a > 0.f ? 4.f * x / (a + d) : (d - a) / (2.f * tb));
    }
  }
  i = min(max(i, 0), s.nb - 1);
  while (i + 1 < s.nb && units_before(s, i + 1, dv) <= r) ++i;
  while (i > 0 && units_before(s, i, dv) > r) --i;
  return i;
}

// What the warps of a CTA need of a segment.
struct alignas(16) Seg {
  int b;         // sequence; -1: the share ends
  int hu, blk;   // unit
  int row0, n;   // the sequence's new tokens
  int ctx, len;
  int keys, t0, t1;
  int slot;      // of the partial result; -1: the output itself
  int it;        // running number of tile t0 in the share
};
static_assert(sizeof(Seg) == 48, "three 16-byte words");

// The unit that goes on behind a CTA's share.
struct Meta {
  int last;  // last CTA that holds a part of it; -1: no such unit
  int hu, blk, row0, n;
};

// Wait, by a whole warp at the end of its part, for copies or products that it started: a CTA that gives up after a
// timeout must not leave them running into memory that it has given back.  Bounded as the other waits are, but not cut
// short by a sibling's abort.  Without a timeout all of it has long been waited for.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity, int code) {
  uint64_t t0 = 0;
  for (uint32_t n = 1; !mbar_try_wait(bar, parity); ++n) {
    if ((n & 63u) != 0u) continue;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > CEA_WAIT_LIMIT_NS) {
      record_error(code);
      break;
    }
  }
  __syncwarp();
}

// The segments of a share pass from the one warp that walks them to the others through a short queue in shared
// memory, so that the walk (64-bit positions) is done once and ahead of its use.
constexpr int kQueue = 8;

struct SegQueue {
  uint8_t* seg;   // kQueue x Seg
  uint32_t full;  // kQueue barriers, one arrival
  uint32_t empty; // kQueue barriers, one arrival per reading warp
  volatile int* abort;
  int code;

  static constexpr int kBytes = kQueue * sizeof(Seg);
  static constexpr int kBars = 2 * kQueue;

  __device__ __forceinline__ void init(int readers) const {
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, readers);
    }
  }
  // by a whole warp
  __device__ __forceinline__ bool put(int i, const Seg& g, int lane) const {
    const uint32_t st = i % kQueue, n = i / kQueue;
    if (n > 0 && !__all_sync(0xffffffffu, mbar_wait(empty + 8 * st, (n - 1) & 1, abort, code))) return false;
    if (lane != 0) return true;
    int4* to = reinterpret_cast<int4*>(seg + st * sizeof(Seg));
    to[0] = make_int4(g.b, g.hu, g.blk, g.row0);
    to[1] = make_int4(g.n, g.ctx, g.len, g.keys);
    to[2] = make_int4(g.t0, g.t1, g.slot, g.it);
    mbar_arrive(full + 8 * st);
    return true;
  }
  __device__ __forceinline__ bool read(int i, Seg& g) const {
    const uint32_t st = i % kQueue, n = i / kQueue;
    if (!mbar_wait(full + 8 * st, n & 1, abort, code)) return false;
    const int4* from = reinterpret_cast<const int4*>(seg + st * sizeof(Seg));
    const int4 x = from[0], y = from[1], z = from[2];
    g = Seg{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
    return true;
  }
  // segment i, by a whole warp; false at the end of the share or after a timeout
  __device__ __forceinline__ bool get(int i, Seg& g, int lane) const {
    const bool ok = __all_sync(0xffffffffu, read(i, g));
    // all lanes' reads come before lane 0's release of the slot: a vote orders no memory, this does
    __syncwarp();
    if (ok && lane == 0) mbar_arrive(empty + 8 * (i % kQueue));
    return ok && g.b >= 0;
  }
};

// Walks this CTA's share: one whole warp, which hands every segment to `take` (and a Seg with b = -1 at the end); the
// unit that goes on behind the share is described in `meta`.  The code is met once per launch, from cold instruction
// caches, so each piece of it stands here once.
template <int BK, bool kOne, typename Take>
__device__ __forceinline__ void walk(const Batch& bt, const Division& dv, bool dead, Meta* meta, const Take& take) {
  const int lane = threadIdx.x & 31, cta = blockIdx.x;
  const int64_t cap = min(static_cast<int64_t>(bt.max_pages) * bt.ps, kMaxLen);
  Share sh;
  SeqUnits s;
  int64_t W = 0, lo = 0, hi = 0, pos = 0;  // the axis, this CTA's share, and where on it the walk is
  int b = dv.B;                            // sequence at lo
  // the axis's length, then the sequence that holds lo: 32 sequences at a time, one a lane
  Seq q = {0, 0, 0, 0};
  int64_t w = 0, end = 0;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int64_t before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < dv.B; b0 += 32) {
      if (pass == 0 || dv.B > 32) {
        q = Seq{0, 0, 0, 0};
        if (b0 + lane < dv.B) {
          q = load_seq(bt, b0 + lane);
          // a length that the table cannot hold, descending offsets, or a broken promise
          const int raw = bt.lens[b0 + lane], o0 = bt.q_off[b0 + lane], o1 = bt.q_off[b0 + lane + 1];
          if (raw < 0 || raw > cap || o0 < 0 || o1 < o0 || o1 > bt.T || (q.n > 0 && (q.n < dv.min_n || q.n > dv.max_n)))
            report(CEA_DEV_BAD_BATCH);
        }
        end = w = seq_units<kOne>(dv, q).S * dv.units_h;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t up = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end += up;
        }
      }
      if (pass == 1) {
        const unsigned hit = __ballot_sync(0xffffffffu, before + end > lo);
        if (hit != 0u) {
          const int l = __ffs(hit) - 1;
          b = b0 + l;
          pos = before + __shfl_sync(0xffffffffu, end - w, l);
          q = Seq{__shfl_sync(0xffffffffu, q.row0, l), __shfl_sync(0xffffffffu, q.n, l),
                  __shfl_sync(0xffffffffu, q.len, l), __shfl_sync(0xffffffffu, q.ctx, l)};
          break;
        }
      }
      before += __shfl_sync(0xffffffffu, end, 31);
    }
    if (pass == 0) {
      W = before;
      sh.n = static_cast<int>(min(static_cast<int64_t>(gridDim.x), max(int64_t(1), W >> dv.min_share_log2)));
      sh.base = div64(W, sh.n);
      sh.rem = static_cast<int>(W - sh.base * sh.n);
      lo = sh.start(min(cta, sh.n));
      hi = sh.start(min(cta + 1, sh.n));
      if (lo >= hi) break;
    } else {
      s = seq_units<kOne>(dv, q);
    }
  }

  Meta behind = {-1, 0, 0, 0, 0};
  int it = 0;
  bool ok = true;
  if (b < dv.B && !dead) {
    // from the start of the sequence to the unit that holds lo
    int64_t r = lo - pos;
    int hu = static_cast<int>(div64(r, s.S));
    r -= hu * s.S;
    int blk = kOne ? 0 : block_at(s, r, dv);
    pos += hu * s.S + (kOne ? 0 : units_before(s, blk, dv));
#pragma unroll 1
    while (pos < hi) {
      const int keys = kOne ? s.len : unit_keys(s, blk, dv.tb, dv.causal);
      const int nt = max(1, (keys + BK - 1) / BK);
      const int t0 = static_cast<int>((max(lo - pos, int64_t(0)) + BK - 1) / BK);
      const int t1 = static_cast<int>(min(static_cast<int64_t>(nt), (hi - pos + BK - 1) / BK));
      if (t0 < t1) {
        const int slot = t0 > 0 ? 2 * cta : t1 < nt ? 2 * cta + 1 : -1;
        if (t0 == 0 && t1 < nt) behind = Meta{sh.cta_of(pos + static_cast<int64_t>(nt - 1) * BK), hu, blk, s.row0, s.n};
        ok = take(Seg{b, hu, blk, s.row0, s.n, s.ctx, s.len, keys, t0, t1, slot, it});
        if (!ok) break;
        it += t1 - t0;
      }
      pos += unit_span(keys, dv);
      if (!kOne && ++blk < s.nb) continue;
      blk = 0;
      if (++hu < dv.units_h) continue;
      hu = 0;
      do {
        if (++b >= dv.B) break;
        s = seq_units<kOne>(dv, load_seq(bt, b));
      } while (s.S == 0);
      if (b >= dv.B) break;
    }
  }
  if (ok) take(Seg{-1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0});
  if (lane == 0) meta[cta] = behind;
}

template <typename A>
struct CombineArgs {
  Division dv;
  const A* part_o;    // [slot][rows][D]
  const A* part_lse;  // [slot][rows], natural log
  const Meta* meta;   // [CTA]
  int rows;           // rows of a slot
  void* out;
  int64_t o_ss, o_sh;
  A* lse;
  int64_t l_sh, l_ss;
  int D, out_dtype, heads_per_kv, head_groups;
};

template <typename A>
__device__ __forceinline__ void store_out(void* out, int64_t at, A v, int dtype) {
  if (dtype == CEA_BF16) reinterpret_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(static_cast<float>(v));
  else if (dtype == CEA_F16) reinterpret_cast<__half*>(out)[at] = __float2half_rn(static_cast<float>(v));
  else reinterpret_cast<A*>(out)[at] = v;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float log_of(float x) { return logf(x); }
__device__ __forceinline__ double log_of(double x) { return log(x); }

constexpr int kCombineThreads = 256;
constexpr int kMaxD = 256;

// 4 columns of a part; `vec`: rows are 16-byte aligned (D a multiple of 4)
__device__ __forceinline__ void load4(const float* p, int left, bool vec, float (&v)[4]) {
  if (vec) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : 0.f;
  }
}
__device__ __forceinline__ void load4(const double* p, int left, bool, double (&v)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : 0.0;
}

// Joins the parts of units that several CTAs worked on:
//   lse = ln sum_i exp(lse_i),  out = sum_i exp(lse_i - lse) out_i
// in the partials' precision, parts in the order of the keys (the result does not depend on timing).  The unit that
// goes on behind CTA c has its first part in slot 2 c + 1 and the others in the slots 2 (c + 1), 2 (c + 2), ...: a share
// is at least a tile long, so every CTA up to the unit's last one holds a part.
// Block (c, y): rows y * RPB ...; 8 / RPB warps share a row's parts, a lane has 4 columns.  Bound by latency and L2: a
// call's partials (at most 2 slots per CTA) are just written, so the weights of 32 parts are formed at once, one a lane,
// and the parts are read four at a time.
template <typename A, int RPB>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const __grid_constant__ CombineArgs<A> a) {
  constexpr int WPR = 8 / RPB;  // warps per row
  constexpr int C = kMaxD / 128;
  __shared__ A acc_s[WPR > 1 ? 8 : 1][WPR > 1 ? kMaxD : 1];
  __shared__ A sum_s[8];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int status = *reinterpret_cast<volatile int*>(&g_cea_status);
  const Meta m = a.meta[c];
  if (status != 0 || m.last < 0) return;  // after a timeout parts may be missing
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.y * RPB + warp / WPR, sub = warp % WPR;
  const int tok = m.blk * a.dv.tb + row / a.dv.group, g = (m.hu % a.head_groups) * a.dv.group + row % a.dv.group;
  const int head = (m.hu / a.head_groups) * a.heads_per_kv + g;
  const bool in = row < a.dv.tb * a.dv.group && tok < m.n && g < a.heads_per_kv;
  const int parts = m.last - c + 1;
  const bool vec = a.D % 4 == 0;
  auto slot = [&](int i) -> int64_t { return i == 0 ? 2 * c + 1 : 2 * (c + i); };
  const int64_t orow = (static_cast<int64_t>(m.row0) + tok) * a.o_ss + head * a.o_sh;
  const int64_t lrow = head * a.l_sh + (static_cast<int64_t>(m.row0) + tok) * a.l_ss;
  A top = -INFINITY, sum = 0;
  A acc[C][4];
#pragma unroll
  for (int j = 0; j < C; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0;
  if (in) {
    for (int i = lane; i < parts; i += 32) top = max(top, a.part_lse[slot(i) * a.rows + row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = top == -INFINITY ? A(0) : top;  // a row no part of which saw a key
    // this warp's parts: sub, sub + WPR, ...
    for (int i0 = 0; i0 * WPR + sub < parts; i0 += 32) {
      const int mine = (i0 + lane) * WPR + sub, here = min(32, (parts - sub - i0 * WPR + WPR - 1) / WPR);
      const A w = mine < parts ? exp_of(a.part_lse[slot(mine) * a.rows + row] - top) : A(0);
      sum += w;
      for (int i = 0; i < here; i += 4) {
        A wi[4], v[4][C][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          wi[k] = __shfl_sync(0xffffffffu, w, (i + k) & 31);
          if (i + k >= here) wi[k] = 0;
          const A* src = a.part_o + (slot((i0 + min(i + k, here - 1)) * WPR + sub) * a.rows + row) * a.D;
#pragma unroll
          for (int j = 0; j < C; ++j) {
            v[k][j][0] = v[k][j][1] = v[k][j][2] = v[k][j][3] = 0;
            if (j * 128 + lane * 4 < a.D) load4(src + j * 128 + lane * 4, a.D - j * 128 - lane * 4, vec, v[k][j]);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < C; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (i + k < here) acc[j][e] += wi[k] * v[k][j][e];
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if constexpr (WPR == 1) {
    if (!in) return;
    const A inv = sum == A(0) ? A(0) : A(1) / sum;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j * 128 + lane * 4 + e < a.D) store_out<A>(a.out, orow + j * 128 + lane * 4 + e, acc[j][e] * inv, a.out_dtype);
    if (lane == 0 && a.lse != nullptr) a.lse[lrow] = sum == A(0) ? A(-INFINITY) : top + log_of(sum);
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc_s[warp][j * 128 + lane * 4 + e] = acc[j][e];
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (!in) return;
    const int w0 = warp / WPR * WPR;
    A total = 0;
#pragma unroll
    for (int w = 0; w < WPR; ++w) total += sum_s[w0 + w];
    const A inv = total == A(0) ? A(0) : A(1) / total;
    for (int d = sub * 32 + lane; d < a.D; d += WPR * 32) {
      A v = 0;
#pragma unroll
      for (int w = 0; w < WPR; ++w) v += acc_s[w0 + w][d];
      store_out<A>(a.out, orow + d, v * inv, a.out_dtype);
    }
    if (sub == 0 && lane == 0 && a.lse != nullptr) a.lse[lrow] = total == A(0) ? A(-INFINITY) : top + log_of(total);
  }
}

// The same for the chunk kernel's slots of 256 rows, laid out [slot][D / 4][row][4] so that its rows (one a thread) are
// written, and read here, in whole lines.  Bound by L2: block (c, y) takes 32 rows, one a lane, and each of its 8 warps
// D / 8 columns; a lane has four parts' statistics and columns in flight at a time.
// One warp a row with a lane per 4 columns took 17 us for 148 split units of 256 rows, bound by the latency of four
// waves of blocks.
constexpr int kWideRows = 256;

template <int D>
__global__ void __launch_bounds__(kCombineThreads) combine_wide_kernel(const __grid_constant__ CombineArgs<float> a) {
  constexpr int C4 = D / 32;  // float4 of a lane
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x;
  const int status = *reinterpret_cast<volatile int*>(&g_cea_status);
  const Meta m = a.meta[c];
  if (status != 0 || m.last < 0) return;  // after a timeout parts may be missing
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.y * 32 + lane;
  const int tok = m.blk * a.dv.tb + row / a.dv.group, head = m.hu * a.dv.group + row % a.dv.group;
  if (row >= a.dv.tb * a.dv.group || tok >= m.n) return;
  const int parts = m.last - c + 1;
  float top = -INFINITY, sum = 0.f;
  float4 acc[C4];
#pragma unroll
  for (int j = 0; j < C4; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int P = 4;
  for (int i = 0; i < parts; i += P) {
    float lse[P], up = top;
    float4 v[P][C4];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      lse[k] = -INFINITY;
#pragma unroll
      for (int j = 0; j < C4; ++j) v[k][j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i + k < parts) {
        const int64_t slot = i + k == 0 ? 2 * c + 1 : 2 * (c + i + k);
        lse[k] = a.part_lse[slot * kWideRows + row];
        const float4* src = reinterpret_cast<const float4*>(a.part_o) + (slot * (D / 4) + warp * C4) * kWideRows + row;
#pragma unroll
        for (int j = 0; j < C4; ++j) v[k][j] = src[j * kWideRows];
      }
    }
#pragma unroll
    for (int k = 0; k < P; ++k) up = fmaxf(up, lse[k]);
    const float ref = up == -INFINITY ? 0.f : up, w = expf(top - ref);
    top = up;
    sum *= w;
#pragma unroll
    for (int j = 0; j < C4; ++j) acc[j] = make_float4(acc[j].x * w, acc[j].y * w, acc[j].z * w, acc[j].w * w);
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const float wk = expf(lse[k] - ref);
      sum += wk;
#pragma unroll
      for (int j = 0; j < C4; ++j) {
        acc[j].x += wk * v[k][j].x;
        acc[j].y += wk * v[k][j].y;
        acc[j].z += wk * v[k][j].z;
        acc[j].w += wk * v[k][j].w;
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t trow = static_cast<int64_t>(m.row0) + tok;
  const int64_t at = trow * a.o_ss + head * a.o_sh + warp * C4 * 4;
#pragma unroll
  for (int j = 0; j < C4; ++j) {
    const float4 o = make_float4(acc[j].x * inv, acc[j].y * inv, acc[j].z * inv, acc[j].w * inv);
    if (a.out_dtype == CEA_F32)
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + at + j * 4) = o;
    else
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + at + j * 4) =
          make_uint2(pack2(o.x, o.y, a.out_dtype == CEA_BF16), pack2(o.z, o.w, a.out_dtype == CEA_BF16));
  }
  if (warp == 0 && a.lse != nullptr)
    a.lse[head * a.l_sh + trow * a.l_ss] = sum == 0.f ? -INFINITY : top + logf(sum);
}

// ------------------------------------------------------------------ append
// New token rows into their pages, bit for bit: one warp per token moves its K and its V rows.  Bound by HBM for
// prompts and by latency for a decoding step, so the loads of the rows are issued before the walk from the token to
// its page (sequence by a 32-way search of the offsets, then the table) and stored after it.
// A row's position is counted back from its sequence's length and end, so rows that the caller's k and v lack change no
// other row's place.  One block more than the rows need looks at all offsets and reports a batch that does not fit.
struct AppendArgs {
  Batch bt;
  const uint8_t* src[2];   // k, v
  uint8_t* dst[2];         // pages
  int64_t src_ss[2], src_sh[2];           // bytes: token, head
  int64_t dst_sp[2], dst_sh[2], dst_ss[2];  // bytes: page, head, slot
  int H;
  kvc::FastDiv units;      // units of U bytes per head row
};

// sequence of row t: the last b with q_off[b] <= t (offsets ascend; empty sequences are passed over), -1 if none
__device__ __forceinline__ int find_seq(const Batch& bt, int t, int lane) {
  int lo = 0, hi = bt.B + 1;  // q_off[lo - 1] <= t (or lo = 0), q_off[hi] > t (or hi = B + 1)
  while (hi - lo > 0) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const bool le = i < hi && bt.q_off[i] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, le));  // offsets ascend: the first c probes hold
    if (c == 0) return lo - 1;
    const int first = lo + (c - 1) * step;  // q_off[first] <= t
    hi = c < 32 ? min(hi, lo + c * step) : hi;
    lo = first + 1;
  }
  return lo - 1;
}

constexpr int kAppendThreads = 128;
constexpr int kAppendUnroll = 4;

template <typename U>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int per = a.H * static_cast<int>(a.units.d);  // units of one token's K (or V)
  // head and byte offset of this lane's units, the same for every token
  int head[kAppendUnroll], byte[kAppendUnroll];
  auto place = [&](int i, int& h, int& at) {
    h = static_cast<int>(kvc::fdiv(i, a.units));
    at = (i - h * static_cast<int>(a.units.d)) * static_cast<int>(sizeof(U));
  };
#pragma unroll
  for (int j = 0; j < kAppendUnroll; ++j) place(j * 32 + lane, head[j], byte[j]);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == gridDim.x - 1) {
    for (int b = threadIdx.x; b < a.bt.B; b += kAppendThreads) {
      const int o0 = a.bt.q_off[b], o1 = a.bt.q_off[b + 1];
      if (o0 < 0 || o1 < o0 || o1 > a.bt.T) report(CEA_DEV_BAD_BATCH);
    }
    return;
  }
  const unsigned stride = (gridDim.x - 1) * (kAppendThreads / 32);
  // unsigned: a stride behind the last of 2^31 - 1 rows is above an int
  for (unsigned row = blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5); row < static_cast<unsigned>(a.bt.T);
       row += stride) {
    const int t = static_cast<int>(row);
    U val[2][kAppendUnroll];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < kAppendUnroll; ++j)
        if (j * 32 + lane < per)
          val[x][j] = *reinterpret_cast<const U*>(a.src[x] + t * a.src_ss[x] + head[j] * a.src_sh[x] + byte[j]);
    const int b = find_seq(a.bt, t, lane);
    if (b < 0 || b >= a.bt.B) continue;  // before the first or behind the last sequence
    const int64_t pos = static_cast<int64_t>(a.bt.lens[b]) - a.bt.q_off[b + 1] + t;
    if (t >= a.bt.q_off[b + 1]) continue;  // offsets that descend
    const int64_t page_i = pos < 0                ? -1
                           : (pos >> 32) == 0 ? static_cast<uint32_t>(pos) / static_cast<uint32_t>(a.bt.ps)
                                              : pos / a.bt.ps;
    const int page = page_i >= 0 && page_i < a.bt.max_pages ? a.bt.table[b * a.bt.table_sb + page_i] : -1;
    if (page < 0 || page >= a.bt.num_pages) {
      if (lane == 0) report(CEA_DEV_BAD_PAGE);
      continue;
    }
    const int64_t slot = pos - page_i * a.bt.ps;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      uint8_t* dst = a.dst[x] + page * a.dst_sp[x] + slot * a.dst_ss[x];
#pragma unroll
      for (int j = 0; j < kAppendUnroll; ++j)
        if (j * 32 + lane < per) *reinterpret_cast<U*>(dst + head[j] * a.dst_sh[x] + byte[j]) = val[x][j];
      for (int i = kAppendUnroll * 32 + lane; i < per; i += 32) {  // rows longer than the loads in flight
        int h, at;
        place(i, h, at);
        *reinterpret_cast<U*>(dst + h * a.dst_sh[x] + at) =
            *reinterpret_cast<const U*>(a.src[x] + t * a.src_ss[x] + h * a.src_sh[x] + at);
      }
    }
  }
}

// ------------------------------------------------------------------ page copy
// Pages src[i] -> dst[i] of every layer's K and V pool.  The pairs travel as kernel arguments (no copy of them to the
// device, and a captured graph keeps its own).  No page is both read and written (checked on the host), so the order
// of the copies does not matter.  Bound by HBM: 16-byte units, kCopyUnroll loads in flight per thread.
constexpr int kCopyPairs = 480;  // a 4 KB argument block
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;

struct CopyArgs {
  uint8_t* pool[2];
  int64_t page_stride[2], layer_stride[2];  // bytes
  int64_t units;                            // units of U bytes per page
  int n, layers;
  int2 pair[kCopyPairs];
};

template <typename U>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  // blockIdx.x walks the chunks of a page, then the pairs; y the layers, z K or V
  constexpr int kChunk = kCopyThreads * kCopyUnroll;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int chunks = static_cast<int>((a.units + kChunk - 1) / kChunk);
  const int i = blockIdx.x / chunks;
  const int64_t u0 = static_cast<int64_t>(blockIdx.x % chunks) * kChunk + threadIdx.x;
  const int2 pr = a.pair[i];
  for (int layer = blockIdx.y; layer < a.layers; layer += gridDim.y) {
    uint8_t* base = (blockIdx.z ? a.pool[1] : a.pool[0]) + layer * a.layer_stride[blockIdx.z];
    const U* src = reinterpret_cast<const U*>(base + pr.x * a.page_stride[blockIdx.z]);
    U* dst = reinterpret_cast<U*>(base + pr.y * a.page_stride[blockIdx.z]);
    U v[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
      if (u0 + j * kCopyThreads < a.units) v[j] = src[u0 + j * kCopyThreads];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
      if (u0 + j * kCopyThreads < a.units) dst[u0 + j * kCopyThreads] = v[j];
  }
}

}  // namespace paged
}  // namespace cea

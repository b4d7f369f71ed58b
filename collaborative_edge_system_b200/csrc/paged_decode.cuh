// Attention over a paged cache for sequences with few new tokens (n_b * G <= 16 query rows per KV head): the form of
// a decoding step and of a few proposed tokens.
//
// HBM-bound: K and V are read once, about 4 FLOP per byte at a group of 4 query heads.  One CTA per SM takes an
// equal share of all key tiles of the batch (paged.cuh), so lengths may differ at will and no CTA idles.  Three
// producer warps stream 64-key K and V tiles into a ring of 192 KB with TMA, one box per page (or part of one) and 64
// columns, each lane looking its box's page up; a warp takes about 60 ns a box and 0.5 us a tile, so the warps take the
// tiles in turn (one warp for all of them: 2.8 TB/s at pages of 8 and 4.5 at 16; the boxes of each tile dealt to four
// warps: 5.3 and 6.1, and 3.8 at D = 64; the tiles in turn: 6.5 and 6.5, and 6.0 at D = 64; 32 sequences of 16384, 8 KV
// heads).  A fourth warp finds the segments of the share ahead of the loads; the ring runs on across them, so the loads
// do not pause while the consumer warps join their results.  Two groups of four consumer warps take the tiles in turn, each
// warp 16 keys, transposed on mma.sync m16n8k16 so that the keys (and then the columns of V) fill the 16 rows and the few
// query rows the 8 columns: S^T = K Q^T, online softmax in the log2 domain down the columns, O^T += V^T P^T.  With
// the query rows on the 16-row side instead, half of each product was padding at 4 or 8 rows.  P is carried as the
// sum of two 16-bit numbers (the value's rounding and the rounding of what that leaves), which doubles the PV products:
// what is lost is 2^-17 of a probability in bf16, and in f16 2^-22 of it or 2^-39 of the row's largest.  In f16 numbers
// below 2^-14 lose bits and those below 2^-25 are 0, so the probabilities there are held as 2^14 times their ratio to the
// running maximum (at most 2^14, of 65504); held with the maximum at 1, keys 17 to 18 nats below one that outweighs them
// counted in the sum and not in the output.  TMA boxes behind the last key are not loaded, and the V fragments of keys
// behind it are zeroed in registers, so slots that hold no token never count, whatever they hold.  A probability of 0 does
// not silence an infinity or a NaN, so the keys that not all rows see are searched for them ahead of the products; the
// product with the remainders leaves them out everywhere (12 sequences with 2 to 5 new tokens 38.6 -> 40 us, the 16-row
// form at D = 64, bound by its instructions, 72 -> 76 us for 32 sequences of 4096 with 4).
#pragma once

#include "decode.cuh"
#include "paged.cuh"

namespace cea {
namespace paged {
namespace dec {

using cea::dec::ldsm_x4;
using cea::dec::ldsm_x4_t;
using cea::dec::mma16816;
using cea::dec::swz;

constexpr int BK = 64;
constexpr int NCW = 8;  // consumer warps: two groups of four
constexpr int NPW = 3;  // producer warps, which take the tiles in turn (a 13th warp would leave 128 registers a thread)
constexpr int ROWS = 16;  // query rows of a slot
constexpr int kWalkWarp = NCW + NPW;
constexpr int NTHREADS = (NCW + NPW + 1) * 32;

template <int D>
struct Layout {
  static constexpr int KBOX = D / 64;
  static constexpr int BOX = BK * 128;  // 64 columns of all 64 keys
  static constexpr int TILE = KBOX * BOX;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int NSTAGE = D == 128 ? 6 : 12;
  // A parity wait is right only for a warp that has seen the phase before last complete.  So a stage is always filled
  // by one producer warp and always read by one group of consumers, each of which meets its phases one by one.
  static_assert(NSTAGE % NPW == 0 && NSTAGE % 2 == 0, "a stage has one producer warp and one consumer group");
  static constexpr int DT = D / 16;
  // buffer of the join: [NCW][DT][32] float4, the fragments of 8 query rows, and their [NCW][8] max, then sum
  static constexpr int OFF_JOIN = NSTAGE * STAGE;
  static constexpr int OFF_STAT = OFF_JOIN + NCW * DT * 32 * 16;
  static constexpr int OFF_QUEUE = OFF_STAT + 2 * NCW * 8 * 4;
  static constexpr int OFF_BAR = OFF_QUEUE + SegQueue::kBytes;
  static constexpr int B_FULL = 0;
  static constexpr int B_EMPTY = B_FULL + NSTAGE;
  static constexpr int B_WRITTEN = B_EMPTY + NSTAGE;  // the join's buffer
  static constexpr int B_READ = B_WRITTEN + 1;
  static constexpr int B_QUEUE = B_READ + 1;
  static constexpr int NBAR = B_QUEUE + SegQueue::kBars;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = OFF_MISC + 16;
  static constexpr int SMEM_ALLOC = BYTES + 1024;
  static_assert(OFF_QUEUE % 16 == 0 && SMEM_ALLOC <= 232448, "shared memory");
};

struct Params {
  Batch bt;
  Division dv;
  const void* q;
  int64_t q_ss, q_sh;
  void* out;
  int64_t o_ss, o_sh;
  float* lse;
  int64_t l_sh, l_ss;
  float* part_o;
  float* part_lse;
  Meta* meta;
  int box;  // rows of a TMA box: divides the page and the tile
  int out_dtype;
  float scale_log2;
};

// log2 of the probability that a row's running maximum is given
template <bool kBF16>
constexpr float kTopLog2 = kBF16 ? 0.f : 14.f;

template <bool kBF16>
__device__ __forceinline__ float round16(float x) {
  if constexpr (kBF16) return __bfloat162float(__float2bfloat16_rn(x));
  return __half2float(__float2half_rn(x));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D, bool kBF16, int NT>
__global__ void __launch_bounds__(NTHREADS, 1)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ Params p) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
  auto bar = [&](int i) -> uint32_t { return sbase + L::OFF_BAR + 8 * i; };
  const SegQueue queue{smem + L::OFF_QUEUE, bar(L::B_QUEUE), bar(L::B_QUEUE + kQueue), abort_flag,
                       CEA_DEV_TIMEOUT_DECODE};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NSTAGE; ++s) {
      mbar_init(bar(L::B_FULL + s), 1);
      mbar_init(bar(L::B_EMPTY + s), NCW / 2);
    }
    mbar_init(bar(L::B_WRITTEN), NCW);
    mbar_init(bar(L::B_READ), NCW);
    queue.init(NCW + NPW);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp == kWalkWarp) {
    int i = 0;
    // after a device-side timeout nothing is computed
    const bool dead = *reinterpret_cast<volatile int*>(&g_cea_status) != 0;
    walk<BK, true>(p.bt, p.dv, dead, p.meta, [&](const Seg& g) -> bool { return queue.put(i++, g, lane); });
    return;
  }

  Seg g;
  if (warp >= NCW) {
    // ---------------------------------------------------------------- producers: one TMA box per lane
    const int nbox = BK / p.box;  // boxes of 64 columns along a tile's keys
    const int box = lane % nbox, half = (lane / nbox) % L::KBOX, is_v = lane / (nbox * L::KBOX);
    const bool mine = is_v < 2;
    const CUtensorMap* map = is_v == 1 ? &tmV : &tmK;
    const uint32_t dst0 = is_v * L::TILE + half * L::BOX + box * p.box * 128;
    const int none = p.bt.num_pages;
    bool ok = true;
    int last = -1;  // tile loaded last
    for (int i = 0; ok && queue.get(i, g, lane); ++i) {
      const int32_t* table = p.bt.table + g.b * p.bt.table_sb;
      for (int t = g.t0 + (warp - NCW + NPW - g.it % NPW) % NPW; t < g.t1; t += NPW) {
        const int at = g.it + (t - g.t0);
        const int st = at % L::NSTAGE;
        const uint32_t n = at / L::NSTAGE;
        const int key = t * BK + box * p.box;
        const bool load = mine && key < g.keys;
        int page = 0, slot = 0;
        if (load) {
          const int page_i = key / p.bt.ps;
          slot = key - page_i * p.bt.ps;
          page = table[page_i];
          if (page < 0 || page >= none) {
            report(CEA_DEV_BAD_PAGE);
            page = none;  // outside the tensor map: reads as zeros
          }
        }
        if (n > 0) ok = mbar_wait(bar(L::B_EMPTY + st), (n - 1) & 1, abort_flag, CEA_DEV_TIMEOUT_DECODE);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int boxes = __popc(__ballot_sync(0xffffffffu, load));
        if (lane == 0) mbar_arrive_expect_tx(bar(L::B_FULL + st), boxes * p.box * 128);
        __syncwarp();
        if (load) tma_load_4d(sbase + st * L::STAGE + dst0, map, bar(L::B_FULL + st), half * 64, slot, g.hu, page);
        last = at;
      }
    }
    // the last load of each of this warp's stages
    for (int at = last; at >= 0 && at > last - L::NSTAGE; at -= NPW)
      drain(bar(L::B_FULL + at % L::NSTAGE), (at / L::NSTAGE) & 1, CEA_DEV_TIMEOUT_DECODE);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int grp = warp >> 2, key0 = (warp & 3) * 16;  // this warp's keys within a tile
  const int G = p.dv.group;
  const int mi = lane >> 3, ri = lane & 7, kr = lane >> 2, c2 = 2 * (lane & 3);

  uint32_t qb[NT][D / 16][2];  // Q^T fragments: rows nt * 8 + kr
  auto load_q = [&]() {
    const int R = g.n * G;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + kr, tok = r / G;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(g.row0) + tok) * p.q_ss +
                            (g.hu * G + r - tok * G) * p.q_sh + c2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qb[nt][kk][0] = r < R ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
        qb[nt][kk][1] = r < R ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
      }
    }
  };
  int joins = 0;
  bool more = queue.get(0, g, lane);
  if (more) load_q();
  for (int i = 1; more; ++i) {
    // last key that rows nt * 8 + c2, + 1 see, -1 for none
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = nt * 8 + c2 + e, seen = g.len - 1;
        lim[nt][e] = r >= g.n * G ? -1 : (p.dv.causal ? min(g.ctx + r / G, seen) : seen);
      }
    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (int t = g.t0 + ((grp ^ g.it) & 1); t < g.t1; t += 2) {
      const int at = g.it + (t - g.t0);
      const int st = at % L::NSTAGE;
      const bool got = mbar_wait(bar(L::B_FULL + st), (at / L::NSTAGE) & 1, abort_flag, CEA_DEV_TIMEOUT_DECODE);
      if (!__all_sync(0xffffffffu, got)) return;
      const uint32_t kt = sbase + st * L::STAGE;
      const uint32_t vt = kt + L::TILE;
      const int left = g.keys - t * BK;  // keys of the unit in this tile
      if (left > key0) {                 // warp-uniform: else none of this warp's keys exists
        float s[NT][2][4];               // two chains of products, added below
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][0][e] = s[nt][1][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t a[4];
          ldsm_x4(swz(kt, key0 + ((mi & 1) << 3) + ri, 2 * kk + (mi >> 1)), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<kBF16>(s[nt][kk & 1], a, qb[nt][kk][0], qb[nt][kk][1]);
        }
        const int kA = t * BK + key0 + kr, kB = kA + 8;
        uint32_t pb[NT][2], pl[NT][2];  // P^T = pb + pl
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = (s[nt][0][e] + s[nt][1][e]) * p.scale_log2;
            x[e] = (e < 2 ? kA : kB) <= lim[nt][e & 1] ? v : -INFINITY;
          }
          float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], off));
            top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], off));
          }
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float nm = fmaxf(m[nt][e], top[e]);
            const float u = nm == -INFINITY ? 0.f : nm, u1 = u - kTopLog2<kBF16>;
            alpha[e] = fast_exp2(m[nt][e] - u);
            m[nt][e] = nm;
            x[e] = fast_exp2(x[e] - u1);
            x[2 + e] = fast_exp2(x[2 + e] - u1);
            l[nt][e] = l[nt][e] * alpha[e] + x[e] + x[2 + e];
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float y0 = x[2 * k], y1 = x[2 * k + 1];
            pb[nt][k] = transpose8x8(pack2(y0, y1, kBF16));
            pl[nt][k] = transpose8x8(pack2(y0 - round16<kBF16>(y0), y1 - round16<kBF16>(y1), kBF16));
          }
          if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              o[nt][j][0] *= alpha[0];
              o[nt][j][1] *= alpha[1];
              o[nt][j][2] *= alpha[0];
              o[nt][j][3] *= alpha[1];
            }
          }
        }
        // V^T fragment words hold keys c2, c2 + 1 of the first or second 8 keys
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (left < key0 + 16) {
          const int k0 = key0 + c2;
          keep0 = (k0 < left ? 0xffffu : 0u) | (k0 + 1 < left ? 0xffff0000u : 0u);
          keep1 = (k0 + 8 < left ? 0xffffu : 0u) | (k0 + 9 < left ? 0xffff0000u : 0u);
        }
        // Keys that not all rows see: a probability of 0 does not silence an infinity or a NaN.  They are added to the rows
        // that see them here, and zeros take their place in this warp's part of the tile.
        if (t * BK + key0 + min(16, left - key0) > (p.dv.causal ? g.ctx : g.len - 1) + 1) {
          uint32_t other = 0;
          for (int i = lane; i < 16 * (D / 8); i += 32) {
            const uint4 w = *reinterpret_cast<const uint4*>(smem + (swz(vt, key0 + (i & 15), i >> 4) - sbase));
            note_other<kBF16>(w.x, other);
            note_other<kBF16>(w.y, other);
            note_other<kBF16>(w.z, other);
            note_other<kBF16>(w.w, other);
          }
          if (__any_sync(0xffffffffu, other != 0u)) {
#pragma unroll 1
            for (int k = 0; k < min(16, left - key0); ++k) {
              const int key = t * BK + key0 + k;
#pragma unroll
              for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  const int d = j * 16 + 8 * x + kr;
                  uint16_t* at = reinterpret_cast<uint16_t*>(smem + (swz(vt, key0 + k, d >> 3) - sbase) + (d & 7) * 2);
                  const uint32_t bits = *at;
                  __syncwarp();  // four lanes share a column
                  if (finite_or_zero<kBF16>(bits) == bits) continue;
                  *at = 0;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                      if (key <= lim[nt][e]) o[nt][j][2 * x + e] += widen16<kBF16>(bits);
                }
              __syncwarp();
            }
            fence_async_smem();  // the stage's next load comes behind these writes
          }
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t a[4];
          ldsm_x4_t(swz(vt, key0 + ((mi >> 1) << 3) + ri, 2 * j + (mi & 1)), a[0], a[1], a[2], a[3]);
          a[0] &= keep0;
          a[1] &= keep0;
          a[2] &= keep1;
          a[3] &= keep1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<kBF16>(o[nt][j], a, pb[nt][0], pb[nt][1]);
          // an infinity counts in the first product only: the second's factor, a remainder, may be 0 or negative
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] = finite_or_zero<kBF16>(a[e]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816<kBF16>(o[nt][j], a, pl[nt][0], pl[nt][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(L::B_EMPTY + st));
    }

    // the next segment's queries travel while this one's results are joined
    const Seg was = g;
    more = queue.get(i, g, lane);
    if (more) load_q();

    // ------------------------------------------------- join the warps' results, in the order of the warps
    float4* os = reinterpret_cast<float4*>(smem + L::OFF_JOIN);
    float* ms = reinterpret_cast<float*>(smem + L::OFF_STAT);
    float* ls = ms + NCW * 8;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt, ++joins) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], off);
      // the reads of the join before
      const bool left_it =
          joins == 0 || mbar_spin(bar(L::B_READ), (joins - 1) & 1, abort_flag, CEA_DEV_TIMEOUT_DECODE);
      if (!__all_sync(0xffffffffu, left_it)) return;
      if (kr == 0) {
        *reinterpret_cast<float2*>(ms + warp * 8 + c2) = make_float2(m[nt][0], m[nt][1]);
        *reinterpret_cast<float2*>(ls + warp * 8 + c2) = make_float2(l[nt][0], l[nt][1]);
      }
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
        os[(warp * L::DT + j) * 32 + lane] = make_float4(o[nt][j][0], o[nt][j][1], o[nt][j][2], o[nt][j][3]);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(L::B_WRITTEN));
      const bool met = mbar_spin(bar(L::B_WRITTEN), joins & 1, abort_flag, CEA_DEV_TIMEOUT_DECODE);
      if (!__all_sync(0xffffffffu, met)) return;
      // warp j of the eight: columns 16 j .. 16 j + 15 of all rows (D = 64: the first four)
      if (warp < L::DT) {
        float v[4] = {0.f, 0.f, 0.f, 0.f}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, lse[2];
        float2 mw[NCW];
#pragma unroll
        for (int w = 0; w < NCW; ++w) {
          mw[w] = *reinterpret_cast<const float2*>(ms + w * 8 + c2);
          top[0] = fmaxf(top[0], mw[w].x);
          top[1] = fmaxf(top[1], mw[w].y);
        }
        const float u0 = top[0] == -INFINITY ? 0.f : top[0], u1 = top[1] == -INFINITY ? 0.f : top[1];
#pragma unroll
        for (int w = 0; w < NCW; ++w) {
          const float w0 = fast_exp2(mw[w].x - u0), w1 = fast_exp2(mw[w].y - u1);
          const float2 lw = *reinterpret_cast<const float2*>(ls + w * 8 + c2);
          const float4 f = os[(w * L::DT + warp) * 32 + lane];
          sum[0] += w0 * lw.x;
          sum[1] += w1 * lw.y;
          v[0] += w0 * f.x;
          v[1] += w1 * f.y;
          v[2] += w0 * f.z;
          v[3] += w1 * f.w;
        }
        lse[0] = sum[0] == 0.f ? -INFINITY : (u0 + (log2f(sum[0]) - kTopLog2<kBF16>)) * kLn2;
        lse[1] = sum[1] == 0.f ? -INFINITY : (u1 + (log2f(sum[1]) - kTopLog2<kBF16>)) * kLn2;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + c2 + e;
          if (r >= was.n * G) continue;
          const int tok = r / G, head = was.hu * G + r - tok * G;
          const int64_t trow = static_cast<int64_t>(was.row0) + tok;
          const int d = warp * 16 + kr;
          const float inv = sum[e] == 0.f ? 0.f : 1.f / sum[e];
          const float x = v[e] * inv, y = v[2 + e] * inv;
          if (was.slot >= 0) {
            float* po = p.part_o + (static_cast<int64_t>(was.slot) * ROWS + r) * D;
            po[d] = x;
            po[d + 8] = y;
            if (warp == 0 && kr == 0) p.part_lse[static_cast<int64_t>(was.slot) * ROWS + r] = lse[e];
          } else {
            const int64_t to = trow * p.o_ss + head * p.o_sh + d;
            store_out<float>(p.out, to, x, p.out_dtype);
            store_out<float>(p.out, to + 8, y, p.out_dtype);
            if (warp == 0 && kr == 0 && p.lse != nullptr) p.lse[head * p.l_sh + trow * p.l_ss] = lse[e];
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(L::B_READ));
    }
  }
}

}  // namespace dec
}  // namespace paged
}  // namespace cea

// Attention over a paged cache for sequences with few new tokens (n_b * G <= 16 query rows per KV head): the form of
// a decoding step and of a few proposed tokens.
//
// HBM-bound: K and V are read once, about 4 FLOP per byte at a group of 4 query heads.  One CTA per SM takes an
// equal share of all key tiles of the batch (paged.cuh), so lengths may differ at will and no CTA idles; a warp
// streams 64-key K and V tiles into a ring of 192 KB with TMA, one box per page (or part of one), its lanes looking
// the pages up and issuing the boxes side by side; the ring runs on across the segments of a share, so the loads do not
// pause while four consumer warps join their results.  Consumer warp w takes keys 16w .. 16w + 15 of a tile for the 16
// (padded) query rows on mma.sync m16n8k16: S = Q K^T, online softmax in the log2 domain, O += P V.  P is carried as
// the sum of two 16-bit numbers (the value's rounding and the rounding of what that leaves, 2^-17 of the value for
// bf16), which doubles the PV products and makes the result as exact as fp32 probabilities; the products are far from
// the bound.  TMA boxes behind the last key are not loaded, and the V fragments of keys behind it are zeroed in
// registers, so slots that hold no token never count, whatever they hold.
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
constexpr int NCW = 4;
constexpr int NTHREADS = (NCW + 1) * 32;
constexpr int ROWS = 16;

template <int D>
struct Layout {
  static constexpr int KBOX = D / 64;
  static constexpr int BOX = BK * 128;  // 64 columns of all 64 keys
  static constexpr int TILE = KBOX * BOX;
  static constexpr int STAGE = 2 * TILE;
  static constexpr int NSTAGE = 196608 / STAGE;
  static constexpr int LDO = D + 4;
  static constexpr int OFF_MERGE = NSTAGE * STAGE;  // [NCW][16] max, sum, then [NCW][16][LDO]
  static constexpr int OFF_BAR = OFF_MERGE + NCW * ROWS * (LDO + 2) * 4;
  static constexpr int OFF_MISC = OFF_BAR + 2 * NSTAGE * 8;
  static constexpr int BYTES = OFF_MISC + 16;
  static constexpr int SMEM_ALLOC = BYTES + 1024;
  static_assert(SMEM_ALLOC <= 232448, "shared memory");
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

template <bool kBF16>
__device__ __forceinline__ float round16(float x) {
  if constexpr (kBF16) return __bfloat162float(__float2bfloat16_rn(x));
  return __half2float(__float2half_rn(x));
}

template <int D, bool kBF16>
__global__ void __launch_bounds__(NTHREADS)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ Params p) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);
  auto full_bar = [&](int s) -> uint32_t { return sbase + L::OFF_BAR + 8 * s; };
  auto empty_bar = [&](int s) -> uint32_t { return sbase + L::OFF_BAR + 8 * (L::NSTAGE + s); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < L::NSTAGE; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), NCW);
    }
    // after a device-side timeout nothing is computed (the shares below are walked without waiting for data)
    *abort_flag = *reinterpret_cast<volatile int*>(&g_cea_status) != 0;
    fence_mbar_init();
  }
  const Share sh = divide(p.bt, p.dv, reinterpret_cast<int64_t*>(smem + L::OFF_MERGE));
  asm volatile("griddepcontrol.launch_dependents;");
  __syncthreads();
  const bool dead = *abort_flag != 0;

  if (warp == NCW) {
    // ---------------------------------------------------------------- producer: one TMA box per lane
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    __syncwarp();
    const int nbox = BK / p.box;  // boxes of 64 columns along a tile's keys
    const int box = lane % nbox, half = (lane / nbox) % L::KBOX, is_v = lane / (nbox * L::KBOX);
    const bool mine = is_v < 2;
    const CUtensorMap* map = is_v == 1 ? &tmV : &tmK;
    const uint32_t dst0 = is_v * L::TILE + half * L::BOX + box * p.box * 128;
    int it = 0;
    bool ok = !dead;
    MetaPair meta;
    for (Segments<BK> g(p.bt, p.dv, sh); ok && !g.done(); g.next()) {
      meta.note(g);
      const int32_t* table = p.bt.table + g.b * p.bt.table_sb;
      for (int t = g.t0; t < g.t1; ++t, ++it) {
        const int st = it % L::NSTAGE;
        const uint32_t n = it / L::NSTAGE;
        const int key = t * BK + box * p.box;
        const bool load = mine && key < g.keys;
        int page = 0, slot = 0;
        if (load) {
          const int page_i = key / p.bt.ps;
          slot = key - page_i * p.bt.ps;
          page = table[page_i];
          if (page < 0 || page >= p.bt.num_pages) {
            report(CEA_DEV_BAD_PAGE);
            page = p.bt.num_pages;  // outside the tensor map: reads as zeros
          }
        }
        if (n > 0) ok = mbar_wait(empty_bar(st), (n - 1) & 1, abort_flag, CEA_DEV_TIMEOUT_DECODE);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int boxes = __popc(__ballot_sync(0xffffffffu, load));
        if (lane == 0) mbar_arrive_expect_tx(full_bar(st), boxes * p.box * 128);
        __syncwarp();
        if (load) tma_load_4d(sbase + st * L::STAGE + dst0, map, full_bar(st), half * 64, slot, g.hu, page);
      }
    }
    if (lane == 0) meta.store(p.meta);
    return;
  }

  // ------------------------------------------------------------------ consumers
  float* ms = reinterpret_cast<float*>(smem + L::OFF_MERGE);  // [NCW][16] max (log2 domain)
  float* ls = ms + NCW * ROWS;                                // [NCW][16] sum
  float* os = ls + NCW * ROWS;                                // [NCW][16][LDO]
  const int G = p.dv.group;
  const int rA = lane >> 2, rB = rA + 8;
  const uint16_t* qg = reinterpret_cast<const uint16_t*>(p.q);
  int it = 0;
  bool ok = !dead;
  for (Segments<BK> g(p.bt, p.dv, sh); ok && !g.done(); g.next()) {
    const int R = g.s.n * G;
    uint32_t qa[D / 16][4];
    {
      auto qrow = [&](int r) -> const uint16_t* {
        return r < R ? qg + (static_cast<int64_t>(g.s.row0) + r / G) * p.q_ss + (g.hu * G + r % G) * p.q_sh : nullptr;
      };
      const uint16_t *qA = qrow(rA), *qB = qrow(rB);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int d0 = kk * 16 + 2 * (lane & 3);
        qa[kk][0] = qA ? *reinterpret_cast<const uint32_t*>(qA + d0) : 0u;
        qa[kk][1] = qB ? *reinterpret_cast<const uint32_t*>(qB + d0) : 0u;
        qa[kk][2] = qA ? *reinterpret_cast<const uint32_t*>(qA + d0 + 8) : 0u;
        qa[kk][3] = qB ? *reinterpret_cast<const uint32_t*>(qB + d0 + 8) : 0u;
      }
    }
    // last key each row sees, -1 for none
    auto limit_of = [&](int r) -> int {
      if (r >= R) return -1;
      return p.dv.causal ? min(g.s.ctx + r / G, g.s.len - 1) : g.s.len - 1;
    };
    const int limA = limit_of(rA), limB = limit_of(rB);

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;

    for (int t = g.t0; t < g.t1; ++t, ++it) {
      const int st = it % L::NSTAGE;
      const bool got = mbar_wait(full_bar(st), (it / L::NSTAGE) & 1, abort_flag, CEA_DEV_TIMEOUT_DECODE);
      ok = __all_sync(0xffffffffu, got);
      if (!ok) break;
      const uint32_t kt = sbase + st * L::STAGE;
      const uint32_t vt = kt + L::TILE;
      const int key0 = warp * 16;        // this warp's keys within the tile
      const int left = g.keys - t * BK;  // keys of the unit in this tile
      if (left > key0) {                 // warp-uniform: else none of this warp's keys exists
        float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        {
          const int mi = lane >> 3, ri = lane & 7;
          const int key = key0 + ((mi >> 1) << 3) + ri;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4(swz(kt, key, 2 * kk + (mi & 1)), b0, b1, b2, b3);
            mma16816<kBF16>(s[0], qa[kk], b0, b1);
            mma16816<kBF16>(s[1], qa[kk], b2, b3);
          }
        }
        float tA = -INFINITY, tB = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = t * BK + key0 + nt * 8 + 2 * (lane & 3) + e;
            s[nt][e] = key <= limA ? s[nt][e] * p.scale_log2 : -INFINITY;
            s[nt][2 + e] = key <= limB ? s[nt][2 + e] * p.scale_log2 : -INFINITY;
            tA = fmaxf(tA, s[nt][e]);
            tB = fmaxf(tB, s[nt][2 + e]);
          }
        }
#pragma unroll
        for (int off = 1; off < 4; off <<= 1) {
          tA = fmaxf(tA, __shfl_xor_sync(0xffffffffu, tA, off));
          tB = fmaxf(tB, __shfl_xor_sync(0xffffffffu, tB, off));
        }
        const float nA = fmaxf(mA, tA), nB = fmaxf(mB, tB);
        const float uA = nA == -INFINITY ? 0.f : nA, uB = nB == -INFINITY ? 0.f : nB;
        const float aA = fast_exp2(mA - uA), aB = fast_exp2(mB - uB);
        mA = nA;
        mB = nB;
        uint32_t pa[4], pl[4];  // P = pa + pl
        {
          float pv[2][4];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            pv[nt][0] = fast_exp2(s[nt][0] - uA);
            pv[nt][1] = fast_exp2(s[nt][1] - uA);
            pv[nt][2] = fast_exp2(s[nt][2] - uB);
            pv[nt][3] = fast_exp2(s[nt][3] - uB);
          }
          lA = lA * aA + pv[0][0] + pv[0][1] + pv[1][0] + pv[1][1];
          lB = lB * aB + pv[0][2] + pv[0][3] + pv[1][2] + pv[1][3];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = pv[i >> 1][(i & 1) * 2], y = pv[i >> 1][(i & 1) * 2 + 1];
            pa[i] = pack2(x, y, kBF16);
            pl[i] = pack2(x - round16<kBF16>(x), y - round16<kBF16>(y), kBF16);
          }
        }
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= aA;
          o[i][1] *= aA;
          o[i][2] *= aB;
          o[i][3] *= aB;
        }
        // V fragment words hold keys 2 (lane & 3), + 1 of the first (b0, b2) or second (b1, b3) 8 keys
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (left < key0 + 16) {
          const int k0 = key0 + 2 * (lane & 3);
          keep0 = (k0 < left ? 0xffffu : 0u) | (k0 + 1 < left ? 0xffff0000u : 0u);
          keep1 = (k0 + 8 < left ? 0xffffu : 0u) | (k0 + 9 < left ? 0xffff0000u : 0u);
        }
        {
          const int mi = lane >> 3, ri = lane & 7;
          const int key = key0 + ((mi & 1) << 3) + ri;
#pragma unroll
          for (int dn = 0; dn < D / 8; dn += 2) {
            uint32_t b0, b1, b2, b3;
            ldsm_x4_t(swz(vt, key, dn + (mi >> 1)), b0, b1, b2, b3);
            b0 &= keep0;
            b1 &= keep1;
            b2 &= keep0;
            b3 &= keep1;
            mma16816<kBF16>(o[dn], pa, b0, b1);
            mma16816<kBF16>(o[dn + 1], pa, b2, b3);
            mma16816<kBF16>(o[dn], pl, b0, b1);
            mma16816<kBF16>(o[dn + 1], pl, b2, b3);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty_bar(st));
    }
    if (!ok) break;

    // ------------------------------------------------- join the four warps' results, in the order of the warps
    lA += __shfl_xor_sync(0xffffffffu, lA, 1);
    lA += __shfl_xor_sync(0xffffffffu, lA, 2);
    lB += __shfl_xor_sync(0xffffffffu, lB, 1);
    lB += __shfl_xor_sync(0xffffffffu, lB, 2);
    asm volatile("bar.sync 1, %0;" ::"n"(NCW * 32));  // the previous segment's reads of the scratch
    if ((lane & 3) == 0) {
      ms[warp * ROWS + rA] = mA;
      ms[warp * ROWS + rB] = mB;
      ls[warp * ROWS + rA] = lA;
      ls[warp * ROWS + rB] = lB;
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const int d = i * 8 + 2 * (lane & 3);
      *reinterpret_cast<float2*>(os + (warp * ROWS + rA) * L::LDO + d) = make_float2(o[i][0], o[i][1]);
      *reinterpret_cast<float2*>(os + (warp * ROWS + rB) * L::LDO + d) = make_float2(o[i][2], o[i][3]);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(NCW * 32));
    const int row = threadIdx.x >> 3, part = threadIdx.x & 7;
    if (row < R) {
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < NCW; ++w) mx = fmaxf(mx, ms[w * ROWS + row]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float wsum = 0.f, wt[NCW];
#pragma unroll
      for (int w = 0; w < NCW; ++w) {
        wt[w] = fast_exp2(ms[w * ROWS + row] - mu);
        wsum += wt[w] * ls[w * ROWS + row];
      }
      const float inv = wsum == 0.f ? 0.f : 1.f / wsum;
      const float lse = wsum == 0.f ? -INFINITY : (mu + log2f(wsum)) * kLn2;
      const int tok = row / G, head = g.hu * G + row % G;
      const int64_t trow = static_cast<int64_t>(g.s.row0) + tok;
      const int slot = segment_slot(g);
      float* po = p.part_o + (static_cast<int64_t>(slot) * ROWS + row) * D;
      const int64_t at = trow * p.o_ss + head * p.o_sh;
      for (int d = 2 * part; d < D; d += 16) {
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < NCW; ++w) {
          const float2 v = *reinterpret_cast<const float2*>(os + (w * ROWS + row) * L::LDO + d);
          x += wt[w] * v.x;
          y += wt[w] * v.y;
        }
        x *= inv;
        y *= inv;
        if (slot >= 0) {
          *reinterpret_cast<float2*>(po + d) = make_float2(x, y);
        } else if (p.out_dtype == CEA_F32) {
          reinterpret_cast<float*>(p.out)[at + d] = x;
          reinterpret_cast<float*>(p.out)[at + d + 1] = y;
        } else {
          const uint32_t w = pack2(x, y, kBF16);
          reinterpret_cast<uint16_t*>(p.out)[at + d] = static_cast<uint16_t>(w);
          reinterpret_cast<uint16_t*>(p.out)[at + d + 1] = static_cast<uint16_t>(w >> 16);
        }
      }
      if (part == 0) {
        if (slot >= 0) p.part_lse[static_cast<int64_t>(slot) * ROWS + row] = lse;
        else if (p.lse != nullptr) p.lse[head * p.l_sh + trow * p.l_ss] = lse;
      }
    }
  }
}

}  // namespace dec
}  // namespace paged
}  // namespace cea

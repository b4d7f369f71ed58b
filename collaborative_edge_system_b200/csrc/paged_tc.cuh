// Attention over a paged cache for chunks of new tokens (n_b * G > 16 query rows per KV head): tcgen05 products.
//
// Tensor-bound on long chunks.  One persistent CTA per SM takes an equal share of all key tiles of the batch
// (paged.cuh).  A unit is 2 x (128 / G) new tokens of one KV head: the G query heads of a group are packed with the
// tokens into the 128 rows of each of two MMA tiles ("halves"), so short chunks fill the rows and every K/V tile
// is read once for all heads that share it.  Q rows (token, head) come from one TMA box of (64, G, 128 / G).
//   warps 0-3 / 4-7   softmax and epilogue of half 0 / 1: one thread per query row (= TMEM lane)
//   warp 8 / 10       the K / V ring: 64-key tiles, one TMA box per page (or part of one), one box per lane
//   warp 9 / 11       MMA issuer of half 0 / 1, which also loads its half's Q
// Tiles of 64 keys leave room in tensor memory for two S buffers per half (2 x (2 x 64 + D) columns), so an issuer keeps
// S two tiles ahead of PV: S_h(c + 2) is pushed behind PV_h(c), whose P_h it overwrites, and a half's softmax finds the
// next scores waiting instead of standing in the chain S -> softmax -> PV.  (With tiles of 128 keys and one buffer, as in
// the dense prefill kernel, that chain set the pace.)  The tile numbers and rings run on across
// segments.  A new segment needs no drain: its Q_h is loaded once the last S_h of the old one is complete, during that
// tile's softmax; its first PV_h, which overwrites O_h, waits for a P_h that the softmax warps write after their
// epilogue has read O_h.
// A row sees keys 0 .. limit; only tiles that reach behind the first token's limit are masked, with one compare per key.
// Slots behind the unit's last key are not loaded or hold anything: their scores are masked, and their V rows are zeroed
// in shared memory before the tile is released to the MMA (a probability of 0 does not silence a NaN).  For the same reason
// the tiles that not all rows see whole are searched for infinities and NaN, which become zeros there and are added by
// the epilogue to the rows that see them, from the pages (a rare path; the search is one pass of the V producer over the
// last one to five tiles of a unit).
// P is rounded to the input type (the MMA's operand; half a step, 2^-8 for bf16 and 2^-11 for f16, independent per key; a
// second term, as the decode kernel has it, would double the PV products, and products bound this kernel), the sum is of
// the unrounded fp32 values; S, statistics and O are fp32.  f16 numbers below 2^-14 lose bits and those below
// 2^-25 are 0, so there P is 2^7 times the probability's ratio to its row's reference (at most 2^15 of 65504: the reference
// may be 2^8 below the maximum): a key counts down to 2^-32 of the largest.
// Measured (bf16, 32/8 heads of 128, pages of 16): 4096 new tokens on 36864, 2.27 to 2.30 ms a call among others, 1015 to
// 1030 TFLOP/s, with the clock pulled down by the power limit (1.99 ms, 1176 TFLOP/s, for a few calls in a captured graph);
// 512 on 8700, 75 us of GPU time, 940 TFLOP/s, 83 to 84 us a call.  A pair of
// 64-key tiles takes some 1600 cycles against 1280 of products and 1024 of exponentials.  Tried and slower: tiles of 128
// keys with one S buffer (91 us for the 512), one issuing warp for both halves, the halves' exponentials by turns,
// a quarter to a half of the exponentials by a polynomial on the multiply-add pipe, the row maximum computed between the
// exponentials of the same tile, three-operand maxima.
#pragma once

#include "attn_tc2.cuh"
#include "paged.cuh"

namespace cea {
namespace paged {
namespace tc {

using cea::tc2::umma_ts;

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int NUM_THREADS = 384;
constexpr int kKWarp = 8, kMmaWarp = 9, kVWarp = 10;  // warp 11: the second issuer
constexpr int kLaunchRegs = 168, kRegsSoftmax = 216, kRegsOther = 72;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsOther <= kLaunchRegs * NUM_THREADS, "register split");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kPCol = 32;  // P_h (pairs of 16 bit) within its S_h buffer
constexpr float kRescaleThreshold = 8.0f;
template <bool kBF16>
constexpr float kTopLog2 = kBF16 ? 0.f : 7.f;  // log2 of P at the row's reference
static_assert(kRescaleThreshold + kTopLog2<false> <= 15.f, "f16 ends at 65504");
static_assert(2 * BM == kWideRows, "rows of a slot");

template <int D>
struct Layout {
  static constexpr int KBOX = D / 64;
  static constexpr int QBOX = BM * 128;  // 64 columns of 128 query rows
  static constexpr int QTILE = KBOX * QBOX;
  static constexpr int BOX = BK * 128;   // 64 columns of 64 keys
  static constexpr int TILE = KBOX * BOX;
  static constexpr int KST = D == 128 ? 5 : 10;
  static constexpr int VST = D == 128 ? 5 : 10;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = OFF_Q + 2 * QTILE;
  static constexpr int OFF_V = OFF_K + KST * TILE;
  static constexpr int OFF_BAR = OFF_V + VST * TILE;
  static constexpr int B_QFULL = 0;  // x2 (per half)
  static constexpr int B_KFULL = B_QFULL + 2;
  static constexpr int B_KEMPTY = B_KFULL + KST;
  static constexpr int B_VFULL = B_KEMPTY + KST;
  static constexpr int B_VEMPTY = B_VFULL + VST;
  static constexpr int B_VTAIL = B_VEMPTY + VST;  // a V tile that is looked at before it counts as full
  // x4: [half][S buffer].  One barrier per buffer: each phase is met before its next one can begin, where a barrier for
  // both would run two phases ahead of a waiter.
  static constexpr int B_SFULL = B_VTAIL + 1;
  static constexpr int B_PFULL = B_SFULL + 4;
  static constexpr int B_PVDONE = B_PFULL + 4;
  static constexpr int B_DRAIN = B_PVDONE + 4;  // x2 (per half): all products are done
  static constexpr int B_QUEUE = B_DRAIN + 2;
  static constexpr int NBAR = B_QUEUE + SegQueue::kBars;
  static constexpr int OFF_QUEUE = (OFF_BAR + NBAR * 8 + 15) / 16 * 16;
  static constexpr int OFF_MISC = OFF_QUEUE + SegQueue::kBytes;
  static constexpr int BYTES = OFF_MISC + 16;
  static constexpr int SMEM_ALLOC = BYTES + 1024;
  static_assert(SMEM_ALLOC <= 232448, "shared memory");
};

struct Params {
  Batch bt;
  Division dv;  // tb = 2 * half
  int half;     // tokens of a half: 128 / G
  int box;      // slots of a TMA box: divides the page and the tile
  const uint16_t* v;
  int64_t v_sp, v_sh, v_ss;  // page, head, slot
  void* out;
  int64_t o_ss, o_sh;
  float* lse;
  int64_t l_sh, l_ss;
  float* part_o;
  float* part_lse;
  Meta* meta;
  int out_dtype;
  float scale_log2;
};

// One thread of a warp that runs in step.  The issuing warps keep in step and wrap only the tcgen05 instructions so:
// their operands are then uniform over the warp and stay in uniform registers.  With a loop of one thread's own
// (`lane == 0`) every product cost 75 to 90 cycles to issue, more than the 48 to 64 that it takes to run.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// The first tile of the unit that its rows do not all see whole (the first token sees the fewest keys).
__device__ __forceinline__ int first_parted(const Params& p, const Seg& g) {
  return max(0, p.dv.causal ? g.ctx + g.blk * p.dv.tb + 1 : g.len) / BK;
}

// Bounded wait of a whole warp (the contract of mbar_wait), short in code.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, volatile int* abort, int code) {
  uint64_t t0 = 0;
  for (uint32_t n = 1; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++n) {
    if ((n & 63u) != 0u) continue;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    const bool late = now - t0 > CEA_WAIT_LIMIT_NS;
    if (__any_sync(0xffffffffu, late || *abort != 0)) {
      if (late) record_error(code);
      *abort = 1;
      return false;
    }
  }
  return true;
}

template <int D, bool kBF16>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params p) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  volatile int* other_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 8);  // a value that is no finite number was met
  auto bar = [&](int i) -> uint32_t { return sbase + L::OFF_BAR + 8 * i; };
  const SegQueue queue{smem + L::OFF_QUEUE, bar(L::B_QUEUE), bar(L::B_QUEUE + kQueue), abort_flag,
                       CEA_DEV_TIMEOUT_PRODUCER};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int h = 0; h < 2; ++h) {
      mbar_init(bar(L::B_QFULL + h), 1);
      mbar_init(bar(L::B_DRAIN + h), 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(bar(L::B_SFULL + 2 * h + b), 1);
        mbar_init(bar(L::B_PFULL + 2 * h + b), 4);  // one arrival per softmax warp
        mbar_init(bar(L::B_PVDONE + 2 * h + b), 1);
      }
    }
    for (int s = 0; s < L::KST; ++s) {
      mbar_init(bar(L::B_KFULL + s), 1);
      mbar_init(bar(L::B_KEMPTY + s), 2);  // released by each half, with or without a product
    }
    for (int s = 0; s < L::VST; ++s) {
      mbar_init(bar(L::B_VFULL + s), 1);
      mbar_init(bar(L::B_VEMPTY + s), 2);
    }
    mbar_init(bar(L::B_VTAIL), 1);
    queue.init(8 + 3);  // the softmax warps, the V producer and the issuers
    *abort_flag = 0;
    *other_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  if (warp == kKWarp && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp >= kKWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == kKWarp || warp == kVWarp) {
      // ---------------------------------------------------------- TMA producers, one box per lane
      const bool is_k = warp == kKWarp;
      const CUtensorMap* map = is_k ? &tmK : &tmV;
      const int nst = is_k ? L::KST : L::VST;
      const uint32_t off = sbase + (is_k ? L::OFF_K : L::OFF_V);
      const int b_full = is_k ? L::B_KFULL : L::B_VFULL, b_empty = is_k ? L::B_KEMPTY : L::B_VEMPTY;
      const int nbox = BK / p.box;
      const int box = lane % nbox, col = lane / nbox;
      const bool mine = col < L::KBOX;
      uint32_t tails = 0;
      int loaded = 0;          // tiles whose full barrier completes by itself
      bool tail_open = false;  // a tail was loaded and not waited for
      auto load_tiles = [&](const Seg& g) -> bool {
        const int32_t* table = p.bt.table + g.b * p.bt.table_sb;
        const int parted = is_k ? INT32_MAX : first_parted(p, g);
        for (int t = g.t0; t < g.t1; ++t) {
          const int u = g.it + (t - g.t0);
          const int st = u % nst;
          const uint32_t n = u / nst;
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
          if (n > 0 && !wait_all(bar(b_empty + st), (n - 1) & 1, abort_flag, CEA_DEV_TIMEOUT_PRODUCER)) return false;
          const int boxes = __popc(__ballot_sync(0xffffffffu, load));
          const int left = g.keys - t * BK;
          const bool tail = t >= parted;  // a V tile that is looked at before it is released
          const uint32_t to = off + st * L::TILE;
          const uint32_t fb = tail ? bar(L::B_VTAIL) : bar(b_full + st);
          if (lane == 0) mbar_arrive_expect_tx(fb, boxes * p.box * 128);
          __syncwarp();
          if (load) tma_load_4d(to + col * L::BOX + box * p.box * 128, map, fb, col * 64, slot, g.hu, page);
          if (tail) {
            tail_open = true;
            if (!wait_all(bar(L::B_VTAIL), tails & 1, abort_flag, CEA_DEV_TIMEOUT_PRODUCER)) return false;
            ++tails;
            tail_open = false;
            uint8_t* tile = smem + L::OFF_V + st * L::TILE;
            for (int i = max(left, 0) * 8 + lane; i < BK * 8; i += 32)
#pragma unroll
              for (int c = 0; c < L::KBOX; ++c)
                *reinterpret_cast<uint4*>(tile + c * L::BOX + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            __syncwarp();
            uint32_t other[4] = {0u, 0u, 0u, 0u};
#pragma unroll 4
            for (int i = lane; i < BK * 8 * L::KBOX; i += 32) {
              const uint4 w = *reinterpret_cast<const uint4*>(tile + i * 16);
              note_other<kBF16>(w.x, other[0]);
              note_other<kBF16>(w.y, other[1]);
              note_other<kBF16>(w.z, other[2]);
              note_other<kBF16>(w.w, other[3]);
            }
            if ((other[0] | other[1] | other[2] | other[3]) != 0u) {  // among what this lane has read
              *other_flag = 1;
#pragma unroll 1
              for (int i = lane; i < BK * 8 * L::KBOX; i += 32) {
                uint4* at = reinterpret_cast<uint4*>(tile + i * 16);
                const uint4 w = *at;
                *at = make_uint4(finite_or_zero<kBF16>(w.x), finite_or_zero<kBF16>(w.y), finite_or_zero<kBF16>(w.z),
                                 finite_or_zero<kBF16>(w.w));
              }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(b_full + st));
          }
          loaded = u + 1;
        }
        return true;
      };
      int i = 0;
      if (is_k) {
        // this warp also walks the share, ahead of the others; after a device-side timeout nothing is computed
        const bool dead = *reinterpret_cast<volatile int*>(&g_cea_status) != 0;
        walk<BK, false>(p.bt, p.dv, dead, p.meta, [&](const Seg& g) -> bool {
          return queue.put(i++, g, lane) && (g.b < 0 || load_tiles(g));
        });
      } else {
        Seg g;
        while (queue.get(i++, g, lane))
          if (!load_tiles(g)) break;
      }
      for (int u = max(0, loaded - nst); u < loaded; ++u)
        drain(bar(b_full + u % nst), (u / nst) & 1, CEA_DEV_TIMEOUT_PRODUCER);
      if (tail_open) drain(bar(L::B_VTAIL), tails & 1, CEA_DEV_TIMEOUT_PRODUCER);
    } else {
      // ---------------------------------------------------------- MMA issuer of half h: one elected thread, the warp in step
      const int h = warp == kMmaWarp ? 0 : 1;
      constexpr uint32_t kIdescQK = idesc_f16(kBF16, false, BM, BK);
      constexpr uint32_t kIdescPV = idesc_f16(kBF16, true, BM, D);
      const uint32_t tS = __shfl_sync(0xffffffffu, tmem, 0) + 256 * h;  // two buffers of BK columns
      const uint32_t tO = tS + 128;
      const uint64_t qdesc = sw128_desc(sbase + L::OFF_Q + h * L::QTILE, 16, 1024);
      const uint64_t kdesc0 = sw128_desc(sbase + L::OFF_K, 16, 1024);
      const uint64_t vdesc0 = sw128_desc(sbase + L::OFF_V, L::BOX, 1024);
      const uint32_t b_s = bar(L::B_SFULL + 2 * h), b_p = bar(L::B_PFULL + 2 * h), b_pv = bar(L::B_PVDONE + 2 * h);
      const uint32_t b_q = bar(L::B_QFULL + h);
      int ks = 0, vs = 0;               // next stage of the K and V rings,
      uint32_t kph = 0, vph = 0;        // and its phase
      uint32_t sb = 0, sph = 0;         // next S buffer, and the phase that its S will complete
      uint32_t pb = 0, pph = 0;         // the same of P
      uint32_t qph = 0;
      uint32_t pending = 0;             // tiles whose PV is to come, two bits each, the oldest low: 1 computed, 2 first
      int npend = 0;
      bool any = false, ok = true;
      bool q_open = false;              // Q_h was loaded and not waited for
      auto issue_pv = [&]() -> bool {
        if (!wait_all(bar(L::B_VFULL) + 8 * vs, vph, abort_flag, CEA_DEV_TIMEOUT_MMA)) return false;
        if (pending & 1u) {
          if (!wait_all(b_p + 8 * pb, pph, abort_flag, CEA_DEV_TIMEOUT_MMA)) return false;
          tc_fence_after();
          const uint64_t vdesc = vdesc0 + static_cast<uint64_t>((vs * L::TILE) >> 4);
          const uint32_t tP = tS + BK * pb + kPCol;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
              umma_ts(tO, tP + kk * 8, vdesc + static_cast<uint64_t>((kk * 16 * 128) >> 4), kIdescPV,
                      (!(pending & 2u) || kk > 0) ? 1u : 0u);
            umma_commit(b_pv + 8 * pb);
            umma_commit(bar(L::B_VEMPTY) + 8 * vs);
          }
          __syncwarp();
          pph ^= pb;
          pb ^= 1u;
        } else if (elect_one()) {
          mbar_arrive(bar(L::B_VEMPTY) + 8 * vs);
        }
        vs = vs + 1 == L::VST ? 0 : vs + 1;
        vph ^= vs == 0 ? 1u : 0u;
        pending >>= 2;
        --npend;
        return true;
      };
      Seg g;
      for (int i = 0; ok && queue.get(i, g, lane); ++i) {
        const int tok = __shfl_sync(0xffffffffu, g.blk * p.dv.tb + h * p.half, 0);
        const bool act = h == 0 || tok < __shfl_sync(0xffffffffu, g.n, 0);
        const int t0 = __shfl_sync(0xffffffffu, g.t0, 0), t1 = __shfl_sync(0xffffffffu, g.t1, 0);
        if (act) {
          // Q_h is free once this half's last S is complete
          if (any && !wait_all(b_s + 8 * (sb ^ 1u), sph ^ (sb ^ 1u), abort_flag, CEA_DEV_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          if (elect_one()) {
            mbar_arrive_expect_tx(b_q, L::KBOX * 128 * p.half * p.dv.group);
#pragma unroll
            for (int kb = 0; kb < L::KBOX; ++kb)
              tma_load_4d(sbase + L::OFF_Q + h * L::QTILE + kb * L::QBOX, &tmQ, b_q, kb * 64, g.hu * p.dv.group,
                          g.row0 + tok, 0);
          }
          __syncwarp();
          q_open = true;
        }
        for (int t = t0; t < t1; ++t) {
          // S runs two tiles ahead of PV; S(c + 2) follows PV(c) in this thread's order, hence overwrites P(c) behind it
          if (npend == 2 && !(ok = issue_pv())) break;
          if (!(ok = wait_all(bar(L::B_KFULL) + 8 * ks, kph, abort_flag, CEA_DEV_TIMEOUT_MMA))) break;
          if (act) {
            if (t == t0) {
              if (!(ok = wait_all(b_q, qph, abort_flag, CEA_DEV_TIMEOUT_MMA))) break;
              qph ^= 1u;
              q_open = false;
            }
            tc_fence_after();
            const uint64_t kdesc = kdesc0 + static_cast<uint64_t>((ks * L::TILE) >> 4);
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                umma_ss(tS + BK * sb, qdesc + (((kk >> 2) * L::QBOX + (kk & 3) * 32) >> 4),
                        kdesc + (((kk >> 2) * L::BOX + (kk & 3) * 32) >> 4), kIdescQK, kk > 0 ? 1u : 0u);
              umma_commit(b_s + 8 * sb);
              umma_commit(bar(L::B_KEMPTY) + 8 * ks);
            }
            __syncwarp();
            sph ^= sb;
            sb ^= 1u;
            any = true;
          } else if (elect_one()) {
            mbar_arrive(bar(L::B_KEMPTY) + 8 * ks);
          }
          ks = ks + 1 == L::KST ? 0 : ks + 1;
          kph ^= ks == 0 ? 1u : 0u;
          pending |= ((act ? 1u : 0u) | (t == t0 ? 2u : 0u)) << (2 * npend);
          ++npend;
        }
      }
      while (ok && npend > 0) ok = issue_pv();
      if (q_open) drain(b_q, qph, CEA_DEV_TIMEOUT_MMA);
      if (elect_one()) umma_commit(bar(L::B_DRAIN + h));
      __syncwarp();
      drain(bar(L::B_DRAIN + h), 0, CEA_DEV_TIMEOUT_MMA);
    }
  } else {
    // ================================================================ softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int h = warp >> 2;
    const int row = threadIdx.x & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 256 * h + lane_base;
    const uint32_t tO = tmem + 256 * h + 128 + lane_base;
    const int G = p.dv.group;
    const int row_tok = row / G, row_head = row - row_tok * G;
    int it = 0;  // tiles this half computed
    bool ok = true;
    Seg g;
    for (int i = 0; ok && queue.get(i, g, lane); ++i) {
      const int tok0 = g.blk * p.dv.tb + h * p.half;
      if (tok0 >= g.n && h == 1) continue;
      const int tok = tok0 + row_tok;
      const bool row_in = row_tok < p.half && tok < g.n;
      const int seen = g.len - 1;
      const int limit = !row_in ? -1 : (p.dv.causal ? min(g.ctx + tok, seen) : seen);
      const int first_limit = p.dv.causal ? min(g.ctx + tok0, seen) : seen;  // of the half's first token
      float m = -INFINITY, l = 0.f;
      for (int t = g.t0; t < g.t1; ++t) {
        const int b = it & 1;
        if (!wait_all(bar(L::B_SFULL + 2 * h + b), (it >> 1) & 1, abort_flag, CEA_DEV_TIMEOUT_SOFTMAX)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[BK];
#pragma unroll
        for (int c = 0; c < BK / 32; ++c) tmem_ld32(tS + BK * b + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
        tmem_wait_ld();
        float mx[8];
#pragma unroll
        for (int a = 0; a < 8; ++a) mx[a] = -INFINITY;
        if (t * BK + BK - 1 > first_limit) {
          const int vis = limit - t * BK;  // keys 0 .. vis of the tile
#pragma unroll
          for (int j = 0; j < BK; ++j) {
            if (j > vis) s[j] = __float_as_uint(-INFINITY);
            mx[j & 7] = fmaxf(mx[j & 7], __uint_as_float(s[j]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < BK; ++j) mx[j & 7] = fmaxf(mx[j & 7], __uint_as_float(s[j]));
        }
        const float tmax =
            fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) *
            p.scale_log2;
        const float m_new = fmaxf(m, tmax);
        const bool rescale = (m != -INFINITY) && (m_new > m + kRescaleThreshold);
        float alpha = 1.f;
        if (m == -INFINITY) {
          m = m_new;
        } else if (rescale) {
          alpha = fast_exp2(m - m_new);
          l *= alpha;
          m = m_new;
        }
        const float neg_m = kTopLog2<kBF16> - (m == -INFINITY ? 0.f : m);
        if (__any_sync(0xffffffffu, rescale)) {  // not at a segment's first tile
          // S_h(it) complete means PV_h(it - 2) complete: the parity wait for PV_h(it - 1) is unambiguous
          if (!wait_all(bar(L::B_PVDONE + 2 * h + (b ^ 1)), ((it - 1) >> 1) & 1, abort_flag, CEA_DEV_TIMEOUT_SOFTMAX)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tO + c * 32, o);
          }
        }
        uint64_t rs2[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) rs2[a] = 0ull;
        const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
        const uint64_t negm2 = f2_pack(neg_m, neg_m);
        {
#pragma unroll
          for (int c = 0; c < BK / 32; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint64_t x = f2_fma(
                  f2_pack(__uint_as_float(s[c * 32 + 2 * e]), __uint_as_float(s[c * 32 + 2 * e + 1])), scale2, negm2);
              float p0, p1;
              f2_unpack(x, p0, p1);
              p0 = fast_exp2(p0);
              p1 = fast_exp2(p1);
              rs2[e & 3] = f2_add(rs2[e & 3], f2_pack(p0, p1));
              pk[e] = pack2(p0, p1, kBF16);
            }
            tmem_st16(tS + BK * b + kPCol + c * 16, pk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L::B_PFULL + 2 * h + b));
        {
          const uint64_t r = f2_add(f2_add(rs2[0], rs2[1]), f2_add(rs2[2], rs2[3]));
          float r0, r1;
          f2_unpack(r, r0, r1);
          l += r0 + r1;
        }
        ++it;
      }
      if (!ok) break;
      // ---------------------------------------------------------------- epilogue of the segment
      // S_h(it - 1) completed, hence PV_h(it - 3) did: the parity wait for PV_h(it - 1) is unambiguous
      ok = wait_all(bar(L::B_PVDONE + 2 * h + ((it - 1) & 1)), ((it - 1) >> 1) & 1, abort_flag, CEA_DEV_TIMEOUT_SOFTMAX);
      if (!ok) break;
      tc_fence_after();
      const float inv_l = l == 0.f ? 0.f : 1.f / l;
      const float lse_row = l == 0.f ? -INFINITY : (m + (log2f(l) - kTopLog2<kBF16>)) * kLn2;
      const int slot = g.slot;
      const int head = g.hu * G + row_head;
      const int64_t trow = static_cast<int64_t>(g.row0) + tok;
      const int64_t obase = trow * p.o_ss + head * p.o_sh;
      const int prow = h * p.half * G + row;  // of the slot: [D / 4][row][4]
      float4* part = reinterpret_cast<float4*>(p.part_o) + static_cast<int64_t>(slot) * (D / 4) * kWideRows + prow;
      // the flag was set before the tile was released, hence before the products that were waited for above
      if (__any_sync(0xffffffffu, *other_flag != 0)) {
        // the keys of searched tiles that this row sees
        const int from = max(g.t0, first_parted(p, g)) * BK, to = min(limit + 1, g.t1 * BK);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld32(tO + c, o);
          tmem_wait_ld();
#pragma unroll 1
          for (int key = from; key < to; ++key) {
            const int page_i = key / p.bt.ps, page = p.bt.table[g.b * p.bt.table_sb + page_i];
            if (page < 0 || page >= p.bt.num_pages) continue;
            const uint4* src = reinterpret_cast<const uint4*>(p.v + page * p.v_sp + g.hu * p.v_sh +
                                                              (key - page_i * p.bt.ps) * p.v_ss + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint4 w = src[e];
              const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t bad = x[k] ^ finite_or_zero<kBF16>(x[k]);
                float lo = __uint_as_float(o[e * 8 + 2 * k]), hi = __uint_as_float(o[e * 8 + 2 * k + 1]);
                if (bad & 0xffffu) lo += widen16<kBF16>(x[k] & 0xffffu);
                if (bad >> 16) hi += widen16<kBF16>(x[k] >> 16);
                o[e * 8 + 2 * k] = __float_as_uint(lo);
                o[e * 8 + 2 * k + 1] = __float_as_uint(hi);
              }
            }
          }
          __syncwarp();
          tmem_st32(tO + c, o);
        }
        tmem_wait_st();
      }
#pragma unroll 1
      for (int c = 0; c < D; c += 64) {
        uint32_t o[64];
        tmem_ld32(tO + c, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
        tmem_ld32(tO + c + 32, *reinterpret_cast<uint32_t(*)[32]>(&o[32]));
        tmem_wait_ld();
        if (row_in) {
#pragma unroll
          for (int e = 0; e < 64; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv_l);
          auto f = [&](int e) { return __uint_as_float(o[e]); };
          if (slot >= 0) {
#pragma unroll
            for (int e = 0; e < 64; e += 4)
              part[((c + e) / 4) * kWideRows] = make_float4(f(e), f(e + 1), f(e + 2), f(e + 3));
          } else if (p.out_dtype == CEA_F32) {
            float* dst = reinterpret_cast<float*>(p.out) + obase + c;
#pragma unroll
            for (int e = 0; e < 64; e += 4)
              *reinterpret_cast<float4*>(dst + e) = make_float4(f(e), f(e + 1), f(e + 2), f(e + 3));
          } else {
            uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + obase + c;
#pragma unroll
            for (int e = 0; e < 64; e += 8)
              *reinterpret_cast<uint4*>(dst + e) = make_uint4(
                  pack2(f(e), f(e + 1), kBF16), pack2(f(e + 2), f(e + 3), kBF16), pack2(f(e + 4), f(e + 5), kBF16),
                  pack2(f(e + 6), f(e + 7), kBF16));
          }
        }
        __syncwarp();  // the next tcgen05.ld is for all lanes of the warp together
      }
      tc_fence_before();
      if (row_in) {
        if (slot >= 0) p.part_lse[static_cast<int64_t>(slot) * kWideRows + prow] = lse_row;
        else if (p.lse != nullptr) p.lse[head * p.l_sh + trow * p.l_ss] = lse_row;
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace tc
}  // namespace paged
}  // namespace cea

// Attention over a paged cache on CUDA cores: fp32 and fp64, and 16-bit inputs whose head size, page size, strides or
// alignment the tensor-core kernels do not take.  Right for every case; the arithmetic is the accumulation type's
// throughout (probabilities are not rounded).
//
// A unit is up to 16 query rows (tokens x query heads of one KV head) against the keys of one sequence, in tiles of 32
// keys.  16 threads share two rows, r and r + 8: thread `sub` holds the scores of keys sub + 16 j and groups of 16-byte
// output columns sub + 16 c of both, so every 16-byte word of K and V that it reads from shared memory, which bounds the
// kernel, feeds two rows (one row a thread: 44 us at the size below; tiles of 64 keys, with half the CTAs on an SM: 41;
// this: 37, and 38 with the rows of a tile that they see different parts of taken one by one).  Rows are padded by 16
// bytes, which keeps the reads free of conflicts.  Online softmax: m' = max(m, max s),
// l' = l e^(m - m') + sum e^(s - m'), o' = o e^(m - m') + sum e^(s - m') v.
// Several threads fetch a key's K and V rows (one page lookup per tile and thread): by cp.async a tile ahead where the
// rows are aligned and need no conversion, else element by element.  The division of the work over the grid is
// paged.cuh's; several CTAs per SM hide one another's latencies.  Fetching element by element into one buffer, with
// scalar reads, took 97 us (fp32, 8 heads of 64, 4 sequences of up to 2048, up to 40 new tokens).
#pragma once

#include "paged.cuh"

namespace cea {
namespace paged {
namespace simt {

constexpr int BQ = 16, BK = 32, TPR = 16, NT = BQ / 2 * TPR;

template <typename A>
struct Params {
  Batch bt;
  Division dv;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_ss, q_sh;          // elements
  int64_t k_sp, k_sh, k_ss;    // page, head, slot
  int64_t v_sp, v_sh, v_ss;
  void* out;
  int64_t o_ss, o_sh;
  A* lse;
  int64_t l_sh, l_ss;
  A* part_o;
  A* part_lse;
  Meta* meta;
  int G, head_groups, D, out_dtype;
  int vec;  // K and V rows are 16-byte aligned and whole in 16-byte words
  double scale;
};

template <typename A, int DMAX>
struct Layout {
  static constexpr int VN = 16 / sizeof(A);        // elements of a 16-byte word
  static constexpr int LD = DMAX + VN;             // of a row in shared memory
  static constexpr int NST = sizeof(A) * DMAX > 1024 ? 1 : 2;  // fp64 rows of 256: one stage is 133 KB
  static constexpr int LP = BK + VN;
  static constexpr int ELEMS = BQ * LD + NST * 2 * BK * LD + BQ * LP;
  static constexpr size_t BYTES = sizeof(A) * ELEMS;
};

template <typename T> __device__ __forceinline__ double widen(T x, double) { return static_cast<double>(to_f32<T>(x)); }
template <> __device__ __forceinline__ double widen<double>(double x, double) { return x; }
template <typename T> __device__ __forceinline__ float widen(T x, float) { return to_f32<T>(x); }

template <typename A> struct Word;
template <> struct Word<float> {
  float4 w;
  __device__ __forceinline__ float operator[](int i) const { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
};
template <> struct Word<double> {
  double2 w;
  __device__ __forceinline__ double operator[](int i) const { return i == 0 ? w.x : w.y; }
};
template <typename A>
__device__ __forceinline__ Word<A> word(const A* p) { return *reinterpret_cast<const Word<A>*>(p); }

__device__ __forceinline__ void cp16(const void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

template <typename T, typename A, int DMAX>
__global__ void __launch_bounds__(NT) attn_kernel(const __grid_constant__ Params<A> p) {
  using L = Layout<A, DMAX>;
  constexpr int VN = L::VN, KPT = BK / TPR;
  constexpr int NC = (DMAX + VN * TPR - 1) / (VN * TPR);  // output words of a thread and row
  constexpr int FPK = NT / BK;                            // threads that fetch a key
  extern __shared__ __align__(16) uint8_t smem_raw[];
  A* qs = reinterpret_cast<A*>(smem_raw);
  A* kv = qs + BQ * L::LD;  // stages of K, then V
  A* ps = kv + L::NST * 2 * BK * L::LD;
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* kp = reinterpret_cast<const T*>(p.k);
  const T* vp = reinterpret_cast<const T*>(p.v);
  const int r0 = threadIdx.x / TPR, sub = threadIdx.x % TPR;  // rows r0 and r0 + 8
  const int words = (p.D + VN - 1) / VN;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  // columns behind D stay zero in every row
  for (int i = threadIdx.x; i < L::ELEMS; i += NT) qs[i] = 0;
  // after a device-side timeout nothing is computed (one thread asks, as all warps must agree)
  const bool dead = __syncthreads_or(threadIdx.x == 0 && *reinterpret_cast<volatile int*>(&g_cea_status) != 0);

  walk<BK, false>(p.bt, p.dv, dead, p.meta, [&](const Seg& g) -> bool {  // every warp alike
    if (g.b < 0) return true;
    const int kvh = g.hu / p.head_groups, g0 = (g.hu % p.head_groups) * p.dv.group;
    int64_t row[2];
    int head[2], limit[2];  // keys 0 .. limit are visible to the row
    bool in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = r0 + 8 * h, tok = g.blk * p.dv.tb + r / p.dv.group, gg = g0 + r % p.dv.group;
      in[h] = r < p.dv.tb * p.dv.group && tok < g.n && gg < p.G;
      head[h] = kvh * p.G + gg;
      row[h] = static_cast<int64_t>(g.row0) + tok;
      limit[h] = !in[h] ? -1 : (p.dv.causal ? min(g.ctx + tok, g.len - 1) : g.len - 1);
    }
    // keys 0 .. all_see are visible to both rows, or to the one that exists
    const int all_see = in[0] && in[1] ? min(limit[0], limit[1]) : max(limit[0], limit[1]);
    const bool busy = __any_sync(0xffffffffu, in[0] || in[1]);  // some row of the warp exists
    // keys of tile t into stage `st`; those behind the unit's last are zeros (their scores are masked)
    auto fetch = [&](int t, int st) {
      const int j = threadIdx.x / FPK, part = threadIdx.x % FPK, key = t * BK + j;
      A* ks = kv + st * 2 * BK * L::LD + j * L::LD;
      A* vs = ks + BK * L::LD;
      int page = -1, slot = 0;
      if (key < g.keys) {
        const int page_i = key / p.bt.ps;
        slot = key - page_i * p.bt.ps;
        page = p.bt.table[g.b * p.bt.table_sb + page_i];
        if (page < 0 || page >= p.bt.num_pages) {
          if (part == 0) report(CEA_DEV_BAD_PAGE);
          page = -1;  // read as zeros
        }
      }
      if (page < 0) {
        for (int d = part; d < p.D; d += FPK) ks[d] = vs[d] = 0;
        return;
      }
      const T* ksrc = kp + page * p.k_sp + kvh * p.k_sh + slot * p.k_ss;
      const T* vsrc = vp + page * p.v_sp + kvh * p.v_sh + slot * p.v_ss;
      if (sizeof(T) == sizeof(A) && p.vec) {
        for (int w = part; w < words; w += FPK) {
          cp16(ks + w * VN, ksrc + w * VN);
          cp16(vs + w * VN, vsrc + w * VN);
        }
      } else {
        for (int d = part; d < p.D; d += FPK) {
          ks[d] = widen(ksrc[d], A(0));
          vs[d] = widen(vsrc[d], A(0));
        }
      }
    };
    __syncthreads();  // the previous segment's reads of qs and of the stages
    if (L::NST == 2) {
      fetch(g.t0, g.t0 & 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (in[h])
        for (int d = sub; d < p.D; d += TPR)
          qs[(r0 + 8 * h) * L::LD + d] = widen(q[row[h] * p.q_ss + head[h] * p.q_sh + d], A(0));
    A m[2], l[2], o[2][NC][VN];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = -INFINITY;
      l[h] = 0;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < VN; ++e) o[h][c][e] = 0;
    }
    for (int t = g.t0; t < g.t1; ++t) {
      const int st = L::NST == 2 ? t & 1 : 0;
      if (L::NST == 1) {
        __syncthreads();  // the previous tile's reads
        fetch(t, 0);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();  // tile t is there, tile t - 1 is done with
      if (L::NST == 2 && t + 1 < g.t1) {
        fetch(t + 1, st ^ 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      if (!busy) continue;
      const A* ks = kv + st * 2 * BK * L::LD;
      const A* vs = ks + BK * L::LD;
      A s[2][KPT];
#pragma unroll
      for (int j = 0; j < KPT; ++j) s[0][j] = s[1][j] = 0;
#pragma unroll 2
      for (int w = 0; w < words; ++w) {
        const Word<A> x0 = word(qs + r0 * L::LD + w * VN), x1 = word(qs + (r0 + 8) * L::LD + w * VN);
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          const Word<A> y = word(ks + (sub + TPR * j) * L::LD + w * VN);
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            s[0][j] += x0[e] * y[e];
            s[1][j] += x1[e] * y[e];
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        A top = -INFINITY;
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          // a key behind the row's view does not count, whatever its product is
          s[h][j] = t * BK + sub + TPR * j <= limit[h] ? s[h][j] * static_cast<A>(p.scale) : A(-INFINITY);
          top = max(top, s[h][j]);
        }
#pragma unroll
        for (int x = 1; x < TPR; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
        const A m_new = max(m[h], top), ref = m_new == A(-INFINITY) ? A(0) : m_new;
        const A alpha = exp_of(m[h] - ref);
        A add = 0;
#pragma unroll
        for (int j = 0; j < KPT; ++j) {
          const A e = exp_of(s[h][j] - ref);
          add += e;
          ps[(r0 + 8 * h) * L::LP + sub + TPR * j] = e;
        }
        m[h] = m_new;
        l[h] = l[h] * alpha + add;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < VN; ++e) o[h][c][e] *= alpha;
      }
      __syncwarp();  // a row's 16 threads are of one warp
      if (min(t * BK + BK, g.keys) - 1 <= all_see) {  // slots behind the last key are zeros
#pragma unroll 2
        for (int j = 0; j < BK; j += VN) {
          const Word<A> e0 = word(ps + r0 * L::LP + j), e1 = word(ps + (r0 + 8) * L::LP + j);
#pragma unroll
          for (int i = 0; i < VN; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const int col = (sub + TPR * c) * VN;
              if (DMAX % (VN * TPR) != 0 && col >= DMAX) continue;  // fp32 rows of 32: 8 words for 16 threads
              const Word<A> y = word(vs + (j + i) * L::LD + col);
#pragma unroll
              for (int e = 0; e < VN; ++e) {
                o[0][c][e] += e0[i] * y[e];
                o[1][c][e] += e1[i] * y[e];
              }
            }
        }
      } else {
        // keys that only some rows see: a probability of 0 does not silence an infinity or a NaN, so each row ends at its
        // last key
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int end = min(BK, limit[h] - t * BK + 1);
#pragma unroll 1
          for (int j = 0; j < end; ++j) {
            const A w = ps[(r0 + 8 * h) * L::LP + j];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const int col = (sub + TPR * c) * VN;
              if (DMAX % (VN * TPR) != 0 && col >= DMAX) continue;
              const Word<A> y = word(vs + j * L::LD + col);
#pragma unroll
              for (int e = 0; e < VN; ++e) o[h][c][e] += w * y[e];
            }
          }
        }
      }
      __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = 1; x < TPR; x <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
      const A inv = l[h] == A(0) ? A(0) : A(1) / l[h];  // no visible key: zeros and -inf
      const A lse = l[h] == A(0) ? A(-INFINITY) : m[h] + log_of(l[h]);
      const int64_t at = row[h] * p.o_ss + head[h] * p.o_sh, part = static_cast<int64_t>(g.slot) * BQ + r0 + 8 * h;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const int d = (sub + TPR * c) * VN + e;
          if (d >= p.D) continue;
          if (g.slot >= 0) p.part_o[part * p.D + d] = o[h][c][e] * inv;
          else if (in[h]) store_out<A>(p.out, at + d, o[h][c][e] * inv, p.out_dtype);
        }
      if (sub == 0) {
        if (g.slot >= 0) p.part_lse[part] = lse;
        else if (in[h] && p.lse != nullptr) p.lse[head[h] * p.l_sh + row[h] * p.l_ss] = lse;
      }
    }
    return true;
  });
}

}  // namespace simt
}  // namespace paged
}  // namespace cea

// Attention over a paged cache on CUDA cores: fp32 and fp64, and 16-bit inputs whose head size, page size, strides or
// alignment the tensor-core kernels do not take.  Right for every case; the arithmetic is the accumulation type's
// throughout (probabilities are not rounded).
//
// A unit is up to 16 query rows (tokens x query heads of one KV head) against the keys of one sequence, in tiles of
// 32 keys: 8 threads per row, thread `sub` holds the scores of keys sub + 8 j and the output columns sub + 8 c.
// Online softmax: m' = max(m, max s), l' = l e^(m - m') + sum e^(s - m'), o' = o e^(m - m') + sum e^(s - m') v.
// The division of the work over the grid is paged.cuh's; several CTAs per SM hide the load latency of one another.
#pragma once

#include "paged.cuh"

namespace cea {
namespace paged {
namespace simt {

constexpr int BQ = 16, BK = 32, TPR = 8, NT = BQ * TPR;

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
  double scale;
};

template <typename A, int DMAX>
constexpr size_t smem_bytes() {
  return sizeof(A) * (BQ * (DMAX + 1) + 2 * BK * (DMAX + 1) + BQ * (BK + 1));
}

template <typename T> __device__ __forceinline__ double widen(T x, double) { return static_cast<double>(to_f32<T>(x)); }
template <> __device__ __forceinline__ double widen<double>(double x, double) { return x; }
template <typename T> __device__ __forceinline__ float widen(T x, float) { return to_f32<T>(x); }

template <typename T, typename A, int DMAX>
__global__ void __launch_bounds__(NT) attn_kernel(const Params<A> p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  constexpr int LD = DMAX + 1;
  A* qs = reinterpret_cast<A*>(smem_raw);
  A* ks = qs + BQ * LD;
  A* vs = ks + BK * LD;
  A* ps = vs + BK * LD;
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* kp = reinterpret_cast<const T*>(p.k);
  const T* vp = reinterpret_cast<const T*>(p.v);
  const int r = threadIdx.x / TPR, sub = threadIdx.x % TPR;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  walk<BK, false>(p.bt, p.dv, false, p.meta, [&](const Seg& g) -> bool {  // every warp alike
    if (g.b < 0) return true;
    const int kvh = g.hu / p.head_groups, g0 = (g.hu % p.head_groups) * p.dv.group;
    const int tok = g.blk * p.dv.tb + r / p.dv.group, gg = g0 + r % p.dv.group;
    const bool in = r < p.dv.tb * p.dv.group && tok < g.n && gg < p.G;
    const int head = kvh * p.G + gg;
    const int64_t row = static_cast<int64_t>(g.row0) + tok;
    // keys 0 .. limit are visible to this row
    const int64_t limit = !in ? -1 : (p.dv.causal ? min(int64_t(g.ctx) + tok, int64_t(g.len) - 1) : g.len - 1);
    __syncthreads();  // the previous segment's reads of qs
    if (in)
      for (int d = sub; d < p.D; d += TPR) qs[r * LD + d] = widen(q[row * p.q_ss + head * p.q_sh + d], A(0));
    A m = -INFINITY, l = 0, o[DMAX / TPR];
#pragma unroll
    for (int c = 0; c < DMAX / TPR; ++c) o[c] = 0;
    for (int t = g.t0; t < g.t1; ++t) {
      const int key0 = t * BK, nk = min(BK, g.keys - key0);
      __syncthreads();  // the previous tile's reads of ks and vs
      for (int i = threadIdx.x; i < BK * p.D; i += NT) {
        const int j = i / p.D, d = i - j * p.D;
        A kv = 0, vv = 0;
        if (j < nk) {
          const int key = key0 + j, page_i = key / p.bt.ps, slot = key - page_i * p.bt.ps;
          const int page = p.bt.table[g.b * p.bt.table_sb + page_i];
          if (page >= 0 && page < p.bt.num_pages) {
            kv = widen(kp[page * p.k_sp + kvh * p.k_sh + slot * p.k_ss + d], A(0));
            vv = widen(vp[page * p.v_sp + kvh * p.v_sh + slot * p.v_ss + d], A(0));
          } else if (d == 0) {
            report(CEA_DEV_BAD_PAGE);  // read as zeros
          }
        }
        ks[j * LD + d] = kv;
        vs[j * LD + d] = vv;
      }
      __syncthreads();
      A s[BK / TPR], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < BK / TPR; ++j) s[j] = 0;
      if (in)
        for (int d = 0; d < p.D; ++d) {
          const A x = qs[r * LD + d];
#pragma unroll
          for (int j = 0; j < BK / TPR; ++j) s[j] += x * ks[(sub + TPR * j) * LD + d];
        }
#pragma unroll
      for (int j = 0; j < BK / TPR; ++j) {
        // a key behind the sequence or the row's view does not count, whatever its product is
        s[j] = key0 + sub + TPR * j <= limit ? s[j] * static_cast<A>(p.scale) : A(-INFINITY);
        top = max(top, s[j]);
      }
#pragma unroll
      for (int o2 = 1; o2 < TPR; o2 <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o2));
      const A m_new = max(m, top), ref = m_new == A(-INFINITY) ? A(0) : m_new;
      const A alpha = exp_of(m - ref);
      A add = 0;
#pragma unroll
      for (int j = 0; j < BK / TPR; ++j) {
        const A e = exp_of(s[j] - ref);
        add += e;
        ps[r * (BK + 1) + sub + TPR * j] = e;
      }
      m = m_new;
      l = l * alpha + add;
      __syncwarp();  // a row's 8 threads are of one warp
#pragma unroll
      for (int c = 0; c < DMAX / TPR; ++c) o[c] *= alpha;
      for (int j = 0; j < BK; ++j) {
        const A e = ps[r * (BK + 1) + j];
#pragma unroll
        for (int c = 0; c < DMAX / TPR; ++c)
          if (sub + TPR * c < p.D) o[c] += e * vs[j * LD + sub + TPR * c];
      }
      __syncwarp();
    }
#pragma unroll
    for (int o2 = 1; o2 < TPR; o2 <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o2);
    const A inv = l == A(0) ? A(0) : A(1) / l;  // no visible key: zeros and -inf
    const A lse = l == A(0) ? A(-INFINITY) : m + log_of(l);
    const int slot = g.slot;
    if (slot < 0) {
      if (in) {
        const int64_t at = row * p.o_ss + head * p.o_sh;
#pragma unroll
        for (int c = 0; c < DMAX / TPR; ++c)
          if (sub + TPR * c < p.D) store_out<A>(p.out, at + sub + TPR * c, o[c] * inv, p.out_dtype);
        if (sub == 0 && p.lse != nullptr) p.lse[head * p.l_sh + row * p.l_ss] = lse;
      }
    } else {
      const int64_t at = static_cast<int64_t>(slot) * BQ + r;
#pragma unroll
      for (int c = 0; c < DMAX / TPR; ++c)
        if (sub + TPR * c < p.D) p.part_o[at * p.D + sub + TPR * c] = o[c] * inv;
      if (sub == 0) p.part_lse[at] = lse;
    }
    return true;
  });
}

}  // namespace simt
}  // namespace paged
}  // namespace cea

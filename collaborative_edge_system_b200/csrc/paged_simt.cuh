// Attention over a paged cache on CUDA cores: fp32 and fp64, and 16-bit inputs whose head size, page size, strides or
// alignment the tensor-core kernels do not take.  Right for every case; the arithmetic is the accumulation type's
// throughout (probabilities are not rounded).
//
// A unit is up to 16 query rows (tokens x query heads of one KV head) against the keys of one sequence, in tiles of
// 32 keys.  8 threads share a row: thread `sub` holds the scores of keys sub + 8 j and groups of 16-byte output
// columns sub + 8 c, so K, V and Q are read from shared memory in 16-byte words without conflicts (rows are padded by
// 16 bytes) and each word feeds 4 to 16 multiply-adds.  Online softmax: m' = max(m, max s),
// l' = l e^(m - m') + sum e^(s - m'), o' = o e^(m - m') + sum e^(s - m') v.
// 4 threads fetch a key's K and V rows (one page lookup per tile and thread): by cp.async a tile ahead where the rows
// are aligned and need no conversion, else element by element.  The division of the work over the grid is paged.cuh's;
// several CTAs per SM hide one another's latencies.  Fetching element by element into one buffer, with scalar reads,
// took 97 us where this takes the time in the table of the measurements (fp32, 4 sequences of up to 2048, 40 new tokens).
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
__global__ void __launch_bounds__(NT, sizeof(A) == 4 && DMAX <= 64 ? 4 : 1) attn_kernel(const __grid_constant__ Params<A> p) {
  using L = Layout<A, DMAX>;
  constexpr int VN = L::VN, NC = DMAX / (VN * TPR);  // output words of a thread
  extern __shared__ __align__(16) uint8_t smem_raw[];
  A* qs = reinterpret_cast<A*>(smem_raw);
  A* kv = qs + BQ * L::LD;  // stages of K, then V
  A* ps = kv + L::NST * 2 * BK * L::LD;
  const T* q = reinterpret_cast<const T*>(p.q);
  const T* kp = reinterpret_cast<const T*>(p.k);
  const T* vp = reinterpret_cast<const T*>(p.v);
  const int r = threadIdx.x / TPR, sub = threadIdx.x % TPR;
  const int words = (p.D + VN - 1) / VN;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  // columns behind D stay zero in every row
  for (int i = threadIdx.x; i < L::ELEMS; i += NT) qs[i] = 0;
  __syncthreads();

  walk<BK, false>(p.bt, p.dv, false, p.meta, [&](const Seg& g) -> bool {  // every warp alike
    if (g.b < 0) return true;
    const int kvh = g.hu / p.head_groups, g0 = (g.hu % p.head_groups) * p.dv.group;
    const int tok = g.blk * p.dv.tb + r / p.dv.group, gg = g0 + r % p.dv.group;
    const bool in = r < p.dv.tb * p.dv.group && tok < g.n && gg < p.G;
    const bool busy = __any_sync(0xffffffffu, in);  // some row of the warp exists
    const int head = kvh * p.G + gg;
    const int64_t row = static_cast<int64_t>(g.row0) + tok;
    // keys 0 .. limit are visible to this row
    const int limit = !in ? -1 : (p.dv.causal ? min(g.ctx + tok, g.len - 1) : g.len - 1);
    // keys of tile t into stage `st`; a key behind the unit's last keeps what is there (its score is masked, its V row
    // zeroed)
    auto fetch = [&](int t, int st) {
      const int j = threadIdx.x >> 2, part = threadIdx.x & 3, key = t * BK + j;
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
        for (int d = part; d < p.D; d += 4) ks[d] = vs[d] = 0;
        return;
      }
      const T* ksrc = kp + page * p.k_sp + kvh * p.k_sh + slot * p.k_ss;
      const T* vsrc = vp + page * p.v_sp + kvh * p.v_sh + slot * p.v_ss;
      if (sizeof(T) == sizeof(A) && p.vec) {
        for (int w = part; w < words; w += 4) {
          cp16(ks + w * VN, ksrc + w * VN);
          cp16(vs + w * VN, vsrc + w * VN);
        }
      } else {
        for (int d = part; d < p.D; d += 4) {
          ks[d] = widen(ksrc[d], A(0));
          vs[d] = widen(vsrc[d], A(0));
        }
      }
    };
    __syncthreads();  // the previous segment's reads of qs and of the stages
    if (in)
      for (int d = sub; d < p.D; d += TPR) qs[r * L::LD + d] = widen(q[row * p.q_ss + head * p.q_sh + d], A(0));
    if (L::NST == 2) {
      fetch(g.t0, g.t0 & 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    A m = -INFINITY, l = 0, o[NC][VN];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < VN; ++e) o[c][e] = 0;
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
      A s[BK / TPR], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < BK / TPR; ++j) s[j] = 0;
#pragma unroll 2
      for (int w = 0; w < words; ++w) {
        const Word<A> x = word(qs + r * L::LD + w * VN);
#pragma unroll
        for (int j = 0; j < BK / TPR; ++j) {
          const Word<A> y = word(ks + (sub + TPR * j) * L::LD + w * VN);
#pragma unroll
          for (int e = 0; e < VN; ++e) s[j] += x[e] * y[e];
        }
      }
#pragma unroll
      for (int j = 0; j < BK / TPR; ++j) {
        // a key behind the row's view does not count, whatever its product is
        s[j] = t * BK + sub + TPR * j <= limit ? s[j] * static_cast<A>(p.scale) : A(-INFINITY);
        top = max(top, s[j]);
      }
#pragma unroll
      for (int x = 1; x < TPR; x <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, x));
      const A m_new = max(m, top), ref = m_new == A(-INFINITY) ? A(0) : m_new;
      const A alpha = exp_of(m - ref);
      A add = 0;
#pragma unroll
      for (int j = 0; j < BK / TPR; ++j) {
        const A e = exp_of(s[j] - ref);
        add += e;
        ps[r * L::LP + sub + TPR * j] = e;
      }
      m = m_new;
      l = l * alpha + add;
      __syncwarp();  // a row's 8 threads are of one warp
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < VN; ++e) o[c][e] *= alpha;
#pragma unroll 2
      for (int j = 0; j < BK; j += VN) {
        const Word<A> e4 = word(ps + r * L::LP + j);
#pragma unroll
        for (int i = 0; i < VN; ++i)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const int col = (sub + TPR * c) * VN;
            const Word<A> y = word(vs + (j + i) * L::LD + col);
#pragma unroll
            for (int e = 0; e < VN; ++e) o[c][e] += e4[i] * y[e];
          }
      }
      __syncwarp();
    }
#pragma unroll
    for (int x = 1; x < TPR; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    const A inv = l == A(0) ? A(0) : A(1) / l;  // no visible key: zeros and -inf
    const A lse = l == A(0) ? A(-INFINITY) : m + log_of(l);
    const int64_t at = row * p.o_ss + head * p.o_sh, part = static_cast<int64_t>(g.slot) * BQ + r;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const int d = (sub + TPR * c) * VN + e;
        if (d >= p.D) continue;
        if (g.slot >= 0) p.part_o[part * p.D + d] = o[c][e] * inv;
        else if (in) store_out<A>(p.out, at + d, o[c][e] * inv, p.out_dtype);
      }
    if (sub == 0) {
      if (g.slot >= 0) p.part_lse[part] = lse;
      else if (in && p.lse != nullptr) p.lse[head * p.l_sh + row * p.l_ss] = lse;
    }
    return true;
  });
}

}  // namespace simt
}  // namespace paged
}  // namespace cea

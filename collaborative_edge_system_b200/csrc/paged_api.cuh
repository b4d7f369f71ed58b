// Entry points of the paged KV cache: argument checks, choice of kernels, launches.  Included by cea_api.cu, whose
// helpers it uses.
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <numeric>
#include <vector>

#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_simt.cuh"
#include "paged_tc.cuh"

namespace {

namespace pg = cea::paged;

int paged_sms();

enum PagedKernel { kPagedTc = 1, kPagedDecode = 2, kPagedSimt = 4 };

int paged_check_table(const char* what, int B, int T, int page_size, int num_pages, int max_pages, const void* off,
                      const void* lens, const void* table) {
  if (B < 0 || T < 0 || page_size < 1 || num_pages < 0 || max_pages < 0)
    return fail(CEA_ERR_INVALID, "%s: sizes B=%d T=%d page_size=%d num_pages=%d max_pages=%d", what, B, T, page_size,
                num_pages, max_pages);
  if (B > 0 && T > 0 && (off == nullptr || lens == nullptr || (table == nullptr && max_pages > 0)))
    return fail(CEA_ERR_INVALID, "%s: null offsets, lengths or page table", what);
  return CEA_OK;
}

int paged_validate(const cea_paged_attn_params* p) {
  const char* what = "cea_paged_attn";
  if (p == nullptr) return fail(CEA_ERR_INVALID, "%s: null params", what);
  if (int e = paged_check_table(what, p->B, p->T, p->page_size, p->num_pages, p->max_pages, p->q_offsets, p->seq_lens,
                                p->page_table))
    return e;
  if (p->Hq < 0 || p->Hkv < 1 || p->D < 1) return fail(CEA_ERR_INVALID, "%s: Hq=%d Hkv=%d D=%d", what, p->Hq, p->Hkv, p->D);
  if (p->Hq % p->Hkv != 0)
    return fail(CEA_ERR_INVALID, "%s: %d query heads cannot share %d KV heads evenly", what, p->Hq, p->Hkv);
  if (p->D > pg::kMaxD) return fail(CEA_ERR_UNSUPPORTED, "%s: head dim %d above %d", what, p->D, pg::kMaxD);
  const int in = p->in_dtype, out = p->out_dtype;
  if (in < CEA_F32 || in > CEA_F64) return fail(CEA_ERR_INVALID, "%s: unknown input dtype %d", what, in);
  if (!(in == CEA_F64 ? out == CEA_F64 : (out == CEA_F32 || out == in)))
    return fail(CEA_ERR_UNSUPPORTED, "%s: output dtype %d not available for input dtype %d", what, out, in);
  if (p->min_q_len < 0 || p->max_q_len < 0 || p->min_q_len > p->max_q_len)
    return fail(CEA_ERR_INVALID, "%s: new tokens per sequence between %d and %d", what, p->min_q_len, p->max_q_len);
  if (!std::isfinite(p->scale)) return fail(CEA_ERR_INVALID, "%s: scale is not a finite number", what);
  if (p->B > 0 && p->T > 0 && p->Hq > 0 && p->max_q_len > 0) {
    if (p->q == nullptr || p->out == nullptr) return fail(CEA_ERR_INVALID, "%s: null q or out", what);
    if (p->num_pages > 0 && (p->k_pages == nullptr || p->v_pages == nullptr))
      return fail(CEA_ERR_INVALID, "%s: null pages", what);
  }
  return CEA_OK;
}

// pages that TMA boxes of at least 8 slots can read: [num_pages, Hkv, page_size, D]
bool paged_tma_ok(const cea_paged_attn_params* p, const void* ptr, const int64_t* st) {
  if (!aligned16(ptr) || p->num_pages < 1) return false;
  for (int i = 0; i < 3; ++i) {
    if ((i == 0 && p->num_pages == 1) || (i == 1 && p->Hkv == 1)) continue;  // unused
    if (st[i] <= 0 || st[i] % 8 != 0 || st[i] * 2 >= (int64_t(1) << 40)) return false;
  }
  return true;
}

bool paged_tensor_ok(const cea_paged_attn_params* p) {
  if (p->in_dtype != CEA_BF16 && p->in_dtype != CEA_F16) return false;
  if ((p->D != 64 && p->D != 128) || p->page_size % 8 != 0) return false;
  return paged_tma_ok(p, p->k_pages, p->k_stride) && paged_tma_ok(p, p->v_pages, p->v_stride);
}

// the decode kernel reads query words of 4 bytes
bool paged_decode_ok(const cea_paged_attn_params* p) {
  return paged_tensor_ok(p) && p->Hq / p->Hkv <= pg::dec::ROWS && (reinterpret_cast<uintptr_t>(p->q) & 3u) == 0 &&
         ((p->q_stride[0] | p->q_stride[1]) & 1) == 0;
}

// the chunk kernel reads Q by TMA, stores 16-byte vectors of a row, and scales the scores' maximum (not the scores)
bool paged_tc_ok(const cea_paged_attn_params* p) {
  if (!paged_tensor_ok(p) || p->Hq / p->Hkv > pg::tc::BM || !(static_cast<float>(p->scale) > 0.f)) return false;
  if (!aligned16(p->q) || !aligned16(p->out)) return false;
  const int vec = p->out_dtype == CEA_F32 ? 4 : 8;
  const int size[2] = {p->T, p->Hq};
  for (int i = 0; i < 2; ++i) {
    if (size[i] == 1) continue;
    if (p->q_stride[i] <= 0 || p->q_stride[i] % 8 != 0 || p->q_stride[i] * 2 >= (int64_t(1) << 40)) return false;
    if (p->o_stride[i] % vec != 0) return false;
  }
  return true;
}

// Which kernels serve a call.  Sequences of up to `few` new tokens go through the decode kernel, which is compiled for 8
// or 16 query rows per KV head; the others through the chunk kernel.  A kernel is launched only if the promised
// numbers of new tokens allow a sequence for it.  Times in us, bf16, 32 query and 8 KV heads where nothing else is said.
// - 9 to 16 rows at D = 128, if no sequence of the call can have fewer: the chunk kernel, which pads them to a tile that
//   the tensor cores take in their stride, while the 16-row form holds twice the accumulators.  Chunk kernel and 16-row
//   form: 36 and 41 (8 sequences of 4096, 4 tokens each), 103 and 106 (32 of them), 40 and 57 (64 of 300 to 600),
//   36 and 41 (32 of 4096, one token, groups of 16), 15 and 17 (one of those).
// - 9 to 16 rows at D = 64: the 16-row form, 76 against 85 (32 of 4096, 4 tokens), 29.5 against 30.4 (groups of 16).
// - up to 16 rows, some of them perhaps 8 or fewer: the 16-row form alone, 35 against 44 and 87 against 97 for the 8-row
//   form with the chunk kernel after it (8 and 32 of 2000 to 4096, 1 to 4 tokens).
// - where longer chunks come too: the 8-row form, and sequences of 9 to 16 rows join the chunks; the 16-row form costs
//   every single token of the batch: 101 against 108 (18 single tokens and two chunks of 389, up to 6000 keys).
// - up to 8 rows: the 8-row form, 44 against 56 for the 16-row form (64 of 600 to 900, one token).
struct PagedChoice {
  int kernels;
  int rows;  // query rows of the decode kernel: 8 or 16
  int few;   // tokens those hold
};

PagedChoice paged_choice(const cea_paged_attn_params* p) {
  PagedChoice c = {0, 8, 0};
  if (p->B == 0 || p->T == 0 || p->Hq == 0 || p->max_q_len == 0) return c;
  const int64_t G = p->Hq / p->Hkv, most = p->max_q_len * G;
  const bool wide = p->D == 128 && std::max(p->min_q_len, 1) * G > 8 && paged_tc_ok(p);
  c.rows = most <= 8 || (most > pg::dec::ROWS && G <= 8) || wide ? 8 : pg::dec::ROWS;
  c.few = static_cast<int>(c.rows / G);
  const bool few = std::max(p->min_q_len, 1) <= c.few, many = p->max_q_len > c.few;
  if ((!few || paged_decode_ok(p)) && (!many || paged_tc_ok(p)))
    c.kernels = (few ? kPagedDecode : 0) | (many ? kPagedTc : 0);
  else
    c.kernels = kPagedSimt;
  return c;
}

int paged_kernels(const cea_paged_attn_params* p) { return paged_choice(p).kernels; }

struct PagedPlan {
  int grid, rows;       // CTAs, rows of a slot
  size_t o, lse, meta, bytes;  // offsets into the workspace
};

PagedPlan paged_plan(int grid, int rows, int D, size_t elem, size_t at) {
  PagedPlan pl;
  pl.grid = grid;
  pl.rows = rows;
  pl.o = at;
  pl.lse = pl.o + align256(elem * 2 * grid * rows * D);
  pl.meta = pl.lse + align256(elem * 2 * grid * rows);
  pl.bytes = pl.meta + align256(sizeof(pg::Meta) * grid);
  return pl;
}

// CTAs of the CUDA-core kernel: as many as fit an SM's shared memory and registers (at 128 a thread); one more per SM
// is a second wave (59 us instead of 44 us at the size in paged_simt.cuh)
template <typename A, int DMAX>
int paged_simt_per_sm() {
  return static_cast<int>(std::max<size_t>(1, std::min<size_t>(4, 227 * 1024 / (pg::simt::Layout<A, DMAX>::BYTES + 1024))));
}

int paged_simt_grid(const cea_paged_attn_params* p) {
  const bool d = p->in_dtype == CEA_F64;
  const int n = p->D <= 32    ? (d ? paged_simt_per_sm<double, 32>() : paged_simt_per_sm<float, 32>())
                : p->D <= 64  ? (d ? paged_simt_per_sm<double, 64>() : paged_simt_per_sm<float, 64>())
                : p->D <= 128 ? (d ? paged_simt_per_sm<double, 128>() : paged_simt_per_sm<float, 128>())
                              : (d ? paged_simt_per_sm<double, 256>() : paged_simt_per_sm<float, 256>());
  return paged_sms() * n;
}

PagedPlan paged_simt_plan(const cea_paged_attn_params* p, size_t at) {
  return paged_plan(paged_simt_grid(p), pg::simt::BQ, p->D, p->in_dtype == CEA_F64 ? 8 : 4, at);
}

PagedPlan paged_decode_plan(const cea_paged_attn_params* p, size_t at) {
  return paged_plan(paged_sms(), pg::dec::ROWS, p->D, 4, at);
}

PagedPlan paged_tc_plan(const cea_paged_attn_params* p, size_t at) {
  return paged_plan(paged_sms(), 2 * pg::tc::BM, p->D, 4, at);
}

pg::Batch paged_batch(const cea_paged_attn_params* p) {
  return pg::Batch{p->q_offsets, p->seq_lens, p->page_table, p->table_stride, p->B, p->T, p->max_pages, p->num_pages,
                   p->page_size};
}

// SMs of the current device, asked for once per device
int paged_sms() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return num_sms();
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    n = num_sms();
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// a launch whose start may overlap the end of the kernel before it on the stream (it waits for it on the device)
template <typename K, typename... Args>
cudaError_t launch_dependent(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename A>
pg::CombineArgs<A> combine_args(const cea_paged_attn_params* p, const pg::Division& dv, const PagedPlan& pl,
                                int head_groups) {
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  pg::CombineArgs<A> c;
  c.dv = dv;
  c.part_o = reinterpret_cast<const A*>(ws + pl.o);
  c.part_lse = reinterpret_cast<const A*>(ws + pl.lse);
  c.meta = reinterpret_cast<const pg::Meta*>(ws + pl.meta);
  c.rows = pl.rows;
  c.out = p->out;
  c.o_ss = p->o_stride[0];
  c.o_sh = p->o_stride[1];
  c.lse = static_cast<A*>(p->lse);
  c.l_sh = p->lse_stride[0];
  c.l_ss = p->lse_stride[1];
  c.D = p->D;
  c.out_dtype = p->out_dtype;
  c.heads_per_kv = p->Hq / p->Hkv;
  c.head_groups = head_groups;
  return c;
}

// rows of the largest unit: none has more than a sequence of the batch
int unit_rows(const cea_paged_attn_params* p, const pg::Division& dv) {
  return static_cast<int>(std::min<int64_t>(dv.tb, p->max_q_len) * dv.group);
}

template <typename A, int RPB>
int launch_combine(const cea_paged_attn_params* p, const pg::Division& dv, const PagedPlan& pl, int head_groups,
                   cudaStream_t s) {
  const cudaError_t e =
      launch_dependent(pg::combine_kernel<A, RPB>, dim3(pl.grid, (unit_rows(p, dv) + RPB - 1) / RPB),
                       pg::kCombineThreads, 0, s, combine_args<A>(p, dv, pl, head_groups));
  return e == cudaSuccess ? CEA_OK : fail(CEA_ERR_CUDA, "combine_kernel: %s", cudaGetErrorString(e));
}

int launch_combine_wide(const cea_paged_attn_params* p, const pg::Division& dv, const PagedPlan& pl, cudaStream_t s) {
  const cudaError_t e =
      launch_dependent(p->D == 128 ? pg::combine_wide_kernel<128> : pg::combine_wide_kernel<64>,
                       dim3(pl.grid, (unit_rows(p, dv) + 31) / 32), pg::kCombineThreads, 0, s,
                       combine_args<float>(p, dv, pl, 1));
  return e == cudaSuccess ? CEA_OK : fail(CEA_ERR_CUDA, "combine_wide_kernel: %s", cudaGetErrorString(e));
}

template <typename T, typename A, int DMAX>
int launch_paged_simt(const cea_paged_attn_params* p, const PagedPlan& pl, cudaStream_t s) {
  const int G = p->Hq / p->Hkv;
  const int group = std::min(G, pg::simt::BQ), groups = (G + group - 1) / group;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  pg::simt::Params<A> a;
  a.bt = paged_batch(p);
  a.dv = pg::Division{p->B, p->Hkv * groups, pg::simt::BQ / group, group, INT64_MAX, 0, p->min_q_len, p->max_q_len, p->causal ? 1 : 0, 16,
                      5};
  a.q = p->q;
  a.k = p->k_pages;
  a.v = p->v_pages;
  a.q_ss = p->q_stride[0];
  a.q_sh = p->q_stride[1];
  a.k_sp = p->k_stride[0];
  a.k_sh = p->k_stride[1];
  a.k_ss = p->k_stride[2];
  a.v_sp = p->v_stride[0];
  a.v_sh = p->v_stride[1];
  a.v_ss = p->v_stride[2];
  a.out = p->out;
  a.o_ss = p->o_stride[0];
  a.o_sh = p->o_stride[1];
  a.lse = static_cast<A*>(p->lse);
  a.l_sh = p->lse_stride[0];
  a.l_ss = p->lse_stride[1];
  a.part_o = reinterpret_cast<A*>(ws + pl.o);
  a.part_lse = reinterpret_cast<A*>(ws + pl.lse);
  a.meta = reinterpret_cast<pg::Meta*>(ws + pl.meta);
  a.G = G;
  a.head_groups = groups;
  a.D = p->D;
  a.out_dtype = p->out_dtype;
  a.scale = p->scale;
  auto k = pg::simt::attn_kernel<T, A, DMAX>;
  constexpr size_t bytes = pg::simt::Layout<A, DMAX>::BYTES;
  const int size = elem_bytes(p->in_dtype);
  bool vec = aligned16(p->k_pages) && aligned16(p->v_pages) && p->D * size % 16 == 0;
  for (int i = 0; i < 3; ++i) vec = vec && p->k_stride[i] * size % 16 == 0 && p->v_stride[i] * size % 16 == 0;
  a.vec = vec;
  allow_smem(k, static_cast<int>(bytes));
  if (const cudaError_t e = launch_dependent(k, dim3(pl.grid), pg::simt::NT, bytes, s, a))
    return fail(CEA_ERR_CUDA, "paged attn_kernel: %s", cudaGetErrorString(e));
  return launch_combine<A, 8>(p, a.dv, pl, groups, s);
}

template <typename T, typename A>
int launch_paged_simt_d(const cea_paged_attn_params* p, const PagedPlan& pl, cudaStream_t s) {
  if (p->D <= 32) return launch_paged_simt<T, A, 32>(p, pl, s);
  if (p->D <= 64) return launch_paged_simt<T, A, 64>(p, pl, s);
  if (p->D <= 128) return launch_paged_simt<T, A, 128>(p, pl, s);
  return launch_paged_simt<T, A, 256>(p, pl, s);
}

// pages [num_pages, Hkv, page_size, D] as a 4-D tensor map (D, slot, head, page) with (64, rows, 1, 1) boxes
bool paged_map(CUtensorMap* map, const cea_paged_attn_params* p, const void* ptr, const int64_t* st, int rows) {
  return make_map(map, p->in_dtype, ptr, p->D, p->page_size, p->Hkv, p->num_pages, st[2], st[1], st[0], rows);
}

int launch_paged_decode(const cea_paged_attn_params* p, const PagedPlan& pl, cudaStream_t s) {
  const int G = p->Hq / p->Hkv;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  pg::dec::Params a;
  a.bt = paged_batch(p);
  const PagedChoice choice = paged_choice(p);
  a.dv = pg::Division{p->B, p->Hkv, choice.few, G, choice.rows, 0, p->min_q_len, p->max_q_len,
                      p->causal ? 1 : 0, 192, 7};
  a.q = p->q;
  a.q_ss = p->q_stride[0];
  a.q_sh = p->q_stride[1];
  a.out = p->out;
  a.o_ss = p->o_stride[0];
  a.o_sh = p->o_stride[1];
  a.lse = static_cast<float*>(p->lse);
  a.l_sh = p->lse_stride[0];
  a.l_ss = p->lse_stride[1];
  a.part_o = reinterpret_cast<float*>(ws + pl.o);
  a.part_lse = reinterpret_cast<float*>(ws + pl.lse);
  a.meta = reinterpret_cast<pg::Meta*>(ws + pl.meta);
  a.box = std::gcd(p->page_size, pg::dec::BK);
  a.out_dtype = p->out_dtype;
  a.scale_log2 = static_cast<float>(p->scale * 1.4426950408889634);
  CUtensorMap mk, mv;
  if (!paged_map(&mk, p, p->k_pages, p->k_stride, a.box) || !paged_map(&mv, p, p->v_pages, p->v_stride, a.box))
    return fail(CEA_ERR_CUDA, "cuTensorMapEncodeTiled failed for the pages");
  cudaError_t err = cudaSuccess;
#define CEA_PDEC(DD, BF)                                                                  \
  do {                                                                                    \
    auto k = choice.rows == 8 ? pg::dec::decode_kernel<DD, BF, 1> : pg::dec::decode_kernel<DD, BF, 2>; \
    allow_smem(k, pg::dec::Layout<DD>::SMEM_ALLOC);                                       \
    err = launch_dependent(k, dim3(pl.grid), pg::dec::NTHREADS, pg::dec::Layout<DD>::SMEM_ALLOC, s, mk, mv, a); \
  } while (0)
  const bool bf = p->in_dtype == CEA_BF16;
  if (p->D == 128) {
    if (bf) CEA_PDEC(128, true); else CEA_PDEC(128, false);
  } else {
    if (bf) CEA_PDEC(64, true); else CEA_PDEC(64, false);
  }
#undef CEA_PDEC
  if (err != cudaSuccess) return fail(CEA_ERR_CUDA, "paged decode_kernel: %s", cudaGetErrorString(err));
  return launch_combine<float, 1>(p, a.dv, pl, 1, s);
}

// q [T, Hq, D] as a tensor map (D, head, token) with boxes of `tokens` x G heads x 64 columns
bool paged_q_map(CUtensorMap* map, const cea_paged_attn_params* p, int G, int tokens) {
  EncodeTiledFn enc = encode_fn();
  if (enc == nullptr) return false;
  // the stride of a dimension of size 1 is never used: give it a legal value
  const int64_t sh = p->Hq == 1 ? p->D : p->q_stride[1], ss = p->T == 1 ? p->D * int64_t(p->Hq) : p->q_stride[0];
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p->D), static_cast<cuuint64_t>(p->Hq),
                              static_cast<cuuint64_t>(p->T), 1};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(ss) * 2,
                                 static_cast<cuuint64_t>(ss) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(G), static_cast<cuuint32_t>(tokens), 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t =
      p->in_dtype == CEA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, t, 4, const_cast<void*>(p->q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_paged_tc(const cea_paged_attn_params* p, const PagedPlan& pl, cudaStream_t s) {
  const int G = p->Hq / p->Hkv;
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  pg::tc::Params a;
  a.bt = paged_batch(p);
  a.half = pg::tc::BM / G;
  a.dv = pg::Division{p->B, p->Hkv, 2 * a.half, G, INT64_MAX, int64_t(paged_choice(p).few) * G + 1,
                      p->min_q_len, p->max_q_len, p->causal ? 1 : 0, 384, 8};
  a.box = std::gcd(p->page_size, pg::tc::BK);
  a.v = static_cast<const uint16_t*>(p->v_pages);
  a.v_sp = p->v_stride[0];
  a.v_sh = p->v_stride[1];
  a.v_ss = p->v_stride[2];
  a.out = p->out;
  a.o_ss = p->o_stride[0];
  a.o_sh = p->o_stride[1];
  a.lse = static_cast<float*>(p->lse);
  a.l_sh = p->lse_stride[0];
  a.l_ss = p->lse_stride[1];
  a.part_o = reinterpret_cast<float*>(ws + pl.o);
  a.part_lse = reinterpret_cast<float*>(ws + pl.lse);
  a.meta = reinterpret_cast<pg::Meta*>(ws + pl.meta);
  a.out_dtype = p->out_dtype;
  a.scale_log2 = static_cast<float>(p->scale * 1.4426950408889634);
  CUtensorMap mq, mk, mv;
  if (!paged_q_map(&mq, p, G, a.half) || !paged_map(&mk, p, p->k_pages, p->k_stride, a.box) ||
      !paged_map(&mv, p, p->v_pages, p->v_stride, a.box))
    return fail(CEA_ERR_CUDA, "cuTensorMapEncodeTiled failed for the queries or the pages");
  cudaError_t err = cudaSuccess;
#define CEA_PTC(DD, BF)                                                                               \
  do {                                                                                                \
    auto k = pg::tc::chunk_kernel<DD, BF>;                                                            \
    if (int e = check_launch_regs(reinterpret_cast<const void*>(k), pg::tc::kLaunchRegs)) return e;   \
    allow_smem(k, pg::tc::Layout<DD>::SMEM_ALLOC);                                                    \
    err = launch_dependent(k, dim3(pl.grid), pg::tc::NUM_THREADS, pg::tc::Layout<DD>::SMEM_ALLOC, s, mq, mk, mv, a); \
  } while (0)
  const bool bf = p->in_dtype == CEA_BF16;
  if (p->D == 128) {
    if (bf) CEA_PTC(128, true); else CEA_PTC(128, false);
  } else {
    if (bf) CEA_PTC(64, true); else CEA_PTC(64, false);
  }
#undef CEA_PTC
  if (err != cudaSuccess) return fail(CEA_ERR_CUDA, "paged chunk_kernel: %s", cudaGetErrorString(err));
  return launch_combine_wide(p, a.dv, pl, s);
}

size_t paged_workspace(const cea_paged_attn_params* p, int kernels) {
  size_t n = 0;
  if (kernels & kPagedDecode) n = paged_decode_plan(p, n).bytes;
  if (kernels & kPagedTc) n = paged_tc_plan(p, n).bytes;
  if (kernels & kPagedSimt) n = paged_simt_plan(p, n).bytes;
  return n;
}

template <typename U>
cudaError_t launch_append(const pg::AppendArgs& a, cudaStream_t s) {
  constexpr int per = pg::kAppendThreads / 32;
  // and a block that checks the offsets
  const int grid = static_cast<int>(std::min<int64_t>((static_cast<int64_t>(a.bt.T) + per - 1) / per, 148 * 16)) + 1;
  return launch_dependent(pg::append_kernel<U>, dim3(grid), pg::kAppendThreads, 0, s, a);
}

}  // namespace

extern "C" {

int cea_paged_attn_kernels(const cea_paged_attn_params* p) {
  if (paged_validate(p) != CEA_OK) return -1;
  return paged_kernels(p);
}

size_t cea_paged_attn_workspace_size(const cea_paged_attn_params* p) {
  if (paged_validate(p) != CEA_OK) return 0;
  return paged_workspace(p, paged_kernels(p));
}

int cea_paged_attn(const cea_paged_attn_params* p, void* stream) {
  if (int e = paged_validate(p)) return e;
  const int kernels = paged_kernels(p);
  if (kernels == 0) return CEA_OK;
  const size_t need = paged_workspace(p, kernels);
  if (p->workspace == nullptr || p->workspace_bytes < need || !aligned16(p->workspace))
    return fail(CEA_ERR_WORKSPACE, "paged attention needs %zu 16-byte aligned workspace bytes, got %zu", need,
                p->workspace_bytes);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  size_t at = 0;
  if (kernels & kPagedDecode) {
    const PagedPlan pl = paged_decode_plan(p, at);
    if (int e = launch_paged_decode(p, pl, s)) return e;
    at = pl.bytes;
  }
  if (kernels & kPagedTc) {
    const PagedPlan pl = paged_tc_plan(p, at);
    if (int e = launch_paged_tc(p, pl, s)) return e;
    at = pl.bytes;
  }
  if (kernels & kPagedSimt) {
    const PagedPlan pl = paged_simt_plan(p, at);
    switch (p->in_dtype) {
      case CEA_F64: return launch_paged_simt_d<double, double>(p, pl, s);
      case CEA_F32: return launch_paged_simt_d<float, float>(p, pl, s);
      case CEA_BF16: return launch_paged_simt_d<__nv_bfloat16, float>(p, pl, s);
      default: return launch_paged_simt_d<__half, float>(p, pl, s);
    }
  }
  return CEA_OK;
}

int cea_paged_append(const cea_paged_append_params* p, void* stream) {
  const char* what = "cea_paged_append";
  if (p == nullptr) return fail(CEA_ERR_INVALID, "%s: null params", what);
  if (int e = paged_check_table(what, p->B, p->T, p->page_size, p->num_pages, p->max_pages, p->q_offsets, p->seq_lens,
                                p->page_table))
    return e;
  if (p->H < 1 || p->D < 1) return fail(CEA_ERR_INVALID, "%s: heads and head dim must be >= 1", what);
  const int eb = p->elem_bytes;
  if (eb != 1 && eb != 2 && eb != 4 && eb != 8) return fail(CEA_ERR_INVALID, "%s: element size %d", what, eb);
  if (p->B == 0 || p->T == 0) return CEA_OK;
  if (!p->k || !p->v || !p->k_pages || !p->v_pages) return fail(CEA_ERR_INVALID, "%s: null k, v or pages", what);
  pg::AppendArgs a{};
  a.bt = pg::Batch{p->q_offsets, p->seq_lens, p->page_table, p->table_stride, p->B, p->T, p->max_pages, p->num_pages,
                   p->page_size};
  const void* src[2] = {p->k, p->v};
  void* dst[2] = {p->k_pages, p->v_pages};
  const int64_t* ss[2] = {p->k_stride, p->v_stride};
  const int64_t* ds[2] = {p->kp_stride, p->vp_stride};
  // the widest unit that divides a row and every row start
  uint64_t bits = static_cast<uint64_t>(p->D) * eb;
  for (int i = 0; i < 2; ++i) {
    a.src[i] = static_cast<const uint8_t*>(src[i]);
    a.dst[i] = static_cast<uint8_t*>(dst[i]);
    a.src_ss[i] = ss[i][0] * eb;
    a.src_sh[i] = ss[i][1] * eb;
    a.dst_sp[i] = ds[i][0] * eb;
    a.dst_sh[i] = ds[i][1] * eb;
    a.dst_ss[i] = ds[i][2] * eb;
    for (int64_t x : {reinterpret_cast<int64_t>(src[i]), reinterpret_cast<int64_t>(dst[i]), a.src_ss[i], a.src_sh[i],
                      a.dst_sp[i], a.dst_sh[i], a.dst_ss[i]})
      bits |= static_cast<uint64_t>(x);
  }
  const int unit = static_cast<int>(std::min<uint64_t>(16, bits & (~bits + 1)));
  a.H = p->H;
  const int64_t units = static_cast<int64_t>(p->D) * eb / unit;
  if (units * p->H > 0x7fffffff) return fail(CEA_ERR_UNSUPPORTED, "%s: %d heads of %d elements", what, p->H, p->D);
  a.units = cea::kvc::make_fastdiv(static_cast<uint32_t>(units));
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  switch (unit) {
    case 16: e = launch_append<uint4>(a, s); break;
    case 8: e = launch_append<uint2>(a, s); break;
    case 4: e = launch_append<uint32_t>(a, s); break;
    case 2: e = launch_append<uint16_t>(a, s); break;
    default: e = launch_append<uint8_t>(a, s); break;
  }
  return e == cudaSuccess ? CEA_OK : fail(CEA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int cea_copy_pages(const cea_copy_pages_params* p, void* stream) {
  const char* what = "cea_copy_pages";
  if (p == nullptr) return fail(CEA_ERR_INVALID, "%s: null params", what);
  if (p->n < 0 || p->layers < 0 || p->num_pages < 0 || p->page_bytes < 0)
    return fail(CEA_ERR_INVALID, "%s: negative size", what);
  if (p->n == 0) return CEA_OK;
  if (!p->src || !p->dst) return fail(CEA_ERR_INVALID, "%s: null indices", what);
  for (int i = 0; i < p->n; ++i)
    if (p->src[i] < 0 || p->src[i] >= p->num_pages || p->dst[i] < 0 || p->dst[i] >= p->num_pages)
      return fail(CEA_ERR_INVALID, "%s: pair %d (%d -> %d) outside a pool of %d pages", what, i, p->src[i], p->dst[i],
                  p->num_pages);
  // every destination once, and none that is also a source: the copies then commute
  try {
    std::vector<int32_t> dst(p->dst, p->dst + p->n), src(p->src, p->src + p->n);
    std::sort(dst.begin(), dst.end());
    std::sort(src.begin(), src.end());
    const auto twice = std::adjacent_find(dst.begin(), dst.end());
    if (twice != dst.end()) return fail(CEA_ERR_INVALID, "%s: page %d is written twice", what, *twice);
    for (size_t i = 0, j = 0; i < src.size() && j < dst.size();) {
      if (src[i] == dst[j]) return fail(CEA_ERR_INVALID, "%s: page %d is both read and written", what, src[i]);
      if (src[i] < dst[j]) ++i; else ++j;
    }
  } catch (const std::exception& e) {
    return fail(CEA_ERR_INVALID, "%s: %s", what, e.what());
  }
  if (p->layers == 0 || p->page_bytes == 0) return CEA_OK;
  if (!p->k_pages || !p->v_pages) return fail(CEA_ERR_INVALID, "%s: null pages", what);
  pg::CopyArgs a{};
  a.pool[0] = static_cast<uint8_t*>(p->k_pages);
  a.pool[1] = static_cast<uint8_t*>(p->v_pages);
  uint64_t bits = static_cast<uint64_t>(p->page_bytes) | reinterpret_cast<uintptr_t>(p->k_pages) |
                  reinterpret_cast<uintptr_t>(p->v_pages);
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? p->v_stride : p->k_stride;
    a.layer_stride[i] = st[0];
    a.page_stride[i] = st[1];
    bits |= static_cast<uint64_t>(st[1]) | (p->layers > 1 ? static_cast<uint64_t>(st[0]) : 0);
  }
  const int unit = static_cast<int>(std::min<uint64_t>(16, bits & (~bits + 1)));
  a.units = p->page_bytes / unit;
  a.layers = p->layers;
  const int64_t chunks = (a.units + pg::kCopyThreads * pg::kCopyUnroll - 1) / (pg::kCopyThreads * pg::kCopyUnroll);
  if (chunks * pg::kCopyPairs > 0x7fffffff) return fail(CEA_ERR_UNSUPPORTED, "%s: pages of %lld bytes", what, (long long)p->page_bytes);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  for (int i0 = 0; i0 < p->n; i0 += pg::kCopyPairs) {
    a.n = std::min(pg::kCopyPairs, p->n - i0);
    for (int i = 0; i < a.n; ++i) a.pair[i] = make_int2(p->src[i0 + i], p->dst[i0 + i]);
    const dim3 grid(static_cast<unsigned>(chunks * a.n), std::min(p->layers, 65535), 2);
    cudaError_t e;
    switch (unit) {
      case 16: e = launch_dependent(pg::copy_pages_kernel<uint4>, grid, pg::kCopyThreads, 0, s, a); break;
      case 8: e = launch_dependent(pg::copy_pages_kernel<uint2>, grid, pg::kCopyThreads, 0, s, a); break;
      case 4: e = launch_dependent(pg::copy_pages_kernel<uint32_t>, grid, pg::kCopyThreads, 0, s, a); break;
      case 2: e = launch_dependent(pg::copy_pages_kernel<uint16_t>, grid, pg::kCopyThreads, 0, s, a); break;
      default: e = launch_dependent(pg::copy_pages_kernel<uint8_t>, grid, pg::kCopyThreads, 0, s, a); break;
    }
    if (e != cudaSuccess) return fail(CEA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  return CEA_OK;
}

}  // extern "C"

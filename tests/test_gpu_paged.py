"""The paged KV cache on the GPU: attention of ragged batches over pages, append and page copy against plain float64
forms, and the cache's own operations."""

import math

import pytest
import torch

import collaborative_edge_system_b200 as cea
import paged_ref as R
from collaborative_edge_system_b200 import _lib, paged

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


def _acc(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def _kernels(x, **kw):
    out = torch.empty_like(x["q"])
    p = paged._attn_params(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"], out, None,
                           kw.get("min_q_len", 0), kw.get("max_q_len"), kw.get("causal", True), kw.get("scale"))
    return _lib.paged_attn_kernels(p)


def _check(x, *, out_dtype=None, with_lse=True, **kw):
    """The call's result against the plain form; rows of no sequence must stay as they were."""
    dtype = x["q"].dtype
    out_dtype = out_dtype or dtype
    T, Hq, D = x["q"].shape
    out = torch.full((T, Hq, D), 77.0, dtype=out_dtype, device=DEV)
    lse = torch.full((Hq, T), 77.0, dtype=_acc(dtype), device=DEV) if with_lse else None
    cea.paged_attend_into(**x, out=out, lse=lse, **kw)
    ref = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"],
                      kw.get("causal", True), kw.get("scale"))
    R.check(out, lse, ref, dtype=dtype, out_dtype=out_dtype, single_p=bool(_kernels(x, **kw) & _lib.PAGED_TC))
    none = ref[0].isnan().all(-1).all(-1).to(DEV)
    assert (out[none] == 77.0).all() and (lse is None or (lse[:, none] == 77.0).all())
    return out


STEPS = [
    ([1], [1]), ([64], [1]), ([65], [1]), ([1000], [1]), ([5, 64, 0, 129, 700, 1], [1] * 6), ([9000, 3, 511], [1, 1, 1]),
    ([40, 300, 77], [2, 0, 3]), ([3, 2, 0, 900], [4, 4, 2, 4]),
]


@pytest.mark.parametrize("lens,counts", STEPS, ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [
    ("bf16", 32, 8, 128, 16), ("f16", 6, 2, 64, 8), ("bf16", 5, 5, 64, 24), ("f16", 4, 1, 128, 128), ("f32", 4, 2, 64, 16),
    ("f64", 3, 3, 20, 5), ("bf16", 4, 2, 80, 16), ("f16", 36, 1, 64, 16), ("f32", 20, 1, 256, 7)])
def test_attention_of_few_new_tokens(dtype, heads, kv_heads, dim, page, lens, counts, causal):
    x = R.batch(lens, counts, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=TYPES[dtype], device=DEV,
                seed=len(lens) * 7 + dim, extra_rows=2)
    _check(x, causal=causal, max_q_len=max(counts))


CHUNKS = [
    ([17], [17]), ([128], [128]), ([200], [33]), ([1200], [600]), ([129, 513, 40], [65, 130, 40]),
    ([300, 700, 5, 0, 64, 90], [1, 260, 0, 0, 64, 17]), ([50, 20, 600], [120, 30, 1]),
]


@pytest.mark.parametrize("lens,counts", CHUNKS, ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [
    ("bf16", 32, 8, 128, 16), ("f16", 6, 2, 64, 8), ("bf16", 5, 5, 64, 40), ("f16", 4, 1, 128, 256), ("f32", 4, 2, 64, 16),
    ("f64", 3, 3, 20, 5), ("f16", 40, 1, 64, 16)])
def test_attention_of_chunks(dtype, heads, kv_heads, dim, page, lens, counts, causal):
    x = R.batch(lens, counts, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=TYPES[dtype], device=DEV,
                seed=len(lens) * 5 + dim, extra_rows=3)
    _check(x, causal=causal)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1], [90, 70]], ids=["step", "chunk"])
def test_accumulation_precision_output_and_scale(dtype, counts):
    x = R.batch([300, 111], counts, heads=8, kv_heads=2, dim=128, page=16, dtype=TYPES[dtype], device=DEV, seed=3)
    _check(x, out_dtype=torch.float32, scale=0.31)
    _check(x, with_lse=False)
    out, lse = cea.paged_attention_with_lse(**x)
    same = torch.empty_like(out)
    cea.paged_attend_into(**x, out=same)
    assert torch.equal(out, same) and lse.dtype == torch.float32
    assert torch.equal(cea.paged_attention(**x), _check(x))


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(128, 1, 64, 16), (160, 1, 128, 8), (130, 2, 64, 1), (64, 64, 64, 32),
                                                     (51, 17, 128, 64), (16, 1, 128, 16), (27, 3, 64, 8)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 0, 3], [70, 1, 9]], ids=["step", "few", "mixed"])
def test_head_groups_from_one_to_all(heads, kv_heads, dim, page, counts):
    x = R.batch([150, 77, 260], counts, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=torch.bfloat16,
                device=DEV, seed=heads)
    _check(x, max_q_len=max(counts))
    _check(x, causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_that_are_not_positive(dtype, scale):
    x = R.batch([300, 111, 0, 5], [90, 1, 1, 9], heads=8, kv_heads=2, dim=64, page=16, dtype=TYPES[dtype], device=DEV, seed=5)
    p = _check(x, scale=scale)
    assert torch.isfinite(p[:91]).all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [100, 37, 64]], ids=["step", "chunk"])
@pytest.mark.parametrize("case", ["slot_major", "fused_q", "odd_q_base", "odd_pages_base", "layer_slice"])
def test_strides_and_alignment(case, counts):
    x = R.batch([200, 333, 64], counts, heads=8, kv_heads=2, dim=64, page=16, dtype=torch.bfloat16, device=DEV, seed=4,
                layout="shd" if case == "slot_major" else "hsd")
    T = x["q"].shape[0]
    if case == "fused_q":
        x["q"] = torch.randn(T, 8 * 64 + 4 * 64, device=DEV).to(torch.bfloat16)[:, : 8 * 64].view(T, 8, 64)
    elif case == "odd_q_base":
        x["q"] = torch.randn(T * 8 * 64 + 1, device=DEV).to(torch.bfloat16)[1:].view(T, 8, 64)
    elif case == "odd_pages_base":
        for n in ("k_pages", "v_pages"):
            flat = torch.empty(x[n].numel() + 1, dtype=torch.bfloat16, device=DEV)
            flat[1:] = x[n].flatten()
            x[n] = flat[1:].view_as(x[n])
    elif case == "layer_slice":
        for n in ("k_pages", "v_pages"):
            x[n] = torch.stack([torch.zeros_like(x[n]), x[n]], 1)[:, 1]
    _check(x)


@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 90, 20]], ids=["step", "chunk"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_page_outside_the_pool_reads_as_zeros_and_is_reported(dtype, counts):
    assert _lib.device_status(clear=True) == 0
    x = R.batch([100, 150, 200], counts, heads=4, kv_heads=2, dim=64, page=16, dtype=TYPES[dtype], device=DEV, seed=6)
    P = x["k_pages"].shape[0]
    good = x["page_table"].clone()
    for bad in (P, -1, 2**31 - 1, -(2**31)):
        x["page_table"] = good.clone()
        x["page_table"][1, 3] = bad
        got = cea.paged_attention(**x)
        assert _lib.device_status(clear=True) == _lib.DEV_BAD_PAGE
        # the same with a page of zeros in the place of the bad one
        y = dict(x, page_table=good.clone())
        y["page_table"][1, 3] = P
        for n in ("k_pages", "v_pages"):
            y[n] = torch.cat([x[n], torch.zeros_like(x[n][:1])])
        assert torch.equal(got, cea.paged_attention(**y))
        assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_batches_that_do_not_fit_the_call_are_reported(dtype):
    assert _lib.device_status(clear=True) == 0
    x = R.batch([60, 40], [1, 20], heads=4, kv_heads=2, dim=64, page=16, dtype=TYPES[dtype], device=DEV, seed=8)
    cap = x["page_table"].shape[1] * 16
    x["page_table"].clamp_(min=0)  # every entry is a page, so that only the length is wrong
    for n in ("k_pages", "v_pages"):
        x[n] = torch.randn(x[n].shape, device=DEV).to(TYPES[dtype])
    full = dict(x, seq_lens=torch.tensor([cap, 40], dtype=torch.int32, device=DEV))
    over = dict(x, seq_lens=torch.tensor([cap + 1000, 40], dtype=torch.int32, device=DEV))
    want = cea.paged_attention(**full)
    assert _lib.device_status(clear=True) == 0
    assert torch.equal(cea.paged_attention(**over), want)  # cut to what the table holds
    assert _lib.device_status(clear=True) == _lib.DEV_BAD_BATCH
    for offsets in ([0, 5, 3], [-4, 1, 21], [0, 1, 400]):
        cea.paged_attention(**dict(x, q_offsets=torch.tensor(offsets, dtype=torch.int32, device=DEV)))
        assert _lib.device_status(clear=True) == _lib.DEV_BAD_BATCH


def test_broken_promises_are_reported():
    assert _lib.device_status(clear=True) == 0
    for dtype in (torch.bfloat16, torch.float32):
        x = R.batch([60, 40], [2, 20], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype, device=DEV, seed=8)
        for kw in ({"max_q_len": 19}, {"min_q_len": 3}, {"max_q_len": 1}):
            cea.paged_attention(**x, **kw)
            assert _lib.device_status(clear=True) == _lib.DEV_BAD_BATCH
        cea.paged_attention(**x, min_q_len=2, max_q_len=20)
        assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("lens,counts", [([1000, 9, 64], [3, 4, 3]), ([5000], [4]), ([300, 0, 65, 3, 700], [4, 0, 3, 3, 4])],
                         ids=["ragged", "one", "empty"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [("bf16", 32, 8, 128, 16), ("f16", 12, 4, 128, 8),
                                                           ("bf16", 8, 2, 64, 16)])
def test_nine_to_sixteen_rows_with_and_without_the_promise(dtype, heads, kv_heads, dim, page, lens, counts, causal):
    # at 128 columns the promise that no sequence has fewer rows changes the kernel
    x = R.batch(lens, counts, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=TYPES[dtype], device=DEV,
                seed=len(lens) * 3 + dim, extra_rows=2)
    promised, open_ = dict(min_q_len=3, max_q_len=4), dict(max_q_len=4)
    assert _kernels(x, **promised) == (_lib.PAGED_TC if dim == 128 else _lib.PAGED_DECODE)
    assert _kernels(x, **open_) == _lib.PAGED_DECODE
    _check(x, causal=causal, **promised)
    _check(x, causal=causal, **open_)
    _check(x, causal=causal, scale=-0.1, **promised)


@pytest.mark.parametrize("dim", [64, 128])
def test_single_tokens_of_wide_groups_among_chunks(dim):
    for lens, counts in (([700, 64, 1], [1, 1, 1]), ([700, 90, 33, 1], [1, 70, 2, 1])):
        x = R.batch(lens, counts, heads=24, kv_heads=2, dim=dim, page=16, dtype=torch.bfloat16, device=DEV, seed=dim)
        _check(x, max_q_len=max(counts))


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 16)])
def test_more_sequences_than_threads(dtype, dim):
    lens = [(i * 37) % 90 for i in range(1500)]
    counts = [min(n, (0, 1, 1, 2, 17, 1, 30)[i % 7]) for i, n in enumerate(lens)]
    x = R.batch(lens, counts, heads=4, kv_heads=2, dim=dim, page=8, dtype=TYPES[dtype], device=DEV, seed=15)
    _check(x)
    x = R.batch(lens, [min(c, 2) for c in counts], heads=4, kv_heads=2, dim=dim, page=8, dtype=TYPES[dtype], device=DEV,
                seed=16)
    _check(x, max_q_len=2)


def test_long_contexts_split_over_the_gpu_and_are_deterministic():
    x = R.batch([60001, 7, 1500], [1, 1, 1], heads=8, kv_heads=1, dim=128, page=16, dtype=torch.bfloat16, device=DEV,
                seed=9)
    a, b = _check(x, max_q_len=1), _check(x, max_q_len=1)
    assert torch.equal(a, b)
    x = R.batch([20011, 900], [70, 5], heads=8, kv_heads=2, dim=64, page=32, dtype=torch.float16, device=DEV, seed=10)
    a, b = _check(x), _check(x)
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [("bf16", 32, 8, 128, 16), ("f16", 32, 8, 64, 16),
                                                           ("bf16", 16, 16, 128, 8), ("bf16", 16, 8, 64, 256)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_long_shares(dtype, heads, kv_heads, dim, page, n):
    """Hundreds of tiles for every CTA: each stage of the rings is reused many times, across many segments."""
    lens = [30011, 700, 12345, 64, 25000, 1, 3333, 9000]
    x = R.batch(lens, [min(n, v) for v in lens], heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=TYPES[dtype],
                device=DEV, seed=dim + page)
    out = torch.empty_like(x["q"])
    lse = torch.empty(heads, x["q"].shape[0], device=DEV)
    for _ in range(3):
        cea.paged_attend_into(**x, out=out, lse=lse, max_q_len=n)
    ref = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"], where=DEV)
    R.check(out, lse, ref, dtype=TYPES[dtype], out_dtype=TYPES[dtype], single_p=bool(_kernels(x, max_q_len=n) & _lib.PAGED_TC))
    assert _lib.device_status(clear=True) == 0


def test_page_offsets_behind_32_bits():
    P, H, ps, D = 70000, 8, 64, 64  # 2.3e9 elements per pool
    k, v = (torch.zeros(P, H, ps, D, dtype=torch.float16, device=DEV) for _ in range(2))
    ids = [P - 1, 1, P - 2, 65536]
    for t in (k, v):
        t[ids] = torch.randn(4, H, ps, D, device=DEV).half()
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    for n in (1, 60):
        x = {"q": torch.randn(n, 16, D, device=DEV).half(), "k_pages": k, "v_pages": v, "page_table": table,
             "seq_lens": torch.tensor([250], dtype=torch.int32, device=DEV),
             "q_offsets": torch.tensor([0, n], dtype=torch.int32, device=DEV)}
        _check(x)
    new = torch.randn(3, H, D, device=DEV).half()
    cea.paged_append(new, new * 2, k, v, table, torch.tensor([64], dtype=torch.int32, device=DEV),
                     torch.tensor([0, 3], dtype=torch.int32, device=DEV))
    assert torch.equal(k[P - 1, :, 61:].transpose(0, 1), new) and torch.equal(v[P - 1, :, 61:].transpose(0, 1), new * 2)
    cea.copy_pages(k, v, [P - 1], [P - 3])
    assert torch.equal(k[P - 3], k[P - 1]) and torch.equal(v[P - 3], v[P - 1])


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [30, 1, 17, 1]], ids=["step", "mixed"])
def test_captured_graph_serves_changing_batches(counts):
    x = R.batch([400, 30, 200, 9], counts, heads=8, kv_heads=2, dim=128, page=16, dtype=torch.bfloat16, device=DEV,
                seed=11, poison=False)
    out = torch.zeros_like(x["q"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cea.paged_attend_into(**x, out=out)  # warm-up on the stream of the capture
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    new = torch.randn(x["q"].shape[0], 2, 128, device=DEV).to(torch.bfloat16)
    with torch.cuda.graph(g):
        cea.paged_append(new, new, x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
        cea.paged_attend_into(**x, out=out)
    for lens in ([400, 30, 200, 9], [399, 40, 100, 1], [32, 33, 0, 8]):
        x["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        x["page_table"].clamp_(min=0)
        x["q"].normal_()
        new.normal_()
        g.replay()
        again = torch.zeros_like(out)
        ref = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
        cea.paged_attend_into(**x, out=again)
        assert torch.equal(out, again)
        R.check(out, None, ref, dtype=torch.bfloat16, out_dtype=torch.bfloat16, single_p=True)
    _lib.device_status(clear=True)  # positions before a short sequence's start were reported by the append


def test_graph_of_a_whole_step_over_layers():
    """Append and attention of several layers in one graph, replayed while lengths grow: the tokens of every step."""
    L, H, D, ps, B = 3, 2, 64, 8, 4
    cache = cea.PagedKVCache(L, 40, ps, H, D, dtype=torch.bfloat16, device=DEV)
    seqs = [cache.add() for _ in range(B)]
    first = cache.extend(seqs, [9, 1, 30, 16])
    k0 = torch.randn(L, first.num_tokens, H, D, device=DEV).to(torch.bfloat16)
    for layer in range(L):
        cache.append(layer, k0[layer], k0[layer], first)
    table = torch.zeros(B, 10, dtype=torch.int32, device=DEV)
    lens, offs = torch.zeros(B, dtype=torch.int32, device=DEV), torch.arange(B + 1, dtype=torch.int32, device=DEV)
    q, k, v = (torch.zeros(L, B, h, D, dtype=torch.bfloat16, device=DEV) for h in (8, H, H))
    out = torch.zeros_like(q)

    def step():
        for layer in range(L):
            cea.paged_append(k[layer], v[layer], cache.k[layer], cache.v[layer], table, lens, offs)
            cea.paged_attend_into(q[layer], cache.k[layer], cache.v[layer], table, lens, offs, out[layer], min_q_len=1,
                                  max_q_len=1)

    batch = cache.extend(seqs, [1] * B)
    table[:, : batch.page_table.shape[1]] = batch.page_table
    lens.copy_(batch.seq_lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(12):
        if turn:
            batch = cache.extend(seqs, [1] * B)
            table.zero_()
            table[:, : batch.page_table.shape[1]] = batch.page_table
            lens.copy_(batch.seq_lens)
        for t in (q, k, v):
            t.normal_()
        graph.replay()
        for layer in range(L):
            ref = R.attention(q[layer], cache.k[layer], cache.v[layer], table, lens, offs)
            R.check(out[layer], None, ref, dtype=torch.bfloat16, out_dtype=torch.bfloat16, single_p=False)
        pos = lens.long() - 1
        at = table.long()[torch.arange(B, device=DEV), pos // ps]
        assert torch.equal(cache.k[:, at, :, pos % ps], k.transpose(0, 1)) and torch.equal(
            cache.v[:, at, :, pos % ps], v.transpose(0, 1))
    assert _lib.device_status(clear=True) == 0


def test_calls_of_all_kernels_one_after_another():
    """Launches overlap the end of the one before: nothing may be read or written before it is through."""
    kinds = [([900, 64, 5000], [300, 64, 17]), ([700, 65, 3], [1, 1, 1]), ([3000, 40], [4, 3]), ([600, 900], [1, 120])]
    xs = [R.batch(lens, counts, heads=32, kv_heads=8, dim=128, page=16, dtype=torch.bfloat16, device=DEV, seed=i)
          for i, (lens, counts) in enumerate(kinds)]
    alone = []
    for x in xs:
        alone.append(cea.paged_attention(**x))
        torch.cuda.synchronize()
    pages = [(torch.empty_like(x["k_pages"]), torch.empty_like(x["v_pages"])) for x in xs]
    for _ in range(100):
        outs = []
        for x, (k, v) in zip(xs, pages):
            # pages filled, read and spoilt again by neighbours in the stream
            k.copy_(x["k_pages"])
            v.copy_(x["v_pages"])
            outs.append(cea.paged_attention(**{**x, "k_pages": k, "v_pages": v}))
            k.fill_(float("nan"))
            v.fill_(float("nan"))
        for a, b in zip(outs, alone):
            assert torch.equal(a, b)
    assert _lib.device_status(True) == 0


def test_two_streams_at_once():
    xs = [R.batch([700 + 50 * i, 90], [1, 40], heads=8, kv_heads=2, dim=64, page=16, dtype=torch.bfloat16, device=DEV,
                  seed=20 + i) for i in range(4)]
    want = [cea.paged_attention(**x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(cea.paged_attention(**x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shards_merge_to_the_whole():
    """Two ranks that hold the two halves of a sequence in their pages: partials with statistics merge exactly."""
    x = R.batch([700], [3], heads=8, kv_heads=2, dim=64, page=16, dtype=torch.float32, device=DEV, seed=12)
    whole, lse = cea.paged_attention_with_lse(**x)
    head = dict(x, seq_lens=torch.tensor([320], dtype=torch.int32, device=DEV))
    tail = dict(x, page_table=x["page_table"][:, 20:].contiguous(), seq_lens=torch.tensor([380], dtype=torch.int32, device=DEV))
    (o1, l1), (o2, l2) = cea.paged_attention_with_lse(**head, causal=False), cea.paged_attention_with_lse(**tail)
    o, l = cea.merge_attention(o1[None], l1[None], o2[None], l2[None])
    assert (o[0] - whole).abs().max() < 2e-6 and (l[0] - lse).abs().max() < 2e-6


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.uint8],
                         ids=lambda d: str(d).replace("torch.", ""))
@pytest.mark.parametrize("H,D,page,pad", [(8, 128, 16, 0), (3, 80, 5, 0), (1, 1, 1, 3), (2, 20, 8, 5), (40, 64, 32, 0)])
def test_append_writes_every_token_to_its_place(dtype, H, D, page, pad):
    lens, counts = [3, 200, 0, 65, 7, 16, 1000], [3, 41, 0, 1, 7, 15, 130]
    x = R.batch(lens, counts, heads=H, kv_heads=H, dim=D, page=page, dtype=torch.float32, device=DEV, seed=13,
                poison=False)
    T = sum(counts) + 4  # the last rows are of no sequence
    fused = (torch.randn(T, 2 * H * D + pad, device=DEV) * 50).to(dtype)
    k, v = fused[:, : H * D].view(T, H, D), fused[:, H * D : 2 * H * D].view(T, H, D)
    pools = [(x[n] * 50).to(dtype) for n in ("k_pages", "v_pages")]
    want = [p.clone() for p in pools]
    row = 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        for i in range(c):
            pos = n - c + i
            pg = int(x["page_table"][b, pos // page])
            want[0][pg, :, pos % page], want[1][pg, :, pos % page] = k[row], v[row]
            row += 1
    cea.paged_append(k, v, pools[0], pools[1], x["page_table"], x["seq_lens"], x["q_offsets"])
    assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
    assert _lib.device_status(clear=True) == 0


def test_append_of_many_sequences_and_slot_major_pages():
    for B in (1, 31, 32, 33, 1000, 1025, 3000):
        lens = [1 + (i * 37) % 60 for i in range(B)]
        counts = [0 if i % 7 == 3 else 1 for i in range(B)]
        x = R.batch(lens, counts, heads=2, kv_heads=2, dim=16, page=8, dtype=torch.float16, device=DEV, seed=B,
                    poison=False, layout="shd")
        T = sum(counts)
        k = torch.randn(T, 2, 16, device=DEV).half()
        want = x["k_pages"].clone()
        b = torch.tensor([i for i in range(B) if counts[i]], device=DEV)
        pos = (x["seq_lens"].long() - 1)[b]
        want[x["page_table"].long()[b, pos // 8], :, pos % 8] = k
        cea.paged_append(k, k, x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
        assert torch.equal(x["k_pages"], want)


def test_append_drops_and_reports_tokens_without_a_page():
    assert _lib.device_status(clear=True) == 0
    x = R.batch([20, 40, 8], [6, 3, 8], heads=2, kv_heads=2, dim=64, page=8, dtype=torch.bfloat16, device=DEV, seed=14,
                poison=False)
    k = torch.randn(17, 2, 64, device=DEV).to(torch.bfloat16)
    before = x["k_pages"].clone()
    x["page_table"][0, 2] = x["k_pages"].shape[0]  # tokens 16 .. 19
    x["seq_lens"][2] = 5                            # three of eight new tokens before the sequence's start
    cea.paged_append(k, k, x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
    assert _lib.device_status(clear=True) == _lib.DEV_BAD_PAGE
    t = x["page_table"].long()
    before[t[0, 1], :, 6:8] = k[:2].transpose(0, 1)
    before[t[1, 4], :, 5:8] = k[6:9].transpose(0, 1)
    before[t[2, 0], :, 0:5] = k[12:17].transpose(0, 1)
    assert torch.equal(x["k_pages"], before)


# ------------------------------------------------------------------------------------------------ page copy
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8], ids=lambda d: str(d).replace("torch.", ""))
@pytest.mark.parametrize("L,P,H,page,D,n", [(1, 4, 1, 1, 1, 2), (3, 40, 2, 8, 20, 17), (2, 1500, 1, 4, 8, 700),
                                            (5, 12, 8, 16, 128, 6), (2, 6, 3, 5, 7, 1)])
@pytest.mark.parametrize("layout", ["hsd", "shd"])
def test_copy_pages(dtype, L, P, H, page, D, n, layout):
    g = torch.Generator().manual_seed(P)
    k, v = ((torch.randn(L, P, H, page, D, generator=g) * 50).to(dtype).to(DEV) for _ in range(2))
    if layout == "shd":
        k, v = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    order = torch.randperm(P, generator=g)
    src, dst = order[:n], order[n : 2 * n]
    src[n // 2 :] = src[0]  # one page to many places
    wk, wv = k.clone(), v.clone()
    wk[:, dst.to(DEV)], wv[:, dst.to(DEV)] = k[:, src.to(DEV)], v[:, src.to(DEV)]
    cea.copy_pages(k, v, src.tolist(), dst.int())
    assert torch.equal(k, wk) and torch.equal(v, wv)


def test_copy_pages_of_one_layer_and_refusals_change_nothing():
    k = torch.randn(10, 2, 4, 8, device=DEV)
    v = torch.randn(10, 2, 4, 8, device=DEV)
    k0, v0 = k.clone(), v.clone()
    for src, dst, word in (([0, 1], [2, 2], "written twice"), ([0, 2], [2, 3], "both read and written"),
                           ([0], [10], "outside"), ([-1], [3], "range"), ([0, 1], [2], "destinations"),
                           ([5], [5], "both")):
        with pytest.raises(ValueError, match=word):
            cea.copy_pages(k, v, src, dst)
    assert torch.equal(k, k0) and torch.equal(v, v0)
    cea.copy_pages(k, v, [], [])
    cea.copy_pages(k, v, [1], [4])
    assert torch.equal(k[4], k0[1]) and torch.equal(v[4], v0[1]) and torch.equal(k[:4], k0[:4])
    with pytest.raises(ValueError, match="contiguous block"):
        cea.copy_pages(k[..., ::2], v[..., ::2], [0], [1])


# ------------------------------------------------------------------------------------------------ the cache
@pytest.mark.parametrize("dtype,page", [(torch.float32, 5), (torch.bfloat16, 8)], ids=["f32", "bf16"])
def test_cache_operations_keep_every_sequence(dtype, page):
    """Extend, append, fork, truncate, free and compact in a random order: each sequence's tokens, read back through
    its pages, are the ones that were appended to it, and its attention is the plain one."""
    import random

    rnd = random.Random(5)
    L, P, H, D = 2, 90, 2, 64
    cache = cea.PagedKVCache(L, P, page, H, D, dtype=dtype, device=DEV)
    want = {}  # id -> list of (k, v) per token [L, H, D]
    for turn in range(60):
        move = rnd.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        ids = sorted(want)
        if move == "add" or not ids:
            want[cache.add()] = []
        elif move == "extend":
            some = rnd.sample(ids, rnd.randint(1, len(ids)))
            counts = [rnd.randint(0, 9) for _ in some]
            free = cache.num_free_pages
            try:
                batch = cache.extend(some, counts)
            except cea.OutOfPages:
                assert cache.num_free_pages == free
                continue
            k, v = (torch.randn(L, batch.num_tokens, H, D, device=DEV).to(dtype) for _ in range(2))
            for layer in range(L):
                cache.append(layer, k[layer], v[layer], batch)
            row = 0
            for s, c in zip(some, counts):
                want[s] = want[s] + [(k[:, row + i], v[:, row + i]) for i in range(c)]
                row += c
            if batch.num_tokens:
                q = torch.randn(batch.num_tokens, 4, D, device=DEV).to(dtype)
                out = cache.attend(1, q, batch)
                ref = R.attention(q, cache.k[1], cache.v[1], batch.page_table, batch.seq_lens, batch.q_offsets)
                R.check(out, None, ref, dtype=dtype, out_dtype=dtype, single_p=True)
        elif move == "fork":
            s = rnd.choice(ids)
            n = rnd.choice([None, rnd.randint(0, len(want[s]))])
            try:
                new = cache.fork(s, n, rnd.randint(1, 3))
            except cea.OutOfPages:
                continue
            for f in new:
                want[f] = want[s][: len(want[s]) if n is None else n]
        elif move == "truncate":
            s = rnd.choice(ids)
            n = rnd.randint(0, len(want[s]))
            cache.truncate(s, n)
            want[s] = want[s][:n]
        elif move == "free" and len(ids) > 3:
            s = rnd.choice(ids)
            cache.free(s)
            del want[s]
        elif move == "compact":
            used = cache.compact()
            assert used == P - cache.num_free_pages
            assert all(p < used for s in ids for p in cache.pages(s))
        for s, tokens in want.items():
            assert cache.length(s) == len(tokens)
            pages = cache.pages(s)
            assert len(pages) == -(-len(tokens) // page)
            if tokens:
                for got, i in ((cache.k, 0), (cache.v, 1)):
                    flat = got[:, pages].transpose(2, 3).reshape(L, -1, H, D)[:, : len(tokens)]
                    assert torch.equal(flat, torch.stack([t[i] for t in tokens], 1))
    for s in list(want):
        cache.free(s)
    assert cache.num_free_pages == P and _lib.device_status(clear=True) == 0

"""Calls of the paged operators at the edges of what they allow: extreme weights and values, batches that do not fit, the
state after a device-side timeout."""

import math

import pytest
import torch

import collaborative_edge_system_b200 as cea
import paged_ref as R
from collaborative_edge_system_b200 import _lib, paged

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "f64": torch.float64}


def _kernels(x, **kw):
    p = paged._attn_params(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"],
                           torch.empty_like(x["q"]), None, kw.get("min_q_len", 0), kw.get("max_q_len"),
                           kw.get("causal", True), kw.get("scale"))
    return _lib.paged_attn_kernels(p)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,n", [("bf16", 16, 8, 64, 1), ("f16", 32, 8, 128, 4), ("bf16", 16, 8, 128, 19),
                                                        ("f16", 8, 8, 64, 70)])
def test_hundreds_of_short_segments_in_every_share(dtype, heads, kv_heads, dim, n):
    """The queue between the warp that walks a share and the others turns over many times, with segments of one tile
    whose readers keep up at different speeds."""
    lens = [n + (i * 7) % 41 for i in range(2500)]
    x = R.batch(lens, [n - i % 2 * (n > 1) for i in range(2500)], heads=heads, kv_heads=kv_heads, dim=dim, page=8,
                dtype=TYPES[dtype], device=DEV, seed=n)
    out = cea.paged_attention(**x, max_q_len=n)
    for _ in range(30):
        assert torch.equal(cea.paged_attention(**x, max_q_len=n), out)
    ref = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"], where=DEV)
    R.check(out, None, ref, dtype=TYPES[dtype], out_dtype=TYPES[dtype], single_p=bool(_kernels(x, max_q_len=n) & _lib.PAGED_TC))
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (15, 5, 128), (5, 1, 64), (14, 2, 128)])
def test_warps_of_the_chunk_kernel_with_rows_of_no_token(heads, kv_heads, dim, out_dtype):
    """Groups that do not divide a tile and chunks that end within a warp's rows, whole and split over the GPU: lanes
    without a token stay in step with those that have one."""
    lens, counts = [17, 40, 300, 9000, 129], [17, 33, 50, 21, 129]
    x = R.batch(lens, counts, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=torch.bfloat16, device=DEV, seed=heads,
                extra_rows=1)
    ref = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
    assert _kernels(x, min_q_len=17) == _lib.PAGED_TC
    for _ in range(5):
        out = torch.full(x["q"].shape, 77.0, dtype=out_dtype, device=DEV)
        lse = torch.full((heads, out.shape[0]), 77.0, device=DEV)
        cea.paged_attend_into(**x, out=out, lse=lse, min_q_len=17)
        R.check(out, lse, ref, dtype=torch.bfloat16, out_dtype=out_dtype, single_p=True)
        assert (out[-1] == 77.0).all() and (lse[:, -1] == 77.0).all()
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("dtype,n,kernel", [("f16", 40, _lib.PAGED_TC), ("bf16", 1, _lib.PAGED_DECODE), ("f32", 1, _lib.PAGED_SIMT)])
def test_the_longest_sequence(dtype, n, kernel, causal):
    """2^31 - 256 keys, one page under every entry of the table: a unit's keys and its cost are above 31 bits.

    All scores are 0 and the values 0 or 1, so every sum of a share (below 2^24) is exact; what is left are the
    statistics of the parts, off by three roundings of ln 2^24 at most, and their weights in the join."""
    page, D, total = 65536, 64, 2**31 - 256
    slot = torch.arange(page)[:, None] * torch.arange(1, D + 1)[None, :]
    ones = (slot % 5 == 0).long()
    x = {"q": torch.zeros(n, 1, D, dtype=TYPES[dtype], device=DEV),
         "k_pages": torch.randn(1, 1, page, D, device=DEV).to(TYPES[dtype]),
         "v_pages": ones.to(TYPES[dtype]).to(DEV)[None, None],
         "page_table": torch.zeros(1, 2**31 // page, dtype=torch.int32, device=DEV),
         "seq_lens": torch.tensor([total], dtype=torch.int32, device=DEV),
         "q_offsets": torch.tensor([0, n], dtype=torch.int32, device=DEV)}
    kw = {"min_q_len": n, "max_q_len": n, "causal": causal}
    assert _kernels(x, **kw) == kernel
    out, lse = cea.paged_attention_with_lse(**x, **kw)
    seen = torch.arange(total - n + 1, total + 1) if causal else torch.full((n,), total)
    ahead = torch.cat([torch.zeros(1, D, dtype=torch.long), ones.cumsum(0)])
    want = (seen // page)[:, None] * ahead[-1] + ahead[seen % page]
    bound = 2 * 3 * math.log(2**24) * 2.0**-24 + 2.0**-20
    assert float((out[:, 0].double().cpu() / (want / seen[:, None].double()) - 1).abs().max()) <= bound
    assert float((lse[0].double().cpu() - seen.double().log()).abs().max()) <= bound + math.log(2**31) * 2.0**-23
    assert _lib.device_status(clear=True) == 0


def test_append_of_as_many_rows_as_32_bits_count():
    """Three rows of two sequences and 2^31 - 4 of none behind them, of a byte each."""
    k = torch.zeros(2**31 - 1, 1, 1, dtype=torch.uint8, device=DEV)
    k[:3, 0, 0] = torch.tensor([7, 8, 9], dtype=torch.uint8)
    k_pages, v_pages = (torch.full((3, 1, 4, 1), 1, dtype=torch.uint8, device=DEV) for _ in range(2))
    cea.paged_append(k, k, k_pages, v_pages, torch.tensor([[2, -1], [0, 1]], dtype=torch.int32, device=DEV),
                     torch.tensor([4, 5], dtype=torch.int32, device=DEV), torch.tensor([0, 2, 3], dtype=torch.int32, device=DEV))
    want = torch.full((3, 4), 1, dtype=torch.uint8)
    want[2, 2], want[2, 3], want[1, 0] = 7, 8, 9
    assert torch.equal(k_pages.view(3, 4).cpu(), want) and torch.equal(v_pages.view(3, 4).cpu(), want)
    assert _lib.device_status(clear=True) == 0


def _time_out():
    """A bounded wait on a flag that nothing sets: the exchange of two ranks of which one never comes."""
    bufs = [torch.zeros(2 * 2 * 4 * 8, device=DEV) for _ in range(2)]
    flags = [torch.zeros(2, dtype=torch.int64, device=DEV) for _ in range(2)]
    out = torch.zeros(1, 1, 4, 4, device=DEV)
    _lib.peer_merge(2, 0, [b.data_ptr() for b in bufs], [f.data_ptr() for f in flags], 1, 8, out, wait_limit_ns=1_000_000)
    torch.cuda.synchronize()
    assert _lib.device_status(clear=False) == _lib.DEV_TIMEOUT_PEER and out.isnan().all()


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("bf16", 64), ("f16", 128), ("f32", 64), ("f64", 64),
                                       ("bf16", 80)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [60, 1, 20]], ids=["step", "mixed"])
def test_attention_computes_nothing_after_a_timeout(dtype, dim, counts):
    x = R.batch([3000, 40, 500], counts, heads=8, kv_heads=2, dim=dim, page=16, dtype=TYPES[dtype], device=DEV, seed=23)
    before = cea.paged_attention(**x)
    _time_out()
    try:
        out = torch.full_like(before, 77.0)
        lse = torch.full((8, out.shape[0]), 77.0, dtype=paged.accumulation_dtype(out.dtype), device=DEV)
        cea.paged_attend_into(**x, out=out, lse=lse)
        assert (out == 77.0).all() and (lse == 77.0).all()
        # data movement depends on no wait and goes on
        k = torch.randn(out.shape[0], 2, dim, device=DEV).to(TYPES[dtype])
        copy = {n: x[n].clone() for n in ("k_pages", "v_pages")}
        cea.paged_append(k, k, **copy, page_table=x["page_table"], seq_lens=x["seq_lens"], q_offsets=x["q_offsets"])
        assert torch.equal(copy["k_pages"][int(x["page_table"][2, 499 // 16]), :, 499 % 16], k[-1])
    finally:
        assert _lib.device_status(clear=True) == _lib.DEV_TIMEOUT_PEER
    assert torch.equal(cea.paged_attention(**x), before)
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("rows", [3, 7, 9, 12])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_append_of_fewer_rows_than_the_batch_has(dtype, rows):
    """The rows that are there go to their own places, and the batch is reported."""
    assert _lib.device_status(clear=True) == 0
    x = R.batch([10, 20, 9], [5, 4, 3], heads=2, kv_heads=2, dim=16, page=4, dtype=dtype, device=DEV, seed=21, poison=False)
    k = torch.randn(rows, 2, 16, device=DEV).to(dtype)
    want = x["k_pages"].clone()
    places = [(0, p) for p in range(5, 10)] + [(1, p) for p in range(16, 20)] + [(2, p) for p in range(6, 9)]
    for row, (b, p) in enumerate(places[:rows]):
        want[int(x["page_table"][b, p // 4]), :, p % 4] = k[row]
    cea.paged_append(k, k, x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
    assert torch.equal(x["k_pages"], want)
    assert _lib.device_status(clear=True) == (0 if rows == 12 else _lib.DEV_BAD_BATCH)


@pytest.mark.parametrize("offsets", [[0, 5, 3, 9], [-4, 1, 5, 9], [0, 5, 9, 400], [0, 2**31 - 1, 9, 9]])
def test_append_reports_offsets_that_do_not_fit(offsets):
    assert _lib.device_status(clear=True) == 0
    x = R.batch([400, 400, 400], [1, 1, 1], heads=2, kv_heads=2, dim=16, page=4, dtype=torch.bfloat16, device=DEV, seed=22)
    k = torch.randn(9, 2, 16, device=DEV).to(torch.bfloat16)
    cea.paged_append(k, k, x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"],
                     torch.tensor(offsets, dtype=torch.int32, device=DEV))
    assert _lib.device_status(clear=True) in (_lib.DEV_BAD_BATCH, _lib.DEV_BAD_PAGE)
    fine = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV)
    cea.paged_append(k, k, x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], fine)
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("rows", [1, 2, 24, 30])
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_attention_of_fewer_rows_than_the_batch_has(dtype, dim, rows):
    """The rows that are there keep their positions, and the batch is reported."""
    assert _lib.device_status(clear=True) == 0
    x = R.batch([700, 90, 33], [2, 60, 1], heads=8, kv_heads=4, dim=dim, page=16, dtype=TYPES[dtype], device=DEV, seed=24)
    ref = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
    x["q"] = x["q"][:rows]
    assert _kernels(x) == (_lib.PAGED_SIMT if dtype == "f32" else _lib.PAGED_DECODE | (_lib.PAGED_TC if rows > 4 else 0))
    out, lse = cea.paged_attention_with_lse(**x)
    assert _lib.device_status(clear=True) == _lib.DEV_BAD_BATCH
    R.check(out, lse, (ref[0][:rows], ref[1][:, :rows], ref[2][:rows], ref[3][:, :rows]), dtype=TYPES[dtype],
            out_dtype=torch.float32, single_p=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tail", ["even", "spread"])
@pytest.mark.parametrize("dim,group,n", [(64, 1, 1), (128, 4, 1), (64, 4, 4), (64, 1, 20), (128, 4, 33)])
def test_one_key_far_above_a_long_tail(dtype, tail, dim, group, n):
    """One key holds nearly all the weight and a value of 0; the output is what is left of the others, 2^-20 to 2^-26 of it
    each.  Queries pick one column of the keys, so the scores are exact.

    A weight's exponent (below 26 in magnitude, log2) takes three roundings of half a step of fp32, the hardware's exp2 is
    good to 2^-22.  Rounded to 16 bits it is off by half a step, 2^-11 or 2^-8 (one number, the chunk kernel) or the square
    of it, 2^-22 or 2^-17 with the second's rounding (two, the decode kernel), in f16 at least by 2^-25 of the unit that
    the kernel holds it in: 2^-7 and 2^-14 of the largest weight.  Products of 16 keys are added one after another, each
    sum cut to fp32 (2^-23), in the decode kernel for two numbers by each of eight warps."""
    N, H, B, page = 32768, 32, 6, 64
    t = TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(dim + n)
    k = torch.zeros(N // page, H, page, dim, dtype=t, device=DEV)
    score = torch.zeros(H, N, device=DEV) if tail == "even" else torch.rand(H, N, generator=g, device=DEV) * 4 - 1
    score[:, 37] = 17.25
    k[:, :, :, 0] = score.to(t).view(H, N // page, page).transpose(0, 1)
    score = k[:, :, :, 0].transpose(0, 1).reshape(H, N).double()
    v = torch.rand(N // page, H, page, dim, generator=g, device=DEV).to(t)
    v[37 // page, :, 37 % page] = 0
    q = torch.zeros(B * n, H * group, dim, dtype=t, device=DEV)
    q[:, :, 0] = 1
    x = {"q": q, "k_pages": k, "v_pages": v,
         "page_table": torch.arange(N // page, dtype=torch.int32, device=DEV).expand(B, -1),  # all read the same pages
         "seq_lens": torch.full((B,), N, dtype=torch.int32, device=DEV),
         "q_offsets": torch.arange(0, B * n + 1, n, dtype=torch.int32, device=DEV)}
    out = torch.empty(q.shape, device=DEV)
    lse = torch.empty(H * group, B * n, device=DEV)
    kw = {"scale": 1.0, "causal": False, "min_q_len": n, "max_q_len": n}
    cea.paged_attend_into(**x, out=out, lse=lse, **kw)
    single = _kernels(x, **kw)
    assert single in (_lib.PAGED_TC, _lib.PAGED_DECODE)
    single = single == _lib.PAGED_TC
    p = torch.softmax(score, -1)
    values = v.transpose(0, 1).reshape(H, N, dim).double()
    want = torch.einsum("hj,hjd->hd", p, values)
    e = 3 * 26 * 2.0**-24 * math.log(2) + 2.0**-22
    half = torch.finfo(t).eps / 2
    relative = (half if single else max(half * half, 2.0**-17 if dtype == "bf16" else 0)) + 2 * e
    relative += (N / 16 if single else 2 * N / 128) * 2.0**-23 + N / 64 * 2.0**-24
    absolute = (2.0**-25 * (2.0**-7 if single else 2.0**-14) * values.sum(1)) if dtype == "f16" else 0.0
    tol = (want * (relative + 2.0**-24) + absolute).repeat_interleave(group, 0)
    off = (out.double() - want.repeat_interleave(group, 0)).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), float((off / want.repeat_interleave(group, 0)).max()))
    stat = torch.logsumexp(score, -1).repeat_interleave(group, 0)[:, None]
    assert float((lse.double() - stat).abs().max()) <= e + (N / 64 + 4 * 18) * 2.0**-24
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,counts", [
    ("bf16", 8, 2, 128, [1, 1, 1]), ("f16", 8, 8, 64, [1, 2, 1]), ("bf16", 16, 4, 64, [4, 3, 1]), ("f16", 4, 1, 128, [30, 20, 1]),
    ("bf16", 4, 4, 64, [70, 2, 1]), ("f32", 4, 2, 64, [3, 20, 1]), ("bf16", 4, 2, 80, [1, 5, 1])])
def test_an_infinite_value_that_a_token_sees_gives_that_infinity(dtype, heads, kv_heads, dim, counts):
    lens = [5000, 200, 1]
    x = R.batch(lens, counts, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=TYPES[dtype], device=DEV, seed=dim)
    plain = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
    for b, key in enumerate([3111, 70, 0]):  # seen by every new token
        page = int(x["page_table"][b, key // 16])
        x["v_pages"][page, :, key % 16, 3] = math.inf
        x["v_pages"][page, :, key % 16, 5] = -math.inf
    for kw in ({}, {"causal": False}):
        out, lse = cea.paged_attention_with_lse(**x, max_q_len=max(counts), **kw)
        assert (out[..., 3] == math.inf).all() and (out[..., 5] == -math.inf).all()
        assert torch.isfinite(lse).all()
        assert torch.isfinite(out[..., [d for d in range(dim) if d not in (3, 5)]]).all()
        if not kw:
            keep = [d for d in range(dim) if d not in (3, 5)]
            R.check(out[..., keep], lse, (plain[0][..., keep], plain[1], plain[2][..., keep], plain[3]), dtype=TYPES[dtype],
                    out_dtype=torch.float32, single_p=bool(_kernels(x, max_q_len=max(counts)) & _lib.PAGED_TC))
    assert _lib.device_status(clear=True) == 0


def _spoilt(lens, counts, heads, kv_heads, dim, dtype, seed, bad):
    """A batch, its plain result, and the same batch with `bad` in some columns of the values of new tokens: of the last but
    one of every sequence that has two, and of every fifth."""
    x = R.batch(lens, counts, heads=heads, kv_heads=kv_heads, dim=dim, page=16, dtype=TYPES[dtype], device=DEV, seed=seed)
    plain = R.attention(x["q"], x["k_pages"], x["v_pages"], x["page_table"], x["seq_lens"], x["q_offsets"])
    sees = torch.zeros(sum(counts), dtype=torch.bool)
    row = 0
    for b, (n_all, n) in enumerate(zip(lens, counts)):
        spoilt = [i for i in range(n) if n > 1 and n_all - n + i >= 0 and (i == n - 2 or (i % 5 == 3 and n > 6))]
        for i in spoilt:
            pos = n_all - n + i
            x["v_pages"][int(x["page_table"][b, pos // 16]), :, pos % 16, 1::7] = bad
        for i in range(n):
            sees[row + i] = any(s <= i for s in spoilt)
        row += n
    return x, plain, sees


LEAKS = {
    _lib.PAGED_SIMT: [("f32", 8, 2, 64, [700, 33, 5], [40, 17, 2]), ("bf16", 4, 2, 80, [90, 300, 40], [3, 130, 40]),
                      ("f64", 3, 3, 20, [50, 20], [9, 20]), ("f16", 6, 2, 64, [90, 9], [70, 9])],
    _lib.PAGED_DECODE: [("bf16", 8, 8, 64, [5000, 8, 65, 1], [8, 8, 5, 1]), ("f16", 32, 8, 128, [700, 64, 2, 3], [2, 2, 2, 2]),
                        ("bf16", 16, 4, 64, [300, 66, 4], [4, 3, 4]), ("f16", 12, 4, 128, [900, 5, 66, 2], [4, 4, 3, 1])],
    _lib.PAGED_TC: [("bf16", 32, 8, 128, [9000, 90, 17, 64], [33, 70, 17, 64]), ("f16", 8, 8, 64, [700, 300, 1000], [700, 257, 20]),
                    ("bf16", 15, 5, 128, [200, 130], [130, 66]), ("f16", 64, 1, 64, [2000, 9], [5, 9])],
}


def _leak_cases(kernel):
    return pytest.mark.parametrize("dtype,heads,kv_heads,dim,lens,counts", LEAKS[kernel], ids=lambda v: str(v).replace(" ", ""))


def _no_leak(kernel, dtype, heads, kv_heads, dim, lens, counts, bad):
    x, plain, sees = _spoilt(lens, counts, heads, kv_heads, dim, dtype, dim + heads, bad)
    if kernel == _lib.PAGED_SIMT and dtype == "f16":  # a shape of the tensor kernels whose rows are not aligned for them
        for n in ("k_pages", "v_pages"):
            flat = torch.empty(x[n].numel() + 1, dtype=x[n].dtype, device=DEV)
            flat[1:] = x[n].flatten()
            x[n] = flat[1:].view_as(x[n])
    kw = {"min_q_len": min(counts), "max_q_len": max(counts)}
    assert _kernels(x, **kw) == kernel
    out, lse = cea.paged_attention_with_lse(**x, **kw)
    keep = torch.ones(dim, dtype=torch.bool)
    keep[1::7] = False
    single = kernel == _lib.PAGED_TC
    check = lambda cols, rows: R.check(  # noqa: E731
        out[rows][..., cols], lse[:, rows], (plain[0][rows][..., cols], plain[1][:, rows], plain[2][rows][..., cols],
                                            plain[3][:, rows]), dtype=TYPES[dtype], out_dtype=out.dtype, single_p=single)
    rows = torch.arange(len(sees))
    check(keep, rows)  # the other columns, of every token
    if bool((~sees).any()):
        check(~keep, rows[~sees])  # the spoilt ones, of the tokens that do not see them
    seen = out[rows[sees]][..., ~keep]
    assert seen.isnan().all() if math.isnan(bad) else (seen == bad).all()
    assert _lib.device_status(clear=True) == 0


BAD = pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=["nan", "inf", "-inf"])


@BAD
@_leak_cases(_lib.PAGED_SIMT)
def test_values_that_a_token_does_not_see_never_reach_it_on_cuda_cores(dtype, heads, kv_heads, dim, lens, counts, bad):
    _no_leak(_lib.PAGED_SIMT, dtype, heads, kv_heads, dim, lens, counts, bad)


@BAD
@_leak_cases(_lib.PAGED_DECODE)
def test_values_that_a_token_does_not_see_never_reach_it_in_the_decode_kernel(dtype, heads, kv_heads, dim, lens, counts, bad):
    _no_leak(_lib.PAGED_DECODE, dtype, heads, kv_heads, dim, lens, counts, bad)


@BAD
@_leak_cases(_lib.PAGED_TC)
def test_values_that_a_token_does_not_see_never_reach_it_in_the_chunk_kernel(dtype, heads, kv_heads, dim, lens, counts, bad):
    _no_leak(_lib.PAGED_TC, dtype, heads, kv_heads, dim, lens, counts, bad)

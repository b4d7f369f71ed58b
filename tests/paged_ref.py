"""Plain float64 forms of the paged-cache operators, and batches to try them on (test infrastructure)."""

import math

import torch


def attention(q, k_pages, v_pages, table, lens, offsets, causal=True, scale=None, where="cpu"):
    """``(out, lse, spread, size)`` in float64 of a ragged batch, sequence by sequence; rows of no sequence are NaN.

    ``spread`` is ``sum_j p_ij |v_j|`` (what a relative error of the probabilities is multiplied by) and ``size`` is
    ``max_j scale sum_d |q_id k_jd|`` (what the relative error of a dot product is multiplied by)."""
    T, Hq, D = q.shape
    H, ps = k_pages.shape[1], k_pages.shape[2]
    G = Hq // H
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=where)
    lse = torch.full((Hq, T), math.nan, dtype=torch.float64, device=where)
    spread, size = out.clone(), torch.zeros(Hq, T, dtype=torch.float64, device=where)
    q, table = q.double().to(where), table.cpu()
    for b, n_all in enumerate(lens.tolist()):
        r0, r1 = int(offsets[b]), int(offsets[b + 1])
        n = r1 - r0
        if n == 0:
            continue
        pages = table[b, : -(-n_all // ps)].long()
        k = k_pages[pages.to(k_pages.device)].to(where).double().transpose(1, 2).reshape(-1, H, D)[:n_all]
        v = v_pages[pages.to(v_pages.device)].to(where).double().transpose(1, 2).reshape(-1, H, D)[:n_all]
        k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        s = torch.einsum("ihd,jhd->hij", q[r0:r1], k) * scale
        big = torch.einsum("ihd,jhd->hij", q[r0:r1].abs(), k.abs()) * abs(scale)
        if causal:
            at = torch.arange(n_all - n, n_all, device=where)
            hidden = torch.arange(n_all, device=where)[None, :] > at[:, None]
            s = s.masked_fill(hidden, -math.inf)
            big = big.masked_fill(hidden, 0.0)
        stat = torch.logsumexp(s, -1) if n_all else torch.full((Hq, n), -math.inf, dtype=torch.float64, device=where)
        p = torch.exp(s - stat.clamp(min=-1e300)[..., None])
        out[r0:r1] = torch.einsum("hij,jhd->ihd", p, v)
        spread[r0:r1] = torch.einsum("hij,jhd->ihd", p, v.abs())
        lse[:, r0:r1] = stat
        size[:, r0:r1] = big.amax(-1) if n_all else 0.0
    return out.cpu(), lse.cpu(), spread.cpu(), size.cpu()


def check(got, got_lse, ref, *, dtype, out_dtype, single_p):
    """Element by element against :func:`attention`'s answer.

    A dot product of D terms is off by at most ``D u size`` (u: 2^-23 for fp32 accumulation on tensor cores, which may
    cut where they do not round, and a rounding a term elsewhere), and the exponent's argument by two roundings of
    its own size more; the hardware's exp2 adds 2^-21.  So a probability is off by a relative ``e``, and as
    numerator and sum both carry it, the output by ``2 e spread``, the statistics by ``e``.  Where the kernel
    rounds the probabilities to the input type (``single_p``) that is half a step of it more, and the output's own
    rounding half a step of its type."""
    out, lse, spread, size = ref
    D = out.shape[-1]
    u = 2.0**-52 if dtype == torch.float64 else 2.0**-23
    e = (D + 2) * u * size + (2.0**-48 if dtype == torch.float64 else 2.0**-20) + 2 * u * size
    rows = ~out.isnan().all(-1).all(-1)
    p_err = (torch.finfo(dtype).eps / 2 if single_p else 0.0) + 2 * e.T[..., None]
    tol = p_err * spread + torch.finfo(out_dtype).eps / 2 * (out.abs() + p_err * spread) + 1e-300
    if out_dtype == torch.float16:
        tol = tol + 2.0**-25  # half a step of the smallest numbers
    d = (got.double().cpu() - out)[rows].abs()
    assert bool((d <= tol[rows]).all()), (float((d / tol[rows]).max()), float(d.max()))
    if got_lse is not None:
        g, w = got_lse.double().cpu()[:, rows], lse[:, rows]
        none = w.isinf()
        assert torch.equal(g[none], w[none])
        off = (g - w).abs()[~none]
        bound = (2 * e[:, rows] + 4 * u * w.abs().clamp(max=1e300))[~none]
        assert bool((off <= bound).all()), float((off / bound).max())


def batch(lens, counts, *, heads, kv_heads, dim, page, dtype, device, seed=0, spare=3, extra_rows=0, poison=True,
          layout="hsd"):
    """A ragged batch over a pool whose unused slots hold NaN and whose table is -1 behind each sequence's pages."""
    g = torch.Generator().manual_seed(seed)
    used = [-(-n // page) for n in lens]
    P = sum(used) + spare
    order = torch.randperm(P, generator=g)
    table = torch.full((len(lens), max(used + [0]) + 2), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at : at + n].int()
        at += n
    k, v = (torch.randn(P, kv_heads, page, dim, generator=g).to(dtype) for _ in range(2))
    if poison:
        full = torch.zeros(P, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(used[b]):
                full[table[b, i].long(), : min(page, n - i * page)] = True
        hole = ~full[:, None, :, None].expand_as(k)
        k, v = k.masked_fill(hole, math.nan), v.masked_fill(hole, math.nan)
    if layout == "shd":  # slots before heads in memory
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    offsets = torch.zeros(len(counts) + 1, dtype=torch.int32)
    offsets[1:] = torch.tensor(counts).cumsum(0)
    T = int(offsets[-1]) + extra_rows
    q = torch.randn(T, heads, dim, generator=g).to(dtype)
    return {"q": q.to(device), "k_pages": _same(k, device), "v_pages": _same(v, device), "page_table": table.to(device),
            "seq_lens": torch.tensor(lens, dtype=torch.int32).to(device), "q_offsets": offsets.to(device)}


def _same(x, device):
    """``x`` on ``device`` with the strides it has."""
    return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=device).copy_(x)

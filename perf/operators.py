"""Measured cases of the paged KV cache: attention of a ragged batch of new tokens over the pages, the write of their
keys and values into the pages, and the copy of pages between places of the pool.

Formulas, for sequence ``b`` with ``n_b`` new tokens (rows ``q_offsets[b] .. q_offsets[b + 1]`` of the flat token
axis) and ``len_b`` cached tokens, the new ones included; token ``p`` lives in page ``table[b, p // ps]``, slot
``p % ps``:

* attention: new token ``i`` is at position ``len_b - n_b + i`` and sees the keys at positions up to its own;
  ``out = softmax(scale q k^T) v``, ``lse = ln(sum exp(scale q k^T))``;
* append: new token ``i``'s key and value rows go to position ``len_b - n_b + i``;
* copy: page ``src[i]`` of every layer's keys and values goes to page ``dst[i]``.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _attend(name, dtype, seqs, len_lo, len_hi, n_lo, n_hi, *, chunks=0, chunk_n=0, heads=32, kv_heads=8, dim=128,
            page=16, lse=False):
    return {"name": name, "kind": "attend", "dtype": dtype, "seqs": seqs, "len_lo": len_lo, "len_hi": len_hi,
            "n_lo": n_lo, "n_hi": n_hi, "chunks": chunks, "chunk_n": chunk_n, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "lse": lse}


def listed():
    return [
        # the smallest call: one conversation's next token, where launches and latency count
        _attend("step_one", "bf16", 1, 1000, 1000, 1, 1),
        # one decoding step of a serving batch whose conversations differ in length
        _attend("step_batch", "bf16", 32, 1003, 32768, 1, 1),
        # a few proposed tokens a sequence, checked at once (multi-head attention of 64-wide heads)
        _attend("verify_few", "f16", 12, 301, 6000, 2, 5, heads=16, kv_heads=16, dim=64, page=32, lse=True),
        # the next piece of one long prompt
        _attend("chunk_short", "bf16", 1, 8700, 8700, 512, 512),
        # the largest: a big piece of a prompt far into its context
        _attend("chunk_long", "bf16", 1, 36864, 36864, 4096, 4096),
        # decoding sequences and pieces of prompts in one batch, statistics kept for a merge with other ranks
        _attend("mixed", "bf16", 18, 517, 6001, 1, 1, chunks=2, chunk_n=389, lse=True),
        # single-precision heads, as the parity configurations use them
        _attend("verify_f32", "f32", 4, 700, 2048, 1, 40, heads=8, kv_heads=8, dim=64, page=16, lse=True),
        # the keys and values of one decoding step
        {"name": "append_step", "kind": "append", "dtype": "bf16", "seqs": 64, "len_lo": 90, "len_hi": 1500,
         "n_lo": 1, "n_hi": 1, "kv_heads": 8, "dim": 128, "page": 16},
        # the keys and values of a ragged batch of prompts
        {"name": "append_prompts", "kind": "append", "dtype": "f16", "seqs": 9, "len_lo": 2500, "len_hi": 6000,
         "n_lo": 1701, "n_hi": 2500, "kv_heads": 8, "dim": 128, "page": 16},
        # conversations forked: the partly filled last page of each is copied in every layer
        {"name": "fork_tails", "kind": "copy", "dtype": "bf16", "layers": 32, "pages": 64, "pairs": 4, "kv_heads": 8,
         "dim": 128, "page": 16},
        # a pool compacted: pages from its end into holes before them
        {"name": "compact_pool", "kind": "copy", "dtype": "f16", "layers": 8, "pages": 1024, "pairs": 384,
         "kv_heads": 8, "dim": 128, "page": 16},
    ]


def _between(rng, lo, hi):
    """A whole number of the range, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "step", "few", "chunk", "chunk", "mixed", "f32", "append", "append", "copy"])
    if kind in ("append",):
        many = rng.random() < 0.5
        n_hi = _between(rng, 100, 2500) if many else rng.choice([1, 1, 4])
        n_lo = max(1, n_hi // 2) if many else 1
        len_hi = n_hi + _between(rng, 1, 3000)
        return {"kind": "append", "dtype": rng.choice(["bf16", "f16", "f32"]), "seqs": _between(rng, 1, 9 if many else 200),
                "len_lo": n_hi, "len_hi": len_hi, "n_lo": n_lo, "n_hi": n_hi, "kv_heads": rng.choice([1, 2, 5, 8]),
                "dim": rng.choice([64, 80, 128]), "page": rng.choice([8, 16, 32, 64])}
    if kind == "copy":
        pages = _between(rng, 40, 1024)
        return {"kind": "copy", "dtype": rng.choice(["bf16", "f16", "f32"]), "layers": _between(rng, 1, 8), "pages": pages,
                "pairs": _between(rng, 1, pages * 3 // 8), "kv_heads": rng.choice([1, 2, 5, 8]),
                "dim": rng.choice([64, 80, 128]), "page": rng.choice([8, 16])}
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 32, 128), (16, 2, 64), (24, 8, 128), (8, 1, 64), (16, 16, 64)])
    page, dtype, lse = rng.choice([8, 16, 32, 64, 128]), rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.5
    if kind == "step":
        hi = _between(rng, 40, 20000)
        c = _attend("", dtype, _between(rng, 1, 32), max(1, hi // _between(rng, 1, 30)), hi, 1, 1)
    elif kind == "few":
        hi = _between(rng, 100, 8000)
        c = _attend("", dtype, _between(rng, 1, 16), max(9, hi // 8), hi, 1, rng.randint(2, 9))
    elif kind == "chunk":
        n = _between(rng, 17, 2048)
        lo = n + _between(rng, 1, 16000)
        c = _attend("", dtype, 1 if n > 600 else rng.randint(1, 3), lo, lo + rng.randint(0, 300), n, n)
    elif kind == "mixed":
        n = _between(rng, 17, 400)
        c = _attend("", dtype, _between(rng, 2, 18), n, n + _between(rng, 100, 5600), 1, 1, chunks=rng.randint(1, 2), chunk_n=n)
    else:
        heads, kv_heads, dim = rng.choice([(8, 8, 64), (4, 2, 32), (8, 2, 80)])
        dtype, n = "f32", _between(rng, 1, 40)
        c = _attend("", dtype, _between(rng, 1, 4), n, n + _between(rng, 10, 2000), 1, n)
    c.pop("name")
    c.update(heads=heads, kv_heads=kv_heads, dim=dim, page=page, lse=lse)
    return c


def _spread(lo, hi, count, turn):
    """``count`` whole numbers spread over ``lo .. hi``, the first of them ``hi``."""
    return [hi - int((i * turn) % 1.0 * (hi - lo + 1)) for i in range(count)]


def _lengths(case):
    """Cached tokens and new tokens of every sequence: fixed by the case's own numbers."""
    total = _spread(case["len_lo"], case["len_hi"], case["seqs"], 0.6180339887)
    new = _spread(case["n_lo"], case["n_hi"], case["seqs"], 0.7548776662)
    for i in range(case.get("chunks", 0)):
        new[-1 - i] = case["chunk_n"] - i * (case["chunk_n"] // 3)
    return [max(t, n) for t, n in zip(total, new)], new


def work(case):
    size = _BYTES[case["dtype"]]
    if case["kind"] == "copy":
        page = case["kv_heads"] * case["dim"] * case["page"] * size
        return {"bytes": 2 * 2 * case["pairs"] * case["layers"] * page, "flops": 0}
    total, new = _lengths(case)
    row = case["kv_heads"] * case["dim"] * size
    if case["kind"] == "append":
        return {"bytes": 2 * 2 * sum(new) * row, "flops": 0}
    out_row = case["heads"] * case["dim"] * size
    seen = sum(n * (t - n) + n * (n + 1) // 2 for t, n in zip(total, new))
    nbytes = 2 * sum(total) * row + 2 * sum(new) * out_row + (4 * sum(new) * case["heads"] if case["lse"] else 0)
    return {"bytes": nbytes, "flops": 4 * case["dim"] * case["heads"] * seen}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)


def _normal(g, dtype, *shape):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    return x.normal_(generator=g)


def prepare(case, seed):
    dtype, g = _TYPES[case["dtype"]], _generator(seed)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "copy":
        shape = (case["layers"], case["pages"], heads, page, dim)
        order = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(int(seed)))
        src, dst = order[: case["pairs"]], order[case["pairs"] : 2 * case["pairs"]]
        return {"case": case, "k_pages": _normal(g, dtype, *shape), "v_pages": _normal(g, dtype, *shape),
                "src": src.to(torch.int32), "dst": dst.to(torch.int32)}
    total, new = _lengths(case)
    used = [-(-t // page) for t in total]
    pool = sum(used) + 7
    # the pages of a cache in use lie in no order; entries behind a sequence's last page are -1
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(int(seed)), dtype=torch.int64).to(torch.int32)
    table = torch.full((len(total), max(used) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at : at + n]
        at += n
    offsets = torch.zeros(len(new) + 1, dtype=torch.int32)
    offsets[1:] = torch.tensor(new, dtype=torch.int32).cumsum(0)
    tokens = sum(new)
    state = {"case": case, "k_pages": _normal(g, dtype, pool, heads, page, dim),
             "v_pages": _normal(g, dtype, pool, heads, page, dim), "table": table.cuda(),
             "lens": torch.tensor(total, dtype=torch.int32).cuda(), "offsets": offsets.cuda(), "n_max": max(new),
             "n_min": min(new), "len_max": max(total)}
    if case["kind"] == "append":
        # k and v are views of one projection's output, as a decoder layer makes them
        both = _normal(g, dtype, tokens, 2 * heads, dim)
        state.update(k=both[:, :heads], v=both[:, heads:])
        return state
    state["q"] = _normal(g, dtype, tokens, case["heads"], dim)
    state["out"] = torch.empty_like(state["q"])
    state["lse"] = torch.empty(case["heads"], tokens, dtype=torch.float32, device="cuda") if case["lse"] else None
    return state


def _positions(s):
    """For every row of the flat token axis: its sequence, its place among the sequence's new tokens, its position."""
    start, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    rows = torch.arange(s["tokens"], device=start.device)
    seq = torch.searchsorted(end, rows, right=True)
    place = rows - start[seq]
    return seq, place, s["lens"].long()[seq] - (end - start)[seq] + place


def _attend_plain(s):
    case, q = s["case"], s["q"]
    seq, place, position = _positions(dict(s, tokens=q.shape[0]))
    seqs, heads, dim, page = len(s["lens"]), case["kv_heads"], case["dim"], case["page"]
    group, most = case["heads"] // heads, s["len_max"]
    # every sequence's keys and values gathered to one padded tensor, [seqs, heads, most, dim]
    table = s["table"].long().clamp(min=0)[:, : -(-most // page)]
    k = s["k_pages"][table].float().transpose(1, 2).reshape(seqs, heads, -1, dim)[:, :, :most]
    v = s["v_pages"][table].float().transpose(1, 2).reshape(seqs, heads, -1, dim)[:, :, :most]
    slots = torch.arange(most, device=q.device)
    v = torch.where((slots < s["lens"].long()[:, None])[:, None, :, None], v, 0.0)
    padded = torch.zeros(seqs, s["n_max"], case["heads"], dim, device=q.device)
    padded[seq, place] = q.float()
    at = torch.full((seqs, s["n_max"]), -1, device=q.device)
    at[seq, place] = position
    padded = padded.view(seqs, s["n_max"], heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, heads, -1, dim)
    score = torch.matmul(padded, k.transpose(2, 3)).mul_(1.0 / math.sqrt(dim))
    hidden = (slots > at[:, :, None]).repeat_interleave(group, dim=1)
    score.masked_fill_(hidden[:, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / total.clamp(min=1e-30)
    out = out.view(seqs, heads, s["n_max"], group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, s["n_max"], -1, dim)
    out = out[seq, place].to(q.dtype)
    if not case["lse"]:
        return out
    lse = (top + total.log()).view(seqs, heads, s["n_max"], group).permute(1, 3, 0, 2).reshape(case["heads"], seqs, -1)
    return out, lse[:, seq, place]


def _append_plain(s):
    seq, _, position = _positions(dict(s, tokens=s["k"].shape[0]))
    page = s["case"]["page"]
    to = s["table"].long()[seq, position // page]
    s["k_pages"][to, :, position % page] = s["k"]
    s["v_pages"][to, :, position % page] = s["v"]
    return s["k_pages"], s["v_pages"]


def _copy_plain(s):
    src, dst = s["src"].long().cuda(), s["dst"].long().cuda()
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    return s["k_pages"], s["v_pages"]


def _run_own(s):
    import collaborative_edge_system_b200 as cea

    kind = s["case"]["kind"]
    if kind == "copy":
        cea.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
        return s["k_pages"], s["v_pages"]
    if kind == "append":
        cea.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["offsets"])
        return s["k_pages"], s["v_pages"]
    cea.paged_attend_into(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["offsets"], s["out"], s["lse"],
                          min_q_len=s["n_min"], max_q_len=s["n_max"])
    return (s["out"], s["lse"]) if s["lse"] is not None else s["out"]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "attend":
        return _attend_plain(state)
    return _append_plain(state) if kind == "append" else _copy_plain(state)


def exact(case, seed):
    s = prepare(case, seed)
    page = case["page"]
    if case["kind"] == "copy":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            k[:, b], v[:, b] = k[:, a].clone(), v[:, a].clone()
        return k, v
    total, new = _lengths(case)
    table = s["table"].cpu()
    if case["kind"] == "append":
        k, v, row = s["k_pages"].double(), s["v_pages"].double(), 0
        for b, (t, n) in enumerate(zip(total, new)):
            p = torch.arange(t - n, t)
            to, slot = table[b][p // page].long().cuda(), (p % page).cuda()
            k[to, :, slot] = s["k"][row : row + n].double()
            v[to, :, slot] = s["v"][row : row + n].double()
            row += n
        return k, v
    heads, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // heads
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(case["heads"], s["q"].shape[0], dtype=torch.float64, device="cuda")
    row = 0
    for b, (t, n) in enumerate(zip(total, new)):
        pages = table[b, : -(-t // page)].long().cuda()
        limit = torch.arange(t - n, t, device="cuda").repeat_interleave(group)[:, None]
        unseen = torch.arange(t, device="cuda")[None, :] > limit
        for h in range(heads):
            keys = s["k_pages"][pages, h].reshape(-1, dim)[:t].double()
            values = s["v_pages"][pages, h].reshape(-1, dim)[:t].double()
            q = s["q"][row : row + n, h * group : (h + 1) * group].double().reshape(-1, dim)
            score = (q @ keys.T / math.sqrt(dim)).masked_fill(unseen, -math.inf)
            stat = torch.logsumexp(score, -1)
            got = torch.exp(score - stat[:, None]) @ values
            out[row : row + n, h * group : (h + 1) * group] = got.view(n, group, dim)
            lse[h * group : (h + 1) * group, row : row + n] = stat.view(n, group).T
        row += n
    return (out, lse) if case["lse"] else out

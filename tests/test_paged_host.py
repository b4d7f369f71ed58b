"""The paged KV cache's host side on the CPU: page accounting, batch descriptions, argument checks."""

import ctypes
import random

import pytest
import torch

import collaborative_edge_system_b200 as cea
from collaborative_edge_system_b200 import _lib, paged

CPU = torch.device("cpu")


class HostCache(paged.PagedKVCache):
    """The cache with its buffers on the CPU and page copies by indexing, to drive its accounting without a GPU."""

    def __init__(self, layers, pages, page_size, heads, dim):
        super().__init__(layers, pages, page_size, heads, dim, dtype=torch.float32, device=torch.device("cuda"))

    def _make_buffers(self, shape, dtype, device):
        self.k, self.v = torch.zeros(shape), torch.zeros(shape)
        self.device = CPU

    def _copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.k[:, dst], self.v[:, dst] = self.k[:, src], self.v[:, src]

    def write(self, seq, values, batch, b):
        """``values`` into the last places of row ``b`` of the batch, in every layer's K."""
        n = int(batch.seq_lens[b])
        for i, x in enumerate(values):
            p = n - len(values) + i
            self.k[:, int(batch.page_table[b, p // self.page_size]), :, p % self.page_size] = x

    def read(self, seq):
        n = self.length(seq)
        return [float(self.k[0, self.pages(seq)[p // self.page_size], 0, p % self.page_size, 0]) for p in range(n)]


def test_allocator_counts_references():
    a = cea.PageAllocator(4)
    assert a.alloc(2) == [0, 1] and a.num_free == 2
    a.share([1])
    a.release([0, 1])
    assert a.num_free == 3 and a.refs == [0, 1, 0, 0]
    with pytest.raises(cea.OutOfPages):
        a.alloc(4)
    assert a.num_free == 3
    assert a.alloc(3) == [0, 2, 3]
    a.release([1])
    with pytest.raises(ValueError):
        a.release([1])
    with pytest.raises(ValueError):
        a.share([1])
    assert a.compaction() == ([3], [1])
    a.move([3], [1])
    assert a.refs == [1, 1, 1, 0] and a.alloc(1) == [3]
    with pytest.raises(ValueError):
        cea.PageAllocator(-1)


@pytest.mark.parametrize("seed", range(6))
def test_random_operations_never_mix_sequences(seed):
    rnd = random.Random(seed)
    cache = HostCache(2, 40, rnd.choice([1, 3, 4]), 1, 2)
    want, stamp = {}, 0.0
    for _ in range(300):
        ids = sorted(want)
        move = rnd.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        if move == "add" or not ids:
            want[cache.add()] = []
        elif move == "extend":
            some = rnd.sample(ids, rnd.randint(1, len(ids)))
            counts = [rnd.randint(0, 5) for _ in some]
            state = (cache.num_free_pages, list(cache.pool.refs), {s: cache.pages(s) for s in ids})
            try:
                batch = cache.extend(some, counts)
            except cea.OutOfPages:
                assert state == (cache.num_free_pages, list(cache.pool.refs), {s: cache.pages(s) for s in ids})
                continue
            for b, (s, c) in enumerate(zip(some, counts)):
                new = [stamp + i for i in range(1, c + 1)]
                stamp += c
                cache.write(s, new, batch, b)
                want[s] = want[s] + new
        elif move == "fork":
            s = rnd.choice(ids)
            n = rnd.randint(0, len(want[s]))
            try:
                for f in cache.fork(s, n, rnd.randint(0, 3)):
                    want[f] = want[s][:n]
            except cea.OutOfPages:
                pass
        elif move == "truncate":
            s = rnd.choice(ids)
            n = rnd.randint(0, len(want[s]))
            cache.truncate(s, n)
            want[s] = want[s][:n]
        elif move == "free":
            s = rnd.choice(ids)
            cache.free(s)
            del want[s]
        else:
            used = cache.compact()
            assert all(p < used for s in ids for p in cache.pages(s))
        counted = [0] * 40
        for s in want:
            assert cache.read(s) == want[s]
            for p in cache.pages(s):
                counted[p] += 1
        assert counted == cache.pool.refs and cache.num_free_pages == counted.count(0)


def test_batch_description():
    b = cea.PagedBatch([[3, 1], [], [2]], [5, 0, 4], [2, 0, 4], CPU)
    assert b.page_table.tolist() == [[3, 1], [-1, -1], [2, -1]] and b.page_table.dtype == torch.int32
    assert b.seq_lens.tolist() == [5, 0, 4] and b.q_offsets.tolist() == [0, 2, 2, 6]
    assert b.positions.tolist() == [3, 4, 0, 1, 2, 3] and b.positions.dtype == torch.int64
    assert (b.num_tokens, b.min_q_len, b.max_q_len, b.last_rows) == (6, 2, 4, [1, 1, 5])
    e = cea.PagedBatch([], [], [], CPU)
    assert e.num_tokens == 0 and e.q_offsets.tolist() == [0] and e.max_q_len == 0


def test_cache_refuses_what_it_cannot_do():
    c = HostCache(1, 4, 4, 1, 1)
    s = c.add()
    c.extend([s], [6])
    for bad in (lambda: c.length(9), lambda: c.fork(s, 7), lambda: c.fork(s, -1), lambda: c.fork(s, 2, -1),
                lambda: c.truncate(s, 7), lambda: c.extend([s, s], [1, 1]), lambda: c.extend([s], [-1]),
                lambda: c.extend([s], [1, 2]), lambda: c.free(3)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(cea.OutOfPages):
        c.extend([s], [11])
    assert c.length(s) == 6 and c.num_free_pages == 2
    c.extend([s], [10])
    assert c.num_free_pages == 0
    with pytest.raises(ValueError):
        cea.PagedKVCache(1, 4, 4, 1, 1, device=CPU)
    with pytest.raises(ValueError):
        cea.PagedKVCache(1, 4, 0, 1, 1, device=torch.device("cuda"))


def test_operators_refuse_cpu_tensors():
    k, t, n, o = torch.zeros(2, 1, 4, 8), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor(
        [0, 1], dtype=torch.int32)
    x = torch.zeros(1, 1, 8)
    with pytest.raises(ValueError, match="CUDA"):
        cea.paged_append(x, x, k, k, t, n, o)
    with pytest.raises(ValueError, match="CUDA"):
        cea.paged_attention(x, k, k, t, n, o)
    with pytest.raises(ValueError, match="CUDA"):
        cea.copy_pages(k, k, [0], [1])


@pytest.fixture
def anywhere(monkeypatch):
    """Checks that come before the kernels, on CPU tensors: what they let pass ends in ``reached``."""
    reached = []
    monkeypatch.setattr(_lib, "device_number", lambda *t: 0)
    for name in ("paged_attn", "paged_append", "copy_pages"):
        monkeypatch.setattr(_lib, name, lambda p, dev: reached.append(p))
    return reached


def _good():
    return {"q": torch.zeros(3, 4, 8), "k_pages": torch.zeros(5, 2, 4, 8), "v_pages": torch.zeros(5, 2, 4, 8),
            "page_table": torch.zeros(2, 3, dtype=torch.int32), "seq_lens": torch.ones(2, dtype=torch.int32),
            "q_offsets": torch.tensor([0, 1, 3], dtype=torch.int32)}


def test_attention_arguments(anywhere):
    cea.paged_attention(**_good())
    p = anywhere.pop()
    assert (p.B, p.T, p.Hq, p.Hkv, p.D, p.page_size, p.num_pages, p.max_pages, p.min_q_len, p.max_q_len) == (
        2, 3, 4, 2, 8, 4, 5, 3, 0, 3)
    assert list(p.k_stride) == [64, 32, 8] and p.table_stride == 3 and p.lse is None
    bad = [("q", torch.zeros(3, 4, 16)), ("q", torch.zeros(3, 4, 8).half()), ("q", torch.zeros(1, 3, 4, 8)),
           ("q", torch.zeros(3, 4, 16)[..., ::2]), ("k_pages", torch.zeros(5, 2, 4, 16)), ("v_pages", torch.zeros(4, 2, 4, 8)),
           ("v_pages", torch.zeros(5, 2, 4, 8).half()), ("page_table", torch.zeros(2, 3, dtype=torch.int64)),
           ("page_table", torch.zeros(3, 3, dtype=torch.int32)), ("seq_lens", torch.ones(2)),
           ("q_offsets", torch.zeros(2, dtype=torch.int32)), ("q_offsets", torch.zeros(6, dtype=torch.int32)[::2]),
           ("page_table", torch.zeros(2, 6, dtype=torch.int32)[:, ::2])]
    for name, value in bad:
        with pytest.raises(ValueError):
            cea.paged_attention(**{**_good(), name: value})
    x, out = _good(), torch.zeros(3, 4, 8)
    for o, l in ((torch.zeros(2, 4, 8), None), (out, torch.zeros(4, 2)), (out, torch.zeros(4, 3).half()),
                 (torch.zeros(3, 4, 16)[..., ::2], None)):
        with pytest.raises(ValueError):
            cea.paged_attend_into(**x, out=o, lse=l)
    with pytest.raises(TypeError):
        cea.paged_attend_into(**{n: t.int() if n in ("q", "k_pages", "v_pages") else t for n, t in x.items()},
                              out=out)
    assert not anywhere


def test_promise_of_the_least_number_holds_for_an_empty_pass(anywhere):
    x = _good()
    x["q"], x["q_offsets"] = x["q"][:0], torch.zeros(3, dtype=torch.int32)
    cea.paged_attention(**x, min_q_len=1)  # says nothing of sequences without new tokens
    p = anywhere.pop()
    assert p.T == 0 and p.min_q_len <= p.max_q_len


def test_append_arguments(anywhere):
    x = _good()
    x.pop("q")
    k = torch.zeros(3, 2, 8)
    cea.paged_append(k, k, **x)
    p = anywhere.pop()
    assert (p.B, p.T, p.H, p.D, p.elem_bytes) == (2, 3, 2, 8, 4) and list(p.k_stride) == [16, 8]
    for a, b in ((k[:2], k), (k[:, :1], k[:, :1]), (k.half(), k.half()), (torch.zeros(3, 2, 16)[..., ::2],) * 2,
                 (k[None], k[None])):
        with pytest.raises(ValueError):
            cea.paged_append(a, b, **x)
    assert not anywhere


def test_copy_arguments(anywhere):
    k = torch.zeros(3, 5, 2, 4, 8)
    cea.copy_pages(k, k.clone(), [0, 1], torch.tensor([2, 3]))
    p = anywhere.pop()
    assert (p.n, p.layers, p.num_pages, p.page_bytes) == (2, 3, 5, 256) and list(p.k_stride) == [5 * 256, 256]
    for args in ((k, k[:2], [0], [1]), (k, k, [0], [1, 2]), (k, k, [2**31], [1]), (k, k, torch.tensor([0.0]), [1]),
                 (k[..., ::2], k[..., ::2], [0], [1]), (k.expand(2, 3, 5, 2, 4, 8), k, [0], [1]),
                 (k[:, :1].expand(3, 5, 2, 4, 8),) * 2 + ([0], [1])):
        with pytest.raises(ValueError):
            cea.copy_pages(*args)
    assert not anywhere


def test_fractions_are_refused(anywhere):
    k = torch.zeros(3, 5, 2, 4, 8)
    with pytest.raises(TypeError):
        cea.copy_pages(k, k, [0.5], [1])
    c = HostCache(1, 4, 4, 1, 2)
    s = c.add()
    c.extend([s], [3])
    for call in (lambda: c.extend([s], [1.5]), lambda: c.fork(s, 2.5), lambda: c.truncate(s, 2.5)):
        with pytest.raises(TypeError):
            call()
    assert c.length(s) == 3 and c.num_free_pages == 3 and not anywhere


# ------------------------------------------------------------------------------------------------ C ABI
def test_records_have_the_layout_of_the_structs():
    for record, cls in ((_lib.PAGED_ATTN_RECORD, _lib.PagedAttnParams), (_lib.PAGED_APPEND_RECORD, _lib.PagedAppendParams)):
        flat, p = [], cls()
        for name, kind in cls._fields_[:-2] if cls is _lib.PagedAttnParams else cls._fields_:
            if hasattr(kind, "_length_"):
                values = [len(flat) + 1 + i for i in range(kind._length_)]
                setattr(p, name, tuple(values))
            else:
                values = [float(len(flat) + 1) if kind is ctypes.c_double else len(flat) + 1]
                setattr(p, name, values[0])
            flat += values
        packed = record.pack(*flat)
        assert bytes(p)[: len(packed)] == packed and ctypes.sizeof(cls) - len(packed) in (0, 16, 20)
        assert not any(bytes(p)[len(packed):])


FAKE = 1 << 20  # never dereferenced: every check here returns before any CUDA call


def _attn():
    p = _lib.PagedAttnParams()
    p.q = p.k_pages = p.v_pages = p.out = p.q_offsets = p.seq_lens = p.page_table = FAKE
    p.B, p.T, p.Hq, p.Hkv, p.D, p.page_size, p.num_pages, p.max_pages, p.max_q_len = 2, 3, 8, 2, 128, 16, 10, 4, 1
    p.q_stride, p.o_stride = (8 * 128, 128), (8 * 128, 128)
    p.k_stride = p.v_stride = (2 * 16 * 128, 16 * 128, 128)
    p.scale, p.causal, p.in_dtype, p.out_dtype = 0.1, 1, _lib.BF16, _lib.BF16
    return p


def test_attention_checks_of_the_c_abi():
    lib = _lib.load()

    def run(**kw):
        p = _attn()
        for n, v in kw.items():
            setattr(p, n, v)
        return lib.cea_paged_attn(ctypes.byref(p), None)

    assert lib.cea_paged_attn(None, None) == _lib.CEA_ERR_INVALID
    for kw in ({"Hq": 3}, {"Hkv": 0}, {"D": 0}, {"page_size": 0}, {"B": -1}, {"T": -1}, {"q": None}, {"out": None},
               {"k_pages": None}, {"q_offsets": None}, {"page_table": None}, {"seq_lens": None}, {"in_dtype": 9},
               {"min_q_len": 2}, {"min_q_len": -1}, {"max_q_len": -1}, {"scale": float("nan")}, {"scale": float("inf")}, {"num_pages": -1}):
        assert run(**kw) == _lib.CEA_ERR_INVALID, kw
    for kw in ({"D": 257}, {"out_dtype": _lib.F16}, {"in_dtype": _lib.F64, "out_dtype": _lib.F32}):
        assert run(**kw) == _lib.CEA_ERR_UNSUPPORTED, kw
    assert run() == _lib.CEA_ERR_WORKSPACE and b"workspace" in lib.cea_last_error()
    for kw in ({"B": 0}, {"T": 0}, {"Hq": 0}, {"max_q_len": 0}):  # nothing to do, nothing to launch
        assert run(**kw, q=None, out=None) == _lib.CEA_OK, kw


def test_choice_of_kernels():
    lib = _lib.load()

    def mask(**kw):
        p = _attn()
        for n, v in kw.items():
            setattr(p, n, v)
        return lib.cea_paged_attn_kernels(ctypes.byref(p))

    assert mask() == _lib.PAGED_DECODE and mask(max_q_len=4) == _lib.PAGED_DECODE  # 4 query heads share a KV head
    assert mask(max_q_len=5) == _lib.PAGED_DECODE | _lib.PAGED_TC and mask(min_q_len=5, max_q_len=5) == _lib.PAGED_TC
    assert mask(q=FAKE + 8, max_q_len=5) == _lib.PAGED_SIMT and mask(q=FAKE + 8) == _lib.PAGED_DECODE
    assert mask(Hq=2 * 64, out=FAKE + 2) == _lib.PAGED_SIMT and mask(Hq=2 * 64) == _lib.PAGED_TC
    for kw in ({"in_dtype": _lib.F32, "out_dtype": _lib.F32}, {"D": 80}, {"page_size": 12}, {"k_pages": FAKE + 2},
               {"v_stride": (2 * 16 * 128, 16 * 128, 132)}, {"num_pages": 0}):
        assert mask(**kw) == _lib.PAGED_SIMT, kw
    assert mask(scale=-1.0) == _lib.PAGED_DECODE and mask(scale=0.0, max_q_len=5) == _lib.PAGED_SIMT
    assert mask(max_q_len=3) == _lib.PAGED_DECODE and mask(min_q_len=3, max_q_len=5) == _lib.PAGED_TC
    # 9 to 16 rows: the chunk kernel at 128 columns if no sequence may have fewer, as it wins there
    assert mask(min_q_len=3, max_q_len=4) == _lib.PAGED_TC and mask(min_q_len=2, max_q_len=4) == _lib.PAGED_DECODE
    assert mask(min_q_len=3, max_q_len=4, scale=-1.0) == _lib.PAGED_DECODE
    assert mask(Hq=32, max_q_len=1) == _lib.PAGED_TC and mask(Hq=32, max_q_len=2) == _lib.PAGED_TC
    assert mask(Hq=32, max_q_len=1, scale=-1.0) == _lib.PAGED_DECODE
    narrow = {"D": 64, "k_stride": (2 * 16 * 64, 16 * 64, 64), "v_stride": (2 * 16 * 64, 16 * 64, 64)}
    assert mask(min_q_len=3, max_q_len=4, **narrow) == _lib.PAGED_DECODE
    assert mask(Hq=32, max_q_len=2, **narrow) == _lib.PAGED_DECODE | _lib.PAGED_TC
    assert mask(T=0) == 0 and mask(D=0) == -1


def test_append_and_copy_checks_of_the_c_abi():
    lib = _lib.load()
    assert lib.cea_paged_append(None, None) == _lib.CEA_ERR_INVALID
    a = _lib.PagedAppendParams()
    a.B, a.T, a.H, a.D, a.page_size, a.num_pages, a.max_pages, a.elem_bytes = 1, 2, 2, 8, 4, 3, 2, 2
    assert lib.cea_paged_append(ctypes.byref(a), None) == _lib.CEA_ERR_INVALID  # null table
    a.q_offsets = a.seq_lens = a.page_table = FAKE
    assert lib.cea_paged_append(ctypes.byref(a), None) == _lib.CEA_ERR_INVALID  # null k
    a.k = a.v = a.k_pages = a.v_pages = FAKE
    a.elem_bytes = 3
    assert lib.cea_paged_append(ctypes.byref(a), None) == _lib.CEA_ERR_INVALID
    a.elem_bytes, a.T = 2, 0
    assert lib.cea_paged_append(ctypes.byref(a), None) == _lib.CEA_OK

    assert lib.cea_copy_pages(None, None) == _lib.CEA_ERR_INVALID

    def copy(src, dst, pages=6, n=None):
        c = _lib.CopyPagesParams()
        s, d = (ctypes.c_int32 * len(src))(*src), (ctypes.c_int32 * len(dst))(*dst)
        c.src, c.dst = ctypes.addressof(s), ctypes.addressof(d)
        c.n, c.layers, c.num_pages, c.page_bytes = len(src) if n is None else n, 0, pages, 64
        return lib.cea_copy_pages(ctypes.byref(c), None)

    assert copy([0, 0, 1], [2, 3, 4]) == _lib.CEA_OK  # no layers: checked, nothing launched
    for src, dst in (([0], [6]), ([6], [0]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([1], [1])):
        assert copy(src, dst) == _lib.CEA_ERR_INVALID, (src, dst)
    assert copy([0], [1], n=-1) == _lib.CEA_ERR_INVALID


def test_calls_run_with_their_tensors_device_current(monkeypatch):
    seen, current = [], [0]

    class Device:
        def __init__(self, n):
            self.n = n

        def __enter__(self):
            self.before, current[0] = current[0], self.n

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda n: 1000 + n, raising=False)
    p = _lib.CopyPagesParams()
    for device in (0, 3):
        _lib._on_device(lambda ref, stream: seen.append((current[0], stream)) or 0, p, device, "call")
    assert seen == [(0, 1000), (3, 1003)] and current == [0]
    with pytest.raises(RuntimeError, match="call"):
        _lib._on_device(lambda ref, stream: _lib.CEA_ERR_CUDA, p, 3, "call")
    assert current == [0]


# ------------------------------------------------------------------------------------------------ generation
class SumModel:
    """Stands for a model: the next token is the sum of the sequence's tokens (read from the cache) modulo 17."""

    device = CPU

    def __init__(self):
        self.passes = []

    def paged_cache(self, num_pages, page_size):
        self.cache = HostCache(1, num_pages, page_size, 1, 1)
        return self.cache

    def forward_paged(self, ids, batch, cache):
        self.passes.append(batch.num_tokens)
        out, ps = [], cache.page_size
        for b in range(len(batch.seq_lens)):
            n, r0, r1 = int(batch.seq_lens[b]), int(batch.q_offsets[b]), int(batch.q_offsets[b + 1])
            at = lambda p: (0, int(batch.page_table[b, p // ps]), 0, p % ps, 0)  # noqa: E731
            for i in range(r0, r1):
                assert int(batch.positions[i]) == n - r1 + i
                cache.k[at(n - r1 + i)] = float(ids[i])
                out.append(sum(float(cache.k[at(p)]) for p in range(n - r1 + i + 1)))
        return torch.tensor(out).view(-1, 1)

    def logits(self, hidden):
        return torch.nn.functional.one_hot(hidden[:, 0].long() % 17, 17).float()


@pytest.mark.parametrize("seed", range(8))
def test_generation_schedules_every_token_once(seed):
    from collaborative_edge_system_b200.llama import generate_paged

    rnd = random.Random(seed)
    prefix = [rnd.randrange(17) for _ in range(rnd.choice([0, 0, 3, 8, 11]))]
    prompts = [[rnd.randrange(17) for _ in range(rnd.randint(0 if prefix else 1, 12))] for _ in range(rnd.randint(1, 7))]
    most, eos, chunk = rnd.randint(1, 9), rnd.choice([None, 3, 5]), rnd.choice([1, 2, 5, 64])
    want = []
    for p in prompts:
        seq, new = prefix + p, []
        while len(new) < most and (not new or new[-1] != eos):
            new.append(sum(seq) % 17)
            seq = seq + new[-1:]
        want.append(new)
    model = SumModel()
    got, scores = generate_paged(model, prompts, most, prefix=prefix, page_size=4, chunk_tokens=chunk, eos_token_id=eos,
                                 return_scores=True)
    assert got == want and [s.argmax(-1).tolist() for s in scores] == want
    assert max(model.passes) <= chunk
    assert sum(model.passes) == len(prefix) + sum(len(p) + len(w) - 1 for p, w in zip(prompts, want))
    assert model.cache.num_free_pages == len(model.cache.pool.refs)


def test_generation_refusals_leave_the_cache_as_it_was():
    from collaborative_edge_system_b200.llama import generate_paged

    model = SumModel()
    cache = model.paged_cache(4, 4)
    mine = cache.add()
    cache.extend([mine], [5])
    with pytest.raises(ValueError):
        generate_paged(model, [[1], []], 2)
    with pytest.raises(ValueError):
        generate_paged(model, [[1]], 2, chunk_tokens=0)
    with pytest.raises(cea.OutOfPages):
        generate_paged(model, [[1] * 6, [2] * 3], 2, cache=cache)
    assert cache.num_free_pages == 2 and cache.length(mine) == 5
    assert generate_paged(model, [[1, 2]], 0) == [[]]
    assert generate_paged(model, [[1, 2]], 3, cache=cache) == [[3, 6, 12]] and cache.num_free_pages == 2

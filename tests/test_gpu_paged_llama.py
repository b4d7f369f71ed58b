"""The paged cache under the LLaMA path on the GPU: generation over pages against the reference engine's float64 logits
and tokens, and against the dense cache."""

import json

import numpy as np
import pytest
import torch

import collaborative_edge_system_b200 as cea
from collaborative_edge_system_b200 import _lib
from collaborative_edge_system_b200.llama import LlamaConfig, LlamaModel, forward_logits, generate_greedy, generate_paged

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None


def _golden_model(gold):
    cfg = LlamaConfig.from_dict(json.loads(str(gold["config"])))
    sd = {k[len("weights/"):]: torch.from_numpy(v) for k, v in gold.items() if k.startswith("weights/")}
    return LlamaModel.from_state_dict(cfg, sd, dtype=torch.float64, device=DEV)


@pytest.mark.parametrize("name", ["sp1", "sp1_eos"])
@pytest.mark.parametrize("page,chunk", [(16, 2048), (4, 5), (3, 1), (1, 7)])
def test_generation_over_pages_matches_reference_engine(golden_llama, name, page, chunk):
    model = _golden_model(golden_llama)
    prompts = json.loads(str(golden_llama["prompts"]))
    gen = json.loads(str(golden_llama[f"{name}/meta"])).get("generate", {})
    tokens, scores = generate_paged(model, prompts, int(golden_llama["new_tokens"]), page_size=page, chunk_tokens=chunk,
                                    return_scores=True, **gen)
    assert tokens == json.loads(str(golden_llama[f"{name}/tokens"]))
    for b in range(len(prompts)):
        assert np.abs(scores[b].cpu().numpy() - golden_llama[f"{name}/scores{b}"]).max() < 1e-10
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize("page", [4, 5])
def test_shared_prefix_gives_the_results_of_whole_prompts(golden_llama, page):
    model = _golden_model(golden_llama)
    comm = cea.ParallelContext(1, 1, 1, device=DEV).sp
    prefix = [3, 14, 15, 92, 65, 35, 89, 79, 32, 38, 46]
    rest = [[5, 9, 2], [42], [70, 71, 1, 2, 3, 4, 5, 6], []]
    want, want_s = generate_greedy(model, [prefix + r for r in rest], 5, comm, return_scores=True)
    cache = model.paged_cache(40, page)
    got, got_s = generate_paged(model, rest, 5, prefix=prefix, cache=cache, chunk_tokens=6, return_scores=True)
    assert got == want and cache.num_free_pages == 40
    for a, b in zip(got_s, want_s):
        assert (a - b).abs().max() < 1e-10


def test_mixed_batches_in_bf16_at_wide_heads():
    """Two layers at 32 / 8 heads of 128 in bf16: logits of prompts taken in pieces, with decoding sequences beside
    them, stay as near to the float32 model's as the whole prompts' do on the dense path."""
    cfg = LlamaConfig.llama3_8b(num_layers=2, vocab_size=2048, intermediate_size=1024)
    m32 = LlamaModel.random(cfg, seed=1, dtype=torch.float32, device=DEV)
    m16 = LlamaModel.random(cfg, seed=1, dtype=torch.bfloat16, device=DEV)
    comm = cea.ParallelContext(1, 1, 1, device=DEV).sp
    g = torch.Generator().manual_seed(0)
    lens = [300, 45, 1, 130]
    ids = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in lens]
    cache = m16.paged_cache(64, 16)
    seqs = [cache.add() for _ in lens]
    got = [[] for _ in lens]
    with torch.no_grad():
        want = [forward_logits(m32, x[None], None, comm)[0] for x in ids]
        dense = [forward_logits(m16, x[None], None, comm)[0] for x in ids]
        at = [0] * len(lens)
        for counts in ([100, 1, 0, 1], [1, 20, 1, 1], [150, 1, 0, 90], [1, 22, 0, 30], [48, 1, 0, 8]):
            batch = cache.extend(seqs, counts)
            flat = torch.cat([x[a : a + c] for x, a, c in zip(ids, at, counts)]).to(DEV)
            logits = m16.logits(m16.forward_paged(flat, batch, cache))
            for b, part in enumerate(logits.split(counts)):
                got[b].append(part)
            at = [a + c for a, c in zip(at, counts)]
    assert at == lens
    for g_, d, w in zip(got, dense, want):
        near = float((torch.cat(g_).float() - w).norm() / w.norm())
        assert near < 5e-2 and near < 1.2 * float((d.float() - w).norm() / w.norm()) + 1e-3
    with pytest.raises(ValueError):
        m16.forward_paged(flat[:-1], batch, cache)
    assert _lib.device_status(clear=True) == 0

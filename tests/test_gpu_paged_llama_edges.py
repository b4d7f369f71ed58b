"""Passes of the LLaMA path over the paged cache that have no tokens."""

import json

import pytest
import torch

from collaborative_edge_system_b200 import _lib
from collaborative_edge_system_b200.llama import LlamaConfig, LlamaModel

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]
DEV = torch.device("cuda", 0) if torch.cuda.is_available() else None


def test_pass_without_new_tokens(golden_llama):
    cfg = LlamaConfig.from_dict(json.loads(str(golden_llama["config"])))
    model = LlamaModel.random(cfg, dtype=torch.bfloat16, device=DEV)
    cache = model.paged_cache(4, 4)
    seqs = [cache.add(), cache.add()]
    ids = torch.tensor([3, 1, 4], device=DEV)
    first = model.forward_paged(ids, cache.extend(seqs, [3, 0]), cache)
    k = cache.k[:, cache.pages(seqs[0])].clone()
    for some, counts in ((seqs, [0, 0]), ([], [])):
        hidden = model.forward_paged(ids[:0], cache.extend(some, counts), cache)
        assert hidden.shape == (0, first.shape[1]) and hidden.dtype == first.dtype and hidden.device == first.device
    assert torch.equal(cache.k[:, cache.pages(seqs[0])].nan_to_num(), k.nan_to_num())
    assert [cache.length(s) for s in seqs] == [3, 0]
    assert _lib.device_status(clear=True) == 0

"""GPU: the LM's serving paths at the edges."""
import pytest
import torch

from flashmhf_b200 import lm
from tests.test_lm_serving_gpu import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
def test_ids_of_empty_places_may_be_anything(captured):
    cfg, m = _model()
    prompt, out = torch.arange(20, device="cuda"), []
    for filler in (0, -1, 300, 2**40):
        cache = lm.PagedKVCache(cfg, 3, 9, page_size=16, max_len=64)
        m.prefill_paged({1: prompt}, cache)
        ids = torch.tensor([filler, 5, filler], device="cuda")
        if captured:
            m.decode_step_paged(torch.zeros_like(ids), cache)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                logits = m.decode_step_paged(ids, cache)
            cache.reserve(1)
            graph.replay()
            cache.advance(1)
        else:
            logits = m.decode_step_paged(ids, cache)
        torch.cuda.synchronize()
        assert cache.lengths.tolist() == cache.held and bool(logits.isfinite().all())
        out.append(logits[1].clone())
    assert all(torch.equal(x, out[0]) for x in out)

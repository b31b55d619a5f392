"""CPU: who owns which page of a PagedKVCache, and what the serving calls of the LM refuse."""
import pytest
import torch

from flashmhf_b200 import lm

CFG = lm.LMConfig(vocab_size=50, hidden_size=128, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1, intermediate_size=128,
                  mhffnmoe_num_heads=2, mhffnmoe_num_kuv_heads=2, mhffnmoe_num_experts=2)


def _begin(cache, b, n):
    counts = [0] * len(cache.held)
    counts[b] = n
    cache.reserve(counts)
    cache.held[b] = 0
    cache.advance(counts)


def test_pages_are_handed_out_and_come_back():
    c = lm.PagedKVCache(CFG, 3, 6, page_size=16, max_len=64, device="cpu")
    assert c.table.shape == (3, 4) and c.cos.shape == (64, 32) and c.lengths.tolist() == [-1] * 3 and c.nbytes() == 0
    _begin(c, 0, 17)
    _begin(c, 2, 16)
    assert [len(o) for o in c.owned] == [2, 0, 1] and len(c.free) == 3
    assert c.table[0, :2].tolist() == c.owned[0] and c.table[2, 0] == c.owned[2][0]
    c.reserve(1)                       # sequence 2 needs its second page, 0 has room, 1 is none
    c.advance(1)
    assert c.held == [18, -1, 17] and [len(o) for o in c.owned] == [2, 0, 2]
    assert c.nbytes() == 2 * 2 * 1 * ((18 + 17) * 64 + 4 * 4)
    assert len(set(sum(c.owned, []) + c.free)) == 6
    with pytest.raises(RuntimeError, match="free pages"):
        c.reserve([0, 33, 0])
    with pytest.raises(RuntimeError, match="max_len"):
        c.reserve([0, 65, 0])
    assert [len(o) for o in c.owned] == [2, 0, 2] and len(c.free) == 2
    c.release(0)
    assert c.held[0] == -1 and len(c.free) == 4 and c.lengths[0] == -1
    _begin(c, 1, 33)
    assert len(c.owned[1]) == 3


def test_prefill_refuses_places_in_use_and_empty_prompts():
    m = lm.DecoderLM(CFG, ffn=lambda x, p, **k: x)
    c = lm.PagedKVCache(CFG, 2, 4, page_size=16, device="cpu")
    _begin(c, 0, 3)
    ids = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="release"):
        m.prefill_paged({0: ids}, c)
    with pytest.raises(ValueError, match="1-D"):
        m.prefill_paged({1: ids[:0]}, c)
    with pytest.raises(ValueError, match="1-D"):
        m.prefill_paged({1: ids[None]}, c)
    with pytest.raises((TypeError, ValueError)):   # CPU tensors: the operators have no CPU path
        m.prefill_paged({1: ids}, c)
    assert c.held == [3, -1] and c.owned[1] == [] and len(c.free) == 3 and c.lengths.tolist() == [-1, -1]     # as before the call
    for b in (2, -1):
        with pytest.raises(ValueError, match="place"):
            m.prefill_paged({b: ids}, c)

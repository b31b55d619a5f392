"""CPU: what callers of the LM's serving paths may do at the edges: empty places, places outside the batch, calls that fail half way."""
import pytest
import torch

from flashmhf_b200 import lm, serving
from tests.test_lm_serving_cpu import CFG, _begin


def _model():
    return lm.DecoderLM(CFG, ffn=lambda x, p, **k: x).init_weights(seed=0)


@pytest.fixture
def plain_operators(monkeypatch):
    """Stand-ins on the CPU that keep shapes and nothing else."""
    monkeypatch.setattr(serving, "paged_append", lambda pages, k, v, *a, q=None, cu_seqlens=None, rotated_keys=False: (q, k if rotated_keys else None))
    monkeypatch.setattr(serving, "paged_attention", lambda q, *a: q)
    monkeypatch.setattr(serving, "prompt_attention", lambda q, *a: q)


@pytest.mark.parametrize("filler", [-1, -100, 50, 2**31])
def test_ids_of_empty_places_may_be_anything(filler, plain_operators):
    """They are looked up in no embedding; the other places' logits do not depend on them."""
    m, out = _model(), []
    for x in (filler, 0):
        c = lm.PagedKVCache(CFG, 3, 6, page_size=16, device="cpu")
        _begin(c, 1, 3)
        c.lengths[1] = 3
        out.append(m.decode_step_paged(torch.tensor([x, 7, x]), c))
        assert c.held == [-1, 4, -1] and c.lengths.tolist() == [-1, 4, -1]
    assert torch.equal(out[0], out[1]) and out[0].shape == (3, 50)


@pytest.mark.parametrize("shape", [(1,), (2,), (4,), (3, 1), ()])
def test_a_step_refuses_ids_of_another_shape(shape, plain_operators):
    m, c = _model(), lm.PagedKVCache(CFG, 3, 6, page_size=16, device="cpu")
    _begin(c, 1, 16)
    with pytest.raises(ValueError, match="ids"):
        m.decode_step_paged(torch.zeros(shape, dtype=torch.int64), c)
    assert c.held == [-1, 16, -1] and len(c.free) == 5


def test_release_forgets_the_pages_and_refuses_places_outside_the_batch():
    """Another sequence may own them: a step that is replayed without `reserve` must meet no page there, not somebody else's."""
    c = lm.PagedKVCache(CFG, 3, 6, page_size=16, max_len=64, device="cpu")
    _begin(c, 0, 40)
    _begin(c, 2, 17)
    for b in (-1, 3, -3):
        with pytest.raises(ValueError, match="place"):
            c.release(b)
    assert c.held == [40, -1, 17] and len(c.free) == 1 and [len(o) for o in c.owned] == [3, 0, 2]
    c.release(0)
    assert c.table[0].tolist() == [-1] * 4 and c.table[2, :2].tolist() == c.owned[2] and len(c.free) == 4
    c.release(0)                      # (of a place that is free already: nothing)
    assert c.held == [-1, -1, 17] and len(c.free) == 4


def test_a_prefill_of_nothing_and_one_that_fails_half_way(plain_operators):
    m, c = _model(), lm.PagedKVCache(CFG, 3, 6, page_size=16, max_len=64, device="cpu")
    _begin(c, 0, 20)
    empty = m.prefill_paged({}, c)
    assert empty.shape == (0, 50) and empty.dtype == m.lm_head.weight.dtype and c.held == [20, -1, -1] and len(c.free) == 4
    good = torch.arange(5)
    for bad in (torch.zeros(40, dtype=torch.int64, device="meta"), torch.full((40,), 99)):      # no data to copy; no such token
        with pytest.raises(Exception):
            m.prefill_paged({1: good, 2: bad}, c)
        assert c.held == [20, -1, -1] and c.owned[1:] == [[], []] and len(c.free) == 4 and c.lengths[1:].tolist() == [-1, -1]
        assert bool((c.table[1:] == -1).all())
    assert m.prefill_paged({2: good}, c).shape == (1, 50) and c.held == [20, -1, 5]


class _Wrapped(torch.nn.Module):
    """Another module around one, as checkpointing or sharding puts it in place."""

    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, *a, **k):
        return self.inner(*a, **k)


def _serve(m):
    c = lm.PagedKVCache(CFG, 2, 6, page_size=16, device="cpu")
    return [m.prefill_paged({0: torch.arange(5), 1: torch.arange(20)}, c), m.decode_step_paged(torch.tensor([3, 4]), c)]


def test_hooked_and_wrapped_layers_take_part_in_serving(plain_operators):
    """As in the forward pass: a hook runs once a layer and pass and may change the output; a module in the place of a layer or its attention is called."""
    m = _model()
    want, seen = _serve(m), []
    parts = [m.model.layers[0], m.model.layers[1].self_attn]
    hooks = [p.register_forward_hook(lambda mod, a, out: seen.append(mod)) for p in parts]
    assert all(torch.equal(a, b) for a, b in zip(_serve(m), want)) and seen == 2 * parts
    for h in hooks:
        h.remove()
    hook = m.model.layers[1].self_attn.register_forward_hook(lambda mod, a, out: out * 0)
    assert not any(torch.equal(a, b) for a, b in zip(_serve(m), want))
    hook.remove()
    m.model.layers[0], m.model.layers[1].self_attn = _Wrapped(m.model.layers[0]), _Wrapped(m.model.layers[1].self_attn)
    assert all(torch.equal(a, b) for a, b in zip(_serve(m), want))

"""GPU: the serving operators together, as the LM uses them: prompts packed into one pass, then steps over the pages, with sequences that end
and begin in between; and the same steps captured and replayed."""
import pytest
import torch

from flashmhf_b200 import lm, serving
from oracle import mhffn_oracle as orc
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu


def _model(heads=4, kv=2, hidden=256, layers=2):
    cfg = lm.LMConfig(vocab_size=300, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads, num_key_value_heads=kv,
                      intermediate_size=128, mhffnmoe_num_heads=2, mhffnmoe_num_kuv_heads=2, mhffnmoe_num_experts=2)
    with torch.device("cuda"):
        m = lm.DecoderLM(cfg).bfloat16().init_weights(3, std=0.05)
    return cfg, m


def _plain_append(pages, k, v, cos, sin, lengths, table, q=None, cu_seqlens=None, rotated_keys=False):
    before, rows = lengths.tolist(), table.tolist()
    new = [1] * len(before) if cu_seqlens is None else (cu_seqlens[1:] - cu_seqlens[:-1]).tolist()
    pos = torch.cat([torch.arange(max(a, 0), max(a, 0) + n) for a, n in zip(before, new)])
    c, s = cos.cpu()[pos], sin.cpu()[pos]
    k32 = ref.rotate(k.cpu().float(), c, s)
    for codes, scale, y in ((pages.k, pages.k_scale, k32), (pages.v, pages.v_scale, v.cpu().float())):
        a, b = codes.float().double().cpu(), scale.double().cpu()
        ref.append(a, b, y.double(), before, new, rows)
        codes.copy_(a.to(torch.float8_e4m3fn).cuda()), scale.copy_(b.float())
    return ref.rotate(q.cpu().float(), c, s).bfloat16().cuda(), k32.bfloat16().cuda() if rotated_keys else None


def _plain_paged(q, pages, lengths, table):
    K, V = ((c.float().double() * s.double()[:, :, None, None]).cpu() for c, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
    o = torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(lengths.tolist()):
        if n > 0:
            at = table[b, :-(-n // K.shape[2])].long().cpu()
            k, v = (x[at].transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n] for x in (K, V))
            o[b] = ref.attend_causal(q[b:b + 1].cpu().double(), k, v, q.shape[-1] ** -0.5)[0][0]
    return o.bfloat16().cuda()


def _plain_prompt(q, k, v, cu):
    cu = cu.tolist()
    parts = [ref.attend_causal(*(x[a:b].cpu().double() for x in (q, k, v)), q.shape[-1] ** -0.5)[0] for a, b in zip(cu, cu[1:])]
    return torch.cat(parts).bfloat16().cuda()


def _run(m, cfg, page_size):
    """Three prompts of unlike lengths, four steps, one sequence ends and another takes its place, three steps more."""
    g = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, 300, (n,), generator=g).cuda()  # noqa: E731
    cache = lm.PagedKVCache(cfg, 4, 40, page_size=page_size, max_len=300)
    out = [m.prefill_paged({0: ids(37), 1: ids(1), 3: ids(150)}, cache)]
    out += [m.decode_step_paged(ids(4), cache)[[0, 1, 3]] for _ in range(4)]
    cache.release(1)
    out.append(m.prefill_paged({1: ids(page_size), 2: ids(5)}, cache))
    out += [m.decode_step_paged(ids(4), cache) for _ in range(3)]
    assert cache.held == [44, page_size + 3, 8, 157] and cache.lengths.tolist() == cache.held
    return out


@pytest.mark.parametrize("page_size", [16, 64])
def test_serving_run_against_plain_operators(page_size, monkeypatch):
    """Every logit of the run, with the operators and with their definitions in their place.  The two differ by bf16 roundings of attention
    outputs (2^-8 and, of weights before they meet the values, 2^-8 more) and what two layers make of them."""
    cfg, m = _model()
    got = _run(m, cfg, page_size)
    monkeypatch.setattr(serving, "paged_append", _plain_append)
    monkeypatch.setattr(serving, "paged_attention", _plain_paged)
    monkeypatch.setattr(serving, "prompt_attention", _plain_prompt)
    want = _run(m, cfg, page_size)
    for a, b in zip(got, want):
        assert a.shape == b.shape and bool(a.isfinite().all()) and orc.rel_l2(a.float(), b.float()) < 2e-2


def test_serving_prefill_is_the_forward_pass():
    """Prompts in one packed pass give the logits of a forward pass over each alone (no 8-bit numbers are read in it)."""
    cfg, m = _model(heads=2, kv=2, hidden=128)
    g = torch.Generator().manual_seed(2)
    prompts = {b: torch.randint(0, 300, (n,), generator=g).cuda() for b, n in ((0, 130), (1, 1), (2, 64))}
    cache = lm.PagedKVCache(cfg, 3, 12, page_size=32)
    got = m.prefill_paged(prompts, cache)
    with torch.no_grad():
        want = torch.cat([m(prompts[b][None])[:, -1] for b in range(3)])
    assert orc.rel_l2(got.float(), want.float()) < 2e-2


def test_serving_steps_captured_and_replayed():
    """A captured step follows lengths and pages: replayed seven times, across page borders, it gives what eager steps give, bit for bit."""
    cfg, m = _model()
    g = torch.Generator().manual_seed(4)
    prompts = {b: torch.randint(0, 300, (n,), generator=g).cuda() for b, n in ((0, 14), (2, 30))}
    steps = torch.randint(0, 300, (7, 3), generator=g).cuda()
    runs = []
    for captured in (False, True):
        cache = lm.PagedKVCache(cfg, 3, 9, page_size=16, max_len=64)
        m.prefill_paged(prompts, cache)
        out = []
        if captured:
            ids = steps[0].clone()
            state = [t.clone() for p in cache.pools for t in p], cache.lengths.clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(2):
                    m.decode_step_paged(ids, cache)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                logits = m.decode_step_paged(ids, cache)
            for t, was in zip([t for p in cache.pools for t in p], state[0]):      # as it was behind the prompts
                t.copy_(was)
            cache.lengths.copy_(state[1])
            cache.held = [14, -1, 30]
        for x in steps:
            if captured:
                ids.copy_(x)
                cache.reserve(1)
                graph.replay()
                cache.advance(1)
                out.append(logits[[0, 2]].clone())
            else:
                out.append(m.decode_step_paged(x, cache)[[0, 2]])
        assert cache.held == [21, -1, 37] and cache.lengths.tolist() == cache.held
        runs.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_operators_on_another_stream_and_two_calls_at_once():
    """Calls on two streams at the same time, each with its own workspace, give what one after the other gives."""
    import flashmhf_b200 as fm
    g = torch.Generator().manual_seed(0)
    pages = fm.KVPages(*(torch.randn(40, 2, 32, 64, generator=g).mul(30).to(torch.float8_e4m3fn).cuda() for _ in range(2)),
                       *(torch.full((40, 2), 0.125, device="cuda") for _ in range(2)))
    table = ref.ints([list(range(0, 20)), list(range(20, 40))])
    qs = [torch.randn(2, 8, 64, generator=g).bfloat16().cuda() for _ in range(8)]
    p = [torch.randn(300, h, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2)]
    cu, lengths = ref.ints([0, 100, 300]), ref.ints([640, 333])
    want = [fm.paged_attention(q, pages, lengths, table) for q in qs], fm.prompt_attention(*p, cu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got, other = [], []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(fm.paged_attention(q, pages, lengths, table))
            other.append(fm.prompt_attention(*p, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0])) and all(torch.equal(o, want[1]) for o in other)


def test_operators_refuse_gradients():
    import flashmhf_b200 as fm
    q, k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True), torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    pages = fm.KVPages.empty(1, 2, 16, 64)
    cos, sin = ref.tables(16, 64)
    calls = (lambda: fm.prompt_attention(q, k, k, ref.ints([0, 3])), lambda: fm.paged_attention(q, pages, ref.ints([1, 0, 0]), ref.ints([[0]] * 3)),
             lambda: fm.paged_append(pages, q, k, cos, sin, ref.ints([0]), ref.ints([[0]]), cu_seqlens=ref.ints([0, 3])))
    for call in calls:
        with pytest.raises(NotImplementedError):
            call()
    with torch.no_grad():
        for call in calls:
            call()
    fm.check_device_status()

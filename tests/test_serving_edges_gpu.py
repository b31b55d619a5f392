"""GPU: the serving operators at the edges of what their documentation allows: scales at the ends of their range, values that are not finite
numbers, pages of very different scales, calls that the status word has to report, and inputs that lie elsewhere in memory than usual."""
import ctypes as C
import math

import pytest
import torch

from tests import serving_ref as ref
from tests.test_serving_gpu import DECODE, _close, _fill, _packed, _pool, _prompt_reference, _starts

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    import flashmhf_b200 as fm
    fm.check_device_status()


@pytest.mark.parametrize("hd,scale,size", [(64, 2.0 ** -102, 2.0 ** 50), (96, -2.0 ** -111, 2.0 ** 55), (64, 0.0, 2.0 ** 58), (128, 2.0 ** -130, 2.0 ** 60),
                                           (64, 2.0 ** 100, 2.0 ** -52)])
def test_prompt_attention_scales_near_the_ends_of_their_range(hd, scale, size):
    """Large queries and keys under a scale that brings their scores back, and the other way round: the scale is taken as it is, however small.
    A score is off by the roundings that test_prompt_attention_scales_and_scores_that_grow counts, and three more: of the scale, of its product with
    log2(e), and of the score times it."""
    import flashmhf_b200 as fm
    n = [130, 40]
    q, k, v = _packed(sum(n), 4, hd, 1, size), _packed(sum(n), 2, hd, 2, size), _packed(sum(n), 2, hd, 3)
    want, want_lse, room = _prompt_reference(q, k, v, n, n, scale, True)
    most = float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * abs(scale)
    off = most * (hd / 16 * 2.0 ** -22 + 6 * 2.0 ** -24)
    o, lse = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), ref.ints(_starts(n)), scale=scale, return_lse=True)
    _close(o, want, room * (1 + 2 * off * 2.0 ** 8), lse, want_lse)


@pytest.mark.parametrize("lq,lk", [(300, 300), (300, 301), (300, 427), (300, 299), (130, 700)])
@pytest.mark.parametrize("bad", [0, 100, 255, 256, 290])
def test_prompt_attention_values_that_are_no_numbers_reach_127_rows_at_most(lq, lk, bad):
    """Whatever the difference between rows and keys: row r sees key c where c <= r + lk - lq, and a value at c that is not a number may reach
    the 127 rows before its own, no other row that does not see it."""
    import flashmhf_b200 as fm
    q, k, v = _packed(lq + 9, 2, 64, 1), _packed(lk + 9, 2, 64, 2), _packed(lk + 9, 2, 64, 3)
    cu_q, cu_k = ref.ints([0, lq, lq + 9]), ref.ints([0, lk, lk + 9])
    clean = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k)
    v[bad] = NAN
    o = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k)
    own = bad - (lk - lq)                      # the first row that sees it
    untouched = torch.ones(lq + 9, dtype=torch.bool)
    untouched[max(0, own - 127):lq] = False
    assert torch.equal(o.cpu()[untouched], clean.cpu()[untouched])
    assert bool(o.cpu()[max(0, own):lq].isnan().all())


def _strict(got, want, room, heaviest, size):
    """One bf16 rounding of the output; weights in fp16 (11 bits of themselves, and 2^-24 of the row's heaviest below that) times values of summed
    size ``size``; and scores and sums in fp32 (2^-16 of the weights)."""
    err = (got.double().cpu() - want).abs()
    most = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -16) * room + 2.0 ** -24 * heaviest * size + 1e-30
    assert bool((err <= most).all()), float((err / most).max())


def _one_head(q, k, v, scale):
    """q [rows, hd], k, v [n, hd] -> output, weighted sizes, heaviest weights, sizes; 64 bits, CPU."""
    w = torch.softmax(q.double() @ k.T * scale, -1)
    return w @ v, w @ v.abs(), w.amax(-1, keepdim=True), v.abs().sum(0)


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("ratio", [6, 12, 26, 30, 50, 80])
@pytest.mark.parametrize("order", [1, -1])
def test_paged_attention_pages_of_very_different_scales(hd, ratio, order):
    """Pages with large values in some dimensions and pages with small ones in the others, 2^ratio apart: each dimension has the accuracy of its
    own values, whichever page comes first."""
    import flashmhf_b200 as fm
    P, n, G = 16, 150, 3
    pages = fm.KVPages.empty(10, 1, P, hd)
    g = torch.Generator().manual_seed(ratio)
    kc = torch.randn(10, 1, P, hd, generator=g).mul(30).to(torch.float8_e4m3fn)
    vc = torch.randn(10, 1, P, hd, generator=g).mul(60).clamp(-448, 448)
    big = torch.zeros(10, dtype=torch.bool)
    big[::order * 3 if order > 0 else 4] = True
    if order < 0:
        big = big.flip(0)
    vc[big, ..., hd // 2:] = 0
    vc[~big, ..., :hd // 2] = 0
    vc = vc.to(torch.float8_e4m3fn)
    scale = torch.where(big, 2.0 ** (ratio // 2), 2.0 ** (ratio // 2 - ratio))[:, None]
    pages.k.copy_(kc), pages.v.copy_(vc), pages.v_scale.copy_(scale), pages.k_scale.fill_(2.0 ** -5)
    K, V = ((c.double() * s).reshape(-1, hd)[:n] for c, s in ((kc, 2.0 ** -5), (vc, scale[:, :, None, None].double())))
    for size in (0.0, 1.0):
        q = (torch.randn(1, G, hd, generator=g) * size).bfloat16()
        o = fm.paged_attention(q.cuda(), pages, ref.ints([n]), ref.ints([list(range(10))]))
        _strict(o[0], *_one_head(q[0], K, V, hd ** -0.5))


def test_a_wait_that_runs_out_is_reported_before_an_index_out_of_range():
    """Both in one run, in either order: neither report hides the other."""
    import flashmhf_b200 as fm
    from flashmhf_b200 import _lib
    lib, stream = _lib.load(), C.c_void_p(torch.cuda.current_stream().cuda_stream)
    pages, q = _pool(3, 1, 16, 64, 0), _packed(1, 2, 64, 0).cuda()
    steps = (lambda: fm.paged_attention(q, pages, ref.ints([20]), ref.ints([[0, 7]])),
             lambda: lib.flashmhf_selftest_bounded_wait(2_000_000, stream))
    for order in ((0, 1), (1, 0)):
        for i in order:
            steps[i]()
        for status in (-9, -11):
            with pytest.raises(_lib.FlashMHFError) as e:
                fm.check_device_status()
            assert e.value.status == status
        fm.check_device_status()


def test_a_captured_launch_that_gave_up_reports_each_time():
    """A captured launch keeps its number: what the status call has read does not keep the next replay from running, or from saying that it gave up."""
    from flashmhf_b200 import _lib
    lib = _lib.load()
    _lib.device_status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert lib.flashmhf_selftest_bounded_wait(2_000_000, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    _lib.device_status()
    for _ in range(3):
        graph.replay()
        with pytest.raises(_lib.FlashMHFError) as e:
            _lib.device_status()
        assert e.value.status == -9 and e.value.code == _lib.SELFTEST_CODE
        _lib.device_status()
    graph.replay()
    graph.replay()               # before anyone has read of the first
    with pytest.raises(_lib.FlashMHFError):
        _lib.device_status()
    _lib.device_status()


def _shifted(x):
    """The same contiguous tensor two bytes behind a 16-byte boundary."""
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    y.copy_(x)
    assert y.is_contiguous() and y.data_ptr() % 16 != 0
    return y


def test_inputs_off_a_16_byte_boundary():
    import flashmhf_b200 as fm
    q, k, v = (_packed(40, h, 64, i).cuda() for i, h in enumerate((4, 2, 2)))
    cu, cos, sin = ref.ints([0, 17, 40]), *ref.tables(64, 64)
    args = (cos, sin, ref.ints([0, 0]), ref.ints([[0, 1], [2, 3]]))
    runs = []
    for f in (lambda x: x, _shifted):
        pages = fm.KVPages.empty(4, 2, 32, 64)
        for t in pages[:2]:
            t.view(torch.uint8).zero_()
        qr, kr = fm.paged_append(pages, f(k), f(v), *args, q=f(q), cu_seqlens=cu, rotated_keys=True)
        runs.append([qr, kr, *(t.view(torch.uint8) for t in pages), fm.prompt_attention(f(q), f(k), f(v), cu),
                     fm.paged_attention(f(q[:2].clone()), pages, ref.ints([17, 23]), args[3])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_what_is_written_in_place_has_a_new_version():
    import flashmhf_b200 as fm
    pages, x = fm.KVPages.empty(2, 2, 16, 64), _packed(3, 2, 64, 0).cuda()
    cos, sin = ref.tables(16, 64)
    was = [t._version for t in pages]
    fm.paged_append(pages, x, x, cos, sin, ref.ints([0]), ref.ints([[0]]), cu_seqlens=ref.ints([0, 3]))
    assert all(t._version > w for t, w in zip(pages, was))
    for call in (lambda out: fm.paged_attention(x[:1], pages, ref.ints([3]), ref.ints([[0]]), out=out[:1]),
                 lambda out: fm.prompt_attention(x, x, x, ref.ints([0, 3]), out=out)):
        out = torch.empty_like(x)
        was, still = out._version, x._version
        call(out)
        assert out._version > was and x._version == still
    with torch.inference_mode():          # (tensors that count no versions)
        fm.prompt_attention(x, x, x, ref.ints([0, 3]), out=torch.empty_like(x))
    scale = torch.ones(1, device="cuda", requires_grad=True)
    saved = (scale * pages.k_scale).sum()            # keeps k_scale for the gradient of `scale`
    with torch.no_grad():
        fm.paged_append(pages, x[:1], x[:1], cos, sin, ref.ints([3]), ref.ints([[0]]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    grad = pages._replace(k=pages.k.detach().requires_grad_())
    for call in (lambda: fm.paged_append(grad, x[:1], x[:1], cos, sin, ref.ints([3]), ref.ints([[0]])),
                 lambda: fm.paged_attention(x[:1], grad, ref.ints([3]), ref.ints([[0]]))):
        with pytest.raises(NotImplementedError):
            call()


def test_outputs_that_lie_over_inputs():
    """The output may take the queries' place; over keys, values or itself it is refused."""
    import flashmhf_b200 as fm
    qkv = _packed(150, 6, 64, 5).cuda()
    cu = ref.ints([0, 20, 150])
    parts = lambda t: (t[:, :2], t[:, 2:4], t[:, 4:])  # noqa: E731
    want = fm.prompt_attention(*parts(qkv), cu)
    x = qkv.clone()
    assert torch.equal(fm.prompt_attention(*parts(x), cu, out=parts(x)[0]), want) and torch.equal(x[:, 2:], qkv[:, 2:])
    q, k, v = (t.contiguous() for t in parts(qkv))
    for out in (k, v, torch.empty(150 * 64 + 128, dtype=torch.bfloat16, device="cuda").as_strided((150, 2, 64), (64, 64, 1))):
        with pytest.raises(ValueError):
            fm.prompt_attention(q, k, v, cu, out=out)
    for bad in parts(x)[1:]:
        with pytest.raises(ValueError):
            fm.prompt_attention(*parts(x), cu, out=bad)
    assert torch.equal(k, parts(qkv)[1]) and torch.equal(v, parts(qkv)[2])
    one = qkv.clone()                       # one query row inside the range of the keys, heads first, several new tokens: views that do not meet
    row, some = parts(one)[0][30:31], ref.ints([0, 1])
    want = fm.prompt_attention(row.clone(), k, v, some, ref.ints([0, 150]))
    assert torch.equal(fm.prompt_attention(row, *parts(one)[1:], some, ref.ints([0, 150]), out=row), want)
    first = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(fm.prompt_attention(*parts(first), cu, out=parts(first)[0]), fm.prompt_attention(*parts(qkv), cu))
    with pytest.raises(ValueError):
        fm.prompt_attention(*parts(first), cu, out=parts(first)[1])
    pages = _pool(4, 2, 32, 64, 0)
    both = _packed(2 * 3, 8, 64, 8).cuda().view(2, 3, 8, 64)
    where = ref.ints([40, 50]), ref.ints([[0, 1], [2, 3]])
    for t in pages[:2]:
        t.view(torch.uint8).copy_(torch.randn(t.shape).to(torch.float8_e4m3fn).view(torch.uint8))
    want = fm.paged_attention(both[:, :, :4].clone(), pages, *where)
    assert torch.equal(fm.paged_attention(both[:, :, :4], pages, *where, out=both[:, :, 4:]), want) and torch.equal(both[:, :, 4:], want)
    with pytest.raises(ValueError):
        fm.paged_attention(both[:, :, :4], pages, *where, out=both[:, :, 1:5])
    q1 = q[:2].clone()
    args = (pages, ref.ints([30, 50]), ref.ints([[0, 1], [2, 3]]))
    for t in pages[:2]:
        t.view(torch.uint8).copy_(torch.randn(t.shape).to(torch.float8_e4m3fn).view(torch.uint8))
    want = fm.paged_attention(q1, *args)
    assert torch.equal(fm.paged_attention(q1, *args, out=q1), want)


def test_the_example_in_the_readme():
    """Its serving lines, run as they stand: the step's output is attention over the prompt and the new token."""
    import os

    import flashmhf_b200 as fm
    from tests.test_serving_gpu import _decode_reference
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")) as f:
        lines = f.read().split("import flashmhf_b200 as fm\n", 1)[1].split("```", 1)[0].splitlines()
    at = [i for i, line in enumerate(lines) if "KVPages" in line or "install_reference_seam" in line]
    n, n_kv, page_size, head_dim, num_pages = [20, 47], 2, 16, 64, 9
    cos, sin = ref.tables(64, head_dim)
    x, y = _packed(sum(n), 8, head_dim, 1).cuda(), _packed(2, 8, head_dim, 2).cuda()
    rows = [[4, 0, 7, 8], [2, 1, 3, 5]]
    names = dict(fm=fm, num_pages=num_pages, n_kv=n_kv, page_size=page_size, head_dim=head_dim, cos=cos, sin=sin, q=x[:, :4], k=x[:, 4:6], v=x[:, 6:],
                 q1=y[:, :4], k1=y[:, 4:6], v1=y[:, 6:], lengths=ref.ints([0, 0]), table=ref.ints(rows), cu=ref.ints(_starts(n)))
    exec("\n".join(lines[at[0]:at[1]]), names)
    want, _, room = _decode_reference(names["q"].cpu()[:, None], names["pages"], [21, 48], rows, head_dim ** -0.5)
    _close(names["o"][:, None], want, room)


def _gpu_reference(q, pages, lengths, table, scale):
    """The definition in 64 bits on the GPU, a sequence at a time -> (o, lse, weighted sizes, heaviest weights, sizes)."""
    o, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    room, heavy, size = torch.zeros_like(o), torch.zeros(q.shape[:3] + (1,), dtype=torch.float64), torch.zeros_like(o)
    kv, P, hd = pages.k.shape[1:]
    G, nq = q.shape[2] // kv, q.shape[1]
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        at = table[b, :-(-n // P)].long()
        k, v = ((c.view(torch.uint8)[at].view(c.dtype).double() * s[at].double()[:, :, None, None]).transpose(0, 1).reshape(kv, -1, hd)[:, :n]
                for c, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        x = torch.einsum("ikgd,knd->ikgn", q[b].double().view(nq, kv, G, hd), k) * scale
        see = torch.arange(n, device="cuda") < n - nq + 1 + torch.arange(nq, device="cuda")[:, None]
        x = x.masked_fill(~see[:, None, None], -math.inf)
        l = torch.logsumexp(x, -1)
        w = torch.exp(x - l[..., None]).nan_to_num(nan=0.0)
        for to, what in ((o, torch.einsum("ikgn,knd->ikgd", w, v)), (room, torch.einsum("ikgn,knd->ikgd", w, v.abs())), (lse, l), (heavy, w.amax(-1)),
                         (size, v.abs().sum(1)[None, :, None].expand(nq, kv, G, hd))):
            to[b] = what.reshape(to[b].shape).cpu()
    return o, lse, room, heavy, size


def _many_units(runs, kv, tiles, B, longest, seed):
    """Ragged lengths, empty sequences among them, whose units of 64 tokens are `runs` to each warp of the GPU and some more."""
    warps = torch.cuda.get_device_properties(0).multi_processor_count * 12
    r = torch.Generator().manual_seed(seed)
    n = [0 if i % 7 == 3 else int(torch.randint(1, longest + 1, (1,), generator=r)) for i in range(B)]
    units = lambda: sum(-(-x // 64) for x in n) * kv * tiles  # noqa: E731
    i = 0
    while units() < runs * warps + 5:
        i += 1
        n[i % B] += 0 if (i % B) % 7 == 3 else 64
    assert units() % warps
    return n


@pytest.mark.parametrize("hd,P,kv,heads,new,B,longest,runs", [
    (64, 16, 4, 8, 1, 60, 4000, 10),          # a warp's run walks over more than 32 pages of 16, and through several sequences
    (64, 64, 8, 8, 1, 150, 900, 3),           # more items than the joining by sixteen warps is for
    (96, 16, 2, 24, 1, 40, 9000, 11), (96, 32, 8, 8, 2, 100, 600, 2),
    (128, 16, 2, 8, 4, 30, 6000, 12), (128, 128, 4, 4, 1, 64, 3000, 6),
    (64, 32, 1, 2, 1, 1, 10, 9), (128, 64, 1, 8, 1, 2, 10, 5),       # one and two long sequences: every warp has a part of one item
])
def test_paged_attention_runs_of_many_units(hd, P, kv, heads, new, B, longest, runs):
    """Every warp has several units of 64 tokens: rings that go round, pages beyond the first 32, runs that end in another item than they began
    in, parts at both ends of a run, items that one warp has alone, and both kernels that join parts."""
    import flashmhf_b200 as fm
    lengths = _many_units(runs, kv, -(-(heads // kv * new) // 8), B, longest, hd + P)
    rows, n_pages = ref.page_tables(lengths, P, seed=hd)
    g = torch.Generator(device="cuda").manual_seed(P)
    codes = [torch.randn(n_pages, kv, P, hd, device="cuda", generator=g).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    pages = fm.KVPages(*codes, *(torch.exp2(torch.randint(-8, -4, (n_pages, kv), device="cuda", generator=g).float()) for _ in range(2)))
    table = ref.ints(rows)
    for b, n in enumerate(lengths):            # what lies behind a sequence's last token is nobody's
        if n % P:
            for c in codes:
                c.view(torch.uint8)[rows[b][n // P], :, n % P:] = 0x7f
    q = torch.randn(B, new, heads, hd, device="cuda", generator=g).bfloat16()
    want, want_lse, room, heavy, size = _gpu_reference(q, pages, lengths, table, hd ** -0.5)
    o, lse = fm.paged_attention(q, pages, ref.ints(lengths), table, return_lse=True)
    _strict(o, want, room, heavy, size)
    _close(o, want, room, lse, want_lse)
    assert torch.equal(fm.paged_attention(q, pages, ref.ints(lengths), table), o)


@pytest.mark.parametrize("hd,P,often", [(64, 16, 0.01), (128, 16, 0.02), (96, 32, 0.3)])
def test_paged_attention_far_scales_anywhere_in_a_run(hd, P, often):
    """A few pages with large values in some dimensions among many with small ones in the others, 2^40 apart, in runs of more pages than a warp knows
    at first."""
    import flashmhf_b200 as fm
    kv, B = 2, 9
    lengths = _many_units(10, kv, 1, B, 60000, hd)
    rows, n_pages = ref.page_tables(lengths, P, seed=hd)
    g = torch.Generator(device="cuda").manual_seed(P)
    codes = [torch.randn(n_pages, kv, P, hd, device="cuda", generator=g).mul_(60).clamp_(-448, 448) for _ in range(2)]
    big = torch.rand(n_pages, kv, device="cuda", generator=g) < often
    codes[1][..., hd // 2:] *= (~big)[:, :, None, None]
    codes[1][..., :hd // 2] *= big[:, :, None, None]
    pages = fm.KVPages(*(c.to(torch.float8_e4m3fn) for c in codes), torch.full((n_pages, kv), 2.0 ** -6, device="cuda"),
                       torch.where(big, 2.0 ** 20, 2.0 ** -20))
    table = ref.ints(rows)
    q = torch.randn(B, 1, 4 * kv, hd, device="cuda", generator=g).bfloat16()
    want, want_lse, room, heavy, size = _gpu_reference(q, pages, lengths, table, hd ** -0.5)
    o, lse = fm.paged_attention(q, pages, ref.ints(lengths), table, return_lse=True)
    _strict(o, want, room, heavy, size)
    _close(o, want, room, lse, want_lse)


@pytest.mark.parametrize("lengths,new,kv,heads,hd,P", DECODE)
def test_paged_attention_to_the_accuracy_of_its_weights(lengths, new, kv, heads, hd, P):
    """The cases of test_paged_attention, with weights of 11 bits."""
    import flashmhf_b200 as fm
    rows, n_pages = ref.page_tables(lengths, P, seed=hd)
    pages = _pool(n_pages, kv, P, hd, seed=P)
    _fill(pages, lengths, rows, seed=2)
    q = torch.randn(len(lengths), new, heads, hd, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    want, _, room, heavy, size = _gpu_reference(q, pages, lengths, ref.ints(rows), hd ** -0.5)
    _strict(fm.paged_attention(q, pages, ref.ints(lengths), ref.ints(rows)), want, room, heavy, size)


def _spread_out(t, dim, extra, fill):
    """The same tensor with `extra` further entries between those of dimension 0, or as a view of heads-first memory (dim 1)."""
    if dim == 1:
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    big = torch.full((t.shape[0], t.shape[1] + extra, *t.shape[2:]), fill, dtype=torch.uint8, device=t.device).repeat_interleave(t.element_size(), -1)
    big = big.view(t.dtype)
    big[:, :t.shape[1]].view(torch.uint8).copy_(t.contiguous().view(torch.uint8))
    return big[:, :t.shape[1]]


@pytest.mark.parametrize("hd,P", [(64, 16), (96, 64), (128, 32)])
def test_strides_of_pools_tables_and_rows(hd, P):
    """Pools whose pages lie further apart than their size, rows with the head as the outer stride, tables that are views of wider ones: the same
    bits as of contiguous tensors, and nothing between the pages is written."""
    import flashmhf_b200 as fm
    kv, heads, before, new = 2, 6, [5, 40, 0], [30, 1, 3 * P + 7]
    rows, n = ref.page_tables([a + b + 1 for a, b in zip(before, new)], P)
    table = ref.ints(rows)
    wide = torch.full((3, table.shape[1] + 9), 10**6, dtype=torch.int32, device="cuda")
    wide[:, 4:4 + table.shape[1]] = table
    cos, sin = ref.tables(600, hd)
    cu, runs = ref.ints(_starts(new)), []
    x = [_packed(sum(new) + 3, h, hd, h).cuda() for h in (heads, kv, kv + 1)]
    x[2] = x[2][:, :kv]
    for far in (False, True):
        pages = _pool(n, kv, P, hd, 1)
        _fill(pages, before, rows, 2)
        f = lambda t: _spread_out(t, 1, 0, 0) if far else t.contiguous()  # noqa: E731
        pages = pages._replace(**{k: _spread_out(getattr(pages, k), 0, 3, 0x55) for k in "kv"}) if far else pages
        t = wide[:, 4:4 + table.shape[1]] if far else table
        q, k, v = (f(y[:-3]) for y in x)
        q1, k1, v1 = (f(y[-3:]) for y in x)
        qr, kr = fm.paged_append(pages, k, v, cos, sin, ref.ints(before), t, q=q, cu_seqlens=cu, rotated_keys=True)
        lengths = ref.ints(before) + cu[1:] - cu[:-1]
        qs, _ = fm.paged_append(pages, k1, v1, cos, sin, lengths, t, q=q1)
        o, lse = fm.paged_attention(f(qs), pages, lengths + 1, t, return_lse=True)
        out = fm.prompt_attention(f(qr), f(kr), v, cu, out=f(torch.empty_like(qr)))
        runs.append([y.contiguous().view(torch.uint8) for y in (qr, kr, qs, o, lse, out, *pages)])
        if far:
            for c in pages[:2]:
                gap = c.view(torch.uint8).as_strided((n, 3 * P * hd), (c.stride(0), 1), c.storage_offset() + kv * P * hd)
                assert bool((gap == 0x55).all())
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("P", [16, 64, 128])
@pytest.mark.parametrize("bad", [-1, 10**6])
def test_packed_append_leaves_out_pages_and_positions_out_of_range(P, bad):
    """A page outside the pool, and rows behind the rotary tables: those are left out and reported, everything else is written as without them."""
    import flashmhf_b200 as fm
    from flashmhf_b200 import _lib
    before, new, hd, kv = [P // 2, 3, 0], [2 * P, P, 2 * P], 64, 2
    total = [a + b for a, b in zip(before, new)]
    rows, n = ref.page_tables(total, P)
    k, v = _packed(sum(new), kv, hd, 1).cuda(), _packed(sum(new), kv, hd, 2).cuda()
    cos, sin = ref.tables(max(total), hd)
    cu = ref.ints(_starts(new))

    def run(rows, positions):
        pages = _pool(n, kv, P, hd, 3)
        _fill(pages, before, rows_good, 4)
        fm.paged_append(pages, k, v, cos[:positions], sin[:positions], ref.ints(before), ref.ints(rows), cu_seqlens=cu)
        return pages

    def reported(code):
        with pytest.raises(_lib.FlashMHFError) as e:
            fm.check_device_status()
        assert e.value.status == -11 and e.value.code == code

    rows_good = [list(r) for r in rows]
    untouched = _pool(n, kv, P, hd, 3)
    _fill(untouched, before, rows_good, 4)
    want = run(rows_good, max(total))
    broken = [list(r) for r in rows]
    broken[0][1] = bad                                       # the first sequence's second page
    got = run(broken, max(total))
    reported(401)
    for a, b, u in zip(got, want, untouched):
        keep = torch.ones(n, dtype=torch.bool)
        keep[rows_good[0][1]] = False
        a, b, u = (t.view(torch.uint8).cpu() if t.dtype == torch.float8_e4m3fn else t.cpu() for t in (a, b, u))
        assert torch.equal(a[keep], b[keep]) and torch.equal(a[~keep], u[~keep])
    positions = P + P // 2                                    # ends inside the second page of every sequence that reaches it
    got = run(rows_good, positions)
    reported(402)
    for b, (n0, m) in enumerate(zip(before, new)):
        for name in "kv":
            a, w, u = (getattr(t, name).view(torch.uint8).cpu() for t in (got, want, untouched))
            for j in range(-(-total[b] // P)):
                lo, hi, page = max(0, n0 - j * P), min(P, total[b] - j * P, max(0, positions - j * P)), rows_good[b][j]
                assert torch.equal(a[page][:, max(lo, hi):], u[page][:, max(lo, hi):])
                if (j + 1) * P <= positions:                  # pages before the border: as without it
                    assert torch.equal(a[page], w[page])
                elif hi > lo:
                    s = getattr(got, name + "_scale")[page].cpu().double()[:, None, None]
                    y = (k if name == "k" else v).cpu()[sum(new[:b]) + j * P + lo - n0:sum(new[:b]) + j * P + hi - n0].float()
                    if name == "k":
                        y = ref.rotate(y, cos.cpu()[j * P + lo:j * P + hi], sin.cpu()[j * P + lo:j * P + hi])
                    codes = ref.to_e4m3(y.double().transpose(0, 1) / s)
                    assert torch.equal(getattr(got, name)[page, :, lo:hi].float().double().cpu(), codes)


def test_a_token_behind_the_rotary_tables_is_not_written():
    import flashmhf_b200 as fm
    from flashmhf_b200 import _lib
    pages, x = _pool(3, 1, 16, 64, 0), _packed(1, 1, 64, 1).cuda()
    before = [t.view(torch.uint8).clone() for t in pages]
    fm.paged_append(pages, x, x, *ref.tables(40, 64), ref.ints([45]), ref.ints([[0, 1, 2]]))
    with pytest.raises(_lib.FlashMHFError):
        fm.check_device_status()
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before, pages))

"""GPU: the serving operators (paged_append, paged_attention, prompt_attention) against their definitions in 64 bits.

Tolerances count roundings.  Codes: keys are rotated in fp32 with every operation rounded, so that against the same fp32 expression
codes and scales are equal bit for bit.  Attention: the output is one bf16 rounding (2^-8 of the value at most) away from a sum whose
weights were rounded to 8 bits or more before they met the values, each by 2^-8 of itself at most: |error| <= 2^-8 |o| + 2^-8 sum w |v|,
with room for the fp32 parts (2 %)."""
import math

import pytest
import torch

from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    import flashmhf_b200 as fm
    fm.check_device_status()


def _pool(n, kv, P, hd, seed):
    """A pool in use: random codes (NaN codes among them: what nobody may read) and random scales."""
    import flashmhf_b200 as fm
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(0, 256, (n, kv, P, hd), generator=g, dtype=torch.uint8).cuda().view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, -3, (n, kv), generator=g).float()).cuda() for _ in range(2)]
    return fm.KVPages(*codes, *scales)


def _fill(pages, total, rows, seed):
    """Finite codes in the rows that sequences hold."""
    g = torch.Generator().manual_seed(seed)
    P = pages.k.shape[2]
    for c in (pages.k, pages.v):
        raw = c.view(torch.uint8)
        for b, n in enumerate(total):
            for j in range(-(-max(n, 0) // P)):
                m = min(P, n - j * P)
                x = torch.randn(c.shape[1], m, c.shape[3], generator=g).mul(60).clamp(-448, 448).to(torch.float8_e4m3fn)
                raw[rows[b][j], :, :m] = x.view(torch.uint8).cuda()


def _values(codes, scale):
    return codes.float().double().cpu() * scale.double().cpu()[:, :, None, None]


# ------------------------------------------------------------------------------------------------ append
APPEND = [  # before, new (None: one token each), kv, heads, hd, P
    ([0], None, 1, 1, 64, 16),
    ([0, 15, 16, 17, 63, 200], None, 2, 4, 64, 16),
    ([31, 32, 33, -1, 5], None, 3, 3, 96, 32),
    ([127, 128, 129, 1000], None, 2, 16, 128, 128),
    ([0], [1], 2, 2, 64, 64),
    ([0, 0, 0], [1, 64, 65], 2, 4, 64, 64),
    ([5, 0, 63, 64, 100], [130, 0, 1, 200, 3], 2, 6, 96, 64),
    ([0, 17, 300], [257, 128, 129], 2, 8, 128, 128),
    ([3, -1, 30], [40, 9, 1], 1, 9, 128, 16),
    ([10, 11], [33, 31], 4, 1, 96, 32),
]


@pytest.mark.parametrize("before,new,kv,heads,hd,P", APPEND)
def test_append(before, new, kv, heads, hd, P):
    import flashmhf_b200 as fm
    counts = new or [1] * len(before)
    total = [max(0, a) + n for a, n in zip(before, counts)]
    rows, n_pages = ref.page_tables(total, P, seed=len(before))
    pages = _pool(n_pages, kv, P, hd, seed=hd + P)
    _fill(pages, before, rows, seed=1)
    T = sum(counts)
    g = torch.Generator().manual_seed(T)
    qkv = (torch.randn(T, heads + 2 * kv, hd, generator=g) * torch.exp(torch.randn(T, 1, 1, generator=g))).bfloat16().cuda()
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    cos, sin = ref.tables(max(total) + 1, hd)
    cu = None if new is None else ref.ints([sum(counts[:i]) for i in range(len(counts) + 1)])
    want = {x: [getattr(pages, x).float().double().cpu(), getattr(pages, x + "_scale").double().cpu()] for x in "kv"}
    first = [sum(counts[:i]) for i in range(len(counts))]
    pos = torch.cat([torch.arange(max(a, 0), max(a, 0) + n) for a, n in zip(before, counts)])
    live = torch.cat([torch.full((n,), a >= 0) for a, n in zip(before, counts)])
    c, s = cos.cpu()[pos], sin.cpu()[pos]
    k32, q32 = ref.rotate(k.cpu().float(), c, s), ref.rotate(q.cpu().float(), c, s)     # fp32, each operation rounded
    for x, y in (("k", k32), ("v", v.cpu().float())):
        ref.append(*want[x], y.double(), before, counts, rows)
    q_rot, k_rot = fm.paged_append(pages, k, v, cos, sin, ref.ints(before), ref.ints(rows), q=q, cu_seqlens=cu, rotated_keys=True)
    for x in "kv":
        got, scale = getattr(pages, x).float().double().cpu(), getattr(pages, x + "_scale").double().cpu()
        assert torch.equal(scale, want[x][1])
        assert torch.equal(got.nan_to_num(nan=1e6), want[x][0].nan_to_num(nan=1e6))
    assert torch.equal(q_rot.cpu()[live], q32.bfloat16()[live]) and torch.equal(k_rot.cpu()[live], k32.bfloat16()[live])
    assert first[0] == 0


def test_append_without_queries_and_twice_is_the_same():
    import flashmhf_b200 as fm
    rows, n_pages = ref.page_tables([70, 20], 32)
    pages = _pool(n_pages, 2, 32, 64, 3)
    _fill(pages, [30, 20], rows, 4)
    k, v = (torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in (1, 2))
    cos, sin = ref.tables(128, 64)
    args = (k, v, cos, sin, ref.ints([30, 20]), ref.ints(rows))
    q, kr = fm.paged_append(pages, *args, cu_seqlens=ref.ints([0, 40, 40]))
    assert q is None and kr is None
    once = [t.clone() for t in pages]
    fm.paged_append(pages, *args, cu_seqlens=ref.ints([0, 40, 40]))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(once, pages))


def test_append_values_without_a_number_and_zeros():
    """NaN and infinities become NaN codes and leave the scale alone; a page of zeros has the smallest scale; a huge value fits."""
    import flashmhf_b200 as fm
    pages = _pool(3, 1, 16, 64, 0)
    k = torch.zeros(3, 1, 64).bfloat16()
    k[0, 0, 0], k[0, 0, 1], k[0, 0, 2], k[0, 0, 3] = NAN, math.inf, -math.inf, 2.0
    k[2, 0, 5] = -3.3e38
    cos, sin = ref.tables(4, 64)
    cos.fill_(1.0), sin.fill_(0.0)
    fm.paged_append(pages, k.cuda(), k.cuda(), cos, sin, ref.ints([0, 0, 0]), ref.ints([[0], [1], [2]]))
    for codes, scale in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        row = codes[:, 0, 0].float().cpu()
        # 2 = 448 * 2^-7.8...: under 2^-7, 256
        assert scale[:, 0].tolist() == [2.0 ** -7, 2.0 ** -60, 2.0 ** 120]
        # (where the sine is 0, an infinite first half makes the second half NaN and the other way round, for the keys)
        assert row[0, :3].isnan().all() and row[0, 3] == 256 and torch.equal(row[1], torch.zeros(64))
        want = torch.tensor([k[2, 0, 5].double().item() / 2.0 ** 120], dtype=torch.float64)
        assert row[2, 5].double() == ref.to_e4m3(want)


def test_append_grows_the_scale_exactly():
    """Small rows first, a large one later: the rows that were there keep their values (to the type's subnormals)."""
    import flashmhf_b200 as fm
    pages = fm.KVPages.empty(1, 1, 64, 64)
    cos, sin = ref.tables(8, 64)
    small = torch.randn(5, 1, 64, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    fm.paged_append(pages, small, small, cos, sin, ref.ints([0]), ref.ints([[0]]), cu_seqlens=ref.ints([0, 5]))
    was = pages.values()[1][0, 0, :5].clone()
    big = torch.full((1, 1, 64), 20.0).bfloat16().cuda()
    fm.paged_append(pages, big, big, cos, sin, ref.ints([5]), ref.ints([[0]]))
    now, scale = pages.values()[1][0, 0, :6], float(pages.v_scale[0, 0])
    assert scale == 2.0 ** -4 and torch.equal(now[5].float().cpu(), torch.full((64,), 20.0))
    assert ((now[:5] - was).abs().float() <= scale * 2.0 ** -10).all()          # half a subnormal step
    normal = was.abs() >= scale * 2.0 ** -6
    assert torch.equal(now[:5][normal], was[normal])


# ------------------------------------------------------------------------------------------------ attention over pages
DECODE = [  # lengths, new, kv, heads, hd, P
    ([1], 1, 1, 1, 64, 16),
    ([0, 1, 2, 15, 16, 17], 1, 2, 4, 64, 16),
    ([100, 33, 32, 31, -1, 64], 1, 1, 8, 96, 32),
    ([257, 3, 128, 640], 1, 2, 16, 128, 128),
    ([1023], 1, 16, 16, 64, 64),
    ([3000, 1, 50], 1, 2, 24, 64, 16),
    ([5, 1, 300], 4, 2, 6, 96, 16),
    ([77, 16, 15, 1], 16, 1, 2, 128, 64),
    ([700, 65], 3, 1, 40, 64, 32),
    ([20000], 1, 2, 8, 128, 64),
    ([513] * 37, 1, 3, 3, 64, 128),
]


def _decode_reference(q, pages, lengths, rows, scale):
    K, V = _values(pages.k, pages.k_scale), _values(pages.v, pages.v_scale)
    B, nq, H, hd = q.shape
    kv, P = K.shape[1], K.shape[2]
    G = H // kv
    o, lse, room = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:3], -math.inf, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b, n in enumerate(lengths):
        if n <= 0:
            continue
        at = torch.tensor(rows[b][:-(-n // P)])
        for h in range(kv):
            k, v = K[at, h].reshape(-1, hd)[:n], V[at, h].reshape(-1, hd)[:n]
            for i in range(nq):
                m = n - (nq - 1 - i)
                if m <= 0:
                    continue
                x = q[b, i, h * G:(h + 1) * G].double() @ k[:m].T * scale
                l = torch.logsumexp(x, -1)
                w = torch.exp(x - l[:, None])
                o[b, i, h * G:(h + 1) * G], lse[b, i, h * G:(h + 1) * G] = w @ v[:m], l
                room[b, i, h * G:(h + 1) * G] = w @ v[:m].abs()
    return o, lse, room


def _close(got, want, room, lse=None, want_lse=None, top=None):
    err, most = (got.double().cpu() - want).abs(), 2.0 ** -8 * want.abs() + 2.0 ** -8 * 1.02 * room + 1e-30
    assert bool((err <= most).all()), float((err / most).max())
    if lse is not None:
        l = lse.double().cpu()
        assert torch.equal(l == -math.inf, want_lse == -math.inf)
        fine = want_lse > -math.inf
        # a score's products are summed in fp32: about hd roundings of 2^-24 of the largest partial sum, far under 1e-4 of the largest score
        assert ((l - want_lse)[fine].abs() <= 1e-4 + 1e-5 * want_lse[fine].abs()).all()


@pytest.mark.parametrize("lengths,new,kv,heads,hd,P", DECODE)
def test_paged_attention(lengths, new, kv, heads, hd, P):
    import flashmhf_b200 as fm
    rows, n_pages = ref.page_tables(lengths, P, seed=hd)
    pages = _pool(n_pages, kv, P, hd, seed=P)
    _fill(pages, lengths, rows, seed=2)
    q = torch.randn(len(lengths), new, heads, hd, generator=torch.Generator().manual_seed(9)).bfloat16()
    want, want_lse, room = _decode_reference(q, pages, lengths, rows, hd ** -0.5)
    o, lse = fm.paged_attention(q.cuda(), pages, ref.ints(lengths), ref.ints(rows), return_lse=True)
    _close(o, want, room, lse, want_lse)
    if new == 1:
        o3 = fm.paged_attention(q[:, 0].cuda(), pages, ref.ints(lengths), ref.ints(rows))
        assert o3.shape == (len(lengths), heads, hd) and torch.equal(o3, o[:, 0])
    o2 = torch.full_like(o, NAN)
    assert fm.paged_attention(q.cuda(), pages, ref.ints(lengths), ref.ints(rows), out=o2) is o2 and torch.equal(o, o2)


def test_paged_attention_scales_that_differ_widely():
    """Pages whose scales are 2^40 apart, and a softmax scale that makes one key win."""
    import flashmhf_b200 as fm
    lengths, P, hd = [200, 90], 16, 64
    rows, n_pages = ref.page_tables(lengths, P)
    pages = _pool(n_pages, 2, P, hd, 0)
    _fill(pages, lengths, rows, 1)
    g = torch.Generator().manual_seed(3)
    pages.v_scale.copy_(torch.exp2(torch.randint(-25, 15, pages.v_scale.shape, generator=g).float()).cuda())
    pages.k_scale.copy_(torch.exp2(torch.randint(-12, -6, pages.v_scale.shape, generator=g).float()).cuda())
    q = (torch.randn(2, 1, 4, hd, generator=g) * 3).bfloat16()
    for scale in (hd ** -0.5, 2.0, 1e-3, -0.5, 0.0):
        want, want_lse, room = _decode_reference(q, pages, lengths, rows, scale)
        o, lse = fm.paged_attention(q.cuda(), pages, ref.ints(lengths), ref.ints(rows), scale=scale, return_lse=True)
        _close(o, want, room, lse, want_lse)


def test_paged_attention_large_queries():
    """Queries near the end of bf16's range and tiny ones: scores stay what they are in fp32."""
    import flashmhf_b200 as fm
    rows, n_pages = ref.page_tables([70], 32)
    pages = _pool(n_pages, 1, 32, 64, 0)
    _fill(pages, [70], rows, 1)
    for size in (2.0 ** 60, 2.0 ** -60):
        q = (torch.randn(1, 1, 2, 64, generator=torch.Generator().manual_seed(5)) * size).bfloat16()
        want, want_lse, room = _decode_reference(q, pages, [70], rows, 0.125 / size)
        o, lse = fm.paged_attention(q.cuda(), pages, ref.ints([70]), ref.ints(rows), scale=0.125 / size, return_lse=True)
        _close(o, want, room, lse, want_lse)


# ------------------------------------------------------------------------------------------------ attention over prompts
PROMPT = [  # rows, keys (None: the same), kv, heads, hd, causal
    ([1], None, 1, 1, 64, True),
    ([100], None, 12, 12, 64, True),
    ([1, 2, 0, 127, 128, 129, 3], None, 2, 4, 64, True),
    ([255, 256, 257, 513], None, 1, 3, 96, True),
    ([300, 5, 700], None, 2, 8, 128, True),
    ([300, 5, 700], None, 2, 8, 128, False),
    ([64, 1, 30, 0], [200, 129, 5, 7], 2, 2, 64, True),
    ([64, 300, 10], [1, 130, 0], 1, 2, 128, True),
    ([40, 200], [333, 2], 3, 3, 96, False),
    ([1, 1, 1], [300, 1, 128], 2, 4, 64, True),
    ([1300], None, 1, 2, 64, True),
    ([7, 0, 30, 1] * 100, None, 1, 7, 64, True),        # several heads a block
    ([200] * 50 + [3, 600], None, 2, 10, 128, True),
    ([90, 150] * 25, [40, 300] * 25, 13, 13, 96, False),
]


def _packed(n, heads, hd, seed, scale=1.0):
    return (torch.randn(n, heads, hd, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16()


def _starts(n):
    return [sum(n[:i]) for i in range(len(n) + 1)]


def _prompt_reference(q, k, v, nq, nk, scale, causal):
    o, lse, room = [], [], []
    for (a, b), (c, d) in zip(zip(_starts(nq), _starts(nq)[1:]), zip(_starts(nk), _starts(nk)[1:])):
        x, l = ref.attend_causal(q[a:b].double(), k[c:d].double(), v[c:d].double(), scale, causal)
        o.append(x)
        lse.append(l)
        room.append(ref.attend_causal(q[a:b].double(), k[c:d].double(), v[c:d].double().abs(), scale, causal)[0])
    return torch.cat(o), torch.cat(lse), torch.cat(room)


@pytest.mark.parametrize("nq,nk,kv,heads,hd,causal", PROMPT)
def test_prompt_attention(nq, nk, kv, heads, hd, causal):
    import flashmhf_b200 as fm
    keys = nk or nq
    q, k, v = _packed(sum(nq), heads, hd, 1, 1.5), _packed(sum(keys), kv, hd, 2), _packed(sum(keys), kv, hd, 3)
    want, want_lse, room = _prompt_reference(q, k, v, nq, keys, hd ** -0.5, causal)
    args = (q.cuda(), k.cuda(), v.cuda(), ref.ints(_starts(nq)), None if nk is None else ref.ints(_starts(keys)))
    o, lse = fm.prompt_attention(*args, causal=causal, return_lse=True)
    _close(o, want, room, lse, want_lse)
    o2 = torch.full_like(o, NAN)
    assert fm.prompt_attention(*args, causal=causal, out=o2) is o2 and torch.equal(o, o2)


def test_prompt_attention_reads_views_and_leaves_other_rows():
    """q, k, v as views of one projection, the output as a view too; rows behind the last sequence and between views stay."""
    import flashmhf_b200 as fm
    n, kv, heads, hd = [37, 150], 2, 4, 64
    T = sum(n) + 9
    qkv = _packed(T, heads + 2 * kv, hd, 4)
    qkv[sum(n):] = NAN
    d = qkv.cuda()
    out = torch.full((T, 2 * heads, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    o = fm.prompt_attention(d[:, :heads], d[:, heads:heads + kv], d[:, heads + kv:], ref.ints(_starts(n)), out=out[:, heads:])
    m = sum(n)
    want, _, room = _prompt_reference(qkv[:m, :heads], qkv[:m, heads:heads + kv], qkv[:m, heads + kv:], n, n, hd ** -0.5, True)
    _close(o[:m], want, room)
    assert bool((out[:, :heads] == 7).all()) and bool((out[m:] == 7).all())


def test_prompt_attention_sequences_do_not_touch_each_other():
    """NaN and infinities in one sequence stay there, wherever its rows lie in a tile of its neighbours."""
    import flashmhf_b200 as fm
    n, heads, hd = [50, 3, 200, 129], 2, 64
    q, k, v = (_packed(sum(n), heads, hd, i) for i in (1, 2, 3))
    for bad in range(4):
        x = [t.clone() for t in (q, k, v)]
        a, b = _starts(n)[bad], _starts(n)[bad + 1]
        for t in x:
            t[a:b] = NAN
            t[a] = math.inf
        o = fm.prompt_attention(*(t.cuda() for t in x), ref.ints(_starts(n)))
        clean = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), ref.ints(_starts(n)))
        keep = torch.ones(sum(n), dtype=torch.bool)
        keep[a:b] = False
        assert torch.equal(o.cpu()[keep], clean.cpu()[keep])


def test_prompt_attention_gives_the_same_bits_among_any_neighbours():
    """Rows next to a sequence's last tile, of another sequence or of none, do not show in it, however large they are."""
    import flashmhf_b200 as fm
    n, heads, hd = [130, 190, 5], 2, 64
    a, b = 130, 320
    q, k, v = (_packed(sum(n), heads, hd, i) for i in (1, 2, 3))
    alone = fm.prompt_attention(q[a:b].cuda(), k[a:b].cuda(), v[a:b].cuda(), ref.ints([0, 190]))
    for size in (1.0, 1e3, 1e30):
        x = [t.clone() for t in (q, k, v)]
        for t in x:
            t[:a] *= size
            t[b:] *= size
        for cu in (_starts(n), [a, b]):
            o = fm.prompt_attention(*(t.cuda() for t in x), ref.ints(cu))
            assert torch.equal(o[a:b], alone)


@pytest.mark.parametrize("hd,scale,size", [(64, -0.5, 1.0), (128, 0.0, 1.0), (64, 2.0, 4.0), (96, 0.1, 60.0), (128, -0.7, 8.0)])
def test_prompt_attention_scales_and_scores_that_grow(hd, scale, size):
    """Scores up to some thousands, growing along the keys, so that the maximum of a row moves by far many times; scales of zero and below it.
    A score is hd / 16 products in fp32, each off by 2^-22 of the sum of its magnitudes at most, and its argument is rounded three times more:
    weights are off by that many times the largest score besides their own rounding."""
    import flashmhf_b200 as fm
    n, heads, kv = [700, 129], 4, 2
    q, k, v = _packed(sum(n), heads, hd, 1, size), _packed(sum(n), kv, hd, 2), _packed(sum(n), kv, hd, 3)
    k = (k * torch.linspace(0.2, 2, sum(n))[:, None, None]).bfloat16()
    want, want_lse, room = _prompt_reference(q, k, v, n, n, scale, True)
    most = float((q.double().abs().amax(0) * 1.0).norm(dim=-1).max() * k.double().norm(dim=-1).max()) * abs(scale)
    off = most * (hd / 16 * 2.0 ** -22 + 3 * 2.0 ** -24)
    o, lse = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), ref.ints(_starts(n)), scale=scale, return_lse=True)
    _close(o, want, room * (1 + 2 * off * 2.0 ** 8), lse, want_lse)


# ------------------------------------------------------------------------------------------------ all of them
def test_two_streams_at_once_and_a_replayed_graph():
    """The three calls in a row, on two streams at once, then captured and replayed with other lengths, pages and prompts: as one by one."""
    import flashmhf_b200 as fm
    hd, kv, heads, P = 64, 2, 4, 16
    cos, sin = ref.tables(600, hd)
    x = _packed(300, heads + 2 * kv, hd, 7).cuda()
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]

    def state(counts, seed):
        rows, n = ref.page_tables([c + 1 for c in counts], P, seed=seed, spare=40 - sum(-(-(c + 1) // P) for c in counts))
        rows = [r + [-1] * (30 - len(r)) for r in rows]
        return _pool(n, kv, P, hd, seed), ref.ints(counts), ref.ints(rows), ref.ints(_starts(counts))

    def run(pages, counts, rows, cu):
        none = torch.zeros_like(counts)
        qr, kr = fm.paged_append(pages, k, v, cos, sin, none, rows, q=q, cu_seqlens=cu, rotated_keys=True)
        o = torch.zeros(300, heads, hd, dtype=torch.bfloat16, device="cuda")
        fm.prompt_attention(qr, kr, v, cu, out=o)
        q1, _ = fm.paged_append(pages, k[:3], v[:3], cos, sin, counts, rows, q=q[:3])
        return o, fm.paged_attention(q1, pages, counts + 1, rows)

    cases = [([100, 3, 190], 1), ([1, 250, 40], 2)]
    want = [run(*state(*c)) for c in cases]
    streams, states = [torch.cuda.Stream() for _ in cases], [state(*c) for c in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(*states[i])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    held = state(*cases[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*held)
    for i in (1, 0, 1):
        for t, new in zip(held[1:], states[i][1:]):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want[i], out))


def test_pages_behind_two_and_four_gigabytes():
    """Offsets of pages that pass 31 and 32 bits, in bytes and in elements."""
    import flashmhf_b200 as fm
    hd, kv, P = 128, 8, 128
    n = 2 ** 32 // (kv * P * hd) + 40
    pages = fm.KVPages.empty(n, kv, P, hd)
    rows = [[n - 1, 3, n // 2 + 1], [n - 7, n // 2 - 1, 5]]
    counts, heads = [300, 270], 8
    x = _packed(sum(counts), heads + 2 * kv, hd, 3).cuda()
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    cos, sin = ref.tables(400, hd)
    fm.paged_append(pages, k, v, cos, sin, ref.ints([0, 0]), ref.ints(rows), cu_seqlens=ref.ints(_starts(counts)))
    small = fm.KVPages(*(t[torch.tensor(sum(rows, []), device="cuda")].clone() if t.dim() == 2 else
                         t.view(torch.uint8)[torch.tensor(sum(rows, []), device="cuda")].clone().view(t.dtype) for t in pages))
    near = [[0, 1, 2], [3, 4, 5]]
    again = fm.KVPages.empty(6, kv, P, hd)
    fm.paged_append(again, k, v, cos, sin, ref.ints([0, 0]), ref.ints(near), cu_seqlens=ref.ints(_starts(counts)))
    for b, (a, m) in enumerate(zip(near, counts)):
        for j, page in enumerate(a):
            rows_here = min(P, m - j * P)
            for one, two in zip(small[:2], again[:2]):
                assert torch.equal(one[page, :, :rows_here].view(torch.uint8), two[page, :, :rows_here].view(torch.uint8))
            assert all(torch.equal(one[page], two[page]) for one, two in zip(small[2:], again[2:]))
    last = q[[counts[0] - 1, sum(counts) - 1]]
    assert torch.equal(fm.paged_attention(last, pages, ref.ints(counts), ref.ints(rows)), fm.paged_attention(last, again, ref.ints(counts), ref.ints(near)))


def test_nothing_to_do():
    import flashmhf_b200 as fm
    pages = fm.KVPages.empty(2, 2, 16, 64)
    cos, sin = ref.tables(4, 64)
    e = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    q, k = fm.paged_append(pages, e(0, 2, 64), e(0, 2, 64), cos, sin, ref.ints([]), ref.ints([]).view(0, 1), q=e(0, 4, 64), rotated_keys=True)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    assert fm.paged_attention(e(0, 4, 64), pages, ref.ints([]), ref.ints([]).view(0, 1)).shape == (0, 4, 64)
    assert fm.prompt_attention(e(0, 4, 64), e(0, 2, 64), e(0, 2, 64), ref.ints([0])).shape == (0, 4, 64)
    o, lse = fm.prompt_attention(e(3, 4, 64).fill_(1), e(0, 2, 64), e(0, 2, 64), ref.ints([0, 3]), ref.ints([0, 0]), return_lse=True)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


def test_indices_out_of_range_are_left_out_and_reported():
    import flashmhf_b200 as fm
    from flashmhf_b200 import _lib
    pages = _pool(3, 1, 16, 64, 0)
    _fill(pages, [40], [[0, 1, 2]], 0)
    q = _packed(1, 2, 64, 0).cuda()

    def reports(call):
        out = call()
        with pytest.raises(_lib.FlashMHFError) as e:
            fm.check_device_status()
        assert e.value.status == -11
        fm.check_device_status()
        return out

    for row, n in (([0, 3, 2], 40), ([0, -1, 2], 40)):
        o = reports(lambda: fm.paged_attention(q, pages, ref.ints([n]), ref.ints([row])))
        assert bool(o.isfinite().all())
    reports(lambda: fm.paged_attention(q, pages, ref.ints([49]), ref.ints([[0, 1, 2]])))
    x, (cos, sin) = _packed(1, 1, 64, 1).cuda(), ref.tables(40, 64)
    before = [t.clone() for t in pages]
    for n, row in ((20, [0, 7, 2]), (20, [0, -5, 2]), (48, [0, 1, 2]), (45, [0, 1, 2]), (2**31 - 1, [0, 1, 2])):
        reports(lambda: fm.paged_append(pages, x, x, cos, sin, ref.ints([n]), ref.ints([row])))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, pages)) or n == 45
    reports(lambda: fm.paged_append(pages, x, x, cos, sin, ref.ints([0]), ref.ints([[0, 1, 2]]), cu_seqlens=ref.ints([0, 2])))
    reports(lambda: fm.prompt_attention(q, x, x, ref.ints([0, 1]), ref.ints([0, 5])))

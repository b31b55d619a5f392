"""Cases of the serving operators: a paged 8-bit key/value cache, what writes it, what reads it, and attention over prompts.

A program that serves the decoder LM packs the prompts of several requests, runs attention over them (`prompt_attention`),
puts their rotated keys and values into pages (`paged_append`), and then generates a token per sequence and step: append, and
attention over the pages (`paged_attention`).  Head layouts are those of the LM configurations in flashmhf_b200/lm.py (12, 16
and 32 heads of 64, as many key/value heads) and generic grouped ones with heads of 96 and 128.

A case is a dict of plain values:

  op         append, decode (attention over pages) or prompt
  B          sequences
  longest    tokens of the longest sequence: already cached (append, decode) or in the prompt (prompt)
  ragged     lengths are spread over 1 .. longest (else all are `longest`); `lens` seeds them, so that they belong to the case
  heads, kv, hd    query heads, key/value heads, head dimension
  page       tokens of a page
  new        append: tokens of the longest new piece, 0 = one token a sequence (a generation step); decode: query tokens a sequence
  causal     prompt: each row sees the keys up to its own
"""
import math
import random

import torch

own = False

#: (heads, kv, hd): the 128M, 370M and 1.3B LMs of flashmhf_b200/lm.py, and grouped layouts.
LAYOUTS = ((12, 12, 64), (16, 16, 64), (32, 32, 64), (32, 8, 128), (32, 4, 128), (24, 8, 96), (16, 2, 64))
E4M3_MAX = 448.0
MIN_EXP = -60           # the smallest scale of a page is 2^-60


def _case(op, name, B, longest, layout, **more):
    c = {"op": op, "B": B, "longest": longest, "ragged": False, "lens": 1, "heads": layout[0], "kv": layout[1], "hd": layout[2], "page": 64, "new": 0,
         "causal": True}
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one generation step of one request through a layer of the 370M model: the shortest call there is
        _case("append", "append_step_1", 1, 777, (16, 16, 64)),
        # one generation step of a large batch with grouped heads; pages at every fill
        _case("append", "append_step_128", 128, 2000, (32, 8, 128), ragged=True),
        # prompts of several requests after earlier turns: pieces that begin and end inside pages
        _case("append", "append_pieces", 7, 1000, (32, 32, 64), ragged=True, new=1601),
        # a full prefill batch of long prompts
        _case("append", "append_prompts_large", 8, 0, (32, 8, 128), new=4096, page=128),
        # one request of the 370M model
        _case("decode", "decode_1", 1, 1023, (16, 16, 64)),
        # a batch of the 1.3B model at uneven lengths
        _case("decode", "decode_32_ragged", 32, 2048, (32, 32, 64), ragged=True),
        # four proposed tokens a sequence are checked in one pass, small pages
        _case("decode", "decode_verify_4", 16, 1500, (24, 8, 96), ragged=True, page=16, new=4),
        # two requests over long documents
        _case("decode", "decode_long_2", 2, 65537, (32, 4, 128)),
        # a full batch at long context: bound by streaming the cache
        _case("decode", "decode_64_large", 64, 8192, (32, 8, 128)),
        # one short prompt of the 128M model
        _case("prompt", "prompt_short", 1, 100, (12, 12, 64)),
        # prompts of very different lengths in one batch of the 370M model
        _case("prompt", "prompt_ragged", 12, 2048, (16, 16, 64), ragged=True),
        # a long prompt with grouped heads
        _case("prompt", "prompt_long", 1, 8192, (32, 8, 128)),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt"])
    layout, page, lens = rng.choice(LAYOUTS), rng.choice([16, 32, 64, 128]), rng.randrange(1, 10**6)
    ragged = rng.random() < 0.7
    if op == "append":
        B = _log(rng, 1, 256)
        if rng.random() < 0.5:
            return _case(op, None, B, rng.randrange(0, 4000), layout, ragged=ragged, lens=lens, page=page)
        new = _log(rng, 2, max(2, 32768 // B))
        return _case(op, None, B, rng.choice([0, rng.randrange(0, 2000)]), layout, ragged=ragged, lens=lens, page=page, new=new)
    if op == "decode":
        B = _log(rng, 1, 128)
        longest = _log(rng, 1, min(100000, 600000 // B))
        while B * longest * layout[1] * layout[2] > 64 * 8192 * 8 * 128:
            longest = longest // 2 + 1
        return _case(op, None, B, longest, layout, ragged=ragged, lens=lens, page=page, new=rng.choice([1, 1, 1, 1, 2, 3, 5, 8]))
    B = _log(rng, 1, 64)
    longest = _log(rng, 1, 8192)
    while B * longest * longest * layout[0] * layout[2] > 8192 * 8192 * 32 * 128 // 2:
        longest = longest * 3 // 4
    return _case(op, None, B, max(1, longest), layout, ragged=ragged, lens=lens, causal=rng.random() < 0.8)


def _spread(case, longest, salt, least):
    """B lengths in least .. longest, one of them the longest; spread over their logarithm where `ragged`."""
    r = random.Random(case["lens"] * 7 + salt)
    B = case["B"]
    if longest <= least or not case["ragged"]:
        return [max(longest, least)] * B
    n = [min(longest, max(least, int(math.exp(r.uniform(math.log(max(least, 1)), math.log(longest + 1)))) - (1 if least == 0 else 0))) for _ in range(B)]
    n[r.randrange(B)] = longest
    return n


def _lengths(case):
    """(tokens in the cache before the call, new tokens of the call) of each sequence."""
    if case["op"] == "append":
        return _spread(case, case["longest"], 1, 0), _spread(case, case["new"], 2, 1) if case["new"] else [1] * case["B"]
    return _spread(case, case["longest"], 1, 1), [max(1, case["new"])] * case["B"]


def _device(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _keys(g, T, heads, hd):
    """Keys as projections make them: a few channels are larger than the rest, and tokens differ in size."""
    channel = 1 + 3 * (torch.rand(heads, hd, device="cuda", generator=g) > 0.95).float()
    return (_randn(g, T, heads, hd) * channel * (0.3 * _randn(g, T, 1, 1)).exp()).bfloat16()


def prepare(case, seed):
    g = _device(seed)
    B, H, n_kv, hd, P = case["B"], case["heads"], case["kv"], case["hd"], case["page"]
    before, new = _lengths(case)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "prompt":
        T = sum(before)
        cu = [0]
        for n in before:
            cu.append(cu[-1] + n)
        # as one projection of the packed tokens lays them out: q, k and v are views of its rows
        qkv = _randn(g, T, H + 2 * n_kv, hd).bfloat16()
        s.update(q=qkv[:, :H], k=qkv[:, H:H + n_kv], v=qkv[:, H + n_kv:], cu=_int32(cu), longest=max(before))
        return s
    total = [a + b for a, b in zip(before, new)] if case["op"] == "append" else before
    need = [-(-n // P) for n in total]
    width, pages = max(need) + 2, sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=g).int()
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    row = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(need, device="cuda"))
    first = torch.tensor([sum(need[:i]) for i in range(B)], device="cuda")
    used = torch.arange(sum(need), device="cuda")
    table[row, used - first[row]] = order[:sum(need)]
    # a cache in use: values of the size that keys and values have, under scales that fit them
    for x in ("k", "v"):
        scale = torch.exp2(torch.randint(-7, -4, (pages, n_kv), device="cuda", generator=g).float())
        codes = (_randn(g, pages, n_kv, P, hd) / scale[:, :, None, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        s[x + "_pages"], s[x + "_scale"] = codes, scale
    s.update(table=table, lengths=_int32(before), longest=max(before))
    if case["op"] == "decode":
        s["q"] = _randn(g, B, new[0], H, hd).bfloat16()
        return s
    T = sum(new)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s.update(q=_randn(g, T, H, hd).bfloat16(), k=_keys(g, T, n_kv, hd), v=_keys(g, T, n_kv, hd), cu=_int32(cu) if case["new"] else None)
    inv = 1.0 / (10000.0 ** (torch.arange(0, hd, 2, device="cuda").double() / hd))
    ang = torch.arange(max(total), device="cuda").double()[:, None] * inv[None]
    s.update(cos=ang.cos().float(), sin=ang.sin().float())
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _where(s, T):
    """Sequence and position of each of the T new tokens."""
    t = torch.arange(T, device="cuda")
    if s["cu"] is None:
        return t, s["lengths"].long()
    b = torch.searchsorted(s["cu"].long(), t, right=True) - 1
    return b, s["lengths"].long()[b] + t - s["cu"].long()[b]


def _rotate(x, c, s):
    x1, x2 = x.float().chunk(2, dim=-1)
    c, s = c[:, None], s[:, None]
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), dim=-1)


def _write(codes, scale, y, page, row, had):
    """Rows y [T, kv, hd] fp32 into their pages; `had` [pages]: rows that a page held before, -1 where the call does not touch it."""
    amax = torch.zeros_like(scale).index_reduce_(0, page, y.abs().amax(-1), "amax")
    m, e = torch.frexp(amax.double() / E4M3_MAX)
    need = torch.exp2(torch.where(m > 0.5, e, e - 1).double().clamp(min=MIN_EXP)).float()
    need = torch.where(amax > 0, need, torch.full_like(need, 2.0 ** MIN_EXP))
    fresh = torch.where((had > 0)[:, None], torch.maximum(scale, need), need)
    now = torch.where((had >= 0)[:, None], fresh, scale)
    P = codes.shape[2]
    old = torch.arange(P, device="cuda")[None, :] < had[:, None]
    again = (codes.float() * (scale / now)[:, :, None, None]).to(torch.float8_e4m3fn)
    raw = torch.where(old[:, None, :, None], again.view(torch.uint8), codes.view(torch.uint8))
    raw[page, :, row] = (y / now[page][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes.view(torch.uint8).copy_(raw)
    scale.copy_(now)


def _plain_append(s):
    T, P = s["k"].shape[0], s["case"]["page"]
    b, pos = _where(s, T)
    page, row = s["table"][b, pos // P].long(), pos % P
    c, sn = s["cos"][pos], s["sin"][pos]
    start = (s["lengths"].long()[b] - pos // P * P).clamp(min=0)       # rows of this token's page that were there before
    had = torch.full((s["k_scale"].shape[0],), -1, device="cuda").index_put_((page,), start)
    q, k = _rotate(s["q"], c, sn), _rotate(s["k"], c, sn)
    _write(s["k_pages"], s["k_scale"], k, page, row, had)
    _write(s["v_pages"], s["v_scale"], s["v"].float(), page, row, had)
    return {"q": q.bfloat16(), "keys": k.bfloat16() if s["cu"] is not None else None}


def _plain_decode(s):
    c, P = s["case"], s["case"]["page"]
    G, nq, L = c["heads"] // c["kv"], s["q"].shape[1], s["longest"]
    pos = torch.arange(L, device="cuda")
    page = s["table"][:, pos // P].long().clamp(min=0)                 # [B, L]
    seen = pos < s["lengths"][:, None]
    read = lambda x: s[x + "_pages"].view(torch.uint8)[page, :, pos % P].view(torch.float8_e4m3fn).float() * s[x + "_scale"][page][..., None]  # noqa: E731
    K = read("k").permute(0, 2, 1, 3)                                  # [B, kv, L, hd]
    V = torch.where(seen[:, :, None, None], read("v"), 0.0).permute(0, 2, 1, 3)
    q = s["q"].float().view(c["B"], nq, c["kv"], G, c["hd"]).permute(0, 2, 3, 1, 4).reshape(c["B"], c["kv"], G * nq, c["hd"])
    i = torch.arange(nq, device="cuda")
    vis = pos[None, None, :] < (s["lengths"][:, None] - (nq - 1 - i)[None, :])[:, :, None]     # [B, nq, L]
    vis = vis[:, None, None].expand(-1, -1, G, -1, -1).reshape(c["B"], 1, G * nq, L)
    a = _softmax(q @ K.transpose(-1, -2) * c["hd"] ** -0.5, vis)
    o = (a @ V).view(c["B"], c["kv"], G, nq, c["hd"]).permute(0, 3, 1, 2, 4).reshape(c["B"], nq, c["heads"], c["hd"])
    return o.bfloat16()


def _softmax(x, visible):
    """Weights of each row over what it sees; zeros where that is nothing."""
    x = x.masked_fill(~visible, -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    return x.div_(x.sum(-1, keepdim=True).clamp(min=1e-30))


def _plain_prompt(s):
    c, L, cu = s["case"], s["longest"], s["cu"].long()
    G, T = c["heads"] // c["kv"], s["q"].shape[0]
    n = cu[1:] - cu[:-1]
    at = torch.arange(L, device="cuda")
    inside = at[None] < n[:, None]                                     # [B, L]
    row = (cu[:-1, None] + at[None]).clamp(max=T - 1)
    q, k, v = (s[x].float()[row].transpose(1, 2) for x in "qkv")       # [B, heads, L, hd]
    v = torch.where(inside[:, None, :, None], v, 0.0)
    see = inside[:, None, None, :]
    if c["causal"]:
        see = see & (at[None, :] <= at[:, None])[None, None]
    x = (q.reshape(c["B"], c["kv"], G * L, c["hd"]) @ k.transpose(-1, -2)).view(c["B"], c["heads"], L, L)
    a = _softmax(x.mul_(c["hd"] ** -0.5), see)
    o = (a.view(c["B"], c["kv"], G * L, L) @ v).view(c["B"], c["heads"], L, c["hd"])
    return o.transpose(1, 2)[inside].bfloat16()


def run(s):
    if own:
        import flashmhf_b200 as fm
        if s["op"] == "prompt":
            return fm.prompt_attention(s["q"], s["k"], s["v"], s["cu"], causal=s["case"]["causal"])
        pages = fm.KVPages(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
        if s["op"] == "decode":
            return fm.paged_attention(s["q"], pages, s["lengths"], s["table"])
        q, keys = fm.paged_append(pages, s["k"], s["v"], s["cos"], s["sin"], s["lengths"], s["table"], q=s["q"], cu_seqlens=s["cu"],
                                  rotated_keys=s["cu"] is not None)
        out = {"q": q, "keys": keys}
    elif s["op"] == "append":
        out = _plain_append(s)
    else:
        return _plain_decode(s) if s["op"] == "decode" else _plain_prompt(s)
    # the cache as it is now: codes (as the numbers they are) and the power of two that multiplies each page and head
    return {**out, **{x: s[x] for x in ("k_pages", "v_pages", "k_scale", "v_scale")}}


def work(case):
    before, new = _lengths(case)
    H, n_kv, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "prompt":
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in before)
        return {"bytes": sum(before) * hd * 2 * (2 * H + 2 * n_kv), "flops": 4 * H * hd * pairs}
    if case["op"] == "decode":
        nq = new[0]
        return {"bytes": sum(before) * n_kv * hd * 2 + 2 * case["B"] * nq * H * hd * 2, "flops": 4 * sum(before) * H * nq * hd}
    T = sum(new)
    moved = 2 * H * 2 + 2 * n_kv * 2 + 2 * n_kv + (2 * n_kv if case["new"] else 0)      # q in and out, k and v in, codes out, rotated keys out
    positions = min(T, max(a + b for a, b in zip(before, new)))
    return {"bytes": T * hd * moved + positions * hd * 4, "flops": T * hd * (3 * H + 5 * n_kv)}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _to_e4m3(x):
    """x in 64 bits to the nearest number with 3 bits behind the point and exponents from -6, ties to even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(s):
    P, hd = s["case"]["page"], s["case"]["hd"]
    before, new = _lengths(s["case"])
    table = s["table"].cpu().tolist()
    out = {x: s[x].double() for x in ("k_pages", "v_pages", "k_scale", "v_scale")}
    q, keys, first = [], [], 0
    for b, (n0, n) in enumerate(zip(before, new)):
        p = torch.arange(n0, n0 + n, device="cuda")
        z = torch.complex(s["cos"][p].double(), s["sin"][p].double())[:, None]
        turn = lambda x: (lambda y: torch.cat((y.real, y.imag), -1))(torch.complex(x[..., :hd // 2].double(), x[..., hd // 2:].double()) * z)  # noqa: E731
        part = slice(first, first + n)
        first += n
        q.append(turn(s["q"][part]))
        keys.append(turn(s["k"][part]))
        for name, y in (("k", keys[-1]), ("v", s["v"][part].double())):
            codes, scale = out[name + "_pages"], out[name + "_scale"]
            for j in range(n0 // P, (n0 + n - 1) // P + 1):
                lo, hi = max(n0, j * P), min(n0 + n, (j + 1) * P)
                page, had = table[b][j], lo - j * P
                rows = y[lo - n0:hi - n0].transpose(0, 1)              # [kv, rows, hd]
                top = rows.abs().amax((1, 2))
                n2 = torch.round(torch.log2(top / E4M3_MAX))           # off by one either way at most: put right below, without logarithms
                n2 = torch.where(top <= E4M3_MAX * torch.exp2(n2 - 1), n2 - 1, torch.where(top <= E4M3_MAX * torch.exp2(n2), n2, n2 + 1))
                want = torch.exp2(n2.clamp(min=MIN_EXP))
                now = torch.maximum(scale[page], want) if had else want
                codes[page, :, :had] = _to_e4m3(codes[page, :, :had] * (scale[page] / now)[:, None, None])
                codes[page, :, had:had + hi - lo] = _to_e4m3(rows / now[:, None, None])
                scale[page] = now
    return {"q": torch.cat(q), "keys": torch.cat(keys) if s["cu"] is not None else None, **out}


def _attend(q, k, v, visible, scale):
    """One head: softmax(scale q k^T) v over what is visible, in 64 bits."""
    x = (q @ k.T * scale).masked_fill(~visible, -math.inf)
    w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
    return torch.nan_to_num(w, nan=0.0) @ v


def exact(case, seed):
    s = prepare(case, seed)
    H, n_kv, hd, P = case["heads"], case["kv"], case["hd"], case["page"]
    G, scale = H // n_kv, 1 / math.sqrt(hd)
    before, new = _lengths(case)
    if case["op"] == "append":
        touched = sum((a + n - 1) // P - a // P + 1 for a, n in zip(before, new))
        return _exact_append(s) if touched < 6000 else None
    if case["B"] * H > 4500:
        return None
    if case["op"] == "decode":
        nq = new[0]
        o = torch.zeros(case["B"], nq, H, hd, dtype=torch.float64, device="cuda")
        for b, n in enumerate(before):
            page = s["table"][b, :-(-n // P)].long()
            pos = torch.arange(n, device="cuda")
            vis = pos[None] < torch.arange(n - nq + 1, n + 1, device="cuda")[:, None]
            for h in range(n_kv):
                k, v = ((s[x + "_pages"].view(torch.uint8)[page, h].view(torch.float8_e4m3fn).double() * s[x + "_scale"][page, h].double()[:, None, None]).reshape(-1, hd)[:n]
                        for x in "kv")
                qs = s["q"][b, :, h * G:(h + 1) * G].double().reshape(nq * G, hd)
                o[b, :, h * G:(h + 1) * G] = _attend(qs, k, v, vis.repeat_interleave(G, 0), scale).view(nq, G, hd)
        return o
    o, first = torch.zeros(sum(before), H, hd, dtype=torch.float64, device="cuda"), 0
    for n in before:
        at = torch.arange(n, device="cuda")
        vis = at[None] <= at[:, None] if case["causal"] else torch.ones(n, n, dtype=torch.bool, device="cuda")
        for h in range(H):
            q, k, v = (s[x][first:first + n, i].double() for x, i in (("q", h), ("k", h // G), ("v", h // G)))
            o[first:first + n, h] = _attend(q, k, v, vis, scale)
        first += n
    return o

"""The token mixer's operators as a decoder's serving loop calls them: block
tables and slot maps for a step's requests, rotary positions written through
to a paged key-value cache, attention of one new token over that cache, and
linear attention with a decay for each head over a recurrent state.

``run`` computes a pass in elementary torch operations, or, with ``own``
true, through ``runnel_amd.native``.  ``exact`` restates each operator in 64
bits from its definition.
"""

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn

# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one decode step's bookkeeping of a small batch: pure latency
        dict(name="tables: 8 decoding", op="tables", requests=8, cached_lo=31, cached_hi=4000,
             new_lo=1, new_hi=1, page=16, pad=0),
        # a step that takes up new prompts next to running ones, padded to a fixed token budget
        dict(name="tables: 509 mixed", op="tables", requests=509, cached_lo=0, cached_hi=9000,
             new_lo=1, new_hi=700, page=32, pad=1003),
        # the token of a batch-1 decode, positions of the three axes equal in kind but far along
        dict(name="rotary: 1 token", op="rotary", tokens=1, pad=0, q_heads=16, kv_heads=2, dim=128,
             rot=64, axes=3, woven=True, adjacent=False, page=16, bits=16, far=200000),
        # a long prompt of video frames (the 8192-token prefill), 8-bit cache, padded rows
        dict(name="rotary: 8192 video", op="rotary", tokens=8189, pad=3, q_heads=16, kv_heads=4, dim=128,
             rot=128, axes=3, woven=False, adjacent=False, page=32, bits=8, far=9000),
        # batch-1 decode over a short context: latency
        dict(name="attention: 1 x 1000", op="attention", requests=1, lo=1000, hi=1000, q_heads=16,
             kv_heads=2, dim=128, page=16, bits=16, window=0),
        # batch-1 decode far into a long context: the split over the cache's length carries it
        dict(name="attention: 1 x 131071", op="attention", requests=1, lo=131071, hi=131071, q_heads=16,
             kv_heads=2, dim=256, page=64, bits=16, window=0),
        # a serving batch of uneven contexts, 8-bit cache
        dict(name="attention: 61 ragged", op="attention", requests=61, lo=17, hi=16000, q_heads=32,
             kv_heads=8, dim=128, page=32, bits=8, window=0),
        # a large batch, one head of keys for each of queries, a window over the last keys
        dict(name="attention: 256 windowed", op="attention", requests=256, lo=700, hi=4100, q_heads=16,
             kv_heads=16, dim=64, page=16, bits=16, window=1024),
        # the recurrent form: one token of one request
        dict(name="linear: 1 token", op="linear", requests=1, lo=1, hi=1, k_heads=16, v_heads=32,
             dk=128, dv=128, delta=True, slots=3),
        # the recurrent form over a serving batch
        dict(name="linear: 127 tokens", op="linear", requests=127, lo=1, hi=1, k_heads=16, v_heads=32,
             dk=128, dv=128, delta=True, slots=140),
        # prompts of uneven lengths in one packed batch, decay only
        dict(name="linear: 9 prompts", op="linear", requests=9, lo=5, hi=1500, k_heads=16, v_heads=16,
             dk=128, dv=64, delta=False, slots=9),
        # one long prompt (the 8192-token prefill)
        dict(name="linear: 8192 tokens", op="linear", requests=1, lo=8192, hi=8192, k_heads=16, v_heads=32,
             dk=128, dv=128, delta=True, slots=1),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "rotary", "attention", "attention", "linear", "linear"])
    if op == "tables":
        new_hi = rng.choice([1, _between(rng, 2, 700)])
        return dict(op=op, requests=_between(rng, 1, 509), cached_lo=rng.choice([0, 1, 31]),
                    cached_hi=_between(rng, 32, 9000), new_lo=rng.choice([0, 1]) if new_hi > 1 else 1,
                    new_hi=new_hi, page=rng.choice([8, 16, 32, 64]), pad=rng.choice([0, _between(rng, 1, 1003)]))
    if op == "rotary":
        kv = rng.choice([1, 2, 4])
        dim = rng.choice([64, 96, 128, 192, 256])
        return dict(op=op, tokens=_between(rng, 1, 5000 if dim > 128 else 8189), pad=rng.choice([0, 1, 5]),
                    q_heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim, rot=rng.choice([32, 64, dim]),
                    axes=rng.choice([1, 3]), woven=rng.random() < 0.5, adjacent=rng.random() < 0.3,
                    page=rng.choice([8, 16, 32, 64]), bits=rng.choice([16, 8]), far=_between(rng, 100, 200000))
    if op == "attention":
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 8, 16])
        hi = _between(rng, 16, 60000)
        most = max(1, min(200, 60000 * 8 // (hi * kv)))
        return dict(op=op, requests=_between(rng, 1, most), lo=rng.choice([1, hi // 16 + 1, hi]), hi=hi,
                    q_heads=heads, kv_heads=kv, dim=rng.choice([64, 96, 128, 192, 256]),
                    page=rng.choice([8, 16, 32, 64]), bits=rng.choice([16, 8]),
                    window=rng.choice([0, 0, _between(rng, 1, 4096)]))
    prompt = rng.random() < 0.6
    hi = _between(rng, 2, 4000) if prompt else 1
    kh = rng.choice([2, 4, 8, 16])
    requests = _between(rng, 1, max(1, min(12, 8000 // hi))) if prompt else _between(rng, 1, 127)
    return dict(op=op, requests=requests, lo=rng.choice([1, hi // 4 + 1, hi]), hi=hi, k_heads=kh,
                v_heads=kh * rng.choice([1, 2]), dk=rng.choice([64, 128]), dv=rng.choice([32, 64, 96, 128]),
                delta=rng.random() < 0.7, slots=requests + rng.choice([0, 5]))


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, even steps of their logarithm."""
    if n == 1:
        return [hi]
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [min(hi, max(lo, int(round(math.exp(a + (b - a) * i / (n - 1)) - 1)))) for i in range(n)]


def _pages_of(length, page):
    return -(-length // page)


def work(case):
    op = case["op"]
    if op == "tables":
        R, page = case["requests"], case["page"]
        cached = _spread(R, case["cached_lo"], case["cached_hi"])
        new = _spread(R, case["new_lo"], case["new_hi"])
        tokens = sum(new)
        pages = sum(_pages_of(c + n, page) - _pages_of(c, page) for c, n in zip(cached, new))
        rows = tokens + case["pad"]
        return {"bytes": 8 * R + 8 * pages + 16 * rows + 4 * (R + 1) + 4 * R + 12, "flops": 0}
    if op == "rotary":
        n, hq, hk, d, rot = (case[k] for k in ("tokens", "q_heads", "kv_heads", "dim", "rot"))
        held = 1 if case["bits"] == 8 else 2
        return {"bytes": n * (hq * d * 4 + 2 * hk * d * (2 + held) + 4 * case["axes"] + 8),
                "flops": n * (hq + hk) * rot * 3}
    if op == "attention":
        held = 1 if case["bits"] == 8 else 2
        lens = _spread(case["requests"], case["lo"], case["hi"])
        if case["window"]:
            lens = [min(x, case["window"]) for x in lens]
        keys, hq, hk, d, R = sum(lens), case["q_heads"], case["kv_heads"], case["dim"], case["requests"]
        return {"bytes": 2 * keys * hk * d * held + R * hq * d * 4
                + 4 * sum(_pages_of(x, case["page"]) for x in lens), "flops": 4 * keys * hq * d}
    lens = _spread(case["requests"], case["lo"], case["hi"])
    n, kh, vh, dk, dv = sum(lens), case["k_heads"], case["v_heads"], case["dk"], case["dv"]
    gates = 8 if case["delta"] else 4
    return {"bytes": n * (4 * kh * dk + 4 * vh * dv + gates * vh) + 8 * len(lens) * vh * dk * dv,
            "flops": n * vh * dk * dv * (8 if case["delta"] else 5)}


# ----------------------------------------------------------------- the inputs


def _rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _perm(g, n):
    return torch.randperm(n, generator=g, device=DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _held(x, bits):
    return x.to(FP8) if bits == 8 else x.to(BF16)


def prepare(case, seed):
    return _PREPARE[case["op"]](case, _rng(seed))


def _prepare_tables(case, g):
    R, page = case["requests"], case["page"]
    cached = _ints(_spread(R, case["cached_lo"], case["cached_hi"]))[_perm(g, R)]
    new = _ints(_spread(R, case["new_lo"], case["new_hi"]))[_perm(g, R)]
    width = _pages_of(case["cached_hi"] + case["new_hi"], page) + 1
    pages = R * width + 7
    ids = _perm(g, pages).to(torch.int32)
    owned = (torch.arange(width, device=DEV)[None] * page) < cached[:, None]
    table = torch.where(owned, ids[:R * width].view(R, width), -1).contiguous()
    mine = torch.zeros(pages, dtype=torch.bool, device=DEV)
    mine[table[owned].long()] = True
    return dict(case=case, cached=cached, new=new, table=table,
                free=ids[~mine[ids.long()]].contiguous(),
                rows=sum(_spread(R, case["new_lo"], case["new_hi"])) + case["pad"])


def _positions(case, g, rows):
    """Positions of text (equal along the axes) or, for several axes, of a
    run of frames of 24 x 32 patches behind a text."""
    start = int(torch.randint(0, case["far"], (1,), generator=g, device=DEV))
    i = torch.arange(rows, device=DEV)
    if case["axes"] == 1:
        return (start + i).to(torch.int32)[None]
    return (start + torch.stack([i // 768, i // 32 % 24, i % 32])).to(torch.int32)


def _sections(case):
    half = case["rot"] // 2
    if case["axes"] == 1:
        return (half,)
    side = half // 3
    return (half - 2 * side, side, side)


def _prepare_rotary(case, g):
    n, rows, hk, d, page = case["tokens"], case["tokens"] + case["pad"], case["kv_heads"], case["dim"], case["page"]
    pages = _pages_of(n, page) + 3
    slots = torch.full((rows,), -1, dtype=torch.int64, device=DEV)
    order = _perm(g, pages)
    i = torch.arange(n, device=DEV) + 1  # (a prompt that goes on behind a cached token)
    slots[:n] = order[i // page] * page + i % page
    half = case["rot"] // 2
    inv = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    packed = _randn(g, rows, case["q_heads"] + 2 * hk, d).to(BF16)  # one projection's output
    q, k, v = packed.split([case["q_heads"], hk, hk], dim=1)
    return dict(case=case, q=q, k=k, v=v, positions=_positions(case, g, rows), inv_freq=inv.float(), slots=slots,
                k_cache=_held(_randn(g, pages, hk, page, d), case["bits"]),
                v_cache=_held(_randn(g, pages, hk, page, d), case["bits"]),
                k_scale=0.03125 if case["bits"] == 8 else 1.0, v_scale=0.0625 if case["bits"] == 8 else 1.0)


def _prepare_attention(case, g):
    R, hk, d, page = case["requests"], case["kv_heads"], case["dim"], case["page"]
    lens = _spread(R, case["lo"], case["hi"])
    width = _pages_of(case["hi"], page)
    pages = sum(_pages_of(x, page) for x in lens) + 5
    lengths = _ints(lens)[_perm(g, R)]
    ids = _perm(g, pages).to(torch.int32)
    owned = (torch.arange(width, device=DEV)[None] * page) < lengths[:, None]
    at = (owned.reshape(-1).cumsum(0) - 1).clamp(min=0).view(R, width)
    table = torch.where(owned, ids[at], -1).contiguous()

    def cache():  # page by page: a whole cache in 32 bits is large
        return torch.cat([_held(_randn(g, min(256, pages - p), hk, page, d), case["bits"])
                          for p in range(0, pages, 256)])

    # queries whose scores have the spread of trained heads (a few keys carry most)
    q = (2.5 * _randn(g, R, case["q_heads"], d)).to(BF16)
    return dict(case=case, q=q, k_cache=cache(), v_cache=cache(), table=table, lengths=lengths,
                scale=d ** -0.5, k_scale=0.5 if case["bits"] == 8 else 1.0,
                v_scale=0.25 if case["bits"] == 8 else 1.0)


def _prepare_linear(case, g):
    R, kh, vh, dk, dv = (case[k] for k in ("requests", "k_heads", "v_heads", "dk", "dv"))
    lens = _ints(_spread(R, case["lo"], case["hi"]))[_perm(g, R)]
    n = sum(_spread(R, case["lo"], case["hi"]))
    cu = torch.zeros(R + 1, dtype=torch.int32, device=DEV)
    cu[1:] = lens.cumsum(0)
    q, k = (torch.nn.functional.normalize(_randn(g, n, kh, dk), dim=-1).to(BF16) for _ in range(2))
    v = _randn(g, n, vh, dv).to(BF16)
    if case["delta"]:  # gates of each token: decays from almost none to strong ones
        rate = torch.exp(torch.empty(vh, device=DEV).uniform_(-4.0, 1.5, generator=g))
        decay = -rate * torch.nn.functional.softplus(_randn(g, n, vh))
        beta = torch.sigmoid(1.5 * _randn(g, n, vh))
    else:  # a fixed rate of each head
        decay = (-(2.0 ** -torch.linspace(1, 8, vh, device=DEV))).expand(n, vh)
        beta = None
    state = 0.3 * _randn(g, case["slots"], vh, dk, dv)
    return dict(case=case, q=q, k=k, v=v, decay=decay, beta=beta, cu=cu, lens=lens, state=state,
                state_out=torch.zeros_like(state), index=_perm(g, case["slots"])[:R].to(torch.int32),
                scale=dk ** -0.5)


_PREPARE = {"tables": _prepare_tables, "rotary": _prepare_rotary, "attention": _prepare_attention,
            "linear": _prepare_linear}


# ------------------------------------------------------------------- the pass


def run(s):
    if own:
        from runnel_amd import native
        return _OWN[s["case"]["op"]](native, s)
    return _PLAIN[s["case"]["op"]](s)


def _values(cache, scale):
    """What a cache holds, as the values it stands for."""
    return (cache.float() * scale).to(BF16) if cache.dtype == FP8 else cache


def _own_tables(native, s):
    t = native.paged_tables(s["cached"], s["new"], s["table"], s["free"], s["case"]["page"], s["rows"])
    return dict(table=s["table"], slots=t.slots, positions=t.positions, requests=t.requests,
                cu=t.cu_seqlens, lengths=t.lengths, counts=t.counts)


def _own_rotary(native, s):
    c = s["case"]
    q = native.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_cache"], s["v_cache"],
                             s["slots"], sections=_sections(c), woven=c["woven"], adjacent=c["adjacent"],
                             k_scale=s["k_scale"], v_scale=s["v_scale"])
    return dict(q=q, k_cache=_values(s["k_cache"], s["k_scale"]), v_cache=_values(s["v_cache"], s["v_scale"]))


def _own_attention(native, s):
    return native.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], scale=s["scale"],
                                  window=s["case"]["window"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_linear(native, s):
    o = native.linear_attention(s["q"], s["k"], s["v"], s["decay"], s["cu"], s["state"], beta=s["beta"],
                                state_index=s["index"], scale=s["scale"], state_out=s["state_out"])
    return dict(out=o, state=s["state_out"])


_OWN = {"tables": _own_tables, "rotary": _own_rotary, "attention": _own_attention, "linear": _own_linear}


def _plain_tables(s):
    page, table, free = s["case"]["page"], s["table"], s["free"].long()
    c, n = s["cached"].long(), s["new"].long()
    R, width = table.shape
    have, need = (c + page - 1) // page, (c + n + page - 1) // page
    take = (need.clamp(max=width) - have).clamp(min=0)
    first = take.cumsum(0) - take
    j = torch.arange(width, device=DEV)[None] - have[:, None]
    at = first[:, None] + j
    given = torch.where(at < len(free), free[at.clamp(0, len(free) - 1)], -1)
    table.copy_(torch.where((j >= 0) & (j < take[:, None]), given, table.long()))
    cu = torch.zeros(R + 1, dtype=torch.int64, device=DEV)
    cu[1:] = n.cumsum(0)
    i = torch.arange(s["rows"], device=DEV)
    live = i < cu[-1]
    r = torch.searchsorted(cu[1:], i, right=True).clamp(max=R - 1)
    pos = c[r] + i - cu[r]
    entry = pos // page
    held = table[r, entry.clamp(0, width - 1)].long()
    slots = torch.where(live & (entry < width) & (held >= 0), held * page + pos % page, -1)
    total = take.sum()
    counts = torch.stack([cu[-1], total.clamp(max=len(free)), (total - len(free)).clamp(min=0)])
    return dict(table=table, slots=slots, positions=torch.where(live, pos, 0).to(torch.int32),
                requests=torch.where(live, r, -1).to(torch.int32), cu=cu.to(torch.int32),
                lengths=(c + n).to(torch.int32), counts=counts.to(torch.int32))


def _axis_of(case):
    """The axis of positions that each frequency turns by."""
    half, sections = case["rot"] // 2, _sections(case)
    i = torch.arange(half, device=DEV)
    if len(sections) == 1:
        return torch.zeros_like(i)
    if not case["woven"]:  # one block of frequencies after the other
        return (i >= sections[0]).long() + (i >= sections[0] + sections[1]).long()
    turn = i % 3  # in turn, until an axis has had its share; the first has the rest
    share = torch.tensor(sections, device=DEV)[turn]
    return torch.where(i // 3 < share, turn, 0)


def _turn(x, cos, sin, case):
    rot = case["rot"]
    x = x.float() if cos.dtype == torch.float32 else x.double()
    cos, sin = cos[:, None], sin[:, None]
    head, rest = x[..., :rot], x[..., rot:]
    if case["adjacent"]:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([head, rest], dim=-1)


def _plain_rotary(s):
    c = s["case"]
    n, page = c["tokens"], c["page"]
    # far positions: the angle in 64 bits, its cosine and sine in 32
    angle = s["positions"].double()[_axis_of(c)].T * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    q, k = _turn(s["q"], cos, sin, c), _turn(s["k"], cos, sin, c)
    slots = s["slots"][:n]
    at = ((slots // page)[:, None], torch.arange(c["kv_heads"], device=DEV)[None], (slots % page)[:, None])
    for cache, x, scale in ((s["k_cache"], k, s["k_scale"]), (s["v_cache"], s["v"].float(), s["v_scale"])):
        x = x[:n] / scale
        if cache.dtype == FP8:
            cache.view(torch.uint8)[at] = x.clamp(-448, 448).to(FP8).view(torch.uint8)
        else:
            cache[at] = x.to(BF16)
    return dict(q=q.to(BF16), k_cache=_values(s["k_cache"], s["k_scale"]), v_cache=_values(s["v_cache"], s["v_scale"]))


def _plain_attention(s):
    c, q = s["case"], s["q"].float()
    R, hq, d = q.shape
    hk = c["kv_heads"]
    pages = s["table"].clamp(min=0).long()

    def keys(cache, scale):  # [R, hk, keys, d]
        x = cache.view(torch.uint8)[pages].view(FP8) if cache.dtype == FP8 else cache[pages]
        x = x.permute(0, 2, 1, 3, 4).float() * scale
        return x.reshape(R, hk, -1, d)

    scores = torch.matmul(q.view(R, hk, hq // hk, d), keys(s["k_cache"], s["k_scale"]).transpose(-1, -2)) * s["scale"]
    j = torch.arange(scores.shape[-1], device=DEV)
    live = j < s["lengths"][:, None]
    if c["window"]:
        live &= j >= s["lengths"][:, None] - c["window"]
    scores = scores.masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, keys(s["v_cache"], s["v_scale"])) / p.sum(-1, keepdim=True)
    return out.reshape(R, hq, d).to(BF16)


def _plain_linear(s):
    c = s["case"]
    R, T, vh, dk, dv = c["requests"], c["hi"], c["v_heads"], c["dk"], c["dv"]
    C = min(64, T)
    pad = -(-T // C) * C
    t = torch.arange(pad, device=DEV)
    live = t < s["lens"][:, None]
    at = torch.where(live, s["cu"][:-1, None] + t, 0).long()

    def rows(x, heads):  # [R, v_heads, pad, width], zeros behind a sequence's end
        x = torch.where(live[..., None, None], x[at].float(), 0.0).transpose(1, 2)
        return x.repeat_interleave(vh // heads, dim=1)

    q, k, v = rows(s["q"], c["k_heads"]) * s["scale"], rows(s["k"], c["k_heads"]), rows(s["v"], vh)
    g = rows(s["decay"][..., None], vh)[..., 0]
    b = rows(s["beta"][..., None], vh) if c["delta"] else None
    index = s["index"].long()
    S = s["state"][index]
    eye = torch.eye(C, device=DEV)
    outs = []
    for i in range(0, pad, C):  # the state passes from chunk to chunk
        Q, K, U, G = q[:, :, i:i + C], k[:, :, i:i + C], v[:, :, i:i + C], g[:, :, i:i + C].double().cumsum(-1)
        D = torch.exp((G[..., :, None] - G[..., None, :]).float().tril()).tril()
        if b is not None:
            B = b[:, :, i:i + C]
            A = (B * torch.matmul(K, K.transpose(-1, -2)) * D).tril(-1)
            U = torch.linalg.solve_triangular(eye + A, B * (U - G.exp().float()[..., None] * torch.matmul(K, S)),
                                              upper=False, unitriangular=True)
        outs.append(G.exp().float()[..., None] * torch.matmul(Q, S)
                    + torch.matmul(torch.matmul(Q, K.transpose(-1, -2)) * D, U))
        left = torch.exp(G[..., -1:] - G).float()[..., None]
        S = G[..., -1].exp().float()[..., None, None] * S + torch.matmul(K.transpose(-1, -2), left * U)
    s["state_out"][index] = S
    o = torch.cat(outs, dim=2).transpose(1, 2).to(BF16)
    n = s["q"].shape[0]
    r = torch.searchsorted(s["cu"][1:].long(), torch.arange(n, device=DEV), right=True)
    return dict(out=o[r, torch.arange(n, device=DEV) - s["cu"].long()[r]], state=s["state_out"])


_PLAIN = {"tables": _plain_tables, "rotary": _plain_rotary, "attention": _plain_attention, "linear": _plain_linear}


# ------------------------------------------------------- the results in 64 bits


def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _exact_tables(case, s):
    return None  # whole numbers


def _exact_rotary(case, s):
    n, page, hk = case["tokens"], case["page"], case["kv_heads"]
    axis = _axis_of(case)
    angle = torch.stack([s["positions"][int(a)].double() * s["inv_freq"][i].double() for i, a in enumerate(axis)], -1)
    q, k = (_turn(s[x], angle.cos(), angle.sin(), case) for x in ("q", "k"))
    out = dict(q=q)
    for name, x in (("k", k), ("v", s["v"].double())):
        cache = (s[name + "_cache"].double() * s[name + "_scale"]).transpose(1, 2).reshape(-1, hk, case["dim"])
        if case["bits"] == 8:  # (what a rounding to 3 bits would give, and not its border's other side)
            x = (x / s[name + "_scale"]).clamp(-448, 448)
            x = x.float().to(FP8).double() * s[name + "_scale"]
        cache[s["slots"][:n]] = x[:n]
        out[name + "_cache"] = cache.view(-1, page, hk, case["dim"]).transpose(1, 2)
    return out


def _exact_attention(case, s):
    R, hq, d = s["q"].shape
    hk, page = case["kv_heads"], case["page"]
    out = torch.zeros((R, hq, d), dtype=torch.float64, device=DEV)
    for r in range(R):
        n = int(s["lengths"][r])
        first = max(0, n - case["window"]) if case["window"] else 0
        pages = s["table"][r, first // page:-(-n // page)].long()
        for h in range(hk):
            k, v = ((s[x].view(torch.uint8)[pages, h].view(FP8) if case["bits"] == 8 else s[x][pages, h])
                    .double().reshape(-1, d)[first % page:n - first // page * page] for x in ("k_cache", "v_cache"))
            mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
            w = torch.softmax(s["q"][r, mine].double() @ k.T * (s["scale"] * s["k_scale"]), dim=-1)
            out[r, mine] = w @ v * s["v_scale"]
    return out


def _exact_linear(case, s):
    R, vh = case["requests"], case["v_heads"]
    each = vh // case["k_heads"]
    index, cu = s["index"].long(), s["cu"].long()
    S = s["state"][index].double()
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV)
    for t in range(case["hi"]):  # token by token
        live = torch.nonzero(s["lens"] > t)[:, 0] if case["lo"] != case["hi"] else torch.arange(R, device=DEV)
        at = cu[live] + t
        q, k = (s[x][at].double().repeat_interleave(each, dim=1) for x in "qk")
        u = s["v"][at].double()
        now = S[live] * s["decay"][at].double().exp()[..., None, None]
        if case["delta"]:
            u = s["beta"][at].double()[..., None] * (u - torch.matmul(k[..., None, :], now)[..., 0, :])
        now += k[..., :, None] * u[..., None, :]
        out[at] = torch.matmul(q[..., None, :], now)[..., 0, :] * s["scale"]
        S[live] = now
    state = s["state_out"].double()
    state[index] = S
    return dict(out=out, state=state)


_EXACT = {"tables": _exact_tables, "rotary": _exact_rotary, "attention": _exact_attention, "linear": _exact_linear}

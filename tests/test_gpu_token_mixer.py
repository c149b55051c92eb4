"""The token mixer's operators on the GPU against their definitions in 64
bits (tests/mixer_ref.py): block tables, rotary positions, the paged cache's
write and its attention, linear attention, and a decoder's use of them
together, eager, on two streams and captured."""

import numpy as np
import pytest
import torch

import mixer_ref as M

pytestmark = pytest.mark.gpu
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def native():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from runnel_amd import _lib, native
    _lib.load()
    return native


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g)


def close(got, ref, tol, name=""):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, the worst by "
                           f"{(got - ref).abs()[bad].max().item():.3g}")


# ---------------------------------------------------------------- refusals


def test_no_rows(native):
    """Calls of no row at all, of no request and of no sequence."""
    def z(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    x, i, c, inv = z(0, 2, 64), z(0, dtype=torch.int32), z(3, 2, 16, 64), z(32, dtype=torch.float32)
    assert [t.shape for t in native.rotary(x, x, i, inv)] == [(0, 2, 64)] * 2
    assert native.rotary_append(x, x, x, i, inv, c, c.clone(), i.long()).shape == (0, 2, 64)
    out, lse = native.paged_attention(x, c, c, z(0, 9, dtype=torch.int32), i, return_lse=True)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    g, st = z(0, 2, dtype=torch.float32), torch.ones(2, 2, 64, 64, device="cuda")
    for cu in ([0], [0, 0, 0]):
        out = native.linear_attention(x, x, x, g, torch.tensor(cu, device="cuda"), st, beta=g)
        assert out.shape == (0, 2, 64) and bool((st == 1).all())
    t = native.paged_tables(z(2, dtype=torch.int32), z(2, dtype=torch.int32), z(2, 3, dtype=torch.int32), i, 16, 0)
    assert t.slots.numel() == 0 and t.counts.tolist() == [0, 0, 0]


def test_wrapper_checks(native):
    """The checks that stand between a tensor and its address."""
    def z(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    c, q, table, lens = z(4, 2, 16, 64), z(1, 2, 64), z(1, 3, dtype=torch.int32), z(1, dtype=torch.int32)

    def attend(k=c, v=c, q=q, table=table, lens=lens, **kw):
        return native.paged_attention(q, k, v, table, lens, **kw)

    turned = z(4, 2, 64, 16).transpose(2, 3)
    for why, kw in (("one type and shape", dict(v=c[:3])), ("one type and shape", dict(v=c.to(E4M3))),
                    ("lie in memory alike", dict(v=z(4, 16, 2, 64).transpose(1, 2))),
                    ("contiguous", dict(k=turned, v=turned)), ("belong to float8", dict(k_scale=0.5)),
                    ("must be bfloat16 or float8", dict(k=c.half(), v=c.half())),
                    ("cache must be", dict(k=c[0], v=c[0])),
                    ("q must be", dict(q=z(1, 2, 96))), ("bfloat16", dict(q=z(1, 2, 64, dtype=torch.float32))),
                    ("block_table must be", dict(table=table[0])), ("block_table must be", dict(table=table[:0])),
                    ("block_table must be int32", dict(table=table.float())),
                    ("lengths must be", dict(lens=z(2, dtype=torch.int32))),
                    ("window", dict(window=-1)), ("window is out of range", dict(window=1 << 33)),
                    ("multiple of the 2 key heads", dict(q=z(1, 3, 64))),
                    ("GPU tensors", dict(q=q.cpu())), ("GPU tensors", dict(lens=lens.cpu())),
                    ("no backward pass", dict(q=q.clone().requires_grad_()))):
        with pytest.raises(ValueError, match=why):
            attend(**kw)
    with torch.no_grad():
        attend(q=q.clone().requires_grad_())
    with pytest.raises(TypeError):
        attend(window=None)
    with pytest.raises(RuntimeError, match="ambiguous"):
        attend(return_lse=z(2))
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode() as fake, pytest.raises(ValueError, match="dispatch to Python"):
        attend(lens=fake.from_tensor(lens))  # has no memory
    # a dimension of one: its stride says nothing
    one = z(1, 2, 16, 64).as_strided((1, 2, 16, 64), (7, 1024, 64, 1))
    assert attend(k=c[:1], v=one).shape == (1, 2, 64)

    inv, pos, x = z(32, dtype=torch.float32), z(2, dtype=torch.int32), z(2, 3, 64)
    for why, args in (("multiple of 8", (z(2, 3, 60), x, pos, inv)), ("k must be", (x, z(3, 3, 64), pos, inv)),
                      ("k must be", (x, z(2, 3, 96), pos, inv)),
                      ("1 to 4 axes", (x, x, z(5, 2, dtype=torch.int32), inv, (8, 8, 8, 4, 4))),
                      ("positions must be", (x, x, pos, inv, (16, 16))),
                      ("int32", (x, x, pos.float(), inv)), ("float32", (x, x, pos, inv.double())),
                      ("contiguous float32", (x, x, pos, z(64, dtype=torch.float32)[::2])),
                      ("sum to half", (x, x, z(2, 2, dtype=torch.int32), inv, (16, 15)))):
        with pytest.raises(ValueError, match=why):
            native.rotary(*args)
    with pytest.raises(TypeError):
        native.rotary(x, x, z(2, 2, dtype=torch.int32), inv, (16, "16"))

    flat = z(3 * 64 * 64 + 64, dtype=torch.float32)
    g, cu, st = z(2, 3, dtype=torch.float32), torch.tensor([0, 2], device="cuda"), z(1, 3, 64, 64, dtype=torch.float32)

    def linear(q=x, k=x, v=x, g=g, cu=cu, st=st, **kw):
        return native.linear_attention(q, k, v, g, cu, st, **kw)

    for why, kw in (("log_decay must be float32", dict(g=g.to(BF16))), ("log_decay must be", dict(g=g[:1])),
                    ("beta must be", dict(beta=g[:, :2])), ("cu_seqlens must be", dict(cu=cu[:0])),
                    ("state must be contiguous", dict(st=st.transpose(2, 3))),
                    ("state_out must be contiguous", dict(state_out=st[:, :2])),
                    ("lie apart", dict(st=flat[:-64].view(1, 3, 64, 64), state_out=flat[64:].view(1, 3, 64, 64))),
                    ("slots for 2 sequences", dict(cu=torch.tensor([0, 1, 2], device="cuda"))),
                    ("state_index must be", dict(state_index=z(2, dtype=torch.int32)))):
        with pytest.raises(ValueError, match=why):
            linear(**kw)
    assert native.linear_attention(x, x, x, g[:1].expand(2, 3), cu, st).shape == (2, 3, 64)

    i = z(2, dtype=torch.int32)
    for why, args in (("block_table must be int32", (i, i, z(2, 4, dtype=torch.int64), i, 16, 2)),
                      ("contiguous", (i, i, z(4, 2, dtype=torch.int32).t(), i, 16, 2)),
                      ("cached must be", (i[:1], i, z(2, 4, dtype=torch.int32), i, 16, 2)),
                      ("rows must not be negative", (i, i, z(2, 4, dtype=torch.int32), i, 16, -1)),
                      ("page_size", (i, i, z(2, 4, dtype=torch.int32), i, 12, 2))):
        with pytest.raises(ValueError, match=why):
            native.paged_tables(*args)


# ---------------------------------------------------------------- the tables


TABLES = [
    # cached, added, page, width, free pages, rows
    ([0], [1], 16, 4, 3, 1),
    ([16, 15, 17], [1, 1, 1], 16, 4, 8, 3),           # at, before and behind a page's end
    ([0, 5, 0, 40], [0, 0, 7, 0], 8, 6, 4, 10),       # nothing to do for most; padded rows
    ([3, 0, 100], [60, 129, 31], 32, 8, 20, 230),
    ([10, 10, 10], [30, 30, 30], 8, 8, 5, 90),        # the free list runs out inside a request
    ([10, 60], [30, 30], 8, 6, 30, 60),               # past the table's width
    ([-4, 2], [5, -3], 8, 4, 4, 8),                   # negative counts as none
    ([7, 0], [50, 50], 16, 8, 40, 33),                # fewer rows than tokens
    ([0, 0], [9, 9], 8, 4, 0, 18),                    # no page left at all
    ([5, 9], [0, 0], 8, 4, 3, 0),                     # no row
    ([1, 2], [1, 1], 8, 0, 3, 2),                     # a table without entries
]


@pytest.mark.parametrize("case", TABLES, ids=range(len(TABLES)))
def test_tables(native, case):
    cached, added, page, width, free, rows = case
    R = len(cached)
    rng = np.random.default_rng(R + page)
    ids = rng.permutation(R * width + free + 1).astype(np.int32)
    table = ids[:R * width].reshape(R, width).copy()
    free = ids[R * width:R * width + free]
    dev = torch.from_numpy(table.copy()).cuda()
    t = native.paged_tables(torch.tensor(cached).cuda(), torch.tensor(added, dtype=torch.int32).cuda(),
                            dev, torch.from_numpy(free.copy()).cuda(), page, rows)
    ref = M.tables(cached, added, table, free, page, rows)
    for got, want in zip((dev, t.slots, t.positions, t.requests, t.cu_seqlens, t.lengths, t.counts), ref):
        assert np.array_equal(got.cpu().numpy(), want)
    assert t.slots.dtype == torch.int64


@pytest.mark.parametrize("R,hi,page", [(1, 5000, 8), (255, 40, 16), (257, 90, 64), (4096, 3, 8)])
def test_tables_many(native, R, hi, page):
    rng = np.random.default_rng(R)
    cached, added = rng.integers(0, hi, R), rng.integers(0, hi, R)
    width = -(-2 * hi // page) + 1
    table = np.full((R, width), -7, dtype=np.int32)
    for r in range(R):
        table[r, :-(-cached[r] // page)] = rng.integers(0, 1000, -(-cached[r] // page))
    free = rng.permutation(R * width).astype(np.int32) + 2000000000  # slots past 32 bits
    rows = int(added.sum()) + 5
    # a view into a wider table: its rows lie apart
    wide = torch.full((R, width + 3), -9, dtype=torch.int32)
    wide[:, :width] = torch.from_numpy(table)
    dev = wide.cuda()
    t = native.paged_tables(torch.from_numpy(cached).cuda(), torch.from_numpy(added).cuda(), dev[:, :width],
                            torch.from_numpy(free).cuda(), page, rows)
    ref = M.tables(cached, added, table, free, page, rows)
    assert np.array_equal(dev[:, :width].cpu().numpy(), ref[0]) and bool((dev[:, width:] == -9).all())
    for got, want in zip((t.slots, t.positions, t.requests, t.cu_seqlens, t.lengths, t.counts), ref[1:]):
        assert np.array_equal(got.cpu().numpy(), want)


def test_tables_sums_that_pass_32_bits(native):
    """The running sums stay at the largest value instead of wrapping."""
    big = 2 ** 31 - 1
    t = native.paged_tables(torch.tensor([big, 0], dtype=torch.int32).cuda(),
                            torch.tensor([big, 5], dtype=torch.int32).cuda(),
                            torch.zeros((2, 1), dtype=torch.int32).cuda(),
                            torch.zeros(1, dtype=torch.int32).cuda(), 1024, 4)
    assert t.cu_seqlens.tolist() == [0, big, big] and t.lengths.tolist() == [big, 5]
    assert t.slots.tolist() == [-1] * 4 and t.requests.tolist() == [0] * 4


# ------------------------------------------------------------------- rotary


ROTARY = [
    # N, Hq, Hk, D, half, sections, woven, adjacent
    (1, 1, 1, 64, 32, None, False, False),
    (5, 4, 2, 128, 64, (24, 20, 20), False, False),
    (3, 3, 1, 96, 16, (6, 5, 5), True, False),
    (1030, 2, 1, 96, 48, (16, 16, 16), True, True),   # four tokens a workgroup, the last with two
    (2, 2, 2, 256, 128, (32, 32, 32, 32), False, True),
    (4, 1, 1, 256, 32, (0, 32), False, False),
    (2, 5, 5, 72, 8, None, False, True),
]


def rotary_inputs(seed, N, hq, hk, D, half, sections, far=200000):
    g = gen(seed)
    axes = 1 if sections is None else len(sections)
    packed = randn(g, N, hq + 2 * hk, D).to(BF16)
    positions = torch.randint(-5, far, (axes, N), generator=g)
    inv = (10000.0 ** (-torch.arange(half) / half)).float()
    return packed, positions, inv


def rotary_tol(x, ref, half, adjacent):
    """One rounding to bf16 of two fp32 products and their sum; the cosine
    and sine within 2^-22 (an angle reduced in 64 bits, rounded to 32, and the
    functions' own error), so 2^-20 of |a| + |b| holds all of it."""
    x = x.double().abs()
    pair = torch.zeros_like(x)
    i = torch.arange(half)
    lo, hi = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    pair[..., lo] = pair[..., hi] = x[..., lo] + x[..., hi]
    return 2.0 ** -8 * ref.abs() + 2.0 ** -20 * pair


@pytest.mark.parametrize("case", ROTARY, ids=range(len(ROTARY)))
def test_rotary(native, case):
    N, hq, hk, D, half, sections, woven, adjacent = case
    packed, positions, inv = rotary_inputs(N, N, hq, hk, D, half, sections)
    d = packed.cuda()
    pos = positions.cuda() if sections else positions[0].cuda()
    q, k = native.rotary(d[:, :hq], d[:, hq:hq + hk], pos, inv.cuda(), sections, woven, adjacent)
    for got, x in ((q, packed[:, :hq]), (k, packed[:, hq:hq + hk])):
        ref = M.rotary(x, positions, inv, sections or (half,), woven, adjacent)
        close(got, ref, rotary_tol(x, ref, half, adjacent))
        assert torch.equal(got[..., 2 * half:].cpu(), x[..., 2 * half:])


def test_rotary_odd_views(native):
    """Rows that no 16-byte load can take are copied first; positions of
    another type and stride."""
    g = gen(3)
    x = randn(g, 6, 4, 131).to(BF16)
    inv = (10000.0 ** (-torch.arange(32) / 32)).float()
    pos = torch.arange(12)[::2]
    d = x.cuda()
    q, k = native.rotary(d[:, :, 1:129], d[:, :2, 3:131], pos.cuda(), inv.cuda())
    for got, y in ((q, x[:, :, 1:129]), (k, x[:, :2, 3:131])):
        ref = M.rotary(y, pos[None], inv, (32,))
        close(got, ref, rotary_tol(y, ref, 32, False))


def cache_of(g, pages, hk, page, D, bits, layout):
    """A cache with leftovers (NaN among them) in the given memory order."""
    x = randn(g, pages, hk, page, D)
    x[..., ::7] = float("nan")
    x = x.to(E4M3 if bits == 8 else BF16).cuda()
    if layout == "rows":  # heads of one token next to each other
        base = torch.zeros((pages, page, hk, D), dtype=x.dtype, device="cuda")
        view = base.transpose(1, 2)
    elif layout == "pair":  # both caches in one tensor, page by page
        base = torch.zeros((pages, 2, hk, page, D), dtype=x.dtype, device="cuda")
        view = base[:, 0]
    else:
        return x
    if bits == 8:
        view.view(torch.uint8).copy_(x.view(torch.uint8))
    else:
        view.copy_(x)
    return view


def raw(t):
    return t.view(torch.uint8 if t.dtype == E4M3 else torch.int16)


@pytest.mark.parametrize("bits,layout", [(16, "heads"), (16, "rows"), (8, "heads"), (8, "pair")])
@pytest.mark.parametrize("N,hq,hk,D,page", [(1, 4, 1, 64, 8), (37, 6, 3, 96, 16), (1500, 2, 2, 128, 32),
                                            (9, 4, 2, 256, 64)])
def test_rotary_append(native, N, hq, hk, D, page, bits, layout):
    half = 16 if D == 96 else D // 2
    sections = (half - 2 * (half // 3), half // 3, half // 3)
    packed, positions, inv = rotary_inputs(N + D, N, hq, hk, D, half, sections)
    g = gen(N)
    pages = -(-N // page) + 2
    kc, vc = cache_of(g, pages, hk, page, D, bits, layout), cache_of(g, pages, hk, page, D, bits, layout)
    slots = torch.randperm(pages * page, generator=g)[:N]
    slots[::5] = -1
    if N > 3:
        slots[3] = pages * page  # behind the cache
    before = raw(kc).cpu().clone(), raw(vc).cpu().clone()
    ks, vs = (0.125, 0.02) if bits == 8 else (1.0, 1.0)
    d = packed.cuda()
    q = native.rotary_append(d[:, :hq], d[:, hq:hq + hk], d[:, hq + hk:], positions.cuda(), inv.cuda(), kc, vc,
                             slots.cuda(), sections, k_scale=ks, v_scale=vs)
    ref = M.rotary(packed[:, :hq], positions, inv, sections)
    close(q, ref, rotary_tol(packed[:, :hq], ref, half, False))
    live = (slots >= 0) & (slots < pages * page)
    at, off = slots[live] // page, slots[live] % page
    for cache, x, old, scale, turned in ((kc, packed[:, hq:hq + hk], before[0], ks, True),
                                         (vc, packed[:, hq + hk:], before[1], vs, False)):
        x = x[live]
        ref = M.rotary(x, positions[:, live], inv, sections) if turned else x.double()
        tol = rotary_tol(x, ref, half, False) if turned else torch.zeros_like(ref)
        if bits == 8:  # half a step of 3 bits, of the smallest step below 2^-6; saturating
            tol = tol + 2.0 ** -4 * ref.abs() + 2.0 ** -10 * scale * 1.0001 + 2.0 ** -22 * ref.abs()
            ref = ref.clamp(-448 * scale, 448 * scale)
        got = cache.cpu()
        close(got[at, :, off].double() * scale, ref, tol)
        now = raw(got).clone()
        now[at, :, off] = old[at, :, off]
        assert torch.equal(now, old)  # nothing else was written


def test_append_special_values(native):
    """NaN stays NaN; in 8 bits infinities and large values saturate."""
    x = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38, -1e5, 448.0, 464.0, 0.0] * 8)
    x = x.to(BF16).view(1, 1, 64).cuda()
    inv = torch.zeros(8, device="cuda")  # no pair turns: cos 1, sin 0, but inf * 0 is NaN
    for dtype in (BF16, E4M3):
        kc, vc = (torch.zeros((1, 1, 8, 64), dtype=dtype, device="cuda") for _ in range(2))
        native.rotary_append(x, x, x, torch.zeros(1, dtype=torch.int32, device="cuda"), inv, kc, vc,
                             torch.tensor([5], device="cuda"))
        got, want = vc[0, 0, 5].cpu().float(), x[0, 0].cpu().float()
        if dtype == E4M3:
            want = want.clamp(-448, 448)
        assert torch.equal(got.isnan(), want.isnan())
        both = [x.nan_to_num(7.0, float("inf"), -float("inf")) for x in (got, want)]
        assert torch.equal(*both)
        tail = kc[0, 0, 5, 16:].cpu().float()
        assert torch.equal(tail.isnan(), want[16:].isnan())


def test_append_refuses_one_cache(native):
    """Keys and values into one place: either could be left there."""
    x, c = torch.zeros(1, 1, 64, dtype=BF16, device="cuda"), torch.zeros(1, 1, 8, 64, dtype=BF16, device="cuda")
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    for k, v, why in ((c, c.view(1, 1, 8, 64), "must be two"), (c.expand(4, 1, 8, 64), c.expand(4, 1, 8, 64), "expanded")):
        with pytest.raises(ValueError, match=why):
            native.rotary_append(x, x, x, i, torch.zeros(8, device="cuda"), k, v, i.long())


# ---------------------------------------------------------------- attention


def attention_inputs(seed, lens, hq, hk, D, page, bits, layout="heads", width=None):
    g = gen(seed)
    R = len(lens)
    need = [-(-max(n, 0) // page) for n in lens]
    width = max(max(need), 1) if width is None else width
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((R, width), -1, dtype=torch.int32)
    p = 0
    for r, n in enumerate(need):
        n = min(n, width)
        table[r, :n] = ids[p:p + n]
        p += n
    kc, vc = (cache_of(g, pages, hk, page, D, bits, layout) for _ in range(2))
    for c in (kc, vc):  # real values where a key is, leftovers elsewhere
        x = randn(g, pages, hk, page, D).to(c.dtype)
        live = torch.zeros(pages, page, dtype=torch.bool)
        for r, n in enumerate(lens):
            for j in range(min(max(n, 0), width * page)):
                live[table[r, j // page], j % page] = True
        new = torch.where(live[:, None, :, None], raw(x), raw(c).cpu())
        raw(c).copy_(new)
    q = (2 * randn(g, R, hq, D)).to(BF16)
    return q, kc, vc, table, torch.tensor(lens, dtype=torch.int32)


def check_attention(native, q, kc, vc, table, lengths, window=0, ks=1.0, vs=1.0, scale=None):
    D = q.shape[2]
    out, lse = native.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), scale=scale, window=window,
                                      k_scale=ks, v_scale=vs, return_lse=True)
    scale = D ** -0.5 if scale is None else scale
    ref, rlse, size, unit = M.attention(q, kc.cpu().float(), vc.cpu().float(), table, lengths, scale, window, ks, vs)
    # a score: D products summed in fp32 and a scaling, each within 2^-24 of
    # the sum of magnitudes; its error e turns a weight by a factor of e^e,
    # and the sum of the weights likewise.  Then 2^-8 for the weights'
    # rounding to bf16 (of v's weighted magnitude) and 2^-8 for the output's;
    # 2^-18 holds the fp32 sums, exponentials and quotients.
    e = (D + 4) * 2.0 ** -24 * unit[..., None]
    close(out, ref, 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -18 + 2.1 * e) * size, "out")
    some = torch.isfinite(rlse)
    assert torch.equal(torch.isfinite(lse.cpu()), some) and not lse.isnan().any()
    assert bool((lse.cpu()[~some] == -torch.inf).all())
    tol = e[..., 0] + 2.0 ** -20 * (1 + rlse.abs())
    assert bool(((lse.cpu().double() - rlse).abs()[some] <= tol[some]).all())
    assert bool((out.cpu()[~some] == 0).all())
    plain = native.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda(), scale=scale, window=window,
                                   k_scale=ks, v_scale=vs)
    assert torch.equal(plain, out)  # equal calls, equal bits
    return out


LENS = [0, 1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_attention_lengths(native, D, bits):
    """Every length around a tile's and a page's ends, NaN behind each."""
    ks, vs = (0.25, 2.0) if bits == 8 else (1.0, 1.0)
    check_attention(native, *attention_inputs(D + bits, LENS, 4, 2, D, 8, bits), ks=ks, vs=vs)


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (16, 1), (17, 1), (40, 1), (5, 5), (24, 2)])
def test_attention_groups(native, hq, hk):
    check_attention(native, *attention_inputs(hq, [50, 1, 0, 200], hq, hk, 64, 16, 16))
    check_attention(native, *attention_inputs(hq, [50, 1, 0, 200], hq, hk, 256, 16, 8))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 299, 300, 1000])
def test_attention_window(native, window):
    """Pages that only keys before the window are on may be gone from the
    table, or taken by other requests."""
    q, kc, vc, table, lengths = attention_inputs(window, LENS, 4, 2, 128, 16, 16)
    for r, n in enumerate(LENS):
        gone = max(0, n - window) // 16
        table[r, :gone] = torch.tensor([-1, 10 ** 6, 0])[torch.arange(gone) % 3].to(torch.int32)
    check_attention(native, q, kc, vc, table, lengths, window=window)


@pytest.mark.parametrize("layout,page,bits", [("rows", 32, 16), ("pair", 64, 8), ("rows", 1024, 8)])
def test_attention_layouts(native, layout, page, bits):
    check_attention(native, *attention_inputs(page, [1, 70, 0, 64, 333], 8, 2, 128, page, bits, layout))


def test_attention_long(native):
    """Split over many workgroups, the lengths uneven."""
    check_attention(native, *attention_inputs(1, [9001, 3, 0, 4500], 6, 2, 128, 16, 16))
    check_attention(native, *attention_inputs(2, [20011], 2, 1, 64, 32, 8), ks=0.5, vs=0.5)


@pytest.mark.parametrize("R", [2, 3, 64, 65, 200, 256, 257])
@pytest.mark.parametrize("bits", [16, 8])
def test_attention_ragged(native, R, bits):
    """A long request or two among short and empty ones, whose parts lie
    anywhere among all requests': in one, two and four runs of 64 requests,
    and more requests than are looked through."""
    lens = [(0, 1, 33, 5, 190, 0, 64)[i * 5 % 7] for i in range(R)]
    lens[R // 2], lens[-1] = 2500, 1300
    if R > 70:
        lens[63], lens[64] = 700, 0
    check_attention(native, *attention_inputs(R, lens, 3, 1, 64, 32, bits))
    # all without a key but one, none at all
    q, kc, vc, table, lengths = attention_inputs(R, lens, 3, 1, 64, 32, bits)
    for keep in (R // 2, None):
        some = torch.tensor([n if i == keep else 0 for i, n in enumerate(lens)], dtype=torch.int32)
        check_attention(native, q, kc, vc, table, some)


@pytest.mark.parametrize("R,hk,D", [(2, 1, 256), (21, 2, 256), (40, 3, 192)])
def test_attention_ragged_wide(native, R, hk, D):
    """Wide heads, whose parts are counted in whole rounds of workgroups."""
    lens = [(40, 1, 0, 150, 65)[i % 5] for i in range(R)]
    lens[1] = 1200
    check_attention(native, *attention_inputs(D + R, lens, 2 * hk, hk, D, 16, 16 if R < 40 else 8))


@pytest.mark.parametrize("hq,hk", [(40, 2), (6, 6)])
def test_attention_ragged_heads(native, hq, hk):
    """Several heads of keys, and more than a tile of query heads to one."""
    lens = [3, 2100, 0, 40, 900, 1, 2, 65, 350]
    check_attention(native, *attention_inputs(5, lens, hq, hk, 64, 16, 16))
    check_attention(native, *attention_inputs(5, lens, hq, hk, 64, 16, 16), window=777)


def test_attention_bad_pages(native):
    """Pages outside the cache, a length past the table and one below 0."""
    q, kc, vc, table, lengths = attention_inputs(5, [100, 100, 64, 40], 4, 2, 64, 8, 16)
    table[0, 3], table[0, 5], table[1, 0] = -1, 10 ** 9, len(kc)
    table[2] = -1
    check_attention(native, q, kc, vc, table, lengths)
    lengths[0], lengths[3] = 10 ** 8, -5
    live = native.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    lengths[0], lengths[3] = table.shape[1] * 8, 0
    same = native.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    assert torch.equal(torch.nan_to_num(live), torch.nan_to_num(same))
    # no table at all
    none = native.paged_attention(q.cuda(), kc, vc, table.cuda()[:, :0], lengths.cuda())
    assert bool((none == 0).all())


@pytest.mark.parametrize("dtype", [E4M3, BF16])
def test_cache_past_32_bits(native, dtype):
    """Pages whose values lie more than 2^31 values (bf16: 2^32 bytes) into
    the cache, written and read; the pages between are nobody's."""
    pages, page, D = 32800, 1024, 64
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 9 GB of the GPU's memory")
    kc, vc = (torch.empty((pages, 1, page, D), dtype=dtype, device="cuda") for _ in range(2))
    ids = [pages - 1, 3, pages - 2]
    for c in (kc, vc):
        raw(c)[ids] = 0
    g = gen(3)
    N = 2 * page + 100
    x = randn(g, N, 3, D).to(BF16).cuda()
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    t = native.paged_tables(torch.zeros(1, dtype=torch.int32, device="cuda"),
                            torch.tensor([N], dtype=torch.int32, device="cuda"), table.clone(),
                            table[0], page, N)
    inv = torch.zeros(8, device="cuda")
    q = native.rotary_append(x[:, :1], x[:, 1:2], x[:, 2:], t.positions, inv, kc, vc, t.slots)
    small = [c[torch.tensor(ids, device="cuda")] if dtype == BF16 else raw(c)[ids].view(dtype) for c in (kc, vc)]
    want = x[:, 1:].to(dtype).cpu().float()
    for i in range(2):
        flat = small[i].cpu().float().reshape(-1, D)
        assert torch.equal(flat[:N], want[:, i]) and bool((flat[N:] == 0).all())
    last = q[-1:].cpu()
    near = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    ref = check_attention(native, last, *small, near, t.lengths.cpu())
    got = native.paged_attention(last.cuda(), kc, vc, table, t.lengths)
    assert torch.equal(got, ref)  # the same values in other places


def test_attention_peaked_scores(native):
    """Scores far apart (one key carries all), of both signs, and all equal."""
    q, kc, vc, table, lengths = attention_inputs(8, [200, 33], 4, 4, 64, 8, 16)
    check_attention(native, (q * 20).to(BF16), kc, vc, table, lengths)
    check_attention(native, q, kc, vc, table, lengths, scale=-0.3)
    check_attention(native, q, kc, vc, table, lengths, scale=0.0)


def test_attention_strided(native):
    """A query that is a slice of a packed projection, a table that is a
    slice of a wider one, lengths of another type."""
    q, kc, vc, table, lengths = attention_inputs(9, [20, 90, 5], 4, 2, 128, 16, 16)
    ref = native.paged_attention(q.cuda(), kc, vc, table.cuda(), lengths.cuda())
    packed = torch.zeros(3, 8, 128, dtype=BF16, device="cuda")
    packed[:, 2:6] = q.cuda()
    wide = torch.full((3, table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = table.cuda()
    got = native.paged_attention(packed[:, 2:6], kc, vc, wide[:, 2:2 + table.shape[1]], lengths.cuda().long())
    assert torch.equal(got, ref)


# --------------------------------------------------------- linear attention


def linear_inputs(seed, lens, kh, vh, dk, dv, delta=True, slots=None, decay="mixed", lead=0, tail=0):
    g = gen(seed)
    N, R = lead + sum(lens) + tail, len(lens)
    q, k = (torch.nn.functional.normalize(randn(g, N, kh, dk), dim=-1).to(BF16) for _ in range(2))
    v = randn(g, N, vh, dv).to(BF16)
    if decay == "mixed":
        a = -torch.exp(torch.empty(N, vh).uniform_(-8, 2, generator=g))
        a[::17] = -torch.inf   # a state forgotten
        a[5::11] = -3.0e38
        a[3::13] = 0.0
    else:
        a = torch.full((1, vh), float(decay)).expand(N, vh)
    beta = torch.sigmoid(2 * randn(g, N, vh)) if delta else None
    if delta:
        beta[::7], beta[1::9] = 1.0, 0.0
    cu = torch.tensor([lead] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)
    state = randn(g, R if slots is None else slots, vh, dk, dv)
    return q, k, v, a, cu, state, beta


def check_linear(native, q, k, v, a, cu, state, beta, index=None, scale=None, inplace=False):
    dk, T = q.shape[2], int((cu[1:] - cu[:-1]).max())
    dev = state.cuda()
    keep = None if inplace else torch.full_like(dev, 7.0)
    out = native.linear_attention(q.cuda(), k.cuda(), v.cuda(), a.cuda(), cu.cuda(), dev,
                                  beta=None if beta is None else beta.cuda(),
                                  state_index=None if index is None else index.cuda(), scale=scale, state_out=keep)
    ref, final, size, fsize = M.linear(q, k, v, a, cu, state, beta, index, scale)
    # two pieces of 8 bits (2^-15 each of a factor, on both of q S and P U),
    # the exponentials and the sums' fp32 (dk + 64 terms), then the rounding
    close(out, ref, 2.0 ** -8 * ref.abs() + (2.0 ** -13 + (dk + 64) * 2.0 ** -23) * size, "out")
    used = set(range(len(cu) - 1)) if index is None else {int(i) for i in index if 0 <= int(i) < len(state)}
    got = (dev if inplace else keep).cpu()
    for i in range(len(state)):
        if i in used:
            # every token adds at most (dk + 64 + 16) roundings of 2^-24 of the
            # terms' magnitude; a token's update shrinks what came before
            close(got[i], final[i], (T + 1) * (dk + 80) * 2.0 ** -24 * fsize[i].amax() + 1e-30, f"state {i}")
            # (and as a whole they are far from all adding up)
            rel = (got[i].double() - final[i]).norm() / final[i].norm().clamp(min=1e-30)
            assert rel <= 2.0 ** -24 * 4 * (dk * (T + 1)) ** 0.5, rel
        else:
            assert torch.equal(got[i], state[i] if inplace else torch.full_like(got[i], 7.0))
    if not inplace:
        assert torch.equal(dev.cpu(), state)
    return out


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [0], [0, 3, 1], [2, 5, 7, 16]])
def test_linear_tokens(native, lens, delta):
    """The recurrent form."""
    for dk, dv, kh, vh in ((128, 128, 2, 4), (64, 16, 1, 3), (128, 48, 2, 2)):
        check_linear(native, *linear_inputs(dk + dv, lens, kh, vh, dk, dv, delta))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lens", [[17], [63], [64], [65], [128], [200], [0, 100, 0], [130, 1, 64, 0, 129]])
def test_linear_chunks(native, lens, delta):
    for dk, dv, kh, vh in ((128, 32, 2, 4), (64, 16, 1, 3)):
        check_linear(native, *linear_inputs(dk + lens[0], lens, kh, vh, dk, dv, delta))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("R", [3, 300])
def test_linear_mixed(native, R, delta):
    """Single tokens, a few and prompts in one batch: by token and in chunks
    in one call, with 300 sequences more than a workgroup lists at once."""
    lens = [[1, 9, 70], [0, 8, 33], [130, 2, 1]][R % 3] if R == 3 else [
        (1, 24, 0, 25, 1, 2, 65, 1, 1, 17)[i * 7 % 10] for i in range(R)]
    kh, vh, dv = (1, 2, 16) if R == 3 else (2, 4, 64)
    check_linear(native, *linear_inputs(R, lens, kh, vh, 64, dv, delta))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lens", [[131], [70, 130, 26, 66], [65, 30, 3, 129]])
@pytest.mark.parametrize("dk", [64, 128])
def test_linear_many_states(native, lens, dk, delta):
    """More states than the chip takes at once, which go through the chunks by
    32 columns: one sequence, several, and several of which one turns out to
    be short, so that by 16 saves a round."""
    vh = 64 if len(lens) == 1 else 32
    check_linear(native, *linear_inputs(dk, lens, 8, vh, dk, 128, delta))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("decay", [0.0, -1e-4, -0.3, -40.0, -float("inf")])
def test_linear_decays(native, decay, delta):
    """One rate for a head, expanded over the tokens: none, slow, and so
    strong that every state is forgotten at once."""
    x = linear_inputs(11, [150, 40], 1, 2, 64, 32, delta, decay=decay)
    check_linear(native, *x)


def test_linear_equal_keys(native):
    """The delta rule's triangular system at its worst conditioned: all keys
    alike, beta 1, no decay."""
    q, k, v, a, cu, state, beta = linear_inputs(4, [130], 1, 1, 128, 16, decay=0.0)
    k[:] = k[:1]
    beta[:] = 1.0
    check_linear(native, q, k, v, a, cu, state, beta)


@pytest.mark.parametrize("lens", [[3, 1, 2], [90, 1, 70]])
@pytest.mark.parametrize("inplace", [True, False])
def test_linear_slots(native, lens, inplace):
    """States of a pool by index, one sequence without a slot, another's
    index past the pool, rows in front of and behind the sequences."""
    x = linear_inputs(6, lens, 1, 2, 64, 32, slots=9, lead=3, tail=70)
    out = check_linear(native, *x, index=torch.tensor([7, -1, 2]), inplace=inplace, scale=0.7)
    assert bool((out[:3] == 0).all()) and bool((out[-70:] == 0).all())
    check_linear(native, *x, index=torch.tensor([0, 9, 8]), inplace=inplace)


@pytest.mark.parametrize("T", [1, 70])
def test_linear_state_past_32_bits(native, T):
    """A slot more than 2^31 values into the pool of states."""
    vh, slots = 32, 4100
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 9 GB of the GPU's memory")
    q, k, v, a, cu, state, beta = (x.cuda() for x in linear_inputs(8, [T, T], 16, vh, 128, 128))
    pool = torch.empty((slots, vh, 128, 128), device="cuda")
    at = torch.tensor([slots - 1, 2], dtype=torch.int32, device="cuda")
    pool[slots - 1], pool[2] = state[0], state[1]
    pool[slots - 2] = 5.0
    got = native.linear_attention(q, k, v, a, cu, pool, beta=beta, state_index=at)
    ref = native.linear_attention(q, k, v, a, cu, state, beta=beta)
    assert torch.equal(got, ref)
    assert torch.equal(pool[slots - 1], state[0]) and torch.equal(pool[2], state[1])
    assert bool((pool[slots - 2] == 5.0).all())


def test_linear_strided(native):
    """q, k and v as slices of one projection, gates with strides."""
    q, k, v, a, cu, state, beta = linear_inputs(2, [100], 2, 2, 64, 64)
    ref = native.linear_attention(q.cuda(), k.cuda(), v.cuda(), a.cuda(), cu.cuda(), state.cuda(), beta=beta.cuda())
    packed = torch.cat([q, k, v], dim=1).cuda()
    gates = torch.stack([a, beta], dim=-1).cuda()
    got = native.linear_attention(packed[:, :2], packed[:, 2:4], packed[:, 4:], gates[..., 0], cu.cuda().long(),
                                  state.cuda(), beta=gates[..., 1])
    assert torch.equal(ref, got)


def test_linear_other_sequences_nan(native):
    """A NaN in one sequence reaches no other, in chunks and by tokens."""
    for lens in ([70, 70, 70], [2, 2, 2]):
        q, k, v, a, cu, state, beta = linear_inputs(8, lens, 1, 2, 64, 16)
        n = lens[0]
        ref, fin = native.linear_attention, state.cuda()
        clean = ref(q.cuda(), k.cuda(), v.cuda(), a.cuda(), cu.cuda(), fin, beta=beta.cuda())
        for x in (q, k, v):
            x[n + 1] = float("nan")
        a, beta = a.clone(), beta.clone()
        a[n], beta[n] = float("nan"), float("inf")
        bad = state.cuda()
        out = ref(q.cuda(), k.cuda(), v.cuda(), a.cuda(), cu.cuda(), bad, beta=beta.cuda())
        for part in (slice(0, n), slice(2 * n, 3 * n)):
            assert torch.equal(out[part], clean[part])
        assert torch.equal(bad[0], fin[0]) and torch.equal(bad[2], fin[2]) and bad[1].isnan().any()
        assert out[n + 1:2 * n].isnan().any()


def test_linear_pieces(native):
    """A prompt in chunks, then token by token, is the whole sequence."""
    q, k, v, a, cu, state, beta = linear_inputs(12, [140], 2, 4, 128, 32, decay=-0.05)
    d = [x.cuda() for x in (q, k, v, a, beta)]
    whole = state.cuda()
    native.linear_attention(*d[:4], cu.cuda(), whole, beta=d[4])
    parts, outs = state.cuda(), []
    for lo, hi in ((0, 100), (100, 137), (137, 138), (138, 140)):
        c = torch.tensor([0, hi - lo], dtype=torch.int32).cuda()
        outs.append(native.linear_attention(*[x[lo:hi] for x in d[:4]], c, parts, beta=d[4][lo:hi]))
    ref, final, size, fsize = M.linear(q, k, v, a, cu, state, beta)
    close(torch.cat(outs), ref, 2.0 ** -8 * ref.abs() + (2.0 ** -13 + 192 * 2.0 ** -23) * size)
    close(parts, final, 141 * 208 * 2.0 ** -24 * fsize.amax())
    close(whole, final, 141 * 208 * 2.0 ** -24 * fsize.amax())


# ------------------------------------------------------------ used together


class Serving:
    """A layer's attention over a paged cache for a few requests: what a
    serving loop keeps, and one step of it."""

    def __init__(self, native, hq, hk, D, page, requests, pages, rows, seed):
        g = gen(seed)
        self.native, self.page, self.rows, self.shape = native, page, rows, (hq, hk, D)
        self.kc, self.vc = (torch.full((pages, hk, page, D), float("nan"), dtype=BF16, device="cuda")
                            for _ in range(2))
        self.table = torch.full((requests, pages // requests), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=g).to(torch.int32).cuda()
        self.cached = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.added = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.inv = (1e6 ** (-torch.arange(D // 4) / (D // 4))).float().cuda()
        self.qkv = torch.zeros(rows, hq + 2 * hk, D, dtype=BF16, device="cuda")

    def step(self):
        """(out of each request's last token, positions): eager or captured."""
        hq, hk, D = self.shape
        t = self.native.paged_tables(self.cached, self.added, self.table, self.free, self.page, self.rows)
        q = self.native.rotary_append(*self.qkv.split([hq, hk, hk], dim=1), t.positions, self.inv, self.kc, self.vc,
                                      t.slots)
        last = q[(t.cu_seqlens[1:] - 1).clamp(min=0).long()]
        return self.native.paged_attention(last, self.kc, self.vc, self.table, t.lengths), t


def dense_last(keys, values, q, scale):
    s = torch.einsum("hd,nhd->hn", q.double(), keys.double()) * scale
    return torch.einsum("hn,nhd->hd", torch.softmax(s, -1), values.double())


@pytest.mark.parametrize("captured", [False, True])
def test_serving_steps(native, captured):
    """Prompts, then single tokens, requests joining at different steps:
    each step's attention against dense attention over all tokens so far."""
    hq, hk, D, rows = 4, 2, 64, 64
    s = Serving(native, hq, hk, D, 8, 3, 60, rows, 1)
    g = gen(2)
    graph = None
    if captured:
        s.step()  # (what the first call of all sets up)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, tables = s.step()
    history = [[] for _ in range(3)]
    cached, free = [0, 0, 0], s.free.cpu()
    for added in ([30, 17, 0], [1, 1, 8], [1, 0, 1], [1, 1, 1], [9, 1, 50]):
        qkv = randn(g, rows, hq + 2 * hk, D).to(BF16)
        s.qkv.copy_(qkv)
        s.cached.copy_(torch.tensor(cached, dtype=torch.int32))
        s.added.copy_(torch.tensor(added, dtype=torch.int32))
        s.free[:len(free)].copy_(free)
        if captured:
            graph.replay()
            eager_out, eager = s.step()  # the program's own work between replays
            torch.cuda.synchronize()
            assert torch.equal(out[[r for r in range(3) if added[r]]], eager_out[[r for r in range(3) if added[r]]])
        else:
            out, tables = s.step()
        i = 0
        for r in range(3):
            for j in range(added[r]):
                history[r].append((cached[r] + j, qkv[i]))
                i += 1
        for r in range(3):
            if not added[r]:
                continue
            pos = torch.tensor([p for p, _ in history[r]])[None]
            rows_r = torch.stack([x for _, x in history[r]])
            turned = M.rotary(rows_r[:, :hq + hk], pos, s.inv.cpu(), (D // 4,)).to(BF16)
            k = turned[:, hq:].repeat_interleave(hq // hk, dim=1)
            v = rows_r[:, hq + hk:].repeat_interleave(hq // hk, dim=1)
            ref = dense_last(k, v, turned[-1, :hq], D ** -0.5)
            # the rounding of the turned q and k may fall to the other side
            # of a border (one step, 2^-7 of a product): small scores' weights
            # move by about 2^-7 |s|; the weights' and the output's roundings
            close(out[r], ref, 2.0 ** -8 * ref.abs() + 2.0 ** -5 * v.double().abs().amax(0))
        taken = int(tables.counts[1])
        assert int(tables.counts[2]) == 0
        free = torch.cat([free[taken:], free[:taken]])
        cached = [c + a for c, a in zip(cached, added)]


def test_decoder_layer(native):
    """One decode step of a decoder layer with each kind of mixer: the mixer's
    output added to h, then the layer's MoE half."""
    from runnel_amd import PostAttentionMoE, RMSNorm, SparseMoeBlock, FusedQuantizedSwitchGLU
    from runnel_amd.switch_layers import QuantizedSwitchLinear
    g = gen(7)
    H, R = 256, 3
    blk = SparseMoeBlock(H, 64, 8, 2, bits=8, device="cuda")
    blk.gate.weight.copy_((0.1 * randn(g, 8, H)).to(BF16))
    for name, o, i in (("gate_proj", 64, H), ("up_proj", 64, H), ("down_proj", H, 64)):
        setattr(blk.switch_mlp, name, QuantizedSwitchLinear.from_float((0.1 * randn(g, 8, o, i)).cuda(), 8))
    blk.switch_mlp = FusedQuantizedSwitchGLU(blk.switch_mlp)
    moe = PostAttentionMoE(RMSNorm(H, device="cuda"), blk)
    h = randn(g, R, H).to(BF16).cuda()
    s = Serving(native, 4, 2, 64, 8, R, 30, R, 3)
    s.added.fill_(1)
    s.qkv.copy_(randn(g, R, 8, 64).to(BF16))
    attended, _ = s.step()
    q, k, v, a, cu, state, beta = (None if x is None else x.cuda()
                                   for x in linear_inputs(3, [1] * R, 2, 4, 64, 64))
    mixed = native.linear_attention(q, k, v, a, cu, state, beta=beta)
    for m in (attended, mixed):
        y = moe(h + m.reshape(R, H))
        assert y.shape == (R, H) and torch.isfinite(y).all()
        assert torch.equal(y, moe(h + m.reshape(R, H)))


def test_streams_share_nothing(native):
    """Calls of each operator on two streams at once equal the calls alone."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for seed in range(2):
        q, kc, vc, table, lengths = attention_inputs(seed, [3000, 10, 900], 4, 2, 128, 16, 16)
        a = [q.cuda(), kc, vc, table.cuda(), lengths.cuda()]
        x = linear_inputs(seed, [300, 20], 2, 4, 128, 32)
        b = [None if y is None else y.cuda() for y in x]
        jobs.append((a, b))

    def both(a, b):
        st = b[5].clone()
        o = native.linear_attention(*b[:5], st, beta=b[6])
        return native.paged_attention(*a), o, st

    alone = [both(*j) for j in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(both(*jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for x, y in zip(r, alone[i]):
                assert torch.equal(x, y)


def test_threads(native):
    """Calls from several Python threads, each on a stream of its own: the
    binding lets others run while it launches, and errors stay with theirs."""
    from concurrent.futures import ThreadPoolExecutor

    q, kc, vc, table, lengths = attention_inputs(2, [1500, 40, 7], 4, 2, 64, 16, 16)
    a = [q.cuda(), kc, vc, table.cuda(), lengths.cuda()]
    b = [None if y is None else y.cuda() for y in linear_inputs(2, [90, 3], 2, 4, 64, 32)]
    want = native.paged_attention(*a), native.linear_attention(*b[:5], b[5].clone(), beta=b[6])
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                assert torch.equal(native.paged_attention(*a), want[0])
                assert torch.equal(native.linear_attention(*b[:5], b[5].clone(), beta=b[6]), want[1])
                with pytest.raises(ValueError, match="page_size" if i % 2 else "rows must not"):
                    native.paged_tables(a[4], a[4], a[3].clone(), a[4], 12 if i % 2 else 16, 1 if i % 2 else -1)
        return i

    with ThreadPoolExecutor(4) as pool:
        assert list(pool.map(work, range(4))) == [0, 1, 2, 3]


def test_two_graphs(native):
    """Two captured graphs of the same operators, replayed in turn and at
    once on two streams."""
    graphs, inputs = [], []
    for seed in range(2):
        q, kc, vc, table, lengths = attention_inputs(seed + 20, [2000, 64, 1], 4, 1, 64, 16, 16)
        a = [q.cuda(), kc, vc, table.cuda(), lengths.cuda()]
        b = [None if y is None else y.cuda() for y in linear_inputs(seed, [100, 33], 1, 2, 64, 32)]
        out_state = torch.zeros_like(b[5])

        def work(a=a, b=b, out_state=out_state):
            return (native.paged_attention(*a),
                    native.linear_attention(*b[:6], beta=b[6], state_out=out_state), out_state)

        ref = [x.clone() for x in work()]
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = work()
        graphs.append((gr, out, ref))
        inputs.append((a, b))  # (a graph does not keep what it reads)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        for (gr, out, ref), st in zip(graphs, streams):
            for x in out:
                x.zero_()
        torch.cuda.synchronize()
        for (gr, out, ref), st in zip(graphs, streams):
            with torch.cuda.stream(st if turn else streams[0]):
                gr.replay()
        torch.cuda.synchronize()
        for gr, out, ref in graphs:
            for x, y in zip(out, ref):
                assert torch.equal(x, y)

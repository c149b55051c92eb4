"""What the token mixer's operators refuse, on the host, before any launch:
the C calls with addresses that are never read, the torch wrappers with CPU
tensors and meta shapes.  No test here launches a kernel."""

import ctypes

import numpy as np
import pytest
import torch

import mixer_ref
from runnel_amd import _lib, native

FAKE = 0x100000
BF16 = torch.bfloat16


def rows(x=FAKE, row=256, head=64, heads=4):
    return _lib.Rows(x, row, head, heads)


def cache(**kw):
    d = dict(k=FAKE, v=FAKE, page_stride=2048, head_stride=1024, row_stride=64, pages=4, page_size=16,
             kv_heads=2, dim=64, bits=16, k_scale=1.0, v_scale=1.0)
    d.update(kw)
    return _lib.PagedCache(*[d[n] for n, _ in _lib.PagedCache._fields_])


def spec(half=32, sections=(32,), woven=0, adjacent=0, ptr=FAKE):
    return _lib.RotarySpec(ptr, half, len(sections), (ctypes.c_int32 * 4)(*sections[:4]), woven, adjacent)


def test_tables_refusals():
    lib = _lib.load()

    def call(requests=2, table=FAKE, stride=4, width=4, free=FAKE, count=3, page=16, n=5, cached=FAKE,
             slots=FAKE):
        return lib.rmoe_paged_tables(cached, FAKE, requests, table, stride, width, free, count, page, n, slots,
                                     FAKE, FAKE, FAKE, FAKE, FAKE, None)

    for bad in (dict(requests=0), dict(requests=4097), dict(page=0), dict(page=4), dict(page=24),
                dict(page=2048), dict(width=-1), dict(stride=3), dict(count=-1), dict(n=-1)):
        assert call(**bad) == _lib.RMOE_EINVAL, bad
    for bad in (dict(cached=None), dict(table=None), dict(free=None), dict(slots=None)):
        assert call(**bad) == _lib.RMOE_ENULL, bad
    assert call(slots=FAKE + 4) == _lib.RMOE_EALIGN


def test_rotary_refusals():
    lib = _lib.load()

    def call(s=None, n=3, dim=64, q=None, k=None, q_out=FAKE, k_out=FAKE, pos=FAKE, axis=3):
        s = spec() if s is None else s
        return lib.rmoe_rotary(ctypes.byref(s), pos, axis, n, dim, ctypes.byref(q or rows()), q_out,
                               ctypes.byref(k or rows(heads=2)), k_out, None)

    for s in (spec(half=0, sections=(0,)), spec(half=12, sections=(12,)), spec(half=136, sections=(136,)),
              spec(half=32, sections=(16, 8)), spec(half=32, sections=(40, -8)),
              spec(half=32, sections=(10, 11, 11), woven=1), spec(half=40, sections=(40,))):
        ok = s.half == 32 and s.woven  # (10 + 11 + 11 fits the turns of three axes)
        if not ok:
            assert call(s) == _lib.RMOE_EINVAL
    assert call(spec(half=32, sections=(8, 12, 12), woven=1)) == _lib.RMOE_EINVAL
    s = spec()
    for axes in (0, 5):
        s.axes = axes
        assert call(s) == _lib.RMOE_EINVAL
    assert call(spec(ptr=None)) == _lib.RMOE_ENULL
    for bad in (dict(n=-1), dict(n=(1 << 25) + 1), dict(dim=12), dict(dim=1032), dict(q=rows(heads=0)),
                dict(q=rows(row=-8)), dict(k=rows(heads=70000))):
        assert call(**bad) == _lib.RMOE_EINVAL, bad
    for bad in (dict(q_out=None), dict(k_out=None), dict(pos=None), dict(q=rows(x=None))):
        assert call(**bad) == _lib.RMOE_ENULL, bad
    for bad in (dict(q_out=FAKE + 8), dict(k_out=FAKE + 2), dict(q=rows(x=FAKE + 8)), dict(k=rows(row=132)),
                dict(k=rows(head=68))):
        assert call(**bad) == _lib.RMOE_EALIGN, bad
    assert call(n=0, q_out=None, k_out=None, pos=None, q=rows(x=None), k=rows(x=None)) == _lib.RMOE_OK


BAD_CACHES = [
    (dict(page_size=4), _lib.RMOE_EINVAL), (dict(page_size=48), _lib.RMOE_EINVAL),
    (dict(dim=80), _lib.RMOE_EINVAL), (dict(dim=512), _lib.RMOE_EINVAL), (dict(bits=4), _lib.RMOE_EBITS),
    (dict(pages=0), _lib.RMOE_EINVAL), (dict(kv_heads=0), _lib.RMOE_EINVAL),
    (dict(page_stride=-8), _lib.RMOE_EINVAL), (dict(k=None), _lib.RMOE_ENULL),
    (dict(v=FAKE + 8), _lib.RMOE_EALIGN), (dict(row_stride=68), _lib.RMOE_EALIGN),
    (dict(bits=8, row_stride=72), _lib.RMOE_EALIGN), (dict(bits=8, k_scale=0.0), _lib.RMOE_EINVAL),
    (dict(bits=8, v_scale=float("nan")), _lib.RMOE_EINVAL),
    (dict(bits=8, v_scale=float("inf")), _lib.RMOE_EINVAL),
]


@pytest.mark.parametrize("bad,code", BAD_CACHES, ids=range(len(BAD_CACHES)))
def test_cache_refusals(bad, code):
    lib = _lib.load()
    c = cache(**bad)
    assert lib.rmoe_paged_attention(ctypes.byref(rows()), ctypes.byref(c), FAKE, 4, 4, FAKE, 2, 0, 0.1, FAKE, None,
                                    FAKE, 1 << 30, None) == code
    assert lib.rmoe_rotary_append(ctypes.byref(spec()), FAKE, 3, 3, ctypes.byref(rows()), FAKE,
                                  ctypes.byref(rows(heads=2)), ctypes.byref(rows(heads=2)), ctypes.byref(c), FAKE,
                                  None) == code


def test_attention_refusals():
    lib = _lib.load()

    def call(q=None, c=None, table=FAKE, width=4, lengths=FAKE, n=2, window=0, scale=0.1, out=FAKE, ws=FAKE,
             size=1 << 30):
        return lib.rmoe_paged_attention(ctypes.byref(q or rows()), ctypes.byref(c or cache()), table, 4, width,
                                        lengths, n, window, scale, out, None, ws, size, None)

    for bad in (dict(q=rows(heads=3)), dict(width=-1), dict(n=-1), dict(window=-1), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(width=1 << 27), dict(n=1 << 24)):
        assert call(**bad) == _lib.RMOE_EINVAL, bad
    for bad in (dict(table=None), dict(lengths=None), dict(out=None), dict(q=rows(x=None))):
        assert call(**bad) == _lib.RMOE_ENULL, bad
    assert call(out=FAKE + 8) == _lib.RMOE_EALIGN
    need = lib.rmoe_paged_attention_workspace_bytes(ctypes.byref(cache()), 4, 2, 4000, 0)
    assert need > 0
    for bad in (dict(size=need - 1), dict(ws=None)):
        assert call(width=4000, **bad) == _lib.RMOE_EWS, bad
    assert call(width=4000, ws=FAKE + 8) == _lib.RMOE_EALIGN
    assert lib.rmoe_paged_attention_workspace_bytes(ctypes.byref(cache()), 3, 2, 4000, 0) == 0
    assert call(n=0, q=rows(x=None), table=None, lengths=None, out=None) == _lib.RMOE_OK


def test_attention_refuses_a_table_backwards():
    lib = _lib.load()
    assert lib.rmoe_paged_attention(ctypes.byref(rows()), ctypes.byref(cache()), FAKE, -4, 4, FAKE, 2, 0, 0.1, FAKE,
                                    None, FAKE, 1 << 30, None) == _lib.RMOE_EINVAL


def test_linear_refusals():
    lib = _lib.load()
    gate = _lib.Gate(FAKE, 4, 1)

    def call(q=None, k=None, v=None, g=gate, b=gate, cu=FAKE, n=100, r=2, dk=64, dv=32, scale=1.0, st=FAKE,
             so=FAKE, slots=2, out=FAKE, ws=FAKE, size=1 << 40):
        return lib.rmoe_linear_attention(
            ctypes.byref(q or rows()), ctypes.byref(k or rows()), ctypes.byref(v or rows()),
            None if g is None else ctypes.byref(g), None if b is None else ctypes.byref(b), cu, n, r, dk, dv, scale,
            st, so, None, slots, out, 1, ws, size, None)

    for bad in (dict(n=-1), dict(r=0), dict(dk=96), dict(dk=256), dict(dv=8), dict(dv=24), dict(dv=1040),
                dict(q=rows(heads=2)), dict(v=rows(heads=6)), dict(scale=float("nan")), dict(slots=-1),
                dict(g=_lib.Gate(FAKE, -1, 1)), dict(b=_lib.Gate(FAKE, 1, -1)), dict(n=1 << 30, r=1),
                dict(r=1 << 30), dict(k=rows(row=1 << 25)), dict(v=rows(row=1 << 25)),
                dict(v=rows(heads=65536), dv=512)):
        assert call(**bad) == _lib.RMOE_EINVAL, bad
    for bad in (dict(g=None), dict(cu=None), dict(st=None), dict(so=None), dict(out=None), dict(q=rows(x=None)),
                dict(b=_lib.Gate(None, 1, 1))):
        assert call(**bad) == _lib.RMOE_ENULL, bad
    for bad in (dict(st=FAKE + 4), dict(so=FAKE + 8), dict(out=FAKE + 2), dict(v=rows(head=36)), dict(ws=FAKE + 8)):
        assert call(**bad) == _lib.RMOE_EALIGN, bad
    need = lib.rmoe_linear_attention_workspace_bytes(100, 2, 4, 4, 64, 1)
    assert need > lib.rmoe_linear_attention_workspace_bytes(100, 2, 4, 4, 64, 0) > 0
    assert lib.rmoe_linear_attention_workspace_bytes(2, 2, 4, 4, 64, 1) == 0
    for bad in (dict(size=need - 1), dict(ws=None)):
        assert call(**bad) == _lib.RMOE_EWS, bad


def test_wrappers_take_gpu_tensors():
    x, i = torch.zeros(2, 4, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    c = torch.zeros(4, 2, 16, 64, dtype=BF16)
    f = torch.zeros(2, 4)
    for call in (lambda: native.paged_tables(i, i, torch.zeros(2, 4, dtype=torch.int32), i, 16, 2),
                 lambda: native.rotary(x, x, i, f[0]),
                 lambda: native.rotary_append(x, x, x, i, f[0], c, c, i.long()),
                 lambda: native.paged_attention(x, c, c, torch.zeros(2, 4, dtype=torch.int32), i),
                 lambda: native.linear_attention(x, x, x, f, i, torch.zeros(1, 4, 64, 64))):
        with pytest.raises(ValueError, match="GPU tensors"):
            call()


def test_wrappers_take_tensors():
    x = torch.zeros(2, 4, 64, dtype=BF16)
    with pytest.raises(TypeError, match="k must be a tensor"):
        native.rotary(x, None, x, x)
    with pytest.raises(TypeError):
        native.paged_tables(x, x, x, x, 16.5, 2)
    with pytest.raises(ValueError, match="page_size is out of range"):
        native.paged_tables(x, x, x, x, 1 << 40, 2)


def test_a_binding_that_was_not_built(monkeypatch):
    import sys

    import runnel_amd
    native._binding()
    monkeypatch.setattr(native, "_mixer", None)
    monkeypatch.delattr(runnel_amd, "_mixer")
    monkeypatch.setitem(sys.modules, "runnel_amd._mixer", None)
    with pytest.raises(RuntimeError, match="_mixer.so is missing"):
        native._binding()


def test_oracle_tables():
    """The tables' oracle on a case worked by hand: pages of 8, a free list
    of two."""
    table, slots, positions, requests, cu, lengths, counts = mixer_ref.tables(
        [7, 0], [2, 9], np.array([[4, -1], [-1, -1]]), [9, 3], 8, 12)
    assert table.tolist() == [[4, 9], [3, -1]]
    assert slots.tolist() == [39, 72, 24, 25, 26, 27, 28, 29, 30, 31, -1, -1]
    assert positions.tolist()[:4] == [7, 8, 0, 1] and requests.tolist()[-2:] == [1, -1]
    assert cu.tolist() == [0, 2, 11] and lengths.tolist() == [9, 9] and counts.tolist() == [11, 2, 1]


def test_oracle_linear():
    """With beta 1, no decay and orthonormal keys the delta rule stores each
    value at its key: reading with a key returns its last value."""
    k = torch.eye(4)[[0, 1, 0, 2]][:, None]
    v = torch.arange(8.0).view(4, 1, 2)
    g = torch.zeros(4, 1)
    out, state, _, _ = mixer_ref.linear(k, k, v, g, [0, 4], torch.zeros(1, 1, 4, 2), torch.ones(4, 1), scale=1.0)
    assert torch.equal(out, v.double())
    assert torch.equal(state[0, 0], torch.tensor([[4.0, 5.0], [2.0, 3.0], [6.0, 7.0], [0.0, 0.0]]).double())

"""Rotary positions of packed rows and rows through a paged cache: the host's
checks and index functions (CPU), the kernels against float64 (GPU)."""
import ctypes as C
import math
import os

import numpy as np
import pytest
import torch

import rows_util as U
from rows_util import DT, ELEM, F64, HALF, Dev

HERE = os.path.dirname(os.path.abspath(__file__))


# ---------------------------------------------------------------- CPU ----

@pytest.fixture(scope="module")
def ri(xh):
    lib = C.CDLL(os.path.join(HERE, "native", "rows_index.so"))
    lib.ri_row_position.restype = C.c_int64
    lib.ri_row_position.argtypes = [C.c_int32, C.c_uint32, C.c_uint32]
    lib.ri_page_of.restype = C.c_int32
    lib.ri_page_of.argtypes = [C.c_void_p] + [C.c_uint32] * 4 + [C.c_int64]
    lib.ri_cache_row.restype = C.c_uint64
    lib.ri_cache_row.argtypes = [C.c_uint32] * 5
    lib.ri_seq_of_row.restype = C.c_uint32
    lib.ri_seq_of_row.argtypes = [C.c_void_p] + [C.c_uint32] * 3
    lib.ri_row_span.argtypes = [C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p]
    return lib


@pytest.mark.parametrize("new", [[1], [3, 0, 2], [0, 0, 5, 0], [0], [1] * 70, [2, 0, 0, 7, 1]])
def test_every_packed_row_has_its_sequence(ri, new):
    cu = np.cumsum([0] + new).astype(np.int32)
    n = int(cu[-1]) + 3                                   # rows behind the last sequence
    for t in range(n):
        got = ri.ri_seq_of_row(cu.ctypes.data, len(new), n, t)
        want = next((b for b in range(len(new)) if cu[b] <= t < cu[b + 1]), len(new))
        assert got == want, (t, got, want)


@pytest.mark.parametrize("cu", [[0, -5, 9], [0, 100, 7], [-3, 4, 2], [5, 5, 5], [2 ** 31 - 1, -2 ** 31, 3]])
def test_malformed_sequences_stay_in_their_rows(ri, cu):
    cu, n = np.array(cu, np.int32), 8
    out = np.zeros(2, np.uint32)
    for b in range(2):
        ri.ri_row_span(cu.ctypes.data, n, b, out.ctypes.data)
        assert 0 <= out[0] <= out[1] <= n
    for t in range(n):
        b = ri.ri_seq_of_row(cu.ctypes.data, 2, n, t)
        assert b <= 2
        if b < 2:
            ri.ri_row_span(cu.ctypes.data, n, b, out.ctypes.data)
            assert out[0] <= t < out[1]


def test_bad_pages_have_no_row(ri):
    table = np.array([[3, -1, 7, 2 ** 31 - 1], [0, 6, -2 ** 31, 5]], np.int32)
    at = lambda b, p: ri.ri_page_of(table.ctypes.data, 4, 7, 4, b, p)  # noqa: E731  (7 pages of 16)
    assert [at(0, p) for p in (0, 15, 16, 32, 48, 63)] == [3, 3, -1, -1, -1, -1]
    assert [at(1, p) for p in (0, 16, 31, 32, 48, 63)] == [0, 6, 6, -1, 5, 5]
    assert [at(b, p) for b in (0, 1) for p in (-1, 64, 2 ** 31, 2 ** 40, -2 ** 40)] == [-1] * 10
    assert ri.ri_row_position(2, 5, 0) == -3 and ri.ri_row_position(-2 ** 31, 2 ** 31, 0) == -2 ** 32
    # rows past 2^32 elements of a large cache
    assert ri.ri_cache_row(2 ** 31 - 2, 8, 7, 10, 1023) == ((2 ** 31 - 2) * 8 + 7) * 1024 + 1023


def rope_spec(xh, **kw):
    base = dict(rot_dim=64, layout=xh.XP_ROPE_HALF, theta=1e4, scaling=xh.XP_ROPE_PLAIN, factor=8.0,
                original_len=8192.0, low=1.0, high=4.0, magnitude=0.0)
    base.update(kw)
    return xh.XpRope(*base.values())


def want_frequencies(spec):
    n, out = spec.rot_dim, []
    for i in range(n // 2):
        f, g = spec.theta ** (-2.0 * i / n), 1.0
        if spec.scaling == 1:
            g = 0.0
        elif spec.scaling == 2:
            g = (spec.original_len * f / (2 * math.pi) - spec.low) / (spec.high - spec.low)
        elif spec.scaling == 3:
            at = [n * math.log(spec.original_len / (2 * math.pi * r)) / (2 * math.log(spec.theta)) for r in (spec.high, spec.low)]
            a, b = (min(max(f(x), 0), n - 1) for f, x in zip((math.floor, math.ceil), at))
            g = 1 - (i - a) / max(b - a, 1e-3)
        g = min(max(g, 0.0), 1.0)
        out.append(f * (g + (1 - g) / spec.factor) if spec.scaling else f)
    return np.array(out)


@pytest.mark.parametrize("scaling", [0, 1, 2, 3])
@pytest.mark.parametrize("rot,theta", [(2, 1e4), (64, 1e4), (128, 5e5), (250, 1e6), (512, 1e6)])
def test_rope_frequencies(xh, scaling, rot, theta):
    spec = rope_spec(xh, rot_dim=rot, theta=theta, scaling=scaling, high=32.0 if scaling == 3 else 4.0)
    np.testing.assert_allclose(xh.rope_frequencies(spec), want_frequencies(spec), rtol=1e-12)


@pytest.mark.parametrize("bad,says", [
    ({"rot_dim": 0}, "rot_dim"), ({"rot_dim": 63}, "rot_dim"), ({"rot_dim": 514}, "rot_dim"), ({"layout": 2}, "layout"),
    ({"theta": 1.0}, "theta"), ({"theta": math.nan}, "theta"), ({"theta": math.inf}, "theta"), ({"scaling": 4}, "scaling"),
    ({"scaling": 1, "factor": 0.5}, "factor"), ({"scaling": 2, "low": 0.0}, "low"), ({"scaling": 2, "high": 1.0}, "high"),
    ({"scaling": 3, "original_len": 0.0}, "original_len"), ({"magnitude": math.inf}, "magnitude")])
def test_rope_refuses_specs(xh, bad, says):
    with pytest.raises(xh.XposeError, match=says) as e:
        xh.rope_frequencies(rope_spec(xh, **bad)) if "rot_dim" not in bad else xh.call(
            "xp_rope_frequencies", rope_spec(xh, **bad), np.empty(300).ctypes.data, 300)
    assert e.value.code == -1


FAKE = 1 << 20      # an aligned address that no refused call touches


def rows_args(xh, **kw):
    r = dict(data=FAKE, stride=8 * 64, heads=8, elem=ELEM["f16"])
    r.update(kw)
    return xh.XpRows(*r.values())


@pytest.mark.parametrize("bad,says", [
    ({"data": None}, "q is null"), ({"elem": 3}, "elem 3"), ({"heads": 0}, "heads"), ({"stride": 511}, "stride"),
    ({"data": FAKE + 1}, "multiples of 2"), ({"stride": 1 << 27}, "2\\^26"), ({"heads": 4, "stride": 256}, "q_out has not")])
def test_rope_refuses_rows(xh, bad, says):
    with pytest.raises(xh.XposeError, match=says):
        xh.call("xp_rope_rows", rows_args(xh), rows_args(xh, **bad), None, None, FAKE, 4, 64, rope_spec(xh), None)


def test_rope_refuses_shapes(xh):
    r = rows_args(xh)
    for args, says in (((r, r, r, None, FAKE, 4, 64, rope_spec(xh), None), "both"),
                       ((r, r, None, None, None, 4, 64, rope_spec(xh), None), "positions"),
                       ((r, r, None, None, FAKE, 4, 62, rope_spec(xh), None), "head_dim"),
                       ((r, r, None, None, FAKE, 4, 514, rope_spec(xh), None), "head_dim"),
                       ((r, r, r, rows_args(xh, elem=0), FAKE, 4, 64, rope_spec(xh), None), "k_out has not")):
        with pytest.raises(xh.XposeError, match=says):
            xh.call("xp_rope_rows", *args)
    xh.call("xp_rope_rows", r, r, None, None, None, 0, 64, rope_spec(xh), None)      # no tokens: nothing to do


def cache_args(xh, **kw):
    c = dict(k=FAKE, v=FAKE, k_scale=None, v_scale=None, elem=ELEM["f16"], n_pages=4, page_size=16, kv_heads=8, head_dim=64)
    c.update(kw)
    return xh.XpPagedKv(*c.values())


def seqs_args(xh, **kw):
    s = dict(n_seq=2, n_tokens=4, cu=FAKE, kv_len=FAKE, pages=FAKE, table=3)
    s.update(kw)
    return xh.XpPagedSeqs(*s.values())


BAD_CACHES = [
    ({"k": None}, "null"), ({"elem": 0}, "elem 0"), ({"elem": 3}, "scales"), ({"k_scale": FAKE}, "scales"),
    ({"elem": 4, "k_scale": FAKE}, "scales"), ({"page_size": 8}, "page_size"), ({"page_size": 48}, "page_size"),
    ({"page_size": 2048}, "page_size"), ({"head_dim": 72}, "head_dim"), ({"head_dim": 272}, "head_dim"),
    ({"kv_heads": 0}, "kv heads"), ({"n_pages": 1 << 31}, "pages"), ({"v": FAKE + 8}, "aligned")]
BAD_SEQS = [({"cu": None}, "null"), ({"kv_len": None}, "null"), ({"pages": None}, "null"),
            ({"n_tokens": 1 << 31}, "tokens"), ({"n_seq": (1 << 24) + 1}, "sequences"), ({"table": (1 << 26) + 1}, "table")]


@pytest.mark.parametrize("call", ["xp_paged_kv_write", "xp_paged_kv_read"])
def test_paged_kv_refuses(xh, call):
    r = rows_args(xh)
    for bad, says in BAD_CACHES:
        with pytest.raises(xh.XposeError, match=says):
            xh.call(call, cache_args(xh, **bad), seqs_args(xh), r, r, None)
    for bad, says in BAD_SEQS:
        with pytest.raises(xh.XposeError, match=says):
            xh.call(call, cache_args(xh), seqs_args(xh, **bad), r, r, None)
    for bad, says in (({"data": FAKE + 2}, "multiples of 16"), ({"stride": 516}, "multiples of 16"), ({"heads": 4}, "heads"),
                      ({"elem": 0}, "elem"), ({"data": None}, "v is null")):
        with pytest.raises(xh.XposeError, match=says):
            xh.call(call, cache_args(xh), seqs_args(xh), r, rows_args(xh, **bad), None)
    for none in ({"n_tokens": 0}, {"n_seq": 0}):
        xh.call(call, cache_args(xh), seqs_args(xh, cu=None, kv_len=None, pages=None, **none), r, r, None)


# ---------------------------------------------------------------- GPU ----

def rope_ref(x, positions, f, layout, rot, magnitude):
    """[token][head][dim] turned in float64, and |x0| + |x1| of each value's pair."""
    y, size = x.to(F64).clone(), x.to(F64).abs()
    angle = positions.to(F64)[:, None] * torch.from_numpy(f)
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    i0, i1 = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == 0 else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = y[..., i0].clone(), y[..., i1].clone()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = (a.abs() + b.abs()) * magnitude
    return y, size


def rope_bound(y, size, elem):
    """The fraction of a turn has 24 bits (half a turn: pi 2^-24 of an angle), sine and cosine 2 ulp of 1 at
    most, magnitude and products and sum a rounding each: (pi + 4 + 1 + 2) 2^-24 < 2^-20 of |x0| + |x1|."""
    return size * 2.0 ** -20 + HALF[elem] * y.abs() * 1.01 + 2.0 ** -25


ROPES = [  # tokens, q heads, k heads, dim, rot, elem, layout, scaling
    (1, 1, 0, 2, 2, "f32", 0, 0), (1, 4, 1, 256, 256, "f32", 0, 0), (16, 4, 1, 256, 256, "bf16", 1, 0),
    (7, 3, 2, 80, 40, "f16", 0, 1), (33, 32, 8, 128, 64, "bf16", 1, 2), (5, 5, 5, 96, 80, "f32", 1, 3),
    (300, 8, 8, 64, 48, "f16", 0, 3), (1029, 4, 1, 256, 240, "f32", 0, 2), (3, 2, 1, 512, 512, "f16", 1, 0),
    (9, 2, 1, 34, 30, "bf16", 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,qh,kh,dim,rot,elem,layout,scaling", ROPES)
def test_gpu_rope(xp, tokens, qh, kh, dim, rot, elem, layout, scaling):
    g = torch.Generator().manual_seed(tokens * 1000 + dim)
    spec = rope_spec(xp, rot_dim=rot, layout=layout, theta=1e6, scaling=scaling, high=32.0 if scaling == 3 else 4.0,
                     magnitude=1.25 if scaling == 3 else 0.0)
    pos = torch.randint(-(1 << 20), 1 << 20, (tokens,), generator=g, dtype=torch.int32)
    pos[0], pos[-1] = 0, 2 ** 31 - 1
    f, m = xp.rope_frequencies(spec), spec.magnitude or 1.0
    heads = [qh] + ([kh] if kh else [])
    x = [torch.randn(tokens, h, dim, generator=g).to(DT[elem]) for h in heads]
    din = [Dev(xp, v) for v in x]
    dout = [Dev(xp, torch.full_like(v, -7.0)) for v in x]
    dpos = Dev(xp, pos)
    view = lambda d, h: U.rows(xp, d, h, elem, h * dim)  # noqa: E731
    k = (view(dout[1], kh), view(din[1], kh)) if kh else (None, None)
    xp.call("xp_rope_rows", view(dout[0], qh), view(din[0], qh), *k, dpos.ptr, tokens, dim, spec, None)
    xp.synchronize()
    for v, d in zip(x, dout):
        want, size = rope_ref(v, pos, f, layout, rot, m)
        got = d.host().to(F64)
        assert torch.equal(got[..., rot:], v[..., rot:].to(F64))
        err = (got - want).abs()
        assert (err <= rope_bound(want, size, elem)).all(), float((err / rope_bound(want, size, elem)).max())
    # turned back in place, on a row step of its own: the input again
    back = Dev(xp, -pos)
    xp.call("xp_rope_rows", view(dout[0], qh), view(dout[0], qh), None, None, back.ptr, tokens, dim, spec, None)
    xp.synchronize()
    if m == 1.0:
        size = rope_ref(x[0], pos, f, layout, rot, m)[1]
        err = (dout[0].host().to(F64) - x[0].to(F64)).abs()
        assert (err <= 2 * rope_bound(size, size, elem) * 1.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("elem,offset,gap", [("f16", 0, 24), ("f32", 3, 5), ("bf16", 1, 0)])
def test_gpu_rope_in_a_fused_row(xp, elem, offset, gap):
    """q and k inside one row with other values around them, which stay."""
    g = torch.Generator().manual_seed(5)
    tokens, qh, kh, dim, rot = 11, 4, 2, 64, 32
    stride = (qh + 2 * kh) * dim + gap
    x = torch.randn(tokens * stride + offset, generator=g).to(DT[elem])
    pos = torch.arange(100, 100 + tokens, dtype=torch.int32)
    d, dpos, spec = Dev(xp, x), Dev(xp, pos), rope_spec(xp, rot_dim=rot)
    q, k = U.rows(xp, d, qh, elem, stride, offset), U.rows(xp, d, kh, elem, stride, offset + qh * dim)
    xp.call("xp_rope_rows", q, q, k, k, dpos.ptr, tokens, dim, spec, None)
    xp.synchronize()
    rows_ = lambda t: t[offset:].reshape(tokens, stride)  # noqa: E731
    got, old = rows_(d.host()), rows_(x)
    n = (qh + kh) * dim
    assert torch.equal(got[:, n:], old[:, n:]) and torch.equal(d.host()[:offset], x[:offset])
    want, size = rope_ref(old[:, :n].reshape(tokens, qh + kh, dim), pos, xp.rope_frequencies(spec), 0, rot, 1.0)
    err = (got[:, :n].reshape(want.shape).to(F64) - want).abs()
    assert (err <= rope_bound(want, size, elem)).all()


def special_rows(x, g):
    """Some rows of zeros, of one value, tiny, huge, and with values that are not finite."""
    x[0] = 0.0
    x[1, 0, 3] = math.nan
    x[2, -1, 1] = -math.inf
    x[3] *= 2.0 ** -14
    x[4, :, 1:] = 0.0
    x[5] = torch.round(x[5] * 4) / 4                      # ties
    x[5, :, 0] = 127.0 / 8
    return x


KVS = [  # new of each sequence, length before, kv heads, dim, rows' elem, cache, page
    ([1], [0], 1, 16, "f32", "i8", 16), ([1] * 5, [0, 15, 16, 17, 300], 1, 256, "f32", "i8", 64),
    ([7, 0, 30, 1], [5, 9, 0, 64], 8, 128, "bf16", "e4m3", 16), ([33, 12], [0, 31], 2, 80, "f16", "i8", 32),
    ([40, 9], [3, 1], 3, 96, "f32", "e4m3", 128), ([20, 20], [10, 100], 4, 64, "f16", "f16", 16),
    ([9, 50], [1, 2], 2, 192, "bf16", "bf16", 32), ([17], [1000], 2, 112, "f32", "f16", 256), ([12], [0], 1, 48, "f16", "e4m3", 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("new,past,kvh,dim,elem,cache,page", KVS)
def test_gpu_paged_kv_round_trip(xp, new, past, kvh, dim, elem, cache, page):
    g = torch.Generator().manual_seed(len(new) * 100 + dim)
    lens = [n + p for n, p in zip(new, past)]
    width = max(-(-n // page) for n in lens)
    pages = len(new) * width + 2
    c = U.Cache(xp, g, cache, pages, page, kvh, dim).upload()
    s = U.Seqs(xp, new, lens, page, pages, n_tokens=sum(new) + 3, g=g)     # three rows behind the last sequence
    n = s.n_tokens
    kv = torch.randn(n, 2 * kvh, dim, generator=g)
    kv = special_rows(kv, g) if n >= 9 else kv
    kv = kv.to(DT[elem])
    d = Dev(xp, kv)
    k, v = U.rows(xp, d, kvh, elem, 2 * kvh * dim), U.rows(xp, d, kvh, elem, 2 * kvh * dim, kvh * dim)
    xp.call("xp_paged_kv_write", c.desc, s.desc, k, v, None)
    xp.synchronize()
    want_code, want_scale = [x.clone() for x in c.code], [None if x is None else x.clone() for x in c.scale]
    for t, b, p in s.tokens():
        g_, i = int(s.table[b, p // page]), p % page
        for w in (0, 1):
            code, scale = U.quantise(kv[t, w * kvh:(w + 1) * kvh], cache)
            want_code[w][g_, :, i] = code
            if scale is not None:
                want_scale[w][g_, :, i] = scale
    for w in (0, 1):
        got = c.dcode[w].host()
        same = got.view(torch.uint8) == want_code[w].view(torch.uint8)
        if cache in ("f16", "bf16"):
            same = same | (torch.isnan(got) & torch.isnan(want_code[w])).repeat_interleave(2, -1)
        if cache == "e4m3":                               # -0 is 0's
            same = same | ((got.to(torch.float32) == 0) & (want_code[w].to(torch.float32) == 0))
        assert same.all(), int((~same).sum())
        if want_scale[w] is not None:
            assert torch.equal(torch.nan_to_num(c.dscale[w].host(), nan=-1.0), torch.nan_to_num(want_scale[w], nan=-1.0))
    # read back: each value rounded once; rows of no sequence stay
    back = Dev(xp, torch.full_like(kv, 5.0))
    kb, vb = U.rows(xp, back, kvh, elem, 2 * kvh * dim), U.rows(xp, back, kvh, elem, 2 * kvh * dim, kvh * dim)
    xp.call("xp_paged_kv_read", c.desc, s.desc, kb, vb, None)
    xp.synchronize()
    got = back.host()
    assert (got[sum(new):] == 5.0).all()
    for t, b, p in s.tokens():
        for w in (0, 1):
            g_, i = int(s.table[b, p // page]), p % page
            sc = want_scale[w]
            x = want_code[w][g_, :, i].to(torch.float32)
            x = (x if sc is None else x * sc[g_, :, i, None]).to(DT[elem])
            y = got[t, w * kvh:(w + 1) * kvh]
            assert torch.equal(torch.nan_to_num(x.to(F64), nan=-9.0), torch.nan_to_num(y.to(F64), nan=-9.0)), (t, w)


@pytest.mark.gpu
@pytest.mark.parametrize("cache", ["i8", "f16"])
def test_gpu_paged_kv_rows_without_a_slot(xp, cache):
    """Bad pages, positions past the table and before the start: dropped when written, NaN when read (rows before the
    start belong to no sequence and stay)."""
    g = torch.Generator().manual_seed(3)
    page, pages, kvh, dim = 16, 6, 2, 32
    table = torch.tensor([[1, -1, 6], [2, 4, 3]], dtype=torch.int32)
    new, lens = [40, 6], [56, 4]                          # rows 16..55 of three entries; rows -2..3
    c = U.Cache(xp, g, cache, pages, page, kvh, dim).upload()
    s = U.Seqs(xp, new, lens, page, pages, table=table)
    kv = torch.randn(46, 2 * kvh, dim, generator=g).to(torch.float16)
    d, old = Dev(xp, kv), [x.host() for x in c.dcode]
    view = lambda t, w: U.rows(xp, t, kvh, "f16", 2 * kvh * dim, w * kvh * dim)  # noqa: E731
    xp.call("xp_paged_kv_write", c.desc, s.desc, view(d, 0), view(d, 1), None)
    back = Dev(xp, torch.full_like(kv, 5.0))
    xp.call("xp_paged_kv_read", c.desc, s.desc, view(back, 0), view(back, 1), None)
    xp.synchronize()
    got = back.host()
    assert torch.isnan(got[:40]).all() and (got[40:42] == 5.0).all() and torch.isfinite(got[42:]).all()
    for w in (0, 1):
        now = c.dcode[w].host().view(torch.uint8)
        touched = (now != old[w].view(torch.uint8)).reshape(pages, kvh, page, -1).any(-1).any(1)
        assert touched[2, :4].all() and int(touched.sum()) == 4


@pytest.mark.gpu
def test_gpu_paged_kv_past_32_bits(xp):
    """Rows whose offsets pass 2^32 bytes and elements, read and attended where they were written."""
    page, kvh, dim = 1024, 8, 256
    pages = (1 << 33) // (page * kvh * dim) // 4 + 2      # 2^31 elements of 16 bits and some: 4.3 GB a plane
    pages = pages * 2 + 1                                 # past 2^32 elements
    g = torch.Generator().manual_seed(8)
    planes = [xp.DeviceBuffer(pages * page * kvh * dim * 2) for _ in range(2)]
    desc = xp.XpPagedKv(planes[0].ptr, planes[1].ptr, None, None, ELEM["f16"], pages, page, kvh, dim)
    table = torch.tensor([[pages - 1], [0]], dtype=torch.int32)
    s = U.Seqs(xp, [3, 3], [3, 3], page, pages, table=table)
    kv = torch.randn(6, 2 * kvh, dim, generator=g).to(torch.float16)
    d, back = Dev(xp, kv), Dev(xp, torch.zeros_like(kv))
    view = lambda t, w: U.rows(xp, t, kvh, "f16", 2 * kvh * dim, w * kvh * dim)  # noqa: E731
    xp.call("xp_paged_kv_write", desc, s.desc, view(d, 0), view(d, 1), None)
    xp.call("xp_paged_kv_read", desc, s.desc, view(back, 0), view(back, 1), None)
    q = torch.randn(6, 2 * kvh, dim, generator=g).to(torch.float16)
    dq, out = Dev(xp, q), Dev(xp, torch.zeros_like(q))
    xp.call("xp_attention_paged", U.rows(xp, out, 2 * kvh, "f16", 2 * kvh * dim), U.rows(xp, dq, 2 * kvh, "f16", 2 * kvh * dim),
            desc, s.desc, 0, 1 / 16, None, 0, None)
    xp.synchronize()
    assert torch.equal(back.host(), kv)
    got = out.host().to(F64)
    for b in (0, 1):
        r = slice(3 * b, 3 * b + 3)
        want, size, most = U.attend(q[r].to(F64), kv[r, :kvh].to(F64), kv[r, kvh:].to(F64), 1 / 16, 0, 0)
        assert ((got[r] - want).abs() <= U.attention_bound(want, size, most, "f16", "f16")).all()
    for p in planes:
        p.close()


@pytest.mark.gpu
def test_gpu_outputs_have_to_be_device_memory(xp):
    host = np.zeros(4096, np.float16)
    r = lambda p: xp.XpRows(p, 64, 1, ELEM["f16"])  # noqa: E731
    dev = Dev(xp, torch.zeros(64, dtype=torch.float16))
    pos = Dev(xp, torch.zeros(1, dtype=torch.int32))
    at = (host.ctypes.data + 15) // 16 * 16
    with pytest.raises(xp.XposeError, match="not device memory"):
        xp.call("xp_rope_rows", r(at), r(dev.ptr), None, None, pos.ptr, 1, 64, rope_spec(xp), None)
    xp.call("xp_rope_rows", r(dev.ptr), r(dev.ptr), None, None, pos.ptr, 1, 64, rope_spec(xp), None)   # and no error is left behind
    xp.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("cache,elem", [("i8", "f32"), ("bf16", "f16")])
def test_gpu_paged_kv_many_sequences(xp, cache, elem):
    """Hundreds of sequences, many without a new row: what is written is what is read, and nothing else is."""
    g = torch.Generator().manual_seed(12)
    n, page, kvh, dim = 700, 16, 2, 32
    new = [(0, 1, 1, 5, 0, 2, 17)[i % 7] for i in range(n)]
    lens = [x + (i * 13) % 30 for i, x in enumerate(new)]
    pages = n * 3 + 1
    c = U.Cache(xp, g, cache, pages, page, kvh, dim).upload()
    s = U.Seqs(xp, new, lens, page, pages, n_tokens=sum(new) + 2, g=g, width=3)
    kv = torch.randn(s.n_tokens, 2 * kvh, dim, generator=g).to(DT[elem])
    d, back = Dev(xp, kv), Dev(xp, torch.full_like(kv, 5.0))
    view = lambda t, w: U.rows(xp, t, kvh, elem, 2 * kvh * dim, w * kvh * dim)  # noqa: E731
    xp.call("xp_paged_kv_write", c.desc, s.desc, view(d, 0), view(d, 1), None)
    xp.call("xp_paged_kv_read", c.desc, s.desc, view(back, 0), view(back, 1), None)
    xp.synchronize()
    got = back.host()
    assert (got[sum(new):] == 5.0).all()
    code, scale = U.quantise(kv[:sum(new)], cache)
    x = code.to(torch.float32)
    x = (x if scale is None else x * scale[..., None]).to(DT[elem])
    assert torch.equal(got[:sum(new)], x)
    # the slots that no token has are as they were
    want = [t.clone() for t in c.code]
    for t, b, p in s.tokens():
        for w in (0, 1):
            want[w][int(s.table[b, p // page]), :, p % page] = code[t, w * kvh:(w + 1) * kvh]
    for w in (0, 1):
        assert torch.equal(c.dcode[w].host().view(torch.uint8), want[w].view(torch.uint8))

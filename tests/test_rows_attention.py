"""Attention of packed rows, over a paged cache and over packed prompts: the
host's checks (CPU), the kernels against float64 (GPU)."""
import math

import numpy as np
import pytest
import torch

import rows_util as U
from rows_util import DT, ELEM, F64, Dev
from test_rows_ops import BAD_CACHES, BAD_SEQS, FAKE, cache_args, rope_ref, rope_spec, rows_args, seqs_args


# ---------------------------------------------------------------- CPU ----

def test_attention_paged_refuses(xh):
    out, q = rows_args(xh), rows_args(xh, data=FAKE * 2)

    def call(cache=None, seqs=None, q=q, out=out, scale=0.1, ws=(None, 0)):
        xh.call("xp_attention_paged", out, q, cache_args(xh, **(cache or {})), seqs_args(xh, **(seqs or {})), 0, scale, *ws, None)

    for bad, says in BAD_CACHES:
        with pytest.raises(xh.XposeError, match=says):
            call(cache=bad)
    for bad, says in BAD_SEQS:
        with pytest.raises(xh.XposeError, match=says):
            call(seqs=bad)
    for bad, says in (({"heads": 7, "stride": 512}, "heads"), ({"data": FAKE + 8}, "multiples"), ({"stride": 500}, "stride"),
                      ({"elem": 4}, "elem"), ({"elem": 0}, "elem"), ({"data": None}, "null")):
        with pytest.raises(xh.XposeError, match=says):
            call(out=rows_args(xh, **bad))
    odd = dict(data=FAKE * 2, heads=7, stride=512)
    for kw, says in ((dict(out=q), "must not be q"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
                     (dict(q=rows_args(xh, **odd), out=rows_args(xh, heads=7)), "multiple of 8"),
                     (dict(ws=(FAKE, 8)), "workspace"), (dict(cache={"elem": ELEM["bf16"]}), "BF16 queries")):
        with pytest.raises(xh.XposeError, match=says):
            call(**kw)
    call(seqs={"n_tokens": 0})
    call(seqs={"n_seq": 0})


def test_attention_packed_refuses(xh):
    r = {n: rows_args(xh, data=FAKE * (i + 1)) for i, n in enumerate(("out", "q", "k", "v"))}

    def call(dim=64, n_seq=2, n=8, cu=FAKE, scale=0.1, ws=(None, 0), **kw):
        x = {**r, **kw}
        xh.call("xp_attention_packed", x["out"], x["q"], x["k"], x["v"], dim, n_seq, n, cu, 0, scale, *ws, None)

    for kw, says in ((dict(dim=72), "head_dim"), (dict(dim=272), "head_dim"), (dict(cu=None), "cu is null"),
                     (dict(n=1 << 31), "too many"), (dict(scale=math.nan), "scale"), (dict(out=r["q"]), "must not be q"),
                     (dict(v=rows_args(xh, heads=4)), "v 4"), (dict(k=rows_args(xh, elem=2)), "all F16 or all BF16"),
                     (dict(q=rows_args(xh, elem=0), out=rows_args(xh, elem=0, data=FAKE * 9)), "all F16 or all BF16"),
                     (dict(k=rows_args(xh, heads=3)), "multiple of 3"), (dict(ws=(FAKE + 4, 1 << 30)), "workspace"),
                     (dict(k=rows_args(xh, data=FAKE + 2)), "multiples of 16")):
        with pytest.raises(xh.XposeError, match=says):
            call(**kw)
    call(n=0, cu=None)
    call(n_seq=0, cu=None)


def test_attention_workspace_sizes(xh):
    assert xh.attention_workspace(0, 0, 4, 1, 256) >= 0
    sizes = [xh.attention_workspace(n, b, 32, 8, 128) for n, b in ((1, 1), (64, 64), (4096, 8), (1 << 20, 1000))]
    assert all(s % 16 == 0 and s < 1 << 30 for s in sizes)
    for bad, says in (((1, 1, 7, 2, 128), "multiple"), ((1, 1, 4, 0, 128), "multiple"), ((1, 1, 4, 1, 100), "head_dim")):
        with pytest.raises(xh.XposeError, match=says):
            xh.attention_workspace(*bad)


# ---------------------------------------------------------------- GPU ----

def workspace(X, n_tokens, n_seq, heads, kvh, dim, use):
    if not use:
        return None, 0
    n = X.attention_workspace(n_tokens, n_seq, heads, kvh, dim)
    # what a former call left: nothing of it may show
    return Dev(X, torch.full((n // 4 + 1,), math.nan)).ptr, n


class Paged:
    """A call over pages, and its sequences in float64."""

    def __init__(self, X, new, past, heads, kvh, dim, elem, cache, page, window=0, seed=1, pad=2, std=1.5, split=True,
                 n_pages=None, table=None):
        g = torch.Generator().manual_seed(seed)
        self.X, self.window, self.scale, self.elem, self.op = X, window, dim ** -0.5, elem, "bf16" if cache == "bf16" else "f16"
        lens = [n + p for n, p in zip(new, past)]
        width = max([-(-n // page) for n in lens] + [1])
        self.pages = n_pages or len(new) * width + 1
        self.c = U.Cache(X, g, cache, self.pages, page, kvh, dim)
        self.s = U.Seqs(X, new, lens, page, self.pages, n_tokens=sum(new) + pad, g=g, table=table)
        self.q = (torch.randn(self.s.n_tokens, heads, dim, generator=g) * std).to(DT[elem])
        self.shape, self.split = (heads, kvh, dim), split

    def run(self, stream=None):
        X, (heads, kvh, dim) = self.X, self.shape
        self.c.upload()
        self.dq, self.dout = Dev(X, self.q), Dev(X, torch.full_like(self.q, 5.0))
        ws = workspace(X, self.s.n_tokens, len(self.s.new), heads, kvh, dim, self.split)
        view = lambda d: U.rows(X, d, heads, self.elem, heads * dim)  # noqa: E731
        self.args = (view(self.dout), view(self.dq), self.c.desc, self.s.desc, self.window, self.scale, *ws)
        X.call("xp_attention_paged", *self.args, stream)
        X.synchronize()
        return self.dout.host()

    def want(self, b):
        """(rows, out, size, most) of sequence b; keys without a row are NaN."""
        n, length = self.s.new[b], self.s.lens[b]
        kv = []
        for w in (0, 1):
            at = [self.c.at(w, self.s.table[b].tolist(), p) for p in range(length)]
            kv.append(torch.stack([torch.full(self.shape[1:], math.nan, dtype=F64) if x is None else x for x in at])
                      if at else torch.empty(0, *self.shape[1:], dtype=F64))
        r = slice(self.s.cu[b], self.s.cu[b] + n)
        return r, *U.attend(self.q[r].to(F64), *kv, self.scale, self.window, length - n)

    def check(self, got):
        assert (got[self.s.cu[-1]:] == 5.0).all(), "rows behind the last sequence"
        for b in range(len(self.s.new)):
            r, want, size, most = self.want(b)
            n, length = self.s.new[b], self.s.lens[b]
            x = got[r].to(F64)
            if n > length:                                # rows before the start belong to no sequence
                assert (x[:n - length] == 5.0).all()
                x, want, size, most = (t[n - length:] for t in (x, want, size, most))
            same = torch.equal(torch.isnan(x), torch.isnan(want)) and torch.equal(x[torch.isinf(want)], want[torch.isinf(want)])
            assert same, b
            fine = torch.isfinite(want)
            bound = U.attention_bound(want, size, most, self.elem, self.op)
            off = ((x - want).abs() / bound)[fine]
            assert not off.numel() or off.max() <= 1, (b, float(off.max()))


PAGED = [  # new, past, heads, kv heads, dim, q elem, cache, page, window
    ([1], [0], 1, 1, 16, "f16", "f16", 16, 0), ([1], [4095], 4, 1, 256, "f32", "f16", 64, 0),
    ([1] * 5, [0, 15, 16, 700, 2049], 8, 2, 128, "bf16", "bf16", 16, 0), ([1] * 3, [1, 63, 1500], 32, 8, 128, "bf16", "i8", 64, 0),
    ([1] * 4, [500, 2, 90, 0], 16, 1, 64, "f32", "e4m3", 32, 0), ([1, 1], [900, 30], 40, 2, 96, "f16", "i8", 128, 0),
    ([1] * 70, [i * 7 for i in range(70)], 4, 2, 64, "f16", "f16", 16, 0), ([1, 1, 0, 1], [300, 5, 7, 800], 4, 1, 256, "f32", "f16", 16, 512),
    ([3], [1200], 8, 8, 64, "bf16", "e4m3", 16, 0), ([17, 0, 1, 33], [100, 50, 400, 0], 12, 4, 192, "f16", "f16", 32, 0),
    ([200, 70], [300, 1], 4, 1, 256, "f32", "f16", 64, 128), ([129], [64], 16, 2, 128, "f16", "e4m3", 64, 0),
    ([100, 28, 300], [0, 513, 77], 32, 8, 128, "bf16", "bf16", 16, 0), ([64], [1000], 6, 2, 80, "f32", "i8", 256, 0),
    ([90], [10], 10, 2, 112, "bf16", "i8", 16, 50), ([65, 1], [0, 0], 7, 7, 48, "f16", "f16", 16, 1),
    ([40, 8], [33, 2], 4, 1, 256, "bf16", "bf16", 1024, 33), ([300], [2000], 4, 1, 256, "f32", "e4m3", 16, 0),
    ([31] * 9, [i * 40 for i in range(9)], 5, 1, 64, "f16", "f16", 16, 0), ([6, 2], [2, 5], 3, 1, 160, "bf16", "f16", 16, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("new,past,heads,kvh,dim,elem,cache,page,window", PAGED)
def test_gpu_attention_paged(xp, new, past, heads, kvh, dim, elem, cache, page, window, split):
    c = Paged(xp, new, past, heads, kvh, dim, elem, cache, page, window, split=split)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("new,cache,elem", [([6], "f16", "f16"), ([1, 90], "bf16", "bf16"), ([2, 70], "i8", "f32")])
def test_gpu_attention_paged_more_rows_than_length(xp, new, cache, elem):
    c = Paged(xp, new, [0] * len(new), 4, 2, 64, elem, cache, 16)
    c.s = U.Seqs(xp, new, [max(0, n - 2) for n in new], 16, c.pages, n_tokens=c.s.n_tokens, table=c.s.table)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("new,past", [([1, 1, 1], [100, 20, 60]), ([70, 3, 90], [100, 30, 0])])
@pytest.mark.parametrize("cache,elem", [("f16", "f16"), ("i8", "bf16"), ("bf16", "bf16"), ("e4m3", "f32")])
def test_gpu_attention_paged_bad_pages(xp, cache, elem, new, past):
    """Queries that see a position without a page get NaN, the others their values."""
    c = Paged(xp, new, past, 4, 2, 64, elem, cache, 16)
    c.s.table[0, 3] = -1
    c.s.table[2, 4] = c.pages
    c.s = U.Seqs(xp, new, c.s.lens, 16, c.pages, n_tokens=c.s.n_tokens, table=c.s.table[:, :8].contiguous())   # and past the table
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("cache,elem,dim", [("f16", "f16", 128), ("bf16", "bf16", 64), ("f16", "f32", 256), ("i8", "f16", 128),
                                            ("e4m3", "bf16", 64)])
def test_gpu_attention_paged_values_that_are_not_finite(xp, cache, elem, dim, window):
    """Rows with NaN and infinities in the cache, in K and in V: what does not see them does not have them."""
    c = Paged(xp, [1, 100, 33], [150, 60, 0], 4, 1, dim, elem, cache, 16, window)
    table, page = c.s.table, 16
    rows = {0: [(1, 30, math.inf)], 1: [(1, 100, math.nan), (0, 140, math.nan), (1, 62, math.inf), (1, 63, -math.inf)],
            2: [(1, 20, -math.inf), (0, 31, math.inf)]}
    for b, bad in rows.items():
        for w, p, x in bad:
            g, i = int(table[b, p // page]), p % page
            if c.c.scale[w] is not None:
                c.c.scale[w][g, :, i] = math.nan
                c.c.code[w][g, :, i] = torch.zeros_like(c.c.code[w][g, :, i])
            else:
                c.c.code[w][g, :, i, 5] = x
    # and behind each sequence's end, in its last page
    for b, length in enumerate(c.s.lens):
        if length % page:
            g = int(table[b, length // page])
            for w in (0, 1):
                if c.c.scale[w] is not None:
                    c.c.scale[w][g, :, length % page:] = math.nan
                else:
                    c.c.code[w][g, :, length % page:] = math.nan
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("elem,cache", [("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "i8"), ("bf16", "e4m3")])
def test_gpu_attention_paged_large_and_small_scores(xp, elem, cache):
    """Scores of hundreds (one weight is all), rows of zeros, and values near the type's ends."""
    for std, new in ((60.0, [1, 40]), (0.0, [1, 40]), (1e-3, [1, 40])):
        c = Paged(xp, new, [300, 77], 8, 2, 128, elem, cache, 16, std=std)
        if cache == "f16":
            c.c.code[1] = (c.c.code[1].float() * 1e4).to(torch.float16)
        elif cache in ("i8", "e4m3"):
            c.c.scale[1] *= 100.0 if elem == "f16" else 1e20
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("elem,cache,new", [("f32", "f16", [1, 1]), ("bf16", "i8", [1, 50])])
def test_gpu_attention_paged_strides_and_graph(xp, elem, cache, new):
    """Rows with others between them; the call captured into a graph and replayed on new lengths."""
    past, heads, kvh, dim, page = [700, 300], 8, 2, 128, 16
    c = Paged(xp, new, past, heads, kvh, dim, elem, cache, page)
    want = c.run()
    c.check(want)
    # the same rows a fused product away, the same output rows two apart
    n, gap = c.s.n_tokens, (heads + 2 * kvh) * dim
    fused = torch.zeros(n, gap, dtype=DT[elem])
    fused[:, :heads * dim] = c.q.reshape(n, -1)
    dq, dout = Dev(xp, fused), Dev(xp, torch.full((n, 2 * heads * dim), 5.0).to(DT[elem]))
    call = (U.rows(xp, dout, heads, elem, 2 * heads * dim), U.rows(xp, dq, heads, elem, gap), *c.args[2:])
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        xp.call("xp_attention_paged", *call, side.cuda_stream)
    for shorter in (0, 5, 13):
        lens = [x - shorter for x in (701, 300 + new[1])]
        c.s.lens = lens
        c.s.dev[1].buf.upload(np.array(lens, np.int32))
        dout.buf.upload(U.raw(torch.full((n, 2 * heads * dim), 5.0).to(DT[elem])))
        graph.replay()
        torch.cuda.synchronize()
        got = dout.host()
        assert (got[:, heads * dim:] == 5.0).all()
        c.check(got[:, :heads * dim].reshape(n, heads, dim))


@pytest.mark.gpu
def test_gpu_attention_calls_repeat_bit_for_bit(xp):
    c = Paged(xp, [1, 1, 1], [4000, 300, 1999], 8, 2, 128, "bf16", "i8", 16)
    first = c.run()
    for _ in range(3):
        assert torch.equal(c.run().view(torch.int16), first.view(torch.int16))


PACKED = [  # lengths, heads, kv heads, dim, elem, window
    ([1], 1, 1, 16, "f16", 0), ([1, 1, 0, 2], 4, 2, 64, "bf16", 0), ([200], 4, 1, 256, "f16", 0), ([333, 1, 64, 65], 8, 2, 128, "bf16", 0),
    ([500], 4, 1, 256, "f16", 100), ([63, 128, 129], 6, 3, 96, "f16", 0), ([90, 400], 7, 7, 80, "bf16", 64), ([1030], 16, 1, 64, "f16", 0),
    ([257], 5, 1, 192, "bf16", 1), ([40] * 33, 2, 1, 48, "f16", 0), ([700], 32, 8, 128, "f16", 17), ([300], 12, 1, 256, "bf16", 0)]


def packed(xp, lens, heads, kvh, dim, elem, window, split=True, pad=3, poison=(), stream=None):
    g = torch.Generator().manual_seed(sum(lens) + dim)
    n = sum(lens) + pad
    row = (heads + 2 * kvh) * dim
    qkv = (torch.randn(n, heads + 2 * kvh, dim, generator=g) * 1.3).to(DT[elem])
    for t, h, d, x in poison:
        qkv[t, heads + h, d] = x
    cu = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32)
    d, dcu, out = Dev(xp, qkv), Dev(xp, cu), Dev(xp, torch.full((n, heads, dim), 5.0).to(DT[elem]))
    view = lambda h, o: U.rows(xp, d, h, elem, row, o * dim)  # noqa: E731
    xp.call("xp_attention_packed", U.rows(xp, out, heads, elem, heads * dim), view(heads, 0), view(kvh, heads), view(kvh, heads + kvh),
            dim, len(lens), n, dcu.ptr, window, dim ** -0.5, *workspace(xp, n, len(lens), heads, kvh, dim, split), stream)
    xp.synchronize()
    got = out.host()
    assert (got[sum(lens):] == 5.0).all()
    for b, length in enumerate(lens):
        r = slice(int(cu[b]), int(cu[b]) + length)
        x = qkv[r].to(F64)
        want, size, most = U.attend(x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:], dim ** -0.5, window, 0)
        y = got[r].to(F64)
        same = torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[torch.isinf(want)], want[torch.isinf(want)])
        assert same, b
        fine = torch.isfinite(want)
        off = ((y - want).abs() / U.attention_bound(want, size, most, elem, elem))[fine]
        assert not off.numel() or off.max() <= 1, (b, float(off.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("lens,heads,kvh,dim,elem,window", PACKED)
def test_gpu_attention_packed(xp, lens, heads, kvh, dim, elem, window, split):
    packed(xp, lens, heads, kvh, dim, elem, window, split)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("dim,elem", [(64, "f16"), (128, "bf16"), (256, "f16")])
def test_gpu_attention_packed_values_that_are_not_finite(xp, dim, elem, window):
    kvh = 2
    bad = [(10, kvh, 3, math.nan), (77, kvh + 1, 0, math.inf), (78, kvh + 1, 0, -math.inf), (130, 0, 7, math.nan), (250, kvh, dim - 1, math.inf)]
    packed(xp, [60, 140, 120], 8, kvh, dim, elem, window, poison=bad)


@pytest.mark.gpu
@pytest.mark.parametrize("cache,elem,page", [("f16", "f32", 16), ("i8", "bf16", 64), ("e4m3", "f16", 32), ("bf16", "bf16", 128)])
def test_gpu_a_server_step(xp, cache, elem, page):
    """A prompt's chunk for one sequence and single tokens for others, through one layer's run of the operators: turned,
    written, attended, on a stream of its own; the chunk's keys are in the cache only through the write."""
    g = torch.Generator().manual_seed(11)
    new, past, heads, kvh, dim = [40, 1, 0, 1], [25, 130, 12, 0], 8, 2, 64
    c = Paged(xp, new, past, heads, kvh, dim, elem, cache, page, pad=0)
    n, row = c.s.n_tokens, (heads + 2 * kvh) * dim
    qkv = torch.randn(n, heads + 2 * kvh, dim, generator=g).to(DT[elem])
    pos = torch.tensor([p for _, _, p in c.s.tokens()], dtype=torch.int32)
    spec = rope_spec(xp, rot_dim=32, scaling=xp.XP_ROPE_BANDS, theta=5e5)
    c.c.upload()
    d, dpos, out = Dev(xp, qkv), Dev(xp, pos), Dev(xp, torch.zeros(n, heads, dim).to(DT[elem]))
    q, k, v = (U.rows(xp, d, h, elem, row, o * dim) for h, o in ((heads, 0), (kvh, heads), (kvh, heads + kvh)))
    ws = workspace(xp, n, len(new), heads, kvh, dim, True)
    side = torch.cuda.Stream()
    st = side.cuda_stream
    xp.call("xp_rope_rows", q, q, k, k, dpos.ptr, n, dim, spec, st)
    xp.call("xp_paged_kv_write", c.c.desc, c.s.desc, k, v, st)
    xp.call("xp_attention_paged", U.rows(xp, out, heads, elem, heads * dim), q, c.c.desc, c.s.desc, 0, c.scale, *ws, st)
    side.synchronize()
    turned = d.host()
    want, size = rope_ref(qkv[:, :heads + kvh], pos, xp.rope_frequencies(spec), 0, 32, 1.0)
    assert ((turned[:, :heads + kvh].to(F64) - want).abs() <= size * 2.0 ** -20 + U.HALF[elem] * want.abs() * 1.01).all()
    assert torch.equal(turned[:, heads + kvh:], qkv[:, heads + kvh:])
    c.q = turned[:, :heads]
    for t, b, p in c.s.tokens():
        for w in (0, 1):
            code, scale = U.quantise(turned[t, heads + w * kvh:heads + (w + 1) * kvh], cache)
            c.c.code[w][int(c.s.table[b, p // page]), :, p % page] = code
            if scale is not None:
                c.c.scale[w][int(c.s.table[b, p // page]), :, p % page] = scale
    c.check(out.host())


def wide_table(new, past, page, positions=8192, seed=5):
    """(page table of `positions` positions a sequence, pages): the pages in use in any order, none behind them."""
    used = [-(-(n + p) // page) for n, p in zip(new, past)]
    order = torch.randperm(sum(used) + 1, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(new), positions // page), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(used) + 1


@pytest.mark.gpu
@pytest.mark.parametrize("new,past,heads,kvh,dim,elem,cache,page,window", PAGED)
def test_gpu_attention_paged_in_wide_tables(xp, new, past, heads, kvh, dim, elem, cache, page, window):
    """Tables with room for 8192 positions, as a server's are: the host takes the call for a long one."""
    table, pages = wide_table(new, past, page)
    c = Paged(xp, new, past, heads, kvh, dim, elem, cache, page, window, n_pages=pages, table=table)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [100, 20, 60]), ([70, 3, 90], [100, 30, 0])])
@pytest.mark.parametrize("cache,elem", [("f16", "f16"), ("i8", "bf16"), ("bf16", "bf16"), ("e4m3", "f32")])
def test_gpu_attention_paged_wide_tables_with_bad_pages(xp, cache, elem, new, past, window):
    table, pages = wide_table(new, past, 16)
    table[0, 3], table[2, 4] = -1, pages
    c = Paged(xp, new, past, 4, 2, 64, elem, cache, 16, window, n_pages=pages, table=table)
    if cache in ("f16", "bf16"):                          # and values that are not finite
        c.c.code[1][int(table[1, 0]), :, 3, 7] = math.inf
        c.c.code[0][int(table[1, 1]), :, 2, 1] = math.nan
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("elem,cache,positions", [("bf16", "i8", 512), ("f16", "f16", 8192), ("f32", "e4m3", 8192)])
def test_gpu_attention_paged_many_sequences(xp, elem, cache, positions, split):
    """More sequences than a wave has lanes several times over, some with no row, a few of a chunk; two share their pages."""
    n = 300
    new = [0 if i % 7 == 3 else 9 if i % 50 == 1 else 1 for i in range(n)]
    past = [(i * 37) % 250 for i in range(n)]
    table, pages = wide_table(new, past, 16, positions)
    new[20] = new[21] = 1
    past[20] = past[21] = 40
    table[21, :3] = table[20, :3] = torch.arange(3)
    c = Paged(xp, new, past, 4, 2, 32, elem, cache, 16, n_pages=pages, table=table, split=split)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 1 << 30, (1 << 32) - 1])
@pytest.mark.parametrize("new,past", [([1, 1], [600, 0]), ([70, 20], [50, 300])])
def test_gpu_attention_paged_least_and_largest_windows(xp, new, past, window):
    for positions in (1024, 8192):
        table, pages = wide_table(new, past, 16, positions)
        c = Paged(xp, new, past, 4, 2, 64, "f16", "f16", 16, window, n_pages=pages, table=table)
        c.check(c.run())


@pytest.mark.gpu
def test_gpu_attention_calls_on_two_streams(xp):
    """Two calls at once, a workspace each, and the one of the other's sizes after it in the same stream."""
    calls = []
    for i, (new, past, elem, cache) in enumerate((([1, 1, 1], [4000, 300, 1999], "bf16", "i8"), ([40, 1, 100], [500, 3000, 0], "f16", "f16"))):
        table, pages = wide_table(new, past, 16)
        c = Paged(xp, new, past, 8, 2, 128, elem, cache, 16, n_pages=pages, table=table, seed=i + 1)
        calls.append((c, c.run()))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for c, _ in calls:
        c.dout.buf.upload(U.raw(torch.full_like(c.q, 5.0)))
    for _ in range(20):
        for (c, _), st in zip(calls, streams):
            xp.call("xp_attention_paged", *c.args, st.cuda_stream)
    torch.cuda.synchronize()
    for c, alone in calls:
        assert torch.equal(c.dout.host().view(torch.int16), alone.view(torch.int16))
        c.check(alone)


@pytest.mark.gpu
@pytest.mark.parametrize("elem,cache", [("f16", "f16"), ("bf16", "i8")])
@pytest.mark.parametrize("cu", [[0, 9, 4, 20], [-5, 30, 30, 2], [7, 3, 50, 1 << 30]])
def test_gpu_malformed_sequences_keep_to_their_rows(xp, elem, cache, cu):
    """A cu that falls or leaves the rows: whatever the call makes of it, nothing outside the descriptors changes."""
    heads, kvh, dim, page, n = 4, 2, 64, 16, 12
    for positions in (64, 8192):
        table, pages = wide_table([9, 9, 9], [20, 3, 30], page, positions)
        c = Paged(xp, [4, 4, 4], [20, 3, 30], heads, kvh, dim, elem, cache, page, n_pages=pages, table=table, pad=0)
        c.s.dev[0].buf.upload(np.array(cu, np.int32))
        c.c.upload()
        guard = torch.full((3 * n, heads, dim), 5.0).to(DT[elem])
        dq, dout = Dev(xp, torch.randn(3 * n, heads, dim).to(DT[elem])), Dev(xp, guard)
        at = lambda d, h: U.rows(xp, d, h, elem, heads * dim, n * heads * dim)  # noqa: E731
        ws = workspace(xp, n, 3, heads, kvh, dim, True)
        xp.call("xp_attention_paged", at(dout, heads), at(dq, heads), c.c.desc, c.s.desc, 0, 0.1, *ws, None)
        xp.call("xp_attention_packed", at(dout, heads), at(dq, heads), at(dq, kvh), at(dq, kvh), dim, 3, n, c.s.dev[0].ptr, 0, 0.1, *ws, None)
        xp.call("xp_paged_kv_write", c.c.desc, c.s.desc, at(dq, kvh), at(dq, kvh), None)
        xp.call("xp_paged_kv_read", c.c.desc, c.s.desc, at(dout, kvh), at(dout, kvh), None)
        xp.synchronize()
        got = dout.host()
        assert (got[:n] == 5.0).all() and (got[2 * n:] == 5.0).all()


def few_of_packed(xp, qkv, got, heads, kvh, dim, elem, window, every):
    """Every `every`-th query of one prompt against float64."""
    x = qkv.to(F64)
    n = x.shape[0]
    for i in sorted(set(range(0, n, every)) | {n - 1}):
        want, size, most = U.attend(x[i:i + 1, :heads], x[:i + 1, heads:heads + kvh], x[:i + 1, heads + kvh:], dim ** -0.5, window, i)
        # (over 4096 keys the bound's sums have up to twice the roundings, 2^-14 for 2^-15)
        bound = U.attention_bound(want, size, most, elem, elem) + 2.0 ** -15 * size
        assert ((got[i:i + 1].to(F64) - want).abs() <= bound).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads,kvh,dim,elem,window", [(5000, 2, 1, 256, "f16", 0), (6001, 3, 1, 128, "bf16", 0), (7000, 4, 1, 64, "f16", 3000),
                                                         (5000, 2, 2, 96, "bf16", 4500)])
def test_gpu_attention_packed_long_prompts_and_graph(xp, n, heads, kvh, dim, elem, window):
    """One long prompt of few heads, whose keys are split; captured, and replayed on another prompt and a shorter one."""
    g = torch.Generator().manual_seed(n)
    row = (heads + 2 * kvh) * dim
    cu = torch.tensor([0, n], dtype=torch.int32)
    d, dcu = Dev(xp, torch.zeros(n, heads + 2 * kvh, dim).to(DT[elem])), Dev(xp, cu)
    out = Dev(xp, torch.zeros(n, heads, dim).to(DT[elem]))
    view = lambda h, o: U.rows(xp, d, h, elem, row, o * dim)  # noqa: E731
    call = (U.rows(xp, out, heads, elem, heads * dim), view(heads, 0), view(kvh, heads), view(kvh, heads + kvh), dim, 1, n, dcu.ptr, window,
            dim ** -0.5, *workspace(xp, n, 1, heads, kvh, dim, True))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        xp.call("xp_attention_packed", *call, side.cuda_stream)
    for length in (n, n, 700):
        qkv = (torch.randn(n, heads + 2 * kvh, dim, generator=g) * 1.3).to(DT[elem])
        d.buf.upload(U.raw(qkv))
        dcu.buf.upload(np.array([0, length], np.int32))
        out.buf.upload(U.raw(torch.full((n, heads, dim), 5.0).to(DT[elem])))
        graph.replay()
        torch.cuda.synchronize()
        got = out.host()
        assert (got[length:] == 5.0).all()
        few_of_packed(xp, qkv[:length], got, heads, kvh, dim, elem, window, max(1, length // 40))
        xp.call("xp_attention_packed", *call, None)       # the same without a graph
        xp.synchronize()
        assert torch.equal(out.host().view(torch.int16), got.view(torch.int16))


@pytest.mark.parametrize("dim", [16, 64, 128, 256])
@pytest.mark.parametrize("heads,kvh", [(1, 1), (32, 8), (40, 1)])
def test_workspace_of_one_sequence_suffices_for_any_number(xh, heads, kvh, dim):
    sizes = (1, 2, 7, 8, 9, 31, 32, 33, 64, 1000, 5000)
    for most in sizes:
        need = xh.attention_workspace(most, 1, heads, kvh, dim)
        for n in (x for x in sizes if x <= most):
            assert all(xh.attention_workspace(n, b, heads, kvh, dim) <= need for b in (1, 2, 5, 64, 4000))


@pytest.mark.gpu
@pytest.mark.parametrize("new,past", [([1, 1], [700, 30]), ([5, 1], [20, 300])])
def test_gpu_attention_paged_more_heads_than_a_tile_has_rows(xp, new, past):
    for positions in (1024, 8192):
        table, pages = wide_table(new, past, 16, positions)
        c = Paged(xp, new, past, 200, 1, 64, "f16", "f16", 16, n_pages=pages, table=table)
        c.check(c.run())

"""What the tests of packed rows and paged caches share: element types on the
host, device views, and the operators restated in float64."""
import ctypes as C
import math

import numpy as np
import torch

from conftest import hold

F64 = torch.float64
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
      "e4m3": torch.float8_e4m3fn}
ELEM = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3, "e4m3": 4}
# the largest relative error of one rounding to the type: half a step
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def raw(t: torch.Tensor) -> np.ndarray:
    return t.contiguous().view(torch.uint8).numpy().reshape(-1)


class Dev:
    """A host tensor's copy in device memory, held until the test ends."""

    def __init__(self, X, t: torch.Tensor):
        self.shape, self.dtype = tuple(t.shape), t.dtype
        self.n = t.numel() * t.element_size()
        self.buf = X.DeviceBuffer(max(self.n, 16))
        if self.n:
            self.buf.upload(raw(t))
        hold(self.buf)
        self.ptr = self.buf.ptr

    def host(self) -> torch.Tensor:
        a = self.buf.download(np.uint8, self.n)
        return torch.from_numpy(a).view(self.dtype).reshape(self.shape)


def rows(X, d: Dev, heads: int, elem: str, stride: int, offset: int = 0):
    return X.XpRows(d.ptr + offset * DT[elem].itemsize, stride, heads, ELEM[elem])


def quantise(x: torch.Tensor, elem: str):
    """(codes as stored, float32 scale of each row or None) of rows, in float64."""
    if elem in ("f16", "bf16"):
        return x.to(DT[elem]), None
    x = x.to(F64)
    top = x.abs().amax(-1)
    finite = torch.isfinite(top)
    safe = torch.where(finite[..., None], x, torch.zeros_like(x))
    top = safe.abs().amax(-1)
    if elem == "i8":
        scale = (top / 127).to(torch.float32).clamp(min=2.0 ** -126)
        code = torch.round(safe / scale.to(F64)[..., None]).to(torch.int8)
    else:
        m, e = torch.frexp(top)
        k = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126)
        scale = torch.exp2(k.to(F64)).to(torch.float32)
        code = (safe / scale.to(F64)[..., None]).to(torch.float32).to(torch.float8_e4m3fn)
    scale = torch.where(top > 0, scale, torch.zeros_like(scale))
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    return code, scale


def values(code: torch.Tensor, scale) -> torch.Tensor:
    x = code.to(torch.float32).to(F64)
    return x if scale is None else x * scale.to(F64)[..., None]


class Cache:
    """Pages of K and V on the host and on the device."""

    def __init__(self, X, g, elem, pages, page, kv_heads, dim, std=1.0):
        self.X, self.elem, self.shape = X, elem, (pages, kv_heads, page, dim)
        kv = [quantise(torch.randn(self.shape, generator=g) * std, elem) for _ in range(2)]
        self.code, self.scale = [c for c, _ in kv], [s for _, s in kv]

    def upload(self):
        self.dcode = [Dev(self.X, c) for c in self.code]
        self.dscale = [None if s is None else Dev(self.X, s) for s in self.scale]
        p, h, n, d = self.shape
        self.desc = self.X.XpPagedKv(self.dcode[0].ptr, self.dcode[1].ptr,
                                     *(None if s is None else s.ptr for s in self.dscale), ELEM[self.elem], p, n, h, d)
        return self

    def at(self, kv: int, table, position: int):
        """Every head's row of a position of a sequence, float64 [kv_heads][dim], or None."""
        page = self.shape[2]
        if position < 0 or position // page >= len(table):
            return None
        g = int(table[position // page])
        if not 0 <= g < self.shape[0]:
            return None
        s = self.scale[kv]
        return values(self.code[kv][g, :, position % page], None if s is None else s[g, :, position % page])


class Seqs:
    """Ragged sequences: new rows, lengths and page tables."""

    def __init__(self, X, new, lens, page, n_pages, n_tokens=None, table=None, width=None, g=None):
        self.new, self.lens, self.page = list(new), list(lens), page
        self.cu = [0]
        for n in self.new:
            self.cu.append(self.cu[-1] + n)
        self.n_tokens = self.cu[-1] if n_tokens is None else n_tokens
        width = width or max([-(-n // page) for n in self.lens] + [1])
        if table is None:
            order = torch.randperm(n_pages, generator=g)[:len(self.new) * width]
            table = order.reshape(len(self.new), width).to(torch.int32)
        self.table = table
        i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        self.dev = [Dev(X, i32(self.cu)), Dev(X, i32(self.lens)), Dev(X, table.contiguous())]
        self.desc = X.XpPagedSeqs(len(self.new), self.n_tokens, *(d.ptr for d in self.dev), table.shape[1])

    def tokens(self):
        """(packed row, sequence, position) of every row that a sequence has."""
        for b, n in enumerate(self.new):
            for i in range(n):
                if self.lens[b] - n + i >= 0:
                    yield self.cu[b] + i, b, self.lens[b] - n + i


def attend(q, keys, vals, scale, window, first):
    """One sequence in float64: q [new][heads][dim], keys and vals [position][kv_heads][dim], query i at
    position first + i. Returns (out, sum_j p_j |v_j|, (largest sum_d |q_d k_d| scale, floor)): the last two bound errors."""
    n, heads, dim = q.shape
    if keys.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q), torch.zeros(n, heads, 2, dtype=F64)
    group = heads // keys.shape[1]
    k, v = (x.repeat_interleave(group, 1).permute(1, 0, 2) for x in (keys, vals))
    place = first + torch.arange(n)[:, None]
    j = torch.arange(keys.shape[0])[None]
    hidden = (j > place) | ((j <= place - window) if window else (j < 0))
    qs = q.permute(1, 0, 2)
    s = ((qs @ k.transpose(1, 2).contiguous()) * scale).masked_fill(hidden, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(hidden.all(-1)[None, :, None], torch.zeros_like(p), p)
    out, size = torch.empty(heads, n, dim, dtype=F64), torch.empty(heads, n, dim, dtype=F64)
    for i in range(n):                       # a value that a query does not see is not multiplied, not even by 0
        see = ~hidden[i]
        out[:, i] = (p[:, i, see][:, None] @ v[:, see])[:, 0]
        size[:, i] = (p[:, i, see][:, None] @ v[:, see].abs())[:, 0]
    most = (qs.abs() @ k.abs().transpose(1, 2) * scale).masked_fill(hidden, 0).nan_to_num(0).amax(-1)
    largest = torch.where(hidden[None, :, :], 0.0, v.abs().nan_to_num(0, posinf=0).amax(-1)[:, None, :]).amax(-1)
    floor = 2.0 ** -30 * (~hidden).sum(-1)[None] * largest
    return out.permute(1, 0, 2), size.permute(1, 0, 2), torch.stack((most, floor), -1).permute(1, 0, 2)


def attention_bound(out, size, most, elem, op):
    """How far an attention output may be from attend()'s, per element, over at most 4096 keys of at most 256
    dims. `size` = sum_j p_j |v_j|, `most` = S, the largest sum_d |q_d k_d| scale of a row, and the floor of its
    weights: F16 ones, the largest at least 2^6 (after a shift that the quotient takes back, and over a power of two
    at most twice the largest scale of an 8-bit cache), are off by 2^-24 at most however small they are: 2^-30 of the
    largest value for each key (nothing beside the rest, unless the value of the key that has all the weight is 0).
    In units of `size`:
      the weights' one rounding to the product's operands, half a step of `op` (two F16 terms, the
      first cut off and the second rounded: 2^-10 2^-11);
      the scores: sums of 256 exact products in blocks of 16 or more with at most 16 + 8 roundings of at most
      S 2^-24, the scales' two more: under 2^-19 S, which moves a weight and the sum of the weights by as
      much each; the exponential's argument, at most 2 S large, has 24 bits and its function 2 ulp: with the
      difference to the maximum under 2^-21 S + 2^-22 for a weight, twice for the quotient: 2^-17 S + 2^-20 in all;
      the sums over the keys: one rounding for each block of 16 or more keys and one rescaling for each of 32
      or more, 4096 / 16 + 4096 / 32 + 16 < 2^9 of 2^-24: 2^-15.
    Last the output's own rounding, and half of the least F16 number."""
    weights = 2.0 ** -21 if elem == "f32" else HALF[op]
    rel = weights + 2.0 ** -15 + 2.0 ** -17 * most[..., :1]
    return (size * rel + (most[..., 1:] if op == "f16" else 0.0) + HALF[elem] * out.abs()) * 1.01 + 2.0 ** -25

"""How the attention of packed rows deals its blocks to workgroups: every block of
every tile once, whatever the lengths (host index functions, no GPU)."""
import ctypes as C
import os
import random

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def rd(xh):
    lib = C.CDLL(os.path.join(HERE, "native", "rows_deal.so"))
    u = C.c_uint32
    lib.rd_walk.argtypes = [C.c_void_p, C.c_void_p] + [u] * 8 + [C.c_int32, C.c_void_p, C.c_void_p]
    return lib


def walk(rd, new, lens, heads, kv_heads, window, row_shift, block_shift, target, most=1 << 20):
    cu = np.cumsum([0] + new).astype(np.int32)
    kv = None if lens is None else np.array(lens, np.int32)
    blocks, waste = C.c_uint32(), C.c_uint32()
    rc = rd.rd_walk(cu.ctypes.data, None if kv is None else kv.ctypes.data, len(new), int(cu[-1]), heads, kv_heads, window, row_shift,
                    block_shift, target, most, C.byref(blocks), C.byref(waste))
    return rc, blocks.value, waste.value


@pytest.mark.parametrize("new,lens,heads,kv_heads,window,row_shift,block_shift", [
    ([1], [1], 1, 1, 0, 4, 6), ([1], [4096], 4, 1, 0, 4, 6), ([1] * 64, [100 * i + 1 for i in range(64)], 32, 8, 0, 4, 7),
    ([512, 1, 0, 300], [15512, 77, 9, 300], 32, 8, 0, 7, 6), ([2000], None, 4, 1, 512, 7, 5), ([2000], None, 4, 1, 0, 7, 5),
    ([333, 1, 64, 65], None, 8, 2, 0, 7, 6), ([40], [10], 7, 7, 0, 7, 6), ([300, 300], [200, 290], 1, 1, 40, 7, 6),
    ([1, 1, 1], [0, -5, 2 ** 31 - 1], 4, 2, 0, 4, 6), ([5000], [9000], 1, 1, 0, 7, 6)])
@pytest.mark.parametrize("target", [8, 512])
def test_every_block_is_dealt_once(rd, new, lens, heads, kv_heads, window, row_shift, block_shift, target):
    rc, blocks, waste = walk(rd, new, lens, heads, kv_heads, window, row_shift, block_shift, target, most=20000)
    assert rc == 0, (rc, blocks, waste)


def test_every_block_is_dealt_once_over_random_calls(rd):
    r = random.Random(7)
    for _ in range(400):
        n = r.choice([1, 2, 5, 70, 130])
        new = [r.choice([0, 1, 1, 2, r.randint(1, 900 if n < 9 else 40)]) for _ in range(n)]
        past = [r.choice([0, r.randint(0, 3000), -r.randint(0, 50)]) for _ in range(n)]
        kv_heads, group = r.choice([(1, 1), (1, 4), (8, 4), (2, 5), (3, 7), (1, 40)])
        lens = None if r.random() < 0.4 else [a + b for a, b in zip(new, past)]
        args = (kv_heads * group, kv_heads, r.choice([0, 0, 1, 17, 128, 1000, 2 ** 31]), r.choice([4, 7, 8]), r.choice([5, 6, 7, 8]),
                r.choice([8, 64, 512]), r.choice([1 << 20, 512]) if lens else sum(new))
        rc, blocks, waste = walk(rd, new, lens, *args)
        assert rc == 0, (rc, new, lens, args)


def test_little_of_a_list_is_gaps(rd):
    """A causal prompt's pairs of tiles are nearly alike, so that runs of equal places are runs of equal work. (A window
    of 512 and 32 tokens fill 9 or 10 blocks of 64, and the list has room for 10: two places of twenty, and the first
    tiles, which see less.)"""
    for new, heads, kv_heads, window, most in (([2000], 4, 1, 0, 60), ([16384], 16, 2, 0, 60), ([1000, 777, 400], 8, 2, 0, 120),
                                               ([8000], 4, 1, 512, 150)):
        rc, blocks, waste = walk(rd, new, None, heads, kv_heads, window, 7, 6, 512, sum(new))
        assert rc == 0 and waste < most, (new, waste)


def test_division_by_the_group(rd):
    r = np.random.default_rng(3)
    for d in [*range(1, 70), 127, 128, 129, 1000, 4096, 65535]:
        top = 2 ** 31 - 1
        q = r.integers(0, top // d, 200)
        n = np.concatenate([r.integers(0, 2 ** 31, 500), q * d, np.maximum(q * d, 1) - 1, [0, 1, top, top - 1, top // d * d, top // d * d - 1]])
        n = n.astype(np.uint32)
        assert rd.rd_by_group(d, n.ctypes.data_as(C.c_void_p), n.size) == 0, d

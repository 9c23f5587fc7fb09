"""Refusals of the paged cache's calls that depend on their arrays' layout, without a GPU."""
import ctypes as C
import random

import pytest

import fusor_attn as fa
from test_paged_cpu import Host, cache_c, message


def read(rows, kv_heads, head_dim, keys, values, row_stride, head_stride, dtype, call="read"):
    """Whether a read into rows of that layout is refused for overlapping (it is refused in any case:
    the pointers are none that CUDA knows)."""
    c = cache_c(heads=2 * kv_heads, kv_heads=kv_heads, head_dim=head_dim)
    h = Host(starts=(0, rows), firsts=(0,), tables=((0,) * 8,), max_rows=rows)
    r = fa._PagedRows(keys, values, row_stride, head_stride, dtype)
    f = fa.lib().fa_paged_read if call == "read" else fa.lib().fa_paged_write
    assert f(C.byref(c), 0, C.byref(h.c), C.byref(r), None) == fa.ERR_ARG
    return "overlap" in message()


@pytest.mark.parametrize("dtype", [fa.F32, fa.BF16])
def test_reads_into_overlapping_rows_are_refused(dtype):
    e, base = (4 if dtype == fa.F32 else 2), 1 << 20
    far = base + (1 << 16)

    def refused(rows, heads, rs, hs, values=far, call="read"):
        return read(rows, heads, 64, base, values, rs, hs, dtype, call)

    assert refused(5, 2, 0, 64) and refused(5, 2, 128, 0) and refused(5, 2, 127, 64)
    assert refused(5, 2, 128, 63) and refused(5, 2, 64, 256)
    assert not refused(5, 2, 128, 64) and not refused(5, 2, 64, 320) and not refused(5, 2, 64, 500)
    # one row, one head: their strides say nothing
    assert not refused(1, 2, 0, 64) and not refused(5, 1, 64, 0) and not refused(1, 1, 0, 0)
    # keys and values side by side in each row, or one array; not in part
    assert not refused(5, 2, 256, 64, base + 128 * e) and not refused(5, 2, 128, 64, base)
    assert refused(5, 2, 256, 64, base + 127 * e) and refused(5, 2, 128, 64, base + 128 * e)
    assert refused(5, 2, 256, 64, base - 64 * e) and not refused(5, 2, 256, 64, base - 128 * e)
    # what is only read may repeat
    assert not refused(5, 2, 0, 0, call="write")


def test_overlaps_as_counted():
    """Random layouts against the elements themselves."""
    rng = random.Random(5)
    seen = set()
    for _ in range(3000):
        rows, heads = rng.randint(1, 4), rng.randint(1, 4)
        d = 64
        rs, hs = (rng.choice([0, 32, 63, 64, 65, 96, 128, 192, 200, 256, 260]) for _ in range(2))
        apart = rng.choice([0, 64, 128, 192, 256, 320, 448, 512, 700, 1024]) * rng.choice([1, -1])
        apart += rng.choice([0, 0, 0, 1, -1])
        base = 1 << 20
        sets = []
        for at in (base, base + apart):
            count = {}
            for i in range(rows):
                for j in range(heads):
                    for x in range(d):
                        y = at + i * rs + j * hs + x
                        count[y] = count.get(y, 0) + 1
            sets.append(count)
        want = max(sets[0].values()) > 1 or (apart != 0 and bool(sets[0].keys() & sets[1].keys()))
        assert read(rows, heads, d, 4 * base, 4 * (base + apart), rs, hs, fa.F32) == want, (
            rows, heads, rs, hs, apart)
        seen.add(want)
    assert seen == {True, False}


def test_norm_weights_are_checked():
    """Weights shorter than a head, of another type or with gaps are refused before the library (whose
    kernels read head_dim floats) is called."""
    import torch

    pages = torch.zeros((1, 3, 2, 16, 64), dtype=torch.bfloat16)
    cache = fa.PagedCache(fa.Shape(1, 4, 2, 64), 3, 16, fa.BF16, keys=pages, values=pages.clone())

    class Batch:
        _ref = None

        def covers(self, *tensors):
            pass

    qkv, out, angles = torch.zeros((2, 512)), torch.zeros((2, 256)), torch.zeros((2, 64))
    good = torch.ones(64)
    for bad in (torch.ones(63), torch.ones(128), torch.ones(64).bfloat16(), torch.ones(64).double(),
                torch.ones(128)[::2], torch.ones((1, 64)), torch.tensor(1.0)):
        for norm in ((bad, good, 1e-6), (good, bad, 1e-6), (bad, None, 1e-6), (None, bad, 1e-6)):
            with pytest.raises(ValueError, match="norm weights"):
                cache.attention_input(0, Batch(), qkv, angles, norm=norm)
            with pytest.raises(ValueError, match="norm weights"):
                cache.attention(0, Batch(), qkv, out, angles, norm=norm)

"""The paged cache's refusals and the host's check of a batch's numbers, without a GPU: every
argument is checked before any launch, and fa_paged_check applies the kernels' own checks to host
copies of row_starts, firsts and tables."""
import ctypes as C

import numpy as np
import pytest

import fusor_attn as fa


def cache_c(**over):
    base = dict(layers=2, heads=8, kv_heads=2, head_dim=128, pages=10, page_size=16, dtype=fa.Q8,
                device=0, keys=4096, values=8192, key_scales=4096, value_scales=8192)
    base.update(over)
    return fa._PagedCache(*[base[n] for n, _ in fa._PagedCache._fields_])


class Host:
    """A batch over host arrays."""

    def __init__(self, starts=(0, 1, 4), firsts=(17, 0), tables=((3, 4), (0, 9)), null=None, **over):
        self.starts = np.array(starts, np.int32)
        self.firsts = np.array(firsts, np.int32)
        self.tables = np.array(tables, np.int32)
        base = dict(sequences=len(firsts), rows=int(starts[-1]), max_rows=8,
                    table_width=self.tables.shape[1], table_stride=self.tables.shape[1],
                    row_starts=self.starts.ctypes.data, firsts=self.firsts.ctypes.data,
                    tables=self.tables.ctypes.data, mask=fa.MASK_CAUSAL, window=0, workspace=4096,
                    workspace_bytes=1 << 40)
        base.update(over)
        if null:
            base[null] = None
        self.c = fa._PagedBatch(*[base[n] for n, _ in fa._PagedBatch._fields_])


def check(cache=None, host=None):
    host = host or Host()
    cache = cache or cache_c()
    return fa.lib().fa_paged_check(C.byref(cache), C.byref(host.c))


def message():
    return fa.lib().fa_last_error().decode()


def test_a_good_batch_passes():
    assert check() == fa.OK
    assert check(host=Host(starts=(0,), firsts=(), tables=np.zeros((0, 2)))) == fa.OK
    assert check(host=Host(starts=(0, 0, 0))) == fa.OK  # sequences without rows
    assert check(host=Host(starts=(0, 1, 4), rows=9)) == fa.OK  # padding rows behind them
    # a prefix's page in two tables; only the pages that new rows lie in are one sequence's own
    assert check(host=Host(starts=(0, 1, 2), firsts=(17, 20), tables=((3, 4), (3, 9)))) == fa.OK


@pytest.mark.parametrize("over,code", [
    (dict(heads=9), fa.ERR_SHAPE), (dict(kv_heads=0), fa.ERR_ARG), (dict(layers=0), fa.ERR_ARG),
    (dict(pages=0), fa.ERR_ARG), (dict(head_dim=80), fa.ERR_UNSUPPORTED),
    (dict(head_dim=32), fa.ERR_UNSUPPORTED), (dict(page_size=8), fa.ERR_ARG),
    (dict(page_size=48), fa.ERR_ARG), (dict(page_size=8192), fa.ERR_ARG),
    (dict(dtype=fa.F32), fa.ERR_UNSUPPORTED), (dict(dtype=7), fa.ERR_ARG),
    (dict(heads=258, kv_heads=2), fa.ERR_UNSUPPORTED)])
def test_shapes_refused(over, code):
    c = cache_c(**over)
    assert check(cache=c) == code
    n = C.c_uint64()
    assert fa.lib().fa_paged_workspace_bytes(C.byref(c), 4, 1, C.byref(n)) == code
    h = Host()
    assert fa.lib().fa_attend_paged(C.byref(c), 0, C.byref(h.c), 16, 1024, fa.BF16, 16, 1024,
                                    fa.BF16, None) == code


@pytest.mark.parametrize("host,code,say", [
    (dict(firsts=(31, 0)), fa.OK, ""),
    (dict(firsts=(32, 0)), fa.ERR_CAPACITY, "every key the span sees"),
    (dict(firsts=(17, 30)), fa.ERR_CAPACITY, "every key the span sees"),
    (dict(firsts=(2**31 - 1, 0)), fa.ERR_CAPACITY, "every key the span sees"),
    (dict(firsts=(-1, 0)), fa.ERR_ARG, "sequence 0"),
    (dict(starts=(0, 5, 4)), fa.ERR_ARG, "sequence 0"),
    (dict(starts=(-1, 1, 4)), fa.ERR_ARG, "sequence 0"),
    (dict(starts=(0, 3, 2), rows=3), fa.ERR_ARG, "sequence 1"),
    (dict(starts=(0, 1, 4), rows=3), fa.ERR_ARG, "sequence 1"),
    (dict(starts=(0, 1, 4), max_rows=2), fa.ERR_ARG, "sequence 1"),
    (dict(tables=((3, 10), (0, 9))), fa.ERR_ARG, "page 10"),
    (dict(tables=((-1, 4), (0, 9))), fa.ERR_ARG, "page -1"),
    (dict(tables=((3, 4), (-2**31, 9))), fa.ERR_ARG, "sequence 1"),
    (dict(tables=((3, 4), (0, -1))), fa.OK, ""),  # a page that the sequence does not reach
    (dict(starts=(0, 1, 4), firsts=(17, 16), tables=((3, 4), (0, 4))), fa.ERR_ARG, "one slot"),
    (dict(starts=(0, 17, 18), firsts=(0, 0), tables=((4, 4), (0, 9)), max_rows=20), fa.ERR_ARG,
     "one slot")])
def test_numbers_refused(host, code, say):
    assert check(host=Host(**host)) == code
    if code != fa.OK:
        assert say in message()


@pytest.mark.parametrize("over,code", [
    (dict(sequences=-1), fa.ERR_ARG), (dict(rows=-1), fa.ERR_ARG), (dict(max_rows=-1), fa.ERR_ARG),
    (dict(sequences=1025), fa.ERR_ARG), (dict(table_stride=1), fa.ERR_ARG),
    (dict(rows=2**28 + 1), fa.ERR_ARG),
    (dict(null="row_starts"), fa.ERR_ARG), (dict(null="firsts"), fa.ERR_ARG),
    (dict(null="tables"), fa.ERR_ARG)])
def test_batches_refused(over, code):
    h = Host(**over)
    assert check(host=h) == code
    c = cache_c()
    assert fa.lib().fa_attend_paged(C.byref(c), 0, C.byref(h.c), 16, 1024, fa.BF16, 16, 1024,
                                    fa.BF16, None) == code
    r = fa._PagedRows(16, 16, 256, 128, fa.F32)
    assert fa.lib().fa_paged_read(C.byref(c), 0, C.byref(h.c), C.byref(r), None) == code
    assert fa.lib().fa_paged_write(C.byref(c), 0, C.byref(h.c), C.byref(r), None) == code


def attend(cache=None, host=None, layer=0, q=16, q_stride=1024, dtype=fa.BF16, out=16,
           out_stride=1024, out_dtype=fa.BF16):
    cache, host = cache or cache_c(), host or Host()
    return fa.lib().fa_attend_paged(C.byref(cache), layer, C.byref(host.c), q, q_stride, dtype, out,
                                    out_stride, out_dtype, None)


def test_attend_refusals_come_before_any_launch():
    assert fa.lib().fa_attend_paged(None, 0, None, None, 0, 0, None, 0, 0, None) == fa.ERR_ARG
    assert attend(layer=2) == fa.ERR_SHAPE and attend(layer=-1) == fa.ERR_SHAPE
    assert attend(q=None) == fa.ERR_ARG and attend(out=None) == fa.ERR_ARG
    assert attend(q_stride=1023) == fa.ERR_SHAPE and attend(out_stride=1023) == fa.ERR_SHAPE
    assert attend(dtype=fa.Q8) == fa.ERR_ARG and attend(out_dtype=5) == fa.ERR_ARG
    assert attend(q=17) == fa.ERR_ARG and attend(out=18, out_dtype=fa.F32) == fa.ERR_ARG
    assert attend(cache=cache_c(keys=None)) == fa.ERR_ARG
    assert attend(cache=cache_c(keys=4104)) == fa.ERR_ARG
    assert attend(cache=cache_c(key_scales=None)) == fa.ERR_ARG
    assert attend(host=Host(mask=fa.MASK_GROUPS)) == fa.ERR_UNSUPPORTED
    assert attend(host=Host(mask=4)) == fa.ERR_ARG
    assert attend(host=Host(mask=fa.MASK_WINDOW, window=0)) == fa.ERR_ARG


def test_input_refusals_come_before_any_launch():
    lib, c, h = fa.lib(), cache_c(), Host()

    def call(rope=fa.ROPE_HALF, angles=16, qkv=16, stride=1536, dtype=fa.F32, q_out=16,
             q_stride=1024):
        return lib.fa_attention_input_paged(C.byref(c), 0, C.byref(h.c), rope, angles, None, qkv,
                                            stride, dtype, q_out, q_stride, None)

    assert call(rope=3) == fa.ERR_ARG and call(angles=None) == fa.ERR_ARG
    assert call(qkv=None) == fa.ERR_ARG and call(stride=1535) == fa.ERR_SHAPE
    assert call(dtype=fa.Q8) == fa.ERR_ARG and call(q_stride=1000) == fa.ERR_SHAPE
    assert call(qkv=18) == fa.ERR_ARG
    assert lib.fa_attention_paged(C.byref(c), 0, C.byref(h.c), fa.ROPE_HALF, None, None, 16, 1536,
                                  fa.F32, 16, 1024, fa.F32, None) == fa.ERR_ARG
    for rows in (None, fa._PagedRows(None, 16, 256, 128, fa.F32),
                 fa._PagedRows(16, 16, -1, 128, fa.F32), fa._PagedRows(16, 16, 256, 128, 9),
                 fa._PagedRows(18, 16, 256, 128, fa.F32)):
        ref = None if rows is None else C.byref(rows)
        assert lib.fa_paged_read(C.byref(c), 0, C.byref(h.c), ref, None) == fa.ERR_ARG
        assert lib.fa_paged_write(C.byref(c), 0, C.byref(h.c), ref, None) == fa.ERR_ARG


def test_pool_tensors_are_checked():
    import torch

    shape = fa.Shape(1, 4, 2, 64)
    good = torch.zeros((1, 3, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(fa.ShapeError):
        fa.PagedCache(shape, 4, 16, fa.BF16, keys=good, values=good)
    with pytest.raises(fa.ShapeError):
        fa.PagedCache(shape, 3, 16, fa.Q8, keys=good, values=good)
    with pytest.raises(fa.FaError):
        fa.PagedCache(shape, 3, 16, fa.F32, keys=good, values=good)
    flags, _ = fa.capabilities()
    assert flags & 16


def test_row_arrays_are_checked():
    """Rows narrower than the heads need (though their stride may be wide enough), angles of another
    type or width: refused before the library is called."""
    import torch
    shape = fa.Shape(1, 4, 2, 64)
    pages = torch.zeros((1, 3, 2, 16, 64), dtype=torch.bfloat16)
    cache = fa.PagedCache(shape, 3, 16, fa.BF16, keys=pages, values=pages.clone())

    class Batch:
        _ref = None

        def covers(self, *tensors):
            pass

    batch = Batch()
    qkv, q = torch.zeros((2, 512)), torch.zeros((2, 256))
    narrow_qkv, narrow = torch.zeros((2, 600))[:, :511], torch.zeros((2, 600))[:, :255]
    angles = torch.zeros((2, 64))
    bad = [
        lambda: cache.attend(0, batch, narrow, q),
        lambda: cache.attend(0, batch, q, narrow),
        lambda: cache.attend(0, batch, q.view(2, 4, 64), q),
        lambda: cache.attention(0, batch, narrow_qkv, q, angles),
        lambda: cache.attention(0, batch, qkv, narrow, angles),
        lambda: cache.attention(0, batch, qkv, q, angles.bfloat16()),
        lambda: cache.attention(0, batch, qkv, q, angles[:, :32]),
        lambda: cache.attention(0, batch, qkv, q, torch.zeros((2, 128))[:, :64]),
        lambda: cache.attention_input(0, batch, narrow_qkv, angles),
        lambda: cache.attention_input(0, batch, qkv, angles, q_out=narrow),
        lambda: cache.attention_input(0, batch, qkv, angles.double()),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()

"""Calls over the paged cache at the edges of what its interface allows, on the GPU: many pieces to
a warp, handles made on one stream and used on another, numbers out of range, against the formulas in 64 bits. The bounds are those of test_paged_gpu.py.
"""
import pytest

import fusor_attn as fa
from test_paged_gpu import CAUSAL, Spans, angles_of, make_cache, run_attend, torch_

pytestmark = pytest.mark.gpu

DIMS = [(14, 2, 64), (32, 8, 128), (8, 2, 256)]


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("dims", [(16, 8, 64), (16, 8, 128), (16, 8, 256)], ids=str)
@pytest.mark.parametrize("rows", [3, 40], ids=["tokens", "chunks"])
def test_many_short_pieces_of_a_warp(dims, dtype, rows):
    """Sequences of a few tiles each, so that every warp takes many pieces one after the other:
    each with its own sequence, head and pages."""
    torch = torch_()
    spans = Spans([(1 + (i * 7) % rows if rows < 8 else 20 + (i * 7) % rows, (i * 37) % 150)
                   for i in range(250)], 16)
    cache, batch, q, out = run_attend(fa.Shape(1, *dims), spans, dtype, CAUSAL)
    again = torch.empty_like(out)
    for _ in range(5):
        cache.attend(0, batch, q, again)
        assert torch.equal(again, out)
    fa.device_status()


# ---- handles made on one stream, used on another -----------------------------------------------

BUSY = 100_000_000  # cycles: tens of milliseconds


def split_run(dtype):
    """A call whose units are shared among many CTAs (so that its counters count), and its output."""
    spans = Spans([(1, 9000), (1, 4000), (70, 3000)], 64)
    cache, batch, q, out = run_attend(fa.Shape(1, 16, 4, 128), spans, dtype, CAUSAL)
    return spans, cache, batch, q, out


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_batch_made_on_a_busy_stream_is_used_on_another(dtype):
    """The batch's counters are zeroed behind long work of the stream that it is made on (in memory
    that held ones); a call on another stream, not ordered with that one by the caller, sees zeros."""
    torch = torch_()
    spans, cache, batch, q, out = split_run(dtype)
    nbytes = batch.workspace.numel()
    del batch
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    ones = torch.ones(nbytes // 4, dtype=torch.int32, device="cuda")
    side, got = torch.cuda.Stream(), torch.zeros_like(out)
    held = [torch.zeros(1 << 20, device="cuda") for _ in range(2)]  # (what the calls below need)
    torch.cuda.synchronize()
    del ones, held
    torch.cuda._sleep(BUSY)
    batch = spans.batch(cache)
    cache.attend(0, batch, q, got, stream=side)
    side.synchronize()
    assert torch.equal(got, out)
    with torch.cuda.stream(side):  # the current stream, too
        torch.cuda._sleep(BUSY // 10)
        later = spans.batch(cache)
        cache.attend(0, batch, q, got)
    cache.attend(0, later, q, got)
    torch.cuda.synchronize()
    assert torch.equal(got, out)
    fa.device_status()


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_batch_dropped_before_its_call_has_run(dtype):
    """The batch's memory is not handed out while another stream's call may still use it."""
    torch = torch_()
    spans, cache, batch, q, out = split_run(dtype)
    nbytes = batch.workspace.numel()
    side, got = torch.cuda.Stream(), torch.zeros_like(out)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
    cache.attend(0, batch, q, got, stream=side)
    del batch
    other = torch.full((nbytes // 4,), 3, dtype=torch.int32, device="cuda")
    torch.cuda.default_stream().synchronize()
    side.synchronize()
    assert torch.equal(got, out)
    assert (other == 3).all()
    fa.device_status()


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_cache_made_on_a_busy_stream_is_used_on_another(dtype):
    """Rows written on another stream are not zeroed away by the pool's own making; a pool dropped
    before its call has run keeps its memory until then."""
    torch = torch_()
    shape = fa.Shape(1, 8, 2, 128)
    spans = Spans([(50, 0), (1, 300)], 16)
    k = torch.randn((spans.rows, 2, 128), device="cuda").bfloat16()
    v = -k
    back = [torch.zeros((2, *k.shape), device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(BUSY)
    cache = fa.PagedCache(shape, spans.pages, 16, dtype)
    batch = spans.batch(cache)
    cache.write(0, batch, k, v, stream=side)
    torch.cuda.synchronize()
    cache.read(0, batch, back[0][0], back[0][1])
    torch.cuda.synchronize()
    top = k.float().abs().amax(-1, keepdim=True)
    step = top / 254 + 1e-5 * top if dtype == fa.Q8 else 0.0
    assert ((back[0][0] - k.float()).abs() <= step).all()
    assert torch.equal(back[0][1], -back[0][0])
    with torch.cuda.stream(side):
        torch.cuda._sleep(BUSY)
    cache.read(0, batch, back[1][0], back[1][1], stream=side)
    size, kind = cache.keys.shape, cache.keys.dtype
    del cache, batch
    other = [torch.full(size, 5, dtype=kind, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    assert torch.equal(back[1], back[0])
    assert all((t == 5).all() for t in other)
    fa.device_status()


# ---- numbers out of range ----------------------------------------------------------------------

@pytest.mark.parametrize("sp", [[(1, 300), (2, 79), (1, 20)], [(100, 201), (1, 64), (40, 0)]],
                         ids=["tokens", "chunks"])
@pytest.mark.parametrize("dims", DIMS, ids=str)
@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_new_rows_own_page_out_of_range(dims, sp, dtype):
    """attention() where pages of new rows are outside the pool: those rows' own queries attend to
    the positions that are left, whatever the workspace held before, and nothing of them is kept."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans(sp, 16)
    cache = make_cache(shape, spans, dtype)
    # (the call's own queries are kept in f32 over 8-bit pages, in bf16 over bf16 pages)
    kind = torch.float32 if dtype == fa.Q8 else torch.bfloat16
    qkv = torch.randn((spans.rows, shape.qkv), device="cuda").to(kind)
    angles = angles_of(spans, dims[2])
    q = torch.empty((spans.rows, shape.width), device="cuda", dtype=kind)
    cache.attention_input(0, spans.batch(cache), qkv, angles, q_out=q)
    fa.device_status()
    good = spans.tables.clone()
    for seq, page, bad in ((0, sp[0][1] // 16 + (sp[0][0] > 1), -1), (1, sp[1][1] // 16, spans.pages)):
        spans.tables.copy_(good)
        spans.tables[seq, page] = bad
        batch = spans.batch(cache)
        batch.workspace[fa.PAGED_COUNTER_BYTES:] = 0xFF  # NaN, in f32 and in bf16
        held = [t.clone() for t in (cache.keys, cache.values)]
        got_q = torch.full_like(q, 7.0)
        cache.attention_input(0, batch, qkv, angles, q_out=got_q)
        with pytest.raises(fa.FaError) as e:
            fa.device_status()
        assert e.value.code == fa.ERR_ARG
        assert torch.equal(got_q, q)
        out = torch.full((spans.rows, shape.width), 5.0, device="cuda")
        want = torch.full_like(out, 6.0)
        cache.attention(0, batch, qkv, out, angles)
        cache.attend(0, batch, q, want)
        with pytest.raises(fa.FaError):
            fa.device_status()
        assert torch.isfinite(out).all() and torch.equal(out, want)
        page_id = int(good[seq, page])  # the page that the table named before: not written
        for t, old in zip((cache.keys, cache.values), held):
            assert torch.equal(t[0, page_id], old[0, page_id])

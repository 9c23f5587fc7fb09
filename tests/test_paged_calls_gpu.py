"""Calls over the paged cache at the edges of what its interface allows, on the GPU: many pieces to
a warp, handles made on one stream and used on another, numbers out of range, 8-bit
scales far apart, against the formulas in 64 bits. The bounds are those of test_paged_gpu.py.
"""
import math

import pytest

import fusor_attn as fa
from test_paged_gpu import (CAUSAL, Spans, angles_of, check_close, held, make_cache, reference,
                            run_attend, torch_, visible)

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


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_batch_after_a_call_that_gave_up(dtype, monkeypatch):
    """Counters left as they were when a wait gave up (put there by hand, and the status with them):
    once the status has been seen, a batch's next call starts from zeros, on any stream; replays of
    a captured call do after a reset."""
    torch = torch_()
    spans, cache, batch, q, out = split_run(dtype)
    got = torch.zeros_like(out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(0, batch, q, got)

    def give_up():
        torch.cuda.synchronize()
        batch.workspace[:fa.PAGED_COUNTER_BYTES] = 1
        got.zero_()
        with monkeypatch.context() as m:
            m.setattr(fa.lib(), "fa_device_status", lambda stream: fa.ERR_TIMEOUT)
            with pytest.raises(fa.FaError) as e:
                fa.device_status()
        assert e.value.code == fa.ERR_TIMEOUT
        torch.cuda.synchronize()

    for stream in (None, torch.cuda.Stream()):
        give_up()
        cache.attend(0, batch, q, got, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, out)
    give_up()
    batch.reset()
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, out)
    assert (batch.workspace[:fa.PAGED_COUNTER_BYTES] == 0).all()
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


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_no_rows_allowed_to_a_sequence(dtype):
    """max_rows 0: a sequence that has rows all the same is left out and reported, as with any other
    number; sequences without rows are in order."""
    torch = torch_()
    shape = fa.Shape(1, 8, 2, 128)
    spans = Spans([(1, 10), (30, 5)], 16)
    cache = make_cache(shape, spans, dtype)
    qkv = torch.randn((31, shape.qkv), device="cuda")
    pools = [t.clone() for t in (cache.keys, cache.values)]
    for call in ("attend", "attention"):
        out = torch.full((31, shape.width), 5.0, device="cuda")
        batch = spans.batch(cache, max_rows=0)
        getattr(cache, call)(0, batch, qkv, out)
        with pytest.raises(fa.CapacityError):
            fa.device_status()
        assert (out == 5.0).all()
    assert torch.equal(cache.keys, pools[0]) and torch.equal(cache.values, pools[1])
    empty = Spans([(0, 10), (0, 5)], 16, pad_rows=4)
    out = torch.full((4, shape.width), 5.0, device="cuda")
    cache.attend(0, empty.batch(cache, max_rows=0), qkv, out)
    fa.device_status()
    assert (out == 5.0).all()


# ---- 8-bit scales far apart --------------------------------------------------------------------

def eight_bit_reference(cache, spans, q, weighty):
    """Outputs of one sequence's causal rows in f64 and their bounds: test_paged_gpu.py's, with the
    scores' errors D taken over the keys that a row sees, or (weighty) over those that have a weight
    in f64, and two changes. D is not small where a huge key is seen: numerator and sum are within
    e^D of what they are without it, so every p_j is within e^(2 D) of it, and with weights and
    values off by w an output by at most ((1 + w) e^(2 D) - 1) x sum_j p_j |v_j| (a row whose D is
    large may give a huge key all of its weight or none: its bound says nothing). The weights go into
    the products in f16, where those below 2^-14 are off by at most 2^-25. The token kernel's weights carry their value's scale s_j and the largest is at
    least 2^6: each is off by at most 2^-31 of the largest p_j s_j. The chunk kernel's go with values
    whose scales are put into [2^8, 2^9), the largest of a tile (which here lie within 2^2 of each
    other, or have units of their own) or each its own: the largest weight is at least 2^7 and its
    scale at least 2^6, and 2^-25 with a scale of at most 2^9 is 2^-29 of the largest p_j s_j. An
    element of at most 127 steps is so off by at most 127 x 2^-29 of it for every position."""
    torch = torch_()
    (rows, first), = spans.spans
    end = first + rows
    heads, kvh, d = cache.shape.heads, cache.shape.kv_heads, cache.shape.head_dim
    k, v = held(cache, 0, *spans.places(0, 0, end))
    page, slot = spans.places(0, 0, end)
    scales = cache.value_scales[0][page, :, slot].double()
    see = visible(CAUSAL, torch.arange(first, end, device="cuda"), end)
    want = torch.zeros((rows, heads * d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(want)
    for h in range(heads):
        cols, kv = slice(h * d, (h + 1) * d), h * kvh // heads
        qh, kh, vh = q[:, cols].double(), k[:, kv], v[:, kv]
        p = torch.softmax(torch.where(see, qh @ kh.T / math.sqrt(d), -math.inf), 1)
        off = (3 * 2.0 ** -11 + 1e-5) * (qh.abs() @ kh.abs().T) + 2.0 ** -14.9 * (
            qh.abs().amax(1, keepdim=True) @ kh.abs().sum(1)[None])
        off = torch.where(p > 0 if weighty else see, off / math.sqrt(d), 0.0).amax(1, keepdim=True)
        want[:, cols] = p @ vh
        tol[:, cols] = ((1 + 3 * 2.0 ** -11 + 1e-4) * torch.exp(2 * off.clamp(max=100)) - 1) * (p @ vh.abs())
        tol[:, cols][off.squeeze(1) > 100] = math.inf  # (e^200 of what p has lost below 1e-308, too)
        tol[:, cols] += end * 127 * 2.0 ** -29 * (p * scales[:, kv]).amax(1, keepdim=True)
    return want, tol


@pytest.mark.parametrize("rows", [2, 60], ids=["token", "chunk"])
@pytest.mark.parametrize("dims", DIMS, ids=str)
@pytest.mark.parametrize("what", ["keys", "values", "both"])
@pytest.mark.parametrize("power", [26, 35])
def test_a_scale_far_above_its_neighbours(dims, rows, what, power):
    """One new position's keys or values 2^26 or 2^35 times its neighbours': the rows before it are
    as precise as without it, whatever tile it shares with their keys."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans([(rows, 90)], 16)
    cache = make_cache(shape, spans, fa.Q8)
    page, slot = spans.places(0, 90 + rows // 2, 91 + rows // 2)
    if what != "values":
        cache.key_scales[0, page, :, slot] *= 2.0 ** power
    if what != "keys":
        cache.value_scales[0, page, :, slot] *= 2.0 ** power
    q = torch.randn((rows, shape.width), device="cuda").bfloat16()
    out = torch.empty((rows, shape.width), device="cuda")
    cache.attend(0, spans.batch(cache), q, out)
    fa.device_status()
    check_close(out, *eight_bit_reference(cache, spans, q, False), False)


@pytest.mark.parametrize("rows", [2, 60], ids=["token", "chunk"])
@pytest.mark.parametrize("dims", DIMS, ids=str)
@pytest.mark.parametrize("at", [0, 37, 91], ids=str)
@pytest.mark.parametrize("power", [9, 26, 35, 60])
def test_a_huge_position_that_no_row_gives_weight(dims, rows, at, power):
    """A position whose keys and values are far above the others' and whose scores lie far below
    them (in 64 bits its weights are exactly zero): every row is what the others make it."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans([(rows, 90)], 16)
    cache = make_cache(shape, spans, fa.Q8)
    page, slot = spans.places(0, at, at + 1)
    cache.keys[0, page, :, slot] = -127  # (queries are positive)
    cache.key_scales[0, page, :, slot] = 2.0 ** power
    cache.value_scales[0, page, :, slot] = 2.0 ** power
    q = torch.rand((rows, shape.width), device="cuda") + 0.5
    out = torch.empty((rows, shape.width), device="cuda")
    cache.attend(0, spans.batch(cache), q, out)
    fa.device_status()
    check_close(out, *eight_bit_reference(cache, spans, q, True), False)


@pytest.mark.parametrize("rows,first", [(2, 3000), (170, 3000), (700, 0)])
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_scales_of_any_size_side_by_side(dims, rows, first):
    """Every position's scales a power of two of their own, over many tiles and shared among CTAs."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans([(rows, first)], 64)
    cache = make_cache(shape, spans, fa.Q8)
    g = torch.Generator(device="cuda").manual_seed(3)
    for t, lo, hi in ((cache.key_scales, -25, 1), (cache.value_scales, -25, 25)):
        t *= 2.0 ** torch.randint(lo, hi, t.shape, generator=g, device="cuda")
    q = torch.randn((rows, shape.width), generator=g, device="cuda").bfloat16()
    out = torch.empty((rows, shape.width), device="cuda")
    batch = spans.batch(cache)
    cache.attend(0, batch, q, out)
    check_close(out, *eight_bit_reference(cache, spans, q, False), False)
    again = torch.empty_like(out)
    cache.attend(0, batch, q, again)
    fa.device_status()
    assert torch.equal(out, again)


@pytest.mark.parametrize("rows", [1, 60], ids=["token", "chunk"])
@pytest.mark.parametrize("dims", DIMS, ids=str)
def test_heads_of_zeros_beside_tiny_values(dims, rows):
    """Blocks of positions whose values are all zero weigh in the sums of rows whose other values are
    tiny, and take nothing from them."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans([(rows, 500)], 16)
    cache = make_cache(shape, spans, fa.Q8)
    cache.value_scales *= 2.0 ** -30
    page, slot = spans.places(0, 128, 256)
    cache.values[0, page, :, slot] = 0
    cache.value_scales[0, page, :, slot] = 0
    q = torch.randn((rows, shape.width), device="cuda").bfloat16()
    out = torch.empty((rows, shape.width), device="cuda")
    cache.attend(0, spans.batch(cache), q, out)
    fa.device_status()
    want, tol = reference(cache, 0, spans, q.double(), CAUSAL)
    up = 2.0 ** 30  # (values are off by at most 2^-58 besides)
    check_close(out.double() * up, want * up, tol * up + 2.0 ** -58 * up, False)


# ---- layouts of rows ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_rows_read_into_one_array_of_keys_and_values(dtype):
    """Keys and values side by side in each row of one array; one array for both holds the values;
    rows that share elements are refused."""
    torch = torch_()
    spans = Spans([(30, 5), (1, 40)], 16)
    cache = make_cache(fa.Shape(1, 8, 4, 128), spans, dtype)
    batch = spans.batch(cache)
    apart = torch.empty((2, spans.rows, 4, 128), device="cuda")
    cache.read(0, batch, apart[0], apart[1])
    both = torch.empty((spans.rows, 2, 4, 128), device="cuda")
    cache.read(0, batch, both[:, 0], both[:, 1])
    one = torch.empty((spans.rows, 4, 128), device="cuda")
    cache.read(0, batch, one, one)
    fa.device_status()
    assert torch.equal(both.transpose(0, 1), apart) and torch.equal(one, apart[1])
    for k, v in ((one[:, :1].expand(-1, 4, -1), apart[1][:, :1].expand(-1, 4, -1)),
                 (one[:1].expand(spans.rows, -1, -1), apart[1][:1].expand(spans.rows, -1, -1)),
                 (both[:-1].flatten(0, 1)[:spans.rows], both.flatten(0, 1)[1:1 + spans.rows])):
        with pytest.raises(fa.FaError) as e:
            cache.read(0, batch, k, v)
        assert e.value.code == fa.ERR_ARG
    cache.write(0, batch, apart[0][:1].expand(spans.rows, -1, -1), apart[1][:1].expand(spans.rows, -1, -1))
    fa.device_status()

"""The paged cache on the GPU: rows written into 8-bit and bf16 pages and read back, and the
attention of single tokens, few rows and chunks over them, against the formulas in 64 bits.

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value (half a step), to f16 by 2^-11.
- A row read back as bf16 is off by the page's rounding (bf16: 2^-8 of the value; 8 bits: half a
  scale, max|x| / 254) and its own 2^-8; in f32 by the page's alone, plus the f32 arithmetic
  (RoPE, norm: a few 2^-23 of the head's largest element).
- An attention output sum_j p_j v_j. Over bf16 pages each weight is rounded once to bf16 (2^-8 of
  it) and a query that is not bf16 is, so that a score is off by at most D = 2^-8 x sum_e |q_e k_e|
  / sqrt(d). Over 8-bit pages weights, keys and values are f16 at worst (2^-11 each; a key or value
  is rounded twice, with its scale), and a query is f16 or held in steps of 2^-14 of its largest
  element (half a step 2^-15, 16256 steps for 2^14): D = 3 x 2^-11 x sum_e |q_e k_e| / sqrt(d) +
  2^-14.9 max|q| sum_e |k_e| / sqrt(d), weights and values 3 x 2^-11. D changes every p_j by at
  most 2 D of it (numerator and sum), so an output is off by at most (weights + 2 D) x sum_j p_j
  |v_j|, and by 2^-8 of itself when it is rounded to bf16 at the end. The products' f32 sums and the
  approximate exponentials add under 1e-4 of the same quantities.
"""
import math

import pytest

import fusor_attn as fa

pytestmark = pytest.mark.gpu

HALF16 = 2.0 ** -8


def torch_():
    import torch
    return torch


class Spans:
    """A batch's numbers: (rows, first) per sequence, tables over a pool in random order."""

    def __init__(self, spans, page_size, spare=5, seed=0, pad_rows=0, width=None):
        torch = torch_()
        self.spans, self.ps = spans, page_size
        g = torch.Generator().manual_seed(seed)
        need = [-(-(r + f) // page_size) for r, f in spans]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g, dtype=torch.int64).to(torch.int32)
        wide = max([1] + need) if width is None else width
        tables = torch.full((len(spans), wide), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            tables[i, :n] = order[at:at + n]
            at += n
        starts = [0]
        for r, _ in spans:
            starts.append(starts[-1] + r)
        self.real_rows = starts[-1]
        self.rows = starts[-1] + pad_rows
        self.max_rows = max([r for r, _ in spans] + [0])
        self.starts = starts
        self.tables_host = tables
        self.row_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.firsts = torch.tensor([f for _, f in spans], dtype=torch.int32, device="cuda")
        self.tables = tables.cuda()

    def batch(self, cache, mask=fa.Mask.causal(), max_rows=None):
        return fa.PagedBatch(cache, self.row_starts, self.firsts, self.tables, self.rows,
                             self.max_rows if max_rows is None else max_rows, mask)

    def places(self, i, lo, hi):
        """(page, slot) of sequence i's positions lo..hi."""
        torch = torch_()
        p = torch.arange(lo, hi)
        return self.tables_host[i][p // self.ps].long().cuda(), (p % self.ps).cuda()


def make_cache(shape, spans, dtype, seed=1, fill="normal"):
    """A cache whose every slot holds values (also the unused ones)."""
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = fa.PagedCache(shape, spans.pages, spans.ps, dtype)
    if dtype == fa.Q8:
        for t, s in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
            t.copy_((40 * torch.randn(t.shape, generator=g, device="cuda")).round().clamp(-127, 127))
            s.copy_((0.5 + torch.rand(s.shape, generator=g, device="cuda")) / 40)
    else:
        for t in (cache.keys, cache.values):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    return cache


def held(cache, layer, page, slot):
    """f64 keys and values of the places (positions, kv_heads, head_dim)."""
    out = []
    for t, s in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        x = t[layer][page, :, slot].double()
        out.append(x if s is None else x * s[layer][page, :, slot].double()[..., None])
    return out


def visible(mask, at, end):
    torch = torch_()
    pos = torch.arange(end, device="cuda")
    if mask.kind == fa.MASK_FULL:
        return torch.ones((len(at), end), dtype=torch.bool, device="cuda")
    see = pos[None] <= at[:, None]
    if mask.kind == fa.MASK_WINDOW:
        see &= pos[None] > at[:, None] - mask.window
    return see


def reference(cache, layer, spans, q, mask, q_bits=0.0):
    """Outputs in f64, and the bound of an f32 output's error (see above). q: f64 rows; q_bits: how
    far the rounding of q to bf16 may be off, relative."""
    torch = torch_()
    eight = cache.dtype == fa.Q8
    q_bits, weights, step = (q_bits + 3 * 2.0 ** -11, 3 * 2.0 ** -11, 2.0 ** -14.9) if eight else (
        q_bits, HALF16, 0.0)
    s = cache.shape
    d, group = s.head_dim, s.heads // s.kv_heads
    out = torch.zeros((spans.rows, s.heads * d), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for i, (rows, first) in enumerate(spans.spans):
        if rows == 0:
            continue
        end = first + rows
        k, v = held(cache, layer, *spans.places(i, 0, end))
        see = visible(mask, torch.arange(first, end, device="cuda"), end)
        r = slice(spans.starts[i], spans.starts[i] + rows)
        for h in range(s.heads):
            qh = q[r, h * d:(h + 1) * d]
            kh, vh = k[:, h // group], v[:, h // group]
            scores = qh @ kh.T / math.sqrt(d)
            # masked keys and values may be anything
            p = torch.softmax(torch.where(see, scores, -math.inf), 1)
            vz = torch.where(see.any(0)[:, None], vh, 0.0)
            out[r, h * d:(h + 1) * d] = p @ vz
            off = qh.abs() @ kh.abs().T / math.sqrt(d)
            off = (q_bits + 1e-5) * torch.where(see, off, 0.0).amax(1, keepdim=True)
            steps = qh.abs().amax(1, keepdim=True) @ kh.abs().sum(1)[None] / math.sqrt(d)
            off = off + step * torch.where(see, steps, 0.0).amax(1, keepdim=True)
            tol[r, h * d:(h + 1) * d] = (weights + 2 * off + 1e-4) * (p @ vz.abs())
    return out, tol


def check_close(got, want, tol, bf16):
    torch = torch_()
    got = got.double()
    assert torch.isfinite(got).all()
    tol = tol + 1e-6 + (HALF16 * (want.abs() + tol) if bf16 else 0.0)
    worst = ((got - want).abs() / tol).max().item() if got.numel() else 0.0
    rel = ((got - want).norm() / want.norm().clamp(min=1e-30)).item()
    print(f"worst {worst:.3f} of the bound, relative L2 {rel:.2e}")
    assert worst <= 1.0


# ---- writes and reads --------------------------------------------------------------------------

def rotate(x, angles, rope):
    torch = torch_()
    if rope == fa.ROPE_NONE:
        return x
    d = x.shape[-1]
    c, s = angles[:, None, :d // 2].double(), angles[:, None, d // 2:].double()
    if rope == fa.ROPE_HALF:
        a, b = x[..., :d // 2], x[..., d // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, b * c + a * s], -1).reshape(x.shape)


def angles_of(spans, d):
    torch = torch_()
    pos = [p for r, f in spans.spans for p in range(f, f + r)] + [0] * (spans.rows - spans.real_rows)
    return torch.from_numpy(fa.rotary_angles(fa.Rotation(base=1e6), d, pos)).cuda()


WRITE_CASES = [
    # heads, kv_heads, d, pages, rows dtype, rope, norm, page_size, spans, padding rows
    (4, 2, 64, fa.Q8, "f32", fa.ROPE_HALF, False, 16, [(1, 0), (3, 14), (0, 9), (40, 5)], 3),
    (4, 2, 64, fa.BF16, "bf16", fa.ROPE_INTERLEAVED, True, 32, [(33, 31), (1, 64)], 0),
    (14, 2, 64, fa.Q8, "bf16", fa.ROPE_HALF, False, 16, [(1, 299), (1, 16), (1, 15)], 2),
    (32, 8, 128, fa.Q8, "bf16", fa.ROPE_HALF, False, 64, [(130, 100)], 0),
    (8, 8, 128, fa.Q8, "f32", fa.ROPE_INTERLEAVED, True, 16, [(5, 3), (2, 130000)], 1),
    (8, 1, 128, fa.BF16, "f32", fa.ROPE_HALF, True, 128, [(17, 120)], 0),
    (8, 2, 256, fa.Q8, "f32", fa.ROPE_NONE, True, 16, [(9, 9)], 0),
    (8, 2, 256, fa.BF16, "bf16", fa.ROPE_HALF, False, 16, [(20, 0), (1, 31)], 0),
    (2, 2, 256, fa.Q8, "bf16", fa.ROPE_INTERLEAVED, False, 4096, [(3, 4094)], 0),
]


@pytest.mark.parametrize("case", WRITE_CASES, ids=[str(i) for i in range(len(WRITE_CASES))])
@pytest.mark.parametrize("odd", [False, True], ids=["aligned", "odd"])
def test_rows_written_and_read_back(case, odd):
    torch = torch_()
    heads, kvh, d, dtype, kind, rope, norm, ps, sp, pad = case
    shape = fa.Shape(2, heads, kvh, d)
    spans = Spans(sp, ps, pad_rows=pad)
    cache = make_cache(shape, spans, dtype)
    before = [t.clone() for t in (cache.keys, cache.values)]
    tdt = torch.float32 if kind == "f32" else torch.bfloat16
    g = torch.Generator(device="cuda").manual_seed(3)
    width = (heads + 2 * kvh) * d
    # odd: rows at an odd element offset and stride, so that no vector load is aligned
    flat = torch.randn((spans.rows, width + (3 if odd else 0)), generator=g, device="cuda").to(tdt)
    qkv = flat[:, 1:1 + width] if odd else flat
    angles = angles_of(spans, d) if rope != fa.ROPE_NONE else None
    weights = None
    if norm:
        weights = tuple(1 + 0.2 * torch.randn(d, generator=g, device="cuda") for _ in range(2))
    q = torch.full((spans.rows, heads * d + (5 if odd else 0)), 7.0, device="cuda", dtype=tdt)
    batch = spans.batch(cache)
    batch.check()
    cache.attention_input(1, batch, qkv, angles, rope, (*weights, 1e-6) if norm else None,
                          q[:, :heads * d])
    fa.device_status()

    x = qkv.double().reshape(spans.rows, -1, d)
    qk, v = x[:, :heads + kvh], x[:, heads + kvh:]
    if norm:
        w = torch.cat([weights[0].expand(heads, d), weights[1].expand(kvh, d)]).double()
        qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    qk = rotate(qk, angles, rope)
    real = spans.real_rows
    got = q[:real, :heads * d].double().reshape(real, heads, d)
    want = qk[:real, :heads]
    # f32: the norm's sum and two roundings, the rotation's three, of the head's largest elements
    fine = 1e-5 * want.abs().amax(-1, keepdim=True)
    tol = fine + (HALF16 * want.abs() if kind == "bf16" else 0)
    assert ((got - want).abs() <= tol).all()
    assert (q[real:] == 7.0).all() and (q[:, heads * d:] == 7.0).all()

    for out_dt in (torch.float32, torch.bfloat16):
        base = torch.full((2, spans.rows, kvh, d + (1 if odd else 0)), 9.0, device="cuda", dtype=out_dt)
        keys, values = base[0, ..., :d], base[1, ..., :d]
        cache.read(1, batch, keys, values)
        for got, want in ((keys, qk[:, heads:]), (values, v)):
            assert (got[real:] == 9.0).all()
            got, want = got[:real].double(), want[:real]
            top = want.abs().amax(-1, keepdim=True)
            tol = 1e-5 * top + (top / 254 if dtype == fa.Q8 else HALF16 * want.abs())
            if out_dt == torch.bfloat16:
                tol = tol + HALF16 * (want.abs() + tol)
            assert ((got - want).abs() <= tol).all()
    fa.device_status()
    # nothing else changed: the other layer, and every slot that no row lies in
    written = torch.zeros((spans.pages, ps), dtype=torch.bool, device="cuda")
    for i, (rows, first) in enumerate(sp):
        if rows:
            written[spans.places(i, first, first + rows)] = True
    for t, old in zip((cache.keys, cache.values), before):
        assert torch.equal(t[0], old[0])
        same = (t[1] == old[1]).all(-1).permute(0, 2, 1)  # page, slot, head
        assert same[~written].all()


def test_eight_bit_rows_at_the_edges():
    """Zeros, tiny heads, a head of one value, an infinity and a NaN."""
    torch = torch_()
    shape = fa.Shape(1, 1, 1, 64)
    spans = Spans([(7, 10)], 16)
    cache = fa.PagedCache(shape, spans.pages, 16, fa.Q8)
    x = torch.zeros((7, 1, 64), device="cuda")
    x[1] = 1e-38
    x[2, 0, 5] = -3.25
    x[3] = torch.linspace(-1, 1, 64)
    x[4] = 3e38
    x[5, 0, 7] = math.inf
    x[6, 0, 9] = math.nan
    batch = spans.batch(cache)
    cache.write(0, batch, x, -x)
    k, v = torch.empty_like(x), torch.empty_like(x)
    cache.read(0, batch, k, v)
    fa.device_status()
    assert (k[:2] == 0).all() and (v[:2] == 0).all()
    top = x[2:5].abs().amax(-1, keepdim=True)
    assert ((k[2:5] - x[2:5]).abs() <= top * (1 / 254 + 1e-6)).all()
    assert torch.equal(k[2:5], -v[2:5])
    assert k[2, 0, 5].item() == pytest.approx(-3.25, rel=1e-6) and (k[2, 0, :5] == 0).all()
    assert torch.isnan(k[5:]).all() and torch.isnan(v[5:]).all()


def test_a_contiguous_caches_block_goes_into_pages_and_back():
    """The rows of a KvCache layer ([kv_head][slot][head_dim]) written into pages through their
    strides, and read back into another one's block."""
    torch = torch_()
    shape = fa.Shape(1, 4, 2, 128)
    rows, capacity = 75, 90
    spans = Spans([(rows, 0)], 32)
    cache = fa.PagedCache(shape, spans.pages, 32, fa.BF16)
    k = torch.randn((2, capacity, 128), device="cuda").bfloat16()
    v = torch.randn((2, capacity, 128), device="cuda").bfloat16()
    batch = spans.batch(cache)
    cache.write(0, batch, k.transpose(0, 1)[:rows], v.transpose(0, 1)[:rows])
    back = fa.KvCache(shape, capacity, fa.BF16)
    ko = torch.zeros((2, capacity, 128), device="cuda", dtype=torch.bfloat16)
    vo = torch.zeros_like(ko)
    cache.read(0, batch, ko.transpose(0, 1)[:rows], vo.transpose(0, 1)[:rows])
    back.put_rows(ko[None], vo[None])
    kb, vb = back.copy_rows(rows)
    assert torch.equal(kb[0], k[:, :rows]) and torch.equal(vb[0], v[:, :rows])
    fa.device_status()


# ---- attention ---------------------------------------------------------------------------------

def run_attend(shape, spans, dtype, mask, rows_dt="bf16", out_dt="bf16", layer=0, seed=5, cache=None,
               max_rows=None):
    torch = torch_()
    cache = make_cache(shape, spans, dtype, seed) if cache is None else cache
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}
    q = (1.3 * torch.randn((spans.rows, shape.width), generator=g, device="cuda")).to(dt[rows_dt])
    out = torch.full((spans.rows, shape.width), 5.0, dtype=dt[out_dt], device="cuda")
    batch = spans.batch(cache, mask, max_rows)
    cache.attend(layer, batch, q, out)
    fa.device_status()
    bits = HALF16 if rows_dt == "f32" and dtype == fa.BF16 else 0.0
    want, tol = reference(cache, layer, spans, q.double(), mask, bits)
    n = spans.real_rows
    check_close(out[:n], want[:n], tol[:n], out_dt == "bf16")
    assert (out[n:] == 5.0).all()
    return cache, batch, q, out


CAUSAL, FULL = fa.Mask.causal(), fa.Mask.full()
SHAPES = [(14, 2, 64), (4, 4, 64), (32, 8, 128), (16, 1, 128), (12, 12, 128), (8, 2, 256),
          (16, 2, 256)]


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("dims", SHAPES, ids=str)
@pytest.mark.parametrize("page_size", [16, 64])
def test_single_tokens(dims, dtype, page_size):
    """Lengths of one to many tiles, around the tile's and the page's ends."""
    shape = fa.Shape(1, *dims)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000, 2049, 0]
    spans = Spans([(1 if n else 0, max(n - 1, 0)) for n in lengths], page_size, pad_rows=2)
    run_attend(shape, spans, dtype, CAUSAL)


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("rows_dt,out_dt", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
def test_single_tokens_row_types(dims, dtype, rows_dt, out_dt):
    spans = Spans([(1, 700), (1, 33)], 16)
    run_attend(fa.Shape(1, *dims), spans, dtype, CAUSAL, rows_dt, out_dt)


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("mask", [CAUSAL, FULL, fa.Mask.window_of(1), fa.Mask.window_of(50),
                                  fa.Mask.window_of(1000)], ids=str)
@pytest.mark.parametrize("dims,rows", [((14, 2, 64), 2), ((32, 8, 128), 4), ((12, 12, 128), 13),
                                       ((16, 2, 256), 2), ((32, 8, 128), 2)], ids=str)
def test_few_rows_under_every_mask(dims, rows, mask, dtype):
    spans = Spans([(rows, 0), (rows, 61), (1, 200), (rows, 777), (rows - 1, 128)], 16)
    run_attend(fa.Shape(1, *dims), spans, dtype, mask)


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_one_long_sequence_is_split_over_the_gpu(dtype):
    spans = Spans([(1, 70000)], 64)
    cache, batch, q, out = run_attend(fa.Shape(2, 16, 8, 128), spans, dtype, CAUSAL, layer=1)
    torch = torch_()
    again = torch.empty_like(out)
    for _ in range(3):  # the merge's order does not depend on who arrives last
        cache.attend(1, batch, q, again)
        assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_many_sequences(dtype):
    """As many as a batch may hold, more than there are CTAs, of a few tiles each."""
    spans = Spans([(1, (37 * i) % 200) for i in range(1024)], 16)
    run_attend(fa.Shape(1, 4, 2, 64), spans, dtype, CAUSAL)


CHUNKS = [
    # dims, spans (rows, first), mask
    ((32, 8, 128), [(300, 0)], CAUSAL),
    ((32, 8, 128), [(129, 1000)], CAUSAL),
    ((32, 8, 128), [(17, 0), (5, 40), (257, 511), (0, 3), (64, 64)], CAUSAL),
    ((12, 12, 128), [(17, 3), (500, 100)], CAUSAL),
    ((14, 2, 64), [(37, 0), (200, 450), (18, 130)], CAUSAL),
    ((4, 4, 64), [(700, 0)], CAUSAL),
    ((8, 2, 256), [(100, 0), (33, 700)], CAUSAL),
    ((16, 2, 256), [(65, 900)], CAUSAL),
    ((48, 2, 128), [(1, 300), (40, 0)], CAUSAL),
    ((128, 1, 64), [(3, 200), (1, 0)], CAUSAL),
    ((32, 8, 128), [(200, 300), (90, 0)], FULL),
    ((14, 2, 64), [(150, 33)], FULL),
    ((32, 8, 128), [(333, 1000), (40, 10)], fa.Mask.window_of(100)),
    ((14, 2, 64), [(333, 1000), (40, 10)], fa.Mask.window_of(1)),
    ((8, 2, 256), [(150, 400)], fa.Mask.window_of(64)),
    ((32, 8, 128), [(1, 900), (1, 30), (150, 300), (2, 64), (1, 0)], CAUSAL),
]


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("case", CHUNKS, ids=[f"{c[0]}-{i}" for i, c in enumerate(CHUNKS)])
def test_chunks(case, dtype):
    dims, sp, mask = case
    spans = Spans(sp, 16 if len(sp) > 1 else 128, pad_rows=len(sp) % 2)
    run_attend(fa.Shape(1, *dims), spans, dtype, mask)


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("rows_dt,out_dt", [("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
def test_chunks_row_types(dims, dtype, rows_dt, out_dt):
    spans = Spans([(70, 230), (45, 0)], 32)
    run_attend(fa.Shape(1, *dims), spans, dtype, CAUSAL, rows_dt, out_dt)


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_chunk_over_a_long_context(dtype):
    spans = Spans([(600, 9000)], 64)
    cache, batch, q, out = run_attend(fa.Shape(2, 16, 4, 128), spans, dtype, CAUSAL, layer=1)
    torch = torch_()
    again = torch.empty_like(out)
    for _ in range(3):
        cache.attend(1, batch, q, again)
        assert torch.equal(again, out)


# ---- what costs such kernels -------------------------------------------------------------------

BOTH = [[(1, 300), (3, 70)], [(100, 201), (40, 0)]]


@pytest.mark.parametrize("sp", BOTH, ids=["tokens", "chunks"])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
@pytest.mark.parametrize("mask", [CAUSAL, fa.Mask.window_of(40)], ids=str)
@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_what_no_row_sees_reaches_no_row(dims, sp, dtype, mask):
    """NaN and infinity in every slot that no row of the batch sees: spare pages, the stale end of
    last pages, the positions before the window."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans(sp, 32)
    cache = make_cache(shape, spans, dtype)
    seen = torch.zeros((spans.pages, 32), dtype=torch.bool, device="cuda")
    for i, (rows, first) in enumerate(sp):
        lo = max(0, first + 1 - mask.window) if mask.kind == fa.MASK_WINDOW else 0
        seen[spans.places(i, lo, first + rows)] = True
    hidden = (~seen)[None, :, None].expand(cache.keys.shape[:-1])
    if dtype == fa.Q8:
        cache.key_scales[hidden] = math.nan
        cache.value_scales[hidden] = math.inf
    else:
        cache.keys[hidden] = math.nan
        cache.values[hidden] = math.inf
    run_attend(shape, spans, dtype, mask, cache=cache)


@pytest.mark.parametrize("rows,first", [(3, 70), (3, 0), (100, 201), (60, 0)])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (16, 2, 256)], ids=str)
@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_a_bad_value_reaches_only_the_rows_that_see_it(dims, rows, first, dtype):
    """The last new position's values are not finite: the rows before it are as without it, the
    rows that see it are not finite."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    if dims[0] // dims[1] > 5 and rows == 3:
        rows = 2
    spans = Spans([(rows, first)], 16)
    cache = make_cache(shape, spans, dtype)
    _, batch, q, out = run_attend(shape, spans, dtype, CAUSAL, cache=cache)
    for bad_row in (rows - 1, rows // 2):
        page, slot = spans.places(0, first + bad_row, first + bad_row + 1)
        pool = cache.value_scales if dtype == fa.Q8 else cache.values
        kept = pool[0, page, :, slot].clone()
        pool[0, page, :, slot] = math.nan if bad_row % 2 else math.inf
        again = torch.empty_like(out)
        cache.attend(0, batch, q, again)
        fa.device_status()
        pool[0, page, :, slot] = kept
        assert torch.equal(again[:bad_row], out[:bad_row])
        assert not torch.isfinite(again[bad_row:]).any()


def test_scores_of_any_size():
    """Queries far outside f16's range over 8-bit pages, and a key with a huge scale."""
    torch = torch_()
    shape = fa.Shape(1, 4, 2, 64)
    spans = Spans([(1, 200)], 16)
    cache = make_cache(shape, spans, fa.Q8)
    batch = spans.batch(cache)
    for size in (1e30, 1e-30):
        q = torch.randn((1, 256), device="cuda") * size
        cache.key_scales.copy_(torch.rand_like(cache.key_scales) / (40 * size))
        out = torch.empty((1, 256), device="cuda")
        cache.attend(0, batch, q, out)
        want, tol = reference(cache, 0, spans, q.double(), CAUSAL)
        check_close(out, want, tol, False)
    fa.device_status()


@pytest.mark.parametrize("size", [1e30, 1e-30])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
def test_chunk_scores_of_any_size(dims, size):
    """The same over chunks, at every head_dim."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans([(70, 130)], 16)
    cache = make_cache(shape, spans, fa.Q8)
    cache.key_scales.copy_(torch.rand_like(cache.key_scales) / (40 * size))
    q = torch.randn((spans.rows, shape.width), device="cuda") * size
    out = torch.empty((spans.rows, shape.width), device="cuda")
    cache.attend(0, spans.batch(cache), q, out)
    fa.device_status()
    check_close(out, *reference(cache, 0, spans, q.double(), CAUSAL), False)


@pytest.mark.parametrize("sp", BOTH, ids=["tokens", "chunks"])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
@pytest.mark.parametrize("mask", [CAUSAL, fa.Mask.window_of(40)], ids=str)
@pytest.mark.parametrize("small", [2.0 ** -14, 2.0 ** -60], ids=["2^-14", "2^-60"])
def test_queries_of_zeros_over_small_keys(dims, sp, mask, small):
    """A row whose query is zero (a padded one) weighs its keys alike, however small they are."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans(sp, 16)
    cache = make_cache(shape, spans, fa.Q8)
    cache.key_scales *= small
    q = torch.randn((spans.rows, shape.width), device="cuda").bfloat16()
    q[::2] = 0
    q[1::4] *= 2.0 ** -100
    out = torch.empty((spans.rows, shape.width), device="cuda")
    cache.attend(0, spans.batch(cache, mask), q, out)
    fa.device_status()
    check_close(out, *reference(cache, 0, spans, q.double(), mask), False)


@pytest.mark.parametrize("sp", BOTH, ids=["tokens", "chunks"])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
@pytest.mark.parametrize("sizes", [(60, -80), (-80, 60), (-40, -40), (-20, 20)], ids=str)
def test_values_of_any_size(dims, sp, sizes):
    """Blocks of positions whose values differ by many powers of two: the weights of the small
    ones count in the sum all the same."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans(sp, 16)
    cache = make_cache(shape, spans, fa.Q8)
    for i, (rows, first) in enumerate(spans.spans):
        for lo in range(0, first + rows, 128):
            page, slot = spans.places(i, lo, min(lo + 128, first + rows))
            cache.value_scales[0, page, :, slot] *= 2.0 ** sizes[lo // 128 % 2]
    q = torch.randn((spans.rows, shape.width), device="cuda").bfloat16()
    out = torch.empty((spans.rows, shape.width), device="cuda")
    cache.attend(0, spans.batch(cache), q, out)
    fa.device_status()
    want, tol = reference(cache, 0, spans, q.double(), CAUSAL)
    up = 2.0 ** -max(sizes)
    # (values are off by at most 2^-58 besides)
    check_close(out.double() * up, want * up, tol * up + 2.0 ** -58 * up, False)


@pytest.mark.parametrize("rows", [2, 60])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
def test_huge_heads_leave_the_others_their_precision(dims, rows):
    """One position's keys and values a million times its neighbours' over 8-bit pages: the rows
    before it are as precise as ever, and so are the rows that give it no weight."""
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans([(rows, 90)], 16)
    cache = make_cache(shape, spans, fa.Q8)
    page, slot = spans.places(0, 91, 92)
    cache.value_scales[0, page, :, slot] *= 1e6
    run_attend(shape, spans, fa.Q8, fa.Mask.causal(), cache=cache)
    cache.key_scales[0, page, :, slot] *= 1e6  # each row gives it all of its weight, or none
    q = torch.randn((spans.rows, shape.width), device="cuda").bfloat16()
    out = torch.empty_like(q)
    cache.attend(0, spans.batch(cache), q, out)
    want, tol = reference(cache, 0, spans, q.double(), fa.Mask.causal())
    # Rows that give the huge key no weight: its score is off by at most 3 x 2^-11 x sum_e |q_e k_e|
    # / sqrt(d) + 2^-14.9 max|q| sum_e |k_e| / sqrt(d) (D above; with sums of 1e6 x 40 terms of
    # about 1 that is thousands), so a score below -100 less that stays below -100.
    d, group = dims[2], dims[0] // dims[1]
    k, _ = held(cache, 0, page, slot)
    for h in range(dims[0]):
        at = slice(h * d, (h + 1) * d)
        qh, kh = q[:, at].double(), k[0, h // group]
        huge = qh @ kh / math.sqrt(d)
        off = 3 * 2.0 ** -11 * (qh.abs() @ kh.abs()) + 2.0 ** -14.9 * qh.abs().amax(1) * kh.abs().sum()
        clear = (huge < -100 - off / math.sqrt(d)) | (torch.arange(rows, device="cuda") == 0)
        got, ref = out[clear, at].double(), want[clear, at]
        if len(got):
            assert ((got - ref).norm() / ref.norm()).item() < 2 * HALF16


@pytest.mark.parametrize("sp", BOTH, ids=["tokens", "chunks"])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_odd_strides_and_offsets(dims, sp, dtype):
    torch = torch_()
    shape = fa.Shape(1, *dims)
    spans = Spans(sp, 16)
    cache, batch, q, out = run_attend(shape, spans, dtype, CAUSAL)
    w = shape.width
    for dt in (torch.bfloat16, torch.float32):
        wide_q = torch.zeros((spans.rows, w + 7), device="cuda", dtype=dt)
        wide_q[:, 3:3 + w] = q
        wide_out = torch.full((spans.rows, w + 9), 3.0, device="cuda", dtype=torch.bfloat16)
        cache.attend(0, batch, wide_q[:, 3:3 + w], wide_out[:, 1:1 + w])
        fa.device_status()
        assert torch.equal(wide_out[:, 1:1 + w], out)
        assert (wide_out[:, 0] == 3.0).all() and (wide_out[:, 1 + w:] == 3.0).all()


@pytest.mark.parametrize("sp", [[(1, 500)], [(50, 450)]], ids=["tokens", "chunk"])
@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_pages_past_32_bit_offsets(sp, dtype):
    """A pool whose last pages lie past 2^32 bytes (and elements) from its start."""
    torch = torch_()
    shape = fa.Shape(1, 8, 4, 128)
    per_page = 4 * 64 * 128
    pages = (1 << 32) // per_page + 40
    free = torch.cuda.mem_get_info()[0]
    if free < 3 * pages * per_page * (1 if dtype == fa.Q8 else 2):
        pytest.skip("not enough free device memory")
    spans = Spans(sp, 64)
    small = make_cache(shape, spans, dtype)
    _, _, q, out = run_attend(shape, spans, dtype, CAUSAL, cache=small)
    cache = fa.PagedCache(shape, pages, 64, dtype)
    shift = pages - spans.pages
    for name in ("keys", "values", "key_scales", "value_scales"):
        if getattr(small, name) is not None:
            getattr(cache, name)[:, shift:] = getattr(small, name)
    spans.tables += shift
    batch = spans.batch(cache)
    got = torch.empty_like(out)
    cache.attend(0, batch, q, got)
    k = torch.empty((spans.rows, 4, 128), device="cuda")
    v = torch.empty_like(k)
    cache.read(0, batch, k, v)
    cache.write(0, batch, k, v)
    k2, v2 = torch.empty_like(k), torch.empty_like(k)
    cache.read(0, batch, k2, v2)
    fa.device_status()
    assert torch.equal(got, out)
    want = held(small, 0, *spans.places(0, sp[0][1], sp[0][1] + sp[0][0]))
    assert torch.allclose(k.double(), want[0], rtol=1e-6) and torch.allclose(v.double(), want[1], rtol=1e-6)
    assert (k2 - k).abs().max() <= k.abs().max() / 127 and (v2 - v).abs().max() <= v.abs().max() / 127


def test_sequences_share_the_pages_of_a_prefix():
    torch = torch_()
    shape = fa.Shape(1, 8, 2, 128)
    spans = Spans([(1, 100), (1, 140), (30, 130)], 16)
    spans.tables_host[1, :6] = spans.tables_host[0, :6]
    spans.tables_host[2, :6] = spans.tables_host[0, :6]
    spans.tables = spans.tables_host.cuda()
    run_attend(shape, spans, fa.Q8, CAUSAL)


# ---- calls out of range ------------------------------------------------------------------------

def test_numbers_out_of_range_are_reported_and_leave_the_rest():
    """Spans and page ids out of range: the kernels' own checks leave such sequences (positions)
    out, the other sequences' rows are as ever, and the status says so once."""
    torch = torch_()
    shape = fa.Shape(1, 4, 2, 64)
    sp = [(1, 100), (2, 60), (1, 30), (40, 20)]
    spans = Spans(sp, 16)
    cache, batch, q, out = run_attend(shape, spans, fa.Q8, CAUSAL)
    kv = torch.randn((spans.rows, 2, 64), device="cuda")

    def calls():
        got = torch.full_like(out, 5.0)
        pools = [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales)]
        cache.attend(0, batch, q, got)
        k, v = torch.full_like(kv, 6.0), torch.full_like(kv, 6.0)
        cache.read(0, batch, k, v)
        cache.write(0, batch, kv, kv)
        torch.cuda.synchronize()
        for t, old in zip((cache.keys, cache.values, cache.key_scales, cache.value_scales), pools):
            t.copy_(old)
        return got, k

    calls()
    fa.device_status()
    # sequence 1's table ends before its last position
    kept = spans.firsts.clone()
    for first in (16 * spans.tables.shape[1] - 1, -5, 2**31 - 1):
        spans.firsts[1] = first
        got, k = calls()
        with pytest.raises(fa.CapacityError):
            fa.device_status()
        fa.device_status()
        assert torch.equal(got[0], out[0]) and torch.equal(got[3:], out[3:])
        assert (got[1:3] == 5.0).all() and (k[1:3] == 6.0).all() and (k[3:] != 6.0).any()
    spans.firsts.copy_(kept)
    # rows that run backwards, or past the call's
    starts = spans.row_starts.clone()
    for at, value in ((2, 0), (4, spans.rows + 1), (4, 2**31 - 1), (0, -1)):
        spans.row_starts[at] = value
        calls()
        with pytest.raises(fa.CapacityError):
            fa.device_status()
        spans.row_starts.copy_(starts)
    # pages outside the pool
    table = spans.tables.clone()
    for bad in (-1, spans.pages, 2**31 - 1, -2**31):
        spans.tables[0, 6] = bad  # positions 96..100 of sequence 0, its new row among them
        got, k = calls()
        with pytest.raises(fa.FaError) as e:
            fa.device_status()
        assert e.value.code == fa.ERR_ARG
        assert torch.equal(got[1:], out[1:]) and torch.isfinite(got[0]).all()
        assert (k[0] == 6.0).all()
        spans.tables.copy_(table)
    # one of the chunk's: its rows see the rest
    spans.tables[3, 1] = -3  # positions 16..31 of sequence 3, whose rows begin at 20
    got, k = calls()
    with pytest.raises(fa.FaError) as e:
        fa.device_status()
    assert e.value.code == fa.ERR_ARG and torch.equal(got[:4], out[:4])
    keys, values = held(cache, 0, *spans.places(3, 0, 60))
    see = visible(CAUSAL, torch.arange(20, 60, device="cuda"), 60)
    see[:, 16:32] = False
    for h in range(4):
        qh = q[4:, 64 * h:64 * (h + 1)].double()
        p = torch.softmax(torch.where(see, qh @ keys[:, h // 2].T / 8.0, -math.inf), 1)
        want, most = p @ values[:, h // 2], p @ values[:, h // 2].abs()
        check_close(got[4:, 64 * h:64 * (h + 1)], want, (HALF16 + 1e-4) * most, True)
    assert (k[4:16] == 6.0).all() and (k[16:] != 6.0).any()
    spans.tables.copy_(table)
    # every page of a sequence: its row sees nothing and is zero
    spans.tables[2] = -7
    got, k = calls()
    with pytest.raises(fa.FaError):
        fa.device_status()
    assert (got[3] == 0).all() and torch.equal(got[4:], out[4:])
    spans.tables.copy_(table)
    got, _ = calls()
    fa.device_status()
    assert torch.equal(got, out)


def test_more_rows_than_max_rows_are_left_out():
    torch = torch_()
    shape = fa.Shape(1, 4, 2, 64)
    spans = Spans([(1, 10), (30, 5)], 16)
    cache = make_cache(shape, spans, fa.BF16)
    q = torch.randn((31, 256), device="cuda")
    for most in (1, 20):
        out = torch.full((31, 256), 5.0, device="cuda")
        batch = spans.batch(cache, max_rows=most)
        cache.attend(0, batch, q, out)
        with pytest.raises(fa.CapacityError):
            fa.device_status()
        assert (out[1:] == 5.0).all() and (out[0] != 5.0).all()


@pytest.mark.parametrize("sp", BOTH, ids=["tokens", "chunks"])
@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
def test_rows_before_the_first_sequence_are_padding(sp, dtype):
    torch = torch_()
    shape = fa.Shape(1, 8, 2, 128)
    spans = Spans(sp, 16)
    lead = 3
    n, kv = spans.rows, (2, 128)
    qkv = torch.randn((lead + n, 12 * 128), device="cuda").bfloat16()
    outs, rows = [], []
    for at in (0, lead):
        cache = make_cache(shape, spans, dtype)
        batch = fa.PagedBatch(cache, spans.row_starts + at, spans.firsts, spans.tables, at + n,
                              spans.max_rows)
        batch.check()
        x = qkv[lead - at:]
        out = torch.full((at + n, shape.width), 5.0, device="cuda", dtype=torch.bfloat16)
        k = torch.full((at + n, *kv), 6.0, device="cuda")
        v = torch.full((at + n, *kv), 7.0, device="cuda")
        cache.attention(0, batch, x, out)
        cache.read(0, batch, k, v)
        fa.device_status()
        assert (out[:at] == 5.0).all() and (k[:at] == 6.0).all() and (v[:at] == 7.0).all()
        outs.append(out[at:])
        rows.append((k[at:], v[at:]))
    assert torch.equal(*outs)
    assert all(torch.equal(a, b) for a, b in zip(*rows))


def test_empty_batches():
    torch = torch_()
    shape = fa.Shape(1, 4, 2, 64)
    none = Spans([], 16)
    cache = fa.PagedCache(shape, 4, 16)
    i32 = dict(dtype=torch.int32, device="cuda")
    for n, width in ((0, 1), (3, 2)):
        batch = fa.PagedBatch(cache, torch.zeros(n + 1, **i32), torch.zeros(n, **i32),
                              torch.zeros((n, width), **i32), 5, 4)
        x = torch.full((5, 512), 2.0, device="cuda")
        out = torch.full((5, 256), 3.0, device="cuda")
        cache.attention(0, batch, x, out)
        cache.attend(0, batch, x, out)
        k = torch.full((5, 2, 64), 4.0, device="cuda")
        cache.read(0, batch, k, k)
        fa.device_status()
        assert (out == 3.0).all() and (k == 4.0).all()
        assert (cache.keys == 0).all()
    del none


# ---- runs of them together ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("dims", [(14, 2, 64), (32, 8, 128), (8, 2, 256)], ids=str)
def test_prompts_then_tokens_as_a_server_runs_them(dims, dtype):
    """Two layers: prompts in chunks of a mixed batch, then decode steps, every step's rows kept by
    the call that attends; each output against f64 attention over the pages as they are then."""
    torch = torch_()
    shape = fa.Shape(2, *dims)
    d = dims[2]
    grow = Spans([(0, 400), (0, 400)], 16, spare=0)  # the tables of two sequences of up to 400
    cache = fa.PagedCache(shape, grow.pages, 16, dtype)
    g = torch.Generator(device="cuda").manual_seed(11)
    steps = [[(150, 0), (0, 0)], [(100, 150), (61, 0)], [(1, 250), (90, 61)], [(1, 251), (1, 151)],
             [(3, 252), (1, 152)], [(1, 255), (1, 153)]]
    for sp in steps:
        spans = Spans(sp, 16)
        spans.tables_host, spans.tables = grow.tables_host, grow.tables
        batch = spans.batch(cache)
        batch.check()
        angles = angles_of(spans, d)
        for layer in range(2):
            qkv = torch.randn((spans.rows, shape.qkv), generator=g, device="cuda").bfloat16()
            out = torch.empty((spans.rows, shape.width), device="cuda", dtype=torch.bfloat16)
            cache.attention(layer, batch, qkv, out, angles)
            fa.device_status()
            x = qkv.double().reshape(spans.rows, -1, d)
            q = rotate(x[:, :dims[0]], angles, fa.ROPE_HALF).reshape(spans.rows, -1)
            want, tol = reference(cache, layer, spans, q, CAUSAL, HALF16)
            check_close(out, want, tol, True)
            k = torch.empty((spans.rows, dims[1], d), device="cuda")
            v = torch.empty_like(k)
            cache.read(layer, batch, k, v)
            turned = rotate(x[:, dims[0]:dims[0] + dims[1]], angles, fa.ROPE_HALF)
            top = turned.abs().amax(-1, keepdim=True)
            lim = top / 254 + 1e-5 * top if dtype == fa.Q8 else HALF16 * turned.abs() + 1e-5
            assert ((k.double() - turned).abs() <= lim).all()


def test_a_captured_step_follows_the_batchs_numbers():
    """One capture of a decode step (attention over the pages, rows kept), replayed as the
    sequences grow: the numbers are read on the device."""
    torch = torch_()
    shape = fa.Shape(1, 8, 2, 128)
    d, n = 128, 3
    grow = Spans([(0, 300)] * n, 16, spare=0)
    cache = make_cache(shape, grow, fa.Q8)
    spans = Spans([(1, 40), (1, 130), (1, 7)], 16)
    spans.tables_host, spans.tables = grow.tables_host, grow.tables
    batch = spans.batch(cache)
    qkv = torch.randn((n, shape.qkv), device="cuda").bfloat16()
    angles = torch.empty((n, d), device="cuda")
    out = torch.empty((n, shape.width), device="cuda", dtype=torch.bfloat16)
    angles.copy_(angles_of(spans, d))
    cache.attention(0, batch, qkv, out, angles)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(0, batch, qkv, out, angles)
    for step in range(4):
        sp = [(1, 40 + 17 * step), (1, 130 + step), (1, 7 + 90 * step)]
        now = Spans(sp, 16)
        now.tables_host = grow.tables_host
        batch.firsts.copy_(now.firsts)
        angles.copy_(angles_of(now, d))
        qkv.copy_(torch.randn_like(qkv))
        graph.replay()
        fa.device_status()
        q = rotate(qkv.double().reshape(n, -1, d)[:, :8], angles, fa.ROPE_HALF).reshape(n, -1)
        want, tol = reference(cache, 0, now, q, CAUSAL, HALF16)
        check_close(out, want, tol, True)


def test_two_batches_on_two_streams():
    torch = torch_()
    shape = fa.Shape(1, 16, 8, 128)
    runs = []
    for i, sp in enumerate(([(1, 20000)], [(1, 15000), (1, 9000)], [(200, 3000)])):
        spans = Spans(sp, 64)
        cache, batch, q, out = run_attend(shape, spans, fa.Q8, CAUSAL, seed=20 + i)
        runs.append((cache, batch, q, out, torch.cuda.Stream(), torch.empty_like(out)))
    torch.cuda.synchronize()
    for _ in range(20):
        for cache, batch, q, out, stream, got in runs:
            cache.attend(0, batch, q, got, stream=stream)
    torch.cuda.synchronize()
    for *_, out, _, got in runs:
        assert torch.equal(got, out)
    fa.device_status()

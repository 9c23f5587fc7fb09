"""The paged cache's operators, measured: keys and values written into pages (quantised to 8 bits
or held in bf16) and read back, single tokens attending over long paged contexts, and chunks of
new tokens attending over a paged cache.

A pool holds `pages` pages of `page_size` positions of every KV head, [layer][page][KV head][slot]
[head_dim]; a sequence's position p lies in slot p % page_size of page tables[sequence][p //
page_size]. 8-bit pages hold round(x * 127 / max|x|) of each (position, KV head) and the f32 scale
max|x| / 127 beside them. A call's rows are those of several sequences one after the other
(row_starts), a sequence's rows at consecutive positions from firsts[sequence].
"""
import math
import random
import sys

import torch

own = False

BASE = 1e6
NEG = float("-inf")


def _fa():
    if "fusor-ai_b200" not in sys.path:
        sys.path.insert(0, "fusor-ai_b200")
    import fusor_attn
    return fusor_attn


# ---- cases -------------------------------------------------------------------------------------

def _case(name, kind, pages, heads, kv_heads, head_dim, sequences, keys, rows, page_size=16,
          rows_type="bf16", window=0, norm=False, lengths=1, long_rows=0):
    """keys: (least, most) positions a sequence holds after the call; rows: (least, most) of them
    that are the call's; long_rows: the rows of the last sequence, where it differs."""
    return {"name": name, "kind": kind, "pages": pages, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "sequences": sequences, "least_keys": keys[0],
            "most_keys": keys[1], "least_rows": rows[0], "most_rows": rows[1],
            "page_size": page_size, "rows_type": rows_type, "window": window, "norm": norm,
            "lengths": lengths, "long_rows": long_rows}


def listed():
    return [
        # one decode step's new tokens of a few users written to 8-bit pages and read back: the
        # smallest call, all latency (14 query heads over 2 KV heads of 64)
        _case("write_step_q8", "write", "q8", 14, 2, 64, 5, (300, 3000), (1, 1)),
        # a prompt's rows written to 8-bit pages (32/8 heads of 128): the write at its largest
        _case("write_prompt_q8", "write", "q8", 32, 8, 128, 3, (2000, 9000), (1500, 5001),
              lengths=2),
        # prompts with head norms and f32 rows, as the gated layers' 8/2 heads of 256 have them
        _case("write_normed_bf16", "write", "bf16", 8, 2, 256, 4, (700, 2500), (300, 1111),
              page_size=32, rows_type="f32", norm=True, lengths=3),
        # whole contexts read back out of 8-bit pages, to be handed to another cache
        _case("read_long_q8", "read", "q8", 32, 8, 128, 2, (60000, 70001), (0, 0), page_size=64,
              lengths=4),
        # a short prefix read out of bf16 pages
        _case("read_prefix_bf16", "read", "bf16", 14, 2, 64, 3, (97, 611), (0, 0), lengths=5),
        # a decode step of 64 users at mixed lengths, 8-bit and bf16 pages
        _case("decode_64_q8", "attend", "q8", 32, 8, 128, 64, (512, 8192), (1, 1), lengths=6),
        _case("decode_64_bf16", "attend", "bf16", 32, 8, 128, 64, (512, 8192), (1, 1),
              lengths=7),
        # one user's decode step over a long context (16/8 heads of 128)
        _case("decode_long_q8", "attend", "q8", 16, 8, 128, 1, (131072, 131072), (1, 1),
              page_size=64, lengths=8),
        # a decode step of a small model for a few users: latency
        _case("decode_few_bf16", "attend", "bf16", 14, 2, 64, 3, (500, 1500), (1, 1),
              lengths=9),
        # a prompt's chunk after what is already cached
        _case("chunk_q8", "attend", "q8", 32, 8, 128, 1, (16384, 16384), (2048, 2048),
              lengths=10),
        # ragged chunks under a sliding window, head_dim 256
        _case("chunk_window_bf16", "attend", "bf16", 8, 2, 256, 5, (1000, 6000), (100, 999),
              page_size=32, window=1024, lengths=11),
        # one whole step of a mixed batch, rows in, written and attended: users decoding beside
        # one prompt's chunk
        _case("step_mixed_q8", "step", "q8", 32, 8, 128, 25, (400, 4000), (1, 1), lengths=12,
              long_rows=389),
    ]


def _log(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "step"])
    heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (32, 8, 128), (16, 8, 128), (12, 12, 128),
                                            (8, 2, 256), (16, 2, 256)])
    case = _case("", kind, rng.choice(["q8", "q8", "bf16"]), heads, kv_heads, head_dim, 1, (1, 1),
                 (1, 1), page_size=rng.choice([16, 32, 64, 128]),
                 rows_type=rng.choice(["bf16", "bf16", "f32"]) if kind == "write" else "bf16",
                 norm=kind != "attend" and rng.random() < 0.3, lengths=rng.randrange(1, 1 << 20))
    del case["name"]
    if kind == "read":
        case["most_keys"] = _log(rng, 50, 60000)
        case["sequences"] = max(1, min(_log(rng, 1, 40), 120000 // case["most_keys"]))
        case["least_keys"] = max(1, case["most_keys"] // rng.choice([1, 2, 7]))
        case["least_rows"] = case["most_rows"] = 0
        return case
    form = rng.choice(["token", "token", "few", "chunk"])
    if kind == "write":
        form = rng.choice(["token", "few", "chunk"])
    most = _log(rng, 64, 100000 if form == "token" else 14000)
    case["most_rows"] = {"token": 1, "few": rng.randrange(2, 9),
                         "chunk": min(most, _log(rng, 17, 2000))}[form]
    # the plain form pads every sequence to the longest: rows x keys of all of them bounded
    room = min(500000 // most, int(3e7 // (most * case["most_rows"])))
    case["sequences"] = max(1, min(_log(rng, 1, 64), room))
    case["most_keys"] = most
    case["least_keys"] = max(1, most // rng.choice([1, 2, 12]))
    case["least_rows"] = 1 if form == "few" else max(1, case["most_rows"] // 3)
    if kind == "attend" and rng.random() < 0.3:
        case["window"] = _log(rng, 16, 4000)
    if kind == "step" and form == "token":
        case["long_rows"] = min(most, _log(rng, 2, 400))
        case["sequences"] = max(1, min(case["sequences"], int(3e7 // (most * case["long_rows"]))))
    return case


def _spans(case):
    """(keys, rows) of every sequence: keys positions after the call, the last rows of them new."""
    r = random.Random(case["lengths"])
    out = []
    for i in range(case["sequences"]):
        keys = r.randint(case["least_keys"], case["most_keys"])
        rows = min(keys, r.randint(case["least_rows"], case["most_rows"]))
        if i == case["sequences"] - 1 and case["long_rows"]:
            rows = min(keys, case["long_rows"])
        if case["kind"] == "read":
            rows = keys
        out.append((keys, rows))
    return out


def _seen(case, keys, rows):
    """Keys that the rows see in all, and distinct positions that any of them sees."""
    w = case["window"]
    pairs = sum(min(p + 1, w) if w else p + 1 for p in range(keys - rows, keys))
    lo = max(0, keys - rows + 1 - w) if w else 0
    return pairs, keys - lo


def work(case):
    kvh, d, heads = case["kv_heads"], case["head_dim"], case["heads"]
    held = kvh * (d + 4 if case["pages"] == "q8" else 2 * d)  # bytes of a position's keys
    esz = 2 if case["rows_type"] == "bf16" else 4
    read = written = flops = 0
    for keys, rows in _spans(case):
        if case["kind"] == "read":
            read += 2 * rows * held
            written += 2 * rows * kvh * d * 2
            flops += 2 * rows * kvh * d
            continue
        if case["kind"] in ("write", "step"):
            read += rows * (heads + 2 * kvh) * d * esz + rows * d * 4
            written += 2 * rows * held
            flops += rows * (heads + 2 * kvh) * d * 3
        if case["kind"] == "write":
            written += rows * heads * d * esz + 2 * rows * kvh * d * 2
            read += 2 * rows * held
        else:
            pairs, distinct = _seen(case, keys, rows)
            read += 2 * distinct * held
            written += rows * heads * d * 2
            flops += 4 * pairs * heads * d
            if case["kind"] == "attend":
                read += rows * heads * d * 2
            else:
                read -= 2 * rows * held  # the step's own rows need no second trip
    return {"bytes": read + written, "flops": flops}


# ---- inputs ------------------------------------------------------------------------------------

def _quantise(x):
    """int8 values and f32 scales of x's last dimension."""
    top = x.abs().amax(-1, keepdim=True)
    q = (x * (127.0 / top)).round().clamp(-127, 127)
    return q.to(torch.int8), (top / 127.0).squeeze(-1)


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    heads, kvh, d, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    spans = _spans(case)
    n = len(spans)
    width = max(-(-keys // ps) for keys, _ in spans)
    pages = sum(-(-keys // ps) for keys, _ in spans) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    tables = torch.zeros((n, width), dtype=torch.int32, device=dev)
    at = 0
    for i, (keys, _) in enumerate(spans):
        used = -(-keys // ps)
        tables[i, :used] = order[at:at + used]
        at += used
    rows = sum(r for _, r in spans)
    starts = [0]
    for _, r in spans:
        starts.append(starts[-1] + r)
    s = {"case": dict(case), "tables": tables, "rows": rows,
         "max_rows": max(r for _, r in spans), "max_keys": max(k for k, _ in spans),
         "row_starts": torch.tensor(starts, dtype=torch.int32, device=dev),
         "firsts": torch.tensor([k - r for k, r in spans], dtype=torch.int32, device=dev)}
    # keys have a few strong channels, values are plain; a sequence's first position is a sink
    # with strong keys and weak values
    shape = (1, pages, kvh, ps, d)
    channel = torch.ones(d, device=dev)
    channel[torch.randperm(d, generator=g, device=dev)[:4]] = 3.0
    channel = channel / channel.square().mean().sqrt()
    k = torch.randn(shape, generator=g, device=dev) * channel
    v = torch.randn(shape, generator=g, device=dev)
    k[0, tables[:, 0].long(), :, 0] *= 1.5
    v[0, tables[:, 0].long(), :, 0] *= 0.05
    if case["pages"] == "q8":
        s["keys"], s["key_scales"] = _quantise(k)
        s["values"], s["value_scales"] = _quantise(v)
    else:
        s["keys"], s["values"] = k.bfloat16(), v.bfloat16()
        s["key_scales"] = s["value_scales"] = None
    del k, v
    rows_type = torch.bfloat16 if case["rows_type"] == "bf16" else torch.float32
    if case["kind"] == "attend":
        s["q"] = (1.5 * torch.randn((rows, heads * d), generator=g, device=dev)).to(rows_type)
    elif case["kind"] in ("write", "step"):
        qkv = torch.randn((rows, heads + 2 * kvh, d), generator=g, device=dev)
        qkv[:, heads:heads + kvh] *= channel
        s["qkv"] = qkv.reshape(rows, -1).to(rows_type)
        pos = torch.cat([torch.arange(k_ - r, k_, device=dev) for k_, r in spans]).double()
        inv = BASE ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        ang = pos[:, None] * inv
        s["angles"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        if case["norm"]:
            s["q_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
            s["k_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
    return s


# ---- the plain form ----------------------------------------------------------------------------

def _places(s):
    """Sequence, page and slot of every row of the call."""
    ps = s["case"]["page_size"]
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["row_starts"].long(), row, right=True) - 1
    pos = s["firsts"].long()[seq] + row - s["row_starts"].long()[seq]
    return seq, pos, s["tables"][seq, pos // ps].long(), pos % ps


def _plain_write(s):
    c = s["case"]
    heads, kvh, d = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float().view(s["rows"], heads + 2 * kvh, d)
    qk, v = x[:, :heads + kvh], x[:, heads + kvh:]
    if c["norm"]:
        inverse = 1.0 / torch.sqrt(qk.square().mean(-1, keepdim=True) + 1e-6)
        weight = torch.cat([s["q_norm"].expand(heads, d), s["k_norm"].expand(kvh, d)])
        qk = qk * inverse * weight
    a, b = qk[..., :d // 2], qk[..., d // 2:]
    cos, sin = s["angles"][:, None, :d // 2], s["angles"][:, None, d // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    _, _, page, slot = _places(s)
    for pool, scales, new in ((s["keys"], s["key_scales"], qk[:, heads:]),
                              (s["values"], s["value_scales"], v)):
        if c["pages"] == "q8":
            ints, scale = _quantise(new)
            pool[0][page, :, slot] = ints
            scales[0][page, :, slot] = scale
        else:
            pool[0][page, :, slot] = new.bfloat16()
    return qk[:, :heads].reshape(s["rows"], heads * d)


def _held(s, pool, scales, page, slot):
    x = s[pool][0][page, :, slot].float()
    return x if s[scales] is None else x * s[scales][0][page, :, slot][..., None]


def _plain_read(s):
    _, _, page, slot = _places(s)
    return {"keys": _held(s, "keys", "key_scales", page, slot).bfloat16(),
            "values": _held(s, "values", "value_scales", page, slot).bfloat16()}


def _plain_attend(s, q):
    """Every sequence padded to the longest and to the most rows."""
    c = s["case"]
    heads, kvh, d, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page_size"]
    n, r, most, group = c["sequences"], s["max_rows"], s["max_keys"], heads // kvh
    pos = torch.arange(most, device="cuda")
    page = s["tables"][:, pos // ps].long()
    slot = (pos % ps).expand(n, most)
    k = _held(s, "keys", "key_scales", page, slot)  # sequence, key, KV head, element
    v = _held(s, "values", "value_scales", page, slot)
    starts, firsts = s["row_starts"].long(), s["firsts"].long()
    j = torch.arange(r, device="cuda")
    there = j < (starts[1:] - starts[:-1])[:, None]
    row = (starts[:-1, None] + j).clamp(max=s["rows"] - 1)
    at = firsts[:, None] + j
    seen = pos <= at[..., None]
    if c["window"]:
        seen &= pos > at[..., None] - c["window"]
    x = q.float().view(-1, kvh, group, d)[row].permute(0, 2, 1, 3, 4).reshape(n, kvh, r * group, d)
    scores = torch.matmul(x, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    scores = scores.view(n, kvh, r, group, most).masked_fill_(~seen[:, None, :, None], NEG)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    o = torch.matmul(scores.view(n, kvh, r * group, most), v.permute(0, 2, 1, 3))
    o = o.view(n, kvh, r, group, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(n, r, heads * d)
    return o[there].bfloat16()


# ---- one pass ----------------------------------------------------------------------------------

def _handles(s):
    """The cache and batch objects that a user's program keeps beside its tensors."""
    if "cache" not in s:
        fa, c = _fa(), s["case"]
        s["cache"] = fa.PagedCache(
            fa.Shape(1, c["heads"], c["kv_heads"], c["head_dim"]), s["keys"].shape[1],
            c["page_size"], fa.Q8 if c["pages"] == "q8" else fa.BF16, keys=s["keys"],
            values=s["values"], key_scales=s["key_scales"], value_scales=s["value_scales"])
        s["batch"] = fa.PagedBatch(
            s["cache"], s["row_starts"], s["firsts"], s["tables"], s["rows"], s["max_rows"],
            fa.Mask.window_of(c["window"]) if c["window"] else fa.Mask.causal())
        s["norm_args"] = (s["q_norm"], s["k_norm"], 1e-6) if c["norm"] and "qkv" in s else None
    return s["cache"], s["batch"]


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        if kind == "write":
            q = _plain_write(s).to(s["qkv"].dtype)
            return {"q": q, **_plain_read(s)}
        if kind == "read":
            return _plain_read(s)
        if kind == "attend":
            return _plain_attend(s, s["q"])
        q = _plain_write(s)
        return {"out": _plain_attend(s, q), **_plain_read(s)}
    cache, batch = _handles(s)
    c = s["case"]

    def rows(width, dtype=torch.bfloat16):
        return torch.empty((s["rows"], width), dtype=dtype, device="cuda")

    def read():
        held = (s["rows"], c["kv_heads"], c["head_dim"])
        k = torch.empty(held, dtype=torch.bfloat16, device="cuda")
        v = torch.empty(held, dtype=torch.bfloat16, device="cuda")
        cache.read(0, batch, k, v)
        return {"keys": k, "values": v}

    width = c["heads"] * c["head_dim"]
    if kind == "write":
        q = rows(width, s["qkv"].dtype)
        cache.attention_input(0, batch, s["qkv"], s["angles"], norm=s["norm_args"], q_out=q)
        return {"q": q, **read()}
    if kind == "read":
        return read()
    out = rows(width)
    if kind == "attend":
        cache.attend(0, batch, s["q"], out)
        return out
    cache.attention(0, batch, s["qkv"], out, s["angles"], norm=s["norm_args"])
    return {"out": out, **read()}


# ---- in 64 bits --------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    heads, kvh, d, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    group, kind = heads // kvh, case["kind"]
    spans = _spans(case)
    if sum(_seen(case, k, r)[0] for k, r in spans) * heads * d > 1.2e12 and kind != "read":
        return None
    starts = s["row_starts"].tolist()
    kept = {}
    if kind in ("write", "step"):
        x = s["qkv"].double().view(s["rows"], heads + 2 * kvh, d)
        turned = []
        for h in range(heads + kvh):
            y = x[:, h]
            if case["norm"]:
                y = y / (y.pow(2).sum(1, keepdim=True) / d + 1e-6).sqrt()
                y = y * (s["q_norm"] if h < heads else s["k_norm"]).double()
            z = torch.complex(y[:, :d // 2], y[:, d // 2:])
            z = z * torch.complex(s["angles"][:, :d // 2].double(), s["angles"][:, d // 2:].double())
            turned.append(torch.cat([z.real, z.imag], 1))
        q = torch.cat(turned[:heads], 1)
        kept = {"keys": torch.stack(turned[heads:], 1), "values": x[:, heads + kvh:]}
        for name, new in kept.items():
            if case["pages"] == "q8":
                step = new.abs().amax(2, keepdim=True) / 127
                kept[name] = torch.round(new / step) * step
            else:
                kept[name] = new.bfloat16().double()
    elif kind == "attend":
        q = s["q"].double()
    read = {"keys": [], "values": []}
    out = torch.empty((s["rows"], heads * d), dtype=torch.float64, device="cuda")
    for i, (keys, rows) in enumerate(spans):
        page = s["tables"][i, :-(-keys // ps)].long()
        held = {}
        for name, scales in (("keys", "key_scales"), ("values", "value_scales")):
            x = s[name][0, page].double()
            if case["pages"] == "q8":
                x = x * s[scales][0, page].double().unsqueeze(-1)
            x = x.transpose(1, 2).reshape(-1, kvh, d)[:keys]
            if name in kept:
                x[keys - rows:] = kept[name][starts[i]:starts[i + 1]]
            held[name] = x
            read[name].append(x[keys - rows:])
        if kind in ("write", "read"):
            continue
        mine = slice(starts[i], starts[i + 1])
        at = torch.arange(keys - rows, keys, device="cuda")[:, None]
        pos = torch.arange(keys, device="cuda")
        hidden = pos > at
        if case["window"]:
            hidden |= pos <= at - case["window"]
        for h in range(heads):
            scores = q[mine, h * d:(h + 1) * d] @ held["keys"][:, h // group].T / math.sqrt(d)
            p = torch.softmax(scores.masked_fill(hidden, NEG), 1)
            out[mine, h * d:(h + 1) * d] = p @ held["values"][:, h // group]
    if kind == "attend":
        return out
    read = {name: torch.cat(x) for name, x in read.items()}
    if kind == "write":
        return {"q": q, **read}
    return read if kind == "read" else {"out": out, **read}

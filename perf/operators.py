"""The cases and the plain forms of the 4-bit paged cache's operators and of the
rotary positions they share:

* ``rotary``     rotation of query and key rows by their positions (half or interleaved
                 pairs, part of the head, tables scaled for long contexts);
* ``append``     the same rotation, then the new tokens' keys and values written to a
                 paged cache in 4 bits, and those tokens read back as the values held;
* ``attention``  decode attention (one query token per request, grouped heads) over
                 that cache, with the base-2 log-sum-exp.

``run`` computes the plain forms with elementary torch operations in 32 bits, or, where
``own`` is true, calls the framework.  ``exact`` gives the same results in 64 bits.

The cache is one record of 2560 bytes per (page of 16 tokens, KV head).  A token's key
and value are each held as 128 codes z of 4 bits with a scale s and a midpoint m (float16)
per group of 32 dimensions, x = (z - 8) * s + m.
"""

import math
import random

import torch

own = False

PAGE, DIM, GROUP, RECORD = 16, 128, 32, 2560
HALF_MAX = 65504.0
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------ cases
def _rotary(name, tokens, first, q_heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
            interleaved=False, adjoint=False, dtype="float16", scaling="none", factor=1.0):
    return dict(name=name, op="rotary", tokens=tokens, first=first, q_heads=q_heads,
                kv_heads=kv_heads, head_dim=head_dim, rotary_dim=rotary_dim,
                interleaved=interleaved, adjoint=adjoint, dtype=dtype, scaling=scaling,
                factor=factor)


def _append(name, batch, min_new, max_new, context, padding=0, q_heads=32, kv_heads=8,
            rotary_dim=128, interleaved=False, dtype="float16", scaling="none", factor=1.0,
            center=True, length_seed=1):
    return dict(name=name, op="append", batch=batch, min_new=min_new, max_new=max_new,
                context=context, padding=padding, q_heads=q_heads, kv_heads=kv_heads,
                rotary_dim=rotary_dim, interleaved=interleaved, dtype=dtype, scaling=scaling,
                factor=factor, center=center, length_seed=length_seed)


def _attention(name, batch, min_len, max_len, q_heads=32, kv_heads=8, dtype="float16",
               center=True, length_seed=1):
    return dict(name=name, op="attention", batch=batch, min_len=min_len, max_len=max_len,
                q_heads=q_heads, kv_heads=kv_heads, dtype=dtype, center=center,
                length_seed=length_seed)


def listed():
    return [
        # one decode step of one request: latency
        _rotary("rotary 1 token", 1, 16383),
        # a prompt of a model that rotates half of each head, neighbouring pairs,
        # positions interpolated to four times the trained length
        _rotary("rotary 8191 interleaved", 8191, 0, rotary_dim=64, interleaved=True,
                dtype="bfloat16", scaling="linear", factor=4.0),
        # the gradient's direction of a long packed batch of small float32 heads
        _rotary("rotary 16385 adjoint", 16385, 0, q_heads=8, kv_heads=2, head_dim=64,
                rotary_dim=64, adjoint=True, dtype="float32"),
        # the longest prompt of the headline workload, frequencies scaled by parts
        _rotary("rotary 49152 by parts", 49152, 0, scaling="parts", factor=8.0),
        # one decode step of one request in a long context
        _append("append 1 token", 1, 1, 1, 49151),
        # one decode step of a batch of 32 with rows padded to a captured batch of 35
        _append("append 32 decode rows", 32, 1, 1, 16384, padding=3, length_seed=5),
        # one prompt of an odd length behind a cached prefix, half of each head rotated
        _append("append 4095 prompt", 1, 4095, 4095, 1001, rotary_dim=64, interleaved=True,
                dtype="bfloat16", center=False),
        # a batch of eight ragged prompts in one call
        _append("append ragged prompts", 8, 1023, 16384, 0, scaling="parts", factor=4.0,
                length_seed=7),
        # the shortest context there is: latency
        _attention("attention 1 token", 1, 1, 1),
        # the headline context, one request
        _attention("attention 49152", 1, 49152, 49152),
        # eight ragged requests
        _attention("attention ragged", 8, 8192, 65536, length_seed=3),
        # one rank's heads of a batch of 32, with eight query heads to a KV head, no centre
        _attention("attention 32 requests", 32, 0, 16384, q_heads=16, kv_heads=2,
                   dtype="bfloat16", center=False, length_seed=11),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(max(low, 1)),
                                                       math.log(high + 1))))))


def _drawn(rng):
    op = rng.choice(("rotary", "append", "attention"))
    seed = rng.randrange(1, 1 << 20)
    scaling = rng.choice(("none", "linear", "parts"))
    factor = 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0))
    dtype = rng.choice(("float16", "bfloat16"))
    kv_heads = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8))
    if op == "rotary":
        head_dim = rng.choice((64, 80, 96, 128, 256))
        rotary_dim = rng.choice((head_dim, head_dim // 2, head_dim // 2 - 6))
        return _rotary("", _spread(rng, 1, 40000), rng.randrange(0, 60000), group * kv_heads,
                       kv_heads, head_dim, rotary_dim, rng.random() < 0.5, rng.random() < 0.3,
                       rng.choice((dtype, "float32")), scaling, factor)
    if op == "append":
        batch = _spread(rng, 1, 64)
        most = _spread(rng, 1, max(1, 65536 // batch))
        return _append("", batch, rng.randint(1, most), most, rng.randrange(0, 50000),
                       rng.choice((0, 0, 1, 5)), group * kv_heads, kv_heads,
                       rng.choice((128, 64, 32, 58)), rng.random() < 0.5, dtype, scaling, factor,
                       rng.random() < 0.5, seed)
    batch = _spread(rng, 1, 64)
    most = _spread(rng, 1, min(131072, 524288 // batch))
    return _attention("", batch, rng.choice((0, 1, most // 2, most)), most, group * kv_heads,
                      kv_heads, dtype, rng.random() < 0.5, seed)


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        case = _drawn(rng)
        if work(case)["bytes"] <= most:
            del case["name"]
            return case


def _lengths(case, low, high):
    """The case's own ragged lengths, whatever the inputs' seed."""
    rng = random.Random(case["length_seed"])
    return [rng.randint(low, high) for _ in range(case["batch"])]


def work(case):
    heads = case["q_heads"], case["kv_heads"]
    if case["op"] == "rotary":
        size = DTYPES[case["dtype"]].itemsize
        n = case["tokens"] * (heads[0] + heads[1])
        table = 4 * case["rotary_dim"] * case["tokens"]
        return {"bytes": 2 * n * case["head_dim"] * size + table + 4 * case["tokens"],
                "flops": 3 * n * case["rotary_dim"]}
    if case["op"] == "append":
        # rows read, rotated queries written, 160 bytes of cache per token and KV head
        # written and read back, and the values held written as rows
        n = sum(_lengths(case, case["min_new"], case["max_new"]))
        row = 2 * DIM
        moved = 2 * heads[0] * row + heads[1] * (2 * row + 2 * 160 + 2 * row)
        return {"bytes": n * (moved + 4 * case["rotary_dim"] + 8),
                "flops": n * (3 * (heads[0] + heads[1]) * case["rotary_dim"]
                              + 8 * heads[1] * DIM)}
    lengths = _lengths(case, case["min_len"], case["max_len"])
    tokens = sum(lengths)
    return {"bytes": tokens * heads[1] * 160 + 4 * sum(-(-n // PAGE) for n in lengths)
            + case["batch"] * heads[0] * (2 * 2 * DIM + 4),
            "flops": 4 * heads[0] * DIM * tokens}


# ----------------------------------------------------------------- inputs
def _frequencies(case):
    """Angles per position of each pair, in 64 bits, and the factor on both tables.

    ``linear`` divides every position by the factor.  ``parts`` divides the frequencies of
    pairs that turn less than once within the trained length (here 8192 positions), keeps
    those that turn more than 32 times, blends the pairs between, and scales the tables."""
    dim, factor, theta = case["rotary_dim"], case["factor"], 1e6
    inv = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if case["scaling"] == "linear":
        return inv / factor, 1.0
    if case["scaling"] == "parts":
        trained = 8192
        pair = lambda turns: dim * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low)
                / max(high - low, 1e-3)).clamp(0, 1)
        return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def _tables(case, positions):
    inv, scale = _frequencies(case)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv.cuda()
    return (angle.cos() * scale).float(), (angle.sin() * scale).float()


def _channels(g, heads, size):
    """Rows as projections give them: unit noise, an offset per channel, some loud channels."""
    offset = torch.randn(heads, size, generator=g, device="cuda")
    loud = torch.where(torch.rand(heads, size, generator=g, device="cuda") < 0.02, 6.0, 1.0)
    return offset * 0.5 * loud, loud


def _packed_rows(case, g, tokens, size, dtype):
    """Query, key and value rows as views of one packed projection's output."""
    hq, hkv = case["q_heads"], case["kv_heads"]
    heads = hq + 2 * hkv
    offset, loud = _channels(g, heads, size)
    rows = torch.empty(tokens, heads, size, dtype=dtype, device="cuda")
    for a in range(0, tokens, 8192):
        b = min(tokens, a + 8192)
        rows[a:b] = torch.randn(b - a, heads, size, generator=g, device="cuda") * loud + offset
    return rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:], offset[hq:hq + hkv], \
        offset[hq + hkv:]


def _tokens_of(case):
    """Per new token its request and its position, and the pages each request holds."""
    new = _lengths(case, case["min_new"], case["max_new"])
    request, position, pages = [], [], []
    for r, n in enumerate(new):
        request += [r] * n
        position += range(case["context"], case["context"] + n)
        pages.append(-(-(case["context"] + n) // PAGE))
    return torch.tensor(request, device="cuda"), torch.tensor(position, device="cuda"), pages


def _append_inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    request, position, pages = _tokens_of(case)
    n, pad = request.numel(), case["padding"]
    q, k, v, k_offset, v_offset = _packed_rows(case, g, n + pad, DIM, DTYPES[case["dtype"]])
    # Each request's pages lie anywhere in the pool.  Only the pages that this call
    # touches are there; the cached prefix's would not be read.
    first = case["context"] // PAGE
    start = torch.tensor([0] + [p - first for p in pages], device="cuda").cumsum(0)
    pool = int(start[-1])
    order = torch.randperm(pool, generator=g, device="cuda")
    slot = order[start[request] + position // PAGE - first] * PAGE + position % PAGE
    padded = torch.full((pad,), -1, dtype=torch.int32, device="cuda")
    state = {"case": case, "q": q, "k": k, "v": v, "pool_pages": pool,
             "positions": torch.cat((position.int(), padded.clamp(min=0))),
             "slots": torch.cat((slot.int(), padded)), "k_center": None, "v_center": None,
             "rows": None}
    if case["center"]:
        shape = (case["batch"], case["kv_heads"], DIM)
        jitter = lambda: 0.1 * torch.randn(shape, generator=g, device="cuda")  # noqa: E731
        state["k_center"] = (k_offset + jitter()).to(q.dtype)
        state["v_center"] = (v_offset + jitter()).to(q.dtype)
        state["rows"] = torch.cat((request.int(), padded.clamp(min=0)))
    return state


def _quantised(x):
    """Codes, scales and midpoints of rows [..., 128] in 32 bits (inputs only)."""
    x = x.view(*x.shape[:-1], DIM // GROUP, GROUP)
    low = x.amin(-1)
    s = ((x.amax(-1) - low) / 15).half()
    m = (low + 8 * s.float()).half()
    z = ((x - m.float()[..., None]) / s.float()[..., None]).round().add_(8).clamp_(0, 15)
    return z.to(torch.uint8).flatten(-2), s, m


def _record(kz, ks, km, vz, vs, vm):
    """Records [pages, Hkv, 2560] of codes [pages, Hkv, 16, 128], scales and midpoints."""
    lead = kz.shape[:2]
    k = kz.view(*lead, PAGE, 4, 4, 8).transpose(-3, -2).reshape(*lead, PAGE, 64, 2)
    v = vz.view(*lead, 2, 4, 2, 4, 8, 4).transpose(-5, -4).transpose(-3, -2)
    v = v.reshape(*lead, PAGE, 64, 2)
    codes = [(c[..., 0] | (c[..., 1] << 4)).flatten(-2) for c in (k, v)]
    metas = [torch.cat((s, m), -1).view(torch.uint8).flatten(-2) for s, m in ((ks, km), (vs, vm))]
    return torch.cat(codes + metas, -1)


def _cache_pages(case, g, pages):
    """Chunks of (first page, codes, scales and midpoints of keys, of values)."""
    heads = case["kv_heads"]
    k_offset, k_loud = _channels(g, heads, DIM)
    v_offset, v_loud = _channels(g, heads, DIM)
    if case["center"]:  # centred rows keep a tenth of their offsets
        k_offset, v_offset = 0.2 * k_offset, 0.2 * v_offset
    step = max(1, 32768 // (PAGE * heads) * 4)
    for a in range(0, pages, step):
        shape = (min(step, pages - a), heads, PAGE, DIM)
        noise = lambda: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
        k = _quantised(noise() * k_loud[:, None] + k_offset[:, None])
        v = _quantised(noise() * v_loud[:, None] + v_offset[:, None])
        yield a, k, v


def _attention_inputs(case, seed, keep):
    g = torch.Generator("cuda").manual_seed(seed)
    lengths = _lengths(case, case["min_len"], case["max_len"])
    pages = [-(-n // PAGE) for n in lengths]
    pool = sum(pages) + 3
    dtype = DTYPES[case["dtype"]]
    q = torch.randn(case["batch"], case["q_heads"], DIM, generator=g, device="cuda")
    q = (q * 1.2).to(dtype)
    center = None
    if case["center"]:
        center = torch.randn(case["batch"], case["kv_heads"], DIM, generator=g, device="cuda")
        center = (0.5 * center).to(dtype)
    order = torch.randperm(pool, generator=g, device="cuda")[:sum(pages)].int()
    records = torch.empty(pool, case["kv_heads"], RECORD, dtype=torch.uint8, device="cuda")
    parts = []
    for a, k, v in _cache_pages(case, g, pool):
        records[a:a + k[0].shape[0]] = _record(*k, *v)
        if keep:
            parts.append((k, v))
    state = {"case": case, "q": q, "center": center, "records": records, "indices": order,
             "indptr": torch.tensor([0] + pages).cumsum(0).int(),
             "last": torch.tensor([(n - 1) % PAGE + 1 if n else 0 for n in lengths],
                                  dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor(lengths, device="cuda"), "pages": max(pages)}
    return state, lengths, parts


def prepare(case, seed):
    if case["op"] == "rotary":
        g = torch.Generator("cuda").manual_seed(seed)
        q, k, _, _, _ = _packed_rows(case, g, case["tokens"], case["head_dim"],
                                     DTYPES[case["dtype"]])
        cos, sin = _tables(case, case["first"] + case["tokens"])
        positions = torch.arange(case["first"], case["first"] + case["tokens"],
                                 dtype=torch.int32, device="cuda")
        return {"case": case, "q": q, "k": k, "cos": cos, "sin": sin, "positions": positions,
                "q_out": torch.zeros(q.shape, dtype=q.dtype, device="cuda"),
                "k_out": torch.zeros(k.shape, dtype=k.dtype, device="cuda")}
    if case["op"] == "append":
        state = _append_inputs(case, seed)
        state["cos"], state["sin"] = _tables(case, case["context"] + case["max_new"])
        state["rotated"] = torch.zeros(state["q"].shape, dtype=state["q"].dtype, device="cuda")
        state["records"] = torch.zeros(state["pool_pages"], case["kv_heads"], RECORD,
                                       dtype=torch.uint8, device="cuda")
        if own:
            from pagegauge_b200.int4 import Int4PagePool
            from pagegauge_b200.runtime import load_append_extension
            state["extension"] = load_append_extension()
            state["pool"] = Int4PagePool(state["pool_pages"], case["kv_heads"],
                                         records=state["records"])
        return state
    state, _, _ = _attention_inputs(case, seed, False)
    state["out"] = torch.empty_like(state["q"])
    state["lse"] = torch.empty(state["q"].shape[:2], dtype=torch.float32, device="cuda")
    if own:
        from pagegauge_b200.wrapper import make_int4_wrapper, plan
        wrapper = make_int4_wrapper(workspace=torch.empty(64 << 20, dtype=torch.uint8,
                                                          device="cuda"))
        plan(wrapper, state["indptr"], state["indices"], state["last"], torch.uint8,
             num_qo_heads=case["q_heads"], num_kv_heads=case["kv_heads"])
        state["wrapper"] = wrapper
    return state


# ------------------------------------------------------------ plain forms
def _rotated(x, cos, sin, interleaved, adjoint):
    """Rows x [T, H, D] of 32 bits turned by cos, sin [T, pairs]; dimensions past the
    pairs stay.  The adjoint turns back."""
    cos, sin = cos[:, None], -sin[:, None] if adjoint else sin[:, None]
    pairs = cos.shape[-1]
    part, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part[..., :pairs], part[..., pairs:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _held(x):
    """The values that the 4-bit cache holds for rows x [T, H, 128] of 32 bits."""
    x = x.clamp(-HALF_MAX, HALF_MAX).unflatten(-1, (DIM // GROUP, GROUP))
    low = x.amin(-1, keepdim=True)
    s = ((x.amax(-1, keepdim=True) - low) * (1.0 / 15.0)).half().float()
    m = (low + 8.0 * s).half().float()
    inverse = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    z = ((x - m) * inverse).round().clamp(-8, 7)
    return (z * s + m).flatten(-2)


def _unpacked(records):
    """Keys and values [..., 16, 128] in 32 bits of records [..., 2560]."""
    lead = records.shape[:-1]
    nibbles = lambda b: torch.stack((b & 15, b >> 4), -1).flatten(-2)  # noqa: E731
    k = nibbles(records[..., :1024]).view(*lead, PAGE, 4, 4, 8).transpose(-3, -2)
    v = nibbles(records[..., 1024:2048]).view(*lead, 2, 2, 4, 8, 4, 4)
    v = v.transpose(-5, -4).transpose(-3, -2)
    out = []
    for z, meta in ((k, records[..., 2048:2304]), (v, records[..., 2304:])):
        meta = meta.contiguous().view(torch.float16).view(*lead, PAGE, 2, 4, 1).float()
        z = z.reshape(*lead, PAGE, 4, GROUP).float() - 8.0
        out.append((z * meta[..., 0, :, :] + meta[..., 1, :, :]).flatten(-2))
    return out


def _plain_append(state):
    case, dtype = state["case"], state["q"].dtype
    keep = state["slots"] >= 0
    at = state["positions"].long()
    cos, sin = state["cos"][at], state["sin"][at]
    turn = lambda x: _rotated(x.float(), cos, sin, case["interleaved"], False)  # noqa: E731
    q, k, v = turn(state["q"]), turn(state["k"]), state["v"].float()
    if state["rows"] is not None:
        k = k - state["k_center"].float()[state["rows"].long()]
        v = v - state["v_center"].float()[state["rows"].long()]
    mask = keep[:, None, None]
    zero = lambda x: torch.where(mask, x, torch.zeros_like(x)).to(dtype)  # noqa: E731
    return zero(q), zero(_held(k)), zero(_held(v))


def _plain_attention(state):
    case, q, indptr = state["case"], state["q"], state["indptr"].to("cuda", non_blocking=True)
    batch, hkv, group = q.shape[0], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    tokens = state["pages"] * PAGE
    if tokens == 0:
        out = torch.zeros_like(q)
        return out, torch.full(q.shape[:2], -math.inf, dtype=torch.float32, device="cuda")
    column = torch.arange(state["pages"], device="cuda")
    begin, end = indptr[:-1, None].long(), indptr[1:, None].long()
    place = (begin + column).clamp(max=state["indices"].numel() - 1)
    ids = torch.where(begin + column < end, state["indices"][place].long(), 0)
    k, v = _unpacked(state["records"][ids])  # [B, pages, Hkv, 16, 128]
    k, v = (x.transpose(1, 2).reshape(batch, hkv, tokens, DIM) for x in (k, v))
    rows = q.float().view(batch, hkv, group, DIM) * (DIM ** -0.5 * math.log2(math.e))
    score = rows @ k.transpose(-1, -2)
    here = torch.arange(tokens, device="cuda") < state["lengths"][:, None]
    here = here[:, None, None]
    score = torch.where(here, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, torch.zeros_like(top))
    p = torch.exp2(score - top)
    total = p.sum(-1, keepdim=True)
    some = total > 0
    out = (p @ v) / torch.where(some, total, torch.ones_like(total))
    if state["center"] is not None:
        out = torch.where(some, out + state["center"].float()[:, :, None], out)
    lse = torch.where(some, total.log2() + top, -math.inf)
    return out.reshape(q.shape).to(q.dtype), lse.reshape(q.shape[:2])


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        if own:
            from pagegauge_b200.rotary import apply_rotary
            return apply_rotary(state["q"], state["k"], state["cos"], state["sin"],
                                state["positions"], interleaved=case["interleaved"],
                                adjoint=case["adjoint"], query_out=state["q_out"],
                                key_out=state["k_out"])
        at = state["positions"].long()
        cos, sin = state["cos"][at], state["sin"][at]
        turn = lambda x: _rotated(x.float(), cos, sin, case["interleaved"],  # noqa: E731
                                  case["adjoint"]).to(x.dtype)
        return turn(state["q"]), turn(state["k"])
    if case["op"] == "append":
        if own:
            state["extension"].rope_append_int4(
                state["q"], state["k"], state["v"], state["cos"], state["sin"],
                state["positions"], state["slots"], state["rotated"], state["records"],
                key_center=state["k_center"], value_center=state["v_center"],
                center_rows=state["rows"], interleaved=case["interleaved"])
            key, value = state["pool"].read(state["slots"], dtype=state["q"].dtype)
            return state["rotated"], key, value
        return _plain_append(state)
    if own:
        return state["wrapper"].run(state["q"], state["records"], value_center=state["center"],
                                    out=state["out"], lse=state["lse"], return_lse=True)
    return _plain_attention(state)


# ------------------------------------------------------------ in 64 bits
def _turned_exactly(x, angle, scale, interleaved, adjoint):
    """Each pair as a complex number times scale * exp(i * angle)."""
    x = x.double()
    turn = torch.polar(torch.full_like(angle, scale), -angle if adjoint else angle)[:, None]
    pairs = angle.shape[-1]
    out = x.clone()
    first, second = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved
                     else (slice(0, pairs), slice(pairs, 2 * pairs)))
    y = torch.complex(x[..., first], x[..., second]) * turn
    out[..., first], out[..., second] = y.real, y.imag
    return out


def _held_exactly(x):
    """(z - 8) s + m of each group of 32 in 64 bits; s and m are float16 by definition."""
    groups = x.reshape(-1, GROUP).clamp(-HALF_MAX, HALF_MAX)
    low, high = groups.min(1).values, groups.max(1).values
    s = ((high - low) / 15).half().double()
    m = (low + 8 * s).half().double()
    z = torch.round((groups - m[:, None]) / torch.where(s > 0, s, 1.0)[:, None])
    z = torch.clamp(z, -8, 7) * (s > 0)[:, None]
    return (z * s[:, None] + m[:, None]).reshape(x.shape)


def exact(case, seed):
    if case["op"] == "attention":
        state, lengths, parts = _attention_inputs(case, seed, True)
        value = lambda side, i: torch.cat([p[side][i] for p in parts])  # noqa: E731
        held = [[value(side, i) for i in range(3)] for side in (0, 1)]
        group = case["q_heads"] // case["kv_heads"]
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(state["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        begin = state["indptr"].tolist()
        for r, n in enumerate(lengths):
            if n == 0:
                continue
            ids = state["indices"][begin[r]:begin[r + 1]].long()
            for h in range(case["kv_heads"]):
                k, v = (((z[ids, h].double() - 8).view(-1, 4, GROUP)
                         * s[ids, h].double().view(-1, 4, 1)
                         + m[ids, h].double().view(-1, 4, 1)).view(-1, DIM)[:n]
                        for z, s, m in held)
                heads = slice(h * group, (h + 1) * group)
                score = state["q"][r, heads].double() @ k.T / math.sqrt(DIM)
                out[r, heads] = torch.softmax(score, -1) @ v
                if state["center"] is not None:
                    out[r, heads] += state["center"][r, h].double()
                lse[r, heads] = torch.logsumexp(score, -1) / math.log(2)
        return out, lse
    inv, scale = _frequencies(case)
    if case["op"] == "rotary":
        state = prepare(case, seed)
        angle = state["positions"].double()[:, None] * inv.cuda()
        return tuple(_turned_exactly(state[x], angle, scale, case["interleaved"],
                                     case["adjoint"]) for x in ("q", "k"))
    state = _append_inputs(case, seed)
    angle = state["positions"].double()[:, None] * inv.cuda()
    q = _turned_exactly(state["q"], angle, scale, case["interleaved"], False)
    k = _turned_exactly(state["k"], angle, scale, case["interleaved"], False)
    v = state["v"].double()
    if case["center"]:
        k -= state["k_center"].double()[state["rows"].long()]
        v -= state["v_center"].double()[state["rows"].long()]
    skipped = state["slots"] < 0
    results = q, _held_exactly(k), _held_exactly(v)
    for x in results:
        x[skipped] = 0
    return results

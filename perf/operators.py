"""Performance cases of the query / key norm with rotation and of the 8-bit key / value cache.

Three kinds of case: ``rope`` (``qk_norm_rope``), ``store`` (``KVCache8.append`` and
the read-back of the blocks it touched) and ``attend`` (``KVCache8.attend``).
"""

import math

import torch

own = False

BLOCK = 64  # tokens of a cache block
DIM = 128   # head dim of the cache
TOP = 448.0  # largest e4m3 value
LEAST_EXPONENT = -60  # exponent of the scale of a block of zeros


def listed():
    return [
        # One new token of a 24-head model, norm over the whole row: latency only.
        dict(name="rope_token", kind="rope", batch=1, rows=1, heads=24, kv_heads=24, dim=128, over="row",
             interleaved=True, far=4096),
        # The DiT's joint sequence (360 video + 32 action rows) between its QKV projection and its attention.
        dict(name="rope_frame", kind="rope", batch=1, rows=392, heads=24, kv_heads=24, dim=128, over="row",
             interleaved=True, far=392),
        # Long prompts of a model with shared key heads, norm of each head, halves rotated, far positions.
        dict(name="rope_long", kind="rope", batch=2, rows=8191, heads=32, kv_heads=8, dim=128, over="head",
             interleaved=False, far=131072),
        # A decode step of 16 sequences: each adds one token to a block that is partly full.
        dict(name="store_token", kind="store", batch=16, rows=1, kv_heads=8, longest=4001, ragged=True),
        # The DiT's text context and prefix of four requests.
        dict(name="store_context", kind="store", batch=4, rows=513, kv_heads=24, longest=121, ragged=True),
        # A long prompt stored at once.
        dict(name="store_prompt", kind="store", batch=2, rows=8001, kv_heads=24, longest=0, ragged=False),
        # One token over a short cache: latency.
        dict(name="attend_token_short", kind="attend", batch=1, rows=1, heads=24, kv_heads=24, longest=577,
             ragged=False, causal=True),
        # A decode step of 16 ragged sequences with shared key heads: bandwidth.
        dict(name="attend_token_batch", kind="attend", batch=16, rows=1, heads=32, kv_heads=8, longest=16381,
             ragged=True, causal=True),
        # The 32 action rows over a history of observations.
        dict(name="attend_action", kind="attend", batch=1, rows=32, heads=24, kv_heads=24, longest=4100,
             ragged=False, causal=False),
        # The video rows over a padded text context.
        dict(name="attend_context", kind="attend", batch=2, rows=360, heads=24, kv_heads=24, longest=513,
             ragged=True, causal=False),
        # A prompt's tail over what is cached of it, causal, shared key heads.
        dict(name="attend_prompt", kind="attend", batch=2, rows=2047, heads=32, kv_heads=8, longest=6143,
             ragged=True, causal=True),
        # The joint sequence over a long history: the largest.
        dict(name="attend_history", kind="attend", batch=1, rows=392, heads=24, kv_heads=24, longest=32768,
             ragged=False, causal=False),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    kind = rng.choice(("rope", "store", "attend"))
    heads, kv_heads = rng.choice(((24, 24), (32, 8), (16, 16), (12, 4), (40, 8), (8, 1), (28, 4)))
    if kind == "rope":
        batch = rng.choice((1, 1, 2, 3, 8))
        return dict(kind=kind, batch=batch, rows=_spread(rng, 1, 16384 // batch), heads=heads, kv_heads=kv_heads,
                    dim=rng.choice((64, 128, 128, 256)), over=rng.choice(("row", "head")),
                    interleaved=rng.random() < 0.5, far=_spread(rng, 16384, 131072))
    batch = rng.choice((1, 2, 3, 5, 16))
    longest = _spread(rng, 1, 32768 // batch)
    if kind == "store":
        return dict(kind=kind, batch=batch, rows=_spread(rng, 1, 16000 // batch), kv_heads=kv_heads,
                    longest=longest if rng.random() < 0.7 else 0, ragged=rng.random() < 0.5)
    # Query rows bounded so that no drawn case exceeds the work of attend_history.
    most = max(1, min(2048, 392 * 32768 * 24 // (2 * batch * longest * heads)))
    rows = 1 if rng.random() < 0.35 else _spread(rng, 1, most)
    return dict(kind=kind, batch=batch, rows=rows, heads=heads, kv_heads=kv_heads, longest=longest,
                ragged=rng.random() < 0.5, causal=rng.random() < 0.5)


def _lengths(case):
    """Cached rows of each sequence: a fixed spread below the longest."""
    longest = case["longest"]
    return [longest - (b * 7919) % (longest // 2 + 1) if case["ragged"] else longest for b in range(case["batch"])]


def _counts(case):
    """Rows that each sequence of a store adds (a ragged batch is padded)."""
    return [case["rows"] - (b * 31) % (case["rows"] // 3 + 1) if case["ragged"] else case["rows"]
            for b in range(case["batch"])]


def _exponent(top):
    """The least e with top <= 448 * 2^e, at least LEAST_EXPONENT (top: float32)."""
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > 0.875)
    return torch.where(top > 0, e, LEAST_EXPONENT).clamp(min=LEAST_EXPONENT)


def _power(e):
    """2^e in float32, exactly (-126 <= e <= 127)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x, e):
    """x / 2^e in e4m3; e broadcasts over x."""
    return (x * _power(-e)).clamp(-TOP, TOP).to(torch.float8_e4m3fn)


def _fp8_rows(blocks, index):
    return blocks.view(torch.uint8)[index].view(torch.float8_e4m3fn).float()


def _filled(shape, generator, device):
    """Blocks of e4m3 values and their scales, as a cache holds them: activations whose size varies by block."""
    size = torch.exp2(torch.randint(-2, 3, (shape[0], shape[1], 1, 1), generator=generator, device=device).float())
    x = torch.empty(shape, device=device).normal_(generator=generator) * size
    e = _exponent(x.abs().amax((2, 3)))
    return _quantise(x, e[:, :, None, None]), _power(e)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)

    def rows(*shape):
        return torch.randn(shape, device=device, generator=g).bfloat16()

    state = dict(case)
    batch, n, kv_heads = case["batch"], case["rows"], case["kv_heads"]
    if case["kind"] == "rope":
        heads, dim = case["heads"], case["dim"]
        packed = rows(batch, n, (heads + 2 * kv_heads) * dim)  # queries, keys and values of one projection
        state["q"], state["k"] = packed[..., :heads * dim], packed[..., heads * dim:(heads + kv_heads) * dim]
        wide = case["over"] == "row"
        state["q_weight"] = (1 + 0.1 * torch.randn(heads * dim if wide else dim, device=device, generator=g)).bfloat16()
        state["k_weight"] = (1 + 0.1 * torch.randn(kv_heads * dim if wide else dim, device=device,
                                                   generator=g)).bfloat16()
        inverse = 10000.0 ** (-torch.arange(dim // 2, device=device, dtype=torch.float64) / (dim // 2))
        angles = torch.arange(case["far"], device=device, dtype=torch.float64)[:, None] * inverse
        state["rope"] = torch.polar(torch.ones_like(angles), angles).to(torch.complex64)
        first = torch.randint(0, case["far"] - n + 1, (batch, 1), device=device, generator=g)
        state["positions"] = (first + torch.arange(n, device=device)).to(torch.int32)
        return state

    lengths = _lengths(case)
    room = max(lengths) + (n if case["kind"] == "store" else 0)
    per = -(-room // BLOCK)
    order = torch.randperm(batch * per, device=device, generator=g)
    state["block_table"] = order.to(torch.int32).view(batch, per)
    shape = (batch * per, kv_heads, BLOCK, DIM)
    state["keys"], state["key_scales"] = _filled(shape, g, device)
    state["values"], state["value_scales"] = _filled(shape, g, device)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    if case["kind"] == "store":
        state["at"] = state["lengths"].clone()
        state["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=device)
        state["first"] = state["at"] // BLOCK * BLOCK  # the first row of the first block that changes
        state["k"], state["v"] = rows(batch, n, kv_heads * DIM), rows(batch, n, kv_heads * DIM)
    else:
        state["q"] = rows(batch, n, case["heads"] * DIM)
    if own:  # the program's handle of the same blocks
        from waminfer_b200.cache import KVCache8

        state["cache"] = KVCache8.of(state["keys"], state["values"], state["key_scales"], state["value_scales"],
                                     state["block_table"], state["lengths"])
    return state


def run(state):
    if state["kind"] == "rope":
        return _rope(state)
    return _store(state) if state["kind"] == "store" else _attend(state)


def _turned(x, heads, weight, cos, sin, eps, interleaved):
    """Norm and rotation of x [batch, rows, heads * dim] in 32 bits."""
    batch, n, width = x.shape
    dim = width // heads
    x = x.float()
    if weight.numel() == dim:
        x = x.view(batch, n, heads, dim)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    x = x.view(batch, n, heads, dim)
    cos, sin = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1)
    else:
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return y.reshape(batch, n, width).bfloat16()


def _rope(s):
    if own:
        from waminfer_b200.rope import qk_norm_rope

        return qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["rope"], s["positions"], s["heads"],
                            s["kv_heads"], 1e-6, s["interleaved"])
    at = s["rope"][s["positions"].long()]
    q = _turned(s["q"], s["heads"], s["q_weight"], at.real, at.imag, 1e-6, s["interleaved"])
    k = _turned(s["k"], s["kv_heads"], s["k_weight"], at.real, at.imag, 1e-6, s["interleaved"])
    return q, k


def _stored(s, x, blocks, scales, ids, row, end):
    """Puts the new rows of x into the blocks `ids` [batch, places] whose rows are `row` [batch, places, 64]."""
    batch, many = ids.shape
    at, kv_heads = s["at"][:, None, None], s["kv_heads"]
    old, new = row < at, (row >= at) & (row < end[:, None, None])
    source = (row - at).clamp(0, s["rows"] - 1).long().view(batch, -1, 1)
    x = x.gather(1, source.expand(-1, -1, x.shape[2])).float()
    x = x.view(batch, many, BLOCK, kv_heads, DIM).transpose(2, 3)
    fresh = new[:, :, None, :, None]
    e = _exponent(torch.where(fresh & x.isfinite(), x.abs(), 0.0).amax((3, 4)))
    e = torch.where(old.any(2)[:, :, None], torch.maximum(torch.frexp(scales[ids])[1] - 1, e), e)
    held = torch.where(fresh, x, _fp8_rows(blocks, ids) * scales[ids][..., None, None])
    codes = _quantise(held, e[..., None, None]).view(torch.uint8)
    codes = torch.where((old | new)[:, :, None, :, None], codes, blocks.view(torch.uint8)[ids])
    blocks.view(torch.uint8)[ids] = codes  # a place that repeats a sequence's last block repeats its values
    scales[ids] = _power(e)


def _read(s, blocks, scales, ids, row, inside):
    """Rows `row` [batch, rows] of each sequence in 16 bits, zeros where not inside."""
    y = blocks.view(torch.uint8)[ids, :, (row % BLOCK).long()].view(torch.float8_e4m3fn).float()
    y = torch.where(inside[:, :, None, None], y * scales[ids][..., None], 0.0)
    return y.flatten(2).bfloat16()


def _store(s):
    span = s["rows"] + BLOCK - 1  # from the first changed block's first row to the last new row
    if own:
        s["cache"].append(s["k"], s["v"], counts=s["counts"], at=s["at"])
        k, v = s["cache"].read(span, start=s["first"])
        return k, v, s["lengths"]
    device, table = s["k"].device, s["block_table"].long()
    end = s["at"] + s["counts"]
    place = (s["at"] // BLOCK)[:, None] + torch.arange(-(-span // BLOCK), device=device)
    place = torch.minimum(place, ((end - 1) // BLOCK)[:, None])
    ids = table.gather(1, place.long())
    row = place[:, :, None] * BLOCK + torch.arange(BLOCK, device=device)
    _stored(s, s["k"], s["keys"], s["key_scales"], ids, row, end)
    _stored(s, s["v"], s["values"], s["value_scales"], ids, row, end)
    s["lengths"].copy_(end)
    row = s["first"][:, None] + torch.arange(span, device=device)
    ids = table.gather(1, (row // BLOCK).clamp(max=table.shape[1] - 1).long())
    inside = row < end[:, None]
    k = _read(s, s["keys"], s["key_scales"], ids, row, inside)
    v = _read(s, s["values"], s["value_scales"], ids, row, inside)
    return k, v, s["lengths"]


def _attend(s):
    if own:
        return s["cache"].attend(s["q"], s["heads"], causal=s["causal"])
    batch, n, heads, kv_heads = s["batch"], s["rows"], s["heads"], s["kv_heads"]
    ids = s["block_table"].long()
    group, room = heads // kv_heads, ids.shape[1] * BLOCK
    k = (_fp8_rows(s["keys"], ids) * s["key_scales"][ids][..., None, None]).transpose(1, 2)
    v = (_fp8_rows(s["values"], ids) * s["value_scales"][ids][..., None, None]).transpose(1, 2)
    k, v = k.reshape(batch, kv_heads, room, DIM), v.reshape(batch, kv_heads, room, DIM)
    q = s["q"].float().view(batch, n, kv_heads, group, DIM).permute(0, 2, 3, 1, 4)
    score = q.reshape(batch, kv_heads, group * n, DIM) @ k.transpose(2, 3) * DIM ** -0.5
    seen = s["lengths"][:, None].expand(batch, n)
    if s["causal"]:
        seen = seen - n + 1 + torch.arange(n, device=q.device)
    seen = torch.arange(room, device=q.device) < seen[..., None]  # [batch, rows, keys]
    seen = seen[:, None, None].expand(-1, -1, group, -1, -1).reshape(batch, 1, group * n, room)
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = weight @ v / torch.where(total > 0, total, 1.0)
    out = out.view(batch, kv_heads, group, n, DIM).permute(0, 3, 1, 2, 4)
    return out.reshape(batch, n, heads * DIM).bfloat16()


def work(case):
    batch, n, kv_heads = case["batch"], case["rows"], case["kv_heads"]
    if case["kind"] == "rope":
        elements = batch * n * (case["heads"] + kv_heads) * case["dim"]
        # Each element in and out, the table's row and the position of each token; weights.
        weights = (case["heads"] + kv_heads if case["over"] == "row" else 2) * case["dim"]
        return {"bytes": 4 * elements + batch * n * (case["dim"] * 4 + 4) + 2 * weights, "flops": 8 * elements}
    if case["kind"] == "store":
        new, span = sum(_counts(case)), n + BLOCK - 1
        # New rows in (16 bits) and out (8 bits); every row of the read-back in (8 bits) where it exists, out (16).
        there = sum(a % BLOCK + c for a, c in zip(_lengths(case), _counts(case)))
        row = 2 * kv_heads * DIM
        return {"bytes": row * (3 * new + there + 2 * batch * span), "flops": 4 * row * new}
    lengths = _lengths(case)
    heads = case["heads"]
    pairs = sum(sum(max(0, m - n + 1 + i) for i in range(n)) if case["causal"] else m * n for m in lengths)
    cached = sum(lengths) * kv_heads * 2 * DIM + sum(-(-m // BLOCK) for m in lengths) * (8 * kv_heads + 4)
    return {"bytes": cached + 4 * batch * n * heads * DIM, "flops": 4 * DIM * heads * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "store": _exact_store, "attend": _exact_attend}[case["kind"]](s)


def _exact_rope(s):
    turn = s["rope"].to(torch.complex128)[s["positions"].long()]
    out = []
    for x, w, heads in ((s["q"], s["q_weight"], s["heads"]), (s["k"], s["k_weight"], s["kv_heads"])):
        x, w = x.double(), w.double()
        whole = x.reshape(x.shape[0], x.shape[1], heads, -1)
        dim = whole.shape[-1]
        if s["over"] == "row":
            whole = whole / ((x ** 2).sum(-1) / x.shape[2] + 1e-6).sqrt()[:, :, None, None] * w.view(heads, dim)
        else:
            whole = whole / ((whole ** 2).sum(-1) / dim + 1e-6).sqrt()[..., None] * w
        if s["interleaved"]:
            z = torch.view_as_complex(whole.reshape(*whole.shape[:-1], dim // 2, 2).contiguous())
            y = torch.view_as_real(z * turn[:, :, None]).flatten(-2)
        else:
            z = torch.complex(whole[..., :dim // 2].contiguous(), whole[..., dim // 2:].contiguous())
            z = z * turn[:, :, None]
            y = torch.cat((z.real, z.imag), -1)
        out.append(y.reshape(x.shape))
    return tuple(out)


def _round_e4m3(x):
    """The nearest e4m3 value (3 fraction bits, least step 2^-9, ties to even), from the format's definition."""
    size = x.abs()
    power = torch.floor(torch.log2(torch.where(size > 0, size, 1.0)))
    power = torch.where(torch.exp2(power) > size, power - 1, power).clamp(min=-6)
    step = torch.exp2(power - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _exact_store(s):
    batch, span = s["batch"], s["rows"] + BLOCK - 1
    at, counts, table = s["at"].tolist(), s["counts"].tolist(), s["block_table"].tolist()
    out = [torch.zeros(batch, span, s["kv_heads"], DIM, dtype=torch.float64, device=s["k"].device) for _ in range(2)]
    for y, x, blocks, scales in ((out[0], s["k"], s["keys"], s["key_scales"]),
                                 (out[1], s["v"], s["values"], s["value_scales"])):
        x = x.double().view(batch, s["rows"], s["kv_heads"], DIM)
        for b in range(batch):
            first, end = at[b] // BLOCK * BLOCK, at[b] + counts[b]
            for low in range(first, end, BLOCK):
                a, z = max(low, at[b]), min(low + BLOCK, end)
                fresh = x[b, a - at[b]:z - at[b]]
                # The least power of two whose 448-fold holds every value.
                need = fresh.abs().amax((0, 2)) / 448
                power = torch.log2(need).round()
                need = torch.where(torch.exp2(power) < need, power + 1, power).clamp(min=-60)
                if low < at[b]:
                    scale = scales[table[b][low // BLOCK]].double()
                    held = blocks[table[b][low // BLOCK]].double()[:, :a - low].transpose(0, 1) * scale[None, :, None]
                    need = torch.maximum(need, torch.log2(scale).round())  # scales are powers of two
                    fresh = torch.cat((held, fresh))
                unit = torch.exp2(need)[None, :, None]
                y[b, low - first:z - first] = _round_e4m3(fresh / unit) * unit
    ends = s["at"] + s["counts"]
    return out[0].flatten(2), out[1].flatten(2), ends


def _exact_attend(s):
    batch, n, heads, kv_heads = s["batch"], s["rows"], s["heads"], s["kv_heads"]
    group = heads // kv_heads
    out = torch.zeros(batch, n, heads, DIM, dtype=torch.float64, device=s["q"].device)
    q = s["q"].double().view(batch, n, heads, DIM)
    lengths, table = s["lengths"].tolist(), s["block_table"].long()
    for b in range(batch):
        for h in range(kv_heads):
            ids = table[b, :-(-lengths[b] // BLOCK)]
            k = (s["keys"][ids, h].double() * s["key_scales"][ids, h].double()[:, None, None]).view(-1, DIM)
            v = (s["values"][ids, h].double() * s["value_scales"][ids, h].double()[:, None, None]).view(-1, DIM)
            k, v = k[:lengths[b]], v[:lengths[b]]
            low = max(0, n - lengths[b]) if s["causal"] else 0  # rows before it see nothing
            score = torch.einsum("igd,jd->igj", q[b, low:, h * group:(h + 1) * group], k) / math.sqrt(DIM)
            if s["causal"]:
                last = lengths[b] - n + torch.arange(low, n, device=k.device)
                hidden = torch.arange(lengths[b], device=k.device)[None] > last[:, None]
                score = score.masked_fill(hidden[:, None], -math.inf)
            out[b, low:, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v
    return out.view(batch, n, heads * DIM)

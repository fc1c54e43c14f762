"""GPU: the 8-bit key / value cache (``waminfer_b200/cache.py``) against the formulas in 64 bits.

Stored values, scales and lengths are equal to the reference's: division by a
power of two is exact, and rounding to e4m3 has one answer.

Attention.  The reference takes the held values exactly.  The kernel's error:
the result's rounding, 2^-8 |out|; the probabilities in f16, 2^-11 of the sum
A = sum p |v| / sum p; scores in fp32, 128 products each (2^-23 of a partial
sum an addition, whichever way the tensor core rounds): 2^-16 B with B the
largest sum |q||k| / sqrt(128), twice (numerator and denominator); sums over N
keys in fp32: N 2^-23 A.  exp2 and its argument are within 2^-20."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BLOCK, DIM = 64, 128


# ------------------------------------------------------------- reference (CPU, float64)
def e4m3(x):
    """The nearest e4m3 value, ties to even, beyond 448 to 448; NaN stays."""
    power = torch.frexp(x)[1].to(torch.float64) - 1
    step = torch.exp2(power.clamp(min=-6) - 3)
    y = torch.round(torch.nan_to_num(x, nan=0.0, posinf=1e4, neginf=-1e4) / step.nan_to_num(1.0)) * step
    y = torch.where(x.isinf(), torch.sign(x) * 448, y.clamp(-448, 448))
    return torch.where(x.isnan(), x, y)


def need(x):
    """Least e >= -60 with max finite |x| <= 448 * 2^e."""
    top = torch.where(x.isfinite(), x.abs(), 0.0).max().item() if x.numel() else 0.0
    e = -60
    while top > 448 * 2.0 ** e:
        e += 1
    return e


class Model:
    """The cache in float64: values as they stand (code * scale) and exponents."""

    def __init__(self, cache):
        self.table = cache.block_table.cpu().tolist()
        self.lengths = cache.lengths.cpu().tolist()
        self.codes = [t.cpu().float().double() for t in (cache.keys, cache.values)]
        self.exps = [torch.log2(t.cpu().double()).round() for t in (cache.key_scales, cache.value_scales)]

    def append(self, k, v, counts=None, at=None):
        heads = self.codes[0].shape[1]
        for b, table in enumerate(self.table):
            n = k.shape[1] if counts is None else max(0, min(counts[b], k.shape[1]))
            start = self.lengths[b] if at is None else at[b]
            end = start + n
            if not 0 <= start <= self.lengths[b] or end > len(table) * BLOCK:
                continue
            places = [i for i in range(start // BLOCK, -(-end // BLOCK))] if end > start else []
            if any(not 0 <= table[i] < self.codes[0].shape[0] for i in range(start // BLOCK, -(-end // BLOCK))):
                continue
            for codes, exps, x in ((self.codes[0], self.exps[0], k), (self.codes[1], self.exps[1], v)):
                x = x[b].cpu().double().view(-1, heads, DIM)
                for i in places:
                    lo, hi = max(start - i * BLOCK, 0), min(end - i * BLOCK, BLOCK)
                    for h in range(heads):
                        new = x[i * BLOCK + lo - start:i * BLOCK + hi - start, h]
                        e = need(new)
                        if lo:
                            old = int(exps[table[i], h])
                            e = max(e, old)
                            codes[table[i], h, :lo] = e4m3(codes[table[i], h, :lo] * 2.0 ** (old - e))
                        exps[table[i], h] = e
                        codes[table[i], h, lo:hi] = e4m3(new * 2.0 ** -e)
            self.lengths[b] = end

    def rows(self, which, b, h):
        ids = self.table[b][:-(-self.lengths[b] // BLOCK)]
        y = self.codes[which][ids, h] * torch.exp2(self.exps[which][ids, h])[:, None, None]
        return y.reshape(-1, DIM)[:self.lengths[b]]

    def same(self, cache):
        assert cache.lengths.tolist() == self.lengths
        for mine, theirs in ((self.codes, (cache.keys, cache.values)), (self.exps, (cache.key_scales, cache.value_scales))):
            for a, t in zip(mine, theirs):
                t = t.cpu().float().double()
                t = torch.log2(t).round() if t.dim() == 2 else t
                assert torch.equal(torch.nan_to_num(a, nan=1e9), torch.nan_to_num(t, nan=1e9))


def rows(g, *shape, size=1.0):
    return (torch.randn(*shape, device=g.device, generator=g) * size).bfloat16()


def make(dev, seed, batch, kv_heads, lengths, spread=0, extra=0, capacity=None):
    """A cache with blocks in random order, filled through float64, stale NaN behind every sequence's last row."""
    from waminfer_b200.cache import KVCache8

    g = torch.Generator(device=dev).manual_seed(seed)
    width = -(-(capacity or max(max(lengths), 1)) // BLOCK)
    pool = batch * width + extra
    keys = torch.empty(pool, kv_heads, BLOCK, DIM, device=dev).normal_(generator=g) * 60
    values = torch.empty(pool, kv_heads, BLOCK, DIM, device=dev).normal_(generator=g) * 60
    table = torch.randperm(pool, device=dev, generator=g)[:batch * width].view(batch, width).to(torch.int32)
    scale = lambda: torch.exp2(torch.randint(-6 - spread, -5 + spread, (pool, kv_heads), device=dev,  # noqa: E731
                                             generator=g).float())
    row = torch.arange(width * BLOCK, device=dev).view(width, BLOCK)
    for b in range(batch):
        stale = (row >= lengths[b])[:, None, :, None].expand(-1, kv_heads, -1, DIM)
        for t in (keys, values):
            t[table[b].long()] = torch.where(stale, float("nan"), t[table[b].long()])
    to = lambda t: t.clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    # Keys stay within a few binades (scores within exp's range), values spread further.
    cache = KVCache8.of(to(keys), to(values), torch.exp2(torch.randint(-7, -4, (pool, kv_heads), device=dev,
                                                                      generator=g).float()), scale(),
                        table, torch.tensor(lengths, dtype=torch.int32, device=dev))
    return cache, g


# ------------------------------------------------------------- storing
@pytest.mark.parametrize("batch,kv_heads,starts,n,size", [
    (1, 1, [0], 1, 1.0),
    (1, 3, [0], 64, 1.0),
    (2, 2, [63, 64], 1, 8.0),      # fills a block with growth; opens one
    (2, 2, [10, 100], 1, 0.01),    # no growth
    (3, 1, [1, 65, 128], 130, 3.0),
    (2, 4, [0, 37], 513, 1.0),
    (1, 1, [5], 200, 1e30),        # the held rows vanish under the new scale
    (1, 2, [70], 3, 1e-30),
])
def test_append(cuda_device, batch, kv_heads, starts, n, size):
    cache, g = make(cuda_device, n + batch, batch, kv_heads, starts, capacity=max(starts) + n + 1, extra=3)
    model = Model(cache)
    packed = rows(g, batch, n, 2 * kv_heads * DIM + 8, size=size)  # rows of a wider projection
    k, v = packed[..., :kv_heads * DIM], packed[..., kv_heads * DIM:2 * kv_heads * DIM]
    cache.append(k, v)
    model.append(k, v)
    model.same(cache)
    assert cache.status() == 0
    # One token at a time gives the same lengths, and values as the rule says.
    for _ in range(3):
        k, v = rows(g, batch, 1, kv_heads * DIM, size=size * 3), rows(g, batch, 1, kv_heads * DIM, size=size * 3)
        cache.append(k, v)
        model.append(k, v)
    model.same(cache)


def test_append_special_values(cuda_device):
    """Zeros, infinities, NaN, the format's borders and ties, the scale's floor."""
    from waminfer_b200.cache import KVCache8

    cache = KVCache8(1, 640, 2, cuda_device)
    model = Model(cache)
    k = torch.zeros(1, 320, 256, device=cuda_device, dtype=torch.bfloat16)
    v = k.clone()
    k[0, 64, :4] = torch.tensor([448.0, 450.0, -464.0, 1.0])
    k[0, 65, 128:132] = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.001])
    ties = torch.arange(128, device=cuda_device) / 64 + 1  # every tie between neighbouring fractions
    v[0, 128, :128], v[0, 129, :128] = ties, -ties * 2.0 ** -9
    v[0, 130, :128] = ties * 2.0 ** -16  # into the subnormals of the block's scale
    v[0, 192, :2] = torch.tensor([1e-25, 3e38])
    k[0, 256, :2] = torch.tensor([1e-38, 1e-39])
    v[0, 256] = float("nan")
    cache.append(k, v)
    model.append(k, v)
    model.same(cache)
    assert cache.key_scales[0, 0].item() == 2.0 ** -60  # a block of zeros
    more = k[:, 64:65] * 0 + 5
    cache.append(more, more)
    model.append(more, more)
    model.same(cache)


def test_append_ragged_replaced_and_refused(cuda_device):
    cache, g = make(cuda_device, 11, 5, 2, [0, 70, 130, 64, 200], capacity=256, extra=2)
    model = Model(cache)
    k, v = rows(g, 5, 100, 256), rows(g, 5, 100, 256)
    k[:, 90:] = float("nan")  # padding that no count reaches
    counts = [0, 90, 1, 64, 56]
    cache.append(k, v, counts=torch.tensor(counts, dtype=torch.int32, device=cuda_device))
    model.append(k, v, counts)
    model.same(cache)
    assert cache.status() == 0 and cache.lengths.tolist() == [0, 160, 131, 128, 256]
    # From an earlier row on; the scales of blocks whose rows all go start anew.
    at = [0, 64, 130, 5, 255]
    k, v = rows(g, 5, 1, 256, size=0.01), rows(g, 5, 1, 256, size=100.0)
    cache.append(k, v, at=torch.tensor(at, dtype=torch.int32, device=cuda_device))
    model.append(k, v, at=at)
    model.same(cache)
    assert cache.lengths.tolist() == [1, 65, 131, 6, 256] and cache.status() == 0
    # Refused, each sequence for itself: full, behind a gap, a negative start, a bad block id; the fifth goes in.
    cache.lengths[4] = 20
    cache.block_table[3, 0] = 99
    model.lengths[4], model.table[3][0] = 20, 99
    at = [2, -1, 131, 6, 20]
    k, v = rows(g, 5, 130, 256), rows(g, 5, 130, 256)
    cache.append(k, v, at=torch.tensor(at, dtype=torch.int32, device=cuda_device))
    model.append(k, v, at=at)
    model.same(cache)
    assert cache.lengths.tolist() == [1, 65, 131, 6, 150]
    assert cache.status() == 2 and cache.status() == 0  # WAMFFN_DEV_BAD_INDEX, then cleared


@pytest.mark.parametrize("count,start", [(1, 0), (200, 0), (70, 63), (33, [0, 1, 64]), (128, [-5, 500, 100])])
def test_read(cuda_device, count, start):
    cache, _ = make(cuda_device, count, 3, 2, [0, 65, 190], spread=20)
    model = Model(cache)
    starts = start if isinstance(start, list) else [start] * 3
    arg = torch.tensor(start, dtype=torch.int32, device=cuda_device) if isinstance(start, list) else start
    got = cache.read(count, arg)
    for which, y in enumerate(got):
        assert y.shape == (3, count, 2 * DIM) and y.dtype == torch.bfloat16
        for b in range(3):
            for h in range(2):
                held = model.rows(which, b, h)
                expect = torch.zeros(count, DIM, dtype=torch.float64)
                for i in range(count):
                    if 0 <= starts[b] + i < held.shape[0]:
                        expect[i] = held[starts[b] + i]
                assert torch.equal(y[b, :, h * DIM:(h + 1) * DIM].cpu().double(), expect)


# ------------------------------------------------------------- attention
def attention(model, q, heads, causal):
    """(out, A, B) of the module's tolerance, float64."""
    batch, nq, _ = q.shape
    kv_heads = model.codes[0].shape[1]
    group = heads // kv_heads
    q = q.cpu().double().view(batch, nq, heads, DIM)
    out, absolute = torch.zeros(batch, nq, heads, DIM, dtype=torch.float64), torch.zeros(batch, nq, heads, DIM,
                                                                                        dtype=torch.float64)
    bound = torch.zeros(batch, nq, heads, 1, dtype=torch.float64)
    for b in range(batch):
        n = model.lengths[b]
        if not n:
            continue
        seen = torch.full((nq,), n) if not causal else (n - nq + 1 + torch.arange(nq)).clamp(min=0)
        hidden = torch.arange(n)[None] >= seen[:, None]
        for h in range(heads):
            k, v = model.rows(0, b, h // group), model.rows(1, b, h // group)
            s = (q[b, :, h] @ k.T / math.sqrt(DIM)).masked_fill(hidden, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            if v.isfinite().all():
                out[b, :, h], absolute[b, :, h] = p @ v, p @ v.abs()
            else:  # a hidden value is not part of the sum, whatever it is
                for i in range(nq):
                    out[b, i, h] = p[i, :seen[i]] @ v[:seen[i]]
                    absolute[b, i, h] = p[i, :seen[i]] @ v[:seen[i]].abs()
            bound[b, :, h] = (q[b, :, h].nan_to_num().abs() @ k.nan_to_num().abs().T).amax(-1, keepdim=True) / math.sqrt(DIM)
    return out.flatten(2), absolute.flatten(2), bound.expand(-1, -1, -1, DIM).flatten(2)


def close(got, ref, keys):
    out, absolute, bound = ref
    got = got.cpu().double()
    wrong = int((got.isnan() != out.isnan()).sum())
    assert not wrong, wrong
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -11 + 2 * 2.0 ** -16 * bound + keys * 2.0 ** -23 + 2.0 ** -20) * absolute
    off = torch.where(out.isnan(), 0.0, (got - out).abs() - tol)
    assert off.max().item() <= 0, (off.max().item(), tol.flatten()[off.argmax()].item())


CASES = [  # batch, nq, heads, kv_heads, lengths, causal
    (1, 1, 1, 1, [1], False),
    (1, 1, 24, 24, [577], True),
    (4, 1, 8, 2, [0, 1, 64, 1000], True),
    (3, 3, 5, 1, [31, 32, 33], True),
    (2, 16, 4, 4, [63, 65], False),
    (2, 5, 4, 1, [300, 2], True),       # 20 packed rows, the first rows of a short sequence see nothing
    (1, 32, 6, 3, [4100], False),
    (2, 33, 3, 3, [129, 40], True),
    (1, 7, 28, 4, [700], True),         # 49 packed rows
    (2, 65, 2, 2, [257, 0], False),
    (2, 130, 4, 2, [400, 100], True),
    (1, 392, 3, 3, [513], False),
    (1, 257, 8, 1, [1111], True),
]


@pytest.mark.parametrize("batch,nq,heads,kv_heads,lengths,causal", CASES)
def test_attend(cuda_device, batch, nq, heads, kv_heads, lengths, causal):
    cache, g = make(cuda_device, nq + heads, batch, kv_heads, lengths, spread=3, extra=2)
    q = rows(g, batch, nq, heads * DIM)
    out = cache.attend(q, heads, causal=causal)
    assert cache.status() == 0
    close(out, attention(Model(cache), q, heads, causal), max(lengths))
    assert torch.equal(out, cache.attend(q, heads, causal=causal))  # the same bits again


@pytest.mark.parametrize("nq,heads,kv_heads,lengths,causal", [
    (1, 1, 1, [9000], True), (4, 2, 2, [8200, 10], True), (30, 1, 1, [9000], False), (150, 2, 1, [7000, 0], True),
    (3, 8, 1, [130, 9001], False)])
def test_attend_in_parts(cuda_device, nq, heads, kv_heads, lengths, causal):
    """Few rows over long sequences: parts of the keys through the workspace, some of them empty; and the same
    call through the C entry without a workspace."""
    import ctypes

    from waminfer_b200 import _lib

    cache, g = make(cuda_device, nq, len(lengths), kv_heads, lengths, spread=2)
    q = rows(g, len(lengths), nq, heads * DIM)
    out = cache.attend(q, heads, causal=causal)
    assert any(cache._needs.values())  # the call was cut into parts
    ref = attention(Model(cache), q, heads, causal)
    close(out, ref, max(lengths))
    whole = torch.full_like(out, float("nan"))
    args = _lib.CacheAttentionArgs(cache._view, _lib.RowsView(q.data_ptr(), q.stride(1), q.stride(0)), whole.data_ptr(),
                                   None, 0, nq, heads, causal, 0)
    _lib.launch(_lib.lib().wamffn_cache_attention, 0, ctypes.byref(args))
    close(whole, ref, max(lengths))
    assert cache.status() == 0


@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("nq,heads,kv_heads,lengths", [(1, 4, 2, [1000, 40]), (20, 2, 2, [300, 1]), (40, 4, 2, [500, 90])])
def test_attend_key_split(cuda_device, split, nq, heads, kv_heads, lengths):
    cache, g = make(cuda_device, split, 2, kv_heads, lengths, spread=2)
    q = rows(g, 2, nq, heads * DIM)
    close(cache.attend(q, heads, causal=True, key_split=split), attention(Model(cache), q, heads, True), max(lengths))


@pytest.mark.parametrize("nq,heads,kv_heads,lengths,causal", [
    (257, 8, 1, [1111], True), (130, 4, 4, [3000, 900], False), (300, 16, 2, [2000], True), (2, 8, 2, [5000, 3], True),
    (9, 6, 2, [777, 64], False), (60, 3, 3, [1500], True)])
def test_attend_gives_the_same_bits_again(cuda_device, nq, heads, kv_heads, lengths, causal):
    """Steps, stages and partial results meet in a fixed order: forty runs back to back, one result."""
    cache, g = make(cuda_device, nq, len(lengths), kv_heads, lengths, spread=3)
    q = rows(g, len(lengths), nq, heads * DIM)
    runs = [cache.attend(q, heads, causal=causal) for _ in range(40)]
    assert all(torch.equal(runs[0], r) for r in runs[1:])
    close(runs[0], attention(Model(cache), q, heads, causal), max(lengths))


@pytest.mark.parametrize("nq", [1, 70])
def test_attend_zero_queries_over_the_smallest_scales(cuda_device, nq):
    """A row of zeros over keys of the least scale: masked keys stay masked, the values' mean comes out."""
    cache, g = make(cuda_device, nq, 1, 2, [70], spread=1)
    cache.key_scales.fill_(2.0 ** -60)
    q = torch.zeros(1, nq, 256, dtype=torch.bfloat16, device=cuda_device)
    for causal in (False, True):
        close(cache.attend(q, 2, causal=causal), attention(Model(cache), q, 2, causal), 70)


@pytest.mark.parametrize("nq", [1, 20, 200])
def test_attend_scales_far_apart(cuda_device, nq):
    """Values of one block 2^40 times another's, a block of zeros, queries of very different sizes and sharp scores."""
    cache, g = make(cuda_device, nq, 1, 2, [450], spread=20)
    cache.value_scales[cache.block_table[0, 2].long()] = 2.0 ** -60
    cache.values.view(torch.uint8)[cache.block_table[0, 2].long()] = 0
    q = rows(g, 1, nq, 4 * DIM) * torch.exp2(torch.randint(-12, 4, (1, nq, 1), device=cuda_device, generator=g).float())
    q = q.bfloat16()
    q[0, 0, :DIM] = 0
    q[..., 7] *= 64  # an outlying dim
    close(cache.attend(q, 4), attention(Model(cache), q, 4, False), 450)


@pytest.mark.parametrize("nq,heads,kv_heads", [(3, 2, 1), (40, 2, 2), (150, 4, 2)])
def test_attend_nan_stays_where_it_is_seen(cuda_device, nq, heads, kv_heads):
    """NaN in a value: only the rows that see the key, only its dim.  NaN in a key: the whole of those rows.
    NaN in a query: its row.  (Stale NaN behind the last row is in every cache of this file.)"""
    cache, g = make(cuda_device, nq, 1, kv_heads, [200], spread=1)
    table = cache.block_table[0].long()
    codes = cache.values.view(torch.uint8)
    codes[table[198 // 64], 0, 198 % 64, 5] = 0x7f
    codes[table[3], 0, 199 % 64, 100] = 0xff
    cache.keys.view(torch.uint8)[table[3], kv_heads - 1, 199 % 64, 0] = 0x7f
    q = rows(g, 1, nq, heads * DIM)
    q[0, 1, DIM + 3] = float("nan")
    for causal in (True, False):
        close(cache.attend(q, heads, causal=causal), attention(Model(cache), q, heads, causal), 200)


@pytest.mark.parametrize("nq", [40, 200])
def test_attend_shares_without_keys(cuda_device, nq):
    """A cluster's CTAs that get no keys hand over nothing, whatever the queries hold: NaN queries stay in their rows."""
    cache, g = make(cuda_device, 6, 3, 2, [0, 64, 130], capacity=1024)
    q = rows(g, 3, nq, 4 * DIM)
    q[:, ::3, :DIM] = float("nan")
    for _ in range(5):
        for split in (0, 2, 8):
            out = cache.attend(q, 4, key_split=split)
            nan = out.view(3, nq, 4, DIM).isnan()
            assert not out[0].any() and nan[1:, ::3, 0].all()
            assert int(nan.sum()) == 2 * len(range(0, nq, 3)) * DIM


def test_attend_bad_blocks_and_lengths(cuda_device):
    """Block ids outside the pool are left out and reported; a length past the table is cut to it."""
    cache, g = make(cuda_device, 1, 2, 2, [190, 190], spread=1)
    q = rows(g, 2, 9, 4 * DIM)
    whole = cache.attend(q, 4)
    cache.block_table[0, 0], cache.block_table[0, 2] = -3, 1 << 20
    out = cache.attend(q, 4)
    assert cache.status() == 2
    assert torch.equal(out[1], whole[1]) and out.isfinite().all()
    middle = Model(cache)
    middle.table[0] = [middle.table[0][1]]
    middle.lengths[0] = 64
    close(out, attention(middle, q, 4, False), 190)
    k, _ = cache.read(64)
    assert cache.status() == 2 and not k[0].any()
    cache.block_table[0] = cache.block_table[1]  # a shared prefix
    cache.lengths.copy_(torch.tensor([10 ** 9, -7]))
    cache.values.view(torch.uint8).bitwise_and_(0x77)  # nothing stale: the cut length reads every row
    cache.keys.view(torch.uint8).bitwise_and_(0x77)
    out = cache.attend(q, 4)
    cut = Model(cache)
    cut.lengths = [192, 0]
    close(out, attention(cut, q, 4, False), 192)
    assert not out[1].any() and cache.status() == 0


def test_refusals(cuda_device):
    from waminfer_b200.cache import KVCache8

    cache = KVCache8(2, 100, 2, cuda_device)
    assert cache.capacity == 128
    good = torch.zeros(2, 3, 256, dtype=torch.bfloat16, device=cuda_device)
    for bad in (good[:1], good[..., :128], good.float(), good.cpu(), good[0]):
        with pytest.raises(ValueError):
            cache.append(bad, good)
        with pytest.raises(ValueError):
            cache.attend(bad, 2)
    with pytest.raises(ValueError, match="differ"):
        cache.append(good, good[:, :2])
    with pytest.raises(ValueError, match="one row"):
        cache.append(good[:, :0], good[:, :0])
    with pytest.raises(ValueError, match="counts"):
        cache.append(good, good, counts=torch.zeros(2, dtype=torch.int64, device=cuda_device))
    with pytest.raises(ValueError, match="at"):
        cache.append(good, good, at=torch.zeros(3, dtype=torch.int32, device=cuda_device))
    with pytest.raises(ValueError, match="multiple"):
        cache.attend(good, 3)
    with pytest.raises(RuntimeError, match="backward"):
        cache.attend(good.clone().requires_grad_(), 2)
    from waminfer_b200._lib import WamffnError
    with pytest.raises(WamffnError, match="key_split"):
        cache.attend(good, 2, key_split=3)
    with pytest.raises(ValueError):
        cache.read(0)
    with pytest.raises(ValueError):
        cache.read(1, -1)
    with pytest.raises(ValueError, match="lengths"):
        KVCache8.of(cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.block_table,
                    cache.lengths.long())
    assert cache.attend(good[:, :0], 2).shape == (2, 0, 256)
    assert not cache.attend(good, 2).any()  # an empty cache


def test_views_and_another_stream(cuda_device):
    """Queries as a chunk of a packed projection, in another row order, unaligned; on a side stream."""
    cache, g = make(cuda_device, 2, 2, 2, [300, 77], spread=1)
    packed = rows(g, 2, 21, 3 * 512)
    q = packed[..., 512:1024]
    expect = cache.attend(q.contiguous(), 4, causal=True)
    assert torch.equal(cache.attend(q, 4, causal=True), expect)
    assert torch.equal(cache.attend(q.transpose(0, 1).contiguous().transpose(0, 1), 4, causal=True), expect)
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(cache.attend(odd, 4, causal=True), expect)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = cache.attend(q, 4, causal=True)
        read = cache.read(10)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there, expect) and torch.equal(read[0], cache.read(10)[0])


def test_a_single_batch_or_row_of_any_stride(cuda_device):
    cache, g = make(cuda_device, 5, 1, 2, [100], capacity=200)
    held = rows(g, 1, 21 * 512 + 3)
    q = held.as_strided((1, 21, 512), (held.shape[1], 512, 1))
    assert q.stride(0) % 8
    plain = q.flatten().view(1, 21, 512)
    assert torch.equal(cache.attend(q, 4, causal=True), cache.attend(plain, 4, causal=True))
    one = rows(g, 1, 1, 257)[..., :256]
    other, _ = make(cuda_device, 5, 1, 2, [100], capacity=200)
    cache.append(one, one)
    other.append(one.flatten().view(1, 1, 256), one.flatten().view(1, 1, 256))
    assert one.stride(1) % 8 and cache.lengths.tolist() == [101] and cache.status() == other.status() == 0
    assert torch.equal(cache.read(1, 100)[0], other.read(1, 100)[0]) and cache.read(1, 100)[0].any()


def test_status_of_calls_on_another_stream(cuda_device):
    from waminfer_b200.cache import KVCache8

    cache = KVCache8(1, 64, 1, cuda_device)
    x = torch.ones(1, 65, DIM, dtype=torch.bfloat16, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # about 50 ms
        cache.append(x, x)  # does not fit
    assert cache.status() == 2 and cache.status() == 0 and cache.lengths.tolist() == [0]


def test_offsets_past_32_bits(cuda_device):
    """Blocks at the end of a pool of 2.6 GB of keys, and query rows past 2^31 elements."""
    from waminfer_b200.cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(3)
    k, v = rows(g, 1, 200, 8 * DIM), rows(g, 1, 200, 8 * DIM)
    small, large = KVCache8(1, 256, 8, cuda_device), KVCache8(1, 256, 8, cuda_device, blocks=40000)
    large.block_table[0] = torch.tensor([39999, 32768, 39000, 1], dtype=torch.int32)
    for cache in (small, large):
        cache.append(k[:, :130], v[:, :130])
        cache.append(k[:, 130:], v[:, 130:])
    for a, b in zip(small.read(200), large.read(200)):
        assert torch.equal(a, b)
    for nq in (1, 30, 300):
        q = rows(g, 1, nq, 16 * DIM)
        assert torch.equal(small.attend(q, 16), large.attend(q, 16))
    assert large.status() == 0
    del large
    one = KVCache8(1, 64, 1, cuda_device)
    one.append(k[:, :40, :DIM], v[:, :40, :DIM])
    q = rows(g, 1, 530000, 32 * DIM)
    tail = one.attend(q, 32)[:, -5:].clone()
    close(tail, attention(Model(one), q[:, -5:], 32, False), 40)


# ------------------------------------------------------------- together
def test_a_decode_run(cuda_device):
    """A prompt, then tokens one by one: norm and rotation, store, attention; eagerly and from one captured step."""
    from waminfer_b200.cache import KVCache8
    from waminfer_b200.rope import qk_norm_rope

    batch, heads, kv_heads, prompt = 2, 8, 2, 100
    g = torch.Generator(device=cuda_device).manual_seed(0)
    qw, kw = rows(g, DIM), rows(g, DIM)
    inverse = 10000.0 ** (-torch.arange(64, device=cuda_device, dtype=torch.float64) / 64)
    angles = torch.arange(200, device=cuda_device, dtype=torch.float64)[:, None] * inverse
    freqs = torch.polar(torch.ones_like(angles), angles).to(torch.complex64)
    cache = KVCache8(batch, 160, kv_heads, cuda_device)

    def step(qkv, positions):
        q, k, v = qkv.split([heads * DIM, kv_heads * DIM, kv_heads * DIM], -1)
        q, k = qk_norm_rope(q, k, qw, kw, freqs, positions, heads, kv_heads, interleaved=False)
        cache.append(k, v)
        return q, k, v, cache.attend(q, heads, causal=True)

    model = Model(cache)
    width = (heads + 2 * kv_heads) * DIM
    q, k, v, out = step(rows(g, batch, prompt, width), None)
    model.append(k, v)
    model.same(cache)
    close(out, attention(model, q, heads, True), prompt)
    static = rows(g, batch, 1, width)
    at = cache.lengths.clone().view(batch, 1)
    before = [t.clone() for t in (cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.lengths)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, k, v, out = step(static, at)
        at += 1
    for t, old in zip((cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.lengths), before):
        assert torch.equal(t, old)  # capture runs nothing
    for i in range(30):
        static.copy_(rows(g, batch, 1, width, size=1 + 0.1 * i))
        graph.replay()
        model.append(k, v)
        if i % 10 == 9:
            model.same(cache)
            close(out, attention(model, q, heads, True), prompt + i)
    assert cache.status() == 0


def test_traced(cuda_device):
    """The calls inside a compiled function: the same cache and results as called one by one."""
    from waminfer_b200.cache import KVCache8
    from waminfer_b200.rope import qk_norm_rope

    g = torch.Generator(device=cuda_device).manual_seed(9)
    qkv, w = rows(g, 2, 5, 4 * DIM), rows(g, DIM)
    freqs = torch.polar(torch.ones(8, 64), torch.rand(8, 64)).to(cuda_device)
    caches = [KVCache8(2, 128, 1, cuda_device) for _ in range(2)]
    at = torch.tensor([0, 0], dtype=torch.int32, device=cuda_device)

    def step(cache, qkv):
        q, k, v = qkv.split([2 * DIM, DIM, DIM], -1)
        q, k = qk_norm_rope(q, k, w, w, freqs, None, 2, 1)
        cache.append(k, v, at=at)
        return cache.attend(q, 2, causal=True) * 1.0, *cache.read(5), *cache.read(3, start=at)

    with torch.no_grad():
        plain = step(caches[0], qkv)
        traced = torch.compile(lambda qkv: step(caches[1], qkv), backend="aot_eager", fullgraph=True)(qkv)
    for a, b in zip(plain, traced):
        assert torch.equal(a, b)
    assert torch.equal(caches[0].lengths, caches[1].lengths) and torch.equal(caches[0].keys.view(torch.uint8),
                                                                             caches[1].keys.view(torch.uint8))


def test_two_graphs_and_two_caches_at_once(cuda_device):
    """Two captured attention steps over different caches, replayed on two streams at the same time."""
    made = [make(cuda_device, i, 2, 4, [900 + 50 * i, 300], spread=1) for i in range(2)]
    jobs = []
    for cache, g in made:
        q = rows(g, 2, 3, 8 * DIM)
        expect = cache.attend(q, 8, causal=True)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph):
            out = cache.attend(q, 8, causal=True)
        jobs.append((graph, side, out, expect, q))  # q stays where the graph reads it
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, side, _, _, _ in jobs:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, expect, _ in jobs:
        assert torch.equal(out, expect)


def test_the_bf16_ops_on_rows_read_back(cuda_device):
    """A cached prefix handed to the bf16 current-frame attention, and the same rows attended in the cache."""
    from waminfer_b200.attention import masked_attention

    cache, g = make(cuda_device, 4, 1, 3, [150])
    q = rows(g, 1, 70, 3 * DIM)
    k, v = cache.read(150)
    theirs = masked_attention(q, k, v, None, 3).float().cpu().double()
    ours = cache.attend(q, 3)
    out, absolute, bound = attention(Model(cache), q, 3, False)
    close(ours, (out, absolute, bound), 150)
    # The bf16 op rounds its probabilities to bf16: 2^-9 of A on top of the result's rounding.
    assert ((theirs - out).abs() <= 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -12) * absolute).all()

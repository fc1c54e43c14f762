"""GPU: the attention over the 8-bit cache on each of its paths, asserted from the plan that the call takes.

Reference and tolerance are those of ``test_gpu_cache.py``."""

import ctypes

import pytest
import torch
from test_gpu_cache import DIM, Model, attention, close, make, rows

pytestmark = pytest.mark.gpu


def call(cache, q, heads, out=None, causal=False, key_split=0, workspace=None):
    """The arguments of one attention call on the C entry."""
    from waminfer_b200 import _lib

    return _lib.CacheAttentionArgs(cache._view, _lib.RowsView(q.data_ptr(), q.stride(1), q.stride(0)),
                                   None if out is None else out.data_ptr(),
                                   None if workspace is None else workspace.data_ptr(),
                                   0 if workspace is None else workspace.numel(), q.shape[1], heads, causal, key_split)


def plan_of(args):
    from waminfer_b200 import _lib

    plan = _lib.CachePlan()
    _lib.check(_lib.lib().wamffn_cache_attention_plan(ctypes.byref(args), ctypes.byref(plan)))
    return plan


def run(args):
    from waminfer_b200 import _lib

    _lib.launch(_lib.lib().wamffn_cache_attention, torch.cuda.current_device(), ctypes.byref(args))


@pytest.mark.parametrize("nq,lengths", [(300, [500]), (12, [9000])])
def test_a_workspace_for_less_than_a_part(cuda_device, nq, lengths):
    """The call does without: every row is written."""
    cache, g = make(cuda_device, nq, 1, 1, lengths, spread=2)
    q = rows(g, 1, nq, 2 * DIM)
    ref = attention(Model(cache), q, 2, True)
    for size in (16, nq * 2 * 130 * 4 - 16):
        workspace = torch.empty(size, dtype=torch.uint8, device=cuda_device)
        out = torch.full_like(q, float("nan"))
        args = call(cache, q, 2, out, True, workspace=workspace)
        assert plan_of(args).parts == 1
        run(args)
        close(out, ref, lengths[0])


# Two tiles of 128 different rows a CTA (tile_rows 256): several steps, the ring of four stages around more than once,
# O rescaled; the last tile of at most 128 rows, which runs as one, beside full ones; clusters; parts; ragged batches.
TWO_TILES = [  # nq, heads, kv_heads, lengths, causal, key_split, parts
    (670, 32, 8, [513], False, 1, 1),            # 2680 packed rows: a last tile of 120
    (670, 8, 2, [513, 130], False, 2, 1),        # the same in clusters, ragged
    (1000, 32, 8, [2000], True, 1, 1),           # 16 tiles, the first rows of a tile see less
    (400, 24, 24, [700, 1], True, 1, 1),
    (150, 24, 24, [900, 70], True, 2, 1),
    (300, 37, 37, [2048], False, 2, 1),          # 300 rows: a last tile of 44
    (392, 16, 4, [2048], False, 4, 1),
    (300, 8, 2, [900], True, 8, 1),
    (128, 32, 8, [4096], False, 8, 1),
    (392, 24, 24, [9000], False, 1, 2),          # parts through the workspace
]


@pytest.mark.parametrize("nq,heads,kv_heads,lengths,causal,key_split,parts", TWO_TILES)
def test_two_tiles_of_rows(cuda_device, nq, heads, kv_heads, lengths, causal, key_split, parts):
    cache, g = make(cuda_device, nq + heads, len(lengths), kv_heads, lengths, spread=3, extra=1)
    q = rows(g, len(lengths), nq, heads * DIM)
    out = cache.attend(q, heads, causal=causal, key_split=key_split)
    workspace = torch.empty(max(cache._needs.values()) or 16, dtype=torch.uint8, device=cuda_device)
    plan = plan_of(call(cache, q, heads, out, causal, key_split, workspace))
    assert plan.tile_rows == 256 and plan.key_split == key_split and min(plan.parts, 2) == parts
    close(out, attention(Model(cache), q, heads, causal), max(lengths))
    for _ in range(5):
        assert torch.equal(out, cache.attend(q, heads, causal=causal, key_split=key_split))
    assert cache.status() == 0


def test_one_tile_of_rows_in_parts(cuda_device):
    """Tiles of 128 rows, each over parts of the keys."""
    cache, g = make(cuda_device, 396, 1, 4, [9000], spread=3, extra=1)
    q = rows(g, 1, 392, 4 * DIM)
    out = cache.attend(q, 4, key_split=1)
    workspace = torch.empty(max(cache._needs.values()), dtype=torch.uint8, device=cuda_device)
    plan = plan_of(call(cache, q, 4, out, key_split=1, workspace=workspace))
    assert plan.tile_rows == 128 and plan.parts > 1
    close(out, attention(Model(cache), q, 4, False), 9000)


def test_two_tiles_of_rows_in_many_parts(cuda_device):
    """128 rows of 40 heads over 32768 rows of 8: checked at some of the queries."""
    cache, g = make(cuda_device, 40, 1, 8, [32768], spread=2)
    q = rows(g, 1, 128, 40 * DIM)
    out = cache.attend(q, 40)
    workspace = torch.empty(max(cache._needs.values()), dtype=torch.uint8, device=cuda_device)
    plan = plan_of(call(cache, q, 40, out, workspace=workspace))
    assert plan.tile_rows == 256 and plan.parts > 1
    some = [0, 25, 26, 51, 76, 102, 127]  # around the tiles' borders, and the last tile of 128 rows
    close(out[:, some], attention(Model(cache), q[:, some], 40, False), 32768)


def test_clusters_of_every_size(cuda_device):
    """Clusters that key_split does not force (3, 5, 6, 7) come from the plan; which shapes take them depends a
    little on the device, so a spread of shapes stands for them."""
    found = set()
    for nq, heads, kv_heads, keys in ((300, 32, 8, 1024), (150, 32, 8, 512), (150, 24, 24, 2048), (65, 32, 8, 2048),
                                      (300, 16, 4, 3000), (200, 10, 5, 1024), (300, 8, 1, 2048), (200, 8, 1, 2048),
                                      (250, 8, 1, 2048)):
        cache, g = make(cuda_device, nq + heads, 1, kv_heads, [keys], spread=2)
        q = rows(g, 1, nq, heads * DIM)
        out = cache.attend(q, heads)
        plan = plan_of(call(cache, q, heads, out))
        found.add((plan.tile_rows, plan.key_split))
        close(out, attention(Model(cache), q, heads, False), keys)
    assert len({split for _, split in found} & {3, 5, 6, 7}) >= 2 and {rows_ for rows_, _ in found} == {128, 256}, found


def test_the_tensors_of_a_cache_are_not_replaced(cuda_device):
    """Calls go by the tensors that the cache was made of: another one in an attribute's place is refused, not
    ignored.  In place they change as ever."""
    cache, g = make(cuda_device, 1, 2, 1, [70, 3], spread=1)
    q = rows(g, 2, 1, DIM)
    for name in ("keys", "values", "key_scales", "value_scales", "block_table", "lengths"):
        old = getattr(cache, name)
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, old.clone())
        with pytest.raises(AttributeError, match=name):
            delattr(cache, name)
        assert getattr(cache, name) is old
    for name in ("batch", "width", "kv_heads", "device"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, 5)
    cache.lengths -= 1
    assert cache.lengths.tolist() == [69, 2]
    close(cache.attend(q, 1), attention(Model(cache), q, 1, False), 70)


@pytest.mark.parametrize("scale", [2.0 ** 120, 2.0 ** 126, 2.0 ** 127, float("inf"), float("nan")])
def test_the_largest_scales(cuda_device, scale):
    """A value block of the largest scale that counts, 2^126, and of scales past it: read, attended, appended to."""
    cache, g = make(cuda_device, 8, 1, 2, [80], capacity=192, spread=1)
    small = torch.randn(cache.values.shape, device=cuda_device, generator=g).clamp(-1, 1)  # results stay finite
    cache.values.copy_(torch.where(cache.values.float().isnan(), float("nan"), small).to(torch.float8_e4m3fn))
    cache.value_scales.fill_(scale)
    model = Model(cache)
    model.exps[1].fill_(120 if scale == 2.0 ** 120 else 126)
    for nq, causal in ((1, True), (9, False), (70, True), (300, False)):
        q = rows(g, 1, nq, 2 * DIM)
        close(cache.attend(q, 2, causal=causal), attention(model, q, 2, causal), 80)
    v = cache.read(80)[1][0]
    for h in range(2):
        assert torch.equal(v[:, h * DIM:(h + 1) * DIM].cpu().double(), model.rows(1, 0, h))
    new = rows(g, 1, 3, 2 * DIM)
    new[0, 0, :6] = torch.tensor([2.0 ** 126, -3e38, float("inf"), -float("inf"), float("nan"), 2.0 ** 117])
    cache.append(new, new)
    model.append(new, new)
    assert cache.status() == 0 and cache.lengths.tolist() == [83]
    held = cache.values[cache.block_table[0, 1].long()].cpu().double()
    assert torch.equal(held[:, :19].nan_to_num(1e9), model.codes[1][model.table[0][1], :, :19].nan_to_num(1e9))
    assert torch.equal(torch.log2(cache.value_scales[cache.block_table[0, 1].long()].cpu().double()),
                       model.exps[1][model.table[0][1]])


def close_held(cache, got, q, heads, keys):
    """The module's tolerance and what it leaves out: the probabilities times the scale of their values, P, are f16
    numbers with a row's largest at 2^5 or more.  Below 2^-14 they are off by up to 2^-25, so by 2^-30 of the largest,
    and the sum over the values (codes, without their scale) by that times sum |code|."""
    model = Model(cache)
    out, absolute, bound = attention(model, q, heads, False)
    batch, nq, _ = q.shape
    group = heads // cache.kv_heads
    extra = torch.zeros(batch, nq, heads, DIM, dtype=torch.float64)
    for b in range(batch):
        n = model.lengths[b]
        ids = model.table[b][:-(-n // 64)]
        for h in range(heads):
            s = q[b].cpu().double().view(nq, heads, DIM)[:, h] @ model.rows(0, b, h // group).T / DIM ** 0.5
            p = torch.softmax(s, -1)
            scale = torch.exp2(model.exps[1][ids, h // group]).repeat_interleave(64)[:n]
            codes = model.codes[1][ids, h // group].reshape(-1, DIM)[:n].abs().nan_to_num().sum(0)
            extra[b, :, h] = 2.0 ** -30 * (p * scale).amax(-1, keepdim=True) * codes
    got = got.cpu().double()
    assert got.isfinite().all()
    tol = 2.0 ** -8 * out.abs() + (2.0 ** -11 + 2 * 2.0 ** -16 * bound + keys * 2.0 ** -23 + 2.0 ** -20) * absolute
    off = (got - out).abs() - tol - extra.flatten(2)
    assert off.max().item() <= 0, (off.max().item(), tol.flatten()[off.argmax()].item())


def far_apart(cache, g, huge, zero, exponent):
    """Ordinary keys and values; block `huge` of the first sequence holds values of 2^exponent, block `zero` none."""
    ids = cache.block_table[0].long()
    cache.value_scales.fill_(2.0 ** -6)
    cache.value_scales[ids[huge]] = 2.0 ** (exponent - 6)
    cache.value_scales[ids[zero]] = 2.0 ** -60
    cache.values.view(torch.uint8)[ids[zero]] = 0
    return ids


# Every place where shares of a row meet: steps of a warp or a tile, warps, the two tiles of the same rows, a cluster,
# parts through the workspace.
MEETINGS = [  # nq, heads, kv_heads, length, key_split
    (1, 2, 1, 128, 1),
    (1, 8, 2, 1100, 0),
    (12, 1, 1, 128, 0),
    (5, 3, 1, 1500, 4),
    (1, 1, 1, 9000, 0),
    (40, 2, 2, 128, 1),
    (40, 2, 2, 700, 8),
    (130, 1, 1, 9000, 0),
    (300, 24, 24, 448, 1),
    (300, 16, 4, 1024, 2),
]


@pytest.mark.parametrize("exponent", [75, 100, 125])
@pytest.mark.parametrize("nq,heads,kv_heads,length,key_split", MEETINGS)
def test_a_block_of_zeros_beside_one_of_huge_values(cuda_device, nq, heads, kv_heads, length, key_split, exponent):
    """All keys keep their share of the normaliser, however far apart the scales of their values lie."""
    cache, g = make(cuda_device, nq + exponent, 1, kv_heads, [length])
    q = rows(g, 1, nq, heads * DIM)
    q[:, ::2] = 0  # equal scores
    blocks = cache.width
    for huge, zero in ((0, 1), (1, 0), (blocks - 1, blocks // 2), (blocks // 2, blocks - 1)):
        if huge != zero:
            far_apart(cache, g, huge, zero, exponent)
            close_held(cache, cache.attend(q, heads, key_split=key_split), q, heads, length)
            cache.values.copy_(torch.where(cache.values.float() == 0, 40.0, cache.values.float()).to(cache.values.dtype))


@pytest.mark.parametrize("exponent", [40, 80, 110])
@pytest.mark.parametrize("nq,heads,kv_heads,length,key_split", MEETINGS)
def test_huge_values_at_low_scores(cuda_device, nq, heads, kv_heads, length, key_split, exponent):
    """Keys whose weight is about 2^-exponent of the others' and whose values are 2^exponent of theirs count as much;
    the queries before and behind those that see it so give them more and less."""
    cache, g = make(cuda_device, nq + exponent, 1, kv_heads, [length])
    blocks = cache.width
    q = torch.zeros(1, nq, heads * DIM, device=cuda_device)
    q.view(1, nq, heads, DIM)[..., 0] = torch.linspace(0.8, 1.2, nq, device=cuda_device)[None, :, None]
    q += torch.randn(q.shape, device=cuda_device, generator=g) * 2.0 ** -8
    q = q.bfloat16()
    for huge, zero in ((0, 1), (1, 0), (blocks - 1, blocks // 2)):
        if huge == zero:
            continue
        ids = far_apart(cache, g, huge, zero, exponent)
        cache.key_scales.fill_(2.0 ** -6)
        cache.key_scales[ids[huge]] = 2.0  # dim 0 of these keys: -ln(2) * exponent * sqrt(128)
        keys = cache.keys.float().clamp(-100, 100)
        keys[ids[huge], :, :, 0] = -exponent * 0.6931 * 128 ** 0.5 / 2
        keys[ids[huge], :, :, 1:] = 0
        cache.keys.copy_(keys.to(cache.keys.dtype))
        cache.values.copy_(torch.where(cache.values.float().abs() > 64, 3.0, cache.values.float()).to(cache.values.dtype))
        close_held(cache, cache.attend(q, heads, key_split=key_split), q, heads, length)


@pytest.mark.parametrize("nq,heads,kv_heads,length,key_split", MEETINGS)
def test_sharp_scores(cuda_device, nq, heads, kv_heads, length, key_split):
    """Blocks hundreds of binades below a row's maximum, before and behind it."""
    cache, g = make(cuda_device, nq, 1, kv_heads, [length], spread=3)
    q = rows(g, 1, nq, heads * DIM, size=24.0)
    close_held(cache, cache.attend(q, heads, key_split=key_split), q, heads, length)


def test_recorded_on_tensors_with_data(cuda_device):
    """A tracer outside the compiler records the calls instead of their results."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from waminfer_b200.cache import KVCache8

    caches = [KVCache8(2, 128, 1, cuda_device) for _ in range(2)]
    g = torch.Generator(device=cuda_device).manual_seed(1)
    at = torch.zeros(2, dtype=torch.int32, device=cuda_device)

    def step(cache, x):
        cache.append(x[..., :DIM], x[..., DIM:], at=at)
        return cache.attend(x, 2, causal=True), *cache.read(5)

    x, y = rows(g, 2, 5, 2 * DIM), rows(g, 2, 5, 2 * DIM)
    recorded = make_fx(lambda x: step(caches[0], x))(x)
    for a, b in zip(recorded(y), step(caches[1], y)):
        assert torch.equal(a, b)
    assert torch.equal(caches[0].keys.view(torch.uint8), caches[1].keys.view(torch.uint8))


@pytest.mark.parametrize("nq,heads,kv_heads,length,key_split", MEETINGS)
def test_huge_queries_and_keys_that_do_not_meet(cuda_device, nq, heads, kv_heads, length, key_split):
    """Queries of 2^100 in one dim, keys of 2^40 in the others: every score is zero, whatever the product of the two
    powers of two that stand for them (past fp32's largest number); the values' mean comes out."""
    cache, g = make(cuda_device, nq, 1, kv_heads, [length], spread=1)
    keys = cache.keys.float()
    keys[..., 5] = torch.where(keys[..., 5].isnan(), keys[..., 5], 0.0)
    cache.keys.copy_(keys.to(cache.keys.dtype))
    cache.key_scales.fill_(2.0 ** 33)
    q = torch.zeros(1, nq, heads * DIM, dtype=torch.bfloat16, device=cuda_device)
    q.view(1, nq, heads, DIM)[..., 5] = 2.0 ** 100
    close(cache.attend(q, heads, key_split=key_split), attention(Model(cache), q, heads, False), length)


@pytest.mark.parametrize("nq", [1, 12, 40, 300])
def test_queries_of_nan_over_blocks_that_are_left_out(cuda_device, nq):
    """A row whose every block lies outside the pool sees nothing: zeros, whatever the query holds; in a sequence with
    one good block it sees that."""
    cache, g = make(cuda_device, nq, 3, 1, [130, 130, 64], spread=1)
    cache.block_table[0] = torch.tensor([-1, 999, 1 << 30], dtype=torch.int32)
    cache.block_table[1, 1:] = -7
    q = rows(g, 3, nq, 2 * DIM)
    q[:, 0, :DIM] = float("nan")
    q[:, 0, DIM] = float("inf")
    for split in (0, 1, 2):
        out = cache.attend(q, 2, key_split=split)
        assert cache.status() == 2
        assert not out[0].any() and out[1:, 0].isnan().all() and out[1:, 1:].isfinite().all()


def test_a_prefix_read_back_for_the_current_frame(cuda_device):
    """Rows stored in 8 bits, read back and handed to the bf16 current-frame attention beside rows of the frame; its
    probabilities are bf16: 2^-9 of A each on top of the result's rounding."""
    from waminfer_b200.attention import current_frame_attention
    from waminfer_b200.cache import KVCache8

    g = torch.Generator(device=cuda_device).manual_seed(2)
    heads, prefix, frame, action = 3, 150, 40, 16
    cache = KVCache8(1, 200, heads, cuda_device)
    cache.append(rows(g, 1, prefix, heads * DIM), rows(g, 1, prefix, heads * DIM))
    qv, kv, vv = (rows(g, 1, frame, heads * DIM) for _ in range(3))
    qa, ka, va = (rows(g, 1, action, heads * DIM) for _ in range(3))
    ck, cv = cache.read(prefix)
    got = torch.cat(current_frame_attention(qv, qa, ck, kv, ka, cv, vv, va, heads), 1).cpu().double()
    model = Model(cache)
    k = torch.cat((torch.stack([model.rows(0, 0, h) for h in range(heads)], 1),
                   torch.cat((kv, ka), 1)[0].cpu().double().view(-1, heads, DIM)))
    v = torch.cat((torch.stack([model.rows(1, 0, h) for h in range(heads)], 1),
                   torch.cat((vv, va), 1)[0].cpu().double().view(-1, heads, DIM)))
    q = torch.cat((qv, qa), 1)[0].cpu().double().view(-1, heads, DIM)
    p = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) / DIM ** 0.5, -1)
    out = torch.einsum("hij,jhd->ihd", p, v).reshape(got.shape)
    absolute = torch.einsum("hij,jhd->ihd", p, v.abs()).reshape(got.shape)
    assert ((got - out).abs() <= 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -12) * absolute).all()

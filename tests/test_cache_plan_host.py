"""CPU: how the attention over the 8-bit cache shares out its work, for a device described in numbers."""

import ctypes
import random

import pytest

from waminfer_b200 import _lib

FAKE = 256  # non-null, 16-byte aligned: the plan reads sizes only
CLUSTERS = (0, 148, 74, 45, 35, 27, 22, 19, 16)  # clusters of 0 .. 8 CTAs on a device of 148 SMs


def attention_args(nq, heads, kv_heads, width, batch=1, causal=0, key_split=0, workspace=0):
    cache = _lib.CacheView(keys=FAKE, values=FAKE, key_scales=FAKE, value_scales=FAKE, block_table=FAKE,
                           table_stride=width, lengths=FAKE, tickets=FAKE, status=FAKE, blocks=batch * width,
                           kv_heads=kv_heads, batch=batch, width=width)
    view = _lib.RowsView(FAKE, heads * 128, nq * heads * 128)
    return _lib.CacheAttentionArgs(cache, view, FAKE, FAKE if workspace else None, workspace, nq, heads, causal, key_split)


def plan_of(args, clusters=CLUSTERS):
    plan = _lib.CachePlan(sm_count=148, clusters=(ctypes.c_int * 9)(*clusters))
    _lib.check(_lib.lib().wamffn_cache_attention_plan(ctypes.byref(args), ctypes.byref(plan)))
    return plan


def covers(plan, rows):
    return plan.row_tiles * plan.tile_rows >= rows > (plan.row_tiles - 1) * plan.tile_rows


@pytest.mark.parametrize("bytes_", [0, 16, 300 * 2 * 130 * 4 - 16, 300 * 2 * 130 * 4, 1 << 30])
def test_a_workspace_of_any_size_leaves_no_row_out(bytes_):
    """Bytes for less than one part count as none."""
    plan = plan_of(attention_args(300, 2, 1, 512, workspace=bytes_))
    assert covers(plan, 600) and plan.parts <= max(1, bytes_ // (300 * 2 * 130 * 4))


def test_every_plan_covers_its_rows():
    rng = random.Random(1)
    log = lambda most: int(2 ** rng.uniform(0, most))  # noqa: E731
    for _ in range(400):
        kv_heads = rng.choice((1, 2, 3, 8, 24))
        nq, group, batch = log(13), rng.choice((1, 2, 4, 7)), log(4)
        args = attention_args(nq, kv_heads * group, kv_heads, log(10), batch, rng.randrange(2),
                              rng.choice((0, 0, 1, 2, 4, 8)), rng.choice((0, log(28))))
        plan = plan_of(args)
        assert covers(plan, nq * group) and 1 <= plan.key_split <= 8 and 1 <= plan.parts <= 32
        assert bool(plan.tensor_cores) == (nq * group > 16)
        if args.key_split:
            assert plan.key_split == args.key_split


def test_the_plan_rejects_what_the_call_rejects():
    lib, plan = _lib.lib(), _lib.CachePlan(sm_count=148)
    args = attention_args(1, 3, 2, 4)
    assert lib.wamffn_cache_attention_plan(ctypes.byref(args), ctypes.byref(plan)) == 1
    assert b"multiple" in lib.wamffn_last_error()
    assert lib.wamffn_cache_attention_plan(None, ctypes.byref(plan)) == 1
    assert lib.wamffn_cache_attention_plan(ctypes.byref(args), None) == 1


def test_a_split_that_the_device_cannot_run_is_refused():
    """No cluster of eight fits: a forced split of eight has no plan, the automatic choice takes another."""
    none = CLUSTERS[:8] + (0,)
    args = attention_args(300, 4, 1, 64, key_split=8)
    plan = _lib.CachePlan(sm_count=148, clusters=(ctypes.c_int * 9)(*none))
    assert _lib.lib().wamffn_cache_attention_plan(ctypes.byref(args), ctypes.byref(plan)) == 3  # unsupported
    assert b"key_split=8" in _lib.lib().wamffn_last_error()
    args = attention_args(300, 4, 1, 64)
    alone = plan_of(args, (0, 148) + (0,) * 7)
    assert alone.key_split == 1 and covers(alone, 1200)

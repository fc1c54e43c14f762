"""CPU: what the norm + rotation and the 8-bit cache refuse, before anything is launched."""

import ctypes

import pytest
import torch

from waminfer_b200 import _lib

FAKE = 256  # non-null, 16-byte aligned: never dereferenced because the call is rejected first


def _rope(**over):
    view = _lib.RowsView(FAKE, 3072, 3072 * 392)
    args = dict(q=view, k=view, q_weight=FAKE, k_weight=FAKE, rope=FAKE, table_stride=64, q_out=FAKE, k_out=FAKE,
                table_rows=392, pairs=64, batch=1, rows=392, heads=24, kv_heads=24, head_dim=128, whole_row=1,
                interleaved=1, eps=1e-6)
    args.update(over)
    return _lib.QkRopeArgs(**args)


@pytest.mark.parametrize("over,code,text", [
    (dict(head_dim=96), 3, b"head_dim"),
    (dict(rows=0), 1, b"rows"),
    (dict(heads=0), 1, b"heads"),
    (dict(q=_lib.RowsView(None, 3072, 0)), 1, b"q is null"),
    (dict(q=_lib.RowsView(FAKE + 2, 3072, 0)), 1, b"aligned"),
    (dict(k=_lib.RowsView(FAKE, 3000, 0)), 1, b"k strides"),
    (dict(k=_lib.RowsView(FAKE, 3076, 0)), 1, b"k strides"),
    (dict(k_weight=None), 1, b"weights"),
    (dict(k_out=FAKE + 8), 1, b"aligned"),
    (dict(pairs=62), 1, b"pairs"),
    (dict(pairs=68), 1, b"pairs"),
    (dict(table_stride=63), 1, b"rope table"),
    (dict(table_rows=391), 1, b"rope table of 391"),
    (dict(positions=FAKE, position_bytes=2), 1, b"positions"),
    (dict(heads=240, q=_lib.RowsView(FAKE, 30720, 0)), 3, b"whole-row"),
])
def test_rope_rejects_before_launching(over, code, text):
    lib = _lib.lib()
    assert lib.wamffn_qk_norm_rope(None, ctypes.byref(_rope(**over))) == code
    assert text in lib.wamffn_last_error()


def _cache(**over):
    args = dict(keys=FAKE, values=FAKE, key_scales=FAKE, value_scales=FAKE, block_table=FAKE, table_stride=4,
                lengths=FAKE, tickets=FAKE, status=FAKE, blocks=8, kv_heads=2, batch=2, width=4)
    args.update(over)
    return _lib.CacheView(**args)


@pytest.mark.parametrize("over,code,text", [
    (dict(blocks=0), 1, b"blocks=0"),
    (dict(batch=0), 1, b"batch=0"),
    (dict(width=0), 1, b"width=0"),
    (dict(kv_heads=40000), 3, b"kv_heads"),
    (dict(blocks=2 ** 30), 3, b"2^31"),
    (dict(lengths=None), 1, b"null"),
    (dict(values=FAKE + 8), 1, b"aligned"),
    (dict(table_stride=3), 1, b"block_table"),
])
def test_cache_is_checked_by_every_entry(over, code, text):
    lib = _lib.lib()
    view = _lib.RowsView(FAKE, 256, 256)
    for entry, args in ((lib.wamffn_cache_append, _lib.CacheAppendArgs(_cache(**over), view, view, None, None, 1)),
                        (lib.wamffn_cache_read, _lib.CacheReadArgs(_cache(**over), None, FAKE, FAKE, 0, 1)),
                        (lib.wamffn_cache_attention, _lib.CacheAttentionArgs(_cache(**over), view, FAKE, None, 0, 1, 2, 0, 0))):
        assert entry(None, ctypes.byref(args)) == code
        assert text in lib.wamffn_last_error()
        assert entry(None, None) == 1


def test_cache_entries_reject_before_launching():
    lib = _lib.lib()
    view, bad = _lib.RowsView(FAKE, 256, 256), _lib.RowsView(FAKE, 200, 256)
    for args, text in ((_lib.CacheAppendArgs(_cache(tickets=None), view, view, None, None, 1), b"tickets"),
                       (_lib.CacheAppendArgs(_cache(), view, view, None, None, 0), b"rows=0"),
                       (_lib.CacheAppendArgs(_cache(), view, bad, None, None, 2), b"v strides"),
                       (_lib.CacheAppendArgs(_cache(), _lib.RowsView(), view, None, None, 2), b"k is null")):
        assert lib.wamffn_cache_append(None, ctypes.byref(args)) == 1
        assert text in lib.wamffn_last_error()
    for args, text in ((_lib.CacheReadArgs(_cache(), None, FAKE, FAKE, 0, 0), b"count=0"),
                       (_lib.CacheReadArgs(_cache(), None, FAKE, FAKE, -1, 1), b"start=-1"),
                       (_lib.CacheReadArgs(_cache(), None, FAKE, None, 0, 1), b"aligned")):
        assert lib.wamffn_cache_read(None, ctypes.byref(args)) == 1
        assert text in lib.wamffn_last_error()
    for args, text in ((_lib.CacheAttentionArgs(_cache(), view, FAKE, None, 0, 0, 2, 0, 0), b"nq=0"),
                       (_lib.CacheAttentionArgs(_cache(), view, FAKE, None, 0, 1, 3, 0, 0), b"multiple"),
                       (_lib.CacheAttentionArgs(_cache(), view, FAKE, None, 0, 1, 2, 0, 3), b"key_split"),
                       (_lib.CacheAttentionArgs(_cache(), view, FAKE, FAKE + 4, 4096, 1, 2, 0, 0), b"workspace"),
                       (_lib.CacheAttentionArgs(_cache(), view, FAKE + 4, None, 0, 1, 2, 0, 0), b"out"),
                       (_lib.CacheAttentionArgs(_cache(), _lib.RowsView(FAKE + 2, 256, 256), FAKE, None, 0, 1, 2, 0, 0),
                        b"aligned")):
        assert lib.wamffn_cache_attention(None, ctypes.byref(args)) == 1
        assert text in lib.wamffn_last_error()


def test_workspace_query_rejects_the_same():
    lib, need = _lib.lib(), ctypes.c_size_t(7)
    args = _lib.CacheAttentionArgs(_cache(), _lib.RowsView(FAKE, 256, 256), None, None, 0, 1, 3, 0, 0)
    assert lib.wamffn_cache_attention_workspace(ctypes.byref(args), ctypes.byref(need)) == 1
    assert b"multiple" in lib.wamffn_last_error() and need.value == 0
    assert lib.wamffn_cache_attention_workspace(None, ctypes.byref(need)) == 1
    assert lib.wamffn_cache_attention_workspace(ctypes.byref(args), None) == 1


def test_python_refuses_what_it_cannot_run():
    from waminfer_b200.cache import KVCache8
    from waminfer_b200.rope import qk_norm_rope

    q, w = torch.zeros(1, 4, 256, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(q, None, w, None, None, None, 2)
    with pytest.raises(RuntimeError, match="backward"):
        qk_norm_rope(q.requires_grad_(), None, w, None, None, None, 2)
    with pytest.raises(ValueError, match="CUDA"):
        KVCache8(1, 64, 1, "cpu")
    blocks = torch.zeros(2, 1, 64, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        KVCache8.of(blocks, blocks, torch.ones(2, 1), torch.ones(2, 1), torch.zeros(1, 2, dtype=torch.int32),
                    torch.zeros(1, dtype=torch.int32))


def test_keys_without_their_weight():
    from waminfer_b200.rope import qk_norm_rope

    q, w = torch.zeros(1, 4, 256, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        qk_norm_rope(q, q, w, None, None, None, 2, 2)

"""Key / value cache in 8 bits and the attention over it, on libwamffn.

The bf16 attention ops (``waminfer_b200/attention.py``) read their cached prefix
and text context in 16 bits.  ``KVCache8`` keeps such rows in e4m3 with one
power-of-two scale for each block of 64 tokens and head: half the memory and half the
bytes an attention over them has to read.

    cache = KVCache8(batch=4, capacity=4096, kv_heads=24, device="cuda")
    cache.append(k, v)                       # [4, rows, 24 * 128] bf16, after the norm and rotation
    out = cache.attend(q, heads=24)          # [4, nq, 24 * 128]
    k, v = cache.read(120)                   # rows back as bf16, e.g. for current_frame_attention

Rows that change at every step (the current frame through the Euler updates)
are replaced in place: ``append(..., at=start)``.  Everything is on the device
(lengths, block table), so all calls can be captured into CUDA graphs.
Inference only: no backward pass.
"""

from __future__ import annotations

import ctypes

import torch
from torch._subclasses.fake_tensor import FakeTensor

from waminfer_b200 import _lib

BLOCK = 64
HEAD_DIM = 128
FORMAT = torch.float8_e4m3fn
# What a cache's calls go by from when it was made.
_FIXED = frozenset(("keys", "values", "key_scales", "value_scales", "block_table", "lengths", "batch", "width",
                    "kv_heads", "device", "_work", "_view", "_needs"))


def _no_gradients(*tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("the 8-bit cache has no backward pass: run it with gradients disabled")


def _rows(t: torch.Tensor, name: str, batch: int, width: int,
          device: torch.device) -> tuple[_lib.RowsView, torch.Tensor]:
    """View of a [batch, rows, width] bf16 operand, and the tensor it views (a
    copy if the kernels cannot read its rows in place)."""
    if t.dim() != 3 or t.dtype != torch.bfloat16 or t.device != device:
        raise ValueError(f"{name} must be a bf16 tensor [batch, rows, heads * {HEAD_DIM}] on {device}")
    count, rows, held = t.shape
    if count != batch or held != width:
        raise ValueError(f"{name} {tuple(t.shape)}: expected [{batch}, rows, {width}]")
    sb, sr, se = t.stride()
    if se != 1 or (count > 1 and sb % 8) or (rows > 1 and (sr % 8 or sr < width)) or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        sb, sr, _ = t.stride()
    return _lib.RowsView(t.data_ptr(), sr, sb), t


def _check(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if t.dtype != dtype or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on {device}, not "
                         f"{t.dtype} {list(t.shape)} on {t.device}")


def _layout(keys, values, key_scales, value_scales, block_table, lengths, work) -> _lib.CacheView:
    """The C view of a cache's tensors; work: [batch] tickets and the status word."""
    (pool, kv_heads), (batch, width) = keys.shape[:2], block_table.shape
    return _lib.CacheView(
        keys=keys.data_ptr(), values=values.data_ptr(), key_scales=key_scales.data_ptr(),
        value_scales=value_scales.data_ptr(), block_table=block_table.data_ptr(), table_stride=width,
        lengths=lengths.data_ptr(), tickets=work.data_ptr(), status=work.data_ptr() + 4 * batch,
        blocks=pool, kv_heads=kv_heads, batch=batch, width=width)


# The calls as ops on the cache's tensors, for traced code (the methods call the library directly otherwise).
@torch.library.custom_op("wam_ffn::cache_append", mutates_args=("keys", "values", "key_scales", "value_scales",
                                                                "lengths", "work"))
def _append_op(k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None, at: torch.Tensor | None,
               keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
               block_table: torch.Tensor, lengths: torch.Tensor, work: torch.Tensor) -> None:
    KVCache8._of(keys, values, key_scales, value_scales, block_table, lengths, work)._append(k, v, counts, at)


@_append_op.register_fake
def _append_fake(k, v, counts, at, keys, values, key_scales, value_scales, block_table, lengths, work):
    return None


@torch.library.custom_op("wam_ffn::cache_read", mutates_args=("work",))
def _read_op(count: int, start: torch.Tensor | None, start_all: int, keys: torch.Tensor, values: torch.Tensor,
             key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
             work: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    cache = KVCache8._of(keys, values, key_scales, value_scales, block_table, lengths, work)
    return cache._read(count, start_all if start is None else start)


@_read_op.register_fake
def _read_fake(count, start, start_all, keys, values, key_scales, value_scales, block_table, lengths, work):
    shape = (block_table.shape[0], count, keys.shape[1] * HEAD_DIM)
    return (keys.new_empty(shape, dtype=torch.bfloat16), keys.new_empty(shape, dtype=torch.bfloat16))


@torch.library.custom_op("wam_ffn::cache_attention", mutates_args=("work",))
def _attend_op(q: torch.Tensor, heads: int, causal: bool, key_split: int, keys: torch.Tensor, values: torch.Tensor,
               key_scales: torch.Tensor, value_scales: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor,
               work: torch.Tensor) -> torch.Tensor:
    cache = KVCache8._of(keys, values, key_scales, value_scales, block_table, lengths, work)
    return cache._attend(q, heads, causal, key_split)


@_attend_op.register_fake
def _attend_fake(q, heads, causal, key_split, keys, values, key_scales, value_scales, block_table, lengths, work):
    return q.new_empty(q.shape)


class KVCache8:
    """Keys and values of ``batch`` sequences in e4m3 blocks of 64 tokens, head dim 128.

    ``capacity`` rows a sequence; ``blocks`` sizes the pool (default: every
    sequence's full capacity, with a table that gives each its own blocks).  With a
    pool of its own size the caller fills ``block_table`` (int32 [batch, width])
    before rows reach those places; a block may stand in several places for reading
    (a shared prefix), one that rows are appended to in one only.

    Tensors: ``keys``, ``values`` [blocks, kv_heads, 64, 128] float8_e4m3fn;
    ``key_scales``, ``value_scales`` float32 [blocks, kv_heads], powers of two from
    2^-60 to 2^126 (a row is value * scale; of another number only the exponent
    counts, cut to that range);
    ``block_table``; ``lengths`` int32 [batch], rows held (lowering an entry drops
    rows).  They are written into, not replaced: the calls go by where they lie, so
    the attributes cannot be bound anew.  Appends to one cache must not overlap in time
    with other calls on it.
    """

    def __init__(self, batch: int, capacity: int, kv_heads: int, device, blocks: int | None = None):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the 8-bit cache lives on a CUDA device")
        if batch < 1 or capacity < 1 or kv_heads < 1 or (blocks is not None and blocks < 1):
            raise ValueError(f"batch={batch} capacity={capacity} kv_heads={kv_heads} blocks={blocks}")
        width = -(-capacity // BLOCK)
        pool = batch * width if blocks is None else blocks
        shape = (pool, kv_heads, BLOCK, HEAD_DIM)
        if blocks is None:
            table = torch.arange(pool, dtype=torch.int32, device=device).view(batch, width)
        else:
            table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self._hold(torch.zeros(shape, dtype=torch.uint8, device=device).view(FORMAT),
                   torch.zeros(shape, dtype=torch.uint8, device=device).view(FORMAT),
                   torch.ones(shape[:2], dtype=torch.float32, device=device),
                   torch.ones(shape[:2], dtype=torch.float32, device=device),
                   table, torch.zeros(batch, dtype=torch.int32, device=device))

    @classmethod
    def of(cls, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor,
           block_table: torch.Tensor, lengths: torch.Tensor) -> "KVCache8":
        """A cache over tensors that the caller holds (laid out as the class describes)."""
        return cls._of(keys, values, key_scales, value_scales, block_table, lengths, None)

    @classmethod
    def _of(cls, keys, values, key_scales, value_scales, block_table, lengths, work):
        self = cls.__new__(cls)
        self._hold(keys, values, key_scales, value_scales, block_table, lengths, work)
        return self

    def _hold(self, keys, values, key_scales, value_scales, block_table, lengths, work=None):
        if keys.dim() != 4 or not keys.is_cuda:
            raise ValueError(f"keys must be a CUDA tensor [blocks, kv_heads, {BLOCK}, {HEAD_DIM}]")
        device, (pool, kv_heads) = keys.device, keys.shape[:2]
        if block_table.dim() != 2:
            raise ValueError("block_table must be [batch, width]")
        batch, width = block_table.shape
        for name, t in (("keys", keys), ("values", values)):
            _check(name, t, FORMAT, (pool, kv_heads, BLOCK, HEAD_DIM), device)
        for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
            _check(name, t, torch.float32, (pool, kv_heads), device)
        _check("block_table", block_table, torch.int32, (batch, width), device)
        _check("lengths", lengths, torch.int32, (batch,), device)
        if min(pool, kv_heads, batch, width) < 1:
            raise ValueError("the cache is empty")
        self.keys, self.values = keys, values
        self.key_scales, self.value_scales = key_scales, value_scales
        self.block_table, self.lengths = block_table, lengths
        self.batch, self.width, self.kv_heads, self.device = batch, width, kv_heads, device
        self._needs: dict[tuple, int] = {}  # workspace of the attention, by its sizes
        self._work = torch.zeros(batch + 1, dtype=torch.int32, device=device) if work is None else work
        self._view = None if isinstance(keys, FakeTensor) else _layout(  # without data there are no addresses
            keys, values, key_scales, value_scales, block_table, lengths, self._work)

    def __setattr__(self, name, value):
        if name in _FIXED and name in self.__dict__ and value is not self.__dict__[name]:  # not x += 1, in place
            raise AttributeError(f"{name} of a cache cannot be replaced: write into it, or make another cache "
                                 "(KVCache8.of)")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        if name in _FIXED:
            raise AttributeError(f"{name} of a cache cannot be deleted")
        object.__delattr__(self, name)

    def _tensors(self):
        return (self.keys, self.values, self.key_scales, self.value_scales, self.block_table, self.lengths, self._work)

    @property
    def capacity(self) -> int:
        """Rows that a sequence can hold."""
        return self.width * BLOCK

    def _index(self, name: str, t: torch.Tensor) -> int:
        if t.dtype != torch.int32 or t.shape != self.lengths.shape or t.device != self.device or not t.is_contiguous():
            _check(name, t, torch.int32, (self.batch,), self.device)
        return t.data_ptr()

    def append(self, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor | None = None,
               at: torch.Tensor | None = None) -> None:
        """Stores k, v [batch, rows, kv_heads * 128] bf16 behind each sequence's
        rows (``at``, int32 [batch]: from that row on, replacing what was there)
        and moves ``lengths``.  ``counts`` (int32 [batch]) says how many of the
        rows are real in a padded batch.

        A block's scale is the least 2^e with |x| <= 448 * 2^e (e >= -60) over
        its finite values; infinities are stored as the largest value, NaN stays.
        When a later row raises the scale of a block, the rows in front of it are
        rounded to the new one.  A sequence whose rows do not fit (past capacity, ``at``
        beyond its length, a block id outside the pool) keeps what it had, and
        ``status`` reports it."""
        _no_gradients(k, v)
        if _lib.traced(k):
            return _append_op(k, v, counts, at, *self._tensors())
        self._append(k, v, counts, at)

    def _append(self, k, v, counts, at):
        width = self.kv_heads * HEAD_DIM
        (k_view, k), (v_view, v) = (_rows(k, "k", self.batch, width, self.device),
                                    _rows(v, "v", self.batch, width, self.device))
        if k.shape != v.shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        if k.shape[1] == 0:
            raise ValueError("append needs at least one row (counts may be zero)")
        args = _lib.CacheAppendArgs(self._view, k_view, v_view, None if counts is None else self._index(
            "counts", counts), None if at is None else self._index("at", at), k.shape[1])
        _lib.launch(_lib.lib().wamffn_cache_append, self.device.index, ctypes.byref(args))

    def read(self, count: int, start: int | torch.Tensor = 0) -> tuple[torch.Tensor, torch.Tensor]:
        """Rows [start, start + count) of every sequence as bf16, k and v
        [batch, count, kv_heads * 128]; ``start`` a number or int32 [batch].
        Rows that a sequence does not hold are zeros."""
        if _lib.traced(self.keys):
            tensor = isinstance(start, torch.Tensor)
            return _read_op(count, start if tensor else None, 0 if tensor else start, *self._tensors())
        return self._read(count, start)

    def _read(self, count, start):
        tensor = isinstance(start, torch.Tensor)
        if count < 1 or (not tensor and not 0 <= start < 2 ** 31):
            raise ValueError(f"read of {count} rows from {start}")
        k = torch.empty((self.batch, count, self.kv_heads * HEAD_DIM), dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        args = _lib.CacheReadArgs(self._view, self._index("start", start) if tensor else None, k.data_ptr(),
                                  v.data_ptr(), 0 if tensor else start, count)
        _lib.launch(_lib.lib().wamffn_cache_read, self.device.index, ctypes.byref(args))
        return k, v

    def attend(self, q: torch.Tensor, heads: int, causal: bool = False, key_split: int = 0) -> torch.Tensor:
        """softmax(q . k / sqrt(128)) . v over each sequence's rows, q [batch,
        nq, heads * 128] bf16, ``heads`` a multiple of ``kv_heads`` (query heads
        [g * heads / kv_heads, ...) share key head g).  ``causal``: the queries
        are the cache's last nq rows, query i sees rows < length - nq + i + 1 (in a
        ragged batch a sequence with fewer queries has them at the end).  A
        row that sees nothing is zeros.  NaN comes out where a row sees it: of a
        query or key in the whole of its heads, of a value in its dim.  key_split:
        CTAs of a cluster sharing a query tile's keys (0 = chosen; 1, 2, 4, 8).

        The lengths stay on the device: the work is shared out for the capacity,
        whatever the sequences hold.  Results do not depend on it, times do: 392
        queries over 577 rows of 24 heads take 18 us in a cache of 640 and 27 us in one
        of 4096, one token over them 5 to 8 us."""
        _no_gradients(q)
        if _lib.traced(q):
            return _attend_op(q, heads, causal, key_split, *self._tensors())
        return self._attend(q, heads, causal, key_split)

    def _attend(self, q, heads, causal, key_split):
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"heads={heads} must be a multiple of the cache's {self.kv_heads}")
        view, q = _rows(q, "q", self.batch, heads * HEAD_DIM, self.device)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        rows = q.shape[1]
        if rows == 0:
            return out
        args = _lib.CacheAttentionArgs(self._view, view, out.data_ptr(), None, 0, rows, heads, causal, key_split)
        held = self._parts(args, rows, heads, bool(causal), key_split)  # kept until the launch, then the stream's
        _lib.launch(_lib.lib().wamffn_cache_attention, self.device.index, ctypes.byref(args))
        return out

    def _parts(self, args, rows: int, heads: int, causal: bool, key_split: int) -> torch.Tensor | None:
        """Gives the call its workspace; few query rows over a long cache ask for one."""
        key = (rows, heads, causal, key_split)
        size = self._needs.get(key)
        if size is None:
            need = ctypes.c_size_t()
            with torch.cuda.device(self.device):
                _lib.check(_lib.lib().wamffn_cache_attention_workspace(ctypes.byref(args), ctypes.byref(need)))
            size = self._needs[key] = need.value
        if not size:
            return None
        held = torch.empty(size, dtype=torch.uint8, device=self.device)
        args.workspace, args.workspace_bytes = held.data_ptr(), size
        return held

    def status(self, clear: bool = True) -> int:
        """Device status word (timeout / bad-index bits); synchronises the device."""
        torch.cuda.synchronize(self.device)  # the calls may be on other streams than the copy below
        value = int(self._work[self.batch])
        if clear and value:
            self._work[self.batch:].zero_()
        return value

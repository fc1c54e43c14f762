"""Query / key norm and position rotation in one pass, on libwamffn.

What runs between the QKV projection (``waminfer_b200/projections.py``) and the
attention ops (``waminfer_b200/attention.py``); the reference's form, whole-row
RMSNorm + RoPE on interleaved pairs, is ``WAMInfer/_triton_inference.py:13-112``.

    q, k, v = projections.qkv(layer, normalized).chunk(3, dim=-1)
    q, k = qk_norm_rope(q, k, attn.norm_q.weight, attn.norm_k.weight, freqs, None, 24, 24)

fp32 inside, one rounding to bf16 at the end.  Inference only, like the rest of
the library: no backward pass.
"""

from __future__ import annotations

import ctypes

import torch

from waminfer_b200 import _lib


def _check_side(x, weight, heads, name):
    """Head dim of q or k after its checks."""
    if x.dim() != 3 or x.dtype != torch.bfloat16 or not x.is_cuda:
        raise ValueError(f"{name} must be a bf16 CUDA tensor [batch, rows, heads * head_dim]")
    width = x.shape[2]
    if heads < 1 or width % heads:
        raise ValueError(f"{name} {tuple(x.shape)} does not hold {heads} heads")
    dim = width // heads
    if weight.dtype != torch.bfloat16 or weight.dim() != 1 or weight.numel() not in (dim, width) or \
            not weight.is_contiguous() or weight.device != x.device:
        raise ValueError(f"{name}_weight must be a contiguous bf16 vector of {dim} (each head) or {width} "
                         f"(the row) on {x.device}")
    return dim


def _in_place(x):
    """Whether the kernel can read the rows of q or k as they lie (but for the start's alignment)."""
    sb, sr, se = x.stride()
    return se == 1 and (sb % 8 == 0 or x.shape[0] <= 1) and (x.shape[1] <= 1 or (sr % 8 == 0 and sr >= x.shape[2]))


def _checked(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved):
    """The call's arguments without its pointers, after all checks of shapes, types and devices."""
    dim = _check_side(q, q_weight, heads, "q")
    batch, rows, width = q.shape
    whole = q_weight.numel() != dim
    if k is not None:
        if k_weight is None:
            raise ValueError("k needs k_weight")
        if _check_side(k, k_weight, kv_heads, "k") != dim or k.shape[:2] != q.shape[:2] or k.device != q.device:
            raise ValueError(f"q {tuple(q.shape)} ({heads} heads) and k {tuple(k.shape)} ({kv_heads} heads) differ in "
                             "batch, rows, head dim or device")
        whole = whole or k_weight.numel() != dim
        if whole and (q_weight.numel() != width or k_weight.numel() != k.shape[2]):
            raise ValueError("q_weight and k_weight must both be for each head or both for the row")
    args = _lib.QkRopeArgs(batch=batch, rows=rows, heads=heads, kv_heads=0 if k is None else kv_heads, head_dim=dim,
                           whole_row=whole, interleaved=interleaved, eps=eps)
    if rope is not None:
        if rope.dtype != torch.complex64 or rope.device != q.device or not (
                rope.dim() == 2 or (rope.dim() == 3 and rope.shape[1] == 1)) or rope.stride(-1) != 1:
            raise ValueError(f"rope must be a complex64 table [positions, pairs] (or [positions, 1, pairs]) on {q.device}")
        args.table_stride, args.table_rows, args.pairs = rope.stride(0), rope.shape[0], rope.shape[-1]
        if positions is not None:
            if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device or \
                    tuple(positions.shape) not in ((rows,), (batch, rows)):
                raise ValueError(f"positions must be int32 or int64, [{rows}] or [{batch}, {rows}], on {q.device}")
            args.position_bytes = positions.element_size()
            args.position_stride = positions.stride(0) if positions.dim() == 2 else 0
    elif positions is not None:
        raise ValueError("positions without a rope table")
    plain = _in_place(q) and (k is None or _in_place(k)) and (rope is None or rope.stride(0) % 2 == 0) and (
        positions is None or rows <= 1 or positions.stride(-1) == 1)
    return bytes(args), plain, q.device.index


# What _checked found for the shapes, strides and types of a call; a decode loop makes the same one over and over.
_CHECKED: dict[tuple, tuple] = {}


def _layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _run(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved):
    if rope is not None and rope.is_conj():  # before anything looks at its strides: the copy may have others
        rope = rope.resolve_conj()
    key = (_layout(q), _layout(k), _layout(q_weight), _layout(k_weight), _layout(rope), _layout(positions), heads,
           kv_heads, eps, interleaved)
    found = _CHECKED.get(key)
    if found is None:
        if len(_CHECKED) >= 4096:
            _CHECKED.clear()
        found = _CHECKED[key] = _checked(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)
    raw, plain, device = found
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    if not plain:  # rows that the kernel cannot read as they lie: copies of them
        if q.numel() == 0:
            return q_out, k_out
        q, k = q.contiguous(), None if k is None else k.contiguous()
        rope = None if rope is None else rope.contiguous()
        positions = None if positions is None else positions.contiguous()
        args = _lib.QkRopeArgs.from_buffer_copy(
            _checked(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)[0])
    else:
        args = _lib.QkRopeArgs.from_buffer_copy(raw)
        if not args.rows * args.batch:
            return q_out, k_out
    q, q_weight = _aligned(q), _aligned(q_weight)
    sb, sr, _ = q.stride()
    args.q = _lib.RowsView(q.data_ptr(), sr, sb)
    args.q_weight, args.q_out = q_weight.data_ptr(), q_out.data_ptr()
    if k is not None:
        k, k_weight = _aligned(k), _aligned(k_weight)
        sb, sr, _ = k.stride()
        args.k = _lib.RowsView(k.data_ptr(), sr, sb)
        args.k_weight, args.k_out = k_weight.data_ptr(), k_out.data_ptr()
    if rope is not None:
        table = _aligned(rope)
        if table is not rope:
            args.table_stride = table.stride(0)
        args.rope = table.data_ptr()
        if positions is not None:
            args.positions = positions.data_ptr()
    _lib.launch(_lib.lib().wamffn_qk_norm_rope, device, ctypes.byref(args))
    return q_out, k_out


@torch.library.custom_op("wam_ffn::qk_norm_rope", mutates_args=())
def _op(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, rope: torch.Tensor | None,
        positions: torch.Tensor | None, heads: int, kv_heads: int, eps: float,
        interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _run(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)


@_op.register_fake
def _fake(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


@torch.library.custom_op("wam_ffn::q_norm_rope", mutates_args=())
def _alone_op(q: torch.Tensor, q_weight: torch.Tensor, rope: torch.Tensor | None, positions: torch.Tensor | None,
              heads: int, eps: float, interleaved: bool) -> torch.Tensor:
    return _run(q, None, q_weight, None, rope, positions, heads, 0, eps, interleaved)[0]


@_alone_op.register_fake
def _alone_fake(q, q_weight, rope, positions, heads, eps, interleaved):
    return q.new_empty(q.shape)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor, k_weight: torch.Tensor | None,
                 rope: torch.Tensor | None, positions: torch.Tensor | None, heads: int, kv_heads: int = 0,
                 eps: float = 1e-6, interleaved: bool = True) -> tuple[torch.Tensor, torch.Tensor | None]:
    """RMS norm of q [batch, rows, heads * head_dim] and k [batch, rows,
    kv_heads * head_dim] and their rotation; returns contiguous (q', k').

    Weights of head_dim values norm each head, of the row's width the whole row
    (the DiT's form).  ``rope`` is a complex64 table [positions, pairs] of
    cos + i sin (``[positions, 1, pairs]`` as the reference passes it), with
    pairs <= head_dim / 2 a multiple of 4; head dims past 2 * pairs are not
    turned; None turns nothing.  Pair i is dims (2i, 2i + 1) when
    ``interleaved``, else (i, i + pairs).  ``positions`` (int32 / int64, [rows]
    or [batch, rows]) picks each row's table entry, None the row's index; one
    outside the table gives a row of NaN.  head_dim 64, 128 or 256.  ``k`` may
    be None (a cross-attention query).
    """
    if torch.is_grad_enabled() and (q.requires_grad or q_weight.requires_grad or (
            rope is not None and rope.requires_grad) or (k is not None and (
                k.requires_grad or (k_weight is not None and k_weight.requires_grad)))):
        raise RuntimeError("qk_norm_rope has no backward pass: run it with gradients disabled")
    if _lib.traced(q):
        if k is None:
            return _alone_op(q, q_weight, rope, positions, heads, eps, interleaved), None
        if k_weight is None:
            raise ValueError("k needs k_weight")
        return _op(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)
    return _run(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)

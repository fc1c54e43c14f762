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


def _side(x, weight, heads, name):
    """Head dim, strides and the operand itself (a copy if the kernel cannot read its rows in place) of q or k."""
    if x.dim() != 3 or x.dtype != torch.bfloat16 or not x.is_cuda:
        raise ValueError(f"{name} must be a bf16 CUDA tensor [batch, rows, heads * head_dim]")
    _, rows, width = x.shape
    if heads < 1 or width % heads:
        raise ValueError(f"{name} {tuple(x.shape)} does not hold {heads} heads")
    dim, n = width // heads, weight.numel()
    if weight.dtype != torch.bfloat16 or weight.dim() != 1 or (n != dim and n != width) or \
            not weight.is_contiguous() or weight.device != x.device:
        raise ValueError(f"{name}_weight must be a contiguous bf16 vector of {dim} (each head) or {width} "
                         f"(the row) on {x.device}")
    sb, sr, se = x.stride()
    if se != 1 or sb % 8 or sr % 8 or x.data_ptr() % 16 or (sr < width and rows > 1):
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        sb, sr, _ = x.stride()
    return dim, _lib.RowsView(x.data_ptr(), sr, sb), x


def _vector(w):
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _run(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved):
    dim, q_view, q_held = _side(q, q_weight, heads, "q")
    batch, rows, width = q.shape
    device = q.device
    whole = q_weight.numel() != dim
    k_view, k_at, k_out = _lib.RowsView(), None, None
    if k is not None:
        if k_weight is None:
            raise ValueError("k needs k_weight")
        k_dim, k_view, k_held = _side(k, k_weight, kv_heads, "k")
        if k_dim != dim or k.shape[:2] != q.shape[:2] or k.device != device:
            raise ValueError(f"q {tuple(q.shape)} ({heads} heads) and k {tuple(k.shape)} ({kv_heads} heads) differ in "
                             "batch, rows, head dim or device")
        whole = whole or k_weight.numel() != dim
        if whole and (q_weight.numel() != width or k_weight.numel() != k.shape[2]):
            raise ValueError("q_weight and k_weight must both be for each head or both for the row")
        k_weight = _vector(k_weight)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        k_at = k_out.data_ptr()
    else:
        kv_heads = 0
    table = places = None
    table_stride = table_rows = pairs = place_bytes = place_stride = 0
    if rope is not None:
        shape = rope.shape
        if rope.dtype != torch.complex64 or rope.device != device or not (
                len(shape) == 2 or (len(shape) == 3 and shape[1] == 1)) or rope.stride(-1) != 1:
            raise ValueError(f"rope must be a complex64 table [positions, pairs] (or [positions, 1, pairs]) on {device}")
        if rope.is_conj():
            rope = rope.resolve_conj()
        table, table_stride, table_rows, pairs = rope.data_ptr(), rope.stride(0), shape[0], shape[-1]
        if table % 16 or table_stride % 2:
            rope = rope.clone(memory_format=torch.contiguous_format)
            table, table_stride = rope.data_ptr(), rope.stride(0)
        if positions is not None:
            shape, kind = positions.shape, positions.dtype
            if (kind != torch.int32 and kind != torch.int64) or positions.device != device or (
                    shape != (batch, rows) and shape != (rows,)):
                raise ValueError(f"positions must be int32 or int64, [{rows}] or [{batch}, {rows}], on {device}")
            if rows > 1 and positions.stride(-1) != 1:
                positions = positions.contiguous()
            places, place_bytes = positions.data_ptr(), 4 if kind == torch.int32 else 8
            place_stride = positions.stride(0) if len(shape) == 2 else 0
    elif positions is not None:
        raise ValueError("positions without a rope table")
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if q.numel() == 0:
        return q_out, k_out
    q_weight = _vector(q_weight)
    args = _lib.QkRopeArgs(q_view, k_view, q_weight.data_ptr(), None if k is None else k_weight.data_ptr(), table,
                           table_stride, places, place_stride, q_out.data_ptr(), k_at, place_bytes, table_rows, pairs,
                           batch, rows, heads, kv_heads, dim, whole, interleaved, eps)
    _lib.launch(_lib.lib().wamffn_qk_norm_rope, device.index, ctypes.byref(args))
    return q_out, k_out


@torch.library.custom_op("wam_ffn::qk_norm_rope", mutates_args=())
def _op(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, rope: torch.Tensor | None,
        positions: torch.Tensor | None, heads: int, kv_heads: int, eps: float,
        interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _run(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)


@_op.register_fake
def _fake(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved):
    return q.new_empty(q.shape), k.new_empty(k.shape)


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
    if torch.is_grad_enabled() and (q.requires_grad or q_weight.requires_grad or (k is not None and (
            k.requires_grad or k_weight.requires_grad))):
        raise RuntimeError("qk_norm_rope has no backward pass: run it with gradients disabled")
    if k is not None and torch.compiler.is_compiling():
        return _op(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)
    return _run(q, k, q_weight, k_weight, rope, positions, heads, kv_heads, eps, interleaved)

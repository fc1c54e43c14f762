"""GPU: query / key norm with the position rotation (``waminfer_b200/rope.py``)
against the formula in 64 bits.

Tolerance: the result is rounded once, half a bf16 step (2^-8 of the value);
before that it is fp32: the norm's factor (a sum of up to 2^15 squares in a
tree, rsqrt, two products) is within 2^-20 of its value, and so are the two
products of the rotation, whose sum may cancel: 2^-20 (|y_a| + |y_b|)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, w, turn, heads, eps, interleaved):
    """(y, the tolerance's |y_a| + |y_b|) in float64; turn [batch, rows, pairs] complex128 or None."""
    batch, rows, width = x.shape
    dim = width // heads
    x, w = x.double(), w.double()
    if w.numel() == dim:
        v = x.view(batch, rows, heads, dim)
        y = v / ((v * v).mean(-1, keepdim=True) + eps).sqrt() * w
    else:
        y = (x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * w).view(batch, rows, heads, dim)
    size = y.abs()
    if turn is not None:
        r = turn.shape[-1]
        a, b = (y[..., 0:2 * r:2], y[..., 1:2 * r:2]) if interleaved else (y[..., :r], y[..., r:2 * r])
        c, s = turn.real[:, :, None], turn.imag[:, :, None]
        both = a.abs() + b.abs()
        turned = (a * c - b * s, a * s + b * c)
        size = size.clone()
        if interleaved:
            y = torch.cat((torch.stack(turned, -1).flatten(-2), y[..., 2 * r:]), -1)
            size[..., :2 * r] = both.repeat_interleave(2, -1)
        else:
            y = torch.cat((*turned, y[..., 2 * r:]), -1)
            size[..., :2 * r] = torch.cat((both, both), -1)
    return y.flatten(2), size.flatten(2)


def check(got, ref):
    y, size = ref
    off = (got.double() - y).abs() - (2.0 ** -8 * y.abs() + 2.0 ** -20 * size)
    assert off.max().item() <= 0, off.max().item()


def table(positions, pairs, dev):
    inverse = 10000.0 ** (-torch.arange(pairs, device=dev, dtype=torch.float64) / pairs)
    angles = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * inverse
    return torch.polar(torch.ones_like(angles), angles).to(torch.complex64)


def case(dev, seed, batch, rows, heads, kv_heads, dim, whole):
    g = torch.Generator(device=dev).manual_seed(seed)
    packed = torch.randn(batch, rows, (heads + 2 * kv_heads) * dim, device=dev, generator=g).bfloat16()
    q, k = packed[..., :heads * dim], packed[..., heads * dim:(heads + kv_heads) * dim]
    qw, kw = ((1 + 0.2 * torch.randn(h * dim if whole else dim, device=dev, generator=g)).bfloat16()
              for h in (heads, kv_heads))
    return q, k, qw, kw, g


@pytest.mark.parametrize("batch,rows,heads,kv_heads,dim,whole,interleaved,pairs,where", [
    (1, 392, 24, 24, 128, True, True, 64, "index"),    # the DiT's joint sequence
    (1, 1, 24, 24, 128, True, True, 64, "row"),        # one token
    (1, 1, 1, 1, 64, False, False, 32, "both"),
    (3, 77, 5, 1, 64, False, True, 32, "both"),
    (2, 129, 8, 2, 256, False, False, 128, "row"),
    (2, 40, 16, 4, 256, True, False, 128, "both"),     # 5120 elements: four vectors a thread
    (1, 9, 100, 28, 256, True, True, 64, "row"),       # 32768 elements, the widest row; half the dims turned
    (2, 1000, 40, 8, 128, False, False, 64, "both"),   # several heads a group of lanes
    (2, 1000, 7, 3, 128, False, True, 4, "index"),     # a short last group, 8 dims turned
    (1, 33, 3, 3, 128, True, False, 20, "row"),
    (2, 50, 6, 6, 128, False, True, 0, "index"),       # no rotation
])
def test_against_the_formula(cuda_device, batch, rows, heads, kv_heads, dim, whole, interleaved, pairs, where):
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, g = case(cuda_device, rows + heads, batch, rows, heads, kv_heads, dim, whole)
    freqs = table(100000, pairs, cuda_device) if pairs else None
    positions = None
    at = torch.arange(rows, device=cuda_device).expand(batch, rows)
    if where == "row":
        positions = torch.randint(0, 100000, (rows,), device=cuda_device, generator=g)
        at = positions.expand(batch, rows)
    elif where == "both":
        at = torch.randint(0, 100000, (batch, rows), device=cuda_device, generator=g)
        positions = at.to(torch.int32)
    turn = freqs[at].to(torch.complex128) if pairs else None
    got = qk_norm_rope(q, k, qw, kw, freqs, positions, heads, kv_heads, 1e-6, interleaved)
    check(got[0], reference(q, qw, turn, heads, 1e-6, interleaved))
    check(got[1], reference(k, kw, turn, kv_heads, 1e-6, interleaved))
    assert got[0].is_contiguous() and got[1].is_contiguous()


def test_extremes(cuda_device):
    """Rows of zeros, of the smallest and of large values; infinities and NaN stay in their row (and head)."""
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, _ = case(cuda_device, 3, 1, 6, 4, 2, 128, False)
    q = q.clone()
    q[0, 0] = 0
    q[0, 1] = 1e-30
    q[0, 2] *= 1e15
    q[0, 3, :128] = float("inf")
    q[0, 4, 200] = float("nan")
    freqs = table(6, 64, cuda_device)
    turn = freqs[None].to(torch.complex128)
    out, _ = qk_norm_rope(q, k, qw, kw, freqs, None, 4, 2)
    y, size = reference(q, qw, turn, 4, 1e-6, True)
    bad = torch.zeros(6, 4, dtype=torch.bool, device=cuda_device)
    bad[3, 0] = bad[4, 1] = True
    wrong = out.view(6, 4, 128).isnan().any(-1)
    assert torch.equal(wrong, bad)
    keep = ~bad[:, :, None].expand(6, 4, 128).reshape(1, 6, 512)
    check(torch.where(keep, out, 0), (torch.where(keep, y, 0), torch.where(keep, size, 0)))


def test_queries_alone_views_and_positions_outside(cuda_device):
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, _ = case(cuda_device, 5, 2, 30, 4, 4, 128, True)
    freqs = table(100, 64, cuda_device)
    turn = freqs[:30][None].to(torch.complex128).expand(2, 30, 64)
    both = qk_norm_rope(q, k, qw, kw, freqs, None, 4, 4)
    alone, none = qk_norm_rope(q, None, qw, None, freqs[:, None], None, 4)  # the reference's [rows, 1, pairs] table
    assert none is None and torch.equal(alone, both[0])
    # Rows in another order, every second row, an unaligned start, a strided table and strided positions.
    shifted = torch.empty(2 * 30 * 512 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(2, 30, 512)
    shifted.copy_(q)
    wide = torch.zeros(100, 131, dtype=torch.complex64, device=cuda_device)
    wide[:, :64] = freqs
    assert torch.equal(qk_norm_rope(shifted, None, qw, None, wide[:, :64], None, 4)[0], alone)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(qk_norm_rope(swapped, None, qw, None, freqs, None, 4)[0], alone)
    positions = torch.arange(60, device=cuda_device)[::2]
    check(qk_norm_rope(q, None, qw, None, freqs, positions, 4)[0],
          reference(q, qw, freqs[positions][None].to(torch.complex128).expand(2, 30, 64), 4, 1e-6, True))
    # A position outside the table: NaN in that row, the others untouched.
    positions = torch.arange(30, device=cuda_device, dtype=torch.int32).repeat(2, 1)
    positions[0, 3], positions[1, 7] = -1, 100
    out, _ = qk_norm_rope(q, None, qw, None, freqs, positions, 4)
    rows = out.isnan()
    assert rows[0, 3].all() and rows[1, 7].all() and int(rows.sum()) == 2 * 512
    keep = ~rows
    assert torch.equal(out[keep], alone[keep])
    assert qk_norm_rope(q[:, :0], None, qw, None, freqs, None, 4)[0].shape == (2, 0, 512)


def test_conjugated_table_of_wider_rows(cuda_device):
    """A lazily conjugated slice: turned the other way, by the slice's own entries."""
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, _ = case(cuda_device, 11, 2, 30, 4, 4, 128, True)
    wide = table(30, 96, cuda_device)
    back = wide.conj()[:, :64]
    assert back.is_conj()
    turn = wide[:, :64].conj().resolve_conj()[None].to(torch.complex128).expand(2, 30, 64)
    for rope in (back, back[:, None]):
        check(qk_norm_rope(q, None, qw, None, rope, None, 4)[0], reference(q, qw, turn, 4, 1e-6, True))


def test_a_single_batch_row_or_table_row_of_any_stride(cuda_device):
    from waminfer_b200.rope import qk_norm_rope

    q, _, qw, _, _ = case(cuda_device, 12, 1, 30, 4, 4, 128, True)
    freqs = table(30, 64, cuda_device)
    held = torch.zeros(1, 30 * 512 + 5, dtype=torch.bfloat16, device=cuda_device)
    held[:, :30 * 512] = q.reshape(1, -1)
    expect = qk_norm_rope(q, None, qw, None, freqs, None, 4)[0]
    view = held.as_strided((1, 30, 512), (held.shape[1], 512, 1))
    assert view.stride(0) % 8 and torch.equal(qk_norm_rope(view, None, qw, None, freqs, None, 4)[0], expect)
    odd = torch.zeros(1, 1, 513, dtype=torch.bfloat16, device=cuda_device)
    odd[..., :512] = q[:, :1]
    one = torch.zeros(1, 65, dtype=torch.complex64, device=cuda_device)
    one[:, :64] = freqs[:1]
    assert torch.equal(qk_norm_rope(odd[..., :512], None, qw, None, one[:, :64], None, 4)[0], expect[:, :1])


def test_captured_and_on_another_stream(cuda_device):
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, g = case(cuda_device, 6, 2, 200, 8, 2, 128, False)
    q, k = q.clone(), k.clone()
    freqs = table(300, 64, cuda_device)
    positions = torch.arange(100, 300, device=cuda_device)
    call = lambda: qk_norm_rope(q, k, qw, kw, freqs, positions, 8, 2)  # noqa: E731
    expect = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(there[0], expect[0]) and torch.equal(there[1], expect[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    q.copy_(torch.randn(q.shape, device=cuda_device, generator=g))
    graph.replay()
    expect = call()
    assert torch.equal(held[0], expect[0]) and torch.equal(held[1], expect[1])


@pytest.mark.parametrize("whole", [False, True])
def test_offsets_past_32_bits(cuda_device, whole):
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, g = case(cuda_device, 9, 1, 1, 32, 4, 64, whole)
    q = torch.randn(1, 1 << 20, 2048, device=cuda_device, generator=g, dtype=torch.bfloat16)  # 2^31 elements
    q = torch.cat((q, q[:, :700]), 1)
    freqs = table(1 << 21, 32, cuda_device)
    out, _ = qk_norm_rope(q, None, qw, None, freqs, None, 32)
    at = torch.arange(q.shape[1] - 700, q.shape[1], device=cuda_device)
    check(out[:, -700:], reference(q[:, -700:], qw, freqs[at][None].to(torch.complex128), 32, 1e-6, True))


def test_the_reference_on_the_same_rows(cuda_device):
    """The reference's rounding points (bf16 after the norm and after the weight) move a value by up to
    three half steps: 3 * 2^-8 of it and of its pair."""
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, _ = case(cuda_device, 8, 1, 392, 24, 24, 128, True)
    freqs = table(392, 64, cuda_device)
    out, _ = qk_norm_rope(q, k, qw, kw, freqs[:, None], None, 24, 24)
    x = q.float()
    n = (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).bfloat16() * qw
    z = torch.view_as_complex(n.double().view(1, 392, 24, 64, 2)) * freqs.to(torch.complex128)[None, :, None]
    y = torch.view_as_real(z).flatten(-3).flatten(2).bfloat16().double().view(1, 392, -1)
    size = z.abs().repeat_interleave(2, -1).flatten(2) * 2 ** 0.5  # |y_a| + |y_b| <= sqrt(2) |z|
    assert ((out.double() - y).abs() <= 4 * 2.0 ** -8 * size + 1e-30).all()

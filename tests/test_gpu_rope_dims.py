"""GPU: dims that the rotation leaves alone keep to themselves (``waminfer_b200/rope.py``); reference and tolerance of
``test_gpu_rope.py``."""

import pytest
import torch
from test_gpu_rope import case, reference, table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,pairs", [(128, 0), (128, 20), (64, 4), (256, 64), (128, 64)])
def test_special_values_stay_in_their_pair(cuda_device, dim, pairs, interleaved, whole):
    """Infinities and NaN in a weight or in a row: a dim past the turned ones, or any without a table, has no partner
    that they could reach."""
    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, _ = case(cuda_device, 21, 2, 9, 3, 2, dim, whole)
    q, qw = q.clone(), qw.clone()
    heads = 3 if whole else 1
    for at, value in ((dim - 1, float("inf")), (2 * pairs, float("nan")), (1, -float("inf")), (dim // 2, float("nan"))):
        if at < dim:
            qw.view(heads, dim)[-1, at] = value
    q[0, 2, dim - 2] = float("inf")
    q[1, 5, 2 * dim + 6] = -float("inf")
    q[1, 6, 3] = float("nan")
    freqs = table(9, pairs, cuda_device) if pairs else None
    turn = freqs[None].to(torch.complex128).expand(2, 9, pairs) if pairs else None
    got, _ = qk_norm_rope(q, k, qw, kw, freqs, None, 3, 2, 1e-6, interleaved)
    y, size = reference(q, qw, turn, 3, 1e-6, interleaved)
    got = got.double()
    assert torch.equal(got.isnan(), y.isnan())
    assert torch.equal(torch.where(got.isinf(), got, 0.0), torch.where(y.isinf(), y, 0.0))
    off = torch.where(y.isfinite(), (got - y).abs() - (2.0 ** -8 * y.abs() + 2.0 ** -20 * size), 0.0)
    assert off.nan_to_num(1.0).max().item() <= 0


def test_queries_alone_traced(cuda_device):
    """The cross-attention form inside a compiled function, with and without a table, and recorded by a tracer on
    tensors with data."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from waminfer_b200.rope import qk_norm_rope

    q, k, qw, kw, g = case(cuda_device, 4, 2, 7, 4, 2, 128, False)
    freqs = table(20, 64, cuda_device)
    positions = torch.randint(0, 20, (2, 7), device=cuda_device, generator=g)

    def step(q):
        return (qk_norm_rope(q, None, qw, None, freqs, positions, 4, eps=1e-5)[0],
                qk_norm_rope(q, None, qw, None, None, None, 4)[0] * 1.0,
                *qk_norm_rope(q, k, qw, kw, freqs, None, 4, 2, interleaved=False))

    with torch.no_grad():
        plain = step(q)
        traced = torch.compile(step, backend="aot_eager", fullgraph=True)(q)
        recorded = make_fx(step)(q)
        other = torch.randn(q.shape, device=cuda_device, generator=g).bfloat16()
        again = recorded(other)
        expect = step(other)
    for a, b in zip((*plain, *expect), (*traced, *again)):
        assert torch.equal(a, b)

"""CPU: what the norm + rotation and the 8-bit cache refuse or trace, on tensors without data."""

import pytest
import torch


def test_a_table_that_wants_gradients_is_refused():
    """No backward pass: like the rows and weights, the table must not be left without its gradient in silence."""
    from waminfer_b200.rope import qk_norm_rope

    q, w = torch.zeros(1, 4, 256, dtype=torch.bfloat16), torch.ones(128, dtype=torch.bfloat16)
    rope = torch.zeros(4, 64, dtype=torch.complex64, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward"):
        qk_norm_rope(q, None, w, None, rope, None, 2)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(q, None, w, None, rope, None, 2)


def calls(x, cache, w, rope, at):
    """Every form of the calls, on [2, 5, 512] rows."""
    from waminfer_b200.rope import qk_norm_rope

    q, k = qk_norm_rope(x, x[..., :256], w, w, rope, None, 4, 2)
    alone, none = qk_norm_rope(x, None, w, None, rope, None, 4)
    assert none is None
    cache.append(k, k)
    cache.append(k, k, counts=at, at=at)
    return (q, k, alone, cache.attend(q, 4), cache.attend(alone, 4, causal=True, key_split=2), *cache.read(3),
            *cache.read(7, start=at))


def fakes():
    from waminfer_b200.cache import KVCache8

    make = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
    return (make(2, 5, 512), KVCache8(2, 100, 2, "cuda"), make(128), make(5, 64, dtype=torch.complex64),
            make(2, dtype=torch.int32))


SHAPES = [(2, 5, 512), (2, 5, 256), (2, 5, 512), (2, 5, 512), (2, 5, 512), (2, 3, 256), (2, 3, 256), (2, 7, 256),
          (2, 7, 256)]


def test_calls_on_tensors_without_data():
    """Shape propagation outside the compiler, as the library's other ops have it."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        out = calls(*fakes())
    assert [tuple(t.shape) for t in out] == SHAPES
    assert all(t.dtype == torch.bfloat16 and t.is_cuda and t.is_contiguous() for t in out)


def test_calls_are_recorded_by_a_tracer():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    with FakeTensorMode():
        x, cache, w, rope, at = fakes()
        graph = make_fx(lambda x: calls(x, cache, w, rope, at))(x).graph
    names = [str(n.target).split(".")[1] for n in graph.nodes if str(n.target).startswith("wam_ffn.")]
    assert names == ["qk_norm_rope", "q_norm_rope", "cache_append", "cache_append", "cache_attention",
                     "cache_attention", "cache_read", "cache_read"]


def test_gradients_are_refused_in_traced_calls_too():
    """A traced append would take the rows and lose their gradient."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, cache, *_ = fakes()
        k = x[..., :256].contiguous()
        wants = k.clone().requires_grad_()
        for call in (lambda: cache.append(wants, k), lambda: cache.append(k, wants), lambda: cache.attend(wants, 2)):
            with pytest.raises(RuntimeError, match="backward"):
                call()
        with torch.no_grad():
            cache.append(wants, wants)
            assert cache.attend(wants, 2).shape == wants.shape


def test_a_cache_takes_attributes_of_the_program():
    """Only what the calls go by is fixed."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        _, cache, *_ = fakes()
    cache.step = 0
    cache.step += 1
    assert cache.step == 1
    del cache.step
    assert not hasattr(cache, "step")
    for name in ("lengths", "batch", "_view"):
        with pytest.raises(AttributeError, match=name):
            setattr(cache, name, object())
        with pytest.raises(AttributeError, match=name):
            delattr(cache, name)

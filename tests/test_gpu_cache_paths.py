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

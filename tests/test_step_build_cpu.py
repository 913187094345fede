"""gkv_step_build, gkv_mrope_* and gkv_prompt_attention without a GPU: refusals of the C ABI and the axis tables."""
import ctypes as C

import numpy as np
import pytest

import glacier_kv as G
from glacier_kv import _lib


def _meta_pool():
    return G.PagedBlockPool(8, 1, 2, 64, 16, allocate_device_arena=False)


def test_device_calls_refuse_missing_pools_and_arenas():
    lib = _lib.lib
    io, qkv, rope, prompt = _lib.gkv_step_io(), _lib.gkv_qkv_io(), _lib.gkv_mrope_desc(), _lib.gkv_prompt_desc()
    pool = _meta_pool()
    for h, code in ((None, _lib.GKV_EINVAL), (pool.handle, _lib.GKV_ESTATE)):
        assert lib.gkv_step_build(h, C.byref(io), 0, None) == code
        assert lib.gkv_mrope_append(h, 0, C.byref(qkv), 0, 2, None, 0, C.byref(rope), None, None) == code
        assert lib.gkv_prompt_attention(h, C.byref(prompt), None) == code
        assert _lib.last_error()
    pool.close()


@pytest.mark.parametrize("sections,rope_dim,interleaved,want", [
    ([4, 2, 2], 16, False, [0, 0, 0, 0, 1, 1, 2, 2]),
    ([4, 2, 2], 16, True, [0, 1, 2, 0, 1, 2, 0, 0]),
    ([0, 4, 4], 16, False, [1, 1, 1, 1, 2, 2, 2, 2]),
    ([8], 16, False, [0] * 8),
    ([8], 16, True, [0] * 8),
    ([2, 2, 2, 2], 16, True, [0, 1, 2, 3, 0, 1, 2, 3]),
    ([1, 3], 8, True, [0, 1, 0, 1]),  # axis 1 takes i % 2 == 1 as long as i < 6
])
def test_axis_tables(sections, rope_dim, interleaved, want):
    rope = G.MultiAxisRope(sections, rope_dim, interleaved=interleaved)
    assert rope.axis[:rope_dim // 2].tolist() == want
    assert np.array_equal(rope.inv_freq, G.rope_inv_freq(10000.0, rope_dim))


@pytest.mark.parametrize("sections,rope_dim", [([4, 2, 3], 16), ([4, 2, 2], 15), ([-1, 5, 4], 16), ([8, 0, 0, 0, 0], 16), ([], 16),
                                               ([200, 56], 512), ([8], -16), ([0], 0)])
def test_axis_table_refusals(sections, rope_dim):
    with pytest.raises(G.ArgumentOutOfRangeError):
        G.MultiAxisRope(sections, rope_dim)


def test_frequency_count_is_checked():
    with pytest.raises(G.ArgumentOutOfRangeError):
        G.MultiAxisRope([4, 2, 2], 16, inv_freq=np.ones(7, np.float32))


def test_step_buffers_refuse_host_tensors():
    import torch

    t = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        G.StepBuffers(torch.zeros(3, 4, dtype=torch.int32), t, t, t, max_tokens=3)

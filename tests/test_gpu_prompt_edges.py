"""gkv_prompt_attention at the edges of what its documentation allows: alignment, scores of minus infinity, bad ranges."""
import math

import pytest

import glacier_kv as G
from operator_refs import assert_within, prompt_reference, prompt_tolerance
from test_gpu_prompt_attention import _inputs, _kind

pytestmark = pytest.mark.gpu


def _at(offset, shape, dtype, mark):
    """(buffer, dense tensor of `shape` that starts `offset` elements into it, with room behind)."""
    import torch

    n = math.prod(shape)
    buf = torch.full((offset + n + 64,), mark, dtype=dtype, device="cuda")
    return buf, buf[offset:offset + n].view(shape)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 128), ("bf16", 64), ("f16", 64), ("f32", 128), ("bf16", 96)])
@pytest.mark.parametrize("sixteens", [0, 1, 2, 3])
def test_rows_on_any_16_byte_boundary(cuda, dtype, d, sixteens):
    """q, k, v and out at every 16-byte boundary, lse at odd floats: nothing beside the rows is written."""
    import torch

    kind, h, hk = _kind(dtype), 4, 2
    off = sixteens * 16 // torch.empty(0, dtype=kind).element_size()
    q, k, v, cu = _inputs([200, 3, 129], h, hk, d, d, dtype, seed=21)
    n = q.shape[0]
    moved = []
    for x in (q, k, v):
        _, y = _at(off, x.shape, kind, 0.0)
        y.copy_(x)
        moved.append(y)
    buf, out = _at(off, (n, h, d), kind, 7.0)
    lbuf, lse = _at(sixteens, (n, h), torch.float32, 7.0)
    assert out.data_ptr() % 16 == 0 and out.data_ptr() % 64 == 16 * sixteens
    pool = G.PagedBlockPool(1, 1, hk, d, 16)
    pool.prompt_attention(*moved, torch.tensor(cu, device="cuda"), out, 1 / math.sqrt(d), lse=lse)
    pool.sync()
    pool.close()
    ref, rlse, size, most = prompt_reference(q, k, v, [int(c) for c in cu], 1 / math.sqrt(d))
    tol, ltol = prompt_tolerance(ref, size, most, d, 200, kind)
    assert_within(out, ref, tol, "out")
    assert_within(lse, rlse, ltol + 2.0 ** -23 * rlse.abs(), "lse")
    for b, o, m in ((buf, off, out.numel()), (lbuf, sixteens, lse.numel())):
        assert bool((b[:o] == 7.0).all()) and bool((b[o + m:] == 7.0).all())


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f32", 64)])
@pytest.mark.parametrize("cut", [1, 127, 128, 200, 256, 300, 511])
@pytest.mark.parametrize("sink", [None, -3.0])
def test_first_keys_score_minus_infinity(cuda, dtype, d, cut, sink):
    """Keys that score -infinity weigh nothing: rows behind them are as if they were not there, and a row that sees no
    other key has 0 / 0, or, with a sink, all its weight there."""
    import torch

    n, h, hk = 600, 4, 2
    q, k, v, _ = _inputs([n], h, hk, d, d, dtype, seed=22)
    q[..., 0] = q[..., 0].abs() + 1
    k[:cut, :, 0] = -math.inf
    sinks = None if sink is None else torch.full((h,), sink, device="cuda")
    pool = G.PagedBlockPool(1, 1, hk, d, 16)
    out, lse = torch.empty_like(q), torch.empty(n, h, device="cuda")
    pool.prompt_attention(q, k, v, torch.tensor([0, n], dtype=torch.int32, device="cuda"), out, 1 / math.sqrt(d), sinks=sinks, lse=lse)
    pool.sync()
    pool.close()
    ref, rlse, size, most = prompt_reference(q[cut:], k[cut:], v[cut:], [0, n - cut], 1 / math.sqrt(d), sinks)
    tol, ltol = prompt_tolerance(ref, size, most, d, n, q.dtype)
    assert_within(out[cut:], ref, tol, "rows behind")
    assert_within(lse[cut:], rlse, ltol + 2.0 ** -23 * rlse.abs(), "lse behind")
    if sink is None:
        assert bool(out[:cut].isnan().all()) and bool((lse[:cut] == -math.inf).all())
    else:
        assert bool((out[:cut] == 0).all())
        assert_within(lse[:cut], torch.full((cut, h), sink, dtype=torch.float64, device="cuda"), torch.tensor(2.0 ** -21 * abs(sink), device="cuda"), "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cu,served", [([0, 40, 30, 100], [(0, 0, 30), (30, 40, 100)]), ([-5, 40, 100], [(40, 40, 100)]),
                                       ([0, 40, 101], [(0, 0, 40)]), ([0, 200, 60], [])])
def test_good_prompts_beside_bad_ranges(cuda, dtype, cu, served):
    """served: (first row of the prompt, first and last row that it alone holds); rows of bad ranges alone stay."""
    import torch

    q, k, v, _ = _inputs([100], 2, 1, 64, 64, dtype, seed=23)
    out = torch.full_like(q, 7.0)
    pool = G.PagedBlockPool(1, 1, 1, 64, 16)
    pool.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), out, 0.125)
    with pytest.raises(G.DeviceError):
        pool.sync()
    pool.sync()
    pool.close()
    free = torch.ones(100, dtype=torch.bool, device="cuda")
    for first, b, e in served:
        ref, _, size, most = prompt_reference(q, k, v, [first, e], 0.125)
        tol, _ = prompt_tolerance(ref, size, most, 64, 100, q.dtype)
        assert_within(out[b:e], ref[b:e], tol[b:e], str((first, b, e)))
        free[first:e] = False
    assert bool((out[free] == 7.0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch", [12, 64, 65, 512, 513, 1030, 3000])
@pytest.mark.parametrize("kind", ["past total", "negative", "first", "last", "several"])
def test_good_prompts_beside_bad_ranges_of_large_batches(cuda, dtype, batch, kind):
    """On both sides of what a block lists: the prompts whose ranges are good keep their results."""
    import numpy as np
    import torch

    rng = np.random.default_rng(batch)
    lens = rng.choice([1, 2, 7, 130, 257], batch).tolist()
    q, k, v, cu = _inputs(lens, 2, 1, 64, 64, dtype, seed=24)
    n = int(cu[-1])
    bad = np.array(cu, np.int64)
    at = {"first": [0], "last": [batch], "several": [batch // 5, batch // 2, batch // 2 + 1, 4 * batch // 5]}.get(kind, [batch // 2])
    bad[at] = -1 if kind in ("negative", "first") else n + 100000
    if kind == "several":
        bad[at[1]] = -5
    good = [b for b in range(batch) if 0 <= bad[b] <= bad[b + 1] <= n]
    assert len(good) == batch - len({x for i in at for x in (i - 1, i) if 0 <= x < batch})
    out = torch.full_like(q, 7.0)
    pool = G.PagedBlockPool(1, 1, 1, 64, 16)
    pool.prompt_attention(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"), out, 0.125)
    with pytest.raises(G.DeviceError):
        pool.sync()
    want = torch.empty_like(q)
    pool.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), want, 0.125)
    pool.sync()
    pool.close()
    rows = torch.zeros(n, dtype=torch.bool, device="cuda")
    for b in good:
        rows[cu[b]:cu[b + 1]] = True
    assert torch.equal(out[rows], want[rows])  # a tile's sums do not depend on where it runs
    assert bool((out[~rows] == 7.0).all())


@pytest.mark.parametrize("dtype,batch", [("bf16", 511), ("bf16", 512), ("bf16", 513), ("f16", 512), ("f32", 64), ("f32", 65)])
def test_batches_around_the_listing_limits(cuda, dtype, batch):
    """The most prompts that a block lists, and one more."""
    import numpy as np

    from test_gpu_prompt_attention import _check

    lens = np.random.default_rng(batch).choice([0, 1, 3, 128, 130, 300], batch).tolist()
    q, k, v, cu = _inputs(lens, 2, 1, 64, 64, dtype, seed=batch)
    _check(q, k, v, cu, 0.125)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_left_out_prompt_is_named(cuda, dtype):
    import torch

    q, k, v, _ = _inputs([100], 2, 1, 64, 64, dtype, seed=25)
    pool = G.PagedBlockPool(1, 1, 1, 64, 16)
    pool.prompt_attention(q, k, v, torch.tensor([0, 101], dtype=torch.int32, device="cuda"), torch.empty_like(q), 0.125)
    with pytest.raises(G.DeviceError, match="prompt"):
        pool.sync()
    pool.close()

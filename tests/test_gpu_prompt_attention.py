"""gkv_prompt_attention against softmax(scale q k^T [, sink]) v in 64 bits."""
import math

import numpy as np
import pytest

import glacier_kv as G
from operator_refs import assert_within, prompt_reference, prompt_tolerance

pytestmark = pytest.mark.gpu


def _kind(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _inputs(lens, heads, heads_kv, d, dv, dtype, seed=0, fused=False, spread=1.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    n = int(cu[-1])
    if fused:
        x = torch.randn(n, heads * d + heads_kv * (d + dv), device="cuda", generator=g).to(_kind(dtype))
        q = x[:, :heads * d].view(n, heads, d)
        k = x[:, heads * d:(heads + heads_kv) * d].view(n, heads_kv, d)
        v = x[:, (heads + heads_kv) * d:].view(n, heads_kv, dv)
    else:
        q, k, v = (torch.randn(n, h, m, device="cuda", generator=g).mul_(spread).to(_kind(dtype))
                   for h, m in ((heads, d), (heads_kv, d), (heads_kv, dv)))
    return q, k, v, cu


def _run(q, k, v, cu, scale, sinks=None, rows=None, mark=7.0):
    import torch

    pool = G.PagedBlockPool(1, 1, k.shape[1], q.shape[2], 16, v_head_dim=v.shape[2], dtype="f32")
    n = q.shape[0]
    out = torch.full((n, q.shape[1], v.shape[2]), mark, dtype=q.dtype, device="cuda")
    lse = torch.full((n, q.shape[1]), mark, device="cuda")
    pool.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), out, scale, sinks=sinks, lse=lse)
    pool.sync()
    pool.close()
    return out, lse


def _check(q, k, v, cu, scale, sinks=None):
    out, lse = _run(q, k, v, cu, scale, sinks)
    ref, rlse, size, most = prompt_reference(q, k, v, [int(c) for c in cu], scale, sinks)
    longest = max(int(b) - int(a) for a, b in zip(cu, cu[1:]))
    tol, ltol = prompt_tolerance(ref, size, most, q.shape[2], longest, q.dtype)
    n = int(cu[-1])
    assert_within(out[:n], ref[:n], tol[:n], "out")
    assert_within(lse[:n], rlse[:n], ltol + 2.0 ** -23 * rlse[:n].abs(), "lse")
    assert bool((out[n:] == 7.0).all()) and bool((lse[n:] == 7.0).all())


LENS = [[1], [2], [63], [64], [65], [127], [128], [129], [255, 1, 257], [1, 1, 1], [300, 17, 0, 64, 1, 513], [0, 0, 5], [1000, 2300]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("dtype,heads,heads_kv,d", [("bf16", 28, 4, 128), ("f16", 4, 1, 64), ("f32", 6, 2, 128), ("bf16", 3, 3, 64),
                                                    ("f16", 8, 1, 128)])
def test_lengths(cuda, lens, dtype, heads, heads_kv, d):
    q, k, v, cu = _inputs(lens, heads, heads_kv, d, d, dtype, seed=sum(lens))
    _check(q, k, v, cu, 1 / math.sqrt(d))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d,dv", [(8, 8), (32, 32), (96, 96), (128, 64), (64, 128), (192, 128), (256, 256), (200, 24)])
def test_head_dims(cuda, dtype, d, dv):
    q, k, v, cu = _inputs([70, 1, 190], 4, 2, d, dv, dtype, seed=d + dv)
    _check(q, k, v, cu, 1 / math.sqrt(d))


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f32", 64), ("f16", 96)])
def test_strides_and_sinks(cuda, dtype, d):
    import torch

    q, k, v, cu = _inputs([200, 3, 140], 8, 2, d, d, dtype, seed=3, fused=True)
    sinks = torch.linspace(-4, 6, 8, device="cuda")
    _check(q, k, v, cu, 1 / math.sqrt(d), sinks)
    # heads before tokens
    t = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    _check(t(q), t(k), t(v), cu, 1 / math.sqrt(d), sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-3, 0.7])
def test_scales(cuda, dtype, scale):
    q, k, v, cu = _inputs([150, 90], 4, 2, 128, 128, dtype, seed=4)
    _check(q, k, v, cu, scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_scores(cuda, dtype):
    """Scores of some hundreds: the running maximum moves by much, and most weights vanish."""
    q, k, v, cu = _inputs([700, 130], 4, 2, 128, 128, dtype, seed=5, spread=6.0)
    _check(q, k, v, cu, 1 / math.sqrt(128))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_growing_scores(cuda, dtype):
    """The maximum moves at every tile."""
    import torch

    q, k, v, cu = _inputs([900], 2, 1, 128, 128, dtype, seed=6)
    ramp = torch.linspace(0, 1, 900, device="cuda")[:, None, None]
    k = (q[:, :1] * 0 + 1.0) * ramp.to(q.dtype) * 4
    _check((q * 0 + 1.0), k.contiguous(), v, cu, 1 / math.sqrt(128))


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 128), ("bf16", 64), ("f16", 64), ("f32", 128), ("f16", 96)])
def test_masked_values_stay_out(cuda, dtype, d):
    """NaN and infinities in later keys and values, in other prompts and behind the last one reach no row that does not
    see them; a row that sees them gets what the formula gives."""
    import torch

    lens = [40, 300, 150]
    q, k, v, cu = _inputs(lens + [30], 4, 2, d, d, dtype, seed=7)
    cu = cu[:4]
    clean = [x.clone() for x in (q, k, v)]
    end = int(cu[3])
    for x in (q, k, v):
        x[end:] = math.nan                    # behind the last prompt
    k[39], v[39] = math.nan, math.inf          # the first prompt's last row
    v[40 + 200, 0, 5] = math.nan               # a value element in the middle of the second
    v[40 + 210, 1, 7] = math.inf
    v[40 + 220, 1, 7] = -math.inf
    v[40 + 290, 0, 3] = -math.inf
    out, lse = _run(q, k, v, cu, 1 / math.sqrt(d))
    ref, rlse, size, most = prompt_reference(*clean, [int(c) for c in cu], 1 / math.sqrt(d))
    tol, ltol = prompt_tolerance(ref, size, most, d, 300, q.dtype)
    seen = torch.zeros_like(ref, dtype=torch.bool)
    seen[39] = True
    seen[240:340, 0:2, 5] = True
    seen[250:340, 2:4, 7] = True
    seen[330:340, 0:2, 3] = True
    assert_within(torch.where(seen, ref, out.double())[:end], ref[:end], tol[:end], "rows that see none")
    rows = torch.ones(end, dtype=torch.bool, device="cuda")
    rows[39] = False
    assert_within(lse[:end][rows], rlse[:end][rows], ltol + 2.0 ** -23 * rlse[:end][rows].abs(), "lse")
    assert bool(out[39].isnan().all())
    assert bool(out[240:340, 0:2, 5].isnan().all())
    assert bool((out[250:260, 2:4, 7] == math.inf).all()) and bool(out[260:340, 2:4, 7].isnan().all())
    assert bool((out[330:340, 0:2, 3] == -math.inf).all())
    assert bool((out[end:] == 7.0).all()) and bool((lse[end:] == 7.0).all())


@pytest.mark.parametrize("cu,bad", [([0, 40, 30, 100], [1]), ([-5, 40, 100], [0]), ([0, 40, 101], [1]), ([0, 200, 60], [0, 1])])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bad_ranges_are_left_out(cuda, dtype, cu, bad):
    import torch

    q, k, v, _ = _inputs([100], 2, 1, 64, 64, dtype, seed=8)
    pool = G.PagedBlockPool(1, 1, 1, 64, 16, dtype="f32")
    out = torch.full_like(q, 7.0)
    pool.prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), out, 0.125)
    with pytest.raises(G.DeviceError):
        pool.sync()
    pool.sync()
    pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_same_result_every_time_and_on_another_stream(cuda, dtype):
    import torch

    q, k, v, cu = _inputs([513, 64, 1200], 8, 2, 128, 128, dtype, seed=9)
    first, lse = _run(q, k, v, cu, 0.09)
    pool = G.PagedBlockPool(1, 1, 2, 128, 16, dtype="bf16")
    c = torch.tensor(cu, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.empty_like(first) for _ in range(3)]
    with torch.cuda.stream(side):
        for o in outs:
            pool.prompt_attention(q, k, v, c, o, 0.09)
    pool.prompt_attention(q, k, v, c, torch.empty_like(first), 0.09)  # two streams at once
    side.synchronize()
    pool.sync()
    assert all(torch.equal(o, first) for o in outs)
    pool.close()


def test_refusals(cuda):
    import torch

    q, k, v, cu = _inputs([10], 4, 2, 64, 64, "bf16")
    c, out = torch.tensor(cu, device="cuda"), torch.empty(10, 4, 64, dtype=torch.bfloat16, device="cuda")
    pool = G.PagedBlockPool(1, 1, 2, 64, 16, dtype="f32")
    bad = G.ArgumentOutOfRangeError
    with pytest.raises(bad):
        pool.prompt_attention(q[:, :3], k, v, c, out[:, :3].contiguous(), 0.1)
    with pytest.raises(bad):
        pool.prompt_attention(q, k, v, c, q, 0.1)
    for scale in (math.nan, math.inf):
        with pytest.raises(bad):
            pool.prompt_attention(q, k, v, c, out, scale)
    wide = torch.zeros(10, 4 * 64 + 4, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(bad):
        pool.prompt_attention(wide[:, :256].view(10, 4, 64), k, v, c, out, 0.1)
    with pytest.raises(bad):
        pool.prompt_attention(wide[:, 4:].view(10, 4, 64), k, v, c, out, 0.1)
    with pytest.raises(ValueError):
        pool.prompt_attention(q, k.float(), v, c, out, 0.1)
    with pytest.raises(ValueError):
        pool.prompt_attention(q, k, v, c.long(), out, 0.1)
    with pytest.raises(ValueError):
        pool.prompt_attention(q, k, v, c, out.float(), 0.1)
    with pytest.raises(ValueError):
        pool.prompt_attention(q, k[:9], v, c, out, 0.1)
    with pytest.raises(ValueError):
        pool.prompt_attention(q, k, v, c, out, 0.1, lse=torch.empty(10, 3, device="cuda"))
    other = G.PagedBlockPool(1, 1, 2, 36, 16, dtype="f32")
    x = [torch.zeros(10, h, 36, device="cuda") for h in (4, 2, 2)]
    with pytest.raises(G.UnsupportedError):
        other.prompt_attention(*x, c, torch.empty_like(x[0]), 0.1)
    # nothing to do
    pool.prompt_attention(q[:0], k[:0], v[:0], c, out[:0], 0.1)
    pool.prompt_attention(q, k, v, c[:1], out, 0.1)
    assert pool.last_launch_count == 0
    pool.close()
    other.close()


@pytest.mark.parametrize("batch", [33, 1024, 1025, 3000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_prompts(cuda, dtype, batch):
    """Batches on both sides of what a block lists, empty prompts and one-token ones among them."""
    rng = np.random.default_rng(batch)
    lens = rng.choice([0, 0, 1, 2, 7, 130, 257], batch).tolist()
    q, k, v, cu = _inputs(lens, 2, 1, 64, 64, dtype, seed=batch)
    _check(q, k, v, cu, 0.125)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f32", 64)])
def test_broadcast_keys_and_values(cuda, dtype, d):
    """One key and value head given as several (a stride of 0), and one row of queries as all."""
    q, k, v, cu = _inputs([150, 40], 4, 1, d, d, dtype, seed=12)
    _check(q, k.expand(-1, 2, -1), v.expand(-1, 2, -1), cu, 0.1)
    _check(q[:1].expand(q.shape[0], -1, -1), k, v, cu, 0.1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_infinite_sinks(cuda, dtype):
    """A sink of minus infinity is none; one of plus infinity takes all the weight."""
    import torch

    q, k, v, cu = _inputs([150, 1], 2, 1, 64, 64, dtype, seed=13)
    out, lse = _run(q, k, v, cu, 0.125, sinks=torch.tensor([-math.inf, math.inf], device="cuda"))
    plain, plain_lse = _run(q, k, v, cu, 0.125)
    assert torch.equal(out[:, 0], plain[:, 0]) and torch.equal(lse[:, 0], plain_lse[:, 0])
    assert bool((out[:, 1] == 0).all()) and bool((lse[:, 1] == math.inf).all())


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f16", 64), ("f32", 128)])
def test_replayed_with_other_lengths(cuda, dtype, d):
    """Captured once, replayed with other prompts in the same buffers; rows behind the last one stay."""
    import torch

    pool = G.PagedBlockPool(1, 1, 2, d, 16, dtype="bf16")
    n, batch = 900, 5
    q, k, v, _ = _inputs([n], 4, 2, d, d, dtype, seed=14)
    cu = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    out, lse = torch.empty(n, 4, d, dtype=q.dtype, device="cuda"), torch.empty(n, 4, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    pool.prompt_attention(q, k, v, cu, out, 0.1, lse=lse, stream=s)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        pool.prompt_attention(q, k, v, cu, out, 0.1, lse=lse, stream=s)
    for lens in ([900, 0, 0, 0, 0], [1, 300, 2, 257, 5], [0, 0, 0, 0, 0], [128, 128, 129, 64, 400]):
        c = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        with torch.cuda.stream(s):
            cu.copy_(torch.from_numpy(c))
            out.fill_(7.0)
            lse.fill_(7.0)
            graph.replay()
        s.synchronize()
        pool.sync(s)
        ref, rlse, size, most = prompt_reference(q, k, v, c.tolist(), 0.1)
        tol, ltol = prompt_tolerance(ref, size, most, d, 900, q.dtype)
        m = int(c[-1])
        assert_within(out[:m], ref[:m], tol[:m], str(lens))
        assert_within(lse[:m], rlse[:m], ltol + 2.0 ** -23 * rlse[:m].abs(), str(lens))
        assert bool((out[m:] == 7.0).all()) and bool((lse[m:] == 7.0).all())
    graph.reset()
    pool.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_overlapping_ranges_are_reported(cuda, dtype):
    """More tiles than the rows of the call have: an error, and the next call is as any other."""
    import torch

    q, k, v, _ = _inputs([2000], 2, 1, 64, 64, dtype, seed=14)
    pool = G.PagedBlockPool(1, 1, 1, 64, 16, dtype="f32")
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    first, then = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    pool.prompt_attention(q, k, v, t([0, 2000] * 40), first, 0.125)
    with pytest.raises(G.DeviceError):
        pool.sync()
    pool.prompt_attention(q, k, v, t([0, 2000]), then, 0.125)
    pool.sync()
    assert bool(((first == 7.0) | (first == then)).all())
    pool.close()

"""gkv_step_build next to the calls that share its step or its tables: the split-KV decode and copy-on-write forks."""
import math

import pytest

import glacier_kv as G

pytestmark = pytest.mark.gpu


def _i32(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _random_arena(pool, g):
    import torch

    for view in (pool.key_view(), pool.value_view()):
        view.copy_(torch.randn(view.shape, device="cuda", generator=g))


def test_split_kv_decode_of_requests_without_tokens(cuda):
    """A rank holds no tokens of a request (its context is 0) or the build left it out: it has no weight in the merge,
    whatever an earlier decode left in the exchange buffers."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(31)
    B, H, HK, D = 4, 8, 2, 128
    pool = G.PagedBlockPool(40, 1, HK, D, 16, dtype="bf16")
    _random_arena(pool, g)
    pool.reserve_step(B, 8, B, H)
    pool.set_static_step()
    comm = G.Comm(G.Comm.unique_id(), 1, 0, cuda.index or 0, timeout_ms=60_000)
    tables = torch.arange(32, dtype=torch.int32, device="cuda").view(B, 8)
    q = torch.randn(B, H, D, device="cuda", generator=g)
    # every parity of the exchange holds rows of all requests before one of them has none
    for ctx, left in (([100, 7, 33, 64], []), ([50, 120, 1, 16], []), ([100, 0, 33, 64], []), ([0, 0, 5, 0], []), ([9, -1, 33, 64], [1]),
                      ([0, 0, 0, 0], [])):
        pool.build_step(G.StepBuffers(tables, _i32(ctx), _i32([0] * B), _i32([]), max_tokens=B))
        merged, plain = torch.full((B, H, D), 7.0, device="cuda"), torch.zeros(B, H, D, device="cuda")
        pool.paged_decode_splitkv_dist(comm, 0, q, merged, H, 1 / math.sqrt(D))
        pool.paged_decode(0, q, plain, H, 1 / math.sqrt(D))
        if left:
            with pytest.raises(G.DeviceError):
                pool.sync()
        pool.sync()
        idle = torch.tensor([c <= 0 for c in ctx], device="cuda")
        assert bool((merged[idle] == 0.0).all()), ctx
        # one rank's block with weight 1, through its lse and back: 3 roundings
        assert bool(((merged - plain).abs() <= 2.0 ** -22 * plain.abs()).all()), ctx
    comm.close()
    pool.close()

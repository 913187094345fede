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


@pytest.mark.parametrize("replayed", [False, True])
def test_a_forked_block_is_rewritten_on_the_device(cuda, replayed):
    """Two requests share a partial block. The one that adds a token first gets a copy of it from append_token; with the
    copy flushed and the new id in its device table, its token lands in the copy and the sibling's block stays."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(32)
    H, HK, D, BS, CTX = 4, 2, 128, 16, 26
    pool = G.PagedBlockPool(12, 1, HK, D, BS)
    _random_arena(pool, g)
    pool.reserve_step(2, 4, 2, H)
    pool.set_static_step()
    a, b = G.BlockTable(pool), G.BlockTable(pool)
    for _ in range(CTX):
        assert a.append_token()[0]
    for block in a.physical_block_ids:
        pool.retain_block(block)
    b.attach_prefix_blocks(a.physical_block_ids, CTX)
    shared = a.get_block_id(1)
    rows = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    for i, t in enumerate((a, b)):
        rows[i, :2] = torch.from_numpy(t.as_span()).cuda()
    io = G.StepBuffers(rows, _i32([CTX, CTX]), _i32([0, 0]), _i32([-1, -1]), max_tokens=2)
    rope = G.MultiAxisRope([D // 2], D)
    q, k, v = (torch.randn(2, n, D, device="cuda", generator=g) for n in (H, HK, HK))
    positions, q_out, out = _i32([[CTX, CTX]]), torch.empty(2, H, D, device="cuda"), torch.zeros(2, H, D, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())

    def step():
        pool.build_step(io, n_new_blocks=0, stream=s)
        pool.mrope_append(0, q, k, v, positions, rope, q_out, stream=s)
        pool.paged_decode(0, q_out, out, H, 1 / math.sqrt(D), stream=s)

    step()  # nothing to add
    s.synchronize()
    if replayed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step()
    keys, values = pool.key_view(), pool.value_view()
    before = [x[shared].clone() for x in (keys, values)]
    torch.cuda.synchronize()
    ok, block, offset = b.append_token()
    assert ok and block != shared and offset == CTX % BS and pool.get_ref_count(shared) == 1
    with pytest.raises(G.InvalidOperationError):  # the copy is still queued: no launch of the step takes it along
        pool.paged_decode(0, q_out, out, H, 1 / math.sqrt(D), stream=s)
    pool.flush_copies(s)
    with torch.cuda.stream(s):
        io.block_tables[1, CTX // BS] = block
        io.new_lens.copy_(_i32([0, 1]))
        q[0].copy_(q[1]), k[0].copy_(k[1]), v[0].copy_(v[1])  # row 0 of the step is request 1's token
        if replayed:
            graph.replay()
        else:
            step()
    s.synchronize()
    pool.sync(s)
    assert io.slots[0].item() == block * BS + CTX % BS and io.ctx_out.tolist() == [CTX, CTX + 1]
    assert all(torch.equal(x[shared], y) for x, y in zip((keys, values), before))
    for x, y in zip((keys, values), before):
        assert torch.equal(x[block][:, :, :CTX % BS], y[:, :, :CTX % BS])
    assert torch.equal(values[block, 0, :, CTX % BS], v[0])
    if replayed:
        graph.reset()
    pool.close()

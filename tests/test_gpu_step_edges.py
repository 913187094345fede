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


def _attended(pool, table, q, position, scale):
    """(out, weighted |v|, largest sum of |q k|) in 64 bits of one query row [heads, dim] over the arena's positions 0 .. position."""
    import torch

    bs, at = pool.block_size, torch.arange(position + 1, device="cuda")
    blocks = torch.tensor(table, device="cuda")[at // bs]
    kk, vv = (x[blocks, 0, :, at % bs].double().repeat_interleave(q.shape[0] // x.shape[2], 1) for x in (pool.key_view(), pool.value_view()))
    s = scale * torch.einsum("hd,thd->ht", q.double(), kk)
    w = torch.softmax(s, 1)
    most = float((abs(scale) * torch.einsum("hd,thd->ht", q.double().abs(), kk.abs())).max())
    return torch.einsum("ht,thd->hd", w, vv), torch.einsum("ht,thd->hd", w, vv.abs()), most


def test_prompts_and_tokens_in_one_step_then_a_further_chunk(cuda):
    """The step's rows go to prompt attention as packed, to the decode gathered by request; a chunk behind stored tokens
    goes through the ordinary layout."""
    import numpy as np
    import torch

    from operator_refs import assert_within, prompt_reference, prompt_tolerance

    g = torch.Generator(device="cuda").manual_seed(33)
    H, HK, D, BS = 4, 2, 64, 16
    scale = 1 / math.sqrt(D)
    ctx, new = [40, 0, 15, 0, 16], [1, 37, 1, 1, 1]  # two prompts, one of them of a single token, and three tokens
    B, cap, width = len(ctx), 48, 6
    pool = G.PagedBlockPool(30, 1, HK, D, BS)
    _random_arena(pool, g)
    pool.reserve_step(B, width, cap, H)
    pool.set_static_step()
    tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    ids = iter(torch.randperm(30, generator=torch.Generator().manual_seed(1)).tolist())
    for b, c in enumerate(ctx):
        for j in range(-(-c // BS)):
            tables[b, j] = next(ids)
    fresh = [next(ids) for c, n in zip(ctx, new) for _ in range(-(-(c + n) // BS) - -(-c // BS))]
    io = G.StepBuffers(tables, _i32(ctx), _i32(new), _i32(fresh), max_tokens=cap)
    rope = G.MultiAxisRope([D // 2], D)
    q, k, v = (torch.randn(cap, n, D, device="cuda", generator=g) for n in (H, HK, HK))
    q_out, k_out, out = torch.empty_like(q), torch.empty_like(k), torch.full_like(q, 7.0)
    pool.build_step(io)
    pool.mrope_append(0, q, k, v, io.positions[None], rope, q_out, k_out)
    pool.prompt_attention(q_out, k_out, v, io.cu_new, out, scale)
    tokens = torch.tensor([b for b, c in enumerate(ctx) if c > 0], device="cuda")
    last = io.cu_new[1:].long() - 1
    decoded = torch.empty(B, H, D, device="cuda")
    pool.paged_decode(0, q_out[last].contiguous(), decoded, H, scale)
    out[last[tokens]] = decoded[tokens]
    pool.sync()
    rows = io.block_tables.tolist()
    cu = io.cu_new.tolist()
    for b, (c, n) in enumerate(zip(ctx, new)):
        if c == 0:
            at = slice(cu[b], cu[b + 1])
            ref, _, size, most = prompt_reference(q_out[at], k_out[at], v[at], [0, n], scale)
            assert_within(out[at], ref, prompt_tolerance(ref, size, most, D, n, torch.float32)[0], f"prompt {b}")
        else:
            ref, size, most = _attended(pool, rows[b], q_out[cu[b]], c, scale)
            assert_within(out[cu[b]], ref, prompt_tolerance(ref, size, most, D, c + 1, torch.float32)[0], f"token {b}")
    assert bool((out[cu[-1]:] == 7.0).all())

    # nine more tokens of request 1 (37 stored)
    pool.set_static_step(False)
    have, more = 37, 9
    table = np.array([rows[1]], np.int32)
    slots = np.array([rows[1][p // BS] * BS + p % BS for p in range(have, have + more)], np.int64)
    pool.upload_step(table, np.array([have + more], np.int32), slots)
    kn, vn, qn = (torch.randn(more, n, D, device="cuda", generator=g) for n in (HK, HK, H))
    pool.kv_append(0, kn, vn)
    chunk = torch.empty(more, H, D, device="cuda")
    pool.paged_prefill(0, qn, chunk, [have], [more], H, scale)
    pool.sync()
    for i in range(more):
        ref, size, most = _attended(pool, rows[1], qn[i], have + i, scale)
        assert_within(chunk[i], ref, prompt_tolerance(ref, size, most, D, have + more, torch.float32)[0], f"chunk {i}")
    pool.close()


def test_arrays_that_overlap_are_refused(cuda):
    """A written array over any other, whole or by one element; arrays that only touch, and empty ones, are not over each other."""
    import torch

    pool = G.PagedBlockPool(8, 1, 2, 64, 16)
    pool.reserve_step(4, 3, 6, 4)
    pool.set_static_step()
    # one buffer of int32 for all: place(name) gives each array's first element in it
    sizes = {"d_ctx_lens": 4, "d_new_lens": 4, "d_new_blocks": 4, "d_block_tables": 12, "d_ctx_out": 4, "d_cu_new": 5, "d_slots": 12,
             "d_positions": 6, "d_counts": 2}
    buf = torch.zeros(64, dtype=torch.int32, device="cuda")
    place, at = {}, 0
    for name in ["d_slots"] + [n for n in sizes if n != "d_slots"]:  # 64-bit slots first: everything touches, nothing overlaps
        place[name] = at
        at += sizes[name]
    io = G.StepBuffers(torch.zeros(4, 3, dtype=torch.int32, device="cuda"), _i32([0] * 4), _i32([0] * 4), _i32([0] * 4), max_tokens=6)

    def build(**moved):
        for name in sizes:
            setattr(io._desc, name, buf.data_ptr() + 4 * {**place, **moved}[name])
        pool.build_step(io)

    build()
    pool.sync()
    order = sorted(place, key=place.get)
    for before, name in zip(order, order[1:]):
        if name in ("d_new_lens", "d_new_blocks") and before in ("d_ctx_lens", "d_new_lens"):
            continue  # inputs may share memory
        with pytest.raises(G.ArgumentOutOfRangeError, match="overlaps"):
            build(**{name: place[name] - 1})
    with pytest.raises(G.ArgumentOutOfRangeError, match="overlaps"):
        build(d_cu_new=place["d_new_lens"])
    build(d_new_lens=place["d_ctx_lens"])
    pool.sync()
    pool.close()


@pytest.mark.parametrize("dtype,heads,heads_kv,dim", [("f32", 4, 2, 64), ("bf16", 28, 4, 128), ("fp8", 28, 4, 128)])
def test_decode_over_a_table_with_a_bad_id(cuda, dtype, heads, heads_kv, dim):
    """The build takes earlier table entries as they are: an id outside the pool is reported, and the other requests are served."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(34)
    B, width = 3, 8
    pool = G.PagedBlockPool(B * width, 1, heads_kv, dim, 16, dtype=dtype)
    for view in (pool.key_view(), pool.value_view()):
        x = torch.randn(view.shape, device="cuda", generator=g)
        view.copy_(x.to(torch.float8_e4m3fn).view(torch.uint8) if dtype == "fp8" else x)
    pool.reserve_step(B, width, B, heads)
    pool.set_static_step()
    tables = torch.arange(B * width, dtype=torch.int32, device="cuda").view(B, width)
    q = torch.randn(B, heads, dim, device="cuda", generator=g)
    outs = []
    for bad in (None, B * width, -1, 2 ** 31 - 1, None):
        t = tables.clone()
        if bad is not None:
            t[1, 3] = bad
        out = torch.full((B, heads, dim), 7.0, device="cuda")
        pool.build_step(G.StepBuffers(t, _i32([100, 128, 17]), _i32([0] * B), _i32([]), max_tokens=B))
        pool.paged_decode(0, q, out, heads, 1 / math.sqrt(dim))
        if bad is not None:
            with pytest.raises(G.DeviceError):
                pool.sync()
        pool.sync()
        outs.append(out)
    assert torch.equal(outs[0], outs[-1]) and bool(outs[0].isfinite().all())
    for out in outs[1:-1]:
        assert torch.equal(out[[0, 2]], outs[0][[0, 2]])
    pool.close()

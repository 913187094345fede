"""gkv_step_build: every output against a request-by-request restatement, and the decode that runs on
the built step bit for bit against the one on the host-uploaded step (the same work list)."""
import math

import numpy as np
import pytest

import glacier_kv as G
from operator_refs import step_reference

pytestmark = pytest.mark.gpu


def _case(rng, ctx, new, bs, spare_width=1, spare_ids=3, short=0):
    """Tables with distinct random ids for ctx, and ids for what new opens (`short` fewer)."""
    old = [-(-max(c, 0) // bs) for c in ctx]
    opened = [max(0, -(-(max(c, 0) + max(n, 0)) // bs) - o) for c, n, o in zip(ctx, new, old)]
    width = max([o + p for o, p in zip(old, opened)] + [1]) + spare_width
    total = sum(old) + sum(opened) + spare_ids
    ids = rng.permutation(total).astype(np.int32)
    tables = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for b, o in enumerate(old):
        tables[b, :o] = ids[at:at + o]
        at += o
    return tables, ids[at:at + sum(opened) - short], total


def _build(pool, ctx, new, tables, ids, max_tokens, batch=None, mark=-7):
    import torch

    t = lambda x: torch.tensor(np.asarray(x, np.int32), device="cuda")  # noqa: E731
    io = G.StepBuffers(t(tables).reshape(len(ctx), -1), t(ctx), t(new), t(ids), max_tokens)
    for x in (io.slots, io.positions, io.cu_new, io.ctx_out):
        x.fill_(mark)
    pool.build_step(io, batch=batch)
    return io


def _check(io, want, mark=-7):
    tables, ctx_out, cu, slots, positions, counts = want[:6]
    assert io.counts.tolist() == counts
    assert io.cu_new.tolist() == cu
    assert io.ctx_out.tolist() == ctx_out
    n = len(slots)
    assert io.slots[:n].tolist() == slots
    assert io.positions[:n].tolist() == positions
    assert bool((io.slots[n:] == mark).all()) and bool((io.positions[n:] == mark).all())
    assert io.block_tables.tolist() == tables


@pytest.mark.parametrize("ctx,new,bs", [
    ([0], [1], 16),                                    # a first token
    ([0], [0], 16),                                    # nothing at all
    ([15, 16, 17], [1, 1, 1], 16),                     # the last slot, a new page, inside a page
    ([0, 5, 16, 31, 0], [33, 11, 0, 1, 16], 16),       # prompts, an idle request, exact pages
    ([3, 0, 100], [1, 40, 7], 1),                      # one-token pages
    ([70, 0, 7], [9, 1, 8], 8),
    ([1000, 1, 0, 4096], [1, 3000, 17, 1], 32),
])
def test_outputs(cuda, ctx, new, bs):
    rng = np.random.default_rng(len(ctx) * 100 + bs)
    tables, ids, total = _case(rng, ctx, new, bs)
    pool = G.PagedBlockPool(total, 1, 2, 64, bs, dtype="bf16")
    cap = sum(new) + 5
    pool.reserve_step(len(ctx) + 1, tables.shape[1], cap, 4)
    pool.set_static_step()
    io = _build(pool, ctx, new, tables, ids, cap)
    pool.sync()
    _check(io, step_reference(ctx, new, tables.tolist(), ids.tolist(), bs, cap))
    pool.close()


@pytest.mark.parametrize("batch", [1, 31, 1023, 1025, 4096])
def test_many_requests(cuda, batch):
    rng = np.random.default_rng(batch)
    ctx = np.minimum(rng.lognormal(3.5, 1.2, batch).astype(int), 900).tolist()
    new = rng.choice([0, 1, 1, 1, 5, 60], batch).tolist()
    tables, ids, total = _case(rng, ctx, new, 16)
    pool = G.PagedBlockPool(total, 1, 1, 32, 16, dtype="bf16")
    pool.reserve_step(batch, tables.shape[1], sum(new) + 2, 1)
    pool.set_static_step()
    io = _build(pool, ctx, new, tables, ids, sum(new) + 2)
    pool.sync()
    _check(io, step_reference(ctx, new, tables.tolist(), ids.tolist(), 16, sum(new) + 2))
    pool.close()


def test_part_of_the_batch(cuda):
    rng = np.random.default_rng(2)
    ctx, new = [20, 16, 40], [1, 1, 3]
    tables, ids, total = _case(rng, ctx, new, 16)
    pool = G.PagedBlockPool(total, 1, 2, 64, 16, dtype="bf16")
    pool.reserve_step(3, tables.shape[1], 8, 4)
    pool.set_static_step()
    io = _build(pool, ctx, new, tables, ids, 8, batch=2)
    pool.sync()
    want = step_reference(ctx[:2], new[:2], tables[:2].tolist(), ids.tolist(), 16, 8)
    assert io.counts.tolist() == want[5] and io.cu_new.tolist() == want[2] + [-7] and io.ctx_out.tolist() == want[1] + [-7]
    assert io.block_tables.tolist() == want[0] + tables[2:].tolist()
    pool.build_step(io, batch=0)
    pool.sync()
    assert io.counts.tolist() == [0, 0] and int(io.cu_new[0]) == 0
    pool.close()


@pytest.mark.parametrize("ctx,new,cap,short", [
    ([20, 16, 16, 5], [1, 1, 1, 1], 8, 1),       # one id too few: the last that opens a page is left out
    ([20, -1, 16], [1, 1, 1], 8, 0),             # a negative length
    ([20, 3, 16], [1, -4, 1], 8, 0),
    ([20, 10, 16], [1, 10, 1], 6, 0),            # rows past max_tokens
    ([20, 3], [1, 2147483647], 6, 0),            # lengths whose sum passes 31 bits
])
def test_requests_left_out(cuda, ctx, new, cap, short):
    rng = np.random.default_rng(cap + short)
    sane = [n if n < 1000 else 0 for n in new]
    tables, ids, total = _case(rng, ctx, sane, 16, short=short)
    pool = G.PagedBlockPool(total, 1, 2, 64, 16, dtype="bf16")
    pool.reserve_step(len(ctx), tables.shape[1], cap, 4)
    pool.set_static_step()
    io = _build(pool, ctx, new, tables, ids, cap)
    with pytest.raises(G.DeviceError):
        pool.sync()
    pool.sync()  # reported once
    if max(new) > 1000:  # too many rows to list: the served request and the tables
        assert io.slots[0].item() == tables[0, 20 // 16] * 16 + 20 % 16 and bool((io.slots[1:] == -1).all())
        assert io.ctx_out.tolist() == [21, 3] and np.array_equal(io.block_tables.cpu().numpy(), tables)
    else:
        want = step_reference(ctx, new, tables.tolist(), ids.tolist(), 16, cap)
        assert want[7]
        _check(io, want)
    pool.close()


def test_a_table_row_that_is_too_short(cuda):
    pool = G.PagedBlockPool(8, 1, 2, 64, 16, dtype="bf16")
    pool.reserve_step(2, 4, 40, 4)
    pool.set_static_step()
    io = _build(pool, [16, 4], [17, 2], [[3, -1], [5, -1]], [1, 2, 4], 40)
    with pytest.raises(G.DeviceError):
        pool.sync()
    _check(io, step_reference([16, 4], [17, 2], [[3, -1], [5, -1]], [1, 2, 4], 16, 40))
    pool.close()


@pytest.mark.parametrize("tables,ids", [([[99, -1]], [2]), ([[1, -1]], [99]), ([[1, -1]], [-1])])
def test_block_ids_outside_the_pool(cuda, tables, ids):
    pool = G.PagedBlockPool(8, 1, 2, 64, 16, dtype="bf16")
    pool.reserve_step(1, 2, 8, 4)
    pool.set_static_step()
    io = _build(pool, [14], [4], tables, ids, 8)
    with pytest.raises(G.DeviceError):
        pool.sync()
    good = lambda i: 0 <= i < 8  # noqa: E731
    want = [tables[0][0] * 16 + 14 if good(tables[0][0]) else -1] * 1
    assert io.slots[0].item() == want[0]
    assert io.slots[2].item() == (ids[0] * 16 if good(ids[0]) else -1)
    pool.close()


def test_refusals(cuda):
    import torch

    z = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    pool = G.PagedBlockPool(8, 1, 2, 64, 16, dtype="bf16")
    io = G.StepBuffers(z(2, 3), z(2), z(2), z(4), max_tokens=6)
    pool.reserve_step(2, 3, 6, 4)
    with pytest.raises(G.InvalidOperationError):
        pool.build_step(io)  # not the static layout
    pool.set_static_step()
    with pytest.raises(G.ArgumentOutOfRangeError):
        pool.build_step(io, batch=3)
    with pytest.raises(G.ArgumentOutOfRangeError):
        pool.build_step(io, n_new_blocks=5)
    with pytest.raises(G.ArgumentOutOfRangeError):
        pool.build_step(G.StepBuffers(z(3, 3), z(3), z(3), z(1), max_tokens=6))  # batch past the reservation
    with pytest.raises(G.ArgumentOutOfRangeError):
        pool.build_step(G.StepBuffers(z(2, 3), z(2), z(2), z(1), max_tokens=7))
    with pytest.raises(ValueError):
        G.StepBuffers(z(2, 3), z(2), z(3), z(1), max_tokens=6)
    with pytest.raises(ValueError):
        G.StepBuffers(z(2, 3).long(), z(2), z(2), z(1), max_tokens=6)
    io._desc.d_ctx_out = io._desc.d_ctx_lens
    with pytest.raises(G.ArgumentOutOfRangeError):
        pool.build_step(io)
    io._desc.d_ctx_out = None
    io._desc.table_stride = 0
    with pytest.raises(G.ArgumentOutOfRangeError):
        pool.build_step(io)
    pool.close()


@pytest.mark.parametrize("dtype,heads,heads_kv,dim", [("f32", 28, 4, 128), ("bf16", 28, 4, 128), ("fp8", 28, 4, 128), ("bf16", 8, 8, 64)])
@pytest.mark.parametrize("kind", ["one long", "mixed", "many short", "few units", "fewer units than workers"])
def test_decode_on_the_built_step(cuda, dtype, heads, heads_kv, dim, kind):
    """The decode right behind the build, and behind an append, equals the uploaded step's bit for bit."""
    import torch

    rng = np.random.default_rng(heads + len(kind))
    ctx = {"one long": [20000], "mixed": [3, 0, 777, 4000, 16, 1, 0, 12000], "many short": rng.integers(0, 40, 300).tolist(),
           "few units": [1, 0, 2, 1], "fewer units than workers": [71, 1, 0, 301, 17, 0, 0, 40]}[kind]
    new = [1 if i % 3 != 1 else 0 for i in range(len(ctx))]
    tables, ids, total = _case(rng, ctx, new, 16)
    pool = G.PagedBlockPool(total, 1, heads_kv, dim, 16, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    for view in (pool.key_view(), pool.value_view()):
        x = torch.randn(view.shape, device="cuda", generator=g)
        view.copy_(x.to(torch.float8_e4m3fn).view(torch.uint8) if dtype == "fp8" else x)
    B, cap = len(ctx), max(1, sum(new))
    pool.reserve_step(B, tables.shape[1], cap, heads)
    pool.set_static_step()
    q = torch.randn(B, heads, dim, device="cuda", generator=g)
    kn, vn = (torch.randn(cap, heads_kv, dim, device="cuda", generator=g) for _ in range(2))
    outs = []
    want = step_reference(ctx, new, tables.tolist(), ids.tolist(), 16, cap)
    for built in (True, False):
        for append in (False, True):
            out = torch.full((B, heads, dim), 3.0, device="cuda")
            if built:
                io = _build(pool, ctx, new, tables, ids, cap)
            else:
                pool.upload_step(np.asarray(want[0], np.int32), np.asarray(want[6], np.int32), np.asarray(want[3], np.int64))
            if append:
                pool.kv_append(0, kn, vn)
            pool.paged_decode(0, q, out, heads, 1 / math.sqrt(dim))
            pool.sync()
            outs.append((out, pool.key_view().clone() if append else None))
    # the first decode ran before any append of the new rows; the third saw them: compare like with like
    assert torch.equal(outs[1][0], outs[3][0]) and torch.equal(outs[1][1], outs[3][1])
    assert torch.equal(outs[2][0], outs[3][0])
    idle = torch.tensor([c == 0 for c in want[6]], device="cuda")
    assert bool((outs[1][0][idle] == 3.0).all())
    pool.close()


def test_more_context_than_the_work_list_counts(cuda):
    """2^31 units and more: slots are built, nothing is decoded, and it is reported."""
    import torch

    pool = G.PagedBlockPool(1, 1, 32, 32, 1024, dtype="bf16")
    B, ctx, width = 40, 16_000_000, 15626
    pool.reserve_step(B, 1, B, 32)
    pool.set_static_step()
    t = lambda n: torch.full((B,), n, dtype=torch.int32, device="cuda")  # noqa: E731
    io = G.StepBuffers(torch.zeros(B, width, dtype=torch.int32, device="cuda"), t(ctx), t(1), t(0), max_tokens=B)  # every request opens a page
    pool.build_step(io)
    with pytest.raises(G.DeviceError):
        pool.sync()
    assert io.positions.tolist() == [ctx] * B and io.slots.tolist() == [ctx % 1024] * B and io.ctx_out.tolist() == [ctx + 1] * B
    out = torch.full((B, 32, 32), 3.0, device="cuda")
    pool.paged_decode(0, torch.zeros_like(out), out, 32, 1.0)
    pool.sync()
    assert bool((out == 3.0).all())
    io.ctx_lens.fill_(5)  # the next step is as any other
    pool.build_step(io)
    pool.paged_decode(0, torch.zeros_like(out), out, 32, 1.0)
    pool.sync()
    assert bool((out == 0.0).all())
    pool.close()


def test_rows_known_on_the_device_alone(cuda):
    """gkv_rope_append takes its rows from the host: refused on a built step, and not behind the next upload."""
    import torch

    pool = G.PagedBlockPool(4, 1, 1, 64, 16)
    pool.reserve_step(1, 2, 4, 1)
    pool.set_static_step()
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pool.build_step(G.StepBuffers(t([[0, -1]]), t([3]), t([1]), t([]), max_tokens=4))
    q, k, v = (torch.zeros(2, 1, 64, device="cuda") for _ in range(3))
    with pytest.raises(G.InvalidOperationError):
        pool.rope_append(0, q, k, v, [3, 4], 1)
    pool.upload_step(np.zeros((1, 1), np.int32), np.array([5], np.int32), np.array([3, 4], np.int64))
    pool.rope_append(0, q, k, v, [3, 4], 1)
    pool.sync()
    pool.close()


def test_a_launch_on_another_stream_orders_nothing(cuda):
    """Behind a build the decode waits for all of it, unless a launch on the build's own stream stands between."""
    import torch

    pool = G.PagedBlockPool(4, 1, 1, 64, 16)
    pool.reserve_step(1, 2, 4, 1)
    pool.set_static_step()
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    io = G.StepBuffers(t([[0, -1]]), t([3]), t([1]), t([]), max_tokens=4)
    x = torch.zeros(4, 1, 64, device="cuda")
    q, out = torch.zeros(1, 1, 64, device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    cu, one, two = t([0, 4]), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    counts = []
    for between in (None, two, one):
        pool.build_step(io, stream=one.cuda_stream)
        if between is not None:
            pool.prompt_attention(x, x, x, cu, torch.empty_like(x), 1.0, stream=between.cuda_stream)
        pool.paged_decode(0, q, out, 1, 1.0, stream=one.cuda_stream)
        counts.append(pool.last_launch_count)
        torch.cuda.synchronize()
    pool.sync()
    assert counts[0] == counts[1] == counts[2] + 1
    pool.close()

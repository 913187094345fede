"""The step operators together: lengths -> tables, slots, positions (build_step) -> rotation and append (mrope_append)
-> prompt attention of the new prompts -> paged decode of the next tokens, eager and replayed from one captured graph."""
import math

import numpy as np
import pytest

import glacier_kv as G
from operator_refs import assert_within, prompt_reference, rope_reference, unit

pytestmark = pytest.mark.gpu

H, HK, D, BS = 8, 2, 128, 16


class Host:
    """Allocation and the 64-bit model of the cache: every request's rotated k and its v, as the arena's type holds them."""

    def __init__(self, pool, rope, n, kind):
        self.pool, self.rope, self.kind = pool, rope, kind
        self.keys, self.values = [[] for _ in range(n)], [[] for _ in range(n)]

    def blocks(self, ctx, new):
        ids = []
        for c, n in zip(ctx, new):
            for _ in range(-(-(c + n) // BS) - -(-c // BS)):
                ok, b = self.pool.try_allocate_block()
                assert ok
                ids.append(b)
        return ids


def _qkv(n, g, kind):
    import torch

    x = torch.randn(n, (H + 2 * HK) * D, device="cuda", generator=g).to(kind)
    return x[:, :H * D].view(n, H, D), x[:, H * D:(H + HK) * D].view(n, HK, D), x[:, (H + HK) * D:].view(n, HK, D)


@pytest.mark.parametrize("kind_name,arena", [("bfloat16", "bf16"), ("float16", "f16"), ("float32", "f32")])
def test_prompts_then_tokens(cuda, kind_name, arena):
    import torch

    kind = getattr(torch, kind_name)
    g = torch.Generator(device="cuda").manual_seed(11)
    lens, scale = [70, 1, 0, 300, 16], 1 / math.sqrt(D)
    B, cap, width = len(lens), 400, 24
    pool = G.PagedBlockPool(60, 1, HK, D, BS, dtype=arena)
    pool.reserve_step(B, width, cap, H)
    pool.set_static_step()
    rope = G.MultiAxisRope([24, 20, 20], D, interleaved=True)
    host = Host(pool, rope, B, kind)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    ctx, new, fresh = i32([0] * B), i32(lens), torch.full((64,), -1, dtype=torch.int32, device="cuda")
    ids = host.blocks([0] * B, lens)
    fresh[:len(ids)] = i32(ids)
    io = G.StepBuffers(tables, ctx, new, fresh, cap)
    pool.build_step(io, n_new_blocks=len(ids))
    n = sum(lens)
    q, k, v = _qkv(cap, g, kind)
    pos = torch.randint(0, 5000, (3, cap), dtype=torch.int32, device="cuda", generator=g)
    q_out, k_out = torch.full((cap, H, D), 7.0, dtype=kind, device="cuda"), torch.full((cap, HK, D), 7.0, dtype=kind, device="cuda")
    out = torch.full((cap, H, D), 7.0, dtype=kind, device="cuda")
    pool.mrope_append(0, q, k, v, pos, rope, q_out, k_out)
    pool.prompt_attention(q_out, k_out, v, io.cu_new, out, scale)
    pool.sync()
    # the attention against its definition on the rotated tensors it was given
    cu = np.concatenate([[0], np.cumsum(lens)]).tolist()
    assert io.cu_new.tolist() == cu
    ref, _, size, _ = prompt_reference(q_out[:n], k_out[:n], v[:n], cu, scale)
    u = 0.0 if kind == torch.float32 else unit(kind)
    assert_within(out[:n], ref, (u + 1e-4) * size + (u + 1e-6) * ref.abs(), "prompt attention")
    assert bool((out[n:] == 7.0).all()) and bool((q_out[n:] == 7.0).all())
    kr, _ = rope_reference(k[:n], pos[:, :n], rope.axis, rope.inv_freq, 0, 1.0)
    for b in range(B):
        host.keys[b].append(kr[cu[b]:cu[b + 1]])
        host.values[b].append(v[cu[b]:cu[b + 1]].double())

    # next tokens: one captured graph, replayed with other lengths, blocks and rows each time
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    qd, kd, vd = (x.clone() for x in _qkv(cap, g, kind))
    pd = torch.zeros(3, cap, dtype=torch.int32, device="cuda")
    q32 = torch.empty(cap, H, D, device="cuda")
    dec = torch.full((B, H, D), 7.0, device="cuda")

    def step():
        pool.build_step(io, stream=s)
        pool.mrope_append(0, qd, kd, vd, pd, rope, q32, stream=s)
        pool.paged_decode(0, q32, dec, H, scale, stream=s)

    with torch.cuda.stream(s):
        ctx.copy_(i32(lens))
        new.zero_()
        step()  # first use, with nothing to append
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    stored = list(lens)
    for turn in range(20):
        # requests 0, 1 and 3 decode; 2 starts late; 4 skips odd turns.  Rows and the decode's queries go by request only
        # where every request adds one token
        add = [1, 1, 1 if turn >= 3 else 0, 1, 1 if turn % 2 == 0 else 0]
        rows = [b for b in range(B) if add[b]]
        ids = host.blocks(stored, add)
        with torch.cuda.stream(s):
            ctx.copy_(i32(stored))
            new.copy_(i32(add))
            fresh.fill_(-1)
            if ids:
                fresh[:len(ids)] = i32(ids)
            a, b_, c = _qkv(cap, g, kind)
            qd.copy_(a), kd.copy_(b_), vd.copy_(c)
            pd.copy_(torch.randint(0, 100000, (3, cap), dtype=torch.int32, device="cuda", generator=g))
            dec.fill_(7.0)
            graph.replay()
        s.synchronize()
        pool.sync(s)
        m = len(rows)
        kr, _ = rope_reference(kd[:m], pd[:, :m], rope.axis, rope.inv_freq, 0, 1.0)
        for i, b in enumerate(rows):
            host.keys[b].append(kr[i:i + 1])
            host.values[b].append(vd[i:i + 1].double())
            stored[b] += 1
        assert io.ctx_out.tolist() == stored
        # the decode reads row b of q32 for request b: hold it to the definition on that
        for b in range(B):
            if stored[b] == 0:
                assert bool((dec[b] == 7.0).all())
                continue
            kk, vv = torch.cat(host.keys[b]), torch.cat(host.values[b])
            for h in range(H):
                w = torch.softmax(scale * (kk[:, h // (H // HK)] @ q32[b, h].double()), 0)
                x = vv[:, h // (H // HK)]
                # keys and values rounded by half a step each (a score by that of sum |q k|), p and q on the tensor path too
                es = (2 * u + 1e-4) * scale * float((kk[:, h // (H // HK)].abs() @ q32[b, h].double().abs()).max())
                tol = (2 * es + 2 * u + 1e-4) * (w @ x.abs())
                assert_within(dec[b, h], w @ x, tol, f"turn {turn} request {b} head {h}")
    graph.reset()
    pool.set_static_step(False)
    pool.close()

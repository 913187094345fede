"""gkv_mrope_append against its formulas in 64 bits."""
import numpy as np
import pytest

import glacier_kv as G
from operator_refs import assert_within, rope_reference, rope_tolerance

pytestmark = pytest.mark.gpu

KIND = {"f32": "float32", "bf16": "bfloat16", "f16": "float16", "fp8": "float8_e4m3fn"}


def _kind(name):
    import torch

    return getattr(torch, KIND[name])


def _slots(rng, n, blocks, bs):
    pages = -(-n // bs)
    ids = rng.permutation(blocks)[:pages]
    return (ids[np.arange(n) // bs] * bs + np.arange(n) % bs).astype(np.int64)


def _cache(pool, n):
    """The arena as values of its type, [blocks, layers, heads, slots, dim]."""
    import torch

    return [x.view(torch.float8_e4m3fn) if pool.dtype == "fp8" else x for x in (pool.key_view(), pool.value_view())]


@pytest.mark.parametrize("n", [1, 3, 37, 1500])
@pytest.mark.parametrize("dtype,out,cache,heads,heads_kv,d,dv,rope_dim,sections,interleaved,style,norm,bias", [
    ("bf16", "bf16", "bf16", 28, 4, 128, 128, 128, [24, 20, 20], False, 0, False, True),
    ("bf16", "f32", "fp8", 28, 4, 128, 128, 128, [24, 20, 20], True, 0, True, False),
    ("f32", "f32", "f32", 8, 2, 64, 64, 32, [4, 6, 6], True, 0, True, True),
    ("f32", "bf16", "f16", 4, 4, 256, 128, 256, [128], False, 1, False, False),
    ("f16", "f16", "bf16", 7, 1, 32, 32, 16, [2, 2, 2, 2], False, 1, True, False),
    ("f16", "f32", "f16", 6, 2, 64, 40, 64, [16, 16], True, 1, False, True),
    ("bf16", "bf16", "f32", 2, 2, 128, 128, 48, [12, 12], False, 0, True, True),
])
def test_formula(cuda, n, dtype, out, cache, heads, heads_kv, d, dv, rope_dim, sections, interleaved, style, norm, bias):
    import torch

    rng = np.random.default_rng(n + d)
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    kind, okind = _kind(dtype), _kind(out)
    fused = r(n, heads * d + heads_kv * (d + dv)).to(kind) if (heads_kv * dv) % 8 == 0 else None
    q = fused[:, :heads * d].view(n, heads, d)
    k = fused[:, heads * d:(heads + heads_kv) * d].view(n, heads_kv, d)
    v = fused[:, (heads + heads_kv) * d:].view(n, heads_kv, dv)
    blocks = -(-n // 16) + 2
    pool = G.PagedBlockPool(blocks, 2, heads_kv, d, 16, v_head_dim=dv, dtype=cache)
    scales = [np.linspace(0.01, 0.03, 2 * heads_kv).astype(np.float32) for _ in range(2)]
    if cache == "fp8":
        pool.set_kv_scales(*scales)
    slots = _slots(rng, n, blocks, 16)
    if n > 2:
        slots[1] = -1
    pool.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), slots)
    rope = G.MultiAxisRope(sections, rope_dim, interleaved=interleaved, style=style, mscale=1.25)
    pos = torch.tensor(rng.integers(0, 1_000_000, (len(sections), n)), dtype=torch.int32, device="cuda")
    w = [1 + 0.1 * r(d) for _ in range(2)] if norm else [None, None]
    b = [r(heads * d), r(heads_kv * d), r(heads_kv * dv)] if bias else [None] * 3
    q_out, k_out, v_out = (torch.full((n, h, m), 9.0, dtype=okind, device="cuda") for h, m in ((heads, d), (heads_kv, d), (heads_kv, dv)))
    before = [x.clone() for x in _cache(pool, n)]
    pool.mrope_append(1, q, k, v, pos, rope, q_out, k_out, v_out, q_bias=b[0], k_bias=b[1], v_bias=b[2], q_norm=w[0], k_norm=w[1])
    pool.sync()
    assert pool.last_launch_count == 1
    args = (pos, rope.axis, rope.inv_freq, style, 1.25)
    qr, qs = rope_reference(q, *args, bias=b[0], weight=w[0])
    kr, ks = rope_reference(k, *args, bias=b[1], weight=w[1])
    vr, vs = rope_reference(v, pos, [], [], 0, 1.0, bias=b[2])
    for got, ref, size, what in ((q_out, qr, qs, "q"), (k_out, kr, ks, "k"), (v_out, vr, vs, "v")):
        assert_within(got, ref, rope_tolerance(ref, size, d, okind), what)
    kept = torch.tensor(slots >= 0, device="cuda")
    st = torch.tensor(slots, device="cuda")[kept]
    for i, (got, was, ref, size) in enumerate(zip(_cache(pool, n), before, (kr, vr), (ks, vs))):
        ref, size = ref[kept], size[kept]
        if cache == "fp8":
            s = torch.tensor(scales[i][heads_kv:], device="cuda").double()[None, :, None]
            ref, size = (ref / s).clamp(-448, 448), size / s
        stored = got.float()[st // 16, 1, :, st % 16]
        assert_within(stored, ref, rope_tolerance(ref, size, d, _kind(cache)), f"cache {i}")
        # nothing else of the arena changed
        rest = got.view(torch.uint8).clone()
        rest[st // 16, 1, :, st % 16] = was.view(torch.uint8)[st // 16, 1, :, st % 16]
        assert torch.equal(rest, was.view(torch.uint8))
    pool.close()


def test_in_place_and_without_keeping(cuda):
    import torch

    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(9, h, 64, device="cuda", generator=g) for h in (4, 2, 2))
    pool = G.PagedBlockPool(2, 1, 2, 64, 16, dtype="f32")
    pool.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), np.arange(9, dtype=np.int64))
    rope = G.MultiAxisRope([16, 8, 8], 64)
    pos = torch.arange(27, dtype=torch.int32, device="cuda").view(3, 9)
    want = torch.empty_like(q)
    pool.mrope_append(0, q, k, v, pos, rope, want)
    pool.mrope_append(0, q, k, v, pos, rope, q)
    pool.sync()
    assert torch.equal(q, want)
    pool.close()


def test_equal_axes_are_plain_rope(cuda):
    """With the same position on every axis the rotation is gkv_rope_append's, up to its angle in 32 bits."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(50, h, 128, device="cuda", generator=g) for h in (8, 2, 2))
    pool = G.PagedBlockPool(4, 2, 2, 128, 16, dtype="f32")
    pool.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), np.arange(50, dtype=np.int64))
    at = np.arange(50, dtype=np.int32) * 3
    rope = G.MultiAxisRope([24, 20, 20], 128, interleaved=True)
    out = torch.empty_like(q)
    pool.mrope_append(0, q, k, v, torch.tensor(at, device="cuda").repeat(3, 1), rope, out)
    plain = q.clone()
    pool.rope_append(1, plain, k, v, at, 8)
    pool.sync()
    # angles up to 147 rad: half a step of them is 2^-17; pairs of size 8 at most
    assert float((out - plain).abs().max()) <= 8 * 2.0 ** -16
    assert float((pool.key_view()[:, 0] - pool.key_view()[:, 1]).abs().max()) <= 8 * 2.0 ** -16
    assert torch.equal(pool.value_view()[:, 0], pool.value_view()[:, 1])
    pool.close()


def test_far_and_negative_positions_keep_their_angle(cuda):
    import torch

    q, k, v = (torch.zeros(4, 1, 64, device="cuda") for _ in range(3))
    q[..., :32] = 1.0  # out = (cos, sin)
    pool = G.PagedBlockPool(1, 1, 1, 64, 16, dtype="f32")
    pool.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), np.arange(4, dtype=np.int64))
    rope = G.MultiAxisRope([32], 64)
    pos = torch.tensor([[2147483647, -1, -2147483648, 123456789]], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    pool.mrope_append(0, q, k, v, pos, rope, out)
    pool.sync()
    theta = pos[0].cpu().numpy().astype(np.longdouble)[:, None] * rope.inv_freq.astype(np.longdouble)
    got = out[:, 0].cpu().numpy()
    # the 64-bit product is off by 2^-53 of an angle of up to 2^31: below 2^-22 rad
    assert np.abs(got[:, :32] - np.cos(theta)).max() <= 2.0 ** -21 + 2.0 ** -22
    assert np.abs(got[:, 32:] - np.sin(theta)).max() <= 2.0 ** -21 + 2.0 ** -22
    pool.close()


def test_bad_slots_are_reported(cuda):
    """In the static layout a slot comes from the device; the host checks the uploaded ones.  Ids past the
    pool give slot -1 there, and the row's q is still written."""
    import torch

    pool = G.PagedBlockPool(4, 1, 1, 64, 16, dtype="bf16")
    pool.reserve_step(1, 2, 3, 1)
    pool.set_static_step()
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    io = G.StepBuffers(t([[77, -1]]), t([2]), t([2]), t([]), max_tokens=3)
    pool.build_step(io)
    q, k, v = (torch.ones(3, 1, 64, device="cuda") for _ in range(3))
    out = torch.full_like(q, 5.0)
    pool.mrope_append(0, q, k, v, t([[2, 3, 4]]), G.MultiAxisRope([32], 64), out)
    with pytest.raises(G.DeviceError):
        pool.sync()
    assert bool((out[:2] != 5.0).all()) and bool((out[2] == 5.0).all())  # two rows in the step
    assert not bool(pool.key_view().any())
    pool.close()


def test_refusals(cuda):
    import torch

    q, k, v = (torch.zeros(4, h, 64, device="cuda") for h in (4, 2, 2))
    pos, rope, out = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), G.MultiAxisRope([16, 8, 8], 64), torch.empty_like(q)
    pool = G.PagedBlockPool(2, 1, 2, 64, 16, dtype="f32")
    with pytest.raises(G.InvalidOperationError):
        pool.mrope_append(0, q, k, v, pos, rope, out)  # no step
    pool.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), np.arange(4, dtype=np.int64))
    bad = G.ArgumentOutOfRangeError
    with pytest.raises(bad):
        pool.mrope_append(1, q, k, v, pos, rope, out)  # layer
    five = [torch.zeros(5, h, 64, device="cuda") for h in (4, 2, 2)]
    with pytest.raises(bad):
        pool.mrope_append(0, *five, torch.zeros(3, 5, dtype=torch.int32, device="cuda"), rope, torch.empty_like(five[0]))  # rows
    with pytest.raises(bad):
        pool.mrope_append(0, q[:, :3], k, v, pos, rope, out[:, :3].contiguous())  # heads
    with pytest.raises(bad):
        pool.mrope_append(0, q, k, v, pos, rope, out, k_out=k)  # an input's address
    shared = torch.empty(4, 2, 64, device="cuda")
    with pytest.raises(bad):
        pool.mrope_append(0, q, k, v, pos, rope, out, k_out=shared, v_out=shared)
    with pytest.raises(bad):
        pool.mrope_append(0, q, k, v, pos, G.MultiAxisRope([16, 8, 8], 64, style=2), out)
    with pytest.raises(bad):
        pool.mrope_append(0, q, k, v, pos, G.MultiAxisRope([32, 16, 16], 128), out)  # rope_dim > head_dim
    with pytest.raises(G.UnsupportedError):
        pool.mrope_append(0, q, k, v, pos, G.MultiAxisRope([4, 4, 2], 20), out)
    wide = torch.zeros(4, 4 * 64 + 2, device="cuda")
    with pytest.raises(bad):
        pool.mrope_append(0, wide[:, 1:257].view(4, 4, 64), k, v, pos, rope, out)  # off the 16-byte boundary
    with pytest.raises(bad):
        pool.mrope_append(0, wide[:, :256].view(4, 4, 64), k, v, pos, rope, out)   # rows off it
    odd = torch.zeros(4 * 64 + 1, device="cuda")[1:]
    with pytest.raises(bad):
        pool.mrope_append(0, q, k, v, pos, rope, out, q_bias=odd)
    with pytest.raises(bad):
        pool.mrope_append(0, q, k, v, pos, rope, out, k_norm=odd[:64])
    with pytest.raises(ValueError):
        pool.mrope_append(0, q, k.half(), v, pos, rope, out)
    with pytest.raises(ValueError):
        pool.mrope_append(0, q, k, v, pos[:2].contiguous(), rope, out)
    with pytest.raises(ValueError):
        pool.mrope_append(0, q, k, v, pos.long(), rope, out)
    with pytest.raises(ValueError):
        pool.mrope_append(0, q.transpose(1, 2), k, v, pos, rope, out)
    other = G.PagedBlockPool(2, 1, 2, 96, 16, dtype="f32")
    other.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), np.arange(4, dtype=np.int64))
    x = [torch.zeros(4, h, 96, device="cuda") for h in (4, 2, 2)]
    with pytest.raises(G.UnsupportedError):
        other.mrope_append(0, *x, pos, G.MultiAxisRope([24, 12, 12], 96), torch.empty_like(x[0]))
    pool.close()
    other.close()


@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("n", [592, 593, 2049, 9472, 9473, 20001])
def test_tokens_of_a_block(cuda, n, static):
    """Counts around those that change how many tokens a block takes; in the static layout fewer rows than reserved."""
    import torch

    rng = np.random.default_rng(n)
    g = torch.Generator(device="cuda").manual_seed(n)
    heads, heads_kv, d, cap = 3, 1, 32, n + 9000 if static else n
    blocks = -(-n // 16)
    pool = G.PagedBlockPool(blocks, 1, heads_kv, d, 16, dtype="f32")
    slots = _slots(rng, n, blocks, 16)
    if static:
        pool.reserve_step(1, 1, cap, heads)
        pool.set_static_step()
    pool.upload_step(np.zeros((1, 1), np.int32), np.ones(1, np.int32), slots)
    q, k, v = (torch.randn(cap, h, d, device="cuda", generator=g) for h in (heads, heads_kv, heads_kv))
    bias = torch.randn(heads * d, device="cuda", generator=g)
    norm = 1 + 0.1 * torch.randn(d, device="cuda", generator=g)
    rope = G.MultiAxisRope([8, 8], d)
    pos = torch.tensor(rng.integers(0, 100_000, (2, cap)), dtype=torch.int32, device="cuda")
    q_out = torch.full_like(q, 9.0)
    pool.mrope_append(0, q, k, v, pos, rope, q_out, q_bias=bias, q_norm=norm)
    pool.sync()
    args = (pos[:, :n], rope.axis, rope.inv_freq, 0, 1.0)
    ref, size = rope_reference(q[:n], *args, bias=bias, weight=norm)
    assert_within(q_out[:n], ref, rope_tolerance(ref, size, d, q.dtype), "q")
    assert bool((q_out[n:] == 9.0).all())
    ref, size = rope_reference(k[:n], *args)
    at = torch.tensor(slots, device="cuda")
    keys, values = (x[:, 0, 0].reshape(-1, d)[at] for x in (pool.key_view(), pool.value_view()))
    assert_within(keys[:, None], ref, rope_tolerance(ref, size, d, q.dtype), "k")
    assert torch.equal(values, v[:n, 0])
    pool.close()

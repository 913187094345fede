"""The step operators' definitions in 64 bits, and what the roundings of their kernels may add up to."""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float8_e4m3fn: 2.0 ** -4}


def unit(dtype):
    """Half a step of the type, relative to the value."""
    return U[dtype]


def step_reference(ctx, new, tables, new_blocks, bs, max_tokens):
    """What gkv_step_build writes, request by request: (tables, ctx_out, cu, slots, positions, counts, step ctx, left out)."""
    tables = [list(r) for r in tables]
    width = len(tables[0]) if tables else 0
    cu, first, slots, positions, ctx_out, step_ctx, left = [0], 0, [], [], [], [], []
    used = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        fits = c >= 0 and n >= 0 and c + n <= width * bs
        c0, n0 = max(c, 0), max(n, 0)
        old = -(-c0 // bs)
        opened = -(-(c0 + n0) // bs) - old if fits else 0
        ok = fits and (n0 == 0 or cu[-1] + n0 <= max_tokens) and (opened == 0 or first + opened <= len(new_blocks))
        if ok:
            tables[b][old:old + opened] = new_blocks[first:first + opened]
            if opened:
                used = first + opened
        for i in range(n0):
            p = c0 + i
            positions.append(p)
            slots.append(tables[b][p // bs] * bs + p % bs if ok else -1)
        cu.append(cu[-1] + n0)
        first += opened
        ctx_out.append(c0 + n0 if ok else c0)
        step_ctx.append(c0 + n0 if ok else 0)
        if not ok:
            left.append(b)
    rows = min(cu[-1], max_tokens)
    return tables, ctx_out, cu, slots[:rows], positions[:rows], [cu[-1], used], step_ctx, left


def prompt_reference(q, k, v, cu, scale, sinks=None):
    """(out, lse, weighted |v|, largest sum of |q k| products) of causal attention in 64 bits; rows outside cu are 0."""
    q, k, v = q.double(), k.double(), v.double()
    h, hk = q.shape[1], k.shape[1]
    out = torch.zeros(q.shape[0], h, v.shape[2], dtype=torch.float64, device=q.device)
    size, lse, most = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device), 0.0
    for b, e in zip(cu, cu[1:]):
        for head in range(h):
            kk, vv = k[b:e, head * hk // h], v[b:e, head * hk // h]
            for i in range(b, e, 1024):
                j = min(e, i + 1024)
                seen = torch.arange(i, j, device=q.device)[:, None] >= torch.arange(b, e, device=q.device)[None]
                s = torch.where(seen, scale * (q[i:j, head] @ kk.T), -math.inf)
                norm = torch.logsumexp(s, 1)
                if sinks is not None:
                    norm = torch.logaddexp(norm, sinks[head].double())
                p = torch.where(seen, torch.exp(s - norm[:, None]), 0.0)
                out[i:j, head], size[i:j, head], lse[i:j, head] = p @ vv, p @ vv.abs(), norm
                most = max(most, abs(scale) * float(torch.where(seen, q[i:j, head].abs() @ kk.abs().T, 0.0).max()))
    return out, lse, size, most


def prompt_tolerance(out, size, most, d, longest, dtype, v_max=8.0):
    """(tolerance of out, of lse).  A score is a sum of d products in 32 bits: off by at most (d + 2) 2^-24 of the sum of
    the products' sizes, and its exponential by that and 2^-21 (base-2 scaling, the exponential unit).  Sums of up to
    `longest` terms in 32 bits add longest 2^-24, taken as its square root times 4 (the order varies, the terms' errors
    are independent).  16-bit types round each p, and the result, by half a step.  fp16 has steps of 2^-24 below 2^-14, so
    there a rounding is off by up to 2^-25 whatever the value: once for the result, and for each of `longest` weights (the
    row's largest is 1 or more, and so is their sum) times values of at most v_max."""
    f = (d + 2) * 2.0 ** -24 * most + 2.0 ** -21 + 4 * math.sqrt(longest) * 2.0 ** -24
    u = 0.0 if dtype == torch.float32 else unit(dtype)
    tiny = 2.0 ** -25 * (1 + longest * v_max) if dtype == torch.float16 else 1e-30
    return (2 * f + u) * size + (u + 2.0 ** -23) * out.abs() + tiny, 2 * f + 2.0 ** -22 * 32


def rope_reference(x, positions, axis, inv_freq, style, mscale, bias=None, weight=None, eps=1e-6):
    """(turned x, |first| + |second| of each element's pair) in 64 bits; x [n, heads, d]."""
    x = x.double()
    if bias is not None:
        x = x + bias.double().view(1, x.shape[1], x.shape[2])
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    half = len(inv_freq)
    size = x.abs()
    if half == 0:
        return x, size
    theta = torch.stack([positions[int(axis[i])].double() * float(inv_freq[i]) for i in range(half)], 1)[:, None]
    at = torch.arange(half, device=x.device)
    first, second = (at, at + half) if style == 0 else (2 * at, 2 * at + 1)
    a, b = x[..., first], x[..., second]
    y = x.clone()
    y[..., first] = (a * theta.cos() - b * theta.sin()) * mscale
    y[..., second] = (b * theta.cos() + a * theta.sin()) * mscale
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(mscale)
    return y, size


def rope_tolerance(y, size, d, dtype):
    """A norm's sum of d squares and its root are off by at most (d + 8) 2^-24, cos and sin by 2^-22, the pair's products
    and sum by 3 roundings; then the destination's half step (and half its smallest subnormal)."""
    tiny = {torch.float16: 2.0 ** -25, torch.float8_e4m3fn: 2.0 ** -10}.get(dtype, 1e-38)
    return size * ((d + 16) * 2.0 ** -24 + 2.0 ** -21) + unit(dtype) * y.abs() + tiny


def assert_within(got, ref, tol, what=""):
    off = (got.double() - ref).abs()
    bad = ~(off <= tol)
    if bool(bad.any()):
        i = int(torch.argmax(torch.where(bad, off / tol, torch.zeros_like(off)).flatten().nan_to_num(math.inf)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got {float(got.flatten()[i])}, "
                             f"want {float(ref.flatten()[i])} +- {float(tol.expand_as(ref).flatten()[i])}")

"""Plain 64-bit forms of the streaming operators, and how far a correct kernel
may be from them."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def seen_mask(queries, keys, window, sinks, frame):
    """bool [queries, keys] of positions (int64 tensors)."""
    fq, fk = queries[:, None] // frame, keys[None, :] // frame
    mask = fk <= fq
    if window is not None:
        mask = mask & ((fq - fk < window) | (fk < sinks))
    return mask


def attend(q, k, v, mask, scale=None):
    """(o, base-2 lse, sum of p |v|) of q [H, n, D] over k, v [Hk, m, D], mask [n, m]; keys that no query sees are
    left out, whatever they hold."""
    used = mask.any(0)
    k, v, mask = k[:, used], v[:, used], mask[:, used]
    group = q.shape[0] // k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(group, 0), v.double().repeat_interleave(group, 0)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    z = (q @ k.transpose(1, 2) * scale).masked_fill(~mask, -math.inf)
    if z.shape[-1] == 0:
        return torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device), torch.zeros_like(q)
    lse = torch.logsumexp(z, -1, keepdim=True)
    p = torch.where(lse > -math.inf, torch.exp(z - lse), 0.0)
    return p @ v, (lse / math.log(2))[..., 0], p @ v.abs()


def check_output(got, o, spread, dtype):
    """P and the output are rounded once each, by at most half a step: |error| <= u (sum p |v| + |o|), and the float32
    sums and exponentials add parts of 1e-4 of that scale."""
    u = HALF_STEP[dtype]
    room = u * (1 + u) * (spread + o.abs()) + 1e-4 * u / HALF_STEP[torch.bfloat16] * spread + 1e-5 * spread + 1e-7
    worst = ((got.double() - o).abs() - room).max().item() if o.numel() else 0.0
    assert worst <= 0, worst


def check_lse(got, lse, dim, size):
    """size: the largest sum |q k| scale of a logit; dim products of exact 16-bit values are added in float32."""
    assert torch.equal(torch.isinf(got), torch.isinf(lse))
    fine = ~torch.isinf(lse)
    if fine.any():
        room = 2.0 ** -24 * (dim * size * 1.4427 + 64 + 4 * lse[fine].abs().max().item())
        worst = (got.double() - lse)[fine].abs().max().item()
        assert worst <= room, (worst, room)


def logit_size(q, k, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else abs(scale)
    finite = lambda t: torch.nan_to_num(t.double(), 0.0, 0.0, 0.0)  # noqa: E731
    return scale * finite(q).norm(dim=-1).max().item() * finite(k).norm(dim=-1).max().item() if q.numel() and k.numel() else 0.0


def turned(x, positions, axes, theta=10000.0, halves=False, joint=False, inverse=False):
    """rotary of x [B, H, N, D] in 64 bits; positions [N, A] or [B, N, A]."""
    x = x.double().clone()
    positions = positions.double() if positions.ndim == 3 else positions.double()[None].expand(x.shape[0], -1, -1)
    base, total = 0, sum(axes)
    for axis, dims in enumerate(axes):
        for j in range(dims // 2):
            freq = theta ** -(2.0 * (base + j) / total if joint else 2.0 * j / dims)
            angle = positions[:, None, :, axis] * freq * (-1 if inverse else 1)
            i = base + j
            a, b = (i, i + total // 2) if halves else (2 * i, 2 * i + 1)
            xa, xb = x[..., a].clone(), x[..., b].clone()
            x[..., a] = xa * angle.cos() - xb * angle.sin()
            x[..., b] = xa * angle.sin() + xb * angle.cos()
        base += dims // 2
    return x


def attend_grad(q, k, v, do, mask, dlse=None, scale=None):
    """(dq, dk, dv) of ``attend`` in 64 bits, and how far a kernel may be that rounds P, dS, the output (which delta is
    made of) and each gradient once, by at most half a step, relative to u."""
    group = q.shape[0] // k.shape[0]
    heads, n, dim = k.shape
    scale = dim ** -0.5 if scale is None else scale
    q, do = q.double(), do.double()
    k, v = k.double().repeat_interleave(group, 0), v.double().repeat_interleave(group, 0)
    z = (q @ k.transpose(1, 2) * scale).masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(z, -1, keepdim=True)
    p = torch.where(lse > -math.inf, torch.exp(z - lse), 0.0)
    o = p @ v
    dp = do @ v.transpose(1, 2)
    delta = (do * o).sum(-1, keepdim=True)
    if dlse is not None:
        delta = delta - dlse.double()[..., None] / math.log(2)
    ds = p * (dp - delta)
    off = p * (do.abs() * (p @ v.abs() + o.abs())).sum(-1, keepdim=True)  # of dS, from P's and the output's rounding
    # float32 sums of dim products in dP, and P's own error of some 2^-17 from the logits', next to u of 2^-11 at least
    noise = p * (do.abs() @ v.abs().transpose(1, 2)) + off + p * delta.abs()
    size = ds.abs() + off + 2.0 ** -6 * noise

    def shared(x):
        return x.reshape(heads, group, n, dim).sum(1)

    dq = scale * ds @ k
    dk, dv = shared(scale * ds.transpose(1, 2) @ q), shared(p.transpose(1, 2) @ do)
    rooms = (abs(scale) * size @ k.abs() + dq.abs(), shared(abs(scale) * size.transpose(1, 2) @ q.abs()) + dk.abs(),
             shared(1.01 * p.transpose(1, 2) @ do.abs()) + dv.abs())
    return (dq, dk, dv), rooms


def check_gradient(got, want, room, dtype, name=""):
    """u times the room, with 2 % for products of roundings, and the float32 arithmetic's 2^-17 of it."""
    u = HALF_STEP[dtype]
    worst = ((got.double() - want).abs() - (1.02 * u + 2.0 ** -17) * room - 1e-7).max().item() if want.numel() else 0.0
    assert worst <= 0, (name, worst)

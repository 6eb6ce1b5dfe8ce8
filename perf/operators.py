"""Operators of streaming video transformers, and the sizes their speed is
measured on: rotary positions over (time, height, width), attention that is
causal over frames with a sliding window and first frames that stay visible
(forward and backward), the write of new keys and values into a paged cache,
and the attention of a chunk of new tokens over that cache.

A case is a dict of plain values. ``listed()`` gives the fixed ones, ``draw``
another of the same ranges; ``prepare`` makes a case's inputs from a seed,
``run`` makes one pass (the operators' plain forms in elementary torch
operations, or with ``own`` the library's), ``work`` counts the bytes and
operations a pass cannot do without, ``exact`` computes the outputs in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

# Values a case holds besides its name:
#   op           rotary | window | append | chunk
#   dtype        bf16 | fp16 | fp32
#   batch        batch items (rotary, window) or sequences (append, chunk)
#   heads, kv_heads, dim
#   grad         the backward pass too
#   token_major  [.., tokens, heads, dim] in memory, as a linear projection leaves it
#   frames, height, width, first   rotary: tokens of a latent grid, its first frame's position
#   axes, theta, halves, joint     rotary: dims of each axis, the base, the pairing, one frequency scale for all axes
#   tokens, window, sinks, frame   window, chunk: sizes of the mask (window and sinks in frames, frame in tokens;
#                                  window 0: everything before stays visible)
#   ragged       window: a padded batch with lengths of its own; append, chunk: sequences of their own sizes
#   chunk, cached, page            append, chunk: most new tokens and most tokens in all of a sequence, tokens of a page
_BASE = dict(dtype="bf16", batch=1, heads=1, kv_heads=1, dim=128, grad=False, token_major=False)
_ROTARY = dict(_BASE, op="rotary", frames=1, height=1, width=1, first=0, axes="44,42,42", theta=10000.0, halves=False,
               joint=False)
_WINDOW = dict(_BASE, op="window", tokens=1, window=0, sinks=0, frame=1, ragged=False)
_CACHE = dict(_BASE, chunk=1, cached=1, page=64, window=0, sinks=0, frame=1, ragged=False)

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One new token in each of 8 sequences: launches and latency are all there is.
        dict(_ROTARY, name="rotary_token", batch=8, heads=32, kv_heads=8, first=30011, axes="32,48,48", halves=True,
             joint=True, theta=1e6),
        # A transformer layer of Wan2.1-1.3B at 480p, Q and K as the projections leave them.
        dict(_ROTARY, name="rotary_480p", batch=2, heads=12, kv_heads=12, frames=21, height=30, width=52, token_major=True),
        # A training step's rotation and its gradient at Wan2.1-14B's 720p size.
        dict(_ROTARY, name="rotary_grad_720p", heads=40, kv_heads=40, frames=21, height=45, width=80, grad=True),
        # A short text-like sequence: a preview, where few workgroups have work.
        dict(_WINDOW, name="window_short", dtype="fp16", batch=2, heads=8, kv_heads=2, dim=64, tokens=509, window=128, sinks=4),
        # A 480p clip, causal over latent frames: the last four frames and the first one stay visible.
        dict(_WINDOW, name="window_480p", heads=12, kv_heads=12, tokens=32760, window=4, sinks=1, frame=1560, token_major=True),
        # A training step on a padded batch with shared key heads and a window in tokens.
        dict(_WINDOW, name="window_grad_ragged", batch=4, heads=16, kv_heads=4, tokens=4099, window=1024, sinks=4, ragged=True,
             grad=True),
        # A training step of the 480p clip.
        dict(_WINDOW, name="window_grad_480p", heads=12, kv_heads=12, tokens=32760, window=4, sinks=1, frame=1560, grad=True),
        # One new token in each of 32 sequences goes into the cache.
        dict(_CACHE, name="append_token", op="append", batch=32, heads=32, kv_heads=8, cached=8192, ragged=True),
        # Three new latent frames of a 480p clip go into the cache, a page a frame.
        dict(_CACHE, name="append_frames", op="append", batch=2, heads=40, kv_heads=40, chunk=4680, cached=32760, page=1560),
        # One new token in each of 32 sequences over long caches.
        dict(_CACHE, name="chunk_token", op="chunk", batch=32, heads=32, kv_heads=8, cached=16384, ragged=True),
        # Three new latent frames of a 480p clip over the last 18 frames and the first one.
        dict(_CACHE, name="chunk_frames", op="chunk", heads=40, kv_heads=40, chunk=4680, cached=32760, page=1560, window=18,
             sinks=1, frame=1560),
        # Prompts of many lengths beside single tokens, sliding window with sinks.
        dict(_CACHE, name="chunk_ragged", op="chunk", batch=12, heads=24, kv_heads=8, chunk=1111, cached=9000, page=32,
             window=4096, sinks=16, ragged=True, token_major=True),
    ]


def _log_uniform(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def _heads(rng, most):
    kv = _log_uniform(rng, 1, most)
    return dict(heads=kv * rng.choice([1, 1, 2, 4]), kv_heads=kv)


def draw(rng):
    most = {}
    for case in listed():
        w = work(case)
        b, f = most.get(case["op"], (0, 0))
        most[case["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        op = rng.choice(["rotary", "window", "window", "append", "chunk", "chunk"])
        if op == "rotary":
            case = dict(_ROTARY, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), batch=rng.choice([1, 1, 2, 3]),
                        frames=_log_uniform(rng, 1, 33), height=_log_uniform(rng, 1, 48), width=_log_uniform(rng, 1, 84),
                        first=_log_uniform(rng, 1, 100000) - 1, axes=rng.choice(["44,42,42", "16,56,56", "32,48,48", "64"]),
                        halves=rng.random() < 0.4, joint=rng.random() < 0.3, theta=rng.choice([256.0, 10000.0, 1e6]),
                        grad=rng.random() < 0.3, token_major=rng.random() < 0.4, **_heads(rng, 40))
        elif op == "window":
            frame = rng.choice([1, 1, 390, 880, 1560, 3600])
            tokens = _log_uniform(rng, 1, 30000) if frame == 1 else frame * rng.randint(1, 21)
            window = 0 if rng.random() < 0.15 else _log_uniform(rng, 16, 4096) if frame == 1 else rng.randint(1, 8)
            case = dict(_WINDOW, dtype=rng.choice(["bf16", "bf16", "fp16"]), batch=rng.choice([1, 1, 2, 3]),
                        dim=rng.choice([64, 128, 128]), tokens=tokens, window=window, frame=frame,
                        sinks=rng.choice([0, 4, 64]) if frame == 1 else rng.choice([0, 1, 1]), ragged=rng.random() < 0.3,
                        grad=rng.random() < 0.5, token_major=rng.random() < 0.4, **_heads(rng, 24))
        else:
            frame = rng.choice([1, 1, 1, 880, 1560])
            page = rng.choice([16, 32, 64, 256]) if frame == 1 else rng.choice([frame, 64])
            cached = _log_uniform(rng, 1, 40000) if frame == 1 else frame * rng.randint(1, 24)
            chunk = (rng.choice([1, 1, _log_uniform(rng, 1, 4096)]) if frame == 1 else frame * rng.choice([1, 3]))
            case = dict(_CACHE, op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), batch=_log_uniform(rng, 1, 48),
                        dim=rng.choice([64, 128, 128]), chunk=min(chunk, cached), cached=cached, page=page, frame=frame,
                        window=0 if rng.random() < 0.5 else _log_uniform(rng, 16, 8192) if frame == 1 else rng.randint(1, 12),
                        sinks=rng.choice([0, 4, 64]) if frame == 1 else rng.choice([0, 1]), ragged=rng.random() < 0.5,
                        token_major=rng.random() < 0.4, **_heads(rng, 40 if frame > 1 else 16))
        w, (b, f) = work(case), most[op]
        plain = _plain_scores(case)
        if w["bytes"] <= b and w["flops"] <= f and plain <= 4e9 and w["bytes"] >= 2048:
            return case


# ---- sizes --------------------------------------------------------------------


def _sequences(case):
    """(new tokens, tokens in all) of every sequence of a cache case; of the
    batch items of a window case, tokens in all."""
    rng = random.Random("%s %s %s" % (case["batch"], case.get("cached", 0), case.get("tokens", 0)))
    new, total = [], []
    for b in range(case["batch"]):
        most = case["cached"] if case["op"] != "window" else case["tokens"]
        n = case.get("chunk", 1)
        if case["ragged"] and b > 0:  # the first one has the full size
            most = rng.randint(max(1, most // 8), most)
            n = min(most, rng.choice([1, rng.randint(1, n), rng.randint(1, n)]))
        new.append(n)
        total.append(most)
    return new, total


def _span(case, position):
    """(visible keys that are sinks only, first key of the window, end) of the token at a position."""
    frame, window, sinks = case["frame"], case["window"], case["sinks"]
    f = position // frame
    low = 0 if window == 0 else max(0, f - window + 1) * frame
    return min(low, sinks * frame), low, (f + 1) * frame


def _visible(case, position, length):
    sink, low, high = _span(case, position)
    return sink + min(high, length) - low


def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    pairs = 0
    new, total = _sequences(case)
    for n, length in zip([0] * len(total) if case["op"] == "window" else new, total):
        first = length - n if case["op"] == "chunk" else 0
        # Token positions grouped by frame see the same keys.
        if case["frame"] == 1:
            pairs += sum(_visible(case, p, length) for p in range(first, length))
        else:
            p = first
            while p < length:
                stop = min(length, (p // case["frame"] + 1) * case["frame"])
                pairs += (stop - p) * _visible(case, p, length)
                p = stop
    return pairs


def _keys_read(case):
    """Keys that some query of a chunk sees, over the sequences."""
    keys = 0
    for n, length in zip(*_sequences(case)):
        sink, low, _ = _span(case, length - n)
        keys += sink + length - low
    return keys


def _plain_scores(case):
    """Scores that the plain form holds at once."""
    if case["op"] == "window":
        _, rows, keys = _bands(case)
        return case["batch"] * case["heads"] * rows * keys
    if case["op"] == "chunk":
        return case["batch"] * case["heads"] * case["chunk"] * (case["cached"] + case["page"])
    return 0


def work(case):
    size, dim = _BYTES[case["dtype"]], case["dim"]
    heads, kv_heads = case["heads"], case["kv_heads"]
    if case["op"] == "rotary":
        tokens = case["batch"] * case["frames"] * case["height"] * case["width"]
        values = float(tokens) * (heads + kv_heads) * dim * (2 if case["grad"] else 1)
        return {"bytes": 2 * values * size, "flops": 3 * values}
    if case["op"] == "window":
        q = float(case["batch"]) * case["tokens"] * heads * dim * size
        kv = float(case["batch"]) * case["tokens"] * kv_heads * dim * size
        flops = 4.0 * dim * heads * _pairs(case)
        if case["grad"]:  # q, k, v, dout in; out and three gradients out; five products more
            return {"bytes": 4 * q + 4 * kv, "flops": 3.5 * flops}
        return {"bytes": 2 * q + 2 * kv, "flops": flops}
    new, _ = _sequences(case)
    rows = float(sum(new))
    if case["op"] == "append":
        return {"bytes": 4 * rows * kv_heads * dim * size, "flops": 0.0}
    return {"bytes": (2 * rows * heads + 2.0 * _keys_read(case) * kv_heads) * dim * size,
            "flops": 4.0 * dim * heads * _pairs(case)}


# ---- inputs -------------------------------------------------------------------


def _normal(gen, shape, dtype, scale=1.0, token_major=False):
    """[.., heads, tokens, dim] (of which token_major has heads and tokens swapped in memory)."""
    if token_major:
        shape = (*shape[:-3], shape[-2], shape[-3], shape[-1])
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)
    return x.transpose(-3, -2) if token_major else x


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, dim = _TYPES[case["dtype"]], case["dim"]
    batch, heads, kv_heads = case["batch"], case["heads"], case["kv_heads"]
    state = {"case": case}
    if case["op"] == "rotary":
        grid = torch.meshgrid(torch.arange(case["frames"], device="cuda") + case["first"],
                              torch.arange(case["height"], device="cuda"), torch.arange(case["width"], device="cuda"),
                              indexing="ij")
        axes = tuple(int(a) for a in case["axes"].split(","))
        positions = torch.stack([g.reshape(-1) for g in grid], -1)[:, :len(axes)]
        if positions.shape[0] == 1:  # single tokens of sequences that are in different places
            positions = torch.randint(0, case["first"] + 1, (batch, 1, len(axes)), generator=gen, device="cuda")
        state["positions"], state["axes"] = positions.contiguous(), axes
        tokens = positions.shape[-2]
        for name, h in (("q", heads), ("k", kv_heads)):
            state[name] = _normal(gen, (batch, h, tokens, dim), dtype, token_major=case["token_major"])
            if case["grad"]:
                state["d" + name] = _normal(gen, (batch, h, tokens, dim), dtype, token_major=case["token_major"])
        return state
    if case["op"] == "window":
        tokens = case["tokens"]
        # Logits with a standard deviation of 2: a few keys carry a row.
        state["q"] = _normal(gen, (batch, heads, tokens, dim), dtype, 2.0, case["token_major"])
        state["k"] = _normal(gen, (batch, kv_heads, tokens, dim), dtype, 1.0, case["token_major"])
        state["v"] = _normal(gen, (batch, kv_heads, tokens, dim), dtype, 1.0, case["token_major"])
        if case["grad"]:
            state["dout"] = _normal(gen, (batch, heads, tokens, dim), dtype, 1.0, case["token_major"])
        state["lengths"] = torch.tensor(_sequences(case)[1], dtype=torch.int32, device="cuda") if case["ragged"] else None
        return state
    new, total = _sequences(case)
    page, rows = case["page"], sum(new)
    needed = [-(-t // page) for t in total]
    pages = sum(needed) + 3
    shape = (pages, kv_heads, page, dim)
    state["k_cache"] = _normal(gen, shape, dtype, 1.0, case["token_major"])
    state["v_cache"] = _normal(gen, shape, dtype, 1.0, case["token_major"])
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.full((batch, max(needed)), -1, dtype=torch.int32)
    at = 0
    for b, count in enumerate(needed):
        table[b, :count] = order[at:at + count]
        at += count
        if case["op"] == "chunk" and case["window"]:  # pages that no query sees any more are given back
            sink, low, _ = _span(case, total[b] - new[b])
            table[b, -(-sink // page):low // page] = -1
    state["table"] = table.cuda()
    state["lengths"] = torch.tensor(total, dtype=torch.int32, device="cuda")
    state["offsets"] = torch.tensor([0] + new, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    if case["op"] == "append":
        state["k"], state["v"] = (_normal(gen, (rows, kv_heads, dim), dtype) for _ in range(2))
    else:
        state["q"] = _normal(gen, (rows, heads, dim), dtype, 2.0)
        state["most"], state["keys"] = max(new), table.shape[1] * page
    return state


# ---- one pass -----------------------------------------------------------------


def run(state):
    return {"rotary": _rotary, "window": _window, "append": _append, "chunk": _chunk}[state["case"]["op"]](state)


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ab-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ab_attention import streaming

    return streaming


def _frequencies(axes, theta, joint):
    """(axis of every pair, its frequency in 64 bits)"""
    axis = [a for a, d in enumerate(axes) for _ in range(d // 2)]
    if joint:
        return axis, [theta ** (-2.0 * i / sum(axes)) for i in range(sum(axes) // 2)]
    return axis, [theta ** (-2.0 * i / d) for d in axes for i in range(d // 2)]


def _turn(x, cos, sin, pairs, halves):
    """x with its pairs turned; cos and sin [.., 1, tokens, pairs]."""
    f = x.float()
    a, b = (f[..., :pairs], f[..., pairs:2 * pairs]) if halves else (f[..., 0:2 * pairs:2], f[..., 1:2 * pairs:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, f[..., 2 * pairs:]], -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    if own:
        lib = _library()
        how = dict(theta=c["theta"], pairing="halves" if c["halves"] else "adjacent", joint=c["joint"])
        if not c["grad"]:
            return lib.rotary(s["q"], s["k"], s["positions"], s["axes"], **how)
        q, k = s["q"].detach().requires_grad_(), s["k"].detach().requires_grad_()
        out = lib.rotary(q, k, s["positions"], s["axes"], **how)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, (q, k), (s["dq"], s["dk"])))
    axis, freq = _frequencies(s["axes"], c["theta"], c["joint"])
    device = s["q"].device
    angle = s["positions"].double()[..., torch.tensor(axis, device=device)] * torch.tensor(freq, dtype=torch.float64, device=device)
    angle = angle[:, None] if angle.ndim == 3 else angle
    cos, sin, pairs = angle.cos().float(), angle.sin().float(), len(axis)
    out = [_turn(s["q"], cos, sin, pairs, c["halves"]), _turn(s["k"], cos, sin, pairs, c["halves"])]
    if c["grad"]:  # the transposed rotation
        out += [_turn(s["dq"], cos, -sin, pairs, c["halves"]), _turn(s["dk"], cos, -sin, pairs, c["halves"])]
    return out


def _bands(case):
    """The plain form's bands: (tokens of a block of queries, queries in all, keys that a block looks at)."""
    rows = case["frame"] if case["frame"] > 1 else 128
    blocks = -(-case["tokens"] // rows)
    span = case["window"] * rows if case["frame"] > 1 else case["window"] + rows - 1
    keys = case["sinks"] * case["frame"] + span
    return rows, blocks * rows, case["tokens"] if case["window"] == 0 or keys >= case["tokens"] else keys


def _window(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    if own:
        lib = _library()
        how = dict(window=c["window"] or None, sinks=c["sinks"], frame=c["frame"], lengths=s["lengths"])
        if not c["grad"]:
            return lib.window_attention(q, k, v, return_lse=True, **how)
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = lib.window_attention(q, k, v, **how)
        return [out.detach(), *torch.autograd.grad(out, (q, k, v), s["dout"])]
    batch, heads, n, dim = q.shape
    kv_heads, device = c["kv_heads"], q.device
    group, frame, window, sinks = heads // kv_heads, c["frame"], c["window"] or n + 1, c["sinks"]
    rows, total, keys = _bands(c)
    blocks, sink_keys = total // rows, sinks * frame
    # The keys of every block of queries, by index, and which of them are there and seen.
    if keys == n:
        at = torch.arange(n, device=device).expand(blocks, n)
        there = torch.ones_like(at, dtype=torch.bool)
    else:
        first = torch.arange(blocks, device=device) * rows - (keys - sink_keys - rows)
        band = first[:, None] + torch.arange(keys - sink_keys, device=device)
        at = torch.cat([torch.arange(sink_keys, device=device).expand(blocks, sink_keys), band], 1)
        there = torch.cat([torch.ones((blocks, sink_keys), dtype=torch.bool, device=device), band >= sink_keys], 1) & (at < n)
        at = at.clamp(0, n - 1)
    pos = torch.arange(total, device=device).reshape(blocks, rows, 1)
    fq, fk = pos // frame, (at // frame)[:, None]
    seen = there[:, None] & (fk <= fq) & ((fq - fk < window) | (fk < sinks)) & (pos < n)
    length = torch.full((batch,), n, device=device) if s["lengths"] is None else s["lengths"].long()
    length = length.reshape(batch, 1, 1, 1)
    seen = (seen & (at[:, None] < length) & (pos < length))[:, None, :, None]  # [batch, 1, blocks, 1, rows, keys]

    def queries(x):  # [batch, kv_heads, blocks, group, rows, dim]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, total - n))
        return x.reshape(batch, kv_heads, group, blocks, rows, dim).transpose(2, 3)

    def tokens(x):
        return x.transpose(2, 3).reshape(batch, heads, total, dim)[:, :, :n]

    def gathered(x):  # [batch, kv_heads, blocks, keys, dim]
        return x.float()[:, :, at.reshape(-1)].reshape(batch, kv_heads, blocks, keys, dim)

    def product(a, b):  # [.., group, rows, x] with [.., x, y] of the same block
        flat = a.reshape(batch, kv_heads, blocks, group * rows, -1)
        return torch.matmul(flat, b).reshape(batch, kv_heads, blocks, group, rows, -1)

    scale = dim ** -0.5
    q32, k32, v32 = queries(q), gathered(k), gathered(v)
    z = product(q32, k32.transpose(-1, -2).contiguous()).mul_(scale).masked_fill_(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = z.sub_(top).exp_()
    norm = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(norm > 0, norm, torch.ones_like(norm)))
    o = product(p, v32)
    out = tokens(o).to(q.dtype)
    if not c["grad"]:
        lse = ((top + norm.log()) / math.log(2)).transpose(2, 3).reshape(batch, heads, total)[:, :, :n]
        return out, lse.contiguous()
    do = queries(s["dout"])
    delta = (do * o).sum(-1, keepdim=True)
    flat = lambda x: x.reshape(batch, kv_heads, blocks, group * rows, -1)  # noqa: E731
    dv = torch.matmul(flat(p).transpose(-1, -2), flat(do))
    ds = product(do, v32.transpose(-1, -2).contiguous()).sub_(delta).mul_(p).mul_(scale)
    dq = tokens(product(ds, k32)).to(q.dtype)
    dk = torch.matmul(flat(ds).transpose(-1, -2), flat(q32))

    def scattered(g):
        full = torch.zeros((batch, kv_heads, n, dim), device=device)
        return full.index_add_(2, at.reshape(-1), g.reshape(batch, kv_heads, blocks * keys, dim)).to(q.dtype)

    return [out, dq, scattered(dk), scattered(dv)]


def _places(s):
    """Of every row of a packed tensor: its sequence, its position, and its place among the sequence's new tokens."""
    offsets, device = s["offsets"].long(), s["offsets"].device
    rows = torch.arange((s["k"] if "k" in s else s["q"]).shape[0], device=device)
    seq = torch.bucketize(rows, offsets[1:], right=True)
    place = rows - offsets[seq]
    new = offsets[1:] - offsets[:-1]
    return seq, s["lengths"].long()[seq] - new[seq] + place, place


def _append(s):
    if own:
        lib = _library()
        cache = lib.PagedCache(s["k_cache"], s["v_cache"])
        lib.append_cache(cache, s["k"], s["v"], s["table"], s["lengths"], s["offsets"])
        return s["k_cache"], s["v_cache"]
    seq, pos, _ = _places(s)
    page = s["case"]["page"]
    at = s["table"].long()[seq, pos // page]
    s["k_cache"][at, :, pos % page] = s["k"]
    s["v_cache"][at, :, pos % page] = s["v"]
    return s["k_cache"], s["v_cache"]


def _chunk(s):
    c, q = s["case"], s["q"]
    if own:
        lib = _library()
        cache = lib.PagedCache(s["k_cache"], s["v_cache"])
        return lib.chunk_attention(q, cache, s["table"], s["lengths"], s["offsets"], window=c["window"] or None,
                                   sinks=c["sinks"], frame=c["frame"], return_lse=True)
    batch, heads, kv_heads, dim = c["batch"], c["heads"], c["kv_heads"], c["dim"]
    most, keys, group, device = s["most"], s["keys"], c["heads"] // c["kv_heads"], q.device
    seq, pos, place = _places(s)
    table = s["table"].long()

    def gathered(cache):  # [batch, kv_heads, keys, dim]
        return cache[table.clamp_min(0)].transpose(1, 2).reshape(batch, kv_heads, keys, dim).float()

    q32 = torch.zeros((batch, most, heads, dim), device=device)
    q32[seq, place] = q.float()
    at = torch.full((batch, most), -1, device=device, dtype=torch.int64)
    at[seq, place] = pos
    key = torch.arange(keys, device=device)
    fq, fk = (at // c["frame"])[..., None], key // c["frame"]
    seen = (fk <= fq) & ((fq - fk < (c["window"] or keys + 1)) | (fk < c["sinks"])) & (at >= 0)[..., None]
    seen &= (key < s["lengths"].long()[:, None])[:, None] & table.ge(0).repeat_interleave(c["page"], 1)[:, None]
    seen = seen[:, None, None]  # [batch, 1, 1, most, keys]
    q32 = q32.reshape(batch, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * most, dim)
    z = torch.matmul(q32, gathered(s["k_cache"]).transpose(-1, -2).contiguous()).mul_(dim ** -0.5)
    z = z.reshape(batch, kv_heads, group, most, keys).masked_fill_(~seen, -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = z.sub_(top).exp_()
    norm = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(norm > 0, norm, torch.ones_like(norm)))
    o = torch.matmul(p.reshape(batch, kv_heads, group * most, keys), gathered(s["v_cache"]))
    o = o.reshape(batch, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
    lse = ((top + norm.log()) / math.log(2)).reshape(batch, kv_heads, group, most).permute(0, 3, 1, 2)
    return o[seq, place].to(q.dtype), lse.reshape(batch, most, heads)[seq, place]


# ---- in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    if case["op"] == "append":
        return None  # copies: there is nothing to compute
    if case["op"] == "window":
        return _exact_window(case, state)
    return _exact_chunk(case, state)


def _exact_rotary(case, state):
    """Every pair as a complex number times e^(i angle)."""
    pairs, angles, base = [], [], 0
    for axis, dims in enumerate(state["axes"]):
        for j in range(dims // 2):
            exponent = 2.0 * (base + j) / sum(state["axes"]) if case["joint"] else 2.0 * j / dims
            angles.append(state["positions"][..., axis].double() * case["theta"] ** -exponent)
        base += dims // 2
    for i in range(base):
        pairs.append((i, i + base) if case["halves"] else (2 * i, 2 * i + 1))
    angle = torch.stack(angles, -1)
    if angle.ndim == 3:
        angle = angle.unsqueeze(1)
    first, second = ([p[i] for p in pairs] for i in (0, 1))

    def turned(x, sign):
        wide = x.double()
        z = torch.complex(wide[..., first], wide[..., second]) * torch.polar(torch.ones_like(angle), sign * angle)
        wide[..., first], wide[..., second] = z.real, z.imag
        return wide

    out = [turned(state["q"], 1.0), turned(state["k"], 1.0)]
    if case["grad"]:
        out += [turned(state["dq"], -1.0), turned(state["dk"], -1.0)]
    return out


def _exact_mask(case, queries, keys):
    """queries, keys: positions"""
    fq, fk = queries[:, None] // case["frame"], keys[None] // case["frame"]
    mask = fk <= fq
    if case["window"]:
        mask &= (fq - fk < case["window"]) | (fk < case["sinks"])
    return mask


def _softmax64(z):
    """(weights, base-2 normaliser) of logits; rows of nothing have no weight."""
    lse = torch.logsumexp(z, -1)
    return torch.where(lse[..., None] > -math.inf, torch.exp(z - lse[..., None]), 0.0), lse / math.log(2)


def _exact_window(case, state):
    q, k, v = state["q"], state["k"], state["v"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
    if case["grad"]:
        dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v))
    scale, group = case["dim"] ** -0.5, case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        length = case["tokens"] if state["lengths"] is None else int(state["lengths"][b])
        for h in range(case["heads"]):
            kh, vh = k[b, h // group, :length].double(), v[b, h // group, :length].double()
            for start in range(0, length, 4096):
                stop = min(length, start + 4096)
                sink, low, _ = _span(case, start)
                end = min(length, _span(case, stop - 1)[2])
                keys = torch.cat([torch.arange(sink, device=q.device), torch.arange(low, end, device=q.device)])
                mask = _exact_mask(case, torch.arange(start, stop, device=q.device), keys)
                qh, kk, vv = q[b, h, start:stop].double(), kh[keys], vh[keys]
                p, lse[b, h, start:stop] = _softmax64((qh @ kk.T * scale).masked_fill(~mask, -math.inf))
                out[b, h, start:stop] = p @ vv
                if case["grad"]:
                    do = state["dout"][b, h, start:stop].double()
                    dp = do @ vv.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                    dq[b, h, start:stop] = ds @ kk
                    dk[b, h // group].index_add_(0, keys, ds.T @ qh)
                    dv[b, h // group].index_add_(0, keys, p.T @ do)
    return [out, dq, dk, dv] if case["grad"] else (out, lse)


def _exact_chunk(case, state):
    q, page, scale = state["q"], case["page"], case["dim"] ** -0.5
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
    table, row = state["table"].tolist(), 0
    for b, (n, length) in enumerate(zip(*_sequences(case))):
        sink, low, _ = _span(case, length - n)
        keys = torch.cat([torch.arange(sink, device=q.device), torch.arange(low, length, device=q.device)])
        at = torch.tensor(table[b], device=q.device)[keys // page].long()
        for h in range(case["kv_heads"]):
            kk, vv = state["k_cache"][at, h, keys % page].double(), state["v_cache"][at, h, keys % page].double()
            group = case["heads"] // case["kv_heads"]
            for g in range(h * group, (h + 1) * group):
                for start in range(0, n, 4096):
                    stop = min(n, start + 4096)
                    mask = _exact_mask(case, length - n + torch.arange(start, stop, device=q.device), keys)
                    z = q[row + start:row + stop, g].double() @ kk.T * scale
                    p, lse[row + start:row + stop, g] = _softmax64(z.masked_fill(~mask, -math.inf))
                    out[row + start:row + stop, g] = p @ vv
        row += n
    return out, lse

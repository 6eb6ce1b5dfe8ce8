"""Plain forms of the operators of drafted tokens, in 64 bits and one sequence at a time."""
import math
import random

import torch

from streaming_reference import attend


def make_tree(n, branch, seed=0):
    """parents of n tokens; branch 0: four lines side by side, 1: a chain, -1: anything, several roots too."""
    rng = random.Random("%s %s %s" % (n, branch, seed))
    tree = []
    for j in range(n):
        if branch < 0:
            tree.append(rng.randint(-1, j - 1) if rng.random() < 0.9 else rng.choice([-7, j, j + 5, 2 ** 31 - 1]))
        elif j == 0:
            tree.append(-1)
        elif branch == 0:
            tree.append(max(0, j - 4))
        else:
            tree.append(max(0, min(j - 1, (j - 1) // branch + (rng.randint(-1, 1) if branch > 1 else 0))))
    return tree


def lines(tree):
    """Of every token, the places on the line down to it, itself last."""
    out = []
    for j, parent in enumerate(tree):
        out.append((out[parent] if 0 <= parent < j else []) + [j])
    return out


def tree_tensors(tree, base):
    """What draft_tree says of one sequence: positions, near as unsigned numbers, above."""
    positions, near, above = [], [], []
    for j, line in enumerate(lines(tree)):
        block = j & ~63
        positions.append(base + len(line) - 1)
        near.append(sum(1 << (i - block) for i in line if i >= block))
        above.append(max([i for i in line if i < block], default=-1))
    return positions, near, above


def tree_mask(tree, base, length, window, sinks, frame):
    """bool [n, length]: what every new token sees of the cache's places (those below 0 do not exist)."""
    n = len(tree)
    of_line = torch.zeros((n, n), dtype=torch.bool)
    for i, parent in enumerate(tree):
        if 0 <= parent < i:
            of_line[i] = of_line[parent]
        of_line[i, i] = True
    position = base + of_line.sum(1) - 1
    there = max(0, -base)  # the first new token that has a place
    key_position = torch.cat([torch.arange(max(base, 0)), position[there:]])
    mask = torch.cat([torch.ones((n, max(base, 0)), dtype=torch.bool), of_line[:, there:]], 1) & (position >= 0)[:, None]
    if window is not None:
        p, t = position[:, None] // frame, key_position[None] // frame
        mask &= (p - t < window) | (t < sinks)
    return mask


def tree_attend(q, cache, table, length, tree, window=None, sinks=0, frame=1, scale=None):
    """(o [n, H, D], lse [n, H], spread) of one sequence's q [n, H, D]; table: its pages."""
    n, page = q.shape[0], cache.k.shape[2]
    mask = tree_mask(tree, length - n, length, window, sinks, frame).to(q.device)
    at = torch.arange(length, device=q.device)
    entry = table.long()[at // page]
    mask &= (entry >= 0) & (entry < cache.k.shape[0])
    entry = entry.clamp(0, cache.k.shape[0] - 1)
    k, v = cache.k[entry, :, at % page].transpose(0, 1), cache.v[entry, :, at % page].transpose(0, 1)
    o, lse, spread = attend(q.transpose(0, 1), k, v, mask, scale)
    return o.transpose(0, 1), lse.transpose(0, 1), spread.transpose(0, 1)


def _clean(x):
    return x if 0 < x < math.inf else 0.0


def verify(target, draft, tokens, tree, uniforms):
    """(path, next) of one sequence: lists of target and draft rows, of tokens, parents and uniforms; sums by math.fsum."""
    vocab = len(target[0])
    last, path = 0, [0]
    w, total = [_clean(x) for x in target[0]], 1.0
    for j in range(1, len(tree)):
        if tree[j] != last:
            continue
        x = tokens[j]
        there = 0 <= x < vocab
        q = 1.0 if draft is None else _clean(draft[last][x]) if there else 0.0
        if there and uniforms[j] * q * total < w[x]:
            last = j
            path.append(j)
            w, total = [_clean(y) for y in target[j]], 1.0
        elif draft is None:
            if there:
                total -= w[x]
                w[x] = 0.0
        else:
            less = [max(a - total * _clean(b), 0.0) for a, b in zip(w, draft[last])]
            rest = math.fsum(less)
            if rest > 0:
                w, total = less, rest
    border = uniforms[0] * math.fsum(w)
    running, found, some = 0.0, -1, -1
    for i, x in enumerate(w):
        if x > 0:
            running += x
            some = i
            if found < 0 and running > border:
                found = i
    return path, found if found >= 0 else some

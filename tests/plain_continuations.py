"""Plain forms, in 64 bits, of the operators that serve many continuations of one prompt."""
import math

import numpy as np
import torch

CUT = 2.0 ** -44                # weights below this share of the largest are not drawn


def kept_tokens(x, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """(ids of the tokens that the filters leave, in the order of ids; their weights relative to the largest logit's)."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    with np.errstate(over="ignore"):
        w = np.exp((x - x.max()) / float(np.float32(temperature)))
    order = np.array(sorted(np.flatnonzero(w >= CUT), key=lambda i: (-x[i], i)), dtype=np.int64)
    if top_k > 0:
        order = order[:top_k]
    if np.float32(top_p) < 1.0:
        sums = np.cumsum(w[order])
        reached = np.flatnonzero(sums >= float(np.float32(top_p)) * sums[-1])
        order = order[:max(1, reached[0] + 1)] if len(reached) else order
    kept = np.sort(order[w[order] >= min(float(np.float32(min_p)), 1.0)])
    return kept, w[kept]


def pick(x, temperature, u, top_k=0, top_p=1.0, min_p=0.0) -> int:
    live = np.where(np.isnan(x), -np.inf, x)
    if not temperature > 0 or not np.isfinite(live.max()):
        return int(np.argmax(live))
    kept, w = kept_tokens(x, temperature, top_k, top_p, min_p)
    sums = np.cumsum(w)
    return int(kept[min(np.searchsorted(sums, float(u) * sums[-1], side="right"), len(kept) - 1)])


def attend(q, k, v, table, positions, scale, window=None):
    """Row by row over the pages of its table. q [n, heads, d], k [pages, kv, page, d], v [pages, kv, d, page] (any float type, on
    the CPU), table [n][pages], positions [n] -> (out [n, heads * d], bound [n, heads * d]), both float64.

    The bound is what the kernel's roundings can add up to. A weight goes in rounded to bfloat16, half a step of 2^-8 of it; so
    does the result. Scores are float32: a dot product of d terms is off by d half steps of 2^-24 of its absolute sum, its scaling, the
    reference's subtraction and the exponential add eight of the score and of one (the references of parts up to 2^8 off one another
    another eight); what a score is off by counts twice, above and below the fraction. Sums over keys are float32, a chain of up
    to as many terms."""
    n, heads, d = q.shape
    kv, page = k.shape[1], k.shape[2]
    out, bound = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, d, dtype=torch.float64)
    for r in range(n):
        hi = int(positions[r])
        lo = max(0, hi + 1 - window) if window else 0
        if hi < 0:
            continue
        ids = list(range(lo, hi + 1))
        rows_k = torch.stack([k[table[r][i // page], :, i % page] for i in ids]).double()          # [keys, kv, d]
        rows_v = torch.stack([v[table[r][i // page], :, :, i % page] for i in ids]).double()
        for h in range(heads):
            qq, kk, vv = q[r, h].double(), rows_k[:, h // (heads // kv)], rows_v[:, h // (heads // kv)]
            s = kk @ qq * scale
            p = torch.softmax(s, 0)
            out[r, h] = p @ vv
            size = p @ vv.abs()
            off = 2.0 ** -24 * (d * float((kk.abs() @ qq.abs()).max()) * abs(scale) + 8 * float(s.abs().max()) + 16 + len(ids))
            bound[r, h] = (2.0 ** -8 * (size + out[r, h].abs()) + 2 * off * size) * 1.01
    return out.reshape(n, -1), bound.reshape(n, -1)


def tables(lengths, new, pages, page, width, n_tokens, leader=None, shared=None, stale=-7):
    """What step_tables leaves in arrays that held `stale`: a dict of lists."""
    n = len(lengths)
    length, new = [max(x, 0) for x in lengths], [max(x, 0) for x in new]
    need = [-(-(a + b) // page) for a, b in zip(length, new)]
    taken = [min(max(s, 0), m) for s, m in zip(shared, need)] if leader is not None else [0] * n
    at, own = 0, []
    for r in range(n):
        own.append([pages[at + i] if at + i < len(pages) else -1 for i in range(need[r] - taken[r])])
        at += need[r] - taken[r]

    def entry(r, j):
        if j >= need[r]:
            return -1
        for _ in range(n):
            if j >= taken[r]:
                return own[r][j - taken[r]] if j < need[r] else -1
            r = leader[r]
            if not 0 <= r < n:
                return -1
        return -1

    starts = [sum(new[:r]) for r in range(n)]
    tokens = [(r, length[r] + i) for r in range(n) for i in range(new[r])]
    kept = tokens[:n_tokens]
    pad = [stale] * (n_tokens - len(kept))
    slots = [entry(r, p // page) * page + p % page if entry(r, p // page) >= 0 else -1 for r, p in kept]
    one, more = [r for r in range(n) if new[r] == 1], [r for r in range(n) if new[r] > 1]
    return {"table": [[entry(r, j) for j in range(width)] for r in range(n)], "seg_start": starts,
            "positions": [p for _, p in kept] + pad, "row_of_token": [r for r, _ in kept] + pad, "slots": slots + pad,
            "lists": one + more + [stale] * (n - len(one) - len(more)), "counts": [len(tokens), at, len(one), len(more)]}

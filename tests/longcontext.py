"""Definitions in 64 bits of the operators on long shared caches (shared prefixes, key weights, eviction), and their inputs."""
import math

import torch

FP8 = torch.float8_e4m3fn


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def pages(g, lens, page, hk, d, dv, dtype, fp8=False, extra=3, poison=True):
    """(k_cache, v_cache, block_table): every sequence owns pages of a shuffled pool; rows no sequence owns are NaN."""
    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + extra
    order = torch.randperm(pool, generator=g).tolist()
    width = max(1, max(counts))
    table = torch.full((len(lens), width), order[-1], dtype=torch.int32)
    at = 0
    k = torch.full((pool, page, hk, d), math.nan if poison and not fp8 else 0.0)
    v = torch.full((pool, page, hk, dv), math.nan if poison and not fp8 else 0.0)
    for b, c in enumerate(counts):
        for j in range(c):
            p = order[at + j]
            n = min(page, lens[b] - j * page)
            k[p, :n] = torch.randn(n, hk, d, generator=g) * (2.0 if fp8 else 1.0)
            v[p, :n] = torch.randn(n, hk, dv, generator=g) * (2.0 if fp8 else 1.0)
            table[b, j] = p
        at += c
    t = FP8 if fp8 else dtype
    return k.to(t), v.to(t), table


def share(k, v, table, starts, prefixes, page):
    """Gives the sequences of each group the prefix of its first one: whole pages by table entry, the rest by value."""
    for g, p in enumerate(prefixes):
        first = starts[g]
        for b in range(first + 1, starts[g + 1]):
            whole, rest = divmod(p, page)
            table[b, :whole] = table[first, :whole]
            if rest:
                for pool in (k, v):
                    x = pool.view(torch.uint8) if pool.dtype == FP8 else pool
                    x[table[b, whole], :rest] = x[table[first, whole], :rest]


def rows(cache, table, n, page, descale=1.0):
    t = torch.arange(n)
    r = cache.float().flatten(0, 1)[table.long()[t // page] * page + t % page] if n else cache.float().flatten(0, 1)[:0]
    return r.double() * (descale if cache.dtype == FP8 else 1.0)


def visible(sq, n, mask_type, window):
    """[sq, n] truth table: key j of row i lies in the window around the diagonal of the mask type (0: none, 1: top left,
    2: bottom right); negative bounds are open."""
    i, j = torch.arange(sq)[:, None], torch.arange(n)[None, :]
    if mask_type == 0:
        return torch.ones(sq, n, dtype=torch.bool)
    left, right = window
    diagonal = i if mask_type == 1 else i + n - sq
    see = torch.ones(sq, n, dtype=torch.bool)
    if left >= 0:
        see &= j >= diagonal - left
    if right >= 0:
        see &= j <= diagonal + right
    return see


def scores(q, k, scale, cap=0.0, slope=None, mask_type=0, window=(-1, -1)):
    """[sq, n] scores of one head in 64 bits, -inf where unseen: q [sq, D], k [n, D]."""
    x = q.double() @ k.T * scale
    if cap > 0:
        x = cap * torch.tanh(x / cap)
    sq, n = x.shape
    if slope is not None:
        i, j = torch.arange(sq)[:, None], torch.arange(n)[None, :]
        if mask_type != 0 and window[0] < 0 and window[1] == 0:
            x = x + slope * j
        else:
            x = x - slope * ((i if mask_type == 1 else i + n - sq) - j).abs()
    return torch.where(visible(sq, n, mask_type, window), x, torch.tensor(-math.inf, dtype=torch.float64))


def attention(q, k, v, scale, **kw):
    """(o [sq, Dv], lse [sq]) of one head in 64 bits; a row that sees nothing gives zeros and -inf."""
    x = scores(q, k, scale, **kw)
    some = torch.isfinite(x).any(1)
    o, lse = torch.zeros(x.shape[0], v.shape[1], dtype=torch.float64), torch.full((x.shape[0],), -math.inf, dtype=torch.float64)
    if some.any():
        seen = torch.isfinite(x[some])
        p = torch.softmax(x[some], 1)
        # a key no row sees does not count, whatever it holds
        o[some] = torch.where(seen.any(0)[None, :], p, 0.0) @ torch.where(seen.any(0)[:, None], v, 0.0)
        lse[some] = torch.logsumexp(x[some], 1)
    return o, lse


def decode(q, kc, vc, lens, table, scale, starts=None, kd=1.0, vd=1.0, slopes=None, **kw):
    """q [B, sq, Hq, D] (or packed [T, Hq, D] with starts) -> (o like q, lse [B, Hq, sq] or [Hq, T])."""
    page, hk = kc.shape[1], kc.shape[2]
    hq, dv = q.shape[-2], vc.shape[3]
    o = torch.zeros(*q.shape[:-1], dv, dtype=torch.float64)
    lse = torch.full((hq, q.shape[0]) if starts is not None else (q.shape[0], hq, q.shape[1]), -math.inf, dtype=torch.float64)
    for b, n in enumerate(lens):
        k, v = rows(kc, table[b], n, page, kd), rows(vc, table[b], n, page, vd)
        for h in range(hq):
            s = None if slopes is None else float(slopes[h] if slopes.dim() == 1 else slopes[b, h])
            qb = q[starts[b]:starts[b + 1], h] if starts is not None else q[b, :, h]
            ob, lb = attention(qb, k[:, h * hk // hq], v[:, h * hk // hq], scale, slope=s, **kw)
            if starts is not None:
                o[starts[b]:starts[b + 1], h], lse[h, starts[b]:starts[b + 1]] = ob, lb
            else:
                o[b, :, h], lse[b, h] = ob, lb
    return o, lse


def key_weights(q, keys, lse, cols, scale, starts=None, before=None, slopes=None, **kw):
    """keys[b]: [n, Hk, D] in 64 bits; the definition of fmha_key_weights, [B, Hk, cols]."""
    hq, hk = q.shape[-2], keys[0].shape[1]
    out = torch.zeros(len(keys), hk, cols, dtype=torch.float64)
    for b, k in enumerate(keys):
        n = min(k.shape[0], cols)
        for h in range(hq):
            s = None if slopes is None else float(slopes[h] if slopes.dim() == 1 else slopes[b, h])
            qb = q[starts[b]:starts[b + 1], h] if starts is not None else q[b, :, h]
            lb = (lse[h, starts[b]:starts[b + 1]] if starts is not None else lse[b, h]).double()
            x = scores(qb, k[:, h * hk // hq], scale, slope=s, **kw)
            e = torch.where(torch.isfinite(lb)[:, None] & torch.isfinite(x), torch.exp(x - lb[:, None]), 0.0)
            out[b, h * hk // hq, :n] += e.sum(0)[:n]
        if before is not None:
            out[b, :, :n] += before[b, :, :n].double()
    return out


def evict(weights, lens, budget, recent, sinks):
    """Kept positions [B][Hk] -> list, by the definition of fmha_cache_evict."""
    out = []
    for b, n in enumerate(lens):
        per_head = []
        for h in range(weights.shape[1]):
            w = [float(x) for x in weights[b, h, :n]] + [0.0] * max(0, n - weights.shape[2])
            w = [-math.inf if math.isnan(x) else x for x in w]
            if n <= budget:
                per_head.append(list(range(n)))
                continue
            middle = sorted(range(sinks, n - recent), key=lambda t: (-w[t], t))[:budget - sinks - recent]
            per_head.append(sorted(set(middle) | set(range(sinks)) | set(range(n - recent, n))))
        out.append(per_head)
    return out

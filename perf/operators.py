"""Workloads of the shared-prefix and cache-eviction operators of ``flash_ck.ops.fmha``.

    fmha_decode_shared_prefix   decode attention of a batch whose sequences share prefixes, each prefix read once
    fmha_key_weights            attention weight each cached key has received, summed over query rows and grouped heads
    fmha_cache_evict            keep the heaviest keys of every (sequence, KV head) and move them to new pages

``run`` computes an operator with elementary torch operations in 32 bits, or, with ``own`` set, through the library.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_FP8 = torch.float8_e4m3fn
_K_DESCALE, _V_DESCALE = 0.5, 0.25


# ---- cases ---------------------------------------------------------------------------------------------------------------
#
# shared   batch sequences in `groups` groups; a group shares up to `prefix` tokens, a sequence has up to `own` more;
#          sq query tokens each (causal among themselves when there are several)
# weights  batch sequences of up to `keys` keys (at least half of them when `full` is set: exactly), sq query rows
# evict    batch sequences of up to `keys` keys, `budget` of them kept per KV head
# `lens` seeds the lengths, so that the work is a property of the case and not of the inputs' seed.

def listed():
    return [
        # a few chats behind one short system prompt: latency
        dict(name="shared_small", op="shared", batch=4, groups=1, sq=1, hq=32, hk=8, d=128, page=16, type="bf16", kv8=False,
             prefix=512, own=64, cap=0.0, lens=1),
        # a batch of requests behind one long instruction, each with its own history
        dict(name="shared_batch", op="shared", batch=32, groups=1, sq=1, hq=32, hk=8, d=128, page=128, type="bf16", kv8=False,
             prefix=4096, own=1024, cap=0.0, lens=2),
        # many questions about one long document: the prefix product no longer hides behind the reads
        dict(name="shared_document", op="shared", batch=64, groups=1, sq=1, hq=64, hk=8, d=128, page=128, type="bf16", kv8=False,
             prefix=32768, own=512, cap=0.0, lens=3),
        # four drafted tokens a step over a quantised cache, three prompts in one batch, ragged lengths
        dict(name="shared_drafts_fp8", op="shared", batch=24, groups=3, sq=4, hq=16, hk=4, d=64, page=64, type="fp16", kv8=True,
             prefix=3001, own=333, cap=0.0, lens=4),
        # wide heads, pages that end inside a tile, capped logits
        dict(name="shared_wide", op="shared", batch=12, groups=2, sq=1, hq=16, hk=4, d=256, page=48, type="bf16", kv8=False,
             prefix=2000, own=200, cap=30.0, lens=5),
        # weights of one step of two short sequences: latency
        dict(name="weights_small", op="weights", batch=2, sq=1, hq=32, hk=8, d=128, page=16, type="fp16", kv8=False, keys=300,
             full=False, lens=6),
        # weights of one decode step of a ragged long-context batch
        dict(name="weights_step", op="weights", batch=16, sq=1, hq=64, hk=8, d=128, page=128, type="bf16", kv8=False, keys=32768,
             full=False, lens=7),
        # the last queries of a prompt as the observation window
        dict(name="weights_window", op="weights", batch=4, sq=33, hq=32, hk=8, d=128, page=128, type="bf16", kv8=False, keys=8191,
             full=True, lens=8),
        # every query of a prompt
        dict(name="weights_prompt", op="weights", batch=1, sq=8192, hq=32, hk=8, d=128, page=128, type="bf16", kv8=False,
             keys=8192, full=True, lens=9),
        # two short sequences brought back to a small budget: latency
        dict(name="evict_small", op="evict", batch=2, hk=8, d=128, page=16, type="fp16", kv8=False, keys=600, budget=256,
             recent=32, sinks=4, lens=10),
        # a serving batch brought back to a quarter of its cache
        dict(name="evict_batch", op="evict", batch=16, hk=8, d=128, page=128, type="bf16", kv8=False, keys=16384, budget=4096,
             recent=256, sinks=4, lens=11),
        # one very long sequence
        dict(name="evict_long", op="evict", batch=1, hk=8, d=64, page=64, type="bf16", kv8=False, keys=131072, budget=8192,
             recent=1024, sinks=16, lens=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of these ranges: the same operators over any of their types, head layouts, lengths and page sizes."""
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = tuple(max(a, b) for a, b in zip(most.get(c["op"], (0, 0)), (w["bytes"], w["flops"])))
    while True:
        hq, hk = rng.choice([(32, 8), (64, 8), (16, 4), (32, 4), (28, 4), (8, 8), (16, 16), (12, 2), (8, 1)])
        c = dict(op=rng.choice(["shared", "weights", "evict"]), hk=hk, d=rng.choice([64, 128, 128, 128, 256]),
                 page=rng.choice([1, 16, 48, 64, 128, 128]), type=rng.choice(["bf16", "fp16"]), kv8=rng.random() < 0.25,
                 lens=rng.randrange(1 << 30))
        if c["op"] == "shared":
            batch = _log_int(rng, 1, 96)
            c.update(batch=batch, groups=min(batch, rng.choice([1, 1, 1, 2, 4])), sq=rng.choice([1, 1, 1, 2, 5]), hq=hq,
                     prefix=_log_int(rng, 1, 32768), own=_log_int(rng, 1, 2048), cap=rng.choice([0.0, 0.0, 0.0, 30.0]))
        elif c["op"] == "weights":
            keys = _log_int(rng, 1, 32768)
            c.update(batch=_log_int(rng, 1, 32), sq=min(keys, rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 8192)])),
                     hq=hq, keys=keys, full=rng.random() < 0.3)
        else:
            keys = _log_int(rng, 1, 131072)
            budget = _log_int(rng, 1, max(1, min(keys, 16384)))
            recent = rng.randint(0, budget // 2)
            c.update(batch=_log_int(rng, 1, 32), keys=keys, budget=budget, recent=recent,
                     sinks=rng.randint(0, min(16, budget - recent)))
        if c["page"] == 1 and max(c.get("keys", 0), c.get("prefix", 0)) > 4096:
            continue  # pages of one token come with short caches
        w = work(c)
        if w["bytes"] <= most[c["op"]][0] and w["flops"] <= most[c["op"]][1]:
            return c


# ---- lengths -------------------------------------------------------------------------------------------------------------

def _shared_lengths(case):
    """(sequence counts of the groups, prefix lengths of the groups, key counts of the sequences)"""
    r = random.Random(case["lens"])
    n, g = case["batch"], case["groups"]
    cuts = [0] + sorted(r.sample(range(1, n), g - 1)) + [n]
    sizes = [b - a for a, b in zip(cuts, cuts[1:])]
    prefix = [case["prefix"]] + [r.randint(0, case["prefix"]) for _ in range(g - 1)]
    lens = [prefix[k] + r.randint(0, case["own"]) for k, s in enumerate(sizes) for _ in range(s)]
    return sizes, prefix, lens


def _lengths(case):
    r = random.Random(case["lens"])
    if case.get("full"):
        return [case["keys"]] * case["batch"]
    low = min(case["keys"], max(case.get("sq", 1), case["keys"] // 4))
    return [case["keys"]] + [r.randint(low, case["keys"]) for _ in range(case["batch"] - 1)]


def work(case):
    """What a pass cannot do without: every input read once, every output written once."""
    hk, d = case["hk"], case["d"]
    e = 1 if case["kv8"] else 2
    if case["op"] == "shared":
        sizes, prefix, lens = _shared_lengths(case)
        n, sq, hq = case["batch"], case["sq"], case["hq"]
        own_tokens = sum(l - p for l, p in zip(lens, [p for p, s in zip(prefix, sizes) for _ in range(s)]))
        pairs = sum(max(0, l - i) for l in lens for i in range(sq))
        return {"bytes": 2 * n * sq * hq * d * 2 + n * sq * hq * 4 + (sum(prefix) + own_tokens) * hk * 2 * d * e,
                "flops": 4 * hq * d * pairs}
    lens = _lengths(case)
    if case["op"] == "weights":
        n, sq, hq = case["batch"], case["sq"], case["hq"]
        pairs = sum(sum(max(0, l - i) for i in range(sq)) for l in lens)
        return {"bytes": n * sq * hq * (d * 2 + 4) + sum(lens) * hk * d * e + 2 * n * hk * case["keys"] * 4, "flops": 2 * hq * d * pairs}
    kept = sum(min(l, case["budget"]) for l in lens)
    return {"bytes": sum(lens) * hk * 4 + kept * hk * 4 * d * e + case["batch"] * hk * (case["keys"] + case["budget"]) * 4,
            "flops": sum(lens) * hk}


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device=g.device, dtype=torch.float32).to(dtype)


def _pool(g, case, pages):
    """A page pool of keys or values; the stored values of a quantised one have twice the spread."""
    if case["kv8"]:
        return _normal(g, pages, case["page"], case["hk"], case["d"], dtype=torch.float32).mul_(2.0).to(_FP8)
    return _normal(g, pages, case["page"], case["hk"], case["d"], dtype=_TYPES[case["type"]])


def _bytes_view(t):
    return t.view(torch.uint8) if t.dtype == _FP8 else t


def _int32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    shuffle = random.Random(seed)
    page, t = case["page"], _TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "shared":
        sizes, prefix, lens = _shared_lengths(case)
        # whole pages of a prefix exist once; its last, partial page is repeated in front of every sequence's own tokens
        rows, pages = [], 0
        for size, p in zip(sizes, prefix):
            common = list(range(pages, pages + p // page))
            pages += len(common)
            for _ in range(size):
                own_pages = -(-lens[len(rows)] // page) - len(common)
                rows.append(common + list(range(pages, pages + own_pages)))
                pages += own_pages
        order = list(range(pages + 1))
        shuffle.shuffle(order)
        width = max(1, max(len(r) for r in rows))
        table = [[order[p] for p in r] + [0] * (width - len(r)) for r in rows]
        s["k"], s["v"] = _pool(g, case, pages + 1), _pool(g, case, pages + 1)
        first = 0
        for size, p in zip(sizes, prefix):
            rest, at = p % page, p // page
            if rest and size > 1:
                others = torch.tensor([table[b][at] for b in range(first + 1, first + size)], device=device)
                for pool in (s["k"], s["v"]):
                    v = _bytes_view(pool)
                    v[others, :rest] = v[table[first][at], :rest]
            first += size
        s["q"] = _normal(g, case["batch"], case["sq"], case["hq"], case["d"], dtype=t)
        s["lens"], s["table"], s["prefix"] = _int32(lens, device), _int32(table, device), _int32(prefix, device)
        starts = [0]
        for size in sizes:
            starts.append(starts[-1] + size)
        s["groups"] = _int32(starts, device)
        s["lse"] = torch.empty(case["batch"], case["hq"], case["sq"], dtype=torch.float32, device=device)
        s["host"] = dict(sizes=sizes, prefix=prefix, lens=lens)
        return s
    lens = _lengths(case)
    counts = [-(-l // page) for l in lens]
    order = list(range(sum(counts) + 1))
    shuffle.shuffle(order)
    width = max(counts)
    table, at = [], 0
    for c in counts:
        table.append(order[at:at + c] + [0] * (width - c))
        at += c
    s["lens"], s["table"] = _int32(lens, device), _int32(table, device)
    s["host"] = dict(lens=lens)
    s["k"] = _pool(g, case, len(order))
    n, hk, keys = case["batch"], case["hk"], case["keys"]
    if case["op"] == "weights":
        s["q"] = _normal(g, n, case["sq"], case["hq"], case["d"], dtype=t)
        # what earlier steps left: of the size that this step adds
        s["before"] = torch.rand(n, hk, keys, generator=g, device=device) * (case["sq"] * case["hq"] / hk / keys)
        s["lse"] = torch.empty(n, case["hq"], case["sq"], device=device)
        for b in range(n):
            for heads, x in _plain_scores(s, b):
                s["lse"][b, heads] = torch.logsumexp(x, dim=-1).flatten(0, 1)
        return s
    s["v"] = _pool(g, case, len(order))
    # accumulated weights have a heavy tail, and many keys have received nothing
    w = torch.exp(2.0 * torch.randn(n, hk, keys, generator=g, device=device))
    s["weights"] = torch.where(torch.rand(n, hk, keys, generator=g, device=device) < 0.3, torch.zeros_like(w), w)
    kept_pages = -(-case["budget"] // page)
    s["new_k"] = torch.zeros(n * kept_pages, page, hk, case["d"], dtype=t, device=device)
    if case["kv8"]:
        s["new_k"] = s["new_k"].to(_FP8)
    s["new_v"] = s["new_k"].clone()
    order = list(range(n * kept_pages))
    shuffle.shuffle(order)
    s["new_table"] = _int32([order[b * kept_pages:(b + 1) * kept_pages] for b in range(n)], device)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------

def _plain_rows(pool, table_row, first, last, page, descale):
    """Tokens first..last-1 of a sequence as fp32 [tokens, heads, head dim]."""
    t = torch.arange(first, last, device=pool.device)
    ids = table_row.long()[t // page] * page + t % page
    rows = _bytes_view(pool).flatten(0, 1)[ids]
    return rows.view(_FP8).float() * descale if pool.dtype == _FP8 else rows.float()


def _plain_cap(x, cap):
    return cap * torch.tanh(x / cap) if cap > 0 else x


def _plain_scores(s, b):
    """Pairs (query heads, scores [KV heads, grouped heads, sq, keys] with unseen keys at -inf) of sequence b, as many KV
    heads at a time as fit 2^28 scores."""
    case, n = s["case"], s["host"]["lens"][b]
    k = _plain_rows(s["k"], s["table"][b], 0, n, case["page"], _K_DESCALE).permute(1, 2, 0)
    group, sq, d = case["hq"] // case["hk"], case["sq"], case["d"]
    q = s["q"][b].float().transpose(0, 1).reshape(case["hk"], group * sq, d)
    seen = torch.arange(n, device=k.device)[None, :] <= torch.arange(n - sq, n, device=k.device)[:, None]
    step = max(1, min(case["hk"], (1 << 28) // (group * sq * n)))
    for h in range(0, case["hk"], step):
        x = torch.matmul(q[h:h + step], k[h:h + step]) / math.sqrt(d)
        x = x.view(-1, group, sq, n).masked_fill_(~seen, -math.inf)
        yield slice(h * group, (h + x.shape[0]) * group), x


def _plain_shared(s):
    case, host = s["case"], s["host"]
    page, sq, hq, hk, d = case["page"], case["sq"], case["hq"], case["hk"], case["d"]
    group, scale, device = hq // hk, 1.0 / math.sqrt(case["d"]), s["q"].device
    out = torch.empty_like(s["q"])
    first = 0
    for size, p in zip(host["sizes"], host["prefix"]):
        seqs = slice(first, first + size)
        lens = s["lens"][seqs].long()
        own_max = max(host["lens"][seqs]) - p
        # rows [hk, size, sq * group, d]
        q = s["q"][seqs].float().view(size, sq, hk, group, d).permute(2, 0, 1, 3, 4).reshape(hk, size, sq * group, d)
        last = (lens[:, None] - sq + 1 + torch.arange(sq, device=device)).repeat_interleave(group, dim=1)  # keys a row sees
        # the prefix once for the whole group, the own tokens padded to the longest
        kp = _plain_rows(s["k"], s["table"][first], 0, p, page, _K_DESCALE).transpose(0, 1)
        vp = _plain_rows(s["v"], s["table"][first], 0, p, page, _V_DESCALE).transpose(0, 1)
        t = p + torch.arange(own_max, device=device)
        at = torch.clamp(t // page, max=s["table"].shape[1] - 1)
        ids = s["table"][seqs].long()[:, at] * page + t % page
        ko, vo = [_bytes_view(x).flatten(0, 1)[ids] for x in (s["k"], s["v"])]
        if case["kv8"]:
            ko, vo = ko.view(_FP8).float() * _K_DESCALE, vo.view(_FP8).float() * _V_DESCALE
        ko, vo = ko.float().permute(2, 0, 1, 3), vo.float().permute(2, 0, 1, 3)
        xp = torch.matmul(q.reshape(hk, size * sq * group, d), kp.transpose(1, 2)).view(hk, size, sq * group, p)
        xo = torch.matmul(q, ko.transpose(2, 3))
        x = torch.cat([xp, xo], dim=-1).mul_(scale)
        x = _plain_cap(x, case["cap"])
        x.masked_fill_(torch.arange(p + own_max, device=device) >= last[..., None], -math.inf)
        m = x.max(dim=-1, keepdim=True).values if x.shape[-1] else x.new_full((*x.shape[:-1], 1), -math.inf)
        e = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        total = e.sum(dim=-1, keepdim=True)
        o = torch.matmul(e[..., :p].reshape(hk, size * sq * group, p), vp).view(hk, size, sq * group, d) + torch.matmul(e[..., p:], vo)
        o = torch.where(total > 0, o / total, torch.zeros_like(o))
        out[seqs] = o.view(hk, size, sq, group, d).permute(1, 2, 0, 3, 4).reshape(size, sq, hq, d).to(out.dtype)
        lse = (m + torch.log(total))[..., 0].view(hk, size, sq, group)
        s["lse"][seqs] = lse.permute(1, 0, 3, 2).reshape(size, hq, sq)
        first += size
    return out, s["lse"]


def _plain_weights(s):
    out = torch.zeros_like(s["before"])
    group = s["case"]["hq"] // s["case"]["hk"]
    for b, n in enumerate(s["host"]["lens"]):
        for heads, x in _plain_scores(s, b):
            p = torch.exp(x - s["lse"][b, heads].view(-1, group, x.shape[2], 1))
            h = slice(heads.start // group, heads.stop // group)
            out[b, h, :n] = s["before"][b, h, :n] + p.sum(dim=(1, 2))
    return out


def _plain_evict(s):
    case = s["case"]
    n, hk, keys, budget, page = case["batch"], case["hk"], case["keys"], case["budget"], case["page"]
    device = s["weights"].device
    t = torch.arange(keys, device=device)
    lens = s["lens"].long()[:, None, None]
    keep_all = (t < case["sinks"]) | (t >= lens - case["recent"])
    w = torch.where(keep_all, math.inf, s["weights"])
    w = torch.where(t < lens, w, -math.inf).expand(n, hk, keys)
    first = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    if keys < budget:
        first = torch.nn.functional.pad(first, (0, budget - keys), value=keys)
    there = torch.arange(budget, device=device) < torch.clamp(lens, max=budget)
    kept = torch.sort(torch.where(there, first, 1 << 40), dim=-1).values
    kept = torch.where(there, kept, -1)
    at = torch.clamp(kept, min=0)
    new_weights = torch.zeros_like(s["weights"])
    new_weights[..., :min(budget, keys)] = torch.where(there, torch.gather(s["weights"], 2, torch.clamp(at, max=keys - 1)), 0.0)[..., :keys]
    pages = torch.gather(s["table"].long()[:, None, :].expand(n, hk, -1), 2, at // page)
    source = (pages * page + at % page) * hk + torch.arange(hk, device=device)[:, None]
    slot = torch.arange(budget, device=device)
    target = (s["new_table"].long()[:, slot // page] * page + slot % page)[:, None, :] * hk + torch.arange(hk, device=device)[:, None]
    source, target = source[there.expand_as(source)], target[there.expand_as(target)]
    for old, new in ((s["k"], s["new_k"]), (s["v"], s["new_v"])):
        _bytes_view(new).view(-1, case["d"])[target] = _bytes_view(old).view(-1, case["d"])[source]
    return kept.to(torch.int32), torch.clamp(s["lens"], max=budget), new_weights


def run(state):
    s, case = state, state["case"]
    scales = dict(k_descale=_K_DESCALE, v_descale=_V_DESCALE) if case["kv8"] else {}
    if case["op"] == "shared":
        if not own:
            return _plain_shared(s)
        from flash_ck.ops import fmha
        mask = dict(mask_type=fmha.MASK_BOTTOM_RIGHT, window=(-1, 0)) if case["sq"] > 1 else {}
        o = fmha.fmha_decode_shared_prefix(s["q"], s["k"], s["v"], s["lens"], s["table"], s["prefix"], cu_groups=s["groups"],
                                           max_group_size=max(s["host"]["sizes"]), max_prefix_len=max(s["host"]["prefix"]),
                                           max_seqlen_k=max(s["host"]["lens"]), logits_soft_cap=case["cap"], lse=s["lse"],
                                           **scales, **mask)
        return o, s["lse"]
    if case["op"] == "weights":
        if not own:
            return _plain_weights(s)
        from flash_ck.ops import fmha
        return fmha.fmha_key_weights(s["q"], s["k"], s["lse"], s["lens"], s["table"], weights=s["before"],
                                     mask_type=fmha.MASK_BOTTOM_RIGHT, window=(-1, 0),
                                     k_descale=_K_DESCALE if case["kv8"] else 1.0)
    if own:
        from flash_ck.ops import fmha
        lens, kept, weights = fmha.fmha_cache_evict(s["k"], s["v"], s["weights"], s["lens"], s["table"], s["new_table"],
                                                    budget=case["budget"], recent=case["recent"], sinks=case["sinks"],
                                                    new_k_cache=s["new_k"], new_v_cache=s["new_v"])
    else:
        kept, lens, weights = _plain_evict(s)
    k, v = s["new_k"], s["new_v"]
    return dict(kept=kept, lens=lens, weights=weights, k=k.float() if case["kv8"] else k, v=v.float() if case["kv8"] else v)


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------------

def _tokens64(pool, table, length, page, descale):
    pages = [pool[p] for p in table[:-(-length // page)]]
    if not pages:
        return torch.zeros(0, *pool.shape[2:], dtype=torch.float64, device=pool.device)
    rows = torch.cat(pages)[:length]
    return rows.float().double() * (descale if pool.dtype == _FP8 else 1.0)


def exact(case, seed):
    s = prepare(case, seed)
    lens, table = s["lens"].tolist(), s["table"].tolist()
    hk, d, page = case["hk"], case["d"], case["page"]
    if case["op"] == "evict":
        return _exact_evict(case, s, lens, table)
    ratio, sq, dev = case["hq"] // hk, case["sq"], s["q"].device
    if case["op"] == "shared":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
        lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device=dev)
    else:
        out = torch.zeros(s["before"].shape, dtype=torch.float64, device=dev)
    for b, length in enumerate(lens):
        k = _tokens64(s["k"], table[b], length, page, _K_DESCALE)
        v = _tokens64(s["v"], table[b], length, page, _V_DESCALE) if case["op"] == "shared" else None
        for h in range(case["hq"]):
            z = s["q"][b, :, h].double() @ k[:, h // ratio].T * d ** -0.5
            if case.get("cap"):
                z = case["cap"] * torch.tanh(z / case["cap"])
            hidden = torch.ones(sq, length, dtype=torch.bool, device=dev).triu(length - sq + 1)
            z[hidden] = -math.inf
            if case["op"] == "weights":
                out[b, h // ratio, :length] += torch.exp(z - s["lse"][b, h].double()[:, None]).sum(0)
                continue
            rows = (~hidden).any(1)
            if bool(rows.any()):
                lse[b, h, rows] = torch.logsumexp(z[rows], 1)
                out[b, rows, h] = torch.softmax(z[rows], 1) @ v[:, h // ratio]
        if case["op"] == "weights":
            out[b, :, :length] += s["before"][b, :, :length].double()
    return (out, lse) if case["op"] == "shared" else out


def _exact_evict(case, s, lens, table):
    hk, page, budget = case["hk"], case["page"], case["budget"]
    weights = s["weights"].cpu().double()
    kept = torch.full((case["batch"], hk, budget), -1, dtype=torch.int32)
    new_weights = torch.zeros_like(weights)
    new_table = s["new_table"].tolist()
    k_old, v_old = [(x.float() if x.dtype == _FP8 else x).cpu() for x in (s["k"], s["v"])]
    k_new, v_new = [(x.float() if x.dtype == _FP8 else x).cpu().double() for x in (s["new_k"], s["new_v"])]
    for b, length in enumerate(lens):
        for h in range(hk):
            w = weights[b, h, :length]
            if length <= budget:
                chosen = list(range(length))
            else:
                middle = range(case["sinks"], length - case["recent"])
                values = w.tolist()
                best = sorted(middle, key=lambda t: -values[t])[:budget - case["sinks"] - case["recent"]]
                chosen = sorted(best + list(range(case["sinks"])) + list(range(length - case["recent"], length)))
            at = torch.tensor(chosen, dtype=torch.long)
            slots = torch.arange(len(chosen))
            kept[b, h, :len(chosen)] = at.int()
            new_weights[b, h, :len(chosen)] = w[at]
            source, target = torch.tensor(table[b])[at // page], torch.tensor(new_table[b])[slots // page]
            k_new[target, slots % page, h] = k_old[source, at % page, h].double()
            v_new[target, slots % page, h] = v_old[source, at % page, h].double()
    return dict(kept=kept, lens=torch.tensor([min(n, budget) for n in lens], dtype=torch.int32), weights=new_weights, k=k_new, v=v_new)

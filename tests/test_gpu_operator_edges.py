"""GPU: the corners of the operators on long shared caches, against their definitions in 64 bits: keys whose scores are not
finite, rows that add nothing, caches with more keys than the weights have columns.

Tolerances are those of test_gpu_key_weights (REL) and test_gpu_shared_prefix (U), derived there."""
import contextlib
import math

import pytest
import torch

import longcontext as lc
from flashck_amd.utils import flags
from helpers import dev

pytestmark = pytest.mark.gpu
REL = 2.5e-5
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _i32(x):
    return dev(torch.tensor(x, dtype=torch.int32))


def _weights_case(seed, lens, sq, hq, hk, d, dtype, page, minus_inf=(), **kw):
    """Inputs of fmha_key_weights; the keys `minus_inf` of every sequence score -inf for every row."""
    g = torch.Generator().manual_seed(seed)
    kc, _, table = lc.pages(g, lens, page, hk, d, d, dtype)
    q = lc.randn(g, len(lens), sq, hq, d, dtype=dtype)
    q[..., 0] = q[..., 0].abs() + 0.5
    for b, n in enumerate(lens):
        for t in minus_inf:
            if t < n:
                kc[table[b, t // page], t % page, :, 0] = -math.inf
    keys = [lc.rows(kc, table[b], n, page) for b, n in enumerate(lens)]
    _, lse = lc.decode(q, kc, torch.zeros_like(kc), lens, table, d ** -0.5, **kw)
    return dict(q=q, kc=kc, table=table, lens=lens, keys=keys, lse=lse.float())


def _weights(fmha, c, **kw):
    return fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(c["lens"]), dev(c["table"]), **kw).cpu()


def _close(got, want, what=""):
    assert got.shape == want.shape and torch.isfinite(got).all(), f"{what}: not finite"
    err = ((got.double() - want).abs() - REL * want).max().item()
    assert err <= 1e-9, f"{what}: off by {err:.3e} beyond the relative bound"


# (sq, hq, hk, d): one and two 16-row blocks in registers, partly and wholly filled; rows in LDS; rows that are streamed
ROWS = [(1, 4, 1, 64), (1, 16, 1, 128), (2, 8, 2, 256), (5, 4, 1, 128), (33, 1, 1, 64), (33, 4, 2, 128), (64, 1, 1, 128),
        (40, 1, 1, 256), (290, 2, 1, 128), (290, 2, 1, 64)]


@pytest.mark.parametrize("mask", [dict(), dict(mask_type=2, window=(-1, 0))])
@pytest.mark.parametrize("sq,hq,hk,d", ROWS)
def test_a_visible_key_of_score_minus_infinity_receives_nothing(fmha, sq, hq, hk, d, mask):
    lens = [sq + 70, 63] if sq < 63 else [sq + 70]
    c = _weights_case(1, lens, sq, hq, hk, d, torch.float16, 64, minus_inf=(5, 40, 62), **mask)
    want = lc.key_weights(c["q"], c["keys"], c["lse"], max(lens), d ** -0.5, **mask)
    assert not want[:, :, 5].any() and not want[:, :, 40].any() and want[:, :, 6].any()
    _close(_weights(fmha, c, max_seqlen_k=max(lens), **mask), want)


@pytest.mark.parametrize("mask", [dict(), dict(mask_type=2, window=(-1, 0))])
@pytest.mark.parametrize("sq,hq,hk,d", ROWS)
def test_rows_whose_lse_is_minus_infinity_add_nothing_whatever_they_hold(fmha, sq, hq, hk, d, mask):
    # padded rows: queries and scores of theirs may be anything
    c = _weights_case(2, [sq + 70], sq, hq, hk, d, torch.bfloat16, 64, **mask)
    g = torch.Generator().manual_seed(3)
    none = torch.rand(1, hq, sq, generator=g) < 0.1
    none[0, hq - 1, sq - 1] = True
    c["lse"][none] = -math.inf
    want = lc.key_weights(c["q"], c["keys"], c["lse"], sq + 70, d ** -0.5, **mask)
    c["q"][none.permute(0, 2, 1)] = math.nan
    _close(_weights(fmha, c, max_seqlen_k=sq + 70, **mask), want)


@pytest.mark.parametrize("cols", [1, 40, 64, 65, 130, 199])
@pytest.mark.parametrize("batch,sq,hq,hk,d", [(64, 1, 8, 8, 64), (64, 5, 32, 8, 64), (1, 33, 4, 2, 128), (2, 33, 1, 1, 64), (1, 290, 2, 1, 64)])
def test_fewer_columns_than_keys(fmha, batch, sq, hq, hk, d, cols):
    # the first two: enough sequences that a wave walks eight tiles.  No tile without a column may be asked for.
    few = min(4, batch)   # sequences 4.. are copies of the first four
    lens = [200 - 7 * b for b in range(few)]
    g = torch.Generator().manual_seed(4)
    kc, _, table = lc.pages(g, lens, 64, hk, d, d, torch.bfloat16)
    q, lse = lc.randn(g, few, sq, hq, d, dtype=torch.bfloat16), torch.full((few, hq, sq), 5.0)
    before = torch.rand(few, hk, cols, generator=g)
    want = lc.key_weights(q, [lc.rows(kc, table[b], n, 64) for b, n in enumerate(lens)], lse, cols, d ** -0.5, before=before)
    copies = lambda x: x.repeat(-(-batch // few), *[1] * (x.dim() - 1))[:batch].contiguous()
    args = (dev(copies(q)), dev(kc), dev(copies(lse)), dev(copies(torch.tensor(lens, dtype=torch.int32))), dev(copies(table)))
    w = dev(copies(before))
    out = fmha.fmha_key_weights(*args, weights=w)
    _close(out.cpu(), copies(want))
    assert fmha.fmha_key_weights(*args, weights=w, out=w) is w and torch.equal(w.cpu(), out.cpu())


def _shared_case(seed, lens, prefix, sq, hq, hk, d, dtype, page):
    """One group: the sequences share the first `prefix` tokens."""
    g = torch.Generator().manual_seed(seed)
    kc, vc, table = lc.pages(g, lens, page, hk, d, d, dtype)
    lc.share(kc, vc, table, [0, len(lens)], [prefix], page)
    return dict(q=lc.randn(g, len(lens), sq, hq, d, dtype=dtype), kc=kc, vc=vc, table=table, lens=lens)


@pytest.mark.parametrize("splits", [1, 2, 20])
def test_a_row_of_nan_is_nan_after_the_merge(fmha, splits):
    # a NaN query, and a query that meets an infinite key: the row's splits are all NaN, or some are; other rows do not notice
    lens = [700, 650, 3]
    c = _shared_case(5, lens, 3, 1, 4, 2, 64, torch.float16, 64)
    c["q"][0, 0, 1] = math.nan
    c["q"][:, 0, 2:, 0] = c["q"][:, 0, 2:, 0].abs() + 0.5
    c["kc"][c["table"][:, 0].long(), 2, 1, 0] = math.inf   # a key of the prefix
    bad = torch.zeros(3, 4, dtype=torch.bool)
    bad[0, 1] = True
    bad[:, 2:] = True
    ref, ref_lse = lc.decode(torch.nan_to_num(c["q"]), torch.nan_to_num(c["kc"], posinf=0.0, nan=0.0), c["vc"], lens, c["table"], 0.125)
    args = (dev(c["q"]), dev(c["kc"]), dev(c["vc"]), _i32(lens), dev(c["table"]))
    lse, lse2 = dev(torch.zeros(3, 4, 1)), dev(torch.zeros(3, 4, 1))
    o = fmha.fmha_decode_paged(*args, num_splits=splits, lse=lse)
    o2 = fmha.fmha_decode_shared_prefix(*args, _i32([3]), num_prefix_splits=1, num_splits=splits, lse=lse2)
    for got, got_lse in ((o, lse), (o2, lse2)):
        got, got_lse = got.cpu()[:, 0], got_lse.cpu()[..., 0]
        assert torch.isnan(got[bad]).all() and torch.isnan(got_lse[bad]).all()
        assert (got.double() - ref[:, 0])[~bad].abs().max() <= (2 * U[torch.float16] + 2.0 ** -20) * 6.0
        assert (got_lse.double() - ref_lse[..., 0])[~bad].abs().max() <= 2e-5


@contextlib.contextmanager
def _checked():
    flags.set_flag_value("FC_DEBUG_KERNEL_INSTANCE", "true")
    try:
        yield
    finally:
        flags.set_flag_value("FC_DEBUG_KERNEL_INSTANCE", "false")


def test_debug_flag_asks_for_the_entries_that_are_read(fmha):
    # two groups; rows of sequences other than a group's first hold no page ids for whole pages of the prefix
    lens, page = [40, 37, 50, 20, 33, 17], 16
    g = torch.Generator().manual_seed(6)
    kc, vc, table = lc.pages(g, lens, page, 1, 64, 64, torch.bfloat16)
    starts, prefixes = [0, 3, 6], [35, 16]
    lc.share(kc, vc, table, starts, prefixes, page)
    q = lc.randn(g, 6, 1, 2, 64, dtype=torch.bfloat16)
    ref, _ = lc.decode(q, kc, vc, lens, table, 0.125)
    rows = table.clone()
    rows[1:3, :2] = -1
    rows[4:, :1] = 10 ** 6
    args = lambda t: (dev(q), dev(kc), dev(vc), _i32(lens), dev(t), _i32(prefixes))
    with _checked():
        o = fmha.fmha_decode_shared_prefix(*args(rows), cu_groups=_i32(starts)).cpu()
        assert (o.double() - ref).abs().max() <= (2 * U[torch.bfloat16] + 2.0 ** -20) * 6.0
        for b, j, kw in ((0, 0, {}), (1, 2, {}), (2, 3, {}), (2, 1, dict(max_group_size=2))):
            bad = rows.clone()
            bad[b, j] = kc.shape[0]
            with pytest.raises(ValueError, match=f"first offending sequence: {b}"):
                fmha.fmha_decode_shared_prefix(*args(bad), cu_groups=_i32(starts), **kw)
        # a step appends through the sequence's own row: sequence 5 is still inside the prefix of its group
        short = [40, 37, 50, 20, 33, 15]
        new = lc.randn(g, 6, 1, 1, 64, dtype=torch.bfloat16)
        step = lambda t, n: fmha.fmha_decode_step(dev(q), dev(new), dev(new), dev(kc), dev(vc), _i32(n), dev(t), prefix_lens=_i32(prefixes),
                                                  cu_groups=_i32(starts))
        step(rows, lens)
        with pytest.raises(ValueError, match="first offending sequence: 5"):
            step(rows, short)


@pytest.mark.parametrize("sq,hq,d", [(1, 4, 64), (33, 2, 64), (290, 2, 64)])
@pytest.mark.parametrize("paged", [True, False])
def test_counts_beyond_what_the_cache_holds_are_cut(fmha, sq, hq, d, paged):
    lens, splits = [128, 100], 2 if sq == 290 else 1
    c = _weights_case(7, lens, sq, hq, 1, d, torch.bfloat16, 64)
    cache, table = c["kc"], c["table"]
    if not paged:   # the second sequence's own row ends the tensor
        cache = torch.stack([torch.nan_to_num(torch.cat([c["kc"][p] for p in table[b].tolist()])) for b in range(2)])
        c["keys"][1] = cache[1].double()
    if paged:
        c["kc"][table[1, 1], 36:] = 0
        c["keys"][1] = lc.rows(c["kc"], table[1], 128, 64)
    want = lc.key_weights(c["q"], c["keys"], c["lse"], 300, d ** -0.5, before=torch.ones(2, 1, 300))
    for n in ([128, 128], [129, 300], [128, 2 ** 31 - 1]):
        out = fmha.fmha_key_weights(dev(c["q"]), dev(cache), dev(c["lse"]), _i32(n), dev(table) if paged else None,
                                    weights=dev(torch.ones(2, 1, 300)), num_row_splits=splits)
        _close(out.cpu(), want, f"{n}")


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("sq,page,window,prefix", [(1, 64, (20, 0), 0), (1, 16, (20, 0), 90), (3, 64, (30, 2), 70), (1, 128, (0, 0), 100), (2, 48, (150, 0), 40)])
def test_values_of_keys_outside_the_window_do_not_matter(fmha, bad, sq, page, window, prefix):
    lens = [prefix + 30, prefix + 101]
    c = _shared_case(8, lens, prefix, sq, 4, 2, 64, torch.bfloat16, page)
    for b, n in enumerate(lens):
        for t in range(max(0, n - sq - window[0])):
            # a key of the prefix may be in the other sequence's window
            if t >= prefix or t < min(lens) - sq - window[0]:
                for pool in (c["kc"], c["vc"]):
                    pool[c["table"][b, t // page], t % page] = bad
    kw = dict(mask_type=2, window=window)
    ref, ref_lse = lc.decode(c["q"], c["kc"], c["vc"], lens, c["table"], 0.125, **kw)
    lse = dev(torch.zeros(2, 4, sq))
    for splits in ((1, 1), (3, 2)):
        o = fmha.fmha_decode_shared_prefix(dev(c["q"]), dev(c["kc"]), dev(c["vc"]), _i32(lens), dev(c["table"]), _i32([prefix]), lse=lse,
                                           num_prefix_splits=splits[0], num_splits=splits[1], **kw).cpu()
        assert torch.isfinite(o.float()).all()
        assert (o.double() - ref).abs().max() <= (2 * U[torch.bfloat16] + 2.0 ** -20) * 6.0
        assert (lse.cpu().double() - ref_lse).abs().max() <= 2e-5


@pytest.mark.parametrize("bounds", [dict(), dict(max_prefix_len=30000, max_seqlen_k=30000), dict(max_prefix_len=64, max_seqlen_k=128)])
def test_every_split_takes_its_part_of_the_keys_whatever_the_bounds(fmha, bounds):
    # a table that can address far more than the sequences have, bounds far above and below what they have
    lens, prefix, nsp, nso = [2048 + 1100, 2048 + 1024, 2048 + 10], 2048, 8, 4
    c = _shared_case(9, lens, prefix, 1, 2, 1, 64, torch.bfloat16, 64)
    table = torch.cat([c["table"], torch.zeros(3, 600, dtype=torch.int32)], dim=1)
    ws = fmha.DecodeWorkspace()
    lse = dev(torch.zeros(3, 2, 1))
    o = fmha.fmha_decode_shared_prefix(dev(c["q"]), dev(c["kc"]), dev(c["vc"]), _i32(lens), dev(table), _i32([prefix]), lse=lse, workspace=ws,
                                       num_prefix_splits=nsp, num_splits=nso, **bounds)
    _, parts = ws.partials(3, 2, nsp + nso, 1, 64, o.device)
    some = torch.isfinite(parts.cpu())[..., 0]
    assert some[:, :, :nsp].all() and some[:2, :, nsp:].all()
    assert some[2, :, nsp].all() and not some[2, :, nsp + 1:].any()   # 10 keys are not cut
    ref, ref_lse = lc.decode(c["q"], c["kc"], c["vc"], lens, c["table"], 0.125)
    assert (o.cpu().double() - ref).abs().max() <= (2 * U[torch.bfloat16] + 2.0 ** -20) * 6.0
    assert (lse.cpu().double() - ref_lse).abs().max() <= 2e-5


def test_a_captured_call_survives_a_workspace_that_grows(fmha):
    c = _shared_case(10, [200, 220], 150, 1, 4, 2, 64, torch.bfloat16, 64)
    big = _shared_case(11, [300] * 12, 150, 1, 4, 2, 64, torch.bfloat16, 64)
    inputs = lambda x: (dev(x["q"]), dev(x["kc"]), dev(x["vc"]), _i32(x["lens"]), dev(x["table"]), _i32([150]))
    args, more = inputs(c), inputs(big)
    ws, out = fmha.DecodeWorkspace(), torch.empty_like(args[0])
    want = fmha.fmha_decode_shared_prefix(*args)
    fmha.fmha_decode_shared_prefix(*args, workspace=ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fmha.fmha_decode_shared_prefix(*args, workspace=ws, out=out)
    fmha.fmha_decode_shared_prefix(*more, workspace=ws)   # outgrows the buffers of the graph
    others = [torch.full((n,), 7.0, device="cuda") for n in (256, 1024, 4096, 16384, 65536) for _ in range(8)]   # would take their place
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all((x == 7.0).all() for x in others)


@pytest.mark.parametrize("splits", [1, 3])
def test_rows_behind_the_last_sequence_stay_as_they_were(fmha, splits):
    lens, starts = [90, 40], [0, 3, 4]
    g = torch.Generator().manual_seed(12)
    kc, vc, table = lc.pages(g, lens, 16, 2, 64, 64, torch.bfloat16)
    q = lc.randn(g, 9, 4, 64, dtype=torch.bfloat16)   # five rows behind the last sequence
    kw = dict(mask_type=2, window=(-1, 0))
    ref, ref_lse = lc.decode(q, kc, vc, lens, table, 0.125, starts=starts, **kw)
    out, lse = dev(torch.full((9, 4, 64), 3.0, dtype=torch.bfloat16)), dev(torch.full((4, 9), 7.0))
    ws = (dev(torch.full((1, 4, splits, 9, 64), 5.0)), dev(torch.full((1, 4, splits, 9), 5.0)))
    fmha.fmha_decode_paged(dev(q), dev(kc), dev(vc), _i32(lens), dev(table), num_splits=splits, cu_seqlens_q=_i32(starts), max_seqlen_q=3,
                           workspace=ws, out=out, lse=lse, **kw)
    out, lse = out.cpu(), lse.cpu()
    assert (out[:4].double() - ref[:4]).abs().max() <= (2 * U[torch.bfloat16] + 2.0 ** -20) * 6.0
    assert (lse[:, :4].double() - ref_lse[:, :4]).abs().max() <= 2e-5
    assert (out[4:] == 3.0).all() and (lse[:, 4:] == 7.0).all()


@pytest.mark.parametrize("window_left", [-1, 40])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_module_steps_over_shared_prefixes(fmha, window_left, packed, fp8):
    """PagedAttention: three steps with prefix_lens and without on caches of their own, the weights of the last step's keys, and an
    eviction: what a serving loop runs.  Bounds of the outputs: both sides within 2 u max|v| of the definition, max|v| < 6."""
    from flashck_amd.nn import PagedAttention
    g = torch.Generator().manual_seed(13)
    lens, page, hq, hk, d = [100, 90, 130, 40, 33], 16, 8, 2, 64
    starts, prefixes, counts = [0, 3, 5], [70, 20], ([2, 1, 0, 3, 2] if packed else [2] * 5)
    kc, vc, table = lc.pages(g, [n + 10 for n in lens], page, hk, d, d, torch.bfloat16, fp8, extra=20, poison=False)
    lc.share(kc, vc, table, starts, prefixes, page)
    kd, vd = (0.5, 0.25) if fp8 else (1.0, 1.0)
    modules = [PagedAttention(hq, hk, d, window_left=window_left, rope_mode=fmha.ROPE_HALF_ROTATED, k_descale=kd, v_descale=vd) for _ in range(2)]
    caches = [(dev(kc.clone()), dev(vc.clone())) for _ in range(2)]
    angles = torch.arange(200)[:, None] * torch.exp(-torch.arange(0, d, 2) / d * 9.0)
    rotary = dict(rotary_cos=dev(torch.cos(angles).to(torch.bfloat16)), rotary_sin=dev(torch.sin(angles).to(torch.bfloat16)))
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    extra = dict(cu_seqlens_knew=_i32(cu), max_seqlen_knew=3) if packed else {}
    shape, total = ((cu[-1],) if packed else (5, 2)), cu[-1]
    now = [_i32(lens), _i32(lens)]
    dt = dev(table)
    for step in range(3):
        q, kn, vn = (lc.randn(g, *shape, h, d, dtype=torch.bfloat16) for h in (hq, hk, hk))
        lse = [dev(torch.zeros(*((hq, total) if packed else (5, hq, 2)))) for _ in range(2)]
        outs, queries = [], []
        for k, m in enumerate(modules):
            queries.append(dev(q.clone()))
            prefix = dict(prefix_lens=_i32(prefixes), cu_groups=_i32(starts)) if k == 0 else {}
            o, n = m.decode_step(queries[k], dev(kn), dev(vn), *caches[k], now[k], dt, lse=lse[k], **rotary, **extra, **prefix)
            outs.append(o.cpu())
            now[k] = n.clone()
        torch.cuda.synchronize()
        assert torch.equal(now[0].cpu(), now[1].cpu())
        for a, b in zip(*caches):
            assert torch.equal(a.cpu().view(torch.uint8), b.cpu().view(torch.uint8))
        assert torch.equal(queries[0].cpu(), queries[1].cpu())   # rotated in place
        assert torch.isfinite(outs[0].float()).all()
        assert (outs[0].double() - outs[1].double()).abs().max() <= 4 * U[torch.bfloat16] * 6.0
        assert (lse[0].cpu() - lse[1].cpu()).abs().max() <= 4e-5
    assert now[0].cpu().tolist() == [n + 3 * c for n, c in zip(lens, counts)]
    more = dict(cu_seqlens_q=_i32(cu), max_seqlen_q=3) if packed else {}
    w = modules[0].key_weights(queries[0], caches[0][0], lse[0], now[0], dt, **more)
    # every row gives its heads a weight of one each
    rows = torch.tensor(counts, dtype=torch.float64)[:, None] * (hq // hk)
    assert (w.cpu().double().sum(dim=2) - rows).abs().max() <= 1e-4 * rows.max()
    if window_left >= 0:
        return
    free = sorted(set(range(kc.shape[0])) - set(table.flatten().tolist()))[:10]
    n_new, kept, _ = modules[0].evict(*caches[0], w, now[0], dt, _i32(free).view(5, 2), budget=32, recent=4)
    torch.cuda.synchronize()
    assert kept.cpu().tolist() == lc.evict(w.cpu(), now[0].cpu().tolist(), 32, 4, 0) and n_new.cpu().tolist() == [32] * 5


# (sizes of the groups, sequences before the first and behind the last, tokens a sequence, query heads of the 1 KV head, head dim)
MANY_GROUPS = [([2] * 10, 0, 0, 1, 16, 64), ([1, 9, 1, 1, 0, 3, 1, 1, 1, 2], 3, 2, 1, 16, 64), ([1] * 12, 5, 0, 2, 8, 128), ([2, 2, 3, 2], 1, 1, 5, 16, 64),
               ([3, 1, 2, 2, 2], 0, 0, 4, 12, 256)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("sizes,before,behind,sq,hq,d", MANY_GROUPS)
def test_many_groups_without_a_bound_on_their_size(fmha, sizes, before, behind, sq, hq, d, packed):
    # so many that the row tiles are not dealt out equally: groups of one tile, of several, empty ones, rows of no group; sequences share
    # whole pages only (page 16, prefixes of 0, 16, 32)
    g = torch.Generator().manual_seed(14)
    starts = [before]
    for s in sizes:
        starts.append(starts[-1] + s)
    batch = starts[-1] + behind
    prefixes = [(0, 32, 16, 32)[k % 4] for k in range(len(sizes))]
    lens = [35 + b % 5 * 9 for b in range(batch)]
    kc, vc, table = lc.pages(g, lens, 16, 1, d, d, torch.bfloat16)
    lc.share(kc, vc, table, starts, prefixes, 16)
    counts = [(sq, 0, 1, sq)[b % 4] for b in range(batch)] if packed else [sq] * batch
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    q = lc.randn(g, *((cu[-1],) if packed else (batch, sq)), hq, d, dtype=torch.bfloat16)
    kw = dict(mask_type=2, window=(-1, 0))
    ref, ref_lse = lc.decode(q, kc, vc, lens, table, d ** -0.5, starts=cu if packed else None, **kw)
    lse = dev(torch.zeros(ref_lse.shape))
    if packed:
        kw.update(cu_seqlens_q=_i32(cu), max_seqlen_q=sq)
    for nsp in (1, 3):
        o = fmha.fmha_decode_shared_prefix(dev(q), dev(kc), dev(vc), _i32(lens), dev(table), _i32(prefixes), cu_groups=_i32(starts), lse=lse,
                                           num_prefix_splits=nsp, num_splits=2, **kw).cpu()
        assert (o.double() - ref).abs().max() <= (2 * U[torch.bfloat16] + 2.0 ** -20) * 6.0
        assert (lse.cpu().double() - ref_lse).abs().max() <= 2e-5

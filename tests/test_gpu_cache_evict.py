"""GPU: eviction from a paged cache by weight: kept positions, lengths, weights and rows are exact."""
import math

import pytest
import torch

import longcontext as lc
from helpers import dev

pytestmark = pytest.mark.gpu


def _i32(x):
    return dev(torch.tensor(x, dtype=torch.int32))


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _run(fmha, seed, lens, hk, d, dtype, page, budget, recent=0, sinks=0, dv=None, weights=None, cols=None, new_page=None, own_pool=False):
    g = torch.Generator().manual_seed(seed)
    fp8 = dtype == lc.FP8
    kept_pages = -(-budget // (new_page or page))
    kc, vc, table = lc.pages(g, lens, page, hk, d, dv or d, torch.bfloat16 if fp8 else dtype, fp8, extra=1 + (0 if own_pool else len(lens) * kept_pages))
    cols = cols or max(max(lens), 1)
    if weights is None:
        weights = torch.rand(len(lens), hk, cols, generator=g)
    used = set(table.flatten().tolist())
    if own_pool:
        nk = torch.zeros(len(lens) * kept_pages, new_page or page, hk, d).to(kc.dtype)
        nv = torch.zeros(len(lens) * kept_pages, new_page or page, hk, dv or d).to(kc.dtype)
        free = torch.randperm(len(lens) * kept_pages, generator=g).tolist()
    else:
        nk, nv = None, None
        free = [p for p in range(kc.shape[0]) if p not in used]
    new_table = torch.tensor(free[:len(lens) * kept_pages], dtype=torch.int32).view(len(lens), kept_pages)
    dk, dvv = dev(kc), dev(vc)
    dnk, dnv = (dev(nk), dev(nv)) if own_pool else (None, None)
    n_new, kept, w_new = fmha.fmha_cache_evict(dk, dvv, dev(weights), _i32(lens), dev(table), dev(new_table), budget=budget, recent=recent,
                                               sinks=sinks, new_k_cache=dnk, new_v_cache=dnv)
    torch.cuda.synchronize()
    n_new, kept, w_new = n_new.cpu(), kept.cpu(), w_new.cpu()
    want = lc.evict(weights, lens, budget, recent, sinks)
    target_k, target_v = (nk, nv) if own_pool else (kc, vc)
    want_k, want_v = target_k.clone(), target_v.clone()
    np_ = target_k.shape[1]
    for b, n in enumerate(lens):
        assert n_new[b] == min(n, budget)
        for h in range(hk):
            w = want[b][h]
            assert kept[b, h].tolist() == w + [-1] * (budget - len(w)), f"sequence {b} head {h}"
            expect = torch.zeros(cols)
            at = torch.tensor([t for t in w if t < cols], dtype=torch.long)
            expect[:len(at)] = weights[b, h, at]
            assert torch.equal(torch.nan_to_num(w_new[b, h], nan=-7.0), torch.nan_to_num(expect, nan=-7.0)), f"sequence {b} head {h}"
            for j, t in enumerate(w):
                want_k[new_table[b, j // np_], j % np_, h] = kc[table[b, t // page], t % page, h]
                want_v[new_table[b, j // np_], j % np_, h] = vc[table[b, t // page], t % page, h]
    got_k, got_v = (dnk, dnv) if own_pool else (dk, dvv)
    assert torch.equal(_bytes(got_k.cpu()), _bytes(want_k)) and torch.equal(_bytes(got_v.cpu()), _bytes(want_v))
    if own_pool:
        assert torch.equal(_bytes(dk.cpu()), _bytes(kc)) and torch.equal(_bytes(dvv.cpu()), _bytes(vc))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, lc.FP8])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 48), (256, 1), (72, 64), (8, 16)])
def test_types_and_shapes(fmha, dtype, d, page):
    _run(fmha, 1, [100, 33, 32, 1, 0, 70], 2, d, dtype, page, 33, recent=4, sinks=2)


@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 64, 0), (64, 0, 64), (64, 30, 34), (64, 0, 0),
                                                 (63, 20, 4), (299, 1, 1), (300, 0, 0), (500, 10, 10)])
@pytest.mark.parametrize("own_pool", [False, True])
def test_budgets(fmha, budget, recent, sinks, own_pool):
    _run(fmha, 2, [300, 64, 65, 299], 2, 64, torch.bfloat16, 16, budget, recent, sinks, own_pool=own_pool)


def test_equal_weights_and_special_values(fmha):
    lens = [200, 200, 200, 200]
    g = torch.Generator().manual_seed(3)
    w = torch.randint(0, 3, (4, 2, 200), generator=g).float()
    w[1] = 0.0
    w[1, :, ::2] = -0.0  # both zeros are equal
    w[2, 0, 10:150] = math.nan
    w[2, 0, 20] = -math.inf  # equal to a NaN: the lower position first
    w[2, 1, 5:100] = math.inf
    w[3] = -torch.rand(2, 200, generator=g)
    for budget, recent, sinks in ((100, 0, 0), (77, 10, 3), (180, 0, 5)):
        _run(fmha, 4, lens, 2, 64, torch.float16, 64, budget, recent, sinks, weights=w)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2049, 4100])
def test_long_rows(fmha, n):
    _run(fmha, 5, [n, n - 1], 1, 8, torch.bfloat16, 64, n // 3, recent=17, sinks=4, own_pool=True)
    g = torch.Generator().manual_seed(n)
    w = torch.randint(0, 2, (2, 1, n), generator=g).float()  # most of the choice is between equals
    _run(fmha, 6, [n, n - 1], 1, 8, torch.bfloat16, 64, n // 2, weights=w, own_pool=True)


def test_fewer_and_more_columns_than_keys(fmha):
    # keys without a column weigh 0; columns behind the kept keys are zeroed
    _run(fmha, 7, [150, 40], 2, 64, torch.bfloat16, 16, 30, recent=5, cols=100)
    _run(fmha, 8, [150, 40], 2, 64, torch.bfloat16, 16, 120, recent=5, cols=20)
    _run(fmha, 9, [150, 40], 2, 64, torch.bfloat16, 16, 30, recent=5, cols=1500)


@pytest.mark.parametrize("dv,new_page", [(32, 16), (128, 48), (64, 1)])
def test_other_page_size_and_value_dim(fmha, dv, new_page):
    _run(fmha, 10, [90, 200], 2, 64, torch.float16, 32, 50, 3, 3, dv=dv, new_page=new_page, own_pool=True)


def test_many_values_close_together(fmha):
    # neighbours that differ in the last bits only
    g = torch.Generator().manual_seed(11)
    base = torch.full((1, 2, 3000), 1.0).view(torch.int32) + torch.randint(-40, 40, (1, 2, 3000), generator=g, dtype=torch.int32)
    _run(fmha, 11, [3000], 2, 8, torch.bfloat16, 64, 700, weights=base.view(torch.float32), own_pool=True)


def test_the_whole_sequence(fmha):
    """Prefill, weights, eviction, and decode steps from the smaller cache with a shared prefix: the run they are made for."""
    g = torch.Generator().manual_seed(12)
    page, hq, hk, d, n = 16, 4, 2, 64, 90
    kc, vc, table = lc.pages(g, [n, n], page, hk, d, d, torch.bfloat16, extra=12, poison=False)
    free = sorted(set(range(kc.shape[0])) - set(table.flatten().tolist()))
    q = lc.randn(g, 2, n, hq, d, dtype=torch.bfloat16)
    lens, scale = [n, n - 20], d ** -0.5
    mask = dict(mask_type=2, window=(-1, 0))
    dk, dvv, dt, dl = dev(kc), dev(vc), dev(table), _i32(lens)
    lse = dev(torch.empty(2, hq, n))
    fmha.fmha_fwd_pagedkv(dev(q), dk, dvv, dl, dt, lse=lse, **mask)
    w = fmha.fmha_key_weights(dev(q), dk, lse, dl, dt, **mask)
    _, ref_lse = lc.decode(q, kc, vc, lens, table, scale, **mask)
    keys = [lc.rows(kc, table[b], m, page) for b, m in enumerate(lens)]
    want_w = lc.key_weights(q, keys, ref_lse, table.shape[1] * page, scale, **mask)
    assert ((w.cpu().double() - want_w).abs() - 1e-4 * want_w).max() <= 1e-9
    budget = 40
    new_table = torch.zeros(2, 5, dtype=torch.int32)
    new_table[:, :3] = torch.tensor(free[:6]).view(2, 3)
    new_table[:, 3:] = torch.tensor(free[6:10]).view(2, 2)
    dnt = dev(new_table)
    n_new, kept, w_new = fmha.fmha_cache_evict(dk, dvv, w, dl, dt, dnt, budget=budget, recent=8, sinks=2)
    torch.cuda.synchronize()
    kept_ref = lc.evict(w.cpu(), lens, budget, 8, 2)
    assert kept.cpu().tolist() == kept_ref and n_new.cpu().tolist() == [budget] * 2
    # two steps of one token each from the evicted cache, sharing the first sequence's kept keys as a prefix of 0 tokens
    cur_k, cur_v = dk.cpu().clone(), dvv.cpu().clone()
    for step in range(2):
        k1, v1, q1 = (lc.randn(g, 2, 1, h, d, dtype=torch.bfloat16) for h in (hk, hk, hq))
        fmha.fmha_fwd_appendkv(None, dk, dvv, dev(k1), dev(v1), n_new, block_table=dnt)
        for b in range(2):
            t = budget + step
            cur_k[new_table[b, t // page], t % page] = k1[b, 0]
            cur_v[new_table[b, t // page], t % page] = v1[b, 0]
        n_new = n_new + 1
        step_lse = dev(torch.empty(2, hq, 1))
        o = fmha.fmha_decode_shared_prefix(dev(q1), dk, dvv, n_new, dnt, _i32([0]), lse=step_lse)
        w_new = fmha.fmha_key_weights(dev(q1), dk, step_lse, n_new, dnt, weights=w_new, out=w_new)
        torch.cuda.synchronize()
        ref, ref_lse = lc.decode(q1, cur_k, cur_v, [budget + step + 1] * 2, new_table, scale)
        assert (o.cpu().double() - ref).abs().max() <= 2 * 2.0 ** -8 * 6
        assert (step_lse.cpu().double() - ref_lse).abs().max() <= 2e-5
    got = w_new.cpu().double()
    assert not got[:, :, budget + 2:].any()
    total = sum(want_w[b, h, torch.tensor(kept_ref[b][h])].sum().item() for b in range(2) for h in range(hk))
    assert abs(got.sum().item() - (total + 2 * 2 * hq)) <= 1e-4 * (total + 2 * 2 * hq)


def test_captured_and_replayed(fmha):
    g = torch.Generator().manual_seed(13)
    lens = [500, 300]
    kc, vc, table = (dev(x) for x in lc.pages(g, lens, 16, 2, 64, 64, torch.bfloat16, extra=20))
    used = set(table.flatten().tolist())
    free = [p for p in range(kc.shape[0]) if p not in used][:16]
    new_table = _i32(free).view(2, 8)
    w, n = torch.rand(2, 2, 500, device="cuda"), _i32(lens)
    outs = dict(out_seqlen=_i32([0, 0]), out_kept=torch.zeros(2, 2, 128, dtype=torch.int32, device="cuda"), out_weights=torch.zeros_like(w))
    kw = dict(budget=128, recent=10, sinks=3)
    fmha.fmha_cache_evict(kc, vc, w, n, table, new_table, **kw, **outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fmha.fmha_cache_evict(kc, vc, w, n, table, new_table, **kw, **outs)
    for step in range(4):
        w.copy_(torch.rand_like(w))
        n.sub_(7)
        graph.replay()
        torch.cuda.synchronize()
        got, rows = [x.clone() for x in outs.values()], _bytes(kc).clone()
        again = fmha.fmha_cache_evict(kc, vc, w, n, table, new_table, **kw)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, again)) and torch.equal(rows, _bytes(kc)), f"replay {step}"


def test_on_another_stream(fmha):
    g = torch.Generator().manual_seed(14)
    lens = [3000, 2000]
    kc, vc, table = (dev(x) for x in lc.pages(g, lens, 64, 2, 64, 64, torch.bfloat16))
    w, n, new_table = torch.rand(2, 2, 3000, device="cuda"), _i32(lens), _i32([3, 0, 5, 1, 7, 2, 4, 6]).view(2, 4)
    pools = [[torch.zeros(8, 64, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(3)]
    run = lambda p: fmha.fmha_cache_evict(kc, vc, w, n, table, new_table, budget=256, new_k_cache=p[0], new_v_cache=p[1])
    first = run(pools[0])
    torch.cuda.synchronize()
    got = []
    for p in pools[1:]:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(run(p))
    torch.cuda.synchronize()
    for p, x in zip(pools[1:], got):
        assert all(torch.equal(a, b) for a, b in zip(first, x)) and all(torch.equal(a, b) for a, b in zip(pools[0], p))


@pytest.mark.parametrize("cols,lens", [(65536, [3000, 700]), (65546, [16390, 64]), (70000, [16100, 16100])])
def test_wide_rows(fmha, cols, lens):
    # rows long enough that several workgroups choose from each; distinct weights, and weights that are mostly equal
    g = torch.Generator().manual_seed(15)
    _run(fmha, 16, lens, 1, 8, torch.bfloat16, 64, 600, 40, 4, cols=cols, own_pool=True)
    w = torch.randint(0, 2, (2, 1, cols), generator=g).float()
    w[0, 0, 100:200] = math.nan
    _run(fmha, 17, lens, 1, 8, torch.bfloat16, 64, 500, 0, 3, cols=cols, weights=w, own_pool=True)
    _run(fmha, 18, lens, 1, 8, torch.bfloat16, 64, 44, 40, 4, cols=cols, own_pool=True)

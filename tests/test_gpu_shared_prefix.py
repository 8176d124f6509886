"""GPU: decode attention over shared prefixes against its definition in 64 bits and against the decode without sharing.

Tolerances.  Scores are products of 16-bit values summed in fp32 (relative error below 2^-20 for these lengths).  The
kernels round the probabilities (a row's common factor apart) to the 16-bit type before the second product, off by at most half a step, u = 2^-8
(bf16) or 2^-11 (fp16) relative, and the result once more.  So |o - o_ref| <= u * sum_j p_j |v_j| + u * |o| <= 2 u max|v|;
the values are normal, max|v| < 6, and 2^-20 more covers the fp32 parts.  The log-sum-exp is fp32 throughout: 2e-5
absolute for |lse| < 16 (a dozen fp32 steps, the hardware's exp2 and log2 being off by about one each)."""
import math

import pytest
import torch

import longcontext as lc
from helpers import dev

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _case(seed, sizes, prefixes, own, hq, hk, d, dtype, page, sq=1, dv=None, fp8=False):
    g = torch.Generator().manual_seed(seed)
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    lens = [prefixes[k] + own[(starts[k] + i) % len(own)] for k, s in enumerate(sizes) for i in range(s)]
    kc, vc, table = lc.pages(g, lens, page, hk, d, dv or d, dtype, fp8)
    lc.share(kc, vc, table, starts, prefixes, page)
    return dict(q=lc.randn(g, len(lens), sq, hq, d, dtype=dtype), kc=kc, vc=vc, table=table, lens=lens, starts=starts,
                prefixes=prefixes)


def _run(fmha, c, lse=True, **kw):
    i32 = lambda x: dev(torch.tensor(x, dtype=torch.int32))
    q = dev(c["q"])
    out_lse = dev(torch.full((q.shape[1], q.shape[0]) if q.dim() == 3 else (q.shape[0], q.shape[2], q.shape[1]), 7.0)) if lse else None
    groups = kw.pop("cu_groups", c["starts"])
    o = fmha.fmha_decode_shared_prefix(q, dev(c["kc"]), dev(c["vc"]), i32(c["lens"]), dev(c["table"]), i32(c["prefixes"]),
                                       cu_groups=None if groups is None else i32(groups), lse=out_lse, **kw)
    torch.cuda.synchronize()
    return o.cpu(), None if out_lse is None else out_lse.cpu()


def _check(o, lse, ref, ref_lse, dtype, what=""):
    assert o.shape == ref.shape and torch.isfinite(o.float()).all(), what
    bound = (2 * U[dtype] + 2.0 ** -20) * 6.0
    err = (o.double() - ref).abs().max().item()
    assert err <= bound, f"{what}: output off by {err:.3e} > {bound:.3e}"
    assert torch.equal(torch.isinf(lse), torch.isinf(ref_lse)), what
    fin = torch.isfinite(ref_lse)
    err = (lse.double() - ref_lse)[fin].abs().max().item() if fin.any() else 0.0
    assert err <= 2e-5, f"{what}: lse off by {err:.3e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d,page", [(8, 2, 64, 64), (8, 2, 128, 128), (4, 4, 128, 16), (8, 1, 256, 48), (4, 2, 256, 64),
                                          (6, 2, 128, 1)])
def test_one_group(fmha, dtype, hq, hk, d, page):
    c = _case(1, [5], [131], [0, 1, 40, 64, 129], hq, hk, d, dtype, page)
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], d ** -0.5)
    for nsp, nso in ((0, 0), (1, 1), (3, 2)):
        o, lse = _run(fmha, c, num_prefix_splits=nsp, num_splits=nso)
        _check(o, lse, *ref, dtype, f"splits {nsp} {nso}")


@pytest.mark.parametrize("splits", [(64, 64), (64, 1), (1, 64)])
def test_most_splits(fmha, splits):
    c = _case(23, [2, 3], [700, 0], [0, 513, 64], 8, 2, 64, torch.bfloat16, 64)
    o, lse = _run(fmha, c, num_prefix_splits=splits[0], num_splits=splits[1])
    _check(o, lse, *lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 0.125), torch.bfloat16, f"{splits}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [0.75, 4.0, 16.0])
def test_scores_that_grow_along_the_keys(fmha, dtype, step):
    # the largest score of every tile outgrows that of the tile before by less and by more than any reference of the
    # exponents may lag behind; rows of the group grow, fall and stay, in one wave.  q = (c, 0, ..), k = (step * tile, ..)
    c = _case(24, [16], [64 * 9], [5, 64], 1, 1, 64, dtype, 64)
    c["q"].zero_()
    c["q"][:, 0, 0, 0] = torch.tensor([1.0, -1.0, 0.0, 0.5] * 4)
    for b, n in enumerate(c["lens"]):
        for t in range(n):
            c["kc"][int(c["table"][b, t // 64]), t % 64, 0, 0] = step * (t // 64)
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 1.0)
    for splits in ((1, 1), (3, 1)):
        o, lse = _run(fmha, c, scale=1.0, num_prefix_splits=splits[0], num_splits=splits[1])
        assert (o.double() - ref[0]).abs().max() <= (2 * U[dtype] + 2.0 ** -20) * 6.0
        # |score| reaches 144: an fp32 step there is 2^-16
        assert (lse.double() - ref[1]).abs().max() <= 1e-4


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 33, 70])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_group_sizes(fmha, rows, d):
    # a row tile that is not full, full, and followed by others; heads of a group share the tile
    c = _case(2 + rows, [rows], [70], [1, 5], 4, 1, d, torch.bfloat16, 64)
    o, lse = _run(fmha, c, num_prefix_splits=2)
    _check(o, lse, *lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], d ** -0.5), torch.bfloat16)


@pytest.mark.parametrize("page", [16, 128])
def test_several_groups_and_none(fmha, page):
    # groups of different sizes and prefixes: none shared, a prefix of one token, no keys at all, one that ends in a page
    c = _case(5, [3, 1, 4, 2], [0, 200, 1, 77], [0, 3, 130], 8, 2, 128, torch.bfloat16, page)
    c["lens"][1] = 0
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 128 ** -0.5)
    for kw in ({}, dict(max_group_size=4, max_prefix_len=200, max_seqlen_k=330), dict(max_group_size=2)):
        o, lse = _run(fmha, c, **kw)
        _check(o, lse, *ref, torch.bfloat16, str(kw))
    assert torch.equal(o[1], torch.zeros_like(o[1])) and torch.isinf(lse[1]).all()


def test_sequences_outside_every_group(fmha):
    c = _case(6, [2, 3, 2], [50, 90, 0], [7, 64], 4, 2, 64, torch.float16, 64)
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 64 ** -0.5)
    c["prefixes"] = [90]
    o, lse = _run(fmha, c, cu_groups=[2, 5])
    _check(o, lse, *ref, torch.float16)
    c["prefixes"] = [0, 90, 0]
    o, lse = _run(fmha, c, cu_groups=[0, 2, 5, 5])
    _check(o, lse, *ref, torch.float16)


def test_prefix_longer_than_the_sequences(fmha):
    # the prefix is cut to what the group's first sequence has; one that ends inside it sees its own part of it
    c = _case(7, [3], [100], [10, 0, 60], 4, 1, 128, torch.bfloat16, 64)
    c["prefixes"] = [10 ** 6]
    c["lens"][0] = 90
    c["lens"][1] = 33
    o, lse = _run(fmha, c)
    _check(o, lse, *lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 128 ** -0.5), torch.bfloat16)
    c["prefixes"] = [-5]
    o, lse = _run(fmha, c)
    _check(o, lse, *lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 128 ** -0.5), torch.bfloat16)


@pytest.mark.parametrize("mask_type,window", [(2, (-1, 0)), (2, (20, 0)), (2, (150, 3)), (1, (-1, 0)), (1, (9, 2)), (2, (0, 0))])
@pytest.mark.parametrize("sq,d", [(1, 64), (3, 128), (5, 256)])
def test_masks(fmha, mask_type, window, sq, d):
    # own tokens fewer than the query tokens: the diagonal reaches back into the prefix; windows that leave it out entirely
    c = _case(8, [4, 2], [70, 9], [0, 2, 80], 4, 2, d, torch.bfloat16, 64, sq=sq)
    kw = dict(mask_type=mask_type, window=window)
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], d ** -0.5, **kw)
    o, lse = _run(fmha, c, num_prefix_splits=2, num_splits=2, **kw)
    _check(o, lse, *ref, torch.bfloat16, f"{kw}")


def test_packed_queries_of_different_lengths(fmha):
    g = torch.Generator().manual_seed(9)
    c = _case(9, [3, 2], [65, 0], [6, 40, 0], 4, 2, 64, torch.bfloat16, 16)
    counts = [1, 0, 4, 2, 3]
    starts_q = [0]
    for n in counts:
        starts_q.append(starts_q[-1] + n)
    c["q"] = lc.randn(g, starts_q[-1] + 2, 4, 64, dtype=torch.bfloat16)  # two rows behind the last sequence
    kw = dict(mask_type=2, window=(-1, 0))
    ref, ref_lse = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 0.125, starts=starts_q, **kw)
    out = dev(torch.full((starts_q[-1] + 2, 4, 64), 3.0, dtype=torch.bfloat16))
    o, lse = _run(fmha, c, cu_seqlens_q=dev(torch.tensor(starts_q, dtype=torch.int32)), max_seqlen_q=4, out=out, **kw)
    n = starts_q[-1]
    _check(o[:n], lse[:, :n], ref[:n], ref_lse[:, :n], torch.bfloat16)
    assert (o[n:] == 3.0).all() and (lse[:, n:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_quantised_cache(fmha, dtype, d, page):
    c = _case(10, [3, 2], [66, 17], [5, 64], 4, 2, d, dtype, page, fp8=True)
    o, lse = _run(fmha, c, k_descale=0.5, v_descale=0.25)
    _check(o, lse, *lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], d ** -0.5, kd=0.5, vd=0.25), dtype)


@pytest.mark.parametrize("d,dv,page", [(72, 40, 64), (192, 128, 64), (128, 64, 16), (8, 8, 32), (40, 256, 48)])
def test_padded_head_dims(fmha, d, dv, page):
    c = _case(11, [4], [75], [9, 70], 4, 2, d, torch.float16, page, dv=dv)
    o, lse = _run(fmha, c)
    _check(o, lse, *lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], d ** -0.5), torch.float16)


@pytest.mark.parametrize("sq", [1, 2])
@pytest.mark.parametrize("page", [16, 64])
def test_alibi_and_soft_cap(fmha, sq, page):
    c = _case(12, [3, 2], [66, 30], [4, 70], 4, 2, 128, torch.bfloat16, page, sq=sq)
    slopes = torch.tensor([0.25, 0.0625, 0.015625, 0.5])
    for kw in (dict(mask_type=2, window=(-1, 0)), dict(mask_type=2, window=(40, 0)), dict()):
        ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 128 ** -0.5, cap=3.0, slopes=slopes, **kw)
        o, lse = _run(fmha, c, alibi_slopes=dev(slopes), logits_soft_cap=3.0, **kw)
        # |score| reaches 70 with the slopes: an fp32 step there is 2^-17, and lse is of that size too
        assert (lse.double() - ref[1]).abs().max() <= 1e-4
        assert (o.double() - ref[0]).abs().max() <= (2 * U[torch.bfloat16] + 1e-4) * 6


def test_keys_behind_a_sequence_and_foreign_table_entries_do_not_matter(fmha):
    # unowned rows are NaN already; entries past a sequence's pages point anywhere valid, and the rows of sequences other than
    # the first need no entries for whole pages of the prefix
    c = _case(13, [3], [128], [1, 63, 64], 4, 1, 64, torch.bfloat16, 64)
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 0.125)
    nan_page = int((torch.isnan(c["kc"].float()).all(dim=3).all(dim=2).all(dim=1)).nonzero()[0])
    c["table"][1:, :2] = nan_page
    o, lse = _run(fmha, c)
    _check(o, lse, *ref, torch.bfloat16)


def test_same_result_as_the_decode_without_sharing(fmha):
    c = _case(14, [6], [300], [1, 20, 90], 8, 2, 128, torch.bfloat16, 128)
    o, lse = _run(fmha, c)
    i32 = lambda x: dev(torch.tensor(x, dtype=torch.int32))
    lse2 = dev(torch.empty_like(lse))
    o2 = fmha.fmha_decode_paged(dev(c["q"]), dev(c["kc"]), dev(c["vc"]), i32(c["lens"]), dev(c["table"]), num_splits=3, lse=lse2)
    torch.cuda.synchronize()
    assert (o.double() - o2.cpu().double()).abs().max() <= 4 * U[torch.bfloat16] * 6
    assert (lse - lse2.cpu()).abs().max() <= 4e-5


def test_results_are_the_same_every_time_and_with_a_kept_workspace(fmha):
    c = _case(15, [20], [150], [3, 64, 70], 8, 2, 128, torch.bfloat16, 64)
    first = _run(fmha, c)
    ws = fmha.DecodeWorkspace()
    for _ in range(3):
        again = _run(fmha, c, workspace=ws)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_without_an_lse(fmha):
    c = _case(16, [2], [20], [1], 4, 4, 64, torch.float16, 16)
    o, _ = _run(fmha, c, lse=False, cu_groups=None)
    assert (o.double() - lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 0.125)[0]).abs().max() <= 2 * U[torch.float16] * 6 + 1e-5


def _device_case(c):
    i32 = lambda x: dev(torch.tensor(x, dtype=torch.int32))
    return dict(q=dev(c["q"]), k_cache=dev(c["kc"]), v_cache=dev(c["vc"]), seqlen_k=i32(c["lens"]), block_table=dev(c["table"]),
                prefix_lens=i32(c["prefixes"]), cu_groups=i32(c["starts"]))


def test_captured_and_replayed(fmha):
    c = _case(17, [5, 3], [131, 40], [3, 64, 70], 8, 2, 128, torch.bfloat16, 64)
    t = _device_case(c)
    lse = torch.empty(8, 8, 1, device="cuda")
    out = torch.empty_like(t["q"])
    fmha.fmha_decode_shared_prefix(**t, out=out, lse=lse)   # warm: the launch opt-ins
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fmha.fmha_decode_shared_prefix(**t, out=out, lse=lse)
    g = torch.Generator().manual_seed(18)
    for step in range(4):
        t["q"].copy_(lc.randn(g, *t["q"].shape, dtype=torch.bfloat16))
        t["seqlen_k"].sub_(1)
        t["prefix_lens"].sub_(1)
        graph.replay()
        torch.cuda.synchronize()
        got, got_lse = out.clone(), lse.clone()
        eager_lse = torch.empty_like(lse)
        eager = fmha.fmha_decode_shared_prefix(**t, lse=eager_lse)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(got_lse, eager_lse), f"replay {step}"


def test_on_another_stream(fmha):
    # two calls at once on two streams, each with a workspace of its own, give what they give alone
    cases = [_case(19 + k, [6], [200], [3, 64, 70], 8, 2, 128, torch.bfloat16, 64) for k in range(2)]
    inputs = [_device_case(c) for c in cases]
    alone = [fmha.fmha_decode_shared_prefix(**t) for t in inputs]
    torch.cuda.synchronize()
    streams, spaces = [torch.cuda.Stream() for _ in range(2)], [fmha.DecodeWorkspace() for _ in range(2)]
    for _ in range(5):
        got = []
        for t, s, ws in zip(inputs, streams, spaces):
            with torch.cuda.stream(s):
                got.append(fmha.fmha_decode_shared_prefix(**t, workspace=ws))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(alone, got))


def test_long_cache_offsets(fmha):
    # pages that lie beyond 2^31 elements and 2^32 bytes of the pools
    c = _case(21, [3], [130], [5, 64], 8, 8, 128, torch.bfloat16, 128)
    pages = 17000   # x 128 x 8 x 128 elements = 2.2e9, 4.5 GB
    n = c["kc"].shape[0]
    kc = torch.zeros(pages, 128, 8, 128, dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    kc[pages - n:], vc[pages - n:] = dev(c["kc"]), dev(c["vc"])
    ref = lc.decode(c["q"], c["kc"], c["vc"], c["lens"], c["table"], 128 ** -0.5)
    t = _device_case(c)
    t.update(k_cache=kc, v_cache=vc, block_table=t["block_table"] + (pages - n))
    lse = torch.empty(3, 8, 1, device="cuda")
    o = fmha.fmha_decode_shared_prefix(**t, lse=lse)
    w = fmha.fmha_key_weights(t["q"], kc, lse, t["seqlen_k"], t["block_table"])
    kept_w, table = torch.rand_like(w), torch.arange(3, dtype=torch.int32, device="cuda").view(3, 1)
    _, kept, _ = fmha.fmha_cache_evict(kc, vc, kept_w, t["seqlen_k"], t["block_table"], table, budget=100)
    torch.cuda.synchronize()
    _check(o.cpu(), lse.cpu(), *ref, torch.bfloat16)
    assert (w.sum(dim=2).cpu() - 1.0).abs().max() <= 1e-4
    kept = kept.cpu()
    for h in (0, 7):
        for j in (0, 99):
            p = int(kept[2, h, j])
            assert torch.equal(kc[2, j, h].cpu(), c["kc"][c["table"][2, p // 128], p % 128, h])
            assert torch.equal(vc[2, j, h].cpu(), c["vc"][c["table"][2, p // 128], p % 128, h])

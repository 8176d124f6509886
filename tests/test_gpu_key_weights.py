"""GPU: the attention weight every cached key receives, against its definition in 64 bits.

Tolerance.  A weight is a sum of terms exp(s - lse) >= 0.  The score s is a sum of products of 16-bit values in fp32 (an error
below 2^-20 of the sum of their magnitudes, itself below 16 here), brought to base 2 in one fused step; lse is the fp32
input.  With |s|, |lse| < 16 the exponent is off by less than 16 * 2^-20 + 3 * 16 * 2^-24 < 2^-15.5 and the exponential
by a few 2^-24 more, so every term, and their sum in fp32, is within 2.5e-5 of its value."""
import pytest
import torch

import longcontext as lc
from helpers import dev

pytestmark = pytest.mark.gpu
REL = 2.5e-5


def _i32(x):
    return dev(torch.tensor(x, dtype=torch.int32))


def _case(seed, lens, sq, hq, hk, d, dtype, page, fp8=False, kd=1.0, starts=None, **kw):
    g = torch.Generator().manual_seed(seed)
    kc, vc, table = lc.pages(g, lens, page, hk, d, d, dtype, fp8)
    q = lc.randn(g, *((starts[-1],) if starts else (len(lens), sq)), hq, d, dtype=dtype)
    _, lse = lc.decode(q, kc, vc, lens, table, d ** -0.5, starts=starts, kd=kd, **kw)
    keys = [lc.rows(kc, table[b], n, page, kd) for b, n in enumerate(lens)]
    return dict(q=q, kc=kc, table=table, lens=lens, lse=lse.float(), keys=keys)


def _check(got, want, lens, what=""):
    got = got.cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    err = ((got.double() - want).abs() - REL * want).max().item()
    assert err <= 1e-9, f"{what}: off by {err:.3e} beyond the relative bound"
    for b, n in enumerate(lens):
        assert not got[b, :, n:].any(), f"{what}: weight behind the last key"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hk,d,page", [(8, 2, 64, 64), (8, 2, 128, 128), (4, 4, 128, 16), (8, 1, 256, 48), (6, 2, 128, 1),
                                          (4, 2, 72, 32), (2, 1, 8, 16)])
def test_one_token(fmha, dtype, hq, hk, d, page):
    lens = [1, 31, 32, 33, 130, 300, 0]
    c = _case(1, lens, 1, hq, hk, d, dtype, page)
    out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), max_seqlen_k=300)
    _check(out, lc.key_weights(c["q"], c["keys"], c["lse"], 300, d ** -0.5), lens)


@pytest.mark.parametrize("mask_type,window", [(0, (-1, -1)), (2, (-1, 0)), (2, (20, 0)), (2, (5, 3)), (1, (-1, 0)), (1, (9, 2))])
@pytest.mark.parametrize("sq,d,page", [(3, 64, 16), (17, 128, 64), (65, 128, 128), (40, 256, 48)])
def test_masks_and_query_runs(fmha, mask_type, window, sq, d, page):
    # bottom right with fewer keys than rows leaves rows that see nothing (lse = -inf)
    lens = [sq, sq + 70, max(1, sq - 2), 200]
    kw = dict(mask_type=mask_type, window=window)
    c = _case(2, lens, sq, 4, 2, d, torch.bfloat16, page, **kw)
    cols = max(lens) + 5
    out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), max_seqlen_k=cols, **kw)
    _check(out, lc.key_weights(c["q"], c["keys"], c["lse"], cols, d ** -0.5, **kw), lens, f"{kw}")


@pytest.mark.parametrize("sq", [1, 9])
def test_accumulates_and_grows(fmha, sq):
    # in place and out of place; fewer columns than keys, and more
    lens = [100, 37]
    c = _case(3, lens, sq, 8, 4, 128, torch.float16, 64)
    g = torch.Generator().manual_seed(4)
    for cols in (64, 100, 150):
        before = torch.rand(2, 4, cols, generator=g)
        want = lc.key_weights(c["q"], c["keys"], c["lse"], cols, 128 ** -0.5, before=before)
        args = (dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]))
        w = dev(before)
        out = fmha.fmha_key_weights(*args, weights=w)
        _check(out, want, lens, f"cols {cols}")
        assert torch.equal(w.cpu(), before)
        assert fmha.fmha_key_weights(*args, weights=w, out=w) is w
        assert torch.equal(w.cpu(), out.cpu())


def test_packed_queries(fmha):
    starts, lens = [0, 3, 3, 40, 41], [50, 9, 37, 130]
    kw = dict(mask_type=2, window=(-1, 0))
    c = _case(5, lens, 0, 8, 2, 64, torch.bfloat16, 16, starts=starts, **kw)
    out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), cu_seqlens_q=_i32(starts),
                                max_seqlen_q=37, max_seqlen_k=130, **kw)
    _check(out, lc.key_weights(c["q"], c["keys"], c["lse"], 130, 0.125, starts=starts, **kw), lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sq", [1, 35])
def test_quantised_keys(fmha, dtype, d, sq):
    lens = [70, 1, 129]
    c = _case(6, lens, sq, 4, 2, d, dtype, 16, fp8=True, kd=0.5)
    out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), max_seqlen_k=129, k_descale=0.5)
    _check(out, lc.key_weights(c["q"], c["keys"], c["lse"], 129, d ** -0.5), lens)


def test_alibi_and_soft_cap(fmha):
    # the cap keeps |score| below 3, the slopes add up to 75: errors of 2^-17 in the exponent
    lens, slopes = [150, 33], torch.tensor([0.25, 0.0625, 0.015625, 0.5])
    for sq, kw in ((1, dict()), (5, dict(mask_type=2, window=(-1, 0))), (33, dict(mask_type=2, window=(40, 0)))):
        c = _case(7, lens, sq, 4, 2, 128, torch.bfloat16, 64, cap=3.0, slopes=slopes, **kw)
        out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), max_seqlen_k=150,
                                    alibi_slopes=dev(slopes), logits_soft_cap=3.0, **kw).cpu()
        want = lc.key_weights(c["q"], c["keys"], c["lse"], 150, 128 ** -0.5, cap=3.0, slopes=slopes, **kw)
        assert ((out.double() - want).abs() - 1e-4 * want).max() <= 1e-9


def test_cache_without_pages(fmha):
    g = torch.Generator().manual_seed(8)
    k, q = lc.randn(g, 3, 90, 2, 128, dtype=torch.bfloat16), lc.randn(g, 3, 2, 4, 128, dtype=torch.bfloat16)
    for lens in (None, [90, 1, 40]):
        keys = [k[b, :n].double() for b, n in enumerate(lens or [90] * 3)]
        lse = torch.stack([torch.stack([lc.attention(q[b, :, h], keys[b][:, h // 2], keys[b][:, h // 2], 128 ** -0.5)[1] for h in range(4)])
                           for b in range(3)]).float()
        out = fmha.fmha_key_weights(dev(q), dev(k), dev(lse), None if lens is None else _i32(lens))
        _check(out, lc.key_weights(q, keys, lse, 90, 128 ** -0.5), lens or [90] * 3)


def test_weights_of_a_row_sum_to_one_and_values_the_mask_hides_do_not_matter(fmha):
    # an infinite key and a NaN key that no row sees, a NaN key that some rows see
    lens, sq = [140], 4
    kw = dict(mask_type=2, window=(30, 0))
    c = _case(9, lens, sq, 2, 1, 64, torch.bfloat16, 64, **kw)
    clean = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), **kw).cpu()
    assert abs(clean.double().sum().item() - 8.0) <= 8 * REL
    kc = c["kc"].clone()
    for t, x in ((3, float("inf")), (100, float("nan")), (139, float("nan"))):
        kc[c["table"][0, t // 64], t % 64] = x
    out = fmha.fmha_key_weights(dev(c["q"]), dev(kc), dev(c["lse"]), _i32(lens), dev(c["table"]), **kw).cpu()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[..., 139] = False
    assert torch.isnan(out[..., 139]).all() and torch.equal(out[keep], clean[keep])


def test_results_are_the_same_every_time(fmha):
    lens = [700, 513]
    kw = dict(mask_type=2, window=(-1, 0))
    c = _case(10, lens, 60, 8, 2, 128, torch.bfloat16, 128, **kw)
    args = (dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]))
    first = fmha.fmha_key_weights(*args, **kw).cpu()
    _check(first, lc.key_weights(c["q"], c["keys"], c["lse"], first.shape[2], 128 ** -0.5, **kw), lens)
    for _ in range(3):
        assert torch.equal(first, fmha.fmha_key_weights(*args, **kw).cpu())


@pytest.mark.parametrize("mask_type,window", [(0, (-1, -1)), (2, (-1, 0)), (2, (60, 5)), (1, (-1, 0))])
@pytest.mark.parametrize("sq,hq,hk,d,page", [(290, 2, 1, 64, 64), (290, 3, 3, 128, 16), (100, 3, 1, 128, 128), (70, 1, 1, 256, 48),
                                             (290, 2, 1, 72, 64)])
def test_long_query_runs(fmha, mask_type, window, sq, hq, hk, d, page):
    # more rows than LDS holds: stages that are full and not, runs that end inside a stage, keys that some waves do not have
    lens = [sq, 277]
    kw = dict(mask_type=mask_type, window=window)
    c = _case(11, lens, sq, hq, hk, d, torch.bfloat16, page, **kw)
    cols = max(lens) + 3
    want = lc.key_weights(c["q"], c["keys"], c["lse"], cols, d ** -0.5, **kw)
    before = torch.rand(2, hk, cols, generator=torch.Generator().manual_seed(1))
    for splits in (1, 3):
        out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), max_seqlen_k=cols,
                                    num_row_splits=splits, **kw)
        _check(out, want, lens, f"{kw} splits {splits}")
        w = dev(before)
        fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), weights=w, out=w,
                              num_row_splits=splits, **kw)
        want_w = want.clone()
        for b, n in enumerate(lens):
            want_w[b, :, :n] += before[b, :, :n].double()
        _check(w, want_w, lens, f"{kw} splits {splits} in place")


def test_long_packed_quantised_and_modified_runs(fmha):
    starts, lens, slopes = [0, 270, 271], [300, 40], torch.tensor([0.25, 0.0625])
    kw = dict(mask_type=2, window=(-1, 0))
    c = _case(12, lens, 0, 2, 1, 64, torch.float16, 16, fp8=True, kd=0.5, starts=starts, **kw)
    out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), cu_seqlens_q=_i32(starts),
                                max_seqlen_q=270, max_seqlen_k=300, k_descale=0.5, num_row_splits=2, **kw)
    _check(out, lc.key_weights(c["q"], c["keys"], c["lse"], 300, 0.125, starts=starts, **kw), lens)
    c = _case(13, lens, 0, 2, 1, 64, torch.bfloat16, 64, starts=starts, cap=3.0, slopes=slopes, **kw)
    out = fmha.fmha_key_weights(dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]), cu_seqlens_q=_i32(starts),
                                max_seqlen_q=270, max_seqlen_k=300, alibi_slopes=dev(slopes), logits_soft_cap=3.0, **kw).cpu()
    want = lc.key_weights(c["q"], c["keys"], c["lse"], 300, 0.125, starts=starts, cap=3.0, slopes=slopes, **kw)
    assert ((out.double() - want).abs() - 2e-4 * want).max() <= 1e-9  # the slopes add up to 75: fp32 steps of 2^-17 there


@pytest.mark.parametrize("sq,hq,splits", [(1, 8, 1), (60, 4, 1), (300, 4, 2)])
def test_captured_and_replayed(fmha, sq, hq, splits):
    lens, kw = [400, 330], dict(mask_type=2, window=(-1, 0))
    c = _case(14, lens, sq, hq, 2, 128, torch.bfloat16, 64, **kw)
    q, lse, n, w = dev(c["q"]), dev(c["lse"]), _i32(lens), torch.zeros(2, 2, 400, device="cuda")
    args = (q, dev(c["kc"]), lse, n, dev(c["table"]))
    kw["num_row_splits"] = splits
    out = torch.empty_like(w)
    fmha.fmha_key_weights(*args, weights=w, out=out, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fmha.fmha_key_weights(*args, weights=w, out=out, **kw)
    for step in range(4):
        q.mul_(0.9)
        n.sub_(3)
        w.copy_(torch.rand_like(w))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, fmha.fmha_key_weights(*args, weights=w, **kw)), f"replay {step}"


def test_on_another_stream(fmha):
    lens, kw = [500, 444], dict(mask_type=2, window=(-1, 0))
    c = _case(15, lens, 300, 4, 2, 128, torch.bfloat16, 64, **kw)
    args = (dev(c["q"]), dev(c["kc"]), dev(c["lse"]), _i32(lens), dev(c["table"]))
    alone = fmha.fmha_key_weights(*args, num_row_splits=2, **kw)
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s in (torch.cuda.Stream(), torch.cuda.Stream()):
            with torch.cuda.stream(s):
                got.append(fmha.fmha_key_weights(*args, num_row_splits=2, **kw))
        torch.cuda.synchronize()
        assert all(torch.equal(alone, x) for x in got)

"""GPU: the log-sum-exp outputs of the forward operators against the definition in 64 bits (fp32 statistics throughout:
2e-5 absolute for |lse| < 16), and outputs that do not change when one is asked for."""
import pytest
import torch

import longcontext as lc
from helpers import dev

pytestmark = pytest.mark.gpu


def _i32(x):
    return dev(torch.tensor(x, dtype=torch.int32))


def _close(got, want):
    got = got.cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    fin = torch.isfinite(want)
    assert (got.double() - want)[fin].abs().max() <= 2e-5


def _ref(q, k, v, **kw):
    hq, hk = q.shape[-2], k.shape[-2]
    return torch.stack([torch.stack([lc.attention(q[b, :, h], k[b][:, h * hk // hq].double(), v[b][:, h * hk // hq].double(), q.shape[-1] ** -0.5, **kw)[1]
                                     for h in range(hq)]) for b in range(q.shape[0])])


@pytest.mark.parametrize("mask", [dict(), dict(mask_type=2, window=(-1, 0)), dict(mask_type=2, window=(9, 0))])
@pytest.mark.parametrize("sq,sk,d", [(5, 70, 64), (140, 100, 128), (33, 65, 256), (20, 64, 72)])
def test_dense(fmha, mask, sq, sk, d):
    g = torch.Generator().manual_seed(1)
    q, k, v = (lc.randn(g, 2, n, h, d, dtype=torch.bfloat16) for n, h in ((sq, 4), (sk, 2), (sk, 2)))
    lse = dev(torch.zeros(2, 4, sq))
    o = fmha.fmha_fwd(dev(q), dev(k), dev(v), lse=lse, **mask)
    plain = fmha.fmha_fwd(dev(q), dev(k), dev(v), **mask)
    torch.cuda.synchronize()
    _close(lse, _ref(q, k, v, **mask))
    assert torch.equal(o.cpu(), plain.cpu())


@pytest.mark.parametrize("d,page", [(64, 64), (128, 16), (256, 64)])
def test_packed_over_pages(fmha, d, page):
    g = torch.Generator().manual_seed(2)
    starts, lens = [0, 3, 140, 141], [3, 170, 40]
    mask = dict(mask_type=2, window=(-1, 0))
    kc, vc, table = lc.pages(g, lens, page, 2, d, d, torch.bfloat16)
    q = lc.randn(g, starts[-1], 4, d, dtype=torch.bfloat16)
    _, want = lc.decode(q, kc, vc, lens, table, d ** -0.5, starts=starts, **mask)
    lse = dev(torch.zeros(4, starts[-1]))
    fmha.fmha_fwd_pagedkv(dev(q), dev(kc), dev(vc), _i32(lens), dev(table), cu_seqlens_q=_i32(starts), max_seqlen_q=137, lse=lse, **mask)
    torch.cuda.synchronize()
    _close(lse, want)
    counts = [-(-n // page) for n in lens]
    indptr = [sum(counts[:b]) for b in range(4)]
    ids = [int(table[b, j]) for b, c in enumerate(counts) for j in range(c)]
    lse.zero_()
    fmha.fmha_batch_prefill(dev(q), dev(kc), dev(vc), _i32(starts), _i32(indptr), _i32(ids), _i32([(n - 1) % page + 1 for n in lens]),
                            max_seqlen_q=137, lse=lse)
    torch.cuda.synchronize()
    _close(lse, want)


def test_varlen_and_quantised(fmha):
    g = torch.Generator().manual_seed(3)
    starts, kstarts = [0, 7, 50], [0, 30, 130]
    q, k, v = (lc.randn(g, n, h, 64, dtype=torch.float16) for n, h in ((50, 4), (130, 2), (130, 2)))
    lse = dev(torch.zeros(4, 50))
    fmha.fmha_fwd_varlen(dev(q), dev(k), dev(v), _i32(starts), _i32(kstarts), 43, lse=lse)
    torch.cuda.synchronize()
    for b in range(2):
        want = _ref(q[None, starts[b]:starts[b + 1]], k[None, kstarts[b]:kstarts[b + 1]], v[None, kstarts[b]:kstarts[b + 1]])
        _close(lse[:, starts[b]:starts[b + 1]], want[0])
    lens = [60, 17]
    kc, vc, table = lc.pages(g, lens, 16, 2, 64, 64, torch.float16, fp8=True)
    q = lc.randn(g, 2, 5, 4, 64, dtype=torch.float16)
    lse = dev(torch.zeros(2, 4, 5))
    fmha.fmha_fwd_pagedkv(dev(q), dev(kc), dev(vc), _i32(lens), dev(table), k_descale=0.5, lse=lse)
    torch.cuda.synchronize()
    _close(lse, lc.decode(q, kc, vc, lens, table, 0.125, kd=0.5, mask_type=2, window=(-1, 0))[1])  # the operator's default mask


@pytest.mark.parametrize("num_splits", [1, 3, 20])
def test_decode(fmha, num_splits):
    g = torch.Generator().manual_seed(4)
    lens = [1, 200, 77, 0]
    kc, vc, table = lc.pages(g, lens, 64, 2, 128, 128, torch.bfloat16)
    q = lc.randn(g, 4, 2, 8, 128, dtype=torch.bfloat16)
    lse = dev(torch.zeros(4, 8, 2))
    args = (dev(q), dev(kc), dev(vc), _i32(lens), dev(table))
    o = fmha.fmha_decode_paged(*args, num_splits=num_splits, lse=lse)
    plain = fmha.fmha_decode_paged(*args, num_splits=num_splits)
    torch.cuda.synchronize()
    _close(lse, lc.decode(q, kc, vc, lens, table, 128 ** -0.5)[1])
    assert torch.equal(o.cpu(), plain.cpu())
    with pytest.raises(NotImplementedError):
        fmha.fmha_decode_paged(*args, num_splits=num_splits, lse=lse, fused=True)

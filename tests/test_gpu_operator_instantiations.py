"""GPU: one small problem for every kernel instantiation a call of the operators on long shared caches can reach (data type, head
dim, row blocks, keys per wave, page addressing, modifiers, quantised caches, padded head dims, merge width), and the long
rows of the eviction.  tests/emu/kernel_coverage.py measures the outcome.

Tolerances are those of test_gpu_key_weights and test_gpu_shared_prefix, derived there; with a soft cap of 3 every |score| is
below 3, so they hold with modifiers as well."""
import pytest
import torch

import longcontext as lc
import test_gpu_cache_evict as evict
from helpers import dev

pytestmark = pytest.mark.gpu
REL = 2.5e-5
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.bfloat16, torch.float16]
FLAGS = ["plain", "mod", "pad", "kv8"]


def _i32(x):
    return dev(torch.tensor(x, dtype=torch.int32))


def _copies(x, n):
    """The first dimension repeated until it has n entries."""
    return x.repeat(-(-n // x.shape[0]), *[1] * (x.dim() - 1))[:n].contiguous()


def _shared(fmha, seed, sizes, prefixes, own, sq, hq, hk, d, dtype, page, flags):
    g = torch.Generator().manual_seed(seed)
    dk, dv = (d - 8, d - 16) if flags == "pad" else (d, d)
    fp8 = flags == "kv8"
    starts = [0]
    for s in sizes:
        starts.append(starts[-1] + s)
    lens = [prefixes[k] + own[(starts[k] + i) % len(own)] for k, s in enumerate(sizes) for i in range(s)]
    kc, vc, table = lc.pages(g, lens, page, hk, dk, dv, dtype, fp8)
    lc.share(kc, vc, table, starts, prefixes, page)
    q = lc.randn(g, len(lens), sq, hq, dk, dtype=dtype)
    kw = dict(mask_type=2, window=(-1, 0))
    if flags == "mod":
        kw["cap"] = 3.0
    ref, ref_lse = lc.decode(q, kc, vc, lens, table, dk ** -0.5, kd=0.5, vd=0.25, **kw)
    cap = kw.pop("cap", 0.0)
    lse = dev(torch.zeros(len(lens), hq, sq))
    if fp8:
        kw.update(k_descale=0.5, v_descale=0.25)
    o = fmha.fmha_decode_shared_prefix(dev(q), dev(kc), dev(vc), _i32(lens), dev(table), _i32(prefixes), cu_groups=_i32(starts), lse=lse,
                                       num_prefix_splits=2, num_splits=2, max_group_size=max(sizes), logits_soft_cap=cap, **kw).cpu()
    assert torch.isfinite(o.float()).all()
    assert (o.double() - ref).abs().max() <= (2 * U[dtype] + 2.0 ** -20) * 6.0
    assert torch.equal(torch.isinf(lse.cpu()), torch.isinf(ref_lse))
    fin = torch.isfinite(ref_lse)
    assert (lse.cpu().double() - ref_lse)[fin].abs().max() <= 2e-5


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("page", [64, 16])
@pytest.mark.parametrize("rows", [40, 160])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16"])
def test_shared_prefix(fmha, dtype, d, rows, page, flags):
    # a group of `rows` packed rows (more than 128: two row blocks per wave at head dims up to 128) and a small one
    _shared(fmha, rows + d + page, [5, 2], [150, 40], [9, 70, 3, 64], rows // 20, 8, 2, d, dtype, page, flags)


@pytest.mark.parametrize("flags", ["plain", "pad"])
@pytest.mark.parametrize("d,hq", [(64, 128), (128, 64), (256, 32)])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16"])
def test_merge_of_many_rows(fmha, dtype, d, hq, flags):
    # enough rows that the merge takes workgroups of 256 threads; sequences 2.. are copies of the first two
    g = torch.Generator().manual_seed(d)
    batch, lens, dk, dv = 128, [33, 70], d, d - 16 if flags == "pad" else d
    kc, vc, table = lc.pages(g, lens, 64, 1, dk, dv, dtype)
    q = lc.randn(g, 2, 1, hq, dk, dtype=dtype)
    ref, ref_lse = lc.decode(q, kc, vc, lens, table, dk ** -0.5)
    lse = dev(torch.zeros(batch, hq, 1))
    o = fmha.fmha_decode_shared_prefix(dev(_copies(q, batch)), dev(kc), dev(vc), dev(_copies(torch.tensor(lens, dtype=torch.int32), batch)),
                                       dev(_copies(table, batch)), _i32([0]), lse=lse, num_prefix_splits=1, num_splits=2).cpu()
    assert (o.double() - _copies(ref, batch)).abs().max() <= (2 * U[dtype] + 2.0 ** -20) * 6.0
    assert (lse.cpu().double() - _copies(ref_lse, batch)).abs().max() <= 2e-5


def _key_weights(fmha, seed, batch, lens, sq, hq, hk, d, dtype, page, flags, **call):
    g = torch.Generator().manual_seed(seed)
    dk, fp8 = (d - 8 if flags == "pad" else d), flags == "kv8"
    kc, _, table = lc.pages(g, lens, page, hk, dk, dk, dtype, fp8)
    q = lc.randn(g, len(lens), sq, hq, dk, dtype=dtype)
    cap = dict(cap=3.0) if flags == "mod" else {}
    keys = [lc.rows(kc, table[b], n, page, 0.5) for b, n in enumerate(lens)]
    _, lse = lc.decode(q, kc, torch.zeros_like(kc), lens, table, dk ** -0.5, kd=0.5, **cap)
    cols = max(lens) + 3
    want = _copies(lc.key_weights(q, keys, lse.float(), cols, dk ** -0.5, **cap), batch)
    out = fmha.fmha_key_weights(dev(_copies(q, batch)), dev(kc), dev(_copies(lse.float(), batch)),
                                dev(_copies(torch.tensor(lens, dtype=torch.int32), batch)), dev(_copies(table, batch)), max_seqlen_k=cols,
                                k_descale=0.5 if fp8 else 1.0, logits_soft_cap=cap.get("cap", 0.0), **call).cpu()
    assert torch.isfinite(out).all()
    assert ((out.double() - want).abs() - REL * want).max() <= 1e-9


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("tiles", [2, 8])
@pytest.mark.parametrize("g", [4, 24])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16"])
def test_key_weights_of_a_step(fmha, dtype, d, g, tiles, flags):
    # one or two blocks of rows; two or (with many sequences) eight tiles of keys per wave
    batch, hk = (64, 8) if tiles == 8 else (2, 2)
    _key_weights(fmha, d + g + tiles, batch, [300, 37], 1, g * hk, hk, d, dtype, 64 if g == 4 else 16, flags)


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16"])
def test_key_weights_of_a_window(fmha, dtype, d, flags):
    _key_weights(fmha, d, 2, [300, 37], 17, 8, 2, d, dtype, 48, flags)


@pytest.mark.parametrize("flags", FLAGS)
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "fp16"])
def test_key_weights_of_a_prompt(fmha, dtype, d, splits, flags):
    # more rows than LDS holds, and enough that two whole pairs of row blocks follow each other
    _key_weights(fmha, d + splits, 1, [300], {64: 140, 128: 75, 256: 70}[d], 4, 1, d, dtype, 64, flags, num_row_splits=splits)


@pytest.mark.parametrize("n,cols", [(20000, 20000), (33000, 65536), (70001, 70001), (140000, 140000), (140000, 131072)])
def test_eviction_of_long_rows(fmha, n, cols):
    # one workgroup and several per row, with parts of a wave shorter and longer than the 1024 weights it walks at once; equal weights that
    # lie in the parts of several workgroups
    evict._run(fmha, n, [n], 1, 8, torch.bfloat16, 64, 3000, recent=100, sinks=7, cols=cols, own_pool=True)
    w = torch.randint(0, 3, (1, 1, cols), generator=torch.Generator().manual_seed(n)).float()
    evict._run(fmha, n + 1, [n], 1, 8, torch.bfloat16, 64, n // 2, weights=w, cols=cols, own_pool=True)

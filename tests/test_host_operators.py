"""Refusals of the operators on long shared caches: nothing is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from flashck_amd import _lib
from flashck_amd.nn import PagedAttention
from flashck_amd.ops import fmha
from flashck_amd.ops.fmha import fmha as F


@pytest.fixture
def ops(monkeypatch):
    """The Python layer with host tensors; a call that gets as far as the library is recorded instead of made."""
    calls = []
    monkeypatch.setattr(F, "_REQUIRE_GPU_TENSORS", False)
    monkeypatch.setattr(F, "_stream", lambda: None)
    monkeypatch.setattr(F, "_call", lambda name, *args: calls.append(name))
    monkeypatch.setattr(F, "_shared_prefix_splits", lambda *a: (2, 2))
    monkeypatch.setattr(F, "_key_weights_row_splits", lambda *a: 1)
    monkeypatch.setattr(F, "_evict_workspace_bytes", lambda *a: 0)
    return calls


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def _shared(**kw):
    a = dict(q=torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16),
             v_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), seqlen_k=_i32(20, 17), block_table=torch.zeros(2, 2, dtype=torch.int32),
             prefix_lens=_i32(16))
    a.update(kw)
    return F.fmha_decode_shared_prefix(**a)


@pytest.mark.parametrize("kw,error", [
    (dict(q=torch.zeros(2, 1, 4, 64)), TypeError),
    (dict(q=torch.zeros(2, 1, 4, 64).to(torch.float8_e4m3fn)), TypeError),
    (dict(q=torch.zeros(3, 1, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 0, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16)[..., ::2]), ValueError),
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.float16)), TypeError),
    (dict(v_cache=torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(seqlen_k=torch.tensor([20, 17])), TypeError),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32)), ValueError),
    (dict(block_table=torch.zeros(2, 0, dtype=torch.int32)), ValueError),
    (dict(prefix_lens=_i32(16, 3)), ValueError),
    (dict(prefix_lens=_i32(16, 3), cu_groups=_i32(0, 2)), ValueError),
    (dict(prefix_lens=torch.zeros(0, dtype=torch.int32), cu_groups=_i32(0)), ValueError),
    (dict(cu_seqlens_q=_i32(0, 1, 2), q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), ValueError),
    (dict(lse=torch.zeros(2, 4, 2)), ValueError),
    (dict(lse=torch.zeros(2, 4, 1, dtype=torch.bfloat16)), TypeError),
    (dict(out=torch.zeros(2, 1, 4, 32, dtype=torch.bfloat16)), ValueError),
    (dict(alibi_slopes=torch.zeros(3)), ValueError),
    (dict(logits_soft_cap=float("inf")), ValueError),
])
def test_shared_prefix_arguments(ops, kw, error):
    with pytest.raises(error):
        _shared(**kw)
    assert ops == []


def test_shared_prefix_reaches_the_library(ops):
    assert _shared().shape == (2, 1, 4, 64) and ops == ["fck_fmha_decode_shared_prefix"]


def _weights(**kw):
    a = dict(q=torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16),
             lse=torch.zeros(2, 4, 1), seqlen_k=_i32(20, 17), block_table=torch.zeros(2, 2, dtype=torch.int32))
    a.update(kw)
    return F.fmha_key_weights(**a)


@pytest.mark.parametrize("kw,error", [
    (dict(lse=torch.zeros(2, 4, 2)), ValueError),
    (dict(lse=torch.zeros(2, 4, 1, dtype=torch.float64)), TypeError),
    (dict(seqlen_k=None), ValueError),
    (dict(block_table=None), ValueError),
    (dict(k_cache=torch.zeros(4, 16, 2, 32, dtype=torch.bfloat16)), ValueError),
    (dict(k_cache=None), TypeError),
    (dict(weights=torch.zeros(2, 4, 32)), ValueError),
    (dict(weights=torch.zeros(2, 2, 0)), ValueError),
    (dict(weights=torch.zeros(2, 2, 32), out=torch.zeros(2, 2, 33)), ValueError),
    (dict(out=torch.zeros(2, 2, 32, dtype=torch.bfloat16)), TypeError),
    (dict(k_cache=torch.zeros(4, 16, 2, 64).to(torch.float8_e4m3fn), k_descale=0.0), ValueError),
])
def test_key_weights_arguments(ops, kw, error):
    with pytest.raises(error):
        _weights(**kw)
    assert ops == []


def test_key_weights_columns(ops):
    assert _weights().shape == (2, 2, 32)
    assert _weights(max_seqlen_k=20).shape == (2, 2, 20)
    assert _weights(out=torch.zeros(2, 2, 25)).shape == (2, 2, 25)
    assert ops == ["fck_fmha_key_weights"] * 3


def _evict(**kw):
    a = dict(k_cache=torch.zeros(8, 16, 2, 64, dtype=torch.bfloat16), v_cache=torch.zeros(8, 16, 2, 32, dtype=torch.bfloat16),
             weights=torch.zeros(2, 2, 32), seqlen_k=_i32(20, 17), block_table=torch.zeros(2, 2, dtype=torch.int32),
             new_block_table=torch.ones(2, 1, dtype=torch.int32), budget=16)
    a.update(kw)
    return F.fmha_cache_evict(**a)


@pytest.mark.parametrize("kw,error", [
    (dict(budget=0), ValueError), (dict(budget=17), ValueError), (dict(recent=-1), ValueError), (dict(sinks=-1), ValueError),
    (dict(recent=10, sinks=7), ValueError), (dict(weights=torch.zeros(2, 3, 32)), ValueError),
    (dict(weights=torch.zeros(2, 2, 32, dtype=torch.float16)), TypeError), (dict(k_cache=torch.zeros(8, 16, 2, 64)), TypeError),
    (dict(v_cache=torch.zeros(8, 16, 2, 64, dtype=torch.float16)), TypeError), (dict(v_cache=torch.zeros(8, 8, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(new_block_table=torch.ones(3, 1, dtype=torch.int32)), ValueError), (dict(new_block_table=torch.ones(2, 1)), TypeError),
    (dict(new_k_cache=torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(new_k_cache=torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16), new_v_cache=torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(out_kept=torch.zeros(2, 2, 15, dtype=torch.int32)), ValueError), (dict(out_weights=torch.zeros(2, 2, 31)), ValueError),
])
def test_evict_arguments(ops, kw, error):
    with pytest.raises(error):
        _evict(**kw)
    assert ops == []


def test_evict_refuses_to_write_what_it_reads(ops):
    table, w, n = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2, 32), _i32(20, 17)
    for kw in (dict(block_table=table, new_block_table=table), dict(weights=w, out_weights=w), dict(seqlen_k=n, out_seqlen=n)):
        with pytest.raises(ValueError):
            _evict(**kw)
    assert ops == []
    _evict(block_table=table, new_block_table=table, new_k_cache=torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16),
           new_v_cache=torch.zeros(2, 16, 2, 32, dtype=torch.bfloat16))
    assert ops == ["fck_fmha_cache_evict"]


def test_debug_flag_checks_the_pages_an_eviction_writes(ops):
    old = _i32(0, 1, 2, 3).view(2, 2)
    k = torch.zeros(8, 16, 2, 64)
    F._validate_new_pages(_i32(20, 17), old, _i32(4, 5).view(2, 1), 16, 16, k, True)
    for new in ((4, 4), (4, 8), (4, -1), (4, 3)):
        with pytest.raises(ValueError):
            F._validate_new_pages(_i32(20, 17), old, _i32(*new).view(2, 1), 16, 16, k, True)
    F._validate_new_pages(_i32(20, 17), old, _i32(4, 3).view(2, 1), 16, 16, k, False)   # a pool of its own
    F._validate_new_pages(_i32(20, 0), old, _i32(4, 99).view(2, 1), 16, 16, k, True)    # an empty sequence writes no page
    F._validate_new_pages(_i32(20, -40), old, _i32(4, 99).view(2, 1), 16, 16, k, True)  # nor does one of negative length


def test_the_step_and_the_module_reach_the_operators(ops, monkeypatch):
    m = PagedAttention(4, 2, 64, 64)
    q, new = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 1, 2, 64, dtype=torch.bfloat16)
    kc = torch.zeros(8, 16, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 2, dtype=torch.int32)
    lse = torch.zeros(2, 4, 1)
    o, n = m.decode_step(q, new, new, kc, kc.clone(), _i32(20, 17), table, prefix_lens=_i32(16), lse=lse)
    assert n.tolist() == [21, 18] and o.shape == q.shape
    m.key_weights(q, kc, lse, n, table)
    m.evict(kc, kc.clone(), torch.zeros(2, 2, 32), n, table, torch.ones(2, 1, dtype=torch.int32), budget=16)
    assert ops == ["fck_fmha_fwd_appendkv", "fck_fmha_decode_shared_prefix", "fck_fmha_key_weights", "fck_fmha_cache_evict"]
    with pytest.raises(ValueError):
        PagedAttention(4, 2, 64, 64, window_left=8).evict(kc, kc, torch.zeros(2, 2, 32), n, table, table, budget=16)


def test_registered():
    from flashck_amd.utils import FlashCKOperationType
    from flashck_amd.utils.registry import get_flashck_functions
    fns = get_flashck_functions(FlashCKOperationType.FMHA.value)
    for name in ("decode_shared_prefix", "key_weights", "cache_evict"):
        assert callable(fns[name])


# ---- the C ABI: errors before any launch -------------------------------------------------------------------------------------

P = ctypes.c_void_p(1 << 20)   # an aligned address that is never read


def _abi_shared(**kw):
    a = dict(q=P, k=P, v=P, o=P, lse=None, lse_acc=P, o_acc=P, sq_start=None, sk=P, bt=P, cu=None, pl=P, batch=2, groups=1, gmax=0, sq=1,
             hq=4, hk=2, d=64, dv=64, qmax=1, nsp=1, nso=1, maxp=0, maxo=0, stride=2, page=16, scale=0.1, wl=-1, wr=-1, mask=0, dtype=4,
             attrs=None, stream=None)
    a.update(kw)
    return _lib.load().fck_fmha_decode_shared_prefix(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), -1), (dict(pl=None), -1), (dict(o_acc=ctypes.c_void_p(8)), -1), (dict(hq=3), -1), (dict(d=12), -2), (dict(d=264), -2),
    (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(mask=4), -1), (dict(dtype=1), -2), (dict(dtype=7), -2), (dict(groups=0), -1),
    (dict(groups=2), -1), (dict(nsp=0), -1), (dict(nso=65), -1), (dict(page=0), -1), (dict(stride=0), -1), (dict(sq=0), -1),
    (dict(batch=1 << 40), -1), (dict(sq=1 << 31, batch=2), -1),
])
def test_abi_shared_prefix(kw, rc):
    assert _abi_shared(**kw) == rc


def test_abi_attributes_that_do_not_apply():
    at = _lib.Attrs()
    at.size = ctypes.sizeof(_lib.Attrs)
    for field, value, rc in (("decode_variant", 1, -1), ("prefill_variant", 1, -1), ("o_scale", 2.0, -1), ("lse", 1 << 20, -1), ("kv_dtype", 3, -2)):
        at = _lib.Attrs()
        at.size = ctypes.sizeof(_lib.Attrs)
        setattr(at, field, value)
        assert _abi_shared(attrs=ctypes.byref(at)) == rc, field
    at = _lib.Attrs()
    at.size = ctypes.sizeof(_lib.Attrs)
    at.bias_type, at.bias, at.bias_row_stride = 1, 1 << 20, 64
    assert _abi_shared(attrs=ctypes.byref(at)) == -2
    at = _lib.Attrs()
    at.size = ctypes.sizeof(_lib.Attrs) - 4
    assert _abi_shared(attrs=ctypes.byref(at)) == -1


def _abi_weights(**kw):
    a = dict(q=P, k=P, lse=P, w=None, out=P, ws=None, sq_start=None, sk=P, bt=P, stride=2, page=16, batch=2, sq=1, skc=0, cols=32, hq=4, hk=2,
             d=64, qmax=1, ns=1, scale=0.1, wl=-1, wr=-1, mask=0, dtype=4, attrs=None, stream=None)
    a.update(kw)
    return _lib.load().fck_fmha_key_weights(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), -1), (dict(lse=None), -1), (dict(out=None), -1), (dict(cols=0), -1), (dict(ns=0), -1), (dict(ns=17), -1), (dict(ns=2), -1),
    (dict(bt=None), -1), (dict(sk=None), -1), (dict(dtype=1), -2), (dict(d=4), -2), (dict(sq=0), -1), (dict(cols=1 << 31), -1), (dict(scale=-1.0), -1),
])
def test_abi_key_weights(kw, rc):
    assert _abi_weights(**kw) == rc


def _abi_evict(**kw):
    a = dict(k=P, v=P, nk=P, nv=P, w=P, nw=ctypes.c_void_p(1 << 21), ws=None, sk=P, nsk=ctypes.c_void_p(1 << 22), kept=P, bt=P, stride=2, page=16, nbt=ctypes.c_void_p(1 << 21),
             nstride=1, npage=16, batch=2, hk=2, d=64, dv=64, cols=32, budget=16, recent=0, sinks=0, dtype=4, stream=None)
    a.update(kw)
    return _lib.load().fck_fmha_cache_evict(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(k=None), -1), (dict(kept=None), -1), (dict(nk=ctypes.c_void_p(8)), -1), (dict(budget=0), -1), (dict(budget=17), -1), (dict(recent=17), -1),
    (dict(recent=9, sinks=8), -1), (dict(sinks=-1), -1), (dict(dtype=0), -2), (dict(d=10), -2), (dict(dv=512), -2), (dict(nbt=P), -1), (dict(nw=P), -1),
    (dict(ws=ctypes.c_void_p(8)), -1), (dict(nsk=P), -1),
    (dict(cols=0), -1), (dict(npage=0), -1), (dict(batch=1 << 30, hk=4), -1),
])
def test_abi_evict(kw, rc):
    assert _abi_evict(**kw) == rc


def test_abi_splits_of_any_sizes():
    lib = _lib.load()
    a, b = ctypes.c_int32(), ctypes.c_int32()
    for sizes in ((1, 1, 1, 1, 1, 1, 64, 1, 1, 256), (64, 1, 64, 64, 8, 1, 128, 32768, 512, 256), (1 << 40, 1, 1, 1, 1, 1, 64, 1, 1, 256),
                  (4, 2, 3, 8, 2, 1, 256, 0, 0, 256), (0, 0, 0, 0, 0, 0, 0, 0, 0, 0), (96, 1, 96, 16, 16, 5, 64, 1 << 30, 1 << 30, 256)):
        assert lib.fck_fmha_shared_prefix_splits(*sizes, ctypes.byref(a), ctypes.byref(b)) == 0
        assert 1 <= a.value <= 64 and 1 <= b.value <= 64, sizes
    for sizes in ((1, 32, 8, 8192, 8192, 128), (1, 8, 8, 1, 1, 64), (1 << 24, 1, 1, 1 << 30, 1 << 30, 256), (0, 0, 0, 0, 0, 0)):
        for mask in (0, 2):
            assert 1 <= lib.fck_fmha_key_weights_row_splits(*sizes, mask, 256) <= 16, sizes


def test_callers_of_the_shorter_attribute_struct_are_served():
    """fck_fmha_attrs grew by its lse fields: a caller with the earlier size gets the same checks as before."""
    lib = _lib.load()
    old = _lib.Attrs.lse.offset
    at = _lib.Attrs()
    at.size, at.logits_soft_cap = old, -1.0
    args = [P, P, P, None, P, None, None, None, 2, 4, 4, 4, 2, 64, 64, 4, 0.1, -1, -1, 0, 4, ctypes.byref(at), None]
    assert lib.fck_fmha_fwd_attrs(*args) == -1 and b"soft_cap" in lib.fck_last_error()
    at.size = old - 8
    assert lib.fck_fmha_fwd_attrs(*args) == -1 and b"size" in lib.fck_last_error()

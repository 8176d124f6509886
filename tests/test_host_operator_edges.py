"""Refusals and host-side choices of the operators on long shared caches: nothing is launched (no GPU needed)."""
import ctypes

import pytest
import torch

from flashck_amd import _lib
from flashck_amd.ops.fmha import fmha as F


def _at(n):
    return ctypes.c_void_p(n << 20)   # an aligned address that is never read


def _abi_evict(**kw):
    a = dict(k=_at(1), v=_at(2), nk=_at(3), nv=_at(4), w=_at(5), nw=_at(6), ws=None, sk=_at(7), nsk=_at(8), kept=_at(9), bt=_at(10), stride=2, page=16,
             nbt=_at(11), nstride=1, npage=16, batch=2, hk=2, d=64, dv=64, cols=32, budget=16, recent=0, sinks=0, dtype=4, stream=None)
    a.update(kw)
    return _lib.load().fck_fmha_cache_evict(*a.values())


@pytest.mark.parametrize("shared", [dict(nk=_at(1)), dict(nv=_at(2)), dict(nk=_at(1), nv=_at(2))])
def test_abi_eviction_refuses_its_own_table_over_a_pool_it_reads(shared):
    assert _abi_evict(nbt=_at(10), **shared) == -1
    assert b"other pages" in _lib.load().fck_last_error()


@pytest.mark.parametrize("sizes", [dict(budget=1 << 27, d=256, dv=256), dict(budget=1 << 30, dtype=1, d=8, dv=8, hk=8),
                                   dict(budget=1 << 20, batch=1 << 16, hk=16)])
def test_abi_eviction_refuses_what_it_cannot_move_before_it_chooses(sizes):
    # a refusal after the choice would leave kept positions and lengths written and no row moved
    assert _abi_evict(npage=1 << 10, nstride=1 << 21, cols=1 << 20, **sizes) == -1
    assert b"one move" in _lib.load().fck_last_error()


def test_abi_eviction_refuses_rows_beyond_its_counters():
    assert _abi_evict(budget=(1 << 31) - 1, dtype=1, d=8, dv=8, hk=1, batch=1, npage=1 << 10, nstride=1 << 21) == -2
    assert _abi_evict(stride=(1 << 20) + 1, page=1 << 10) == -2


def _abi_shared(**kw):
    a = dict(q=_at(1), k=_at(2), v=_at(3), o=_at(4), lse=None, lse_acc=_at(5), o_acc=_at(6), sq_start=_at(7), sk=_at(8), bt=_at(9), cu=_at(10), pl=_at(11),
             batch=2, groups=1, gmax=0, sq=2, hq=4, hk=2, d=64, dv=64, qmax=1, nsp=1, nso=1, maxp=0, maxo=0, stride=2, page=16, scale=0.1, wl=-1,
             wr=-1, mask=0, dtype=4, attrs=None, stream=None)
    a.update(kw)
    return _lib.load().fck_fmha_decode_shared_prefix(*a.values())


def _abi_weights(**kw):
    a = dict(q=_at(1), k=_at(2), lse=_at(3), w=None, out=_at(4), ws=None, sq_start=_at(5), sk=_at(6), bt=_at(7), stride=2, page=16, batch=2, sq=2, skc=0,
             cols=32, hq=4, hk=2, d=64, qmax=1, ns=1, scale=0.1, wl=-1, wr=-1, mask=0, dtype=4, attrs=None, stream=None)
    a.update(kw)
    return _lib.load().fck_fmha_key_weights(*a.values())


@pytest.mark.parametrize("call,sizes", [
    (_abi_shared, dict(batch=1 << 22, sq=1 << 30, qmax=1 << 30, hq=1 << 11, hk=1)),   # rows of a group: 2^63
    (_abi_shared, dict(batch=1 << 22, sq=1 << 30, qmax=1 << 30, hq=1 << 12, hk=1)),   # 2^64
    (_abi_shared, dict(batch=1 << 30, hq=1 << 30, hk=1 << 30)),
    (_abi_shared, dict(groups=1 << 30, hq=1 << 30, hk=1 << 30)),
    (_abi_weights, dict(batch=1 << 30, hq=1 << 30, hk=1 << 30, cols=1 << 30)),
    (_abi_weights, dict(sq=1 << 30, qmax=1 << 30, hq=1 << 30, hk=1)),
])
def test_abi_sizes_whose_products_leave_64_bits_are_refused(call, sizes):
    assert call(**sizes) == -1
    assert b"beyond 32 bits" in _lib.load().fck_last_error()


def test_abi_choices_for_sizes_whose_products_leave_64_bits():
    lib = _lib.load()
    a, b = ctypes.c_int32(), ctypes.c_int32()
    most = 1 << 24
    for sizes in ((most, most, most, most, 1, most), (1, 1, most, most, 1, 1 << 16), (1, 1, 1, 1, 1, most), (most, most, most, most, most, most)):
        assert lib.fck_fmha_shared_prefix_splits(*sizes, 128, 1 << 20, 1 << 20, 256, ctypes.byref(a), ctypes.byref(b)) == 0
        assert 1 <= a.value <= 64 and 1 <= b.value <= 64, sizes
    for sizes in ((1, most, 1, (1 << 31) - 1, 1 << 20, 256), (1, most, 1, 1 << 30, (1 << 31) - 1, 64)):
        assert lib.fck_fmha_key_weights_row_splits(*sizes, 2, 256) == 1, sizes
    assert lib.fck_fmha_cache_evict_workspace_bytes(1 << 30, 1 << 30, 1 << 20, 256) == 0
    assert lib.fck_fmha_cache_evict_workspace_bytes((1 << 31) - 1, (1 << 31) - 1, 1 << 20, 256) == 0


def test_default_splits_hold_for_a_sequence_without_the_prefix():
    # B, groups, group size, Hq, Hk, tokens, head dim; longest prefix, keys behind it, longest sequence
    for sizes in ((32, 2, 32, 32, 8, 1, 128), (4, 1, 4, 32, 8, 1, 128), (8, 2, 4, 16, 4, 1, 64), (64, 1, 64, 64, 8, 1, 128), (24, 3, 24, 16, 4, 4, 64)):
        batch, _, _, hq, hk, sq, d = sizes
        for prefix, own, longest in ((32768, 232, 33000), (32768, 1, 32768), (512, 64, 576), (1, 4096, 4097)):
            ns = F._default_shared_prefix_splits(*sizes, prefix, own, longest)
            assert all(1 <= n <= 64 for n in ns)
            alone = F.num_splits_heuristic(batch, hq, hk, sq, longest, d)
            assert ns[1] >= min(alone, -(-longest // 2048)), (sizes, prefix, own, longest, ns)


def test_missing_bounds_leave_the_prefix_its_splits(monkeypatch):
    seen, call = [], F._call
    monkeypatch.setattr(F, "_REQUIRE_GPU_TENSORS", False)
    monkeypatch.setattr(F, "_stream", lambda: None)
    monkeypatch.setattr(F, "_call", lambda name, *args: seen.append(args) if name == "fck_fmha_decode_shared_prefix" else call(name, *args))
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    cache = torch.zeros(1, 128, 8, 128, dtype=torch.bfloat16)
    for pages in (64, 256, 1024):
        F.fmha_decode_shared_prefix(torch.zeros(32, 1, 32, 128, dtype=torch.bfloat16), cache, cache, i32(*[5000] * 32),
                                    torch.zeros(32, pages, dtype=torch.int32), i32(4096))
        args = seen[-1]
        # one group of 128 packed rows and 8 KV heads: as many prefix splits as make its items fill the chip, whatever the table addresses
        assert args[21] >= 16 and args[22] >= 2, args[21:23]


def test_an_outgrown_workspace_buffer_stays_allocated():
    # a graph captured with the smaller buffers goes on writing to them
    import gc
    import weakref
    ws, device = F.DecodeWorkspace(), torch.device("cpu")
    ws.partials(2, 4, 3, 1, 64, device)
    ws.lengths(2, device)
    old = [weakref.ref(x) for x in (ws._o_acc, ws._lse_acc, ws._seqlen)]
    o, lse = ws.partials(2, 4, 9, 1, 64, device)
    ws.lengths(5, device)
    gc.collect()
    assert all(x() is not None for x in old) and ws._o_acc is not old[0]()
    # growing one row at a time: what is held stays within a small multiple of what is needed
    for rows in range(1, 400):
        o, lse = ws.partials(1, 4, 8, rows, 64, device)
        assert o.shape == (1, 4, 8, rows, 64) and lse.shape == (1, 4, 8, rows)
    held = sum(x.numel() for x in [ws._o_acc, ws._lse_acc, *ws._outgrown])
    assert held <= 5 * (o.numel() + lse.numel())


def test_a_missing_bound_on_the_groups_takes_them_for_average(monkeypatch):
    seen, call = [], F._call
    monkeypatch.setattr(F, "_REQUIRE_GPU_TENSORS", False)
    monkeypatch.setattr(F, "_stream", lambda: None)
    monkeypatch.setattr(F, "_call", lambda name, *args: seen.append(args) if name == "fck_fmha_decode_shared_prefix" else call(name, *args))
    cache = torch.zeros(1, 64, 8, 128, dtype=torch.bfloat16)
    cu, lens = torch.arange(65, dtype=torch.int32) * 4, torch.full((256,), 1100, dtype=torch.int32)
    for bound in (0, 4, 256, 1000):
        F.fmha_decode_shared_prefix(torch.zeros(256, 1, 32, 128, dtype=torch.bfloat16), cache, cache, lens, torch.zeros(256, 20, dtype=torch.int32),
                                    torch.full((64,), 1024, dtype=torch.int32), cu_groups=cu, max_group_size=bound)
    # no bound, the exact one, and bounds that say nothing: the same splits; the library is told of the exact one only
    assert len({a[21:23] for a in seen}) == 1 and [a[14] for a in seen] == [0, 4, 0, 0]

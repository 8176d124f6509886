"""Refusals and host-side choices of the operators on long shared caches: nothing is launched (no GPU needed)."""
import ctypes

import pytest

from flashck_amd import _lib


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

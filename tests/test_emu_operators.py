"""The GPU tests of the operators on long shared caches, on the wave64 emulator (see test_emu_kernels.py): the unchanged
kernel sources, CPU tensors against guard pages.  By default the cases of QUICK run, with FCK_EMU_FULL=1 all of them
(`FCK_EMU_FULL=1 python -m pytest tests/test_emu_operators.py -n 8`: about two minutes on 8 cores)."""
import importlib
import os

import pytest
import torch

import test_emu_kernels as emu

GPU_MODULES = ["test_gpu_shared_prefix", "test_gpu_key_weights", "test_gpu_cache_evict", "test_gpu_lse"]
# need a real device
NEEDS_DEVICE = {"test_captured_and_replayed", "test_on_another_stream", "test_long_cache_offsets"}

QUICK = {
    "test_emu_shared_prefix__one_group[8-2-64-64-dtype0]", "test_emu_shared_prefix__group_sizes[64-17]",
    "test_emu_shared_prefix__sequences_outside_every_group", "test_emu_shared_prefix__prefix_longer_than_the_sequences",
    "test_emu_shared_prefix__masks[3-128-2-window0]", "test_emu_shared_prefix__masks[1-64-1-window4]",
    "test_emu_shared_prefix__packed_queries_of_different_lengths", "test_emu_shared_prefix__quantised_cache[16-64-dtype0]",
    "test_emu_shared_prefix__padded_head_dims[72-40-64]", "test_emu_shared_prefix__padded_head_dims[8-8-32]",
    "test_emu_shared_prefix__keys_behind_a_sequence_and_foreign_table_entries_do_not_matter",
    "test_emu_shared_prefix__without_an_lse", "test_emu_key_weights__one_token[2-1-8-16-dtype0]",
    "test_emu_key_weights__masks_and_query_runs[3-64-16-2-window1]", "test_emu_key_weights__packed_queries",
    "test_emu_key_weights__accumulates_and_grows[1]", "test_emu_key_weights__quantised_keys[1-64-dtype0]",
    "test_emu_key_weights__cache_without_pages", "test_emu_cache_evict__types_and_shapes[64-16-dtype0]",
    "test_emu_cache_evict__types_and_shapes[72-64-dtype2]", "test_emu_cache_evict__budgets[False-64-30-34]",
    "test_emu_cache_evict__budgets[True-1-0-0]", "test_emu_cache_evict__equal_weights_and_special_values",
    "test_emu_cache_evict__long_rows[1025]", "test_emu_cache_evict__fewer_and_more_columns_than_keys",
    "test_emu_cache_evict__the_whole_sequence", "test_emu_lse__varlen_and_quantised", "test_emu_lse__decode[3]",
    "test_emu_lse__packed_over_pages[64-64]",
}

_mods = [importlib.import_module(m) for m in GPU_MODULES]
for _m in _mods:
    for _name in dir(_m):
        _fn = getattr(_m, _name)
        if _name.startswith("test_") and callable(_fn) and _name not in NEEDS_DEVICE:
            globals()[f"test_emu_{_m.__name__[9:]}__{_name[5:]}"] = _fn
del _fn


@pytest.fixture(autouse=True)
def _quick_set(request):
    if os.environ.get("FCK_EMU_FULL") != "1" and request.node.name not in QUICK:
        pytest.skip("not in the emulator's quick set; FCK_EMU_FULL=1 runs it")


@pytest.fixture(scope="module")
def fmha():
    import ctypes
    import build_emu
    import helpers
    from flashck_amd import _lib
    from flashck_amd.ops import fmha as ops
    from flashck_amd.ops.fmha import fmha as F
    lib = ctypes.CDLL(build_emu.build())
    for name, (res, args) in _lib.SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    saved = (_lib._lib, F._REQUIRE_GPU_TENSORS, F._stream, torch.cuda.synchronize, helpers.DEVICE, [(m, m.dev) for m in _mods])
    _lib._lib, F._REQUIRE_GPU_TENSORS, F._stream = lib, False, (lambda: None)
    torch.cuda.synchronize = lambda *a, **k: None
    helpers.DEVICE = "cpu"
    for m in _mods:
        m.dev = emu._cpu
    try:
        yield ops
    finally:
        _lib._lib, F._REQUIRE_GPU_TENSORS, F._stream, torch.cuda.synchronize, helpers.DEVICE, devs = saved
        for m, d in devs:
            m.dev = d

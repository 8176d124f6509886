"""The GPU tests of the operators' corners and of their kernel instantiations on the wave64 emulator (see test_emu_kernels.py):
the unchanged kernel sources, CPU tensors against guard pages.  By default without the cases of SLOW, with FCK_EMU_FULL=1 all."""
import importlib
import os
import re

import pytest
import torch

import test_emu_kernels as emu

GPU_MODULES = ["test_gpu_operator_edges", "test_gpu_operator_instantiations"]
NEEDS_DEVICE = {"test_a_captured_call_survives_a_workspace_that_grows"}
# seconds each; the other cases reach the same code, or a case that stays in does
SLOW = re.compile(r"mask1|fewer_columns_than_keys\[64-.-.*-(1|40|64|130|199)\]|fewer_columns_than_keys\[64-5|infinity_receives_nothing\[290-2-1-64"
                  r"|instantiations__(?!.*(bf16-64.*(kv8|plain)|fp16-128-160-16-pad|20000-20000))")

_mods = [importlib.import_module(m) for m in GPU_MODULES]
for _m in _mods:
    for _name in dir(_m):
        _fn = getattr(_m, _name)
        if _name.startswith("test_") and callable(_fn) and _name not in NEEDS_DEVICE:
            globals()[f"test_emu_{_m.__name__[9:]}__{_name[5:]}"] = _fn
del _fn
_devs = _mods + [importlib.import_module("test_gpu_cache_evict")]   # whose helper the tests of long rows call


@pytest.fixture(autouse=True)
def _quick_set(request):
    if os.environ.get("FCK_EMU_FULL") != "1" and SLOW.search(request.node.name):
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
    saved = (_lib._lib, F._REQUIRE_GPU_TENSORS, F._stream, torch.cuda.synchronize, helpers.DEVICE, [(m, m.dev) for m in _devs])
    _lib._lib, F._REQUIRE_GPU_TENSORS, F._stream = lib, False, (lambda: None)
    torch.cuda.synchronize = lambda *a, **k: None
    helpers.DEVICE = "cpu"
    for m in _devs:
        m.dev = emu._cpu
    try:
        yield ops
    finally:
        _lib._lib, F._REQUIRE_GPU_TENSORS, F._stream, torch.cuda.synchronize, helpers.DEVICE, devs = saved
        for m, d in devs:
            m.dev = d

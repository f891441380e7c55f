"""The C++ host module of fp8, sampling and paging (csrc/serving_host.cpp), bound to the loaded library's entry points."""
from __future__ import annotations

import ctypes as C

from . import _lib as L

_module = None


def host():
    global _module
    if _module is None:
        try:
            from . import _serving_host as m
        except ImportError as e:
            raise ImportError(f"mingmoe/_serving_host.so is missing or does not load ({e}): build it with "
                              "`python ming-voice_b200/mingmoe/build.py` (or __graft_entry__.build())") from e
        lib = L.lib()
        m.bind(*(C.cast(f, C.c_void_p).value for f in (lib.mv_fp8_linear, lib.mv_fp8_linear_scratch_bytes, lib.mv_sample,
                                                       lib.mv_plan_step)))
        _module = m
    return _module

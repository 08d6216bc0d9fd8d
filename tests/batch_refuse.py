"""Refusals without a GPU: a call that is invalid returns before it touches the device, so it can be made
on a context that has none (zeroed memory of more than a context's size)."""
from __future__ import annotations

import ctypes

from nibblemac_amd.nmx import load_library

HIP = ("hipError", "launch", "hipFunc", "no ROCm", "invalid device")


def refuses(name, what, *args):
    """The call fails with a message of its own, before any call of the runtime."""
    lib = load_library()
    ctx = ctypes.create_string_buffer(4096)
    at = ctypes.cast(ctx, ctypes.c_void_p)
    rc = getattr(lib, name)(at, *[ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args])
    msg = lib.nmx_error(at).decode()
    assert rc == -1 and msg.startswith(name + ":"), (what, rc, msg)
    assert not any(h in msg for h in HIP), (what, msg)

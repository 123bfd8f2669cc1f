"""Build the C++ front end of the fine-tuning operators in-tree: ``gpubridge_b200/lib/gb_ops.so``.

One host-only translation unit (``csrc_torch/gb_ops.cpp``: autograd nodes over the kernels of the
native library) against torch's headers, linked to ``libgpubridge_b200.so`` beside it.  Built like
the ``torch.distributed`` front end (``_build_c10d``), and like it a must on a GPU machine: an
operator on a CUDA tensor builds it on the spot where it is missing, or fails.
"""
from __future__ import annotations

import hashlib
import importlib.util
import os
import sys
import time

from gpubridge_b200.ops import _build

NAME = "gb_ops"
SRC = os.path.join(_build.PKG, "csrc_torch", "gb_ops.cpp")
OUT = os.path.join(_build.LIB_DIR, NAME + ".so")
WORK = os.path.join(_build.OBJ, "ops")
STAMP = OUT + ".stamp"


def _digest() -> str:
    import torch
    with open(SRC, "rb") as fh:
        return hashlib.sha256(fh.read() + torch.__version__.encode()).hexdigest()[:16]


def stale() -> bool:
    """True when the module is missing or was built from another source or another torch."""
    if not (os.path.exists(OUT) and os.path.exists(STAMP)):
        return True
    with open(STAMP) as fh:
        return fh.read().strip() != _digest()


def build(verbose: bool = False) -> str:
    """Compile when the source is newer than the module; returns the module's path."""
    if not os.path.exists(_build.LIB) or stale():
        _build.build()
    if not stale():
        return OUT
    from torch.utils import cpp_extension
    os.makedirs(WORK, exist_ok=True)
    lock = os.path.join(WORK, "lock")          # torch waits for it without a limit; a killed build leaves it behind
    try:
        if time.time() - os.path.getmtime(lock) > 600:
            os.remove(lock)
    except OSError:
        pass
    cpp_extension.load(
        name=NAME, sources=[SRC], with_cuda=True, extra_cflags=["-O2", "-std=c++17"],
        extra_ldflags=[f"-L{_build.LIB_DIR}", "-lgpubridge_b200", "-Wl,-rpath,'$$ORIGIN'",
                       f"-Wl,-rpath,{_build.LIB_DIR}"],
        build_directory=WORK, verbose=verbose, is_python_module=False)
    os.replace(os.path.join(WORK, NAME + ".so"), OUT)
    with open(STAMP, "w") as fh:
        fh.write(_digest())
    return OUT


_module = None


def load():
    """The extension module (built first when missing or stale)."""
    global _module
    if _module is None:
        import torch  # noqa: F401 - libtorch must be loaded before the extension
        from gpubridge_b200.ops import _lib
        _lib.lib()                              # the kernels, from the one place they are loaded
        spec = importlib.util.spec_from_file_location(NAME, build())
        _module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_module)
        sys.modules[NAME] = _module
    return _module


def launches() -> int:
    """Kernels launched through the front end so far (0 where it was never loaded)."""
    return 0 if _module is None else _module.launches()


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv))

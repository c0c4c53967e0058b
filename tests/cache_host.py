"""The cache kernels' arithmetic of single values, compiled for the host from the kernels' headers."""
import ctypes
import os
import subprocess

from tests.conftest import PKG_DIR


def library(source, at):
    """`source` (C++, with the kernels' headers in reach) as a library in the folder `at`."""
    src, lib = str(at / "host.cpp"), str(at / "host.so")
    with open(src, "w") as f:
        f.write(source)
    hipcc = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "bin", "hipcc")
    subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-O1",
                    "-std=c++17", "-ffp-contract=off", "-fPIC", "-shared",
                    "-I" + os.path.join(PKG_DIR, "csrc"), src, "-o", lib], check=True)
    return ctypes.CDLL(lib)

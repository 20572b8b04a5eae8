"""Builds the in-tree native libraries: tierstream_b200/libtierstream.so and libtsb_engine.so (nvcc + g++ for
sm_100a, tierstream_b200/csrc/Makefile), the operators on torch tensors (tierstream_b200/_torch_ops.so), and the checkers
under oracle/ (oracle/Makefile)."""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def _make(directory, extra=()):
    jobs = str(max(1, min(16, os.cpu_count() or 1)))
    subprocess.run(["make", "-j", jobs, *extra], cwd=directory, check=True)


def build(oracle=True):
    _make(os.path.join(HERE, "csrc"))
    import torch
    from torch.utils import cpp_extension
    paths = [p for p in cpp_extension.include_paths("cuda") if os.path.isdir(p)]
    _make(os.path.join(HERE, "csrc"), ["torch", "TORCH_INC=" + " ".join(paths),
                                       "TORCH_LIB=" + os.path.join(os.path.dirname(torch.__file__), "lib"),
                                       "PY_INC=" + sysconfig.get_path("include"),
                                       "TORCH_FLAGS=-D_GLIBCXX_USE_CXX11_ABI=%d" % torch.compiled_with_cxx11_abi()])
    if oracle:
        # the reference checkout beside this repository, when present, for the reference harness
        ref = os.path.normpath(os.path.join(ROOT, "..", "reference"))
        extra = ["REF=" + ref] if os.path.isdir(os.path.join(ref, "src")) else ["REF=/nonexistent"]
        _make(os.path.join(ROOT, "oracle"), extra)


if __name__ == "__main__":
    build(oracle="--no-oracle" not in sys.argv)

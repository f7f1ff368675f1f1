"""Properties of the 8-bit floating point operators and of counter-based dropout that show without a GPU: the order of steps in
a kernel's source, what the package needs to be imported, refusals."""

import os
import shutil
import subprocess
import sys

import approxtorch_b200 as at

PKG = os.path.dirname(os.path.abspath(at.__file__))


def _kernel(source, name, end):
    """The text of one kernel."""
    with open(os.path.join(PKG, "csrc", source)) as f:
        text = f.read()
    start = text.index(f"\n{name}(")
    return text[start:text.index(end, start)]


def test_split_kernel_returns_tensor_memory_before_it_waits_for_its_cluster():
    """tcgen05.alloc has no time limit: a block that holds columns and waits for another block may wait for ever."""
    body = _kernel("fp8_gemm.cu", "fp8_split_kernel", "fp8_bias_kernel")
    alloc, free, wait = body.index("tcgen05.alloc"), body.index("tcgen05.dealloc"), body.index("f8_cluster_sync()")
    assert alloc < free < wait and "barrier.cluster" not in body[:free]


def test_patience_of_the_products_waits():
    from approxtorch_b200.backend import _C
    assert _C.lib.atb_fp8_patience(5) == 1 << 18
    assert _C.lib.atb_fp8_patience(-1) == 5 and _C.lib.atb_fp8_patience(1 << 30) == 1 << 18 and _C.lib.atb_fp8_patience(-1) == 1 << 18


def test_products_fill_what_they_leave_out():
    """Every wait of the two kernels is bounded by the launch's patience or is the wait for what is in flight at the end."""
    import re
    text = _kernel("fp8_gemm.cu", "fp8_gemm_kernel", "// ---- host side")
    calls = re.findall(r"f8_wait(?:<[^(]*>)?\(.*", text)
    assert len(calls) >= 12 and all("patience)" in c for c in calls)
    assert text.count("f8_report(p.error)") == 2


def test_package_works_without_the_native_binding(tmp_path):
    """Where the binding cannot be built (no headers of torch, no host compiler that takes them, another torch), everything that
    goes through the C ABI is there as before, and the operators that need it say why they do not run."""
    for name in ("approxtorch_b200", "include"):
        shutil.copytree(os.path.join(os.path.dirname(PKG), name), tmp_path / name, ignore=shutil.ignore_patterns("_binding.so", "__pycache__"))
    with open(tmp_path / "approxtorch_b200" / "csrc" / "binding" / "binding.cpp", "w") as f:
        f.write("#error no headers\n")
    code = """
import torch, approxtorch_b200 as at
from approxtorch_b200.backend import _C, ops
assert at.__file__.startswith({root!r}) and _C.lib.atb_version() >= 100 and torch.ops.approxtorch is not None
at.nn.Linear_fp8(4, 4)
for call in (lambda: ops.drop_threshold(0.5), lambda: ops.dropout(torch.zeros(3), 0.5, None), lambda: at.nn.gemm_fp8.linear_fp8(None, None)):
    try:
        call()
    except ImportError as e:
        assert "native binding" in str(e), e
    else:
        raise AssertionError("no error")
assert not hasattr(_C, "something else")
print("whole")
""".format(root=str(tmp_path))
    run = lambda *args: subprocess.run([sys.executable, *args], cwd=tmp_path, capture_output=True, text=True)   # noqa: E731
    done = run("-c", code)
    assert done.returncode == 0 and "whole" in done.stdout, done.stderr
    done = run("-m", "approxtorch_b200.build")
    assert done.returncode == 0 and done.stdout.strip().endswith("libapproxtorch_b200.so") and "no counter-based dropout" in done.stderr

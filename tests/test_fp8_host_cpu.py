"""Properties of the 8-bit floating point operators and of counter-based dropout that show without a GPU: the order of steps in
a kernel's source, what the package needs to be imported, refusals."""

import os

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

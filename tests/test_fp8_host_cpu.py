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

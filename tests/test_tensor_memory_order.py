"""Kernels that take tensor memory let the next kernel of the stream in only when they have it.

A kernel that is let in early may become resident beside a CTA that still asks for its tensor memory, take some itself and then wait for that CTA's kernel to
end: if what is left is not enough for it, both wait for good. Nothing here needs a device: the order is read from the source.
"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xn_b200", "csrc")


def _kernels(name):
    """Kernels that take tensor memory: (name, source)."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    parts = re.split(r"__global__", text)[1:]
    return [(re.search(r"(\w+_kernel|\w+)\(const", p).group(1), p) for p in parts if re.search(r"tcgen05\.alloc|tmem_alloc[<(]", p)]


SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu") and "tcgen05.alloc" in open(os.path.join(CSRC, f)).read())


def test_the_kernels_are_found():
    assert {"xnq_imma.cu", "xnq_kv_prompt.cu", "xnq_prefill.cu"} <= set(SOURCES)
    assert all(len(_kernels(f)) == 1 for f in SOURCES)


@pytest.mark.parametrize("name", SOURCES)
def test_tensor_memory_before_the_next_kernel(name):
    for kernel, text in _kernels(name):
        taken = [m.start() for m in re.finditer(r"tcgen05\.alloc|tmem_alloc[<(]", text)]
        let_in = [m.start() for m in re.finditer(r"pdl_launch_dependents\(\)", text)]
        assert let_in and max(taken) < min(let_in) or not let_in, f"{name}: {kernel} lets the next kernel in before it has its tensor memory"
        after = text[max(taken):]
        assert not let_in or after.index("__syncthreads()") < after.index("pdl_launch_dependents()"), f"{name}: {kernel}: the warp that allocates is not waited for"

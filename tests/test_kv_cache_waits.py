"""Kernels of the quantized KV cache are let in while the kernel before them is still at work, so that what that one writes is there for them only behind their own
wait: no fence stands for it, nor another kernel's wait. Nothing here needs a device: the order is read from the source."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xn_b200", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.startswith("xnq_kv_"))


def _text(name):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    return re.sub(r'"(?:[^"\\]|\\.)*"', '""', text)


def _bodies(name):
    """(kernel, what stands between its braces)"""
    out = []
    for part in _text(name).split("__global__")[1:]:
        m = re.search(r"(\w+_kernel)\(", part)
        begin = end = part.index("{", part.index(")", m.end()))
        depth = 0
        while depth or end == begin:
            depth += {"{": 1, "}": -1}.get(part[end], 0)
            end += 1
        out.append((m.group(1), part[begin + 1:end - 1]))
    return out


KERNELS = [(f, k, body) for f in SOURCES if f.endswith(".cu") for k, body in _bodies(f)]


def test_the_kernels_are_found():
    assert {"kv_store_kernel", "kv_load_kernel", "kv_attend_split_kernel", "kv_attend_prompt_kernel", "kv_attend_join_kernel", "kv_attend_join_packed_kernel", "kv_reserve_small_kernel",
            "kv_reserve_clear_kernel", "kv_reserve_mark_kernel", "kv_reserve_give_kernel", "kv_plan_kernel", "kv_plan_trees_kernel", "kv_keep_kernel"} == {k for _, k, _ in KERNELS}


@pytest.mark.parametrize("name,kernel,body", KERNELS, ids=[k for _, k, _ in KERNELS])
def test_every_kernel_waits_whatever_its_arguments_are(name, kernel, body):
    always = [m.start() for m in re.finditer(r"pdl_wait\(\);", body)
              if body[:m.start()].count("{") == body[:m.start()].count("}") and body[:m.start()].rstrip()[-1] in ";{}"]
    assert always, f"{name}: {kernel} does not always wait"
    left = [m.start() for m in re.finditer(r"\breturn\b", body[:always[0]])]
    assert all("pdl_wait();" in body[:at] for at in left), f"{name}: {kernel} ends without having waited"


@pytest.mark.parametrize("name", SOURCES)
def test_nothing_is_read_as_what_never_changes(name):
    """Page tables, plans and pages are written by kernels that overlap the ones that read them: no load through the read-only path, which is for data that nobody
    writes while the kernel lives."""
    found = re.findall(r"__ldg\w*|__restrict__", _text(name)) + re.findall(r"ld\.global[\w.]*\.nc", open(os.path.join(CSRC, name)).read())
    assert not found, (name, found)

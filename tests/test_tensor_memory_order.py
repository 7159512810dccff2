"""A kernel that lets the next ones start before it has its tensor memory may never get it: one of them takes the columns and holds
them while it waits for this kernel, which waits for the columns.  Allocation has no bounded form, so the order of the two is read
from the sources: nothing here makes it happen."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "flyweight_b200" / "csrc"
ALLOC = re.compile(r"\btmem_alloc(_pair)?\(|tcgen05\.alloc")
LET_GO = re.compile(r"\bpdl_(launch_dependents|entry)\(")


def kernels(text):
    """The bodies of a source's kernels, by name, without comments."""
    text = re.sub(r"//[^\n]*", "", text)
    found = {}
    for head in re.finditer(r"__global__", text):
        name = re.compile(r"(\w+)\s*\((?:const )?(?:__grid_constant__|const|\w+[ *&])").search(text, text.index(")", head.end()) + 1)
        start = text.index("{", name.end())
        depth, at = 0, start
        while True:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
            if depth == 0:
                break
        found[name.group(1)] = text[start:at]
    return found


def lets_go_too_early(body):
    alloc, go = ALLOC.search(body), LET_GO.search(body)
    return bool(alloc and go and go.start() < alloc.start())


@pytest.mark.parametrize("source,names", [("attention_prefix_tcgen05.cu", {"prefix_tcgen05_kernel"}),
                                          ("gemm_int8.cu", {"gemm_int8_tile_kernel", "gemm_int8_pair_kernel"})])
def test_tensor_memory_comes_before_the_next_kernel(source, names):
    bodies = kernels((CSRC / source).read_text())
    assert {name for name, body in bodies.items() if ALLOC.search(body)} == names
    assert [name for name in sorted(names) if lets_go_too_early(bodies[name])] == []


def test_the_wrong_order_is_found():
    text = "__global__ void __launch_bounds__(64, 1) k(const int n) { pdl_wait(); %s if (w) { %s } }"
    go, alloc = "pdl_launch_dependents();", "tmem_alloc(at, 256);"
    assert lets_go_too_early(kernels(text % (go, alloc))["k"]) and not lets_go_too_early(kernels(text % (alloc, go))["k"])

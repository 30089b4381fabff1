"""Rules that the CUDA sources keep and that no run can show to be kept: a race may give the right values for years.  Read from the text of
minml_b200/csrc, so it needs no GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(__file__), "..", "minml_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"/\*.*?\*/", " ", re.sub(r"//[^\n]*", " ", text), flags=re.S)


def closing(text, start, pair):
    """Index behind the bracket that closes the one at `start`."""
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == pair[0]) - (text[i] == pair[1])
        if depth == 0:
            return i + 1
    raise AssertionError("unbalanced source")


def kernels(text):
    """(name, parameters, body) of every __global__ function"""
    for m in re.finditer(r"__global__", text):
        head = re.compile(r"\b(kernel_\w+)\s*\(").search(text, m.end())
        if head is None:
            continue
        end = closing(text, head.end() - 1, "()")
        brace = text.index("{", end)
        if text[end:brace].strip():
            continue  # no definition
        yield head.group(1), text[head.end():end - 1], text[brace:closing(text, brace, "{}")]


FILES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


@pytest.mark.parametrize("name", FILES)
def test_overlapped_kernels_read_coherently(name):
    """A kernel that starts under the tail of the one ahead (it calls wait_for_previous_grid) may find memory still being written when it
    begins.  __ldg and pointers that are const and __restrict__ promise memory that nobody writes while the kernel runs: they go through the
    path that is not coherent, and the compiler may move them ahead of the wait."""
    text = source(name)
    found = [k for k in kernels(text) if "wait_for_previous_grid" in k[2]]
    for kernel, parameters, body in found:
        for p in parameters.split(","):
            assert not ("__restrict__" in p and "*" in p), (kernel, p.strip())
    if found:
        assert "__ldg" not in text and "ld.global.nc" not in text
        overlapped = " ".join(body for _, _, body in found)
        for m in re.finditer(r"__device__[^;{]*?\b(\w+)\s*\(([^{;]*?)\)\s*(?:const)?\s*\{", text):
            if re.search(r"\b%s\b" % m.group(1), overlapped):
                assert "__restrict__" not in m.group(2), m.group(1)


def test_the_rule_sees_what_it_is_about():
    text = "__global__ void __launch_bounds__(256) kernel_a(const float *__restrict__ x, int n) { wait_for_previous_grid(); f({ 1 }); } __global__ void kernel_b(int *y) { }"
    found = list(kernels(text))
    assert [k[0] for k in found] == ["kernel_a", "kernel_b"]
    assert "__restrict__" in found[0][1] and found[0][2].endswith("f({ 1 }); }")
    assert sum(len(list(kernels(source(f)))) for f in FILES) > 60


@pytest.mark.parametrize("name", FILES)
def test_arrivals_without_a_cluster_release_report_no_writes(name):
    """arrive_at_leader orders nothing that its thread wrote for the other CTA of the pair; it may only say that accumulators have been read."""
    barriers = re.findall(r"arrive_at_leader\(smem_u32\(&bars\.(\w+)", source(name))
    assert set(barriers) <= {"tmem_empty", "au_empty"}, barriers

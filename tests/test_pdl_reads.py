"""Kernels launched before the kernel ahead of them has ended (pdl.cuh) read no memory through
the read-only path: CUDA allows it only for data that nobody writes while the kernel is
resident, and the compiler may move such a load above the wait. Checked in the sources: a stale
read depends on timing and cannot be provoked on purpose."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kimi-k3-for-me_b200", "csrc")


def code(name):
    """The file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")) and '#include "pdl.cuh"' in code(f))


def test_sources_are_found():
    assert {"head.cu", "topk.cu"} <= set(SOURCES)


@pytest.mark.parametrize("name", SOURCES)
@pytest.mark.parametrize("word", ["__restrict__", "__ldg", "ld.global.nc", "__ldcv"])
def test_no_read_only_loads(name, word):
    at = [i + 1 for i, line in enumerate(code(name).split("\n")) if word in line]
    assert not at, f"{name}: {word} on lines {at} (comments removed)"


@pytest.mark.parametrize("name", SOURCES)
def test_every_kernel_waits_before_it_releases(name):
    """Each __global__ function waits for the kernels before it, then lets the next one start."""
    kernels = re.split(r"__global__", code(name))[1:]
    assert kernels
    for k in kernels:
        body = k[k.index("\n{"):k.index("\n}")]
        assert body.count("pdl_wait();") == 1 and body.count("pdl_release();") == 1, k[:80]
        assert body.index("pdl_wait();") < body.index("pdl_release();")

"""Distributed shared memory may be reached once every CTA of the cluster runs,
and only a cluster barrier says so.  Each kernel that maps another CTA's shared
memory has one before the first use (read off the sources, on the CPU)."""
import os
import re

import pytest

from conftest import REPO

CSRC = os.path.join(REPO, "cuda-repo_b200", "csrc")


def _kernels():
    """(file:name, body without comments) of every kernel."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"__global__", text):
            start = text.index("{", m.end())
            depth, end = 1, start + 1
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            kernel = re.search(r"(\w+_kernel)\s*\(", text[m.end():start]).group(1)
            yield "%s:%s" % (name, kernel), text[start:end]


KERNELS = dict(_kernels())
REMOTE = [k for k, body in KERNELS.items() if "mapa_shared" in body]


def test_kernels_are_found():
    assert len(KERNELS) >= 8
    assert {"quantize.cu:quantize_strips_kernel", "spmm24_kernel.cuh:spmm24_pair_kernel",
            "spmm24_prefill.cuh:spmm24_prefill_int8_kernel"} <= set(REMOTE)


@pytest.mark.parametrize("kernel", REMOTE)
def test_a_cluster_barrier_comes_before_remote_shared_memory(kernel):
    body = KERNELS[kernel]
    barrier = re.search(r"cluster_sync\(\)|cluster_wait_acquire\(\)", body)
    assert barrier and barrier.start() < body.index("mapa_shared")

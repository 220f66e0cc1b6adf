"""CPU, from the kernels' sources: a kernel that takes tensor memory lets its
dependents start (pdl_trigger) only once it has it.

A dependent kernel that takes all of an SM's tensor memory before it waits for
its predecessor would otherwise hold what the predecessor's block on that SM
still waits for, and neither would ever end."""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "parakeet.cpp_b200", "csrc", "kernels")


def kernels():
    """(file, text) of each __global__ function, comments taken out."""
    for name in sorted(os.listdir(SRC)):
        if not name.endswith(".cu"):
            continue
        with open(os.path.join(SRC, name)) as f:
            text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
        parts = re.split(r"\b__global__\b", text)[1:]
        for i, body in enumerate(parts):
            yield "%s:%d" % (name, i), body


TAKES = [(at, body) for at, body in kernels() if re.search(r"\btmem_alloc(_2sm)?\(", body)]


def test_there_are_such_kernels():
    assert {at.split(":")[0] for at, _ in TAKES} >= {"gemm.cu", "attention_tc.cu", "decode_attn_tc.cu"}


@pytest.mark.parametrize("at,body", TAKES, ids=[at for at, _ in TAKES])
def test_dependents_start_after_the_allocation(at, body):
    alloc = re.search(r"\btmem_alloc(_2sm)?\(", body).start()
    # every thread is behind the allocation where the block has met after it
    met = re.search(r"__syncthreads\(\)|cluster_sync\(\)", body[alloc:])
    assert met
    first = re.search(r"\bpdl_trigger\(\)", body)
    assert first is None or first.start() > alloc + met.start(), at

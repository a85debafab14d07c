"""Kernels with tensor memory in a chain of programmatic launches.

A kernel may take its tensor memory before it waits for the kernel ahead. If that
one released its dependents while a block of its own still had to ask for tensor
memory, the two could wait for each other for ever. So every kernel that
allocates does it before it releases; that it cannot be seen to fail (the blocks
of today's kernels do not fit one SM together) is why the order is read from the
source here."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "sm120-norm-fusion-kernels_b200" / "csrc"
ALLOCATE = re.compile(r"\b(?:tmem_alloc(?:_pair)?\(|open_block<)")
RELEASE = re.compile(r"\brelease_downstream_grid\(\)")


def kernels():
    for path in sorted(CSRC.glob("*.cu")):
        for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\s*\([^{;]*\)\s*\{(.*?)\n\}", path.read_text(),
                             re.S):
            if ALLOCATE.search(m[2]):
                yield pytest.param(m[2], id=m[1])


def test_the_kernels_are_found():
    assert {p.id for p in kernels()} >= {"prompt_tc_kernel", "prefix_tc_kernel", "qkv_gemm_kernel",
                                         "qkv_gemm_pair_kernel"}


@pytest.mark.parametrize("body", list(kernels()))
def test_tensor_memory_is_taken_before_dependents_are_released(body):
    assert RELEASE.search(body).start() > max(m.start() for m in ALLOCATE.finditer(body))

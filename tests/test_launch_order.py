"""CPU: the order of two steps at the start of the kernels, read from their sources.  A kernel that tells the next one to start (programmatic
dependent launch) before it holds its tensor memory can wait for ever: the next kernel's block may take the columns first and waits
itself for the end of the kernel in front."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "light-tensor_b200", "csrc")
ALLOCATES = r"\btmem_alloc(?:_pair)?\("
STARTS_NEXT = r"\bgriddep_launch_dependents\(\)"


def kernels():
    """(file, name, body) of every kernel."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__\s+void[^{;]*?\b(\w+_kernel)\s*\(", text):
            at = text.index("{", m.end())
            depth, end = 0, at
            for end in range(at, len(text)):
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                if depth == 0:
                    break
            yield os.path.basename(path), m.group(1), text[at:end]


FOUND = [k for k in kernels() if re.search(ALLOCATES, k[2])]


def test_the_kernels_are_found():
    assert {name for _, name, _ in FOUND} >= {"gemm_tc_kernel", "gemm_tc_pair_kernel", "gemv_kernel", "conv_direct_kernel", "mlp_fused_kernel",
                                              "gemm_small_kernel", "cache_attention_tc_kernel"}


@pytest.mark.parametrize("file,name,body", FOUND, ids=[k[1] for k in FOUND])
def test_the_next_kernel_starts_after_the_allocation(file, name, body):
    calls = [m.start() for m in re.finditer(STARTS_NEXT, body)]
    assert calls, f"{file}: {name} never lets the next kernel start"
    assert min(calls) > re.search(ALLOCATES, body).start(), f"{file}: {name} lets the next kernel start before it holds its tensor memory"

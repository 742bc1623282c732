"""CPU: the codes that bounded waits leave when they run out, read from the sources.  A code names its wait: kernels of different kinds
share none, and no code of one kernel stands at two waits."""
import glob
import os
import re
from collections import Counter

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "light-tensor_b200", "csrc")


def codes():
    """file -> the codes of its waits (0xRSS: role, first slot)."""
    got = {}
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        found = [int(c, 16) for call in re.findall(r"\bwait\w*\([^;]*?0x[0-9A-F]{3,4}u[^;]*?[;{]", text) for c in re.findall(r"\b0x([0-9A-F]{3,4})u\b", call)]
        found += [int(c, 16) for call in re.findall(r"\bmbar_wait\([^;]*;", text) for c in re.findall(r"\b0x([0-9A-F]{3,4})u\b", call)]
        if found:
            got[os.path.basename(path)] = set(found)
    return got


def occurrences(file):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    return Counter(re.findall(r"\b0x[0-9A-F]{3}u\b", text))


def test_kernels_of_different_kinds_share_no_role():
    found = codes()
    kinds = {"ltq_mlp_fused.cu": "chain", "ltq_gemm_small.cu": "small", "ltq_cache_attention_tc.cu": "attention", "ltq_selftest.cu": "selftest"}
    assert set(kinds) < set(found)
    roles = {}
    for file, values in found.items():
        for role in {v >> 8 for v in values}:
            roles.setdefault(role, set()).add(kinds.get(file, "product"))
    assert all(len(k) == 1 for k in roles.values()), {hex(r): k for r, k in roles.items() if len(k) > 1}


def test_a_code_stands_at_one_wait():
    for file in ("ltq_mlp_fused.cu", "ltq_gemm_small.cu", "ltq_cache_attention_tc.cu"):
        twice = [c for c, n in occurrences(file).items() if n > 1]
        assert not twice, (file, twice)


def test_what_is_not_a_wait_has_a_word_of_its_own():
    """Refused arguments of the cache kernels never go into the word of the waits."""
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        for target, value in re.findall(r"atomicCAS\(([^,]+), 0u, ([^)]+)\)", open(path).read()):
            assert value == "code" if not target.endswith("refused") else value.startswith("REFUSED_"), (path, target, value)

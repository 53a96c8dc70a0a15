"""Kernels that are launched while the one before them on the stream still runs (launch_overlapped) look at and write nothing in global memory before they have waited for it:
read in the sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipgpt_b200", "csrc")
# what reaches global memory, as the kernels write it; prefetches of a tensor map's descriptor and addresses taken are not among them
ACCESS = re.compile(r"__ldg\(|__ldcg\(|__stcg\(|atomic\w+\(|load_values|store_values|reinterpret_cast<(?:const )?(?:u?int4|float4|uint2) \*>\(|\b\w+\[[^\]]*\] = ")
SHARED = re.compile(r"__shared__|smem|_s\[|\bs_\w+\[|\bsh\[")


def _kernels():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*|__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", f.read())
        for m in re.finditer(r"__global__[^;{]*?\b(\w+)\s*\(", text):
            open_at = text.find("{", m.end())
            depth, i = 0, open_at
            while True:
                depth += {"{": 1, "}": -1}.get(text[i], 0)
                i += 1
                if depth == 0:
                    break
            body = text[open_at:i]
            if "dependency_wait()" in body:
                yield os.path.basename(path), m.group(1), body


KERNELS = list(_kernels())


def test_some_are_found():
    assert len(KERNELS) > 10


@pytest.mark.parametrize("path,name,body", KERNELS, ids=[f"{p}:{n}" for p, n, _ in KERNELS])
def test_nothing_before_the_wait(path, name, body):
    before = body[:body.index("dependency_wait()")]
    last = before.rstrip().splitlines()[-1] if before.strip() else ""
    assert not re.search(r"\bif\s*\([^)]*\)\s*$", before), f"{path}: {name} waits on a condition: {last}"
    if name == "zero_table_kernel":              # stores zeros beside a kernel that has waited in every block, and reads nothing
        assert not re.search(r"__ldg|__ldcg|load_values|= \*|atomic", body) and all("from_float<G>(0.0f)" in x or "make_uint4(0u, 0u, 0u, 0u)" in x for x in before.splitlines() if re.search(r"\] = ", x))
        return
    for line in before.splitlines():
        if ACCESS.search(line) and not SHARED.search(line):
            raise AssertionError(f"{path}: {name} before its wait: {line.strip()}")

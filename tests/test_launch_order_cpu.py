"""Kernels launched to start before the kernel ahead of them has ended (programmatic stream serialization): what they may do before
their wait, read from the sources. Tensor memory is allocated without a limit on the wait, so two kernels that hold some of it while
one waits for the other's end would never finish."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "grilly2_b200", "csrc")
WAIT = re.compile(r"GQ_GRID_DEP_SYNC\(\)|griddepcontrol\.wait")


def _code(path):
    text = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    return re.sub(r"//[^\n]*", "", text)


def _kernels(text):
    """name -> body of every __global__ function."""
    out = {}
    for m in re.finditer(r"__global__\b", text):
        at = text.index("{", m.end())
        name = re.findall(r"(\w+)\s*\([^()]*(?:\([^()]*\)[^()]*)*\)\s*$", text[m.end():at])[-1]
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        out[name] = text[at:end]
    return out


FILES = sorted(glob.glob(os.path.join(CSRC, "*.cu")))


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_tensor_memory_is_allocated_behind_the_wait(path):
    text = _code(path)
    kernels = _kernels(text)
    for name, body in kernels.items():
        alloc, wait = body.find("tmem_alloc("), WAIT.search(body)
        if alloc < 0 or not wait or wait.start() < alloc:
            continue
        # before its wait: only right behind a kernel of the same call that has none and whose first statement is the wait
        launches = [m.group(1) for m in re.finditer(r"launch_after\(\s*(\w+)", text)]
        assert name in launches, name
        for i, launched in enumerate(launches):
            if launched == name:
                ahead = launches[i - 1] if i else None
                if ahead not in kernels:  # a launcher of its own: its callers launch the conversion first
                    ahead = "x_planes_kernel" if "launch_after(x_planes_kernel" in text else ahead
                assert ahead in kernels and "tmem_alloc(" not in kernels[ahead], (name, ahead)
                assert kernels[ahead].lstrip("{ \n").startswith("GQ_GRID_DEP_SYNC();"), (name, ahead)


def test_the_sources_are_read_as_meant():
    found = {n: b for f in FILES for n, b in _kernels(_code(f)).items()}
    assert {"paged_attn_kernel", "gemv_q4_umma_kernel", "gemv_q4_lanes_kernel", "gemm_i8_q8_kernel", "x_digits_kernel", "x_planes_kernel"} <= set(found)
    body = found["paged_attn_kernel"]
    assert 0 < body.index("GQ_GRID_DEP_SYNC();") < body.index("tmem_alloc(")
    assert not re.search(r"\b(?:c|s)\.\w+\[|request_of|table", body[:body.index("GQ_GRID_DEP_SYNC();")])  # and reads no device memory

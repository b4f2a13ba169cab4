"""CPU: rules that the 4-bit layers, the RMSNorms and the rotary positions keep at their limits."""
import ctypes
import importlib
import os
import re

import pytest
import torch
import torch.nn as nn

PKG = "hunyuan3d-tools_b200"


@pytest.fixture(scope="module")
def lib(build_mod):
    return importlib.import_module(PKG + ".csrc._binding").configure(build_mod.load_library())


# ---- order of the kernels' first steps ------------------------------------------------------
def test_tensor_memory_is_taken_before_the_next_kernel_may_start(build_mod):
    """A dependent kernel takes its tensor memory and then waits for this grid to end; a CTA of this grid that is still
    without would wait for those columns for good.  So no function lets the next kernel start ahead of its allocation, and a
    block-wide barrier lies between the two."""
    csrc = os.path.dirname(build_mod.__file__)
    found = 0
    for name in sorted(f for f in os.listdir(csrc) if f.endswith(".cu")):
        with open(os.path.join(csrc, name)) as f:
            functions = re.split(r"^}", f.read(), flags=re.M)      # a function ends at a brace in the first column
        for body in functions:
            takes = [m.start() for m in re.finditer(r"\btmem_alloc_[12]cta\(", body)]
            starts = [m.start() for m in re.finditer(r"\bpdl_launch_dependents\(\)", body)]
            if not takes or not starts:
                continue
            found += 1
            assert min(starts) > max(takes), f"{name}: the next kernel may start before tensor memory is taken"
            assert "__syncthreads()" in body[max(takes):min(starts)], f"{name}: no barrier behind the allocation"
    assert found == 5

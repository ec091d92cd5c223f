"""The order of loads that a kernel's waits count, in the code of the library built here."""
import os
import re
import shutil
import subprocess

import pytest

from nnr_amd import _lib
from test_kernel_resources import code_objects

OBJDUMP = next((p for p in (shutil.which("llvm-objdump"), "/opt/rocm/llvm/bin/llvm-objdump") if p and os.path.exists(p)), None)


@pytest.fixture(scope="module")
def once_kernel(tmp_path_factory):
    """Instructions of the prompts' kernel that holds keys and values once (fp32, heads of 256, two groups of waves)"""
    if OBJDUMP is None:
        pytest.skip("llvm-objdump is not here")
    with open(_lib.LIB_PATH, "rb") as f:
        data = f.read()
    path = tmp_path_factory.mktemp("code") / "co.elf"
    for image in code_objects(data):
        if b"prompt_kernelILi0ELi256ELi2E" not in image:
            continue
        path.write_bytes(image)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, capture_output=True, text=True).stdout
        found = re.search(r"^\S* ?<\S*prompt_kernelILi0ELi256ELi2E[^>]*>:\n(.*?)(?=^\S* ?<\S+>:\n|\Z)", text, re.M | re.S)
        return [re.sub(r"\s*//.*", "", line).strip() for line in found.group(1).splitlines()]
    raise AssertionError("no such kernel in the library")


def test_first_keys_before_first_values(once_kernel):
    """The first barrier of the tiles' loop waits until 16 loads are left, which are the values': the keys' 16 are all
    asked for before them, through a descriptor of their own."""
    end = next(i for i, x in enumerate(once_kernel) if re.match(r"s_waitcnt vmcnt\(16\) lgkmcnt\(0\)", x))
    assert once_kernel[end + 1].startswith("s_barrier")
    via = [re.search(r"s\[\d+:\d+\]", x).group() for x in once_kernel[:end] if x.startswith("buffer_load_dwordx4") and x.endswith("lds")]
    assert len(via) == 32 and len(set(via[:16])) == 1 and len(set(via[16:])) == 1 and via[0] != via[16], via

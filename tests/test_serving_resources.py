"""The serving operators' kernels keep nothing in scratch memory (their variants are
chosen by what fits in registers). From the metadata of the library built here."""
import re

import pytest

from test_kernel_resources import scratch  # noqa: F401 (a fixture)


@pytest.mark.parametrize("pattern,least", [(r"rotary", 1), (r"kv_copy_pages_kernel", 1), (r"kv_move_tokens_kernel", 8), (r"kv_tree_kernel", 6),
                                           (r"prompt_kernelILi\dELi(64|96|128)E", 18)])
def test_no_scratch(scratch, pattern, least):  # noqa: F811
    found = {n: b for n, b in scratch.items() if re.search(pattern, n)}
    assert len(found) >= least and not any(found.values()), {n: b for n, b in found.items() if b}


def test_prompts_of_wide_heads(scratch):  # noqa: F811
    """Two sets of 128 accumulator registers where a tile holds infinities or NaNs, and
    nothing in scratch memory but those. (96 registers of 4 bytes at most.)"""
    found = {n: b for n, b in scratch.items() if "prompt_kernel" in n and "ELi256E" in n}
    assert len(found) >= 3 and max(found.values()) <= 384, found

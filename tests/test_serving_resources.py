"""The serving operators' kernels keep nothing in scratch memory (their variants are
chosen by what fits in registers). From the metadata of the library built here."""
import re

import pytest

from test_kernel_resources import scratch  # noqa: F401 (a fixture)


@pytest.mark.parametrize("pattern,least", [(r"rotary", 1), (r"kv_copy_pages_kernel", 1), (r"kv_move_tokens_kernel", 8), (r"kv_tree_kernel", 6),
                                           (r"prompt_kernel", 27)])
def test_no_scratch(scratch, pattern, least):  # noqa: F811
    found = {n: b for n, b in scratch.items() if re.search(pattern, n)}
    assert len(found) >= least and not any(found.values()), {n: b for n, b in found.items() if b}

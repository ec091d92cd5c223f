"""The decoder operators' kernels keep nothing in scratch memory (their variants are
chosen by what fits in registers). From the metadata of the library built here."""
import re

import pytest

from test_kernel_resources import scratch  # noqa: F401 (a fixture)


@pytest.mark.parametrize("pattern,least", [(r"kv_attn_kernel", 48), (r"kv_join_kernel", 4), (r"kv_(write|read)_kernel", 48),
                                           (r"nbits_kernel", 100), (r"nbits_tile_kernel", 30), (r"nbits_pack_kernel", 1)])
def test_no_scratch(scratch, pattern, least):  # noqa: F811
    found = {n: b for n, b in scratch.items() if re.search(pattern, n)}
    assert len(found) >= least and not any(found.values()), {n: b for n, b in found.items() if b}

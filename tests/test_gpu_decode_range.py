"""Operators of a decoder's step where ranges, sizes and rows are far apart, against float64."""
import pytest
import torch

import nnr_amd

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("typed", [False, True])
def test_workspace_made_before_the_call(dev, t, typed):
    """A workspace of the size that attention_workspace names serves the call, which
    writes nothing behind it; shapes at which the types' sizes differ."""
    H, hd, page = 8, 128, 64
    for B, S, heads, per, prefix in ((8, 64, 32, 64, 0), (32, 1, 32, 8, 4096)):
        pages = prefix // page + 4
        cache = nnr_amd.KVCache(pages, H, hd, page_size=page)
        td = torch.full((B, per), pages - 1, dtype=torch.int32, device=dev)
        pt = torch.arange(prefix // page, dtype=torch.int32, device=dev)
        lens = torch.full((B,), S, dtype=torch.int32, device=dev)
        k = torch.randn((1, S, H, hd), device=dev).to(t)
        cache.write(k, k, td[:1], lens[:1])
        q = torch.randn((B, S, heads, hd), device=dev).to(t)
        n = cache.attention_workspace(B, S, heads, per, prefix, **(dict(dtype=t) if typed else {}))
        buf = torch.full((n + 4096,), 77, dtype=torch.uint8, device=dev)
        kw = dict(prefix_table=pt, prefix_len=prefix)
        y = cache.attention(q, td, lens, workspace=buf[:n], **kw)
        assert torch.equal(y, cache.attention(q, td, lens, **kw))
        assert (buf[n:] == 77).all()

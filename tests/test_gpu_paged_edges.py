"""The paged cache's calls at the edges of what the header allows: addresses, tables and contents that the shapes in
test_gpu_paged.py do not meet. Cases and tolerances are those of its Case."""
import ctypes

import numpy as np
import pytest

from test_gpu_paged import Case, _half

pytestmark = pytest.mark.gpu


# One sequence over 9,000 tokens and many over a long prefix (tiles in parts, joined by row and by tile; both kernels).
CUT = [(16, 8, 128, [(9000, [(1, 2000)])], 0), (16, 8, 128, [(9000, [(1, 2000)])], 700), (32, 8, 64, [(5000, [(3, 9)] * 12)], 0),
       (32, 8, 64, [(5000, [(40, 90)] * 12), (300, [(70, 70)])], 0), (8, 2, 256, [(4000, [(1, 5), (30, 40)])], 0)]


@pytest.mark.parametrize("heads,kv,D,groups,after", CUT)
@pytest.mark.parametrize("at", [16, 32, 48, 240])
def test_workspace_at_any_multiple_of_16(ctx, dev, heads, kv, D, groups, after, at):
    """Parts are stored 32 bytes at a time; a workspace at 16 past a multiple of 32 serves as any other, and nothing is
    written before or behind it."""
    import torch
    c = Case(ctx, dev, groups, heads, kv, D, 32, after=after, seed=at)
    n = c.ws.numel()
    whole = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=dev)
    lead = -whole.data_ptr() % 256 + at
    c.ws = whole[lead:lead + n]
    torch.cuda.synchronize()
    c.call()
    ctx.sync(60000)
    c.check()
    assert (whole[:lead] == 0xA5).all() and (whole[lead + n:] == 0xA5).all()

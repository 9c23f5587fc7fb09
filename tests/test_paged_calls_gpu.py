"""Calls over the paged cache at the edges of what its interface allows, on the GPU: many pieces to
a warp, against the formulas in 64 bits. The bounds are those of test_paged_gpu.py.
"""
import pytest

import fusor_attn as fa
from test_paged_gpu import CAUSAL, Spans, run_attend, torch_

pytestmark = pytest.mark.gpu

DIMS = [(14, 2, 64), (32, 8, 128), (8, 2, 256)]


@pytest.mark.parametrize("dtype", [fa.Q8, fa.BF16], ids=["q8", "bf16"])
@pytest.mark.parametrize("dims", [(16, 8, 64), (16, 8, 128), (16, 8, 256)], ids=str)
@pytest.mark.parametrize("rows", [3, 40], ids=["tokens", "chunks"])
def test_many_short_pieces_of_a_warp(dims, dtype, rows):
    """Sequences of a few tiles each, so that every warp takes many pieces one after the other:
    each with its own sequence, head and pages."""
    torch = torch_()
    spans = Spans([(1 + (i * 7) % rows if rows < 8 else 20 + (i * 7) % rows, (i * 37) % 150)
                   for i in range(250)], 16)
    cache, batch, q, out = run_attend(fa.Shape(1, *dims), spans, dtype, CAUSAL)
    again = torch.empty_like(out)
    for _ in range(5):
        cache.attend(0, batch, q, again)
        assert torch.equal(again, out)
    fa.device_status()

"""GPU: PagedDecoder where test_gpu_paged_batch.py does not reach."""
from __future__ import annotations

import pytest
import torch

from test_gpu_paged_batch import small_engine

pytestmark = pytest.mark.gpu


def test_prefill_scratch_does_not_grow_with_the_layers(rib):
    """A prompt's rows pass through one layer's scratch: 24 layers take no more memory beside the pool than 2 do.
    A cache of all layers would be 2 x 2 heads x 4096 rows x 128 dims x 2 bytes = 4 MB a layer more."""
    grown = []
    for layers in (2, 24):
        e = small_engine(rib, layers=layers)
        pool = rib.PagePool.for_engine(e, pages=80, page_rows=64)
        d = rib.PagedDecoder(e, pool, slots=1, max_rows=5000)
        d.remove(d.add([1] * 4096))  # first-call set-up
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        d.add(list(range(900)) + [7] * 3196)
        torch.cuda.synchronize()
        grown.append(torch.cuda.max_memory_allocated() - before)
        del d, pool, e
    assert grown[1] <= grown[0] + (4 << 20), grown

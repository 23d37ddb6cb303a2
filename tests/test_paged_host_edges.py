"""CPU: paged-cache calls at the edges of what they take, and the page accounting of PagedDecoder.  No call here
reaches a kernel launch."""
from __future__ import annotations

import pytest

from test_paged_host import EINVAL, FAKE, cache

MOST = 0x7f000000


@pytest.mark.parametrize("keep,new_rows", [(MOST + 1, MOST + 1), (2 ** 31 - 1, 2 ** 31 - 1), (32, MOST + 1),
                                           (32, 2 ** 31 - 1)])
def test_evict_refuses_more_rows_than_its_loops_count(rib, keep, new_rows):
    """A thread of the selection writes every 512th to 8192nd of `keep` rows (and of the score rows behind them),
    counting in 32 bits: for a keep within that many of 2^31 the count would wrap and the thread write far below its
    buffer.  Refused before anything is launched."""
    L = rib.load_library()
    status = L.rib_paged_evict(cache(), FAKE, 2, 2, FAKE, 3, 32, FAKE, 128, 64, keep, 4, 8, FAKE, FAKE, FAKE, 64, 32,
                               new_rows, None)
    assert status == EINVAL


def test_attention_refuses_more_tiles_than_a_run_counts(rib):
    """A CTA counts the tiles of its run in 32 bits. Sequences that share their pages (a table stride of 0) can add up
    to more than the 148 x 2 or x 3 CTAs count: the run's length would wrap, and the join would read records that
    nothing wrote."""
    L = rib.load_library()
    many = cache(seqs=1 << 20, nkv=1 << 10, width=MOST // 256, page_rows=256, table_stride=0)
    status = L.rib_paged_decode_attention(many, FAKE, 1 << 16, 64, FAKE, 1 << 20, 1 << 10, MOST, 0.125, FAKE, None, 0, 0,
                                          None, 0, 0, FAKE, 1 << 40, None)
    assert status == EINVAL


def test_attention_refuses_a_scale_beyond_fp32_in_log2_units(rib):
    """scale * log2 e has to be finite in FP32: beyond it a score of 0 would be 0 times infinity."""
    L = rib.load_library()
    ws = L.rib_paged_decode_workspace_bytes(3, 64, 4, 64, 0)
    for scale in (2.4e38, 3.4e38):
        assert L.rib_paged_decode_attention(cache(), FAKE, 256, 64, FAKE, 3, 4, 64, scale, FAKE, None, 0, 0, None, 0, 0,
                                            FAKE, ws, None) == EINVAL

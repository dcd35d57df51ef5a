"""chunk_attention where its definition is easy to miss: windows of sequences that are longer than
their table."""
import pytest
import torch

from helm_amd.kernels import attention as ka
from test_chunk_attention import Batch


# ── windows and tables ───────────────────────────────────────────────────────

@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(79, 0), (80, 0), (81, 3), (100, 0), (119, 1), (120, 0), (10 ** 9, 5),
                                          (2 ** 31 - 1, 0), (2 ** 40, 0)])
@pytest.mark.parametrize("seqs", [[(100, 20), (100, 1)], [(120, 1), (70, 1), (79, 1), (85, 1)]])
def test_a_window_as_long_as_the_table_hides_keys_of_longer_sequences(seqs, window, sinks):
    """The table ends at token 80, the rows stand behind it: a row at p sees the keys from p - window + 1
    to 79 (equal scores and values of +-1: every key too many or too few shows)."""
    b = Batch((8, 2, 64), 16, seqs, window, sinks, flat=True, spare=0).cuda()
    table = b.d_table[:, :5].contiguous()
    out = torch.full_like(b.d_q, 7.0)
    ka.chunk_attention(b.d_q, b.pool, table, b.d_lens, b.d_starts, 16, window, sinks, out=out)
    b.check(out.cpu(), b.exact(coverage=80))
    if all(k == 1 for _, k in seqs):
        out = ka.window_decode_attention(b.d_q, b.pool, table, b.d_lens, 16, window, sinks)
        b.check(out.cpu(), b.exact(coverage=80))


@pytest.mark.gpu
def test_windows_past_2_to_the_30():
    """No position passes 2^31 - 2: from 2^31 - 1 on a window is none.  Below, up to 2^30 are supported."""
    b = Batch((4, 2, 64), 16, [(5, 2), (0, 1)], flat=True).cuda()
    for window in (2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 63):
        b.window = window
        b.check(b.run(), b.exact())
    for window in (2 ** 30 + 1, 2 ** 31 - 2):
        b.window = window
        with pytest.raises(RuntimeError, match="2\\^30"):
            b.run()

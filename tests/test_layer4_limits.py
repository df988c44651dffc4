"""Where the entry points of a 4-bit cache stop for sizes beyond a launch, on the host."""
import pytest

from test_layer4_refusals import cache4
from test_layer_refusals import F16, INVALID, UNSUPPORTED, refused, seqs, t


@pytest.mark.parametrize("D,most", [(64, 1 << 27), (96, (1 << 27) - 8), (128, (1 << 27) - 8)])
def test_write_limit(mi, D, most):
    """A workgroup of the write has 256 threads for 8 tokens of 96 and 128 elements, 16 of 64, and a grid fewer than 2^32
    threads: the last count that fits and the first that does not."""
    c = cache4(mi, n_head_kv=1, head_dim=D)
    for n, st, text in ((most, INVALID, "null context"), (most + 1, UNSUPPORTED, "launch limits")):
        x = t(mi, F16, [D, n, 1, 3])
        refused(mi, mi.lib().mi355_kv_cache4_write(None, c, seqs(mi), x, x, None), st, text)

"""Attention over the paged 8-bit cache at the limits of its arguments."""
import pytest
import torch

from tests.test_kv_cache_gpu import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [70, 9]])
def test_a_window_that_hides_nothing(device, new):
    """As large as the table, and as 64 bits hold: what a call without a window gives, bit for bit."""
    c = Case(new, [3000, 90], 4, 2, 64, 16, 80)
    want, lse = c.check()
    room = c.table.shape[1] * 16
    for window in (room - 1, room, 1 << 31, 1 << 40, (1 << 62) + 1, (1 << 63) - 1):
        got, lse2 = c.call(window=window)
        c.compare(got, lse2, c.want())
        if window >= room:
            assert torch.equal(got, want) and torch.equal(lse2, lse)
    c.check(window=2999)
    c.check(window=2998)

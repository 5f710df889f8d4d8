"""Shared-prefix attention where a group's start lies below the one before it: nobody shares, whatever the groups' sizes add up to,
and every sequence from the first start to the last is attention over its own pages."""

import numpy as np
import pytest

from tests.test_gpu_shared import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("batch,end", [(4, 3), (70, 68), (1100, 1098)])
def test_a_member_too_short_for_a_group_that_overlaps(dtype, batch, end):
    """Place 1 lies in the first group, whose shared positions it has, and in the range of the third, whose it has not.  The groups'
    sizes add up to no more than the batch."""
    lens = np.full(batch, 100)
    lens[1] = 20

    def edit(table, n_pages):
        table[1, 0] = table[0, 0]  # the first group's shared positions
    c = Case(dtype, 2, 1, 64, 16, lens, [(list(range(batch)), 0)], blind=False, edit=edit)
    c.lists = lambda: (list(range(end)) + [-1] * (batch - end), [0, 2, 1, end], [16, 0, 48])
    c.run(name="starts that go back")


def test_only_the_last_start_goes_back():
    c = Case("float16", 2, 1, 64, 16, [80, 90, 70, 60, 50], [(list(range(5)), 0)], blind=False)
    c.lists = lambda: ([0, 1, 2, 3, -1], [0, 2, 5, 4], [32, 16, 48])
    c.run(name="the last start goes back")

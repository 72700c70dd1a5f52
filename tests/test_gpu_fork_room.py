"""paged_cache_fork_forward: what a row is to write to and has no page for is missing, in pools that are dealt out in one launch and in larger ones; room ends with the table."""
import pytest

from paged_cases import Cache
from test_gpu_tree_pages import check_fork, uses_of

pytestmark = pytest.mark.gpu
SPARE = [60, 17000]                                                           # free pages: counts in LDS, and more than that holds


@pytest.mark.parametrize("spare", SPARE)
def test_a_page_kept_in_part_that_the_source_has_not(spare):
    """The row goes on where it has no page, and says so; pages that are kept whole stay as the source has them."""
    cache = Cache([70, 70], 1, 64, 16, seed=3, spare=spare, width=8)
    cache.table[cache.table >= cache.pool] = -1
    cache.table[0, 4], cache.table[1, 1] = -1, -1
    (table, _, missing), _ = check_fork(cache, uses_of(cache), [0, 0, 1, 1, 0], [70, 64, 70, 20, 70], [80, 80, 80, 40, 100], layers=1)
    assert missing.tolist() == [1, 0, 0, 1, 1]
    assert (table[:, :5] < 0).tolist() == [[False] * 4 + [True], [False] * 5, [False, True, False, False, False], [False, True, False, True, True], [False] * 4 + [True]]


def test_missing_of_a_pool_and_of_a_source_together():
    """Two free pages for rows that want two, one and two, of which the first and the last go on in a page that their source has not."""
    cache = Cache([40, 40, 40], 1, 64, 16, seed=4, spare=3, width=6)
    cache.table[cache.table >= cache.pool] = -1
    cache.table[0, 2] = cache.table[2, 2] = -1                                # (two pages more that nobody holds)
    uses = uses_of(cache)
    uses[[p for p in range(cache.pool) if uses[p] == 0][2:]] = 1
    (table, _, missing), _ = check_fork(cache, uses, [0, 1, 2], [40, 40, 40], [80, 64, 80], layers=1)
    assert missing.tolist() == [1, 1, 3] and (table[:, 2:5] >= 0).tolist() == [[False, True, True], [True, False, False], [False, False, False]]


@pytest.mark.parametrize("spare", SPARE)
def test_room_ends_with_the_table(spare):
    """What is asked for behind a table of four pages is cut off, as it is documented."""
    cache = Cache([35, 16], 1, 64, 16, seed=5, spare=spare, width=4)
    cache.table[cache.table >= cache.pool] = -1
    (table, _, missing), _ = check_fork(cache, uses_of(cache), [0, 1, 0, -1, 1], [35, 16, 2**31 - 1, 0, 16], [64, 65, 0, 2**31 - 1, 0], layers=1)
    assert missing.tolist() == [0] * 5 and (table >= 0).sum(1).tolist() == [4, 4, 3, 4, 1]

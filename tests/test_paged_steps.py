"""A step over a paged cache is good for the rows as they were when it was made: one that would give a row pages of another is refused."""
import pytest
import torch

from helpers import pkg


def cache():
    return pkg().PagedKVCache(8, 16, 2, 64, 3, device="cpu")


def refused(call):
    with pytest.raises(pkg().Ab2Error) as e:
        call()
    assert e.value.status == -7


def test_a_step_is_committed_once():
    c = cache()
    s = c.step([0, 1], [20, 3])
    c.commit(s)
    refused(lambda: c.commit(s))
    assert [c.seq_len(r) for r in range(3)] == [20, 3, 0]
    a, b = c.step([0], [1]), c.step([0], [2])   # of two for the same tokens one
    c.commit(b)
    refused(lambda: c.commit(a))
    c.commit(c.step([0], [1], into=a))
    assert c.seq_len(0) == 23


@pytest.mark.parametrize("length", [0, 5, 20])   # the last frees the step's pages and leaves the length
def test_a_row_that_was_cut_needs_another_step(length):
    c = cache()
    c.commit(c.step([0], [20]))
    s = c.step([0, 1], [30, 1])
    k = torch.zeros(31, 2, 64)
    c.truncate(length, 0)
    other = c.step([2], [60])                   # takes pages that the step's table names
    refused(lambda: c.commit(s))
    refused(lambda: c.append(s, k, k))
    refused(lambda: c.attention(s, k, 1.0))
    assert c.seq_len(0) == length and c.seq_len(1) == 0
    c.commit(other)
    held = [p for row in c._pages for p in row]
    assert len(held) == len(set(held))
    c.clear()
    refused(lambda: c.commit(other))
    c.commit(c.step([0, 1], [1, 1], into=s))    # made anew, it is good again
    assert [c.seq_len(r) for r in range(3)] == [1, 1, 0]


def test_other_rows_may_be_cut():
    c = cache()
    c.commit(c.step([0, 1, 2], [10, 20, 30]))
    s = c.step([0, 1], [1, 1])
    c.truncate(3, 2)
    c.commit(s)
    assert [c.seq_len(r) for r in range(3)] == [11, 21, 3]


def test_a_table_is_never_narrower_than_its_rows():
    c = cache()
    c.commit(c.step([0], [40]))
    with pytest.raises(pkg().Ab2Error):
        c.step([0], [30], room=-60)
    assert c.free_pages() == 8 - 3 and len(c._pages[0]) == 3


def test_a_step_that_a_caller_put_together():
    c = cache()
    made = c.step([0], [5])
    own = pkg().PagedStep(made.rows, made.new, made.table, made.lens, made.starts, made.tokens, made.max_new, made.packed)
    c.truncate(0, 1)
    c.commit(own)
    assert c.seq_len(0) == 5

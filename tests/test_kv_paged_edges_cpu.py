"""Paged KV cache without a GPU, at its edges: steps that are taken back, masks, and calls that are refused before a launch."""
import pytest
import torch

from test_kv_paged_cpu import _cache, _consistent, _run


def _two(lengths=(20, 10)):
    c = _cache(batch=2, pages=9, page=16)
    c.extend(lengths)
    _run(c, max(lengths), positions=2)
    return c


@pytest.mark.parametrize("begun", [False, True])
def test_a_step_that_did_not_run_leaves_no_rows(begun):
    """release and crop while a step is under way (not run at all, or by the first layer only) count the rows before it alone: the
    step's were not written in every layer."""
    for take, want in ((lambda c: c.release(0), [0, 10]), (lambda c: c.crop(-1), [19, 9]), (lambda c: c.crop(0), [20, 10]),
                       (lambda c: c.release([]), [20, 10]), (lambda c: c.truncate([20, 7]), [20, 7]),
                       (lambda c: c.reset(), [0, 0])):
        c = _two()
        c.extend([3, 24])
        if begun:
            c.layers[0].begin(24, False, 2)
        take(c)
        assert c.lengths == want and not c._left and c.new.tolist() == [0, 0]
        assert c.get_seq_length() == max(want) and c.positions(1).tolist() == [[n] for n in want]
        _consistent(c)
        _run(c, 1, positions=2)  # and the next step goes on from there
        assert c.lengths == [n + 1 for n in want]
        _consistent(c)


def test_truncate_refuses_rows_that_were_not_written():
    c = _two()
    c.extend([3, 24])
    for bad in ([21, 10], [20, 34]):
        with pytest.raises(ValueError, match="rows that it has"):
            c.truncate(bad)
    assert c._left and c.lengths == [23, 34]  # refused before anything changed
    _consistent(c)
    _run(c, 24, positions=2)
    c.truncate([21, 34])
    assert c.lengths == [21, 34]
    _consistent(c)

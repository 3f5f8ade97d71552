"""Who appends to a last page that several sequences hold, as tests/pages_ref.py defines it: no
sequence loses a token that it still has, however short the pool."""
import numpy as np
import pytest

import pages_ref


def start(n_pages, page, b, max_pages):
    return (pages_ref.Pages(np.zeros(n_pages, np.int32), np.full((b, max_pages), -1, np.int32), np.zeros(b, np.int32), page),
            pages_ref.Contents(n_pages, page, b))


def take(p, c, name, arg, m):
    if name == "grow":
        _, copies, seq, _, slot = p.grow(arg, m)
        c.grow(copies, seq, slot)
    else:
        for x in (p, c):
            x.trim(arg) if name == "trim" else x.fork(arg, arg.shape[1])
    c.check(p.table, p.lens)


def test_a_sequence_that_is_left_out_keeps_its_tokens():
    """The one that would copy finds no page, a shorter one asks for the page as well."""
    p, c = start(2, 16, 3, 2)
    for name, arg in (("grow", [5, 0, 0]), ("fork", [[0, 0, 0]]), ("grow", [1, 1, 1]), ("fork", [[0, 2, 1]]), ("grow", [0, 1, 1])):
        take(p, c, name, np.array(arg), 9)
    assert p.lens.tolist() == [6, 7, 5] and p.left_out == 1
    p, c = start(1, 16, 3, 2)
    for name, arg in (("grow", [6, 0, 0]), ("fork", [[0, 0, 0]]), ("trim", [9, 0, 3]), ("grow", [1, 0, 1])):
        take(p, c, name, np.array(arg), 9)
    assert p.lens.tolist() == [7, 0, 3] and p.left_out == 1


@pytest.mark.parametrize("seed", range(20))
def test_holders_of_many_lengths(seed):
    rng = np.random.default_rng(seed)
    groups, beams = int(rng.integers(1, 6)), int(rng.integers(2, 6))
    b, m = groups * beams, int(rng.integers(5, 60))
    p, c = start(int(b * rng.choice([0.7, 1, 2])) + 1, 16, b, 4)
    steps = pages_ref.holders_of_many_lengths(rng, b, beams, 16, 4, m, 40)
    next(steps)
    while True:
        try:
            name, arg = steps.send(p.lens)
        except StopIteration:
            break
        take(p, c, name, arg, m)

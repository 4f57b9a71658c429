"""Block tables where the ring of free pages has no room for all that is given back (pages held twice): what is dropped is not counted, so that no page of a table becomes free."""
import numpy as np
import pytest

from oracle import sight as S
from tests.test_gpu_tree import check_tables


def cases():
    """(table, pages, starts, counts, ring, state): pages given back beside others that are taken from a ring with little room or none; small tables, and those of two launches."""
    r = np.random.default_rng(1)
    for B, M in ((1, 4), (3, 7), (8, 64), (2, 2500), (600, 3)):
        for free in (0, 1, 2, 3):  # places that the ring has, or all of them are full
            npages = B * M + 2
            before = np.where(r.random((B, M)) < 0.5, r.integers(0, npages, (B, M)), -1).astype(np.int32)
            starts, counts = r.integers(0, M * 16, B), r.integers(0, 40, B)
            yield before, npages, starts, counts, r.permutation(npages).astype(np.int32), np.array([r.integers(npages), npages - free, 0], np.int32)
    # three tokens' pages taken, two given back, all pages free before
    yield np.array([[3, 2, -1, -1, -1]], np.int32), 8, [64], [16], np.arange(8, dtype=np.int32), np.array([0, 8, 0], np.int32)


def as_lists(before, table, npages, ring, state):
    """The free pages after a call, from its table: those before it, without what was taken, then what was given back, as far as there is room."""
    free = [int(ring[(state[0] + i) % npages]) for i in range(state[1])]
    held = lambda t: (t >= 0) & (t < npages)  # noqa: E731
    given = [int(p) for p in before[held(before) & ~held(table)]]
    taken = int((held(table) & ~held(before)).sum())
    return free[taken:] + given[:npages - len(free)], free[:taken]


def check(before, npages, starts, counts, ring, state, after):
    table, next_ring, next_state, _ = after
    want, taken = as_lists(before, table, npages, ring, state)
    got = [int(next_ring[(next_state[0] + i) % npages]) for i in range(next_state[1])]
    assert got == want and len(got) + len(taken) <= npages
    return len(taken), len(got)


def test_the_oracle_keeps_taken_pages_out_of_the_ring():
    moved = 0
    for before, npages, starts, counts, ring, state in cases():
        for window, sinks in ((20, 0), (40, 17)):
            after = S.tables(before, 16, npages, starts, counts, None, 40, window, sinks, ring, state)
            moved += check(before, npages, starts, counts, ring, state, after)[0]
    assert moved > 100


@pytest.mark.gpu
def test_pages_that_the_ring_has_no_room_for(et):
    for before, npages, starts, counts, ring, state in cases():
        for window, sinks in ((20, 0), (40, 17)):
            for in_place in (False, True):
                check_tables(et, before, 16, npages, starts, counts, None, 40, window, sinks, ring, state, in_place)

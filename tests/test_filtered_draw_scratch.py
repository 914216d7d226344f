"""The draw's scratch on the host: where its pieces begin, and how many bytes it has."""
import ctypes

import pytest

from tlie_amd import ops


@pytest.mark.parametrize("rows,vocab", [(1, 20000), (1, 28000), (3, 20480), (35, 24576), (1, 32000), (7, 50261), (64, 128256), (65, 128256)])
def test_pieces_begin_at_multiples_of_16_bytes(rows, vocab):
    """Classes are read 16 bytes at a time, with an odd number of rows times parts too."""
    parts = ops.draw_parts(rows, vocab)
    starts = (ctypes.c_longlong * 7)()
    ops.library().tlie_draw_scratch(rows, parts, starts)
    lists, states, stats, class_mass, class_count, sums, end = starts
    assert parts > 0 and all(start % 16 == 0 for start in (lists, states, stats, class_mass, class_count)) and sums % 8 == 0
    places = rows * parts
    sizes = [(lists, rows * 2048 * 40), (states, rows * 32), (stats, places * 16), (class_mass, places * 1024 * 8), (class_count, places * 1024 * 4), (sums, places * 8)]
    at = 0
    for start, size in sorted(sizes):
        assert start == at
        at += size
    assert end == at == rows * (ops.DRAW_ROW_BYTES + parts * ops.DRAW_PART_BYTES)


def test_a_scratch_that_does_not_begin_so_is_refused():
    draw = ops._entry("tlie_draw", "piipppppiipppp")
    assert draw(4096, 1, 32000, 4096, 4096, None, None, None, 0, 8, 4096 + 8, 4096, None, None) == -1      # (refused before any launch: no GPU is needed)

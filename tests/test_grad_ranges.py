"""Where the gradient tile's loads of weights and scales end: never past the arrays, whatever
the last step of 64 rows holds.

A block of that step may begin past the last row.  Its scalar offset then has to stay within
the buffer, as the range check subtracts it from the buffer's size; values read there would
meet zeros of d, so that no result can show them.  The ranges are walked on the CPU by the
kernel's own offsets (grad_ranges.cpp)."""

import random

import pytest

import host_program


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_loads_end_with_the_matrix(bits, gs):
    rng = random.Random(1000 * bits + gs)
    shapes = [(n, gs * k) for n in (*range(1, 140), 9001, 17408) for k in (1, 5)]
    shapes += [(rng.randint(1, 5000), gs * rng.randint(1, 8192 // gs)) for _ in range(40)]
    # the longest rows of few, and the most rows: the last sizes taken, the first refused
    row = 2 ** 31 // 64 * 8 // bits
    shapes += [(n, row - gs) for n in (1, 2, 63, 64)]
    refused = [(1, row), (64, row), (65, row // 2), (2, 2 ** 28)]
    lines = host_program.run("grad_ranges.cpp", [f"{bits} {gs} {n} {k}" for n, k in shapes + refused])
    for shape, line in zip(shapes, lines):
        assert line == "1 0 0 1", (shape, line)
    for shape, line in zip(refused, lines[len(shapes):]):
        assert line.split()[0] == "0", (shape, line)

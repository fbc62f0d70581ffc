"""Where the gated few-row kernel's loads of weights and scales end (never past the arrays, of
which every byte is read), and that its LDS fits, walked on the CPU by the kernel's own
offsets (glu_ranges.cpp)."""

import random

import pytest

import host_program


@pytest.mark.parametrize("gs", [32, 64, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_loads_end_with_the_matrix(bits, gs):
    rng = random.Random(1000 * bits + gs)
    shapes = [(n, gs * k) for n in (1, 7, 8, 9, 130) for k in (1, 2, 3, 5, 8, 9, 16)]
    shapes += [(rng.randint(1, 300), gs * rng.randint(1, 8192 // gs)) for _ in range(30)]
    shapes += [(8, 65536), (3, 131072 + gs)]
    lines = host_program.run("glu_ranges.cpp", [f"{bits} {gs} {n} {k}" for n, k in shapes])
    for shape, line in zip(shapes, lines):
        past, read, lds = map(int, line.split())
        assert past == 0 and read == 1 and 0 < lds < 160 * 1024, (shape, line)

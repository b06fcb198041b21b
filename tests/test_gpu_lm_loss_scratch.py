"""Scratch of the cross entropy calls against the bounds that their
descriptions give (the queries alone: nothing is allocated)."""
import random

import pytest

pytestmark = pytest.mark.gpu

MB = 1 << 20


def up(n, m):
    return -(-n // m) * m


def copies(rows, vocab, width, x_ld, w_ld):
    """What operands that cannot be read in place take, rows rounded up to 16 bytes."""
    one = up(width, 8) * 2
    return (rows * one + 256 if rows > 1 and x_ld % 8 else 0) + (vocab * one + 256 if vocab > 1 and w_ld % 8 else 0)


def shapes():
    rng = random.Random(5)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
    fixed = [(1, 1, 1), (16, 32768, 4096), (8192, 131072, 4096), (4096, 131072, 4608), (4096, 131072, 4096), (65536, 131072, 4096),
             (65537, 131072, 4096), (777, 50001, 1150), (8192, 131072, 4095), (1 << 23, 1 << 20, 64), (1 << 24, 4096, 8),
             (128, 1 << 24, 512), (129, 1 << 24, 512), (1024, 131072, 4096)]
    return fixed + [(log(1, 1 << 20), log(1, 1 << 20), log(1, 1 << 14)) for _ in range(1500)]


def test_scratch_is_as_documented(cuda):
    from bafe_b200._binding import lib
    for rows, vocab, width in shapes():
        for ld in (up(width, 8), up(width, 8) + 1):
            query = lambda gradient: lib.bafe_cuda_linear_cross_entropy_workspace(None, ld, None, ld, rows, vocab, width, gradient)
            more = copies(rows, vocab, width, ld, ld)
            need = query(0)
            sums = 1 * MB if rows <= 128 else min(16 * rows * -(-vocab // 256), 128 * MB + 16 * rows) + 4 * rows
            assert 0 < need <= more + sums + 1024, (rows, vocab, width, need)
            need = query(1)
            sums = max(1024 * MB if rows * width < 20 * 10 ** 6 else 0, 4 * rows * up(width, 4))
            g = min(2 * rows * up(vocab, 64), max(512 * MB, 8192 * rows))
            assert 0 < need <= more + g + sums + 1024, (rows, vocab, width, need)
